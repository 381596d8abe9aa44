// fast_math.cuh -- exponentials of the attention-weight kernels to fp32 accuracy, on both
// pipes that can compute them, and TMEM loads that overlap with them.
#pragma once

#include "b200_common.cuh"

namespace smolb200 {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float fast_exp2f(float x)   // MUFU: 16 a clock and SM, error 2^-22
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// d = a * b + c and d = a + b for pairs of floats (f32x2: twice the rate of scalar FMA).
__device__ __forceinline__ void pair_fma(float &d0, float &d1, float a0, float a1, float b0, float b1, float c0,
                                         float c1)
{
    asm("{\n\t.reg .b64 a, b, c, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d0), "=f"(d1)
        : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void pair_add(float &d0, float &d1, float a0, float a1, float b0, float b1)
{
    asm("{\n\t.reg .b64 a, b, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d0), "=f"(d1)
        : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}

// 2^x for a pair on the FMA pipe: n = round(x) by adding 1.5 * 2^23, f = x - n in
// [-1/2, 1/2], 2^f from a degree-5 polynomial fitted for relative error (7.5e-8; 2.1e-7
// with its fp32 roundings, as ex2.approx), n added to the exponent.  x below -126 counts as
// -126, so what should vanish is at most 2^-126; x must not exceed 127.
__device__ __forceinline__ void pair_exp2_poly(float x0, float x1, float &e0, float &e1)
{
    constexpr float kMagic = 12582912.0f;
    x0 = fmaxf(x0, -126.f);
    x1 = fmaxf(x1, -126.f);
    float j0, j1, n0, n1, f0, f1, p0, p1;
    pair_add(j0, j1, x0, x1, kMagic, kMagic);
    pair_add(n0, n1, j0, j1, -kMagic, -kMagic);
    pair_fma(f0, f1, n0, n1, -1.f, -1.f, x0, x1);
    pair_fma(p0, p1, 0x1.5c08e4p-10f, 0x1.5c08e4p-10f, f0, f1, 0x1.3d0c52p-7f, 0x1.3d0c52p-7f);
    pair_fma(p0, p1, p0, p1, f0, f1, 0x1.c6b6e4p-5f, 0x1.c6b6e4p-5f);
    pair_fma(p0, p1, p0, p1, f0, f1, 0x1.ebf918p-3f, 0x1.ebf918p-3f);
    pair_fma(p0, p1, p0, p1, f0, f1, 0x1.62e428p-1f, 0x1.62e428p-1f);
    pair_fma(p0, p1, p0, p1, f0, f1, 0x1.000002p+0f, 0x1.000002p+0f);
    e0 = __uint_as_float(__float_as_uint(p0) + (__float_as_uint(j0) << 23));
    e1 = __uint_as_float(__float_as_uint(p1) + (__float_as_uint(j1) << 23));
}

// 16 consecutive 32-bit TMEM columns (lane addressing as tmem_ld32), and the wait for every
// load of this thread; the wait names the registers, so no use of them moves above it.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait16(uint32_t (&r)[16])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}

// f(first column, 16 values) for `n16` groups of 16 columns from taddr on, the next group's
// load in flight during each call.
template <typename F>
__device__ __forceinline__ void for_columns(uint32_t taddr, int n16, F &&f)
{
    uint32_t a[16], b[16];
    tmem_ld16(taddr, a);
    tmem_wait16(a);
#pragma unroll 1
    for (int i = 0; i < n16; i += 2) {
        tmem_ld16(taddr + i * 16 + 16, b);
        f(i * 16, a);
        tmem_wait16(b);
        if (i + 1 >= n16) break;
        tmem_ld16(taddr + (i + 2 < n16 ? i * 16 + 32 : 0), a);
        f(i * 16 + 16, b);
        tmem_wait16(a);
    }
}

}  // namespace smolb200
