// fast_math.cuh -- building blocks of the attention-weight kernels: exponentials of packed
// score pairs, and TMEM loads that overlap with them.
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

// Two floats in a register pair.  Values that come from consecutive registers (a TMEM load)
// and constants packed once outside a loop cost no moves.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float lo, float hi)
{
    f32x2 d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
    return d;
}
__device__ __forceinline__ void unpack2(f32x2 v, float &lo, float &hi)
{
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c)
{
    f32x2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b)
{
    f32x2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ f32x2 exp2_2(f32x2 x)
{
    float a, b;
    unpack2(x, a, b);
    return pack2(fast_exp2f(a), fast_exp2f(b));
}

// 2^x for a pair on the FMA pipe: n = round(x) by adding 1.5 * 2^23, f = x - n in [-1/2, 1/2],
// 2^f from a degree-5 polynomial, n added to the exponent field.  The polynomial is the minimax
// one for relative error, fitted here by Lawson's reweighted least squares: 7.5e-8 off,
// 1.55e-7 with its coefficients rounded to fp32 (the constant is a step above 1), 2.1e-7 with the
// roundings of its evaluation, on a par with ex2.approx.  x outside [-126, 127] counts as
// the nearer end; NaN gives the largest finite float, which no sum of probabilities reaches.
__device__ __forceinline__ float clamp_exp(float x)
{
    float y;
    asm("max.NaN.f32 %0, %1, 0fC2FC0000;" : "=f"(y) : "f"(x));   // -126
    asm("min.NaN.f32 %0, %1, 0f42FE0000;" : "=f"(y) : "f"(y));   // 127
    return y;
}
__device__ __forceinline__ f32x2 both(float c) { return pack2(c, c); }
__device__ __forceinline__ f32x2 exp2_2_poly(f32x2 x)
{
    constexpr float kMagic = 12582912.0f;
    float a, b;
    unpack2(x, a, b);
    x = pack2(clamp_exp(a), clamp_exp(b));
    const f32x2 j = add2(x, both(kMagic));
    const f32x2 f = fma2(add2(j, both(-kMagic)), both(-1.f), x);
    f32x2 p = fma2(both(0x1.5c08e4p-10f), f, both(0x1.3d0c52p-7f));
    p = fma2(p, f, both(0x1.c6b6e4p-5f));
    p = fma2(p, f, both(0x1.ebf918p-3f));
    p = fma2(p, f, both(0x1.62e428p-1f));
    p = fma2(p, f, both(0x1.000002p+0f));
    float p0, p1, j0, j1;
    unpack2(p, p0, p1);
    unpack2(j, j0, j1);
    return pack2(__uint_as_float(__float_as_uint(p0) + (__float_as_uint(j0) << 23)),
                 __uint_as_float(__float_as_uint(p1) + (__float_as_uint(j1) << 23)));
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
