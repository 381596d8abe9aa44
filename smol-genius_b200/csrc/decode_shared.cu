// decode_shared.cu -- single-token decode over a pooled cache with rows that many
// sequences share, and with each key's attention probability added to a running weight.
//
// For query head h of sequence b, over the visible keys j of its shared prefix and its
// own rows:  x_j = scale * q.k_j (capped),  out = sum_j e^(x_j - m) v_j / sum_j e^(x_j - m).
// The sums split over any partition of the keys, each part with its own m, so three
// kernels do one step:
//   prefix  the rows of a shared prefix against the query heads of ALL its sequences, on
//           tcgen05: a 128-row tile holds (sequence, head of the KV group) pairs, so a
//           prefix row is read once per tile instead of once per sequence;
//   split   every sequence's own rows (mma.sync over a TMA ring, keys as the M dimension);
//           with weights it also keeps the scores of the own keys;
//   merge   combines the parts of a row and, with weights, adds
//           sum_h e^(x_hj - M_h) / L_h to the weight of own key j.
//
// Precision.  Scores, maxima, sums and outputs of the parts are fp32.  K is bf16 and V
// fp16 in the cache.  fp32 queries enter the bf16 products as three bf16 terms (24 bits:
// two left the scores 4e-6 off), bf16 queries as they are.  The probabilities multiply V
// as fp16: one term (2^-12) where the output is rounded to bf16 (2^-9) anyway, the value
// and its remainder (2^-23) where the output is fp32.
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <mutex>

#include "b200_common.cuh"
#include "runtime.h"

namespace smolb200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kSms = 148;

struct SharedParams {
    CUtensorMap tk, tv;             // [pool_rows, kv_dim], boxes of 64 columns
    const void *q;                  // [n_seqs, n_heads*hd] fp32 or bf16
    const int64_t *prefix_row0;
    const int *prefix_len, *prefix_seq0;
    const int64_t *seq_row0;
    const int *kv_len;
    float *part_o;                  // [n_seqs*n_heads][slots][hd]
    float2 *part_ml;                // [n_seqs*n_heads][slots]: reference point (log2 units), sum
    float *scores;                  // [n_seqs*n_kv_heads][score_rows][score_cols], log2 units; NULL: not kept
    void *out;
    const float *weights_in;
    float *weights_out;
    long long weights_stride;
    unsigned *err;
    int q_is_bf16, out_is_bf16;
    int n_seqs, n_heads, n_kv_heads, group, n_qgroups;
    int n_prefixes, max_prefix_len, max_prefix_seqs;
    int prefix_chunk, prefix_slots; // keys of one prefix part; parts of the longest prefix
    int chunk, max_chunks;          // the same for own rows
    int slots;                      // prefix_slots + max_chunks
    int max_kv_len, score_rows, score_cols;
    int window;
    float scale, softcap;
};

__device__ __forceinline__ float fast_exp2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// x0, x1 as TERMS packed bf16 pairs whose sum is x to 8*TERMS bits.
template <int TERMS>
__device__ __forceinline__ void split_bf16(float x0, float x1, uint32_t (&t)[TERMS])
{
#pragma unroll
    for (int i = 0; i < TERMS; ++i) {
        t[i] = pack_bf16x2(x0, x1);
        x0 -= bf16lo_f32(t[i]);
        x1 -= bf16hi_f32(t[i]);
    }
}

// p0, p1 as fp16: the rounded pair and what the rounding left.
__device__ __forceinline__ void split_f16(float p0, float p1, uint32_t &hi, uint32_t &lo)
{
    hi = pack_f16x2(p0, p1);
    const __half2 h = *reinterpret_cast<const __half2 *>(&hi);
    lo = pack_f16x2(p0 - __low2float(h), p1 - __high2float(h));
}

// Sequences [s0, s1) of prefix g and its length, clipped to what the host announced
// (kErrBadArgs is flagged where that cuts something off).
__device__ __forceinline__ void prefix_range(const SharedParams &p, int g, int &s0, int &s1, int &len, bool flag)
{
    s0 = p.prefix_seq0[g];
    s1 = p.prefix_seq0[g + 1];
    len = p.prefix_len[g];
    bool bad = s0 < 0 || s1 > p.n_seqs || len < 0 || len > p.max_prefix_len;
    s0 = max(s0, 0);
    s1 = min(s1, p.n_seqs);
    len = min(max(len, 0), p.max_prefix_len);
    if (s1 - s0 > p.max_prefix_seqs) {
        s1 = s0 + p.max_prefix_seqs;
        bad = true;
    }
    if (bad && flag) atomicOr(p.err, kErrBadArgs);
}

// Own keys [ks, n) of sequence b that are visible; n is clipped to max_kv_len.
__device__ __forceinline__ void own_range(const SharedParams &p, int b, int &ks, int &n)
{
    n = min(max(p.kv_len[b], 0), p.max_kv_len);
    ks = (p.window > 0 && n > p.window) ? n - p.window : 0;
}

// ===========================================================================
// prefix
// ===========================================================================
// CTA = (query tile, KV head and chunk of keys, prefix): softmax warpgroups of one packed
// row per thread (thread = TMEM lane), a TMA producer warp and a tcgen05 issuer warp.
//   S = Q K^T  (QT bf16 terms of Q, fp32 in TMEM, two buffers)
//   P = 2^(S*scale*log2e - m) as PT fp16 terms over S's columns
//   O += P V
// Head dims 64 and 128 run two softmax warpgroups on alternate key tiles, each with an O
// and a reference point of its own, joined at the end: the exponentials of a tile take
// longer than its products (one warpgroup left the tensor pipe 34 % busy).  Head dim 256,
// whose O fills half of TMEM, runs one.
// Row r of tile t is query head (r' % group) of sequence s0 + r'/group, r' = 128 t + r.
constexpr int kBM = 128;
constexpr float kMoveLog2 = 8.0f;

template <int HD, int QT>
struct PrefixShape {
    // Key tile: 128; 64 / 32 where the query terms of head dim 256 (64 KB each) leave less room.
    static constexpr int BN = HD == 256 ? (QT == 3 ? 32 : 64) : 128;
    static constexpr int kStages = HD == 256 && QT == 3 ? 1 : 2;
    static constexpr int kSub = HD / 64;
    static constexpr int kQSubBytes = kBM * 128;
    static constexpr int kQTermBytes = kSub * kQSubBytes;
    static constexpr int kKvSubBytes = BN * 128;
    static constexpr int kKvBytes = kSub * kKvSubBytes;
    static constexpr int kOffK = QT * kQTermBytes;
    static constexpr int kOffV = kOffK + kStages * kKvBytes;
    static constexpr int kOffBar = kOffV + kStages * kKvBytes;
    static constexpr int kUsed = kOffBar + 256 + 1024;
    static_assert(kUsed <= 227 * 1024, "shared memory");
    // one CTA per SM: each allocates all 512 TMEM columns
    static constexpr int kSmemBytes = kUsed > 118 * 1024 ? kUsed : 118 * 1024;
    static constexpr int kGroups = HD == 256 ? 1 : 2;   // softmax warpgroups
    static constexpr int kSoftmax = kGroups * kBM;
    static constexpr int kThreads = kSoftmax + 64;
    static constexpr int kTmO = 2 * BN;                 // O of warpgroup w at kTmO + w * HD
    static constexpr int kTmCols = 512;
    static_assert(kTmO + kGroups * HD <= kTmCols, "TMEM");
};

struct PrefixBars {
    uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_done[2], o_final, mma_done;
    uint32_t tmem_base;
    int lo_min;
};

template <int HD, int QT, int PT>
__global__ void __launch_bounds__(PrefixShape<HD, QT>::kThreads, 1) prefix_kernel(const __grid_constant__ SharedParams p)
{
    using S = PrefixShape<HD, QT>;
    constexpr int BN = S::BN, ST = S::kStages, NG = S::kGroups;
    constexpr int kProducer = NG * 4, kIssuer = kProducer + 1;
    static_assert(sizeof(PrefixBars) <= 256, "barriers");
    griddep_wait();
    griddep_trigger();
    const int qt = blockIdx.x;
    const int kvh = blockIdx.y / p.prefix_slots, c = blockIdx.y % p.prefix_slots;
    const int g = blockIdx.z;
    int s0, s1, plen;
    prefix_range(p, g, s0, s1, plen, threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0);
    if (s1 <= s0 || qt * kBM >= (s1 - s0) * p.group) return;   // no rows in this tile

    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    PrefixBars *bars = reinterpret_cast<PrefixBars *>(smem + S::kOffBar);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

    // this softmax thread's packed row and its first visible prefix key
    const int pr = qt * kBM + static_cast<int>(threadIdx.x) % kBM;
    const int b = s0 + pr / p.group, head = kvh * p.group + pr % p.group;
    const bool row_valid = warp < kProducer && b < s1;
    int lo = 0;
    if (row_valid && p.window > 0) {
        int ks, n;
        own_range(p, b, ks, n);
        lo = max(0, plen + n - p.window);
    }
    if (threadIdx.x == 0) {
        bars->lo_min = plen;
        mbar_init(smem_u32(&bars->q_full), S::kSoftmax);
        for (int s = 0; s < 2; ++s) {
            mbar_init(smem_u32(&bars->k_full[s]), 1);
            mbar_init(smem_u32(&bars->k_empty[s]), 1);
            mbar_init(smem_u32(&bars->v_full[s]), 1);
            mbar_init(smem_u32(&bars->v_empty[s]), 1);
            mbar_init(smem_u32(&bars->s_full[s]), 1);
            mbar_init(smem_u32(&bars->p_full[s]), kBM);
            mbar_init(smem_u32(&bars->o_done[s]), 1);
        }
        mbar_init(smem_u32(&bars->o_final), 1);
        mbar_init(smem_u32(&bars->mma_done), 1);
        fence_mbar_init();
    }
    __syncthreads();
    if (row_valid && lo < plen) atomicMin(&bars->lo_min, lo);
    __syncthreads();
    // keys of this part: the chunks count from the first key any row of the tile sees
    const int key_lo = bars->lo_min + c * p.prefix_chunk;
    const int key_hi = min(plen, key_lo + p.prefix_chunk);
    const int n_tiles = key_hi > key_lo ? (key_hi - key_lo + BN - 1) / BN : 0;
    const long long slot = (static_cast<long long>(b) * p.n_heads + head) * p.slots + c;
    if (n_tiles == 0) {
        if (row_valid && threadIdx.x < kBM) p.part_ml[slot] = make_float2(-INFINITY, 0.f);
        return;
    }
    const long long row_base = p.prefix_row0[g] + key_lo;

    if (warp == kIssuer) {
        tmem_alloc(smem_u32(&bars->tmem_base), S::kTmCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bars->tmem_base;
    uint8_t *sK = smem + S::kOffK;
    uint8_t *sV = smem + S::kOffV;

    if (warp == kProducer) {
        // ================= TMA producer =================
        if (lane == 0) {
            tma_prefetch_desc(&p.tk);
            tma_prefetch_desc(&p.tv);
            int nk = 0, nv = 0;   // K and V tiles issued
            auto load = [&](bool is_v, int j) -> bool {
                const int st = j % ST;
                const uint32_t full = smem_u32(is_v ? &bars->v_full[st] : &bars->k_full[st]);
                const uint32_t empty = smem_u32(is_v ? &bars->v_empty[st] : &bars->k_empty[st]);
                if (j >= ST && !mbar_wait(empty, (j / ST - 1) & 1, p.err, kErrWaitTmaEmpty)) return false;
                mbar_arrive_expect_tx(full, S::kKvBytes);
                uint8_t *dst = (is_v ? sV : sK) + st * S::kKvBytes;
#pragma unroll
                for (int sub = 0; sub < S::kSub; ++sub)
                    tma_load_2d(smem_u32(dst + sub * S::kKvSubBytes), is_v ? &p.tv : &p.tk, full, kvh * HD + sub * 64,
                                static_cast<int>(row_base + j * BN));
                return true;
            };
            bool ok = true;
            for (int j = 0; j < n_tiles && ok; ++j) {   // K runs one tile ahead of V
                if ((ok = load(false, j))) ++nk;
                if (ok && j >= 1 && (ok = load(true, j - 1))) ++nv;
            }
            if (ok && load(true, n_tiles - 1)) ++nv;
            for (int j = max(0, nk - ST); j < nk; ++j)
                if (!mbar_wait(smem_u32(&bars->k_full[j % ST]), (j / ST) & 1, p.err, kErrDrain)) break;
            for (int j = max(0, nv - ST); j < nv; ++j)
                if (!mbar_wait(smem_u32(&bars->v_full[j % ST]), (j / ST) & 1, p.err, kErrDrain)) break;
        }
    } else if (warp == kIssuer) {
        // ================= tcgen05 issuer (converged warp, one elected lane issues) =================
        constexpr uint32_t idesc_s = umma_idesc_f16(kBM, BN, true, false);
        constexpr uint32_t idesc_pv = umma_idesc_f16(kBM, HD, false, true);
        const uint32_t q_addr = smem_u32(smem);
        auto issue_pv = [&](int j) -> bool {
            const int st = j % ST, sb = j & 1;
            // the softmax threads waited for V(j) themselves before they arrived here
            if (!mbar_wait_warp(smem_u32(&bars->p_full[sb]), (j >> 1) & 1, p.err, kErrWaitSoftmax)) return false;
            if (!mbar_wait_warp(smem_u32(&bars->v_full[st]), (j / ST) & 1, p.err, kErrWaitTmaFull)) return false;
            tc_fence_after();
            const uint32_t v_addr = smem_u32(sV + st * S::kKvBytes);
#pragma unroll
            for (int t = PT - 1; t >= 0; --t)   // the remainders first: the smaller sums
#pragma unroll
                for (int kk = 0; kk < BN / 16; ++kk) {
                    const uint64_t bd = umma_sdesc_sw128(v_addr + kk * 16 * 128, S::kKvSubBytes, 1024);
                    // columns of P: see the softmax (32-key groups: 16 of values, 16 of remainders)
                    umma_ts_elect(tmem + S::kTmO + (j % NG) * HD, tmem + sb * BN + (kk >> 1) * 32 + t * 16 + (kk & 1) * 8, bd,
                                  idesc_pv, (j >= NG || t < PT - 1 || kk > 0) ? 1u : 0u);
                }
            umma_commit_elect(smem_u32(&bars->o_done[j % NG]));
            umma_commit_elect(smem_u32(&bars->v_empty[st]));
            return true;
        };
        bool ok = mbar_wait_warp(smem_u32(&bars->q_full), 0, p.err, kErrWaitSoftmax);
        // Two warpgroups: P V of tile j - 2, whose P lies in the buffer of S(j), goes before
        // S(j).  One: S(j) goes first, so that it runs during the softmax of tile j - 1.
        for (int j = 0; j < n_tiles && ok; ++j) {
            const int st = j % ST;
            if (NG == 2 && j >= 2 && !(ok = issue_pv(j - 2))) break;
            if (!(ok = mbar_wait_warp(smem_u32(&bars->k_full[st]), (j / ST) & 1, p.err, kErrWaitTmaFull))) break;
            tc_fence_after();
            const uint32_t k_addr = smem_u32(sK + st * S::kKvBytes);
            const uint32_t s_col = tmem + (j & 1) * BN;
#pragma unroll
            for (int t = QT - 1; t >= 0; --t)
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk) {
                    const uint32_t off = (kk & 3) * 32;
                    const uint64_t ad =
                        umma_sdesc_sw128(q_addr + t * S::kQTermBytes + (kk >> 2) * S::kQSubBytes + off, 16, 1024);
                    const uint64_t bd = umma_sdesc_sw128(k_addr + (kk >> 2) * S::kKvSubBytes + off, 16, 1024);
                    umma_ss_elect(s_col, ad, bd, idesc_s, (t < QT - 1 || kk > 0) ? 1u : 0u);
                }
            umma_commit_elect(smem_u32(&bars->s_full[j & 1]));
            umma_commit_elect(smem_u32(&bars->k_empty[st]));
            if (NG == 1 && j >= 1) ok = issue_pv(j - 1);
        }
        if (ok && NG == 2 && n_tiles >= 2) ok = issue_pv(n_tiles - 2);
        if (ok && issue_pv(n_tiles - 1)) umma_commit_elect(smem_u32(&bars->o_final));
        // every MMA must be complete before TMEM is released
        umma_commit_elect(smem_u32(&bars->mma_done));
        mbar_wait_warp(smem_u32(&bars->mma_done), 0, p.err, kErrDrain);
    } else {
        // ================= softmax =================
        // This warp's query rows as QT bf16 terms in the 128B-swizzled K-major layout, kLoad
        // 8-element pieces in flight per lane (one at a time took 11 us of an 18 us call at
        // 512 prefix keys).  Rows past the last sequence stay unwritten: a row of Q only
        // reaches its own row of S and O, and those rows are neither used nor stored.
        constexpr int kVecs = HD / 8, kLoad = 4, kRows = 32 / NG;   // rows loaded by a warp
        const int lr = warp * kRows;
        if (s0 + (qt * kBM + lr) / p.group < s1) {
            for (int i0 = lane; i0 < kRows * kVecs; i0 += 32 * kLoad) {
                uint4 raw[kLoad][2];
#pragma unroll
                for (int n = 0; n < kLoad; ++n) {
                    const int i = i0 + 32 * n;
                    const int rr = qt * kBM + lr + i / kVecs;
                    const int rb = s0 + rr / p.group, rh = kvh * p.group + rr % p.group;
                    const long long off = (static_cast<long long>(rb) * p.n_heads + rh) * HD + (i % kVecs) * 8;
                    if (rb < s1) {
                        if (p.q_is_bf16) {
                            raw[n][0] = __ldg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p.q) + off));
                        } else {
                            const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const float *>(p.q) + off);
                            raw[n][0] = __ldg(src);
                            raw[n][1] = __ldg(src + 1);
                        }
                    }
                }
#pragma unroll
                for (int n = 0; n < kLoad; ++n) {
                    const int i = i0 + 32 * n;
                    const int r = lr + i / kVecs, e = (i % kVecs) * 8;
                    if (s0 + (qt * kBM + r) / p.group >= s1) continue;
                    const uint32_t at = (e / 64) * S::kQSubBytes + sw128_offset(r, (e % 64) / 8);
                    const uint32_t u[8] = {raw[n][0].x, raw[n][0].y, raw[n][0].z, raw[n][0].w,
                                           raw[n][1].x, raw[n][1].y, raw[n][1].z, raw[n][1].w};
                    uint32_t t[4][QT];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if (p.q_is_bf16) {
                            t[k][0] = u[k];
#pragma unroll
                            for (int q = 1; q < QT; ++q) t[k][q] = 0u;
                        } else {
                            split_bf16<QT>(__uint_as_float(u[2 * k]), __uint_as_float(u[2 * k + 1]), t[k]);
                        }
                    }
#pragma unroll
                    for (int q = 0; q < QT; ++q)
                        *reinterpret_cast<uint4 *>(smem + q * S::kQTermBytes + at) =
                            make_uint4(t[0][q], t[1][q], t[2][q], t[3][q]);
                }
            }
        }
        fence_proxy_async_smem();
        mbar_arrive(smem_u32(&bars->q_full));
        const int wg = warp / 4;
        const bool warp_live = s0 + (qt * kBM + (warp % 4) * 32) / p.group < s1;
        const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp % 4) * 32) << 16);
        const uint32_t o_col = lane_base + S::kTmO + wg * HD;
        const float cap = p.softcap, inv_cap = cap > 0.f ? 1.f / cap : 0.f;
        const float mul = cap > 0.f ? 1.f : p.scale * kLog2e;
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int j = wg; j < n_tiles; j += NG) {
            const int sb = j & 1;
            ok = mbar_wait_warp(smem_u32(&bars->s_full[sb]), (j >> 1) & 1, p.err, kErrWaitMma);
            if (!ok) break;
            if (!warp_live && key_hi - (key_lo + j * BN) >= BN) {   // no row here, no V rows to clear
                mbar_arrive(smem_u32(&bars->p_full[sb]));
                continue;
            }
            tc_fence_after();
            const uint32_t s_col = lane_base + sb * BN;
            const int key0 = key_lo + j * BN;
            const bool whole = __all_sync(0xffffffffu, row_valid && key0 >= lo && key0 + BN <= key_hi);
            // The row's keys in groups of 32 columns, once for the maximum and once for the
            // exponentials: S is read twice, but the code stays small (fully unrolled over the
            // tile it was fetched from memory for every short call).
            float mx = -INFINITY;
#pragma unroll 1
            for (int q = 0; q < BN / 32; ++q) {
                uint32_t rr[32];
                tmem_ld32(s_col + q * 32, rr);
                tmem_ld_wait();
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const int key = key0 + q * 32 + i;
                        if (!row_valid || key < lo || key >= key_hi) rr[i] = 0xff800000u;   // -inf
                    }
                }
                float pm[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) pm[i] = fmaxf(__uint_as_float(rr[2 * i]), __uint_as_float(rr[2 * i + 1]));
#pragma unroll
                for (int i = 8; i < 32; i += 8)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        pm[k] = fmaxf(pm[k], fmaxf(__uint_as_float(rr[i + 2 * k]), __uint_as_float(rr[i + 2 * k + 1])));
                mx = fmaxf(mx, fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3])));
            }
            if (cap > 0.f) {   // the cap is monotonic: the maximum's capped score is the capped maximum
                if (mx != -INFINITY) mx = cap * tanhf(mx * p.scale * inv_cap) * kLog2e;
            } else {
                mx *= mul;
            }
            // The reference m of a row is the first maximum it meets; it moves only when a
            // maximum passes it by more than 2^8 (P stays below 256 in fp16), so O is rescaled
            // rarely.  NaN scores keep m and reach P.
            const bool fresh = m == -INFINITY;
            const bool move = mx > m + kMoveLog2 || (fresh && mx != -INFINITY);
            if (__any_sync(0xffffffffu, move && !fresh)) {
                const float f = move && !fresh ? fast_exp2(m - mx) : 1.f;
                l *= f;
                // not the first tile; O holds the earlier ones' P V: scale it once they are complete
                ok = mbar_wait_warp(smem_u32(&bars->o_done[wg]), (j / NG - 1) & 1, p.err, kErrWaitMma);
                if (!ok) break;
                tc_fence_after();
#pragma unroll 1
                for (int q = 0; q < HD / 32; ++q) {
                    uint32_t ro[32];
                    tmem_ld32(o_col + q * 32, ro);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) ro[i] = __float_as_uint(__uint_as_float(ro[i]) * f);
                    tmem_st32(o_col + q * 32, ro);
                }
            }
            if (move) m = mx;
            const float negm = m != -INFINITY ? -m : 0.f;
            // P over S, in place by groups: columns 32q .. 32q+15 take the fp16 pairs of the
            // group's 32 keys, 32q+16 .. 32q+31 what their rounding left (PT == 2).
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
            for (int q = 0; q < BN / 32; ++q) {
                uint32_t rr[32];
                tmem_ld32(s_col + q * 32, rr);
                tmem_ld_wait();
                if (cap > 0.f) {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        rr[i] = __float_as_uint(cap * tanhf(__uint_as_float(rr[i]) * p.scale * inv_cap) * kLog2e);
                }
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const int key = key0 + q * 32 + i;
                        if (!row_valid || key < lo || key >= key_hi) rr[i] = 0xff800000u;
                    }
                }
                uint32_t w[32];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float e0 = fast_exp2(fmaf(__uint_as_float(rr[2 * i]), mul, negm));
                    const float e1 = fast_exp2(fmaf(__uint_as_float(rr[2 * i + 1]), mul, negm));
                    acc[i & 3] += e0 + e1;
                    if (PT == 2) split_f16(e0, e1, w[i], w[16 + i]);
                    else w[i] = pack_f16x2(e0, e1), w[16 + i] = 0u;
                }
                tmem_st32(s_col + q * 32, w);
            }
            l += (acc[0] + acc[1]) + (acc[2] + acc[3]);
            // Rows of the V tile past the part's last key may hold anything (another
            // sequence's rows, unwritten memory): 0 * NaN would reach O, so they are zeroed.
            const int nv = key_hi - key0;
            if (nv < BN) {
                ok = mbar_wait_warp(smem_u32(&bars->v_full[j % ST]), (j / ST) & 1, p.err, kErrWaitTmaFull);
                if (!ok) break;
                uint8_t *vt = sV + (j % ST) * S::kKvBytes;
                for (int i = threadIdx.x % kBM; i < (BN - nv) * 8 * S::kSub; i += kBM) {
                    const int sub = i / ((BN - nv) * 8), k = i % ((BN - nv) * 8);
                    *reinterpret_cast<uint4 *>(vt + sub * S::kKvSubBytes + nv * 128 + k * 16) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async_smem();
            }
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(smem_u32(&bars->p_full[sb]));
        }
        // o_done may be two phases behind here (a parity wait could not tell), hence o_final
        if (ok) ok = mbar_wait_warp(smem_u32(&bars->o_final), 0, p.err, kErrWaitMma);
        // after a wait that ran out the part counts as empty (the device error word is set)
        if (!ok) m = -INFINITY, l = 0.f;
        float M = m, f[2] = {1.f, 0.f};   // the row's reference, and each warpgroup's factor to it
        const int half = threadIdx.x % kBM;
        if (NG == 2) {
            float2 *ml = reinterpret_cast<float2 *>(sK);   // the K tiles are no longer needed
            ml[wg * kBM + half] = make_float2(m, l);
            named_bar_sync(1, S::kSoftmax);
            const float2 a = ml[half], d = ml[kBM + half];
            M = fmaxf(a.x, d.x);
            f[0] = a.x == -INFINITY ? 0.f : fast_exp2(a.x - M);
            f[1] = d.x == -INFINITY ? 0.f : fast_exp2(d.x - M);
            l = f[0] * a.y + f[1] * d.y;
        }
        if (__any_sync(0xffffffffu, row_valid && M != -INFINITY)) {
            tc_fence_after();
            float *dst = p.part_o + slot * HD;
#pragma unroll 1
            for (int c0 = wg * (HD / NG); c0 < (wg + 1) * (HD / NG); c0 += 32) {
                uint32_t r0[32], r1[32];
                tmem_ld32(lane_base + S::kTmO + c0, r0);
                if (NG == 2 && n_tiles > 1) tmem_ld32(lane_base + S::kTmO + HD + c0, r1);
                tmem_ld_wait();
                if (NG == 2) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        float x = f[0] != 0.f ? f[0] * __uint_as_float(r0[i]) : 0.f;
                        if (n_tiles > 1 && f[1] != 0.f) x += f[1] * __uint_as_float(r1[i]);
                        r0[i] = __float_as_uint(x);
                    }
                }
                if (row_valid) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<uint4 *>(dst + c0 + i) = make_uint4(r0[i], r0[i + 1], r0[i + 2], r0[i + 3]);
                }
            }
        }
        if (row_valid && wg == 0) p.part_ml[slot] = make_float2(M, l);
        tc_fence_before();
    }
    __syncthreads();
    if (warp == kIssuer) {
        tc_fence_after();
        tmem_dealloc(tmem, S::kTmCols);
    }
}

// ===========================================================================
// split: a sequence's own rows
// ===========================================================================
// CTA = (chunk of keys, KV head and up to 8 of its query heads, sequence).  Warp 4 streams
// 64-key tiles of K and V through a TMA ring; warps 0-3 take 16 keys of each tile:
//   S^T(16 keys x 8 heads) = K . Q^T,  O^T(hd x 8 heads) += V^T . P^T   (mma.sync)
// so one tile in shared memory serves every query head of the KV head.
constexpr int kKeysPerTile = 64;
constexpr int kConsumerWarps = 4;
constexpr int kSplitThreads = (kConsumerWarps + 1) * 32;
constexpr int kSubtileBytes = kKeysPerTile * 128;

template <int HD>
struct SplitShape {
    static constexpr int kSubtiles = HD / 64;
    static constexpr int kTileBytes = kSubtiles * kSubtileBytes;
    static constexpr int kStageBytes = 2 * kTileBytes;
    static constexpr int kStages = HD == 256 ? 1 : (HD == 128 ? 3 : 4);
    static constexpr int kQRowFloats = HD + 8;
    static constexpr int kQBytes = 8 * kQRowFloats * 4;
    static constexpr int kRedBytes = kConsumerWarps * 8 * (HD + 2) * 4;
    static_assert(kRedBytes <= kStageBytes, "the merge of the warps reuses one stage");
    static constexpr int kSmemBytes = kStages * kStageBytes + kQBytes + 256 + 1024;
};

template <int HD, int QT, int PT>
__global__ void __launch_bounds__(kSplitThreads, 2) split_kernel(const __grid_constant__ SharedParams p)
{
    using S = SplitShape<HD>;
    constexpr int KSTEPS = HD / 16;
    // After a prefix kernel, whose CTAs have all passed their own wait when this grid starts,
    // the inputs are complete and nothing here depends on it: the two run side by side, and
    // this grid only may not end before it (the merge waits for this grid alone).
    if (p.prefix_slots == 0) griddep_wait();
    griddep_trigger();
    const int b = blockIdx.z;
    const int kvh = blockIdx.y / p.n_qgroups, qg = blockIdx.y % p.n_qgroups;
    const int c = blockIdx.x;
    int ks, n;
    own_range(p, b, ks, n);
    const int key0 = ks + c * p.chunk;
    if (key0 >= n) {
        if (p.prefix_slots > 0) griddep_wait();
        return;
    }
    const int nkeys = min(p.chunk, n - key0);
    const int ntiles = (nkeys + kKeysPerTile - 1) / kKeysPerTile;
    const int h_first = kvh * p.group + qg * 8;
    const int nh = min(8, p.group - qg * 8);
    const long long row_base = p.seq_row0[b] + key0;

    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float *qs = reinterpret_cast<float *>(smem + S::kStages * S::kStageBytes);
    uint64_t *full_bar = reinterpret_cast<uint64_t *>(smem + S::kStages * S::kStageBytes + S::kQBytes);
    uint64_t *empty_bar = full_bar + S::kStages;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) {
            mbar_init(smem_u32(&full_bar[s]), 1);
            mbar_init(smem_u32(&empty_bar[s]), kConsumerWarps);
        }
        fence_mbar_init();
    }
    __syncthreads();

    if (warp == kConsumerWarps) {
        if (lane == 0) {
            tma_prefetch_desc(&p.tk);
            tma_prefetch_desc(&p.tv);
            int issued = 0;
            for (int t = 0; t < ntiles; ++t) {
                const int s = t % S::kStages;
                if (t >= S::kStages &&
                    !mbar_wait(smem_u32(&empty_bar[s]), (t / S::kStages - 1) & 1, p.err, kErrWaitTmaEmpty))
                    break;
                const uint32_t fb = smem_u32(&full_bar[s]);
                mbar_arrive_expect_tx(fb, S::kStageBytes);
                const uint32_t kdst = smem_u32(smem + s * S::kStageBytes), vdst = kdst + S::kTileBytes;
                const int y = static_cast<int>(row_base + t * kKeysPerTile);
#pragma unroll
                for (int sub = 0; sub < S::kSubtiles; ++sub) {
                    tma_load_2d(kdst + sub * kSubtileBytes, &p.tk, fb, kvh * HD + sub * 64, y);
                    tma_load_2d(vdst + sub * kSubtileBytes, &p.tv, fb, kvh * HD + sub * 64, y);
                }
                ++issued;
            }
            for (int t = max(0, issued - S::kStages); t < issued; ++t)
                if (!mbar_wait(smem_u32(&full_bar[t % S::kStages]), (t / S::kStages) & 1, p.err, kErrDrain)) break;
        }
        return;
    }
    const int g = lane >> 2, tq = lane & 3;   // key row / head column of a fragment
    {   // the CTA's query rows as fp32, one padded row per head
        const long long off = (static_cast<long long>(b) * p.n_heads + h_first) * HD;
        for (int v = threadIdx.x; v < nh * HD / 8; v += kConsumerWarps * 32) {
            const int e = v * 8;
            float *dst = qs + (e / HD) * S::kQRowFloats + e % HD;
            if (p.q_is_bf16) {
                const uint4 w = __ldg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p.q) + off + e));
                const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    dst[2 * k] = bf16lo_f32(u[k]);
                    dst[2 * k + 1] = bf16hi_f32(u[k]);
                }
            } else {
                const float4 *src = reinterpret_cast<const float4 *>(static_cast<const float *>(p.q) + off + e);
                reinterpret_cast<float4 *>(dst)[0] = __ldg(src);
                reinterpret_cast<float4 *>(dst)[1] = __ldg(src + 1);
            }
        }
        named_bar_sync(1, kConsumerWarps * 32);
    }
    uint32_t qf[KSTEPS][2][QT];   // Q^T as B fragments, QT bf16 terms
    {
        const bool valid = g < nh;
        const float *qrow = qs + (valid ? g : 0) * S::kQRowFloats;
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const float2 v = *reinterpret_cast<const float2 *>(qrow + kk * 16 + half * 8 + tq * 2);
                split_bf16<QT>(valid ? v.x : 0.f, valid ? v.y : 0.f, qf[kk][half]);
            }
    }
    const float cap = p.softcap, inv_cap = cap > 0.f ? 1.f / cap : 0.f;
    const float scale2 = p.scale * kLog2e;
    float *sc_out = nullptr;   // scores of the two heads of this lane, key 0 of the chunk
    if (p.scores && 2 * tq < nh)
        sc_out = p.scores + ((static_cast<long long>(b) * p.n_kv_heads + kvh) * p.score_rows + key0) * p.score_cols +
                 qg * 8 + 2 * tq;
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
    float o[KSTEPS][4];
#pragma unroll
    for (int i = 0; i < KSTEPS; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    bool ok = true;
    for (int t = 0; t < ntiles; ++t) {
        const int s = t % S::kStages;
        if (!mbar_wait_warp(smem_u32(&full_bar[s]), (t / S::kStages) & 1, p.err, kErrWaitTmaFull)) {
            ok = false;
            break;
        }
        const int kb = t * kKeysPerTile + warp * 16;
        const int nv = nkeys - kb;   // valid keys of this warp's block
        if (nv > 0) {
            const uint32_t kbase = smem_u32(smem + s * S::kStageBytes), vbase = kbase + S::kTileBytes;
            float acc[4] = {0.f, 0.f, 0.f, 0.f}, low[4] = {0.f, 0.f, 0.f, 0.f};   // low: the smaller terms
            const int row = warp * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
            for (int kk = 0; kk < KSTEPS; ++kk) {
                uint32_t a0, a1, a2, a3;
                ldsm_x4(kbase + (kk >> 2) * kSubtileBytes + sw128_offset(row, (kk & 3) * 2 + (lane >> 4)), a0, a1, a2,
                        a3);
                mma_bf16_16816(acc, a0, a1, a2, a3, qf[kk][0][0], qf[kk][1][0]);
#pragma unroll
                for (int q = 1; q < QT; ++q) mma_bf16_16816(low, a0, a1, a2, a3, qf[kk][0][q], qf[kk][1][q]);
            }
            float x[4];   // (key g, head 2tq) (g, 2tq+1) (g+8, 2tq) (g+8, 2tq+1), log2 units
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float raw = QT > 1 ? acc[i] + low[i] : acc[i];
                x[i] = cap > 0.f ? cap * tanhf(raw * p.scale * inv_cap) * kLog2e : raw * scale2;
                if (g + (i >> 1) * 8 >= nv) x[i] = -INFINITY;
            }
            if (sc_out) {
                if (g < nv)
                    *reinterpret_cast<float2 *>(sc_out + static_cast<long long>(kb + g) * p.score_cols) =
                        make_float2(x[0], x[1]);
                if (g + 8 < nv)
                    *reinterpret_cast<float2 *>(sc_out + static_cast<long long>(kb + g + 8) * p.score_cols) =
                        make_float2(x[2], x[3]);
            }
            float mb0 = fmaxf(x[0], x[2]), mb1 = fmaxf(x[1], x[3]);
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) {
                mb0 = fmaxf(mb0, __shfl_xor_sync(0xffffffffu, mb0, off));
                mb1 = fmaxf(mb1, __shfl_xor_sync(0xffffffffu, mb1, off));
            }
            const float mn0 = fmaxf(m_run[0], mb0), mn1 = fmaxf(m_run[1], mb1);
            // a row whose scores are all -inf so far keeps exponentials of exactly 0
            const float n0 = mn0 == -INFINITY ? 0.f : -mn0, n1 = mn1 == -INFINITY ? 0.f : -mn1;
            const float corr0 = fast_exp2(m_run[0] + n0), corr1 = fast_exp2(m_run[1] + n1);
            m_run[0] = mn0;
            m_run[1] = mn1;
            const float p0 = fast_exp2(x[0] + n0), p1 = fast_exp2(x[1] + n1);
            const float p2 = fast_exp2(x[2] + n0), p3 = fast_exp2(x[3] + n1);
            l_run[0] = l_run[0] * corr0 + (p0 + p2);
            l_run[1] = l_run[1] * corr1 + (p1 + p3);
#pragma unroll
            for (int i = 0; i < KSTEPS; ++i) {
                o[i][0] *= corr0;
                o[i][1] *= corr1;
                o[i][2] *= corr0;
                o[i][3] *= corr1;
            }
            uint32_t pb[PT][2];   // P^T as B fragments, keys 0-7 and 8-15
            {
                uint32_t h0, h1, r0 = 0, r1 = 0;
                if (PT == 2) {
                    split_f16(p0, p1, h0, r0);
                    split_f16(p2, p3, h1, r1);
                    pb[PT - 1][0] = movmatrix_t(r0);
                    pb[PT - 1][1] = movmatrix_t(r1);
                } else {
                    h0 = pack_f16x2(p0, p1);
                    h1 = pack_f16x2(p2, p3);
                }
                pb[0][0] = movmatrix_t(h0);
                pb[0][1] = movmatrix_t(h1);
            }
            const int mm = lane >> 3;
            const int vrow = warp * 16 + (lane & 7) + (mm >> 1) * 8;
            const bool tail = nv < 16;   // rows past the last key may hold anything: masked to 0
            const uint32_t mlo = (2 * tq < nv ? 0x0000ffffu : 0u) | (2 * tq + 1 < nv ? 0xffff0000u : 0u);
            const uint32_t mhi = (2 * tq + 8 < nv ? 0x0000ffffu : 0u) | (2 * tq + 9 < nv ? 0xffff0000u : 0u);
#pragma unroll
            for (int db = 0; db < KSTEPS; ++db) {
                uint32_t a0, a1, a2, a3;
                ldsm_x4_t(vbase + (db >> 2) * kSubtileBytes + sw128_offset(vrow, (db & 3) * 2 + (mm & 1)), a0, a1, a2,
                          a3);
                if (tail) {
                    a0 &= mlo;
                    a1 &= mlo;
                    a2 &= mhi;
                    a3 &= mhi;
                }
#pragma unroll
                for (int q = PT - 1; q >= 0; --q) mma_f16_16816(o[db], a0, a1, a2, a3, pb[q][0], pb[q][1]);
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&empty_bar[s]));
    }
    // ---- join the four warps; per warp and head: [m, l] then O[hd] ----
    float *red = reinterpret_cast<float *>(smem);
    constexpr int kRowF = HD + 2;
    named_bar_sync(1, kConsumerWarps * 32);
    {
        float l0 = l_run[0], l1 = l_run[1];
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, off);
            l1 += __shfl_xor_sync(0xffffffffu, l1, off);
        }
        float *w0 = red + (warp * 8 + 2 * tq) * kRowF, *w1 = w0 + kRowF;
        if (!ok) {   // a wait ran out (the device error word is set): this warp counts as empty
            m_run[0] = m_run[1] = -INFINITY;
            l0 = l1 = 0.f;
        }
        if (g == 0) {
            w0[0] = m_run[0];
            w0[1] = l0;
            w1[0] = m_run[1];
            w1[1] = l1;
        }
#pragma unroll
        for (int db = 0; db < KSTEPS; ++db) {
            const int d0 = 2 + db * 16 + g;
            w0[d0] = o[db][0];
            w1[d0] = o[db][1];
            w0[d0 + 8] = o[db][2];
            w1[d0 + 8] = o[db][3];
        }
    }
    named_bar_sync(1, kConsumerWarps * 32);
    for (int idx = threadIdx.x; idx < nh * HD; idx += kConsumerWarps * 32) {
        const int h = idx / HD, d = idx % HD;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kConsumerWarps; ++w) M = fmaxf(M, red[(w * 8 + h) * kRowF]);
        float acc = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kConsumerWarps; ++w) {
            const float mw = red[(w * 8 + h) * kRowF];
            const float f = mw == -INFINITY ? 0.f : fast_exp2(mw - M);
            if (f != 0.f) acc += f * red[(w * 8 + h) * kRowF + 2 + d];
            sum += f * red[(w * 8 + h) * kRowF + 1];
        }
        const long long slot =
            (static_cast<long long>(b) * p.n_heads + h_first + h) * p.slots + p.prefix_slots + c;
        p.part_o[slot * HD + d] = acc;
        if (d == 0) p.part_ml[slot] = make_float2(M, sum);
    }
    if (p.prefix_slots > 0) griddep_wait();
}

// ===========================================================================
// merge
// ===========================================================================
// CTA = (part of the work of one KV head, KV head, sequence).  The first out_blocks CTAs
// join 128 outputs of one query head each: warp w takes every 8th part (512 contiguous
// bytes), then the warps meet in shared memory.  The others, with weights, add the
// probabilities of kMergeKeys own keys each.  Every warp finds the M and L it needs
// itself: the (m, l) pairs of a head are few and the warps of a CTA share them in L1.
constexpr int kMergeThreads = 256;
constexpr int kMergeKeys = 1024;
constexpr int kMergeOuts = 128;

// M and 1/L of a head whose parts [first, last) have the pairs ml (the whole warp).
__device__ __forceinline__ void head_sum(const float2 *ml, int first, int last, float &M, float &inv)
{
    const int lane = threadIdx.x % 32;
    M = -INFINITY;
    for (int c = first + lane; c < last; c += 32) M = fmaxf(M, ml[c].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    float L = 0.f;
    for (int c = first + lane; c < last; c += 32) {
        const float2 v = ml[c];
        if (v.x != -INFINITY) L += fast_exp2(v.x - M) * v.y;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    inv = L != 0.f ? 1.f / L : 0.f;   // NaN stays NaN
}

template <int HD>
__global__ void __launch_bounds__(kMergeThreads) merge_kernel(const __grid_constant__ SharedParams p)
{
    griddep_wait();
    griddep_trigger();
    const int b = blockIdx.z, kvh = blockIdx.y;
    int ks, n;
    own_range(p, b, ks, n);
    const int out_blocks = (p.group * HD + kMergeOuts - 1) / kMergeOuts;
    const int j0 = (static_cast<int>(blockIdx.x) - out_blocks) * kMergeKeys;
    if (j0 >= 0 && j0 >= n) return;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (blockIdx.x == 0 && kvh == 0 && threadIdx.x == 0 && (p.kv_len[b] > p.max_kv_len || p.kv_len[b] < 0))
        atomicOr(p.err, kErrBadArgs);
    // whether the sequence has a prefix (its parts were then all written)
    bool has_prefix = false;
    for (int g = lane; g < p.n_prefixes; g += 32) {
        int s0, s1, len;
        prefix_range(p, g, s0, s1, len, false);
        has_prefix |= b >= s0 && b < s1;
    }
    has_prefix = __any_sync(0xffffffffu, has_prefix);
    const int first = has_prefix ? 0 : p.prefix_slots;
    const int last = p.prefix_slots + (n > ks ? (n - ks + p.chunk - 1) / p.chunk : 0);
    const long long row0 = static_cast<long long>(b) * p.n_heads + kvh * p.group;

    if (j0 < 0) {
        // four outputs per lane; head dim 64: two heads per CTA
        __shared__ float4 red[kMergeThreads];
        const int e = blockIdx.x * kMergeOuts + lane * 4;
        constexpr int kHeads = HD < kMergeOuts ? kMergeOuts / HD : 1;   // heads in this CTA
        const int h0 = blockIdx.x * kMergeOuts / HD;
        float M = -INFINITY, inv = 0.f;
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            if (h0 + i >= p.group) break;
            float Mi, invi;
            head_sum(p.part_ml + (row0 + h0 + i) * p.slots, first, last, Mi, invi);
            if (e / HD == h0 + i) M = Mi, inv = invi;
        }
        const bool live = e / HD < p.group;
        const float2 *ml = p.part_ml + (row0 + e / HD) * p.slots;
        const float *src = p.part_o + (row0 + e / HD) * p.slots * HD + e % HD;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        constexpr int kLoad = 4, kWarps = kMergeThreads / 32;   // parts in flight, parts side by side
        for (int c0 = first + warp; live && c0 < last; c0 += kLoad * kWarps) {
            float f[kLoad];
            float4 v[kLoad];
#pragma unroll
            for (int i = 0; i < kLoad; ++i) {
                const int c = c0 + i * kWarps;
                f[i] = c < last ? ml[c].x : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < kLoad; ++i) {   // an empty part has no output written
                v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (f[i] != -INFINITY)
                    v[i] = *reinterpret_cast<const float4 *>(src + static_cast<long long>(c0 + i * kWarps) * HD);
                f[i] = f[i] != -INFINITY ? fast_exp2(f[i] - M) : 0.f;
            }
#pragma unroll
            for (int i = 0; i < kLoad; ++i)
                a.x += f[i] * v[i].x, a.y += f[i] * v[i].y, a.z += f[i] * v[i].z, a.w += f[i] * v[i].w;
        }
        red[threadIdx.x] = a;
        __syncthreads();
        if (warp != 0 || !live) return;
#pragma unroll
        for (int w = 1; w < kWarps; ++w) {
            const float4 v = red[w * 32 + lane];
            a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
        }
        a.x *= inv, a.y *= inv, a.z *= inv, a.w *= inv;
        const long long at = row0 * HD + e;
        if (p.out_is_bf16)
            *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.out) + at) =
                make_uint2(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w));
        else
            *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + at) = a;
        return;
    }
    __shared__ float s_M[8], s_inv[8];
    constexpr int kPer = kMergeKeys / kMergeThreads;
    float w[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) w[i] = 0.f;
    const long long own = static_cast<long long>(b) * p.n_kv_heads + kvh;
    auto load_pair = [&](const float *sc, int h, float2 (&x)[kPer]) {   // score_cols is even: 8-byte loads
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int j = j0 + i * kMergeThreads + static_cast<int>(threadIdx.x);
            x[i] = j >= ks && j < n ? *reinterpret_cast<const float2 *>(sc + static_cast<long long>(j) * p.score_cols + h)
                                    : make_float2(-INFINITY, -INFINITY);
        }
    };
    float w_in[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int j = j0 + i * kMergeThreads + static_cast<int>(threadIdx.x);
        w_in[i] = p.weights_in && j < n ? p.weights_in[own * p.weights_stride + j] : 0.f;
    }
    for (int h0 = 0; h0 < p.group; h0 += 8) {
        const int nh = min(8, p.group - h0);
        const float *sc = p.scores + own * p.score_rows * p.score_cols + h0;
        float2 x[kPer];
        load_pair(sc, 0, x);   // in flight while the sums are found
        if (warp < nh) {
            float M, inv;
            head_sum(p.part_ml + (row0 + h0 + warp) * p.slots, first, last, M, inv);
            if (lane == 0) s_M[warp] = M, s_inv[warp] = inv;
        }
        __syncthreads();
        for (int h = 0; h < nh; h += 2) {
            if (h > 0) load_pair(sc, h, x);
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                if (x[i].x != -INFINITY) w[i] += fast_exp2(x[i].x - s_M[h]) * s_inv[h];
                if (h + 1 < nh && x[i].y != -INFINITY) w[i] += fast_exp2(x[i].y - s_M[h + 1]) * s_inv[h + 1];
            }
        }
        __syncthreads();
    }
    const long long base = own * p.weights_stride;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int j = j0 + i * kMergeThreads + static_cast<int>(threadIdx.x);
        if (j < n) p.weights_out[base + j] = w_in[i] + w[i];
    }
}

// ===========================================================================
// host
// ===========================================================================
int div_up(long long a, long long b) { return static_cast<int>((a + b - 1) / b); }

// Keys per part of the own rows: about 8 CTAs per SM, multiples of 64 keys, at most 2048.
int own_chunk(long long units, int max_kv_len)
{
    long long c = (units * (max_kv_len > 0 ? max_kv_len : 1) + kSms * 8 - 1) / (kSms * 8);
    c = (c + kKeysPerTile - 1) / kKeysPerTile * kKeysPerTile;
    return static_cast<int>(c < kKeysPerTile ? kKeysPerTile : c > 2048 ? 2048 : c);
}

// Most parts own_chunk() makes for any length up to max_kv_len: ceil(L/64) while the
// chunk is 64, at most ceil(1184/units) while it grows with the length, ceil(L/2048) after.
int own_slots(long long units, int max_kv_len)
{
    const int len = max_kv_len > 0 ? max_kv_len : 1;
    int small = div_up(len, kKeysPerTile);
    const int by_work = div_up(kSms * 8, units);
    if (small > by_work) small = by_work;
    const int big = div_up(len, 2048);
    return small > big ? small : big;
}

// Parts of a prefix: one CTA per SM over the query tiles and KV heads of all prefixes, no
// part under 128 keys, and none over kMaxPart: the tensor core truncates when it adds to an
// accumulator, which left a part of 6208 keys 1.3e-5 off (1024: 2e-6).
constexpr int kMaxPart = 1024;
int prefix_parts(int n_prefixes, int max_prefix_len, int max_prefix_seqs, int n_heads, int n_kv_heads)
{
    if (n_prefixes <= 0 || max_prefix_len <= 0 || max_prefix_seqs <= 0) return 0;
    const long long units = static_cast<long long>(n_prefixes) * n_kv_heads *
                            div_up(static_cast<long long>(max_prefix_seqs) * (n_heads / n_kv_heads), kBM);
    int parts = static_cast<int>(kSms / units);
    if (parts < 1) parts = 1;
    const int most = div_up(max_prefix_len, 128), least = div_up(max_prefix_len, kMaxPart);
    return parts < least ? least : parts < most ? parts : most;
}

struct SharedLayout {
    size_t part_ml, scores, total;   // part_o at 0
};

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

SharedLayout shared_layout(int n_seqs, int max_kv_len, int slots, int n_heads, int n_kv_heads, int hd, bool weights)
{
    SharedLayout L;
    const size_t items = static_cast<size_t>(n_seqs) * n_heads * slots;
    L.part_ml = align256(items * hd * 4);
    L.scores = L.part_ml + align256(items * 8);
    const size_t cols = (n_heads / n_kv_heads + 1) & ~1;
    L.total = L.scores +
              (weights ? align256(static_cast<size_t>(n_seqs) * n_kv_heads * (max_kv_len > 0 ? max_kv_len : 1) * cols * 4)
                       : 0);
    return L;
}

// Raises the dynamic shared-memory limit of a kernel, once per kernel and device.
bool allow_smem(const void *kernel, int bytes)
{
    static std::mutex mu;
    static const void *done[16][64];
    static int n_done[16] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 16) {
        cudaGetLastError();
        return false;
    }
    std::lock_guard<std::mutex> lock(mu);
    for (int i = 0; i < n_done[dev]; ++i)
        if (done[dev][i] == kernel) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
        cudaGetLastError();
        return false;
    }
    if (n_done[dev] < 64) done[dev][n_done[dev]++] = kernel;
    return true;
}

template <int HD, int QT, int PT>
int launch_shared(cudaStream_t st, SharedParams &p, const uint16_t *k_pool, const uint16_t *v_pool, int64_t pool_rows)
{
    const int kv_dim = p.n_kv_heads * HD;
    if (p.prefix_slots > 0) {
        using S = PrefixShape<HD, QT>;
        if (!make_tmap_2d(&p.tk, k_pool, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, kv_dim, pool_rows, 64, S::BN) ||
            !make_tmap_2d(&p.tv, v_pool, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, kv_dim, pool_rows, 64, S::BN) ||
            !allow_smem(reinterpret_cast<const void *>(prefix_kernel<HD, QT, PT>), S::kSmemBytes))
            return SMOL_B200_ERR_CUDA;
        const dim3 grid(div_up(static_cast<long long>(p.max_prefix_seqs) * p.group, kBM),
                        p.n_kv_heads * p.prefix_slots, p.n_prefixes);
        if (launch_kernel(prefix_kernel<HD, QT, PT>, grid, dim3(S::kThreads), S::kSmemBytes, st, p) != cudaSuccess)
            return SMOL_B200_ERR_CUDA;
    }
    if (p.max_kv_len > 0) {
        using S = SplitShape<HD>;
        if (!make_tmap_2d(&p.tk, k_pool, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, kv_dim, pool_rows, 64, kKeysPerTile) ||
            !make_tmap_2d(&p.tv, v_pool, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, kv_dim, pool_rows, 64, kKeysPerTile) ||
            !allow_smem(reinterpret_cast<const void *>(split_kernel<HD, QT, PT>), S::kSmemBytes))
            return SMOL_B200_ERR_CUDA;
        const dim3 grid(p.max_chunks, p.n_kv_heads * p.n_qgroups, p.n_seqs);
        if (launch_kernel(split_kernel<HD, QT, PT>, grid, dim3(kSplitThreads), S::kSmemBytes, st, p) != cudaSuccess)
            return SMOL_B200_ERR_CUDA;
    }
    const int blocks = div_up(p.group * HD, kMergeOuts) + (p.scores ? div_up(p.max_kv_len, kMergeKeys) : 0);
    if (launch_kernel(merge_kernel<HD>, dim3(blocks, p.n_kv_heads, p.n_seqs), dim3(kMergeThreads), 0, st, p) !=
        cudaSuccess)
        return SMOL_B200_ERR_CUDA;
    return SMOL_B200_OK;
}

template <int HD>
int launch_shared_hd(cudaStream_t st, SharedParams &p, const uint16_t *k, const uint16_t *v, int64_t rows)
{
    if (p.q_is_bf16)
        return p.out_is_bf16 ? launch_shared<HD, 1, 1>(st, p, k, v, rows) : launch_shared<HD, 1, 2>(st, p, k, v, rows);
    return p.out_is_bf16 ? launch_shared<HD, 3, 1>(st, p, k, v, rows) : launch_shared<HD, 3, 2>(st, p, k, v, rows);
}

bool sizes_ok(int n_seqs, int max_kv_len, int n_heads, int n_kv_heads, int head_dim)
{
    return n_seqs > 0 && n_seqs <= 65535 && max_kv_len >= 0 && n_heads > 0 && n_kv_heads > 0 &&
           n_heads % n_kv_heads == 0 && n_heads <= 65535 && (head_dim == 64 || head_dim == 128 || head_dim == 256);
}

long long own_units(int n_seqs, int n_heads, int n_kv_heads)
{
    return static_cast<long long>(n_seqs) * n_kv_heads * ((n_heads / n_kv_heads + 7) / 8);
}

}  // namespace

size_t decode_shared_workspace_bytes(int n_seqs, int max_kv_len, int n_prefixes, int max_prefix_len,
                                     int max_prefix_seqs, int n_heads, int n_kv_heads, int head_dim, bool weights)
{
    if (!sizes_ok(n_seqs, max_kv_len, n_heads, n_kv_heads, head_dim)) return 0;
    const int slots = own_slots(own_units(n_seqs, n_heads, n_kv_heads), max_kv_len) +
                      prefix_parts(n_prefixes, max_prefix_len, max_prefix_seqs, n_heads, n_kv_heads);
    return shared_layout(n_seqs, max_kv_len, slots, n_heads, n_kv_heads, head_dim, weights).total;
}

int decode_attention_shared(cudaStream_t st, void *out, int out_is_bf16, const void *q, int q_is_bf16,
                            const uint16_t *k_pool, const uint16_t *v_pool, int64_t pool_rows,
                            const int64_t *prefix_row0, const int *prefix_len, const int *prefix_seq0, int n_prefixes,
                            int max_prefix_len, int max_prefix_seqs, const int64_t *seq_row0, const int *kv_len,
                            int n_seqs, int max_kv_len, int n_heads, int n_kv_heads, int head_dim, float scale,
                            int window, float softcap, const float *weights_in, float *weights_out,
                            int64_t weights_stride, void *workspace, size_t workspace_bytes)
{
    if (n_seqs <= 0) return SMOL_B200_OK;
    if (!sizes_ok(n_seqs, max_kv_len, n_heads, n_kv_heads, head_dim) || !out || !q || !k_pool || !v_pool ||
        !seq_row0 || !kv_len || pool_rows <= 0 || pool_rows >= (1ll << 31) || n_prefixes < 0 || n_prefixes > 65535 ||
        max_prefix_len < 0 || max_prefix_seqs < 0 || max_prefix_seqs > n_seqs)
        return SMOL_B200_ERR_ARGS;
    if (n_prefixes > 0 && (!prefix_row0 || !prefix_len || !prefix_seq0)) return SMOL_B200_ERR_ARGS;
    if ((reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool) | reinterpret_cast<uintptr_t>(q) |
         reinterpret_cast<uintptr_t>(out)) & 15)
        return SMOL_B200_ERR_ARGS;
    if (!(scale > 0.f)) return SMOL_B200_ERR_ARGS;
    if (weights_in && !weights_out) return SMOL_B200_ERR_ARGS;
    if (weights_out && weights_stride < max_kv_len) return SMOL_B200_ERR_ARGS;
    if (max_prefix_len == 0 || max_prefix_seqs == 0) n_prefixes = 0;

    SharedParams p;
    memset(&p, 0, sizeof(p));
    const long long units = own_units(n_seqs, n_heads, n_kv_heads);
    if (n_kv_heads * ((n_heads / n_kv_heads + 7) / 8) > 65535) return SMOL_B200_ERR_ARGS;
    p.group = n_heads / n_kv_heads;
    p.n_qgroups = (p.group + 7) / 8;
    p.chunk = own_chunk(units, max_kv_len);
    p.max_chunks = max_kv_len > 0 ? div_up(max_kv_len, p.chunk) : 0;
    p.prefix_slots = prefix_parts(n_prefixes, max_prefix_len, max_prefix_seqs, n_heads, n_kv_heads);
    if (p.prefix_slots > 0) p.prefix_chunk = (div_up(max_prefix_len, p.prefix_slots) + 63) / 64 * 64;
    if (static_cast<long long>(n_kv_heads) * p.prefix_slots > 65535) return SMOL_B200_ERR_ARGS;
    p.slots = p.prefix_slots + p.max_chunks;
    if (p.slots < 1) p.slots = 1;
    const size_t need = decode_shared_workspace_bytes(n_seqs, max_kv_len, n_prefixes, max_prefix_len, max_prefix_seqs,
                                                      n_heads, n_kv_heads, head_dim, weights_out != nullptr);
    if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15))
        return SMOL_B200_ERR_WORKSPACE;
    const SharedLayout L = shared_layout(n_seqs, max_kv_len, p.slots, n_heads, n_kv_heads, head_dim,
                                         weights_out != nullptr);
    uint8_t *base = static_cast<uint8_t *>(workspace);
    p.part_o = reinterpret_cast<float *>(base);
    p.part_ml = reinterpret_cast<float2 *>(base + L.part_ml);
    p.scores = weights_out ? reinterpret_cast<float *>(base + L.scores) : nullptr;
    p.score_rows = max_kv_len;
    p.score_cols = (p.group + 1) & ~1;
    p.q = q;
    p.out = out;
    p.q_is_bf16 = q_is_bf16 ? 1 : 0;
    p.out_is_bf16 = out_is_bf16 ? 1 : 0;
    p.prefix_row0 = prefix_row0;
    p.prefix_len = prefix_len;
    p.prefix_seq0 = prefix_seq0;
    p.seq_row0 = seq_row0;
    p.kv_len = kv_len;
    p.weights_in = weights_in;
    p.weights_out = weights_out;
    p.weights_stride = weights_stride;
    p.err = device_error_word();
    if (!p.err) return SMOL_B200_ERR_CUDA;
    p.n_seqs = n_seqs;
    p.n_heads = n_heads;
    p.n_kv_heads = n_kv_heads;
    p.n_prefixes = n_prefixes;
    p.max_prefix_len = max_prefix_len;
    p.max_prefix_seqs = max_prefix_seqs;
    p.max_kv_len = max_kv_len;
    p.window = window;
    p.scale = scale;
    p.softcap = softcap;
    // every kernel waits for its predecessor before reading anything
    PdlScope pdl(g_api_pdl);
    switch (head_dim) {
    case 64: return launch_shared_hd<64>(st, p, k_pool, v_pool, pool_rows);
    case 128: return launch_shared_hd<128>(st, p, k_pool, v_pool, pool_rows);
    default: return launch_shared_hd<256>(st, p, k_pool, v_pool, pool_rows);
    }
}

}  // namespace smolb200
