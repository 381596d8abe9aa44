// prefill_weights.cu -- the attention weight each cached key receives from the rows of a
// prompt:  w_j += sum over rows i and the query heads h of j's KV head of
//          p_hij = e^(x_hij - lse_hi),  x = scale * q.k (capped), lse_hi = log sum_j e^x_hij
//
// Two passes of the same tiles, S = X Y^T on tcgen05 with fp32 accumulators in TMEM:
//   stats  X = 128 rows (query, head of the KV group), Y = key tiles: every thread owns a
//          row and keeps its reference point and sum; the sums give lse;
//   sums   X = 128 keys, Y = row tiles: every thread owns a KEY, so the sum over rows is
//          a sum in its register, with the rows' lse broadcast from shared memory.  With
//          a single row tile the roles of the two operands in the products change: the
//          rows stay in shared memory, key tiles stream and each is complete by itself.
// The probabilities themselves are never stored.  Bound: two exponentials per visible
// (row, key) pair at 16 per clock and SM; a tile's products take half as long.
//
// Both passes cut their long axis into parts of at most kMaxTiles tiles, whose results a
// small kernel joins in a fixed order, so that causal work spreads evenly and few rows
// against many keys still fill the GPU.  Two CTAs share an SM: one's loads and ends
// hide behind the other's exponentials.
#include <string.h>

#include <mutex>

#include "b200_common.cuh"
#include "fast_math.cuh"
#include "runtime.h"

namespace smolb200 {
namespace {

constexpr int kTile = 128;
constexpr int kMaxTiles = 16;
constexpr int kExpThreads = 256;              // two warpgroups, on alternate tiles
constexpr int kThreads = kExpThreads + 64;    // + TMA producer warp, tcgen05 issuer warp
constexpr float kSumLimit = 1.152921504606847e18f;   // 2^60: a tile's row sum beyond this moves the reference

enum Mode { kStats = 0, kSums = 1, kSumsOneRowTile = 2 };

template <int HD>
struct WShape {
    static constexpr int kSub = HD / 64;
    static constexpr int kSubBytes = kTile * 128;
    static constexpr int kTileBytes = kSub * kSubBytes;
    static constexpr int kStages = HD == 64 ? 4 : 2;
    static constexpr int kOffY = kTileBytes;
    static constexpr int kOffCols = kOffY + kStages * kTileBytes;
    // per warpgroup, twice: -lse, first and past-last visible key of 128 rows
    static constexpr int kColBytes = 2 * 2 * kTile * 12;
    static constexpr int kOffBar = kOffCols + kColBytes;
    static constexpr int kSmemBytes = kOffBar + 256 + 1024;
    static constexpr int kCtas = HD == 256 ? 1 : 2;          // per SM
    static_assert(kSmemBytes <= (HD == 256 ? 227 : 113) * 1024, "shared memory");
};

struct WParams {
    CUtensorMap tq, tk;   // (column, head, row, batch); boxes 64 x group x qp x 1 and 64 x 1 x 128 x 1
    float2 *stat_parts;   // [batch][n_kv_heads][rows][parts]: reference (log2 units), sum
    float *lse;           // [batch][n_kv_heads][rows], log2 units; +inf for a row without keys
    float *sum_parts;     // [parts][batch][n_kv_heads][seq_k]
    const float *weights_in;
    float *weights_out;
    long long weights_stride;
    unsigned *err;
    int batch, seq_q, seq_k, n_kv_heads, group, qp;   // qp: queries of a row tile
    int row_tiles, key_tiles;
    int stat_tiles, n_stat_parts;   // key tiles of a stats part; parts
    int sum_tiles, n_sum_parts;     // the same for sums (row tiles; key tiles with one row tile)
    int mask_kind, q_offset, prefix_len, window;
    int q_bytes;                    // bytes of a row tile's boxes (all sub-tiles)
    float scale, softcap;
};

struct WBars {
    uint64_t x_full, y_full[4], y_empty[4], d_full[2], d_empty[2], done;
    uint32_t tmem_base;
};

// sum += 2^(v*mul + off) for 16 columns; kPoly of every 8 pairs on the FMA pipe, the rest on
// MUFU.  A pair takes 16 MUFU cycles of a scheduler, or 12 issue slots on the FMA pipe.
#ifndef SMOL_WEIGHTS_POLY
#define SMOL_WEIGHTS_POLY 3
#endif
constexpr int kPoly = SMOL_WEIGHTS_POLY;
__device__ __forceinline__ void add_exp2(const uint32_t (&v)[16], float mul, const float (&off)[16], float (&acc)[4])
{
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float x0, x1, e0, e1;
        pair_fma(x0, x1, __uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]), mul, mul, off[2 * i], off[2 * i + 1]);
        if ((i * kPoly) % 8 < kPoly) {
            pair_exp2_poly(x0, x1, e0, e1);
        } else {
            e0 = fast_exp2f(x0);
            e1 = fast_exp2f(x1);
        }
        pair_add(acc[2 * (i & 1)], acc[2 * (i & 1) + 1], acc[2 * (i & 1)], acc[2 * (i & 1) + 1], e0, e1);
    }
}

// Keys [lo, hi) that query i sees (both non-decreasing in i).
__device__ __forceinline__ void row_keys(const WParams &p, int i, int &lo, int &hi)
{
    const int pos = p.q_offset + i;
    hi = p.mask_kind == SMOL_MASK_CAUSAL      ? pos + 1
         : p.mask_kind == SMOL_MASK_PREFIX_LM ? max(pos + 1, p.prefix_len)
                                              : p.seq_k;
    hi = min(max(hi, 0), p.seq_k);
    lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
    if (lo > hi) lo = hi;
}

// Row tiles [t0, t1) with a row that sees a key of [k0, k1).
__device__ __forceinline__ void key_rows(const WParams &p, int k0, int k1, int &t0, int &t1)
{
    int i0 = 0, i1 = p.seq_q;
    if (p.mask_kind == SMOL_MASK_CAUSAL || (p.mask_kind == SMOL_MASK_PREFIX_LM && k0 >= p.prefix_len))
        i0 = max(0, k0 - p.q_offset);
    if (p.window > 0) {   // lo < k1: pos <= k1 + window - 2
        const long long last = static_cast<long long>(k1) + p.window - 2 - p.q_offset;
        if (last + 1 < i1) i1 = static_cast<int>(max(last + 1, 0ll));
    }
    t0 = i0 / p.qp;
    t1 = i1 > i0 ? (i1 + p.qp - 1) / p.qp : t0;
}

template <int HD, int MODE>
__global__ void __launch_bounds__(kThreads, WShape<HD>::kCtas) weights_kernel(const __grid_constant__ WParams p)
{
    using S = WShape<HD>;
    constexpr int ST = S::kStages;
    griddep_wait();
    griddep_trigger();
    const int kvh = blockIdx.y, b = blockIdx.z;
    const int part = MODE == kStats ? blockIdx.x % p.n_stat_parts : blockIdx.x % p.n_sum_parts;
    // x: the tile that stays (rows for stats and for one row tile, keys else); [t0, t1): the tiles that stream
    int x = MODE == kStats ? blockIdx.x / p.n_stat_parts : blockIdx.x / p.n_sum_parts;
    int t0, t1;
    if constexpr (MODE == kStats) {
        x = p.row_tiles - 1 - x;   // causal rows see more keys the later they are: those first
        int lo, hi, unused;
        row_keys(p, x * p.qp, lo, unused);
        row_keys(p, min(p.seq_q, (x + 1) * p.qp) - 1, unused, hi);
        t0 = max(lo / kTile, part * p.stat_tiles);
        t1 = min((hi + kTile - 1) / kTile, (part + 1) * p.stat_tiles);
    } else if constexpr (MODE == kSums) {
        key_rows(p, x * kTile, min(p.seq_k, (x + 1) * kTile), t0, t1);
        t0 += part * p.sum_tiles;
        t1 = min(t1, t0 + p.sum_tiles);
    } else {
        t0 = part * p.sum_tiles;
        t1 = min(p.key_tiles, t0 + p.sum_tiles);
    }
    const int n = max(0, t1 - t0);
    const long long unit = static_cast<long long>(b) * p.n_kv_heads + kvh;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    WBars *bars = reinterpret_cast<WBars *>(smem + S::kOffBar);
    if (n > 0) {
        if (threadIdx.x == 0) {
            mbar_init(smem_u32(&bars->x_full), 1);
            for (int s = 0; s < ST; ++s) {
                mbar_init(smem_u32(&bars->y_full[s]), 1);
                mbar_init(smem_u32(&bars->y_empty[s]), 1);
            }
            for (int s = 0; s < 2; ++s) {
                mbar_init(smem_u32(&bars->d_full[s]), 1);
                mbar_init(smem_u32(&bars->d_empty[s]), 128);
            }
            mbar_init(smem_u32(&bars->done), 1);
            fence_mbar_init();
        }
        // a row tile fills qp*group of the 128 rows; the rest must be finite (they meet lse = +inf)
        if (p.qp * p.group < kTile) {
            const int first = p.qp * p.group * 8, per = kTile * 8 - first;   // 16-byte units of a sub-tile
            for (int i = threadIdx.x; i < per * S::kSub * (1 + ST); i += kThreads) {
                const int sub = i / per, u = first + i % per;
                *reinterpret_cast<uint4 *>(smem + sub * S::kSubBytes + u * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
        }
        if (warp == 9) {
            tmem_alloc(smem_u32(&bars->tmem_base), 256);
            tmem_relinquish();
        }
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
    }
    const uint32_t tmem = n > 0 ? bars->tmem_base : 0;

    if (warp == 8) {
        // ================= TMA producer =================
        if (lane == 0 && n > 0) {
            tma_prefetch_desc(&p.tq);
            tma_prefetch_desc(&p.tk);
            auto load = [&](uint32_t dst, uint32_t bar, bool rows, int t) {
                mbar_arrive_expect_tx(bar, rows ? p.q_bytes : S::kTileBytes);
#pragma unroll
                for (int sub = 0; sub < S::kSub; ++sub) {
                    if (rows) tma_load_4d(dst + sub * S::kSubBytes, &p.tq, bar, sub * 64, kvh * p.group, t * p.qp, b);
                    else tma_load_4d(dst + sub * S::kSubBytes, &p.tk, bar, sub * 64, kvh, t * kTile, b);
                }
            };
            load(smem_u32(smem), smem_u32(&bars->x_full), MODE != kSums, x);
            int issued = 0;
            for (int t = 0; t < n; ++t) {
                const int st = t % ST;
                if (t >= ST && !mbar_wait(smem_u32(&bars->y_empty[st]), (t / ST - 1) & 1, p.err, kErrWaitTmaEmpty))
                    break;
                load(smem_u32(smem + S::kOffY + st * S::kTileBytes), smem_u32(&bars->y_full[st]), MODE == kSums, t0 + t);
                ++issued;
            }
            mbar_wait(smem_u32(&bars->x_full), 0, p.err, kErrDrain);
            for (int t = max(0, issued - ST); t < issued; ++t)
                if (!mbar_wait(smem_u32(&bars->y_full[t % ST]), (t / ST) & 1, p.err, kErrDrain)) break;
        }
    } else if (warp == 9) {
        // ================= tcgen05 issuer =================
        if (n > 0) {
            constexpr uint32_t idesc = umma_idesc_f16(kTile, kTile, true, false);
            const uint32_t x_addr = smem_u32(smem);
            bool ok = mbar_wait_warp(smem_u32(&bars->x_full), 0, p.err, kErrWaitTmaFull);
            for (int t = 0; t < n && ok; ++t) {
                const int st = t % ST, d = t & 1;
                if (t >= 2) ok = mbar_wait_warp(smem_u32(&bars->d_empty[d]), (t / 2 - 1) & 1, p.err, kErrWaitSoftmax);
                if (ok) ok = mbar_wait_warp(smem_u32(&bars->y_full[st]), (t / ST) & 1, p.err, kErrWaitTmaFull);
                if (!ok) break;
                tc_fence_after();
                const uint32_t y_addr = smem_u32(smem + S::kOffY + st * S::kTileBytes);
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk) {
                    const uint32_t off = (kk >> 2) * S::kSubBytes + (kk & 3) * 32;
                    const uint64_t xd = umma_sdesc_sw128(x_addr + off, 16, 1024);
                    const uint64_t yd = umma_sdesc_sw128(y_addr + off, 16, 1024);
                    // rows of S: the tile whose rows are reduced over the other's
                    umma_ss_elect(tmem + d * kTile, MODE == kSumsOneRowTile ? yd : xd, MODE == kSumsOneRowTile ? xd : yd,
                                  idesc, kk > 0 ? 1u : 0u);
                }
                umma_commit_elect(smem_u32(&bars->d_full[d]));
                umma_commit_elect(smem_u32(&bars->y_empty[st]));
            }
            umma_commit_elect(smem_u32(&bars->done));
            mbar_wait_warp(smem_u32(&bars->done), 0, p.err, kErrDrain);
        }
    } else {
        // ================= exponentials: thread r of a warpgroup owns row r of S =================
        const int wg = warp / 4, r = threadIdx.x % kTile;
        const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp % 4) * 32) << 16);
        const float cap = p.softcap, inv_cap = cap > 0.f ? 1.f / cap : 0.f;
        const float mul = cap > 0.f ? 1.f : p.scale * kLog2e;
        const long long rows = static_cast<long long>(p.seq_q) * p.group;
        // this warpgroup's two column sets: -lse, then the first and the past-last visible key
        float *cols = reinterpret_cast<float *>(smem + S::kOffCols) + wg * 2 * 3 * kTile;
        // A wait that runs out (the device error word is set) skips the tiles that follow, but
        // every warp keeps to the barriers it shares with the others.
        bool ok = true;
        auto capped = [&](uint32_t (&v)[16]) {
            if (cap > 0.f) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    v[i] = __float_as_uint(cap * tanhf(__uint_as_float(v[i]) * p.scale * inv_cap) * kLog2e);
            }
        };
        const int r_query = r / p.group;   // query of this thread's row or column within a row tile
        const bool r_used = r < p.qp * p.group;
        // -lse of this thread's column of row tile t (-inf: nothing is added)
        auto neg_lse = [&](int t) -> float {
            const bool valid = r_used && t * p.qp + r_query < p.seq_q;
            return valid ? -p.lse[unit * rows + static_cast<long long>(t) * p.qp * p.group + r] : -INFINITY;
        };
        // Column set `set` = row tile t.  One barrier: a set is written again two tiles later.
        // Returns whether a NaN is among the lse: it has to reach the weights.
        auto load_cols = [&](int t, int set, float nl) -> bool {
            int lo = 0, hi = 0;
            if (r_used && t * p.qp + r_query < p.seq_q) row_keys(p, t * p.qp + r_query, lo, hi);
            float *c = cols + set * 3 * kTile;
            c[r] = nl;
            reinterpret_cast<int *>(c)[kTile + r] = lo;
            reinterpret_cast<int *>(c)[2 * kTile + r] = hi;
            int any;
            asm volatile("{ .reg .pred p, q; setp.ne.b32 p, %1, 0; barrier.cta.red.or.pred q, %2, %3, p; selp.b32 %0, 1, 0, q; }"
                         : "=r"(any)
                         : "r"(nl != nl ? 1 : 0), "r"(1 + wg), "r"(kTile)
                         : "memory");
            return any != 0;
        };
        // whether every row of row tile t sees all of keys [k0, k1)
        auto all_visible = [&](int t, int k0, int k1) -> bool {
            int lo, hi, unused;
            row_keys(p, t * p.qp, unused, hi);
            row_keys(p, min(p.seq_q, (t + 1) * p.qp) - 1, lo, unused);
            return lo <= k0 && hi >= k1;
        };

        if constexpr (MODE == kStats) {
            const int i = x * p.qp + r_query;
            const bool valid = r_used && i < p.seq_q;
            const bool live = __any_sync(0xffffffffu, valid);
            int lo = 0, hi = 0;
            if (valid) row_keys(p, i, lo, hi);
            float m = -INFINITY, l = 0.f;
            for (int t = wg; t < n; t += 2) {
                if (ok) ok = mbar_wait_warp(smem_u32(&bars->d_full[wg]), (t / 2) & 1, p.err, kErrWaitMma);
                if (live && ok) {
                    tc_fence_after();
                    const uint32_t s_col = lane_base + wg * kTile;
                    const int key0 = (t0 + t) * kTile;
                    // rows past the last one may see anything: they are not stored
                    const bool whole = __all_sync(0xffffffffu, !valid || (key0 >= lo && key0 + kTile <= hi));
                    auto hide = [&](int c0, uint32_t (&v)[16]) {
                        if (!whole) {
#pragma unroll
                            for (int c = 0; c < 16; ++c)
                                if (key0 + c0 + c < lo || key0 + c0 + c >= hi) v[c] = 0xff800000u;   // -inf
                        }
                    };
                    // fp32 sums need no maximum close by, only no overflow: a row's reference is
                    // the maximum of the first keys it meets and moves when a tile's sum passes 2^60
                    bool need = __any_sync(0xffffffffu, m == -INFINITY && key0 < hi && key0 + kTile > lo);
                    float lt = 0.f;
                    for (int pass = 0; pass < 2; ++pass) {
                        if (need) {
                            float mx = -INFINITY;
                            for_columns(s_col, kTile / 16, [&](int c0, uint32_t (&v)[16]) {
                                hide(c0, v);
#pragma unroll
                                for (int c = 0; c < 16; ++c) mx = fmaxf(mx, __uint_as_float(v[c]));
                            });
                            if (mx != -INFINITY)
                                mx = cap > 0.f ? cap * tanhf(mx * p.scale * inv_cap) * kLog2e : mx * mul;
                            const bool move = m == -INFINITY || (pass == 1 && !(lt <= kSumLimit));
                            if (move && mx != -INFINITY) {
                                if (m != -INFINITY) l *= fast_exp2f(m - mx);
                                m = mx;
                            }
                        }
                        const float negm = m != -INFINITY ? -m : 0.f;
                        float acc[4] = {0.f, 0.f, 0.f, 0.f};
                        if (whole && !need) {
                            float off[16];
#pragma unroll
                            for (int c = 0; c < 16; ++c) off[c] = negm;
                            // a score may still be far above m (the sum then passes the limit):
                            // the polynomial's exponent must not wrap, so the scores' maximum is
                            // kept beside the sum
                            float top = -INFINITY;
                            for_columns(s_col, kTile / 16, [&](int c0, uint32_t (&v)[16]) {
                                capped(v);
#pragma unroll
                                for (int c = 0; c < 16; c += 2)
                                    top = fmaxf(top, fmaxf(__uint_as_float(v[c]), __uint_as_float(v[c + 1])));
                                add_exp2(v, mul, off, acc);
                            });
                            lt = fmaf(top, mul, negm) > 60.f ? INFINITY : (acc[0] + acc[1]) + (acc[2] + acc[3]);
                        } else {
                            for_columns(s_col, kTile / 16, [&](int c0, uint32_t (&v)[16]) {
                                capped(v);
                                hide(c0, v);
#pragma unroll
                                for (int c = 0; c < 16; ++c)
                                    acc[c & 3] += fast_exp2f(fmaf(__uint_as_float(v[c]), mul, negm));
                            });
                            lt = (acc[0] + acc[1]) + (acc[2] + acc[3]);
                        }
                        need = __any_sync(0xffffffffu, !(lt <= kSumLimit));
                        if (!need) break;
                    }
                    l += lt;
                    tc_fence_before();
                }
                mbar_arrive(smem_u32(&bars->d_empty[wg]));
            }
            if (!ok) m = -INFINITY, l = 0.f;
            float2 *other = reinterpret_cast<float2 *>(smem + S::kOffCols);
            if (wg == 1) other[r] = make_float2(m, l);
            named_bar_sync(3, kExpThreads);
            if (wg == 0 && valid) {
                const float2 o = other[r];
                const float M = fmaxf(m, o.x);
                float L = 0.f;
                if (m != -INFINITY) L += l * fast_exp2f(m - M);
                if (o.x != -INFINITY) L += o.y * fast_exp2f(o.x - M);
                const long long row = unit * rows + static_cast<long long>(x) * p.qp * p.group + r;
                if (p.n_stat_parts == 1) p.lse[row] = M == -INFINITY ? INFINITY : M + log2f(L);
                else p.stat_parts[row * p.n_stat_parts + part] = make_float2(M, L);
            }
        } else {
            // sum over the first n16 * 16 columns of the tile in this warpgroup's buffer, columns
            // described by `set`, of 2^(S - lse) for key `key`; `whole`: the key sees them all
            auto tile_sum = [&](int key, int set, int n16, bool whole) -> float {
                const float *c = cols + set * 3 * kTile;
                const int *c_lo = reinterpret_cast<const int *>(c) + kTile, *c_hi = c_lo + kTile;
                float acc[4] = {0.f, 0.f, 0.f, 0.f};
                for_columns(lane_base + wg * kTile, n16, [&](int c0, uint32_t (&v)[16]) {
                    capped(v);
                    float off[16];
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const float4 e = *reinterpret_cast<const float4 *>(c + c0 + i);
                        off[i] = e.x, off[i + 1] = e.y, off[i + 2] = e.z, off[i + 3] = e.w;
                    }
                    if (whole) {
                        add_exp2(v, mul, off, acc);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float y = fast_exp2f(fmaf(__uint_as_float(v[i]), mul, off[i]));
                            if (key >= c_lo[c0 + i] && key < c_hi[c0 + i]) acc[i & 3] += y;
                        }
                    }
                });
                return (acc[0] + acc[1]) + (acc[2] + acc[3]);
            };
            // columns of row tile t that hold rows
            auto used_cols = [&](int t) -> int { return min(p.qp, p.seq_q - t * p.qp) * p.group; };
            if constexpr (MODE == kSums) {
                const int k0 = x * kTile, key = k0 + r, k1 = min(p.seq_k, k0 + kTile);
                float sum = 0.f;
                float nl = wg < n ? neg_lse(t0 + wg) : 0.f;
                for (int t = wg; t < n; t += 2) {
                    const int set = (t >> 1) & 1, used = used_cols(t0 + t);
                    const bool nan = load_cols(t0 + t, set, nl);
                    if (t + 2 < n) nl = neg_lse(t0 + t + 2);   // in flight during this tile
                    if (ok) ok = mbar_wait_warp(smem_u32(&bars->d_full[wg]), (t / 2) & 1, p.err, kErrWaitMma);
                    if (ok) {
                        tc_fence_after();
                        sum += tile_sum(key, set, (used + 15) / 16, !nan && used % 16 == 0 && all_visible(t0 + t, k0, k1));
                        tc_fence_before();
                    }
                    mbar_arrive(smem_u32(&bars->d_empty[wg]));
                }
                named_bar_sync(3, kExpThreads);   // the columns are no longer read
                float *other = reinterpret_cast<float *>(smem + S::kOffCols);
                if (wg == 1) other[r] = sum;
                named_bar_sync(3, kExpThreads);
                if (wg == 0 && key < p.seq_k) {
                    sum += other[r];
                    if (p.n_sum_parts == 1) {
                        const long long at = unit * p.weights_stride + key;
                        p.weights_out[at] = (p.weights_in ? p.weights_in[at] : 0.f) + sum;
                    } else {
                        p.sum_parts[(static_cast<long long>(part) * p.batch * p.n_kv_heads + unit) * p.seq_k + key] = sum;
                    }
                }
            } else {
                const int used = used_cols(0);
                const bool nan = n > 0 ? load_cols(0, 0, neg_lse(0)) : false;
                for (int t = wg; t < n; t += 2) {
                    const int k0 = (t0 + t) * kTile, key = k0 + r;
                    const long long at = unit * p.weights_stride + key;
                    const float before = p.weights_in && key < p.seq_k ? p.weights_in[at] : 0.f;
                    if (ok) ok = mbar_wait_warp(smem_u32(&bars->d_full[wg]), (t / 2) & 1, p.err, kErrWaitMma);
                    float sum = 0.f;
                    if (ok) {
                        tc_fence_after();
                        sum = tile_sum(key, 0, (used + 15) / 16,
                                       !nan && used % 16 == 0 && all_visible(0, k0, min(p.seq_k, k0 + kTile)));
                        tc_fence_before();
                    }
                    mbar_arrive(smem_u32(&bars->d_empty[wg]));
                    if (key < p.seq_k) p.weights_out[at] = before + sum;
                }
            }
        }
    }
    if (n > 0) {
        tc_fence_before();
        __syncthreads();
        if (warp == 9) {
            tc_fence_after();
            tmem_dealloc(tmem, 256);
        }
    }
}

// lse of every row from its parts, `width` (a power of two up to 32) lanes to a row.
__global__ void __launch_bounds__(256) weights_lse_kernel(float *lse, const float2 *parts, long long rows, int n_parts,
                                                          int width)
{
    griddep_wait();
    griddep_trigger();
    const long long t = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    const long long r = t / width;
    const int lane = static_cast<int>(t % width);
    float M = -INFINITY, L = 0.f;
    if (r < rows)
        for (int c = lane; c < n_parts; c += width) M = fmaxf(M, parts[r * n_parts + c].x);
    for (int o = width / 2; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    if (r < rows)
        for (int c = lane; c < n_parts; c += width) {
            const float2 v = parts[r * n_parts + c];
            if (v.x != -INFINITY) L += v.y * fast_exp2f(v.x - M);
        }
    for (int o = width / 2; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    if (r < rows && lane == 0) lse[r] = M == -INFINITY ? INFINITY : M + log2f(L);
}

// weights_out = weights_in + the parts, in order (no parts: a copy).
__global__ void __launch_bounds__(256) weights_add_kernel(float *out, const float *in, long long stride,
                                                          const float *parts, int n_parts, int seq_k, int n_kv_heads)
{
    griddep_wait();
    griddep_trigger();
    const int j = blockIdx.x * 256 + threadIdx.x;
    if (j >= seq_k) return;
    const long long unit = static_cast<long long>(blockIdx.z) * n_kv_heads + blockIdx.y;
    const long long units = static_cast<long long>(gridDim.z) * n_kv_heads;
    float s = 0.f;
#pragma unroll 4
    for (int c = 0; c < n_parts; ++c) s += parts[(c * units + unit) * seq_k + j];
    out[unit * stride + j] = (in ? in[unit * stride + j] : 0.f) + s;
}

// How the two passes are cut: parts of at most kMaxTiles tiles, shorter ones where the CTAs
// would not fill the GPU, but no more of them than run at once.
struct WPlan {
    int qp, row_tiles, key_tiles, stat_tiles, n_stat_parts, sum_tiles, n_sum_parts;
    size_t lse, sum_parts, total;   // stat_parts at 0
};

WPlan weights_plan(int batch, int seq_q, int seq_k, int n_heads, int n_kv_heads, int head_dim)
{
    WPlan w;
    const int group = n_heads / n_kv_heads;
    const long long units = static_cast<long long>(batch) * n_kv_heads;
    auto up = [](long long a, long long b) { return static_cast<int>((a + b - 1) / b); };
    auto al = [](size_t x) { return (x + 255) & ~size_t(255); };
    w.qp = kTile / group;
    w.row_tiles = up(seq_q, w.qp);
    w.key_tiles = up(seq_k, kTile);
    const long long at_once = 148 * (head_dim > 128 ? WShape<256>::kCtas : WShape<128>::kCtas);
    // tiles of a part for `stay` staying tiles per unit and `stream` streaming ones
    auto cut = [&](long long stay, int stream, int &tiles, int &parts) {
        long long n = units * stay > 0 ? at_once / (units * stay) : 1;
        const int least = up(stream, kMaxTiles);
        if (n < least) n = least;
        if (n > stream) n = stream;
        tiles = n > 0 ? up(stream, n) : 1;
        parts = up(stream, tiles);
    };
    cut(w.row_tiles, w.key_tiles, w.stat_tiles, w.n_stat_parts);
    if (w.row_tiles == 1) cut(1, w.key_tiles, w.sum_tiles, w.n_sum_parts);
    else cut(w.key_tiles, w.row_tiles, w.sum_tiles, w.n_sum_parts);
    const size_t rows = static_cast<size_t>(units) * seq_q * group;
    w.lse = w.n_stat_parts > 1 ? al(rows * w.n_stat_parts * 8) : 0;
    w.sum_parts = w.lse + al(rows * 4);
    w.total = w.sum_parts +
              (w.row_tiles > 1 && w.n_sum_parts > 1 ? al(static_cast<size_t>(units) * seq_k * w.n_sum_parts * 4) : 0);
    return w;
}

template <int HD, int MODE>
int launch_pass(cudaStream_t st, const WParams &p, int x_tiles, int parts)
{
    using S = WShape<HD>;
    static std::mutex mu;
    static bool done[16] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 16) {
        cudaGetLastError();
        return SMOL_B200_ERR_CUDA;
    }
    {
        std::lock_guard<std::mutex> lock(mu);
        if (!done[dev]) {
            if (cudaFuncSetAttribute(weights_kernel<HD, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     S::kSmemBytes) != cudaSuccess) {
                cudaGetLastError();
                return SMOL_B200_ERR_CUDA;
            }
            done[dev] = true;
        }
    }
    const dim3 grid(static_cast<unsigned>(x_tiles) * parts, p.n_kv_heads, p.batch);
    return launch_kernel(weights_kernel<HD, MODE>, grid, dim3(kThreads), S::kSmemBytes, st, p) == cudaSuccess
               ? SMOL_B200_OK
               : SMOL_B200_ERR_CUDA;
}

template <int HD>
int launch_weights(cudaStream_t st, const WParams &p)
{
    int rc = launch_pass<HD, kStats>(st, p, p.row_tiles, p.n_stat_parts);
    if (rc != SMOL_B200_OK) return rc;
    if (p.n_stat_parts > 1) {
        const long long rows = static_cast<long long>(p.batch) * p.n_kv_heads * p.seq_q * p.group;
        int width = 1;
        while (width < 32 && width < p.n_stat_parts) width *= 2;
        if (launch_kernel(weights_lse_kernel, dim3(static_cast<unsigned>((rows * width + 255) / 256)), dim3(256), 0, st,
                          p.lse, static_cast<const float2 *>(p.stat_parts), rows, p.n_stat_parts, width) != cudaSuccess)
            return SMOL_B200_ERR_CUDA;
    }
    if (p.row_tiles == 1) return launch_pass<HD, kSumsOneRowTile>(st, p, 1, p.n_sum_parts);
    return launch_pass<HD, kSums>(st, p, p.key_tiles, p.n_sum_parts);
}

}  // namespace

size_t prefill_weights_workspace_bytes(int batch, int seq_q, int seq_k, int n_heads, int n_kv_heads, int head_dim)
{
    if (batch <= 0 || seq_q < 0 || seq_k < 0 || n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads ||
        n_heads / n_kv_heads > kTile || head_dim <= 0 || head_dim > 256 || head_dim % 8)
        return 0;
    return weights_plan(batch, seq_q, seq_k, n_heads, n_kv_heads, head_dim).total;
}

int prefill_attention_weights(cudaStream_t st, const float *weights_in, float *weights_out, int64_t weights_stride,
                              const uint16_t *q, int64_t q_row_stride, int64_t q_batch_stride, const uint16_t *k,
                              int64_t k_row_stride, int64_t k_batch_stride, int batch, int seq_q, int seq_k,
                              int n_heads, int n_kv_heads, int head_dim, float scale, int mask_kind, int q_offset,
                              int prefix_len, int window, float softcap, void *workspace, size_t workspace_bytes)
{
    if (batch <= 0 || seq_k == 0) return SMOL_B200_OK;
    if (!weights_out || !q || !k || seq_q < 0 || seq_k < 0 || n_heads <= 0 || n_kv_heads <= 0 ||
        n_heads % n_kv_heads != 0 || n_heads / n_kv_heads > kTile || batch > 65535 || n_kv_heads > 65535 ||
        head_dim <= 0 || head_dim > 256 || head_dim % 8 || weights_stride < seq_k || !(scale > 0.f))
        return SMOL_B200_ERR_ARGS;
    if (mask_kind != SMOL_MASK_CAUSAL && mask_kind != SMOL_MASK_PREFIX_LM && mask_kind != SMOL_MASK_FULL)
        return SMOL_B200_ERR_ARGS;
    constexpr int kFar = 1 << 29;   // positions and window differences stay within an int
    if (seq_q > kFar || seq_k > kFar || q_offset > kFar || q_offset < -kFar) return SMOL_B200_ERR_ARGS;
    if (window >= 2 * kFar) window = 0;   // every key
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k)) & 15) return SMOL_B200_ERR_ARGS;
    if ((q_row_stride | k_row_stride) & 7 || (batch > 1 && ((q_batch_stride | k_batch_stride) & 7)))
        return SMOL_B200_ERR_ARGS;
    if (q_row_stride < static_cast<int64_t>(n_heads) * head_dim ||
        k_row_stride < static_cast<int64_t>(n_kv_heads) * head_dim)
        return SMOL_B200_ERR_ARGS;
    const WPlan w = weights_plan(batch, seq_q, seq_k, n_heads, n_kv_heads, head_dim);
    if (!workspace || workspace_bytes < w.total || (reinterpret_cast<uintptr_t>(workspace) & 15))
        return SMOL_B200_ERR_WORKSPACE;
    if (static_cast<long long>(w.row_tiles) * w.n_stat_parts > 0x7fffffffLL ||
        static_cast<long long>(w.key_tiles) * w.n_sum_parts > 0x7fffffffLL)
        return SMOL_B200_ERR_ARGS;

    WParams p;
    memset(&p, 0, sizeof(p));
    p.group = n_heads / n_kv_heads;
    p.qp = w.qp;
    p.weights_in = weights_in;
    p.weights_out = weights_out;
    p.weights_stride = weights_stride;
    p.batch = batch;
    p.seq_q = seq_q;
    p.seq_k = seq_k;
    p.n_kv_heads = n_kv_heads;
    uint8_t *base = static_cast<uint8_t *>(workspace);
    p.stat_parts = reinterpret_cast<float2 *>(base);
    p.lse = reinterpret_cast<float *>(base + w.lse);
    p.sum_parts = reinterpret_cast<float *>(base + w.sum_parts);
    PdlScope pdl(g_api_pdl);
    const bool joined = w.row_tiles > 1 && w.n_sum_parts > 1;
    if (seq_q > 0) {
        const int kernel_hd = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
        const int64_t qb = batch > 1 ? q_batch_stride : static_cast<int64_t>(seq_q) * q_row_stride;
        const int64_t kb = batch > 1 ? k_batch_stride : static_cast<int64_t>(seq_k) * k_row_stride;
        // columns past head_dim read as zero (outside the tensor)
        if (!make_tmap_4d(&p.tq, q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, head_dim, n_heads, seq_q, batch, head_dim,
                          q_row_stride, qb, 64, p.group, w.qp) ||
            !make_tmap_4d(&p.tk, k, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, head_dim, n_kv_heads, seq_k, batch, head_dim,
                          k_row_stride, kb, 64, 1, kTile))
            return SMOL_B200_ERR_CUDA;
        p.q_bytes = kernel_hd / 64 * 128 * p.group * w.qp;
        p.err = device_error_word();
        if (!p.err) return SMOL_B200_ERR_CUDA;
        p.row_tiles = w.row_tiles;
        p.key_tiles = w.key_tiles;
        p.stat_tiles = w.stat_tiles;
        p.n_stat_parts = w.n_stat_parts;
        p.sum_tiles = w.sum_tiles;
        p.n_sum_parts = w.n_sum_parts;
        p.mask_kind = mask_kind;
        p.q_offset = q_offset;
        p.prefix_len = prefix_len;
        p.window = window;
        p.scale = scale;
        p.softcap = softcap;
        const int rc = kernel_hd == 64    ? launch_weights<64>(st, p)
                       : kernel_hd == 128 ? launch_weights<128>(st, p)
                                          : launch_weights<256>(st, p);
        if (rc != SMOL_B200_OK) return rc;
    }
    if (seq_q == 0 || joined) {
        if (launch_kernel(weights_add_kernel, dim3((seq_k + 255) / 256, n_kv_heads, batch), dim3(256), 0, st,
                          weights_out, weights_in, static_cast<long long>(weights_stride),
                          static_cast<const float *>(p.sum_parts), seq_q == 0 ? 0 : w.n_sum_parts, seq_k,
                          n_kv_heads) != cudaSuccess)
            return SMOL_B200_ERR_CUDA;
    }
    return SMOL_B200_OK;
}

}  // namespace smolb200
