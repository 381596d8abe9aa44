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
// (row, key) pair at 16 per clock and SM, 60 us for 4096 causal rows of 16/8 heads of 128,
// which take 109; a pass's products alone take 800 clocks a 128 x 128 tile, its exponentials
// 1000, one waits for the other for 1100 to 1360.  (256-column products, two buffers of S in
// turn: 120 us.)
//
// One persistent CTA per SM.  The visible tiles of all staying tiles, laid end to end, are cut
// into one contiguous run per CTA, so that causal work spreads evenly (whole items of up to
// 8 tiles left the fullest CTA 40 % above the mean) and few rows against many keys still
// fill the GPU; where a run ends inside a staying tile, the pieces are joined in a fixed
// order by a small kernel.  Loads and products run ahead of the exponentials.  Two tiles
// stay where they fit: streaming a tile for 128 rows alone is bound by L2 (11.5 TB/s: 27 us
// of the stats pass at 4096 causal rows, 16/8 heads of 128).
#include <string.h>

#include <mutex>

#include "b200_common.cuh"
#include "fast_math.cuh"
#include "runtime.h"

namespace smolb200 {
namespace {

constexpr int kTile = 128;
constexpr int kGroups = 4;                    // warpgroups of exponentials, a 128-column buffer of S each
constexpr int kExpThreads = kGroups * 128;
constexpr int kThreads = kExpThreads + 64;    // + TMA producer warp, tcgen05 issuer warp
constexpr int kLseRing = 8;                   // row tiles whose lse are in shared memory
constexpr float kSumLimit = 1.152921504606847e18f;   // 2^60: a tile's row sum beyond this moves the reference

// the *OneRowTile forms: at most 128 packed rows per (batch, KV head)
enum Mode { kStats = 0, kSums = 1, kStatsOneRowTile = 2, kSumsOneRowTile = 3 };

template <int HD, int MODE>
struct WShape {
    static constexpr int kSub = HD / 64;
    static constexpr int kSubBytes = kTile * 128;
    static constexpr int kTileBytes = kSub * kSubBytes;
    static constexpr int kStay = HD == 256 || MODE >= kStatsOneRowTile ? 1 : 2;   // tiles that stay
    // A staying tile's streaming tiles go to kWays warpgroups in turn.  Four meet in shared
    // memory at the end of a step, two leave a result each.
    static constexpr int kWays = 4 / kStay;
    static constexpr bool kMeet = kWays == 4 && MODE != kSumsOneRowTile;
    static constexpr int kResults = kMeet ? 1 : kWays;
    static constexpr int kXBytes = kStay * kTileBytes;
    // the next staying tiles load ahead where there is room (stats need no lse beside them)
    static constexpr int kXStages = HD == 64 || (HD == 128 && MODE != kSums) ? 2 : 1;
    static constexpr int kStages = HD == 256 ? 2 : HD == 128 && MODE == kStats ? 3 : 4;
    static constexpr int kRing = MODE == kSums || MODE == kSumsOneRowTile ? kLseRing : 0;
    static constexpr int kOffY = kXStages * kXBytes;
    static constexpr int kOffLse = kOffY + kStages * kTileBytes;
    static constexpr int kOffMeet = kOffLse + kRing * kTile * 4;   // [step parity][warpgroup][128]
    static constexpr int kOffBar = kOffMeet + (kMeet ? 2 * kGroups * kTile * 8 : 0);
    static constexpr int kUsed = kOffBar + 256 + 1024;
    static_assert(kUsed <= 227 * 1024, "shared memory");
    // one CTA per SM: each allocates all 512 TMEM columns
    static constexpr int kSmemBytes = kUsed > 118 * 1024 ? kUsed : 118 * 1024;
};

struct WParams {
    CUtensorMap tq, tk;   // (column, head, row, batch); boxes 64 x group x qp x 1 and 64 x 1 x 128 x 1
    float2 *stat_parts;   // [batch][n_kv_heads][rows][pieces]: reference (log2 units), sum
    float *nlse;          // [batch][n_kv_heads][row_tiles][128]: -lse, log2 units; -inf without keys or row
    float *sum_parts;     // [pieces][batch][n_kv_heads][seq_k]
    const float *weights_in;
    float *weights_out;
    long long weights_stride;
    unsigned *err;
    int batch, seq_q, seq_k, n_kv_heads, group, qp;   // qp: queries of a row tile
    int row_tiles, key_tiles;
    int stay, pieces;               // staying steps per unit; slots of partial results
    long long unit_tiles, run;      // visible streaming tiles (and step costs) of a unit, of a CTA
    long long stat_unit_tiles, stat_run;   // those of the stats pass, for the sums of one row tile
    int stat_pieces;
    int mask_kind, q_offset, prefix_len, window;
    int q_bytes;                    // bytes of a row tile's boxes (all sub-tiles)
    float scale, softcap;
};

struct WBars {
    uint64_t x_full[2], x_empty[2], y_full[4], y_empty[4], d_full[4], d_empty[4], done;
    uint32_t tmem_base;
};

// Keys [lo, hi) that query i sees (both non-decreasing in i).
__host__ __device__ __forceinline__ int imin(int a, int b) { return a < b ? a : b; }
__host__ __device__ __forceinline__ int imax(int a, int b) { return a > b ? a : b; }

__host__ __device__ __forceinline__ void row_keys(const WParams &p, int i, int &lo, int &hi)
{
    const int pos = p.q_offset + i;
    hi = p.mask_kind == SMOL_MASK_CAUSAL      ? pos + 1
         : p.mask_kind == SMOL_MASK_PREFIX_LM ? imax(pos + 1, p.prefix_len)
                                              : p.seq_k;
    hi = imin(imax(hi, 0), p.seq_k);
    lo = p.window > 0 ? imax(0, pos - p.window + 1) : 0;
    if (lo > hi) lo = hi;
}

// Row tiles [t0, t1) with a row that sees a key of [k0, k1).
__host__ __device__ __forceinline__ void key_rows(const WParams &p, int k0, int k1, int &t0, int &t1)
{
    int i0 = 0, i1 = p.seq_q;
    if (p.mask_kind == SMOL_MASK_CAUSAL || (p.mask_kind == SMOL_MASK_PREFIX_LM && k0 >= p.prefix_len))
        i0 = imax(0, k0 - p.q_offset);
    if (p.window > 0) {   // lo < k1: pos <= k1 + window - 2
        const long long last = static_cast<long long>(k1) + p.window - 2 - p.q_offset;
        if (last + 1 < i1) i1 = last + 1 > 0 ? static_cast<int>(last + 1) : 0;
    }
    t0 = i0 / p.qp;
    t1 = i1 > i0 ? (i1 + p.qp - 1) / p.qp : t0;
}

// Streaming tiles [t0, t1) of staying step x (kStay tiles of rows for the stats, of keys for
// the sums).
__host__ __device__ __forceinline__ void stream_range(const WParams &p, int mode, int kstay, int x, int &t0, int &t1)
{
    if (mode == kStats || mode == kStatsOneRowTile) {
        int lo, hi, unused;
        row_keys(p, x * kstay * p.qp, lo, unused);
        const int last = (x + 1) * kstay < p.row_tiles ? (x + 1) * kstay * p.qp : p.seq_q;
        row_keys(p, last - 1, unused, hi);
        t0 = lo / kTile;
        t1 = (hi + kTile - 1) / kTile;
    } else if (mode == kSums) {
        key_rows(p, x * kstay * kTile, (x + 1) * kstay < p.key_tiles ? (x + 1) * kstay * kTile : p.seq_k, t0, t1);
    } else {
        t0 = 0;
        t1 = p.key_tiles;
    }
    if (t1 < t0) t1 = t0;
}

// acc += 2^(v*mul + off) for 16 columns.  MUFU takes 16 cycles of a scheduler for a pair, the
// FMA pipe 4 for its product and sum and 16 more for a polynomial.  kPoly of every 8 pairs go
// there: 111.5 us with 0, 106.3 with 1, 106.5 with 2, 108.8 with 3 (4096 causal rows, 16/8 heads
// of 128).
constexpr int kPoly = 1;
template <typename Off>
__device__ __forceinline__ void add_exp2(const uint32_t (&v)[16], f32x2 mul2, Off &&off, f32x2 &acc0, f32x2 &acc1)
{
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const f32x2 x = fma2(pack2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), mul2, off(i));
        const f32x2 e = (i * kPoly) % 8 < kPoly ? exp2_2_poly(x) : exp2_2(x);
        if (i & 1) acc1 = add2(acc1, e);
        else acc0 = add2(acc0, e);
    }
}

// A staying step costs its CTA time beside its tiles: loads that nothing hides, and for causal
// rows the tiles on the mask's border.  When the runs are cut it counts as this many streaming
// tiles more, in front of its own (fits of the time of each CTA's run, in clocks: stats 2194 a
// tile and 4590 a step, sums 2725 and 786, head dim 128; one row tile: stats 412 and 4638, sums
// 890 and 4369).  4096 causal rows, 16/8 heads: 110.7 us with 1 for all, 106.0 so; 32 rows
// against 16384 keys: 22.2 and 19.4.
__host__ __device__ constexpr int step_cost(int mode)
{
    return mode == kStats ? 2 : mode == kSums ? 1 : mode == kStatsOneRowTile ? 8 : 5;
}

// One CTA's run, staying step by staying step: step x of unit (b, kvh) against streaming tiles
// [t0, t0 + n), as piece `piece` of that step.
struct WRun {
    int unit, x, t0, n, piece;
    long long skip;       // of step x's cost and tiles, what lies before the run
    long long left;       // cost and tiles of the run from there on
};

__device__ __forceinline__ void run_next(WRun &w)
{
    ++w.x;
    w.skip = 0;
    w.piece = 0;
}

template <int HD, int MODE>
__device__ __forceinline__ bool run_step(const WParams &p, WRun &w)
{
    while (w.left > 0) {
        if (w.x == p.stay) {
            w.x = 0;
            if (++w.unit == p.batch * p.n_kv_heads) return false;
        }
        int t0, t1;
        stream_range(p, MODE, WShape<HD, MODE>::kStay, w.x, t0, t1);
        const long long size = t1 > t0 ? t1 - t0 + step_cost(MODE) : 0;
        const long long end = min(size, w.skip + w.left);   // the run's share of the step: [skip, end)
        const int first = static_cast<int>(max(w.skip - step_cost(MODE), 0ll));
        w.t0 = t0 + first;
        w.n = static_cast<int>(max(end - step_cost(MODE), 0ll)) - first;
        w.left -= end - w.skip;
        if (w.n > 0) return true;
        run_next(w);
    }
    return false;
}

// The run of CTA `cta`, found by one warp: tile number cta * run, then the staying step that
// holds it by a scan over the steps of a unit.
template <int HD, int MODE>
__device__ WRun find_run(const WParams &p, int cta)
{
    const int lane = threadIdx.x % 32;
    WRun w;
    const long long start = cta * p.run;
    w.unit = static_cast<int>(start / p.unit_tiles);
    const long long in_unit = start - w.unit * p.unit_tiles;
    const long long all = p.unit_tiles * p.batch * p.n_kv_heads;
    w.left = min(p.run, all - start);
    w.x = 0, w.skip = 0, w.piece = 0, w.t0 = 0, w.n = 0;
    long long before = 0;   // tiles of the steps before this batch of 32
    for (int x0 = 0; x0 < p.stay; x0 += 32) {
        int t0 = 0, t1 = 0;
        if (x0 + lane < p.stay) stream_range(p, MODE, WShape<HD, MODE>::kStay, x0 + lane, t0, t1);
        const int mine = t1 > t0 ? t1 - t0 + step_cost(MODE) : 0;
        int sum = mine;   // inclusive within the warp
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += y;
        }
        const long long first = before + sum - mine;
        const unsigned hit = __ballot_sync(0xffffffffu, first <= in_unit && in_unit < first + mine);
        if (hit) {
            const int l = __ffs(hit) - 1;
            const long long f = __shfl_sync(0xffffffffu, first, l);
            w.x = x0 + l;
            w.skip = in_unit - f;
            w.piece = cta - static_cast<int>((w.unit * p.unit_tiles + f + step_cost(MODE)) / p.run);
            return w;
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    w.left = 0;
    return w;
}

// Runs of length `run` that tiles [first, first + n) lie in.
__device__ __forceinline__ int pieces_at(long long first, int n, long long run)
{
    return n > 0 ? static_cast<int>((first + n - 1) / run - first / run) + 1 : 0;
}

// Pieces of staying step x of `unit` (the whole block asks for one step).
__device__ int step_pieces(const WParams &p, int mode, int kstay, int unit, int x)
{
    __shared__ long long s_sum[32];
    long long sum = 0;
    for (int i = threadIdx.x; i < x; i += blockDim.x) {
        int t0, t1;
        stream_range(p, mode, kstay, i, t0, t1);
        if (t1 > t0) sum += t1 - t0 + step_cost(mode);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (threadIdx.x % 32 == 0) s_sum[threadIdx.x / 32] = sum;
    __syncthreads();
    long long f = unit * p.unit_tiles + step_cost(mode);
    for (int i = 0; i < static_cast<int>(blockDim.x / 32); ++i) f += s_sum[i];
    int t0, t1;
    stream_range(p, mode, kstay, x, t0, t1);
    return pieces_at(f, t1 - t0, p.run);
}

// A piece (reference, sum) of a row's statistics counted from M.  Without a reference its sum is
// 0 (no key seen) or NaN (every score is), which has to reach the row.
__device__ __forceinline__ float piece_sum(float2 v, float M)
{
    return v.x == -INFINITY ? v.y : v.y * fast_exp2f(v.x - M);
}
__device__ __forceinline__ float negative_lse(float M, float L)
{
    return M == -INFINITY && L == 0.f ? -INFINITY : -(M + log2f(L));
}

__device__ __forceinline__ const float *lse_of(const WParams &p, int unit, int row_tile)
{
    return p.nlse + (static_cast<long long>(unit) * p.row_tiles + row_tile) * kTile;
}

// `bytes` (a multiple of 16, both addresses too) from global to shared memory, counted by `bar`.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
                 : "memory");
}

template <int HD, int MODE>
__global__ void __launch_bounds__(kThreads, 1) weights_kernel(const __grid_constant__ WParams p)
{
    using S = WShape<HD, MODE>;
    constexpr int ST = S::kStages, XS = S::kXStages, NX = S::kStay;
    constexpr int kProducer = kGroups * 4, kIssuer = kProducer + 1;
    constexpr bool kOne = MODE == kSumsOneRowTile, kRows = MODE == kStats || MODE == kStatsOneRowTile;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    WBars *bars = reinterpret_cast<WBars *>(smem + S::kOffBar);
    static_assert(sizeof(WBars) <= 256, "barriers");
    if (threadIdx.x == 0) {
        for (int s = 0; s < XS; ++s) {
            mbar_init(smem_u32(&bars->x_full[s]), 1);
            mbar_init(smem_u32(&bars->x_empty[s]), 1);
        }
        for (int s = 0; s < ST; ++s) {
            mbar_init(smem_u32(&bars->y_full[s]), 1);
            mbar_init(smem_u32(&bars->y_empty[s]), 1);
        }
        for (int s = 0; s < 4; ++s) {
            mbar_init(smem_u32(&bars->d_full[s]), 1);
            mbar_init(smem_u32(&bars->d_empty[s]), 128);
        }
        mbar_init(smem_u32(&bars->done), 1);
        fence_mbar_init();
    }
    // a row tile fills qp*group of each 128 rows; the rest must be finite
    if (p.qp * p.group < kTile) {
        for (int i = threadIdx.x; i < S::kOffLse / 16; i += kThreads)
            *reinterpret_cast<uint4 *>(smem + i * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
    }
    WRun w = find_run<HD, MODE>(p, blockIdx.x);
    // Everything above is the kernel's own and may run while the kernels before this one finish.
    // TMEM only after the wait: a CTA that held it while an earlier kernel's CTA on the same SM
    // still had to allocate would wait for that kernel for good.
    griddep_wait();
    griddep_trigger();
    if (warp == kIssuer) {
        tmem_alloc(smem_u32(&bars->tmem_base), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bars->tmem_base;

    if (warp == kProducer) {
        // ================= TMA producer =================
        if (lane == 0) {
            tma_prefetch_desc(&p.tq);
            tma_prefetch_desc(&p.tk);
            // 128 rows of the queries (rows: row tile t) or keys (key tile t); past the last: zeros
            auto load = [&](uint32_t dst, uint32_t bar, bool rows, int t) {
                const int b = w.unit / p.n_kv_heads, kvh = w.unit % p.n_kv_heads;
#pragma unroll
                for (int sub = 0; sub < S::kSub; ++sub) {
                    if (rows) tma_load_4d(dst + sub * S::kSubBytes, &p.tq, bar, sub * 64, kvh * p.group, t * p.qp, b);
                    else tma_load_4d(dst + sub * S::kSubBytes, &p.tk, bar, sub * 64, kvh, t * kTile, b);
                }
            };
            int nx = 0, ny = 0;   // staying steps, streaming tiles issued
            bool ok = true;
            for (; ok && run_step<HD, MODE>(p, w); run_next(w)) {
                const int xs = nx % XS;
                if (nx >= XS && !(ok = mbar_wait(smem_u32(&bars->x_empty[xs]), (nx / XS - 1) & 1, p.err, kErrWaitTmaEmpty)))
                    break;
                const uint32_t xb = smem_u32(&bars->x_full[xs]);
                mbar_arrive_expect_tx(xb, NX * (MODE == kSums ? S::kTileBytes : p.q_bytes));
#pragma unroll
                for (int i = 0; i < NX; ++i)
                    load(smem_u32(smem + xs * S::kXBytes + i * S::kTileBytes), xb, MODE != kSums, w.x * NX + i);
                ++nx;
                for (int t = 0; t < w.n; ++t, ++ny) {
                    const int st = ny % ST;
                    if (ny >= ST &&
                        !(ok = mbar_wait(smem_u32(&bars->y_empty[st]), (ny / ST - 1) & 1, p.err, kErrWaitTmaEmpty)))
                        break;
                    const uint32_t yb = smem_u32(&bars->y_full[st]);
                    mbar_arrive_expect_tx(yb, MODE == kSums ? p.q_bytes + kTile * 4 : S::kTileBytes);
                    load(smem_u32(smem + S::kOffY + st * S::kTileBytes), yb, MODE == kSums, w.t0 + t);
                    if (MODE == kSums)   // a slot is free 8 tiles later: S of those was read before Y's slot was
                        bulk_load(smem_u32(smem + S::kOffLse) + ny % kLseRing * kTile * 4, lse_of(p, w.unit, w.t0 + t),
                                  kTile * 4, yb);
                }
            }
            for (int i = max(0, nx - XS); i < nx; ++i)
                if (!mbar_wait(smem_u32(&bars->x_full[i % XS]), (i / XS) & 1, p.err, kErrDrain)) break;
            for (int i = max(0, ny - ST); i < ny; ++i)
                if (!mbar_wait(smem_u32(&bars->y_full[i % ST]), (i / ST) & 1, p.err, kErrDrain)) break;
        }
    } else if (warp == kIssuer) {
        // ================= tcgen05 issuer =================
        constexpr uint32_t idesc = umma_idesc_f16(kTile, kTile, true, false);
        int nx = 0, ny = 0;
        bool ok = true;
        for (; ok && run_step<HD, MODE>(p, w); run_next(w)) {
            const int xs = nx % XS;
            ok = mbar_wait_warp(smem_u32(&bars->x_full[xs]), (nx / XS) & 1, p.err, kErrWaitTmaFull);
            for (int t = 0; t < w.n && ok; ++t, ++ny) {
                const int st = ny % ST;
                ok = mbar_wait_warp(smem_u32(&bars->y_full[st]), (ny / ST) & 1, p.err, kErrWaitTmaFull);
                const uint32_t y_addr = smem_u32(smem + S::kOffY + st * S::kTileBytes);
#pragma unroll
                for (int i = 0; i < NX; ++i) {
                    const int n = ny * NX + i, d = n % 4;   // buffers of S in turn
                    if (ok && n >= 4) ok = mbar_wait_warp(smem_u32(&bars->d_empty[d]), (n / 4 - 1) & 1, p.err, kErrWaitSoftmax);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t x_addr = smem_u32(smem + xs * S::kXBytes + i * S::kTileBytes);
#pragma unroll
                    for (int kk = 0; kk < HD / 16; ++kk) {
                        const uint32_t off = (kk >> 2) * S::kSubBytes + (kk & 3) * 32;
                        const uint64_t xd = umma_sdesc_sw128(x_addr + off, 16, 1024);
                        const uint64_t yd = umma_sdesc_sw128(y_addr + off, 16, 1024);
                        // rows of S: the side that is not summed over
                        umma_ss_elect(tmem + d * kTile, kOne ? yd : xd, kOne ? xd : yd, idesc, kk > 0 ? 1u : 0u);
                    }
                    umma_commit_elect(smem_u32(&bars->d_full[d]));
                }
                umma_commit_elect(smem_u32(&bars->y_empty[st]));
            }
            umma_commit_elect(smem_u32(&bars->x_empty[xs]));
            ++nx;
        }
        umma_commit_elect(smem_u32(&bars->done));
        mbar_wait_warp(smem_u32(&bars->done), 0, p.err, kErrDrain);
    } else {
        // ================= exponentials: thread r of a warpgroup owns row r of S =================
        // Use n of the buffers of S (streaming tile g0 + t of this CTA, staying tile i: n = (g0 + t) *
        // NX + i) is buffer n % 4, and warpgroup n % 4 reads it.
        const int wg = warp / 4, r = threadIdx.x % kTile;
        const int stay = wg % NX;                       // the staying tile this warpgroup works for
        constexpr int kStep = 4 / NX;                   // and every kStep-th streaming tile of the CTA
        const uint32_t s_col = tmem + (static_cast<uint32_t>((warp % 4) * 32) << 16) + wg * kTile;
        const uint32_t d_full = smem_u32(&bars->d_full[wg]), d_empty = smem_u32(&bars->d_empty[wg]);
        const float cap = p.softcap, inv_cap = cap > 0.f ? 1.f / cap : 0.f;
        const float mul = cap > 0.f ? 1.f : p.scale * kLog2e;
        const f32x2 mul2 = pack2(mul, mul);
        const long long rows = static_cast<long long>(p.seq_q) * p.group;
        bool ok = true;   // false after a wait that ran out (the device error word is set)
        auto capped = [&](uint32_t (&v)[16]) {
            if (cap > 0.f) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    v[i] = __float_as_uint(cap * tanhf(__uint_as_float(v[i]) * p.scale * inv_cap) * kLog2e);
            }
        };
        // columns outside [lo, hi) become -inf: their exponentials are 0 whatever the scores hold
        auto hide = [](int c0, uint32_t (&v)[16], int lo, int hi) {
#pragma unroll
            for (int c = 0; c < 16; ++c)
                if (c0 + c < lo || c0 + c >= hi) v[c] = 0xff800000u;
        };
        auto total = [](f32x2 a, f32x2 b) -> float {
            float x, y;
            unpack2(add2(a, b), x, y);
            return x + y;
        };
        // sum of 2^(S - lse) over columns [lo, hi) of this warpgroup's buffer, lse (negated) in
        // shared memory; `whole`: over all n16 * 16
        auto tile_sum = [&](const float *nl, int n16, bool whole, int lo, int hi) -> float {
            if (whole) {
                f32x2 acc0 = 0, acc1 = 0;
                for_columns(s_col, n16, [&](int c0, uint32_t (&v)[16]) {
                    capped(v);
                    ulonglong2 o[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[i] = *reinterpret_cast<const ulonglong2 *>(nl + c0 + 4 * i);
                    add_exp2(v, mul2, [&](int i) { return i & 1 ? o[i / 2].y : o[i / 2].x; }, acc0, acc1);
                });
                const float s = total(acc0, acc1);
                // beyond any sum of 128 probabilities: a NaN or an infinity, which MUFU alone keeps
                if (!__any_sync(0xffffffffu, !(s <= kSumLimit))) return s;
            }
            float s = 0.f;
            for_columns(s_col, n16, [&](int c0, uint32_t (&v)[16]) {
                capped(v);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float y = fast_exp2f(fmaf(__uint_as_float(v[i]), mul, nl[c0 + i]));
                    if (c0 + i >= lo && c0 + i < hi) s += y;
                }
            });
            return s;
        };
        // Columns [lo, hi) of row tile t whose rows see key `key` (rows see contiguous keys, in order,
        // so a key is seen by contiguous rows).
        auto columns_of = [&](int key, int t, int &lo, int &hi) {
            const int q0 = p.q_offset + t * p.qp;   // position of the tile's first query
            long long first = 0, last = p.qp;       // queries [first, last) of the tile
            if (p.mask_kind == SMOL_MASK_CAUSAL || (p.mask_kind == SMOL_MASK_PREFIX_LM && key >= p.prefix_len))
                first = key - q0;
            if (p.window > 0) last = static_cast<long long>(key) + p.window - q0;
            const int used = min(p.qp, p.seq_q - t * p.qp);
            lo = static_cast<int>(min(max(first, 0ll), static_cast<long long>(used))) * p.group;
            hi = static_cast<int>(min(max(last, 0ll), static_cast<long long>(used))) * p.group;
        };

        int g0 = 0, steps = 0;             // streaming tiles and staying steps before this one
        int one_unit = -1, one_slot = 0;   // one row tile: the unit whose lse are in shared memory, and where
        for (; run_step<HD, MODE>(p, w); run_next(w), ++steps) {
            const int n = w.n;
            const long long unit = w.unit;
            const int first = (wg / NX - g0 % kStep + kStep) % kStep;
            if constexpr (kRows) {
                const int rt = w.x * NX + stay;
                const int i = rt * p.qp + r / p.group;
                const bool valid = r < p.qp * p.group && i < p.seq_q;
                int lo = 0, hi = 0;
                if (valid) row_keys(p, i, lo, hi);
                float m = -INFINITY, l = 0.f;
                for (int t = first; t < n; t += kStep) {
                    if (ok) ok = mbar_wait_warp(d_full, ((g0 + t) / kStep) & 1, p.err, kErrWaitMma);
                    const int key0 = (w.t0 + t) * kTile;
                    // a warp none of whose rows sees a key of the tile skips it
                    if (ok && __any_sync(0xffffffffu, valid && key0 < hi && key0 + kTile > lo)) {
                        tc_fence_after();
                        // rows past the last one may see anything: they are not stored
                        const bool whole = __all_sync(0xffffffffu, !valid || (key0 >= lo && key0 + kTile <= hi));
                        // fp32 sums need no maximum close by, only no overflow: a row's reference is a
                        // maximum of the first tile it meets (of 16 scores where it sees them all) and
                        // moves when a tile's sum passes 2^60
                        bool need = __any_sync(0xffffffffu, m == -INFINITY && key0 < hi && key0 + kTile > lo);
                        float lt = 0.f;
                        for (int pass = 0; pass < 2; ++pass) {
                            if (need) {
                                float mx = -INFINITY;
                                for_columns(s_col, whole && pass == 0 ? 1 : kTile / 16, [&](int c0, uint32_t (&v)[16]) {
                                    if (!whole) hide(c0, v, lo - key0, hi - key0);
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
                            const f32x2 neg2 = pack2(negm, negm);
                            if (whole && pass == 0) {
                                f32x2 acc0 = 0, acc1 = 0;
                                for_columns(s_col, kTile / 16, [&](int c0, uint32_t (&v)[16]) {
                                    capped(v);
                                    add_exp2(v, mul2, [&](int) { return neg2; }, acc0, acc1);
                                });
                                lt = total(acc0, acc1);
                            } else {   // the border of the mask; scores that passed the limit, NaN among them
                                float acc[2] = {0.f, 0.f};
                                for_columns(s_col, kTile / 16, [&](int c0, uint32_t (&v)[16]) {
                                    capped(v);
                                    if (!whole) hide(c0, v, lo - key0, hi - key0);
#pragma unroll
                                    for (int c = 0; c < 16; ++c)
                                        acc[c & 1] += fast_exp2f(fmaf(__uint_as_float(v[c]), mul, negm));
                                });
                                lt = acc[0] + acc[1];
                            }
                            need = __any_sync(0xffffffffu, !(lt <= kSumLimit));
                            if (!need) break;
                        }
                        l += lt;
                        tc_fence_before();
                    }
                    mbar_arrive(d_empty);
                }
                if (!ok) m = -INFINITY, l = 0.f;
                if (S::kMeet) {
                    float2 *box = reinterpret_cast<float2 *>(smem + S::kOffMeet) + (steps & 1) * kGroups * kTile;
                    box[wg * kTile + r] = make_float2(m, l);
                    named_bar_sync(1, kExpThreads);
                    if (wg == 0) {
                        for (int i = 1; i < kGroups; ++i) m = fmaxf(m, box[i * kTile + r].x);
                        l = 0.f;
                        for (int i = 0; i < kGroups; ++i) {
                            const float2 v = box[i * kTile + r];
                            l += piece_sum(v, m);
                        }
                    }
                }
                if (valid && (!S::kMeet || wg == 0))
                    p.stat_parts[(unit * rows + static_cast<long long>(rt) * p.qp * p.group + r) * p.pieces +
                                 w.piece * S::kResults + (S::kMeet ? 0 : wg / NX)] = make_float2(m, l);
            } else {
                const int used = kOne ? (min(p.qp, p.seq_q) * p.group + 15) / 16 : kTile / 16;
                float *ring = reinterpret_cast<float *>(smem + S::kOffLse);
                if (kOne && one_unit != w.unit) {
                    // the rows' -lse from their pieces, four lanes to a row
                    one_unit = w.unit;
                    one_slot ^= 1;
                    int t0, t1;
                    stream_range(p, kStatsOneRowTile, 1, 0, t0, t1);
                    const int pieces = pieces_at(w.unit * p.stat_unit_tiles + step_cost(kStatsOneRowTile), t1 - t0, p.stat_run);
                    const int row = threadIdx.x / 4, part = threadIdx.x % 4;
                    const float2 *src = p.stat_parts + (unit * rows + row) * p.stat_pieces;
                    float M = -INFINITY, L = 0.f;
                    if (row < rows)
                        for (int c = part; c < pieces; c += 4) M = fmaxf(M, src[c].x);
                    M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, 1));
                    M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, 2));
                    if (row < rows)
                        for (int c = part; c < pieces; c += 4) {
                            const float2 v = src[c];
                            L += piece_sum(v, M);
                        }
                    L += __shfl_xor_sync(0xffffffffu, L, 1);
                    L += __shfl_xor_sync(0xffffffffu, L, 2);
                    if (part == 0) ring[one_slot * kTile + row] = negative_lse(M, L);
                    named_bar_sync(1, kExpThreads);   // the slot before is still read: two in turn
                }
                float sum = 0.f;
                for (int t = first; t < n; t += kStep) {
                    // this thread's key, and the row tile
                    const int key = (kOne ? w.t0 + t : w.x * NX + stay) * kTile + r, rt = kOne ? 0 : w.t0 + t;
                    const long long at = unit * p.weights_stride + key;
                    const float before = kOne && p.weights_in && key < p.seq_k ? p.weights_in[at] : 0.f;
                    int lo, hi;
                    columns_of(key, rt, lo, hi);
                    // columns past the tile's rows have -lse = -inf: they add 0, or the polynomial's least value
                    // 2^-126, which only a sum that is itself next to the smallest normal float shows
                    const bool whole = __all_sync(0xffffffffu, lo == 0 && hi == min(p.qp, p.seq_q - rt * p.qp) * p.group);
                    if (ok) ok = mbar_wait_warp(d_full, ((g0 + t) / kStep) & 1, p.err, kErrWaitMma);
                    float one = 0.f;
                    if (ok && __any_sync(0xffffffffu, hi > lo && key < p.seq_k)) {
                        tc_fence_after();
                        one = tile_sum(ring + (kOne ? one_slot : (g0 + t) % kLseRing) * kTile, used, whole, lo, hi);
                        tc_fence_before();
                    }
                    mbar_arrive(d_empty);
                    if (!kOne) sum += one;
                    else if (key < p.seq_k) p.weights_out[at] = before + one;
                }
                if (!kOne) {
                    const int key = (w.x * NX + stay) * kTile + r;
                    if (S::kMeet) {
                        float *box = reinterpret_cast<float *>(smem + S::kOffMeet) + (steps & 1) * kGroups * kTile;
                        box[wg * kTile + r] = sum;
                        named_bar_sync(1, kExpThreads);
                        if (wg == 0) sum = (box[r] + box[kTile + r]) + (box[2 * kTile + r] + box[3 * kTile + r]);
                    }
                    if (key < p.seq_k && (!S::kMeet || wg == 0))
                        p.sum_parts[(static_cast<long long>(w.piece * S::kResults + (S::kMeet ? 0 : wg / NX)) * p.batch *
                                         p.n_kv_heads + unit) * p.seq_k + key] = sum;
                }
            }
            g0 += n;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kIssuer) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// -lse of the rows of a row tile from their pieces, `width` (a power of two, 2 to 32) lanes to
// a row and 256 / width rows to a block: 128 entries a tile, -inf where no row is.
__global__ void __launch_bounds__(256) weights_lse_kernel(const __grid_constant__ WParams p, int kstay, int results, int width)
{
    griddep_wait();
    griddep_trigger();
    const int blocks = kTile * width / 256;   // of a tile
    const int unit = blockIdx.y, tile = blockIdx.x / blocks;
    const int n = step_pieces(p, kStats, kstay, unit, tile / kstay) * results;
    const int lane = threadIdx.x % width, in_tile = blockIdx.x % blocks * (256 / width) + threadIdx.x / width;
    const long long rows = static_cast<long long>(p.seq_q) * p.group;
    const long long row = static_cast<long long>(tile) * p.qp * p.group + in_tile;
    const bool valid = in_tile < p.qp * p.group && row < rows;
    const float2 *src = p.stat_parts + (unit * rows + row) * p.pieces;
    float M = -INFINITY, L = 0.f;
    if (valid)
        for (int c = lane; c < n; c += width) M = fmaxf(M, src[c].x);
    for (int o = width / 2; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    if (valid)
        for (int c = lane; c < n; c += width) {
            const float2 v = src[c];
            L += piece_sum(v, M);
        }
    for (int o = width / 2; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    if (lane == 0)
        p.nlse[(static_cast<long long>(unit) * p.row_tiles + tile) * kTile + in_tile] = negative_lse(M, L);
}

// weights_out = weights_in + the pieces of each key tile, in order (kstay 0: a copy).
__global__ void __launch_bounds__(kTile) weights_add_kernel(const __grid_constant__ WParams p, int kstay, int results)
{
    griddep_wait();
    griddep_trigger();
    const int unit = blockIdx.y;
    const int j = blockIdx.x * kTile + threadIdx.x;
    const int n = kstay > 0 ? step_pieces(p, kSums, kstay, unit, blockIdx.x / kstay) * results : 0;
    if (j >= p.seq_k) return;
    const long long units = static_cast<long long>(p.batch) * p.n_kv_heads;
    float s = 0.f;
#pragma unroll 4
    for (int c = 0; c < n; ++c) s += p.sum_parts[(c * units + unit) * p.seq_k + j];
    const long long at = unit * p.weights_stride + j;
    p.weights_out[at] = (p.weights_in ? p.weights_in[at] : 0.f) + s;
}

// Sizes that do not depend on the mask.  A run is no shorter than a `most`-th of the streaming
// tiles, so a staying step lies in at most most + 1 runs.
struct WPlan {
    int qp, row_tiles, key_tiles;
    int stat_kstay, stat_stay, stat_most, sum_kstay, sum_stay, sum_most;
    int stat_pieces, sum_pieces, results;   // slots of a row / key; results of a piece (not one row tile)
    size_t lse, sums, total;   // the stats pieces at 0
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
    const bool one = w.row_tiles <= 1;
    const int two = head_dim > 128 ? 1 : 2;
    auto most = [&](long long stay, int stream) {
        const long long n = units * stay > 0 ? up(148, units * stay) : 1;
        return static_cast<int>(n < 8 ? (stream < 8 ? stream : 8) : (n < stream ? n : stream));
    };
    w.stat_kstay = one ? 1 : two;
    w.stat_stay = up(w.row_tiles, w.stat_kstay);
    w.stat_most = most(w.stat_stay, w.key_tiles);
    w.results = two == 2 ? WShape<128, kStats>::kResults : WShape<256, kStats>::kResults;
    w.stat_pieces = (w.stat_most + 1) * (one ? WShape<128, kStatsOneRowTile>::kResults : w.results);
    w.sum_kstay = one ? 1 : two;
    w.sum_stay = one ? 1 : up(w.key_tiles, two);
    w.sum_most = one ? up(148, units) : most(w.sum_stay, w.row_tiles);
    w.sum_pieces = one ? 0 : (w.sum_most + 1) * w.results;
    const size_t rows = static_cast<size_t>(units) * seq_q * group;
    w.lse = al(rows * w.stat_pieces * 8);
    w.sums = w.lse + al(static_cast<size_t>(units) * w.row_tiles * kTile * 4);
    w.total = w.sums + al(static_cast<size_t>(units) * seq_k * w.sum_pieces * 4);
    return w;
}

int sm_count()
{
    static int cached[16] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 16) {
        cudaGetLastError();
        return 0;
    }
    if (!cached[dev] && cudaDeviceGetAttribute(&cached[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    return cached[dev];
}

// Completes p for one pass (the runs, from the mask) and launches it.
template <int HD, int MODE>
int launch_pass(cudaStream_t st, WParams &p, int stay, int stream, int most, int pieces)
{
    using S = WShape<HD, MODE>;
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
    p.stay = stay;
    p.pieces = pieces;
    p.unit_tiles = 0;
    for (int x = 0; x < stay; ++x) {
        int t0, t1;
        stream_range(p, MODE, S::kStay, x, t0, t1);
        if (t1 > t0) p.unit_tiles += t1 - t0 + step_cost(MODE);
    }
    const long long all = p.unit_tiles * p.batch * p.n_kv_heads;
    const int sms = sm_count();
    if (sms <= 0) return SMOL_B200_ERR_CUDA;
    p.run = (all + sms - 1) / sms;
    const long long least = (stream + most - 1) / (most > 0 ? most : 1);
    if (p.run < least) p.run = least;
    if (p.run < 1) p.run = 1;
    if (all == 0) return SMOL_B200_OK;   // no row sees a key
    const dim3 grid(static_cast<unsigned>((all + p.run - 1) / p.run));
    return launch_kernel(weights_kernel<HD, MODE>, grid, dim3(kThreads), S::kSmemBytes, st, p) == cudaSuccess
               ? SMOL_B200_OK
               : SMOL_B200_ERR_CUDA;
}

template <int HD>
int launch_weights(cudaStream_t st, WParams &p, const WPlan &w)
{
    const unsigned units = static_cast<unsigned>(p.batch) * p.n_kv_heads;
    if (w.row_tiles == 1) {
        const int rc = launch_pass<HD, kStatsOneRowTile>(st, p, w.stat_stay, w.key_tiles, w.stat_most, w.stat_pieces);
        if (rc != SMOL_B200_OK) return rc;
        p.stat_unit_tiles = p.unit_tiles;
        p.stat_run = p.run;
        p.stat_pieces = w.stat_pieces;
        return launch_pass<HD, kSumsOneRowTile>(st, p, 1, w.key_tiles, w.sum_most, 0);
    }
    int rc = launch_pass<HD, kStats>(st, p, w.stat_stay, w.key_tiles, w.stat_most, w.stat_pieces);
    if (rc != SMOL_B200_OK) return rc;
    // about four results a lane: a step lies in at most key_tiles / run + 2 runs
    long long pieces = (w.key_tiles / p.run + 2) * w.results;
    if (pieces > w.stat_pieces) pieces = w.stat_pieces;
    int width = 2;
    while (width < 32 && width * 4 < pieces) width *= 2;
    if (launch_kernel(weights_lse_kernel, dim3(static_cast<unsigned>(w.row_tiles) * (kTile * width / 256), units),
                      dim3(256), 0, st, p, w.stat_kstay, w.results, width) != cudaSuccess)
        return SMOL_B200_ERR_CUDA;
    rc = launch_pass<HD, kSums>(st, p, w.sum_stay, w.row_tiles, w.sum_most, w.sum_pieces);
    if (rc != SMOL_B200_OK) return rc;
    return launch_kernel(weights_add_kernel, dim3(w.key_tiles, units), dim3(kTile), 0, st, p, w.sum_kstay, w.results) ==
                   cudaSuccess
               ? SMOL_B200_OK
               : SMOL_B200_ERR_CUDA;
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
    if (static_cast<long long>(seq_q) * (n_heads / n_kv_heads) > 0x7fffffffLL ||
        static_cast<long long>(batch) * n_kv_heads > 65535)
        return SMOL_B200_ERR_ARGS;   // row numbers, the grids of the joining kernels
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
    p.nlse = reinterpret_cast<float *>(base + w.lse);
    p.sum_parts = reinterpret_cast<float *>(base + w.sums);
    PdlScope pdl(g_api_pdl);
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
        p.mask_kind = mask_kind;
        p.q_offset = q_offset;
        p.prefix_len = prefix_len;
        p.window = window;
        p.scale = scale;
        p.softcap = softcap;
        const int rc = kernel_hd == 64    ? launch_weights<64>(st, p, w)
                       : kernel_hd == 128 ? launch_weights<128>(st, p, w)
                                          : launch_weights<256>(st, p, w);
        if (rc != SMOL_B200_OK) return rc;
    }
    if (seq_q == 0 && launch_kernel(weights_add_kernel, dim3(w.key_tiles, batch * n_kv_heads), dim3(kTile), 0, st, p, 0,
                                    0) != cudaSuccess)
        return SMOL_B200_ERR_CUDA;
    return SMOL_B200_OK;
}

}  // namespace smolb200
