// decode_shared.cu -- single-token decode over a pooled cache with rows that many
// sequences share, and with each key's attention probability added to a running weight.
//
// For query head h of sequence b, over the visible keys j of its shared prefix and its
// own rows:  x_j = scale * q.k_j (capped),  out = sum_j e^(x_j - m) v_j / sum_j e^(x_j - m).
// The sums split over any partition of the keys, each part with its own m, so three
// kernels do one step:
//   prefix  the rows of a shared prefix against the query heads of ALL its sequences, on
//           tcgen05: a 128-row tile holds (sequence, head of the KV group) pairs, so a
//           prefix row is read once per tile instead of once per sequence (kFewRows packed
//           rows at most: left to the split kernel);
//   split   every sequence's own rows (mma.sync over a TMA ring, keys as the M dimension);
//           with weights it also keeps the scores of the own keys;
//   merge   combines the parts of a row and, with weights, adds
//           sum_h e^(x_hj - M_h) / L_h to the weight of own key j.
// Bound: HBM for large batches (decode weights, 64 sequences of 1024 to 8192 keys, 8 KV heads of
// 128: 202 us for 1.23 GB, 0.93 of the copy rate), latency for small ones (one sequence of 513
// keys: 6.6 us, two launches).
//
// Precision.  Scores, maxima, sums and outputs of the parts are fp32.  K is bf16 and V
// fp16 in the cache.  fp32 queries enter the bf16 products as three bf16 terms (24 bits:
// two left the scores 4e-6 off), bf16 queries as they are.  The probabilities multiply V
// as an fp16 value and its remainder (2^-23), for bf16 outputs too: their one rounding is
// that of the output.  (The value alone is 2^-12 off, which turned one bf16 output in 11 to
// its neighbour; the remainder costs 64 sequences on 8192 shared keys 48.6 us against 46.4,
// 64 sequences of 1024 to 8192 own keys 202.6 against 201.2.)
#include <string.h>

#include <mutex>

#include "b200_common.cuh"
#include "fast_math.cuh"
#include "runtime.h"

namespace smolb200 {
namespace {

constexpr int kSms = 148;

struct SharedParams {
    CUtensorMap tk, tv;             // [pool_rows, kv_dim], boxes of 64 columns x 64 rows (PrefixShape's kBoxRows)
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
    unsigned group_inv;             // ceil(2^31 / group): (u * group_inv) >> 31 is u / group while u * group < 2^31
    int n_prefixes, max_prefix_len, max_prefix_seqs;
    int idle_prefixes;              // prefixes announced without rows or sequences: only looked over
    int prefix_chunk, prefix_slots; // keys of one prefix part; parts of the longest prefix
    int prefix_qtiles;              // query tiles of the largest group (few rows: of 8 rows)
    int prefix_items;               // query tiles x parts x KV heads x prefixes; 0: few rows
    int prefix_ctas;                // CTAs of the prefix kernel at most
    int prefix_units;               // few rows: query tiles x prefixes, taken by the split kernel
    int chunk, max_chunks;          // the same for own rows
    int slots;                      // prefix_slots + max_chunks
    int max_kv_len, score_rows, score_cols;
    int window;
    float scale, softcap;
};

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
    bool bad = s0 < 0 || s1 > p.n_seqs || s0 > s1 || len < 0 || len > p.max_prefix_len;
    s0 = min(max(s0, 0), p.n_seqs);   // any values: 0 <= s0 <= s1 <= n_seqs
    s1 = max(min(s1, p.n_seqs), s0);
    len = min(max(len, 0), p.max_prefix_len);
    if (s1 - s0 > p.max_prefix_seqs) {
        s1 = s0 + p.max_prefix_seqs;
        bad = true;
    }
    if (bad && flag) atomicOr(p.err, kErrBadArgs);
}

// Own keys [ks, n) that a sequence of kv_len rows sees; n is clipped to max_kv_len.
__device__ __forceinline__ void own_keys(const SharedParams &p, int kv_len, int &ks, int &n)
{
    n = min(max(kv_len, 0), p.max_kv_len);
    ks = (p.window > 0 && n > p.window) ? n - p.window : 0;
}
__device__ __forceinline__ void own_range(const SharedParams &p, int b, int &ks, int &n)
{
    own_keys(p, p.kv_len[b], ks, n);
}

// ===========================================================================
// prefix
// ===========================================================================
// Item = (query tile, part of the keys, KV head, prefix); persistent CTAs take items in turn:
// softmax warpgroups of one packed row per thread (thread = TMEM lane), a TMA producer warp
// that runs ahead into the next item, and a tcgen05 issuer warp.
//   S = Q K^T  (QT bf16 terms of Q, fp32 in TMEM, two buffers)
//   P = 2^(S*scale*log2e - m) as an fp16 value and its remainder over S's columns
//   O += P V
// Head dims 64 and 128 run two softmax warpgroups on alternate key tiles, each with an O
// and a reference point of its own, joined at the end: the exponentials of a tile take
// longer than its products (one warpgroup left the tensor pipe 34 % busy).  Head dim 256,
// whose O fills half of TMEM, runs one.
// Row r of tile t is query head (r' % group) of sequence s0 + r'/group, r' = 128 t + r.
constexpr int kBM = 128;
// A row's reference point lies kHeadLog2 below the maximum it is taken from and moves when a
// later maximum lies kMoveLog2 above that one, so the largest probability of a row is 2^7 to 2^15:
// fp16 holds 65504, and what its steps of 2^-24 below 2^-14 cost a small probability counts
// against 2^7 (with the maximum at 1, 900 keys at 2^-22.3 beside a sink without value were 8 % off).
constexpr float kHeadLog2 = 7.0f, kMoveLog2 = 8.0f;

template <int HD, int QT>
struct PrefixShape {
    // Key tile: 128; 64 / 32 where the query terms of head dim 256 (64 KB each) leave less room.
    static constexpr int BN = HD == 256 ? (QT == 3 ? 32 : 64) : 128;
    static constexpr int kStages = HD == 256 && QT == 3 ? 1 : 2;
    static constexpr int kBoxRows = BN < 64 ? BN : 64;   // of a TMA copy: 64 fits the split kernel too
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
    // once an item's products are complete its Q makes room for the warpgroups' (m, l) and
    // then for 2 KB of staged output per warp
    static_assert(kGroups * 4 * 2048 <= kQTermBytes, "staging");
};

struct PrefixBars {
    uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_done[2], o_final, mma_done;
    uint32_t tmem_base;
};

// Query tiles and parts of prefix g.
__device__ __forceinline__ int prefix_tiles(const SharedParams &p, int s0, int s1)
{
    return s1 > s0 ? ((s1 - s0) * p.group + kBM - 1) / kBM : 0;
}
__device__ __forceinline__ int prefix_parts_of(const SharedParams &p, int plen)
{
    return (plen + p.prefix_chunk - 1) / p.prefix_chunk;
}

// One item's geometry, found by each warp for itself.
struct PrefixItem {
    int qt, kvh, c, g;
    int s0, s1, plen;        // sequences and length of the prefix
    int b0, h0, rows;        // row 0 of the tile is head h0 of the group of sequence b0; its rows in use
    int key_lo, key_hi;      // keys of the part
    int n_tiles;
};

// Up to 32 prefixes: lane g knows prefix g, and items are numbered over the query tiles and
// parts that exist, so that CTAs get equal counts of them.  More: over those of the largest
// group and longest prefix.
struct PrefixTable {
    int s0, s1, plen;
    int items;               // of prefixes 0 .. lane
    int all;
};

__device__ __forceinline__ PrefixTable prefix_table(const SharedParams &p, bool flag)
{
    PrefixTable t;
    t.s0 = t.s1 = t.plen = 0;
    t.items = 0;
    t.all = p.prefix_items;
    if (p.n_prefixes > 32) return t;
    const int lane = threadIdx.x % 32;
    if (lane < p.n_prefixes) {
        prefix_range(p, lane, t.s0, t.s1, t.plen, flag);
        t.items = prefix_tiles(p, t.s0, t.s1) * prefix_parts_of(p, t.plen) * p.n_kv_heads;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, t.items, o);
        if (lane >= o) t.items += y;
    }
    t.all = __shfl_sync(0xffffffffu, t.items, 31);
    return t;
}

// (sequence, query head) of row r < 128 of the tile; a division would take some 30 instructions,
// and a call this short fetches most of its instructions from memory.
__device__ __forceinline__ long long packed_row(const SharedParams &p, const PrefixItem &it, int r)
{
    const unsigned u = static_cast<unsigned>(it.h0 + r);
    const int q = static_cast<int>((static_cast<unsigned long long>(u) * p.group_inv) >> 31);
    return static_cast<long long>(it.b0 + q) * p.n_heads + it.kvh * p.group + (static_cast<int>(u) - q * p.group);
}

template <int BN>
__device__ __forceinline__ PrefixItem prefix_item(const SharedParams &p, const PrefixTable &t, int k, bool flag)
{
    PrefixItem it;
    int qtiles = p.prefix_qtiles, parts = p.prefix_slots;
    if (p.n_prefixes <= 32) {
        it.g = __popc(__ballot_sync(0xffffffffu, t.items <= k));
        const int before = __shfl_sync(0xffffffffu, t.items, it.g > 0 ? it.g - 1 : 0);
        if (it.g > 0) k -= before;
        it.s0 = __shfl_sync(0xffffffffu, t.s0, it.g);
        it.s1 = __shfl_sync(0xffffffffu, t.s1, it.g);
        it.plen = __shfl_sync(0xffffffffu, t.plen, it.g);
        qtiles = prefix_tiles(p, it.s0, it.s1);
        parts = prefix_parts_of(p, it.plen);
    }
    // query tiles fastest: those that share keys run at the same time
    it.qt = k % qtiles;
    k /= qtiles;
    it.c = k % parts;
    k /= parts;
    it.kvh = k % p.n_kv_heads;
    if (p.n_prefixes > 32) {
        it.g = k / p.n_kv_heads;
        prefix_range(p, it.g, it.s0, it.s1, it.plen, flag && it.qt == 0 && it.c == 0 && it.kvh == 0);
    }
    it.n_tiles = 0;
    it.key_lo = it.key_hi = 0;
    it.b0 = it.s0 + it.qt * kBM / p.group;
    it.h0 = it.qt * kBM - (it.b0 - it.s0) * p.group;
    it.rows = min(kBM, (it.s1 - it.s0) * p.group - it.qt * kBM);
    if (it.rows <= 0) return it;
    // parts count from the first key any row of the tile sees
    int lo = 0;
    if (p.window > 0) {
        const int b1 = it.b0 + (it.h0 + it.rows - 1) / p.group + 1;   // sequences of the tile: [b0, b1)
        lo = it.plen;
        for (int b = it.b0 + static_cast<int>(threadIdx.x % 32); b < b1; b += 32) {
            int ks, n;
            own_range(p, b, ks, n);
            lo = min(lo, max(0, it.plen + n - p.window));
        }
        lo = __reduce_min_sync(0xffffffffu, lo);
    }
    it.key_lo = lo + it.c * p.prefix_chunk;
    it.key_hi = min(it.plen, it.key_lo + p.prefix_chunk);
    if (it.key_hi > it.key_lo) it.n_tiles = (it.key_hi - it.key_lo + BN - 1) / BN;
    return it;
}

template <int HD, int QT>
__global__ void __launch_bounds__(PrefixShape<HD, QT>::kThreads, 1) prefix_kernel(const __grid_constant__ SharedParams p)
{
    using S = PrefixShape<HD, QT>;
    constexpr int BN = S::BN, ST = S::kStages, NG = S::kGroups;
    constexpr int kProducer = NG * 4, kIssuer = kProducer + 1;
    static_assert(sizeof(PrefixBars) <= 256, "barriers");
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    PrefixBars *bars = reinterpret_cast<PrefixBars *>(smem + S::kOffBar);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (threadIdx.x == 0) {
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
    // TMEM only after the wait: a CTA that held it while an earlier kernel's CTA on the same SM
    // still had to allocate would wait for that kernel for good.  The trigger comes after the
    // wait: the split kernel, which does not wait itself, starts only once every CTA here has
    // triggered, and so once every kernel before this one has completed.
    griddep_wait();
    griddep_trigger();
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

    const PrefixTable table = prefix_table(p, blockIdx.x == 0 && warp == 0);
    // Items with key tiles are numbered n_items = 0, 1, ... and their tiles g = 0, 1, ... over the
    // whole CTA; every barrier's phase follows from these numbers.
    if (warp == kProducer) {
        // ================= TMA producer (one lane issues; the geometry takes the warp) =================
        if (lane == 0) {
            tma_prefetch_desc(&p.tk);
            tma_prefetch_desc(&p.tv);
        }
        int nk = 0, nv = 0;   // K and V tiles issued
        int v_kvh = 0, v_row = 0;   // V tile nv, owed until K tile nv + 1 is issued
        bool ok = true;
        auto load = [&](bool is_v, int n, int kvh, int row) -> bool {
            const int st = n % ST;
            bool good = true;
            if (lane == 0) {
                const uint32_t full = smem_u32(is_v ? &bars->v_full[st] : &bars->k_full[st]);
                const uint32_t empty = smem_u32(is_v ? &bars->v_empty[st] : &bars->k_empty[st]);
                good = n < ST || mbar_wait(empty, (n / ST - 1) & 1, p.err, kErrWaitTmaEmpty);
                if (good) {
                    mbar_arrive_expect_tx(full, S::kKvBytes);
                    uint8_t *dst = (is_v ? sV : sK) + st * S::kKvBytes;
#pragma unroll
                    for (int sub = 0; sub < S::kSub; ++sub)
#pragma unroll
                        for (int r = 0; r < BN; r += S::kBoxRows)
                            tma_load_2d(smem_u32(dst + sub * S::kKvSubBytes + r * 128), is_v ? &p.tv : &p.tk, full,
                                        kvh * HD + sub * 64, row + r);
                }
            }
            return __shfl_sync(0xffffffffu, good, 0);
        };
        for (int k = blockIdx.x; k < table.all && ok; k += gridDim.x) {
            const PrefixItem it = prefix_item<BN>(p, table, k, lane == 0);
            if (it.n_tiles == 0) continue;
            const int row0 = static_cast<int>(p.prefix_row0[it.g] + it.key_lo);
            for (int j = 0; j < it.n_tiles && ok; ++j) {   // K runs one tile ahead of V
                if (!(ok = load(false, nk, it.kvh, row0 + j * BN))) break;
                ++nk;
                if (nv < nk - 1) {
                    if (!(ok = load(true, nv, v_kvh, v_row))) break;
                    ++nv;
                }
                v_kvh = it.kvh;
                v_row = row0 + j * BN;
            }
        }
        if (ok && nv < nk && load(true, nv, v_kvh, v_row)) ++nv;
        if (lane == 0) {
            for (int j = max(0, nk - ST); j < nk; ++j)
                if (!mbar_wait(smem_u32(&bars->k_full[j % ST]), (j / ST) & 1, p.err, kErrDrain)) break;
            for (int j = max(0, nv - ST); j < nv; ++j)
                if (!mbar_wait(smem_u32(&bars->v_full[j % ST]), (j / ST) & 1, p.err, kErrDrain)) break;
        }
        __syncwarp();
    } else if (warp == kIssuer) {
        // ================= tcgen05 issuer (converged warp, one elected lane issues) =================
        constexpr uint32_t idesc_s = umma_idesc_f16(kBM, BN, true, false);
        constexpr uint32_t idesc_pv = umma_idesc_f16(kBM, HD, false, true);
        const uint32_t q_addr = smem_u32(smem);
        int n_items = 0, g0 = 0;
        // P V of tile j of the item whose first tile has number g0
        auto issue_pv = [&](int j) -> bool {
            const int g = g0 + j, st = g % ST, sb = g & 1;
            if (!mbar_wait_warp(smem_u32(&bars->p_full[sb]), (g >> 1) & 1, p.err, kErrWaitSoftmax)) return false;
            if (!mbar_wait_warp(smem_u32(&bars->v_full[st]), (g / ST) & 1, p.err, kErrWaitTmaFull)) return false;
            tc_fence_after();
            const uint32_t v_addr = smem_u32(sV + st * S::kKvBytes);
#pragma unroll
            for (int t = 1; t >= 0; --t)   // the remainders first: the smaller sums
#pragma unroll
                for (int kk = 0; kk < BN / 16; ++kk) {
                    const uint64_t bd = umma_sdesc_sw128(v_addr + kk * 16 * 128, S::kKvSubBytes, 1024);
                    // columns of P: see the softmax (32-key groups: 16 of values, 16 of remainders)
                    umma_ts_elect(tmem + S::kTmO + (g % NG) * HD, tmem + sb * BN + (kk >> 1) * 32 + t * 16 + (kk & 1) * 8, bd,
                                  idesc_pv, (j >= NG || t < 1 || kk > 0) ? 1u : 0u);
                }
            umma_commit_elect(smem_u32(&bars->o_done[g % NG]));
            umma_commit_elect(smem_u32(&bars->v_empty[st]));
            return true;
        };
        bool ok = true;
        for (int k = blockIdx.x; k < table.all && ok; k += gridDim.x) {
            const PrefixItem it = prefix_item<BN>(p, table, k, false);
            if (it.n_tiles == 0) continue;
            // Q is written after the item before was read out, so its O may be overwritten too
            ok = mbar_wait_warp(smem_u32(&bars->q_full), n_items & 1, p.err, kErrWaitSoftmax);
            // Two warpgroups: P V of tile j - 2, whose P lies in the buffer of S(j), goes before
            // S(j).  One: S(j) goes first, so that it runs during the softmax of tile j - 1.  But
            // the softmax clears V rows of a last tile that the keys do not fill, and tells by the
            // parity of v_full that they have landed.  With one V slot that parity is the one of
            // tile j - 2, so tile j - 1 must have landed before S(j) can be seen: P V of tile
            // j - 1, issued after a wait for it, goes first there.
            const bool v_first = NG == 1 && ST == 1 && (it.key_hi - it.key_lo) % BN != 0;
            for (int j = 0; j < it.n_tiles && ok; ++j) {
                const int g = g0 + j, st = g % ST;
                const bool pv_first = NG == 2 ? j >= 2 : v_first && j >= 1 && j + 1 == it.n_tiles;
                if (pv_first && !(ok = issue_pv(j - NG))) break;
                if (!(ok = mbar_wait_warp(smem_u32(&bars->k_full[st]), (g / ST) & 1, p.err, kErrWaitTmaFull))) break;
                tc_fence_after();
                const uint32_t k_addr = smem_u32(sK + st * S::kKvBytes);
                const uint32_t s_col = tmem + (g & 1) * BN;
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
                umma_commit_elect(smem_u32(&bars->s_full[g & 1]));
                umma_commit_elect(smem_u32(&bars->k_empty[st]));
                if (NG == 1 && j >= 1 && !pv_first) ok = issue_pv(j - 1);
            }
            if (ok && NG == 2 && it.n_tiles >= 2) ok = issue_pv(it.n_tiles - 2);
            if (ok) ok = issue_pv(it.n_tiles - 1);
            if (ok) umma_commit_elect(smem_u32(&bars->o_final));
            g0 += it.n_tiles;
            ++n_items;
        }
        // every MMA must be complete before TMEM is released
        umma_commit_elect(smem_u32(&bars->mma_done));
        mbar_wait_warp(smem_u32(&bars->mma_done), 0, p.err, kErrDrain);
    } else {
        // ================= softmax =================
        const int wg = warp / 4, tid = threadIdx.x % kBM;
        const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp % 4) * 32) << 16);
        const float cap = p.softcap, inv_cap = cap > 0.f ? 1.f / cap : 0.f;
        const float mul = cap > 0.f ? 1.f : p.scale * kLog2e;
        int n_items = 0, g0 = 0;
        bool ok = true;   // false after a wait that ran out (the device error word is set)
        for (int k = blockIdx.x; k < table.all; k += gridDim.x) {
            const PrefixItem it = prefix_item<BN>(p, table, k, false);
            // this thread's packed row
            const bool row_valid = tid < it.rows;
            const long long row = packed_row(p, it, tid), slot = row * p.slots + it.c;
            if (it.n_tiles == 0) {
                if (row_valid && wg == 0) p.part_ml[slot] = make_float2(-INFINITY, 0.f);
                continue;
            }
            int lo = 0;   // the row's first visible prefix key
            if (row_valid && p.window > 0) {
                int ks, n;
                own_range(p, static_cast<int>(row / p.n_heads), ks, n);
                lo = max(0, it.plen + n - p.window);
            }
            // This warp's share of the query rows as QT bf16 terms in the 128B-swizzled K-major
            // layout, kLoad 8-element pieces in flight per lane (one at a time took 11 us of an
            // 18 us call at 512 prefix keys).  Rows past the last sequence stay as they are: a row
            // of Q only reaches its own row of S and O, and those are neither used nor stored.
            if (n_items > 0) named_bar_sync(1, S::kSoftmax);   // the last item's staging has been read
            constexpr int kVecs = HD / 8, kLoad = QT == 1 ? 8 : 4, kRows = 32 / NG;   // rows loaded by a warp
            const int lr = warp * kRows;
            if (lr < it.rows) {
#pragma unroll 1
                for (int i0 = lane; i0 < kRows * kVecs; i0 += 32 * kLoad) {
                    uint4 raw[kLoad][QT == 1 ? 1 : 2];
#pragma unroll
                    for (int n = 0; n < kLoad; ++n) {
                        const int i = i0 + 32 * n;
                        const int r = lr + i / kVecs;
                        if (i < kRows * kVecs && r < it.rows) {
                            const long long off = packed_row(p, it, r) * HD + (i % kVecs) * 8;
                            if constexpr (QT == 1) {
                                raw[n][0] =
                                    __ldg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p.q) + off));
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
                        if (i >= kRows * kVecs || r >= it.rows) continue;
                        uint8_t *at = smem + (e / 64) * S::kQSubBytes + sw128_offset(r, (e % 64) / 8);
                        if constexpr (QT == 1) {
                            *reinterpret_cast<uint4 *>(at) = raw[n][0];
                        } else {
                            const uint32_t u[8] = {raw[n][0].x, raw[n][0].y, raw[n][0].z, raw[n][0].w,
                                                   raw[n][1].x, raw[n][1].y, raw[n][1].z, raw[n][1].w};
                            uint32_t t[4][QT];
#pragma unroll
                            for (int i2 = 0; i2 < 4; ++i2)
                                split_bf16<QT>(__uint_as_float(u[2 * i2]), __uint_as_float(u[2 * i2 + 1]), t[i2]);
#pragma unroll
                            for (int q = 0; q < QT; ++q)
                                *reinterpret_cast<uint4 *>(at + q * S::kQTermBytes) =
                                    make_uint4(t[0][q], t[1][q], t[2][q], t[3][q]);
                        }
                    }
                }
            }
            fence_proxy_async_smem();
            tc_fence_before();
            mbar_arrive(smem_u32(&bars->q_full));
            const bool warp_live = (warp % 4) * 32 < it.rows;
            float m = -INFINITY, l = 0.f;
            // this warpgroup's tiles: numbers g with g % NG == wg; the first of the item is the
            // wg'th or, where the item starts on an odd number, the other
            for (int j = NG == 2 ? (g0 + wg) & 1 : 0; j < it.n_tiles; j += NG) {
                const int g = g0 + j, sb = g & 1;
                if (ok) ok = mbar_wait_warp(smem_u32(&bars->s_full[sb]), (g >> 1) & 1, p.err, kErrWaitMma);
                if (!ok) break;
                const int key0 = it.key_lo + j * BN;
                const int nv = it.key_hi - key0;   // valid keys of the tile (may be more)
                if (!warp_live && nv >= BN) {      // no row here, no V rows to clear
                    mbar_arrive(smem_u32(&bars->p_full[sb]));
                    continue;
                }
                tc_fence_after();
                const uint32_t s_col = lane_base + sb * BN, o_col = lane_base + S::kTmO + (g % NG) * HD;
                const bool whole = __all_sync(0xffffffffu, row_valid && key0 >= lo && nv >= BN);
                // The row's keys in groups of 32 columns, once for the maximum and once for the
                // exponentials: S is read twice, but the code stays small (fully unrolled over the
                // tile it was fetched from memory for every short call).
                auto hide = [&](int q, uint32_t (&rr)[32]) {
                    if (!whole) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const int key = key0 + q * 32 + i;
                            if (!row_valid || key < lo || key >= it.key_hi) rr[i] = 0xff800000u;   // -inf
                        }
                    }
                };
                float mx = -INFINITY;
#pragma unroll 1
                for (int q = 0; q < BN / 32; ++q) {
                    uint32_t rr[32];
                    tmem_ld32(s_col + q * 32, rr);
                    tmem_ld_wait();
                    hide(q, rr);
                    float pm[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        pm[i] = fmaxf(__uint_as_float(rr[2 * i]), __uint_as_float(rr[2 * i + 1]));
#pragma unroll
                    for (int i = 8; i < 32; i += 8)
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            pm[u] =
                                fmaxf(pm[u], fmaxf(__uint_as_float(rr[i + 2 * u]), __uint_as_float(rr[i + 2 * u + 1])));
                    mx = fmaxf(mx, fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3])));
                }
                if (cap > 0.f) {   // the cap is monotonic: the maximum's capped score is the capped maximum
                    if (mx != -INFINITY) mx = cap * tanhf(mx * p.scale * inv_cap) * kLog2e;
                } else {
                    mx *= mul;
                }
                // The reference m of a row comes from the first maximum it meets; it moves only when
                // a maximum passes that one by more than 2^8 (P stays below 2^15 in fp16), so O is
                // rescaled rarely.  NaN scores keep m and reach P.
                mx -= kHeadLog2;
                const bool fresh = m == -INFINITY;
                const bool move = mx > m + kMoveLog2 || (fresh && mx != -INFINITY);
                if (j >= NG && __any_sync(0xffffffffu, move && !fresh)) {
                    const float f = move && !fresh ? fast_exp2f(m - mx) : 1.f;
                    l *= f;
                    // O holds the earlier tiles' P V: scale it once they are complete
                    ok = mbar_wait_warp(smem_u32(&bars->o_done[wg]), (g / NG - 1) & 1, p.err, kErrWaitMma);
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
                // group's 32 keys, 32q+16 .. 32q+31 what their rounding left.
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
                    hide(q, rr);
                    uint32_t w[32];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float e0 = fast_exp2f(fmaf(__uint_as_float(rr[2 * i]), mul, negm));
                        const float e1 = fast_exp2f(fmaf(__uint_as_float(rr[2 * i + 1]), mul, negm));
                        acc[i & 3] += e0 + e1;
                        split_f16(e0, e1, w[i], w[16 + i]);
                    }
                    tmem_st32(s_col + q * 32, w);
                }
                l += (acc[0] + acc[1]) + (acc[2] + acc[3]);
                // Rows of the V tile past the part's last key may hold anything (another
                // sequence's rows, unwritten memory): 0 * NaN would reach O, so they are zeroed.
                // (P V of the tile before in this slot was issued before S(g), so its phase of
                // v_full is over and the parity names this tile's.)
                if (nv < BN) {
                    ok = mbar_wait_warp(smem_u32(&bars->v_full[g % ST]), (g / ST) & 1, p.err, kErrWaitTmaFull);
                    if (!ok) break;
                    uint8_t *vt = sV + (g % ST) * S::kKvBytes;
                    for (int i = tid; i < (BN - nv) * 8 * S::kSub; i += kBM) {
                        const int sub = i / ((BN - nv) * 8), u = i % ((BN - nv) * 8);
                        *reinterpret_cast<uint4 *>(vt + sub * S::kKvSubBytes + nv * 128 + u * 16) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async_smem();
                }
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(smem_u32(&bars->p_full[sb]));
            }
            // o_done may be two phases behind here (a parity wait could not tell), hence o_final
            if (ok) ok = mbar_wait_warp(smem_u32(&bars->o_final), n_items & 1, p.err, kErrWaitMma);
            if (!ok) m = -INFINITY, l = 0.f;   // the part counts as empty
            tc_fence_after();
            float M = m, f[2] = {1.f, 0.f};   // the row's reference, and each warpgroup's factor to it
            bool have[2] = {true, false};     // whether a warpgroup had tiles
            if (NG == 2) {
                float2 *ml = reinterpret_cast<float2 *>(smem);   // Q is no longer needed
                ml[wg * kBM + tid] = make_float2(m, l);
                named_bar_sync(1, S::kSoftmax);
                const float2 a = ml[tid], d = ml[kBM + tid];
                M = fmaxf(a.x, d.x);
                f[0] = a.x == -INFINITY ? 0.f : fast_exp2f(a.x - M);
                f[1] = d.x == -INFINITY ? 0.f : fast_exp2f(d.x - M);
                l = f[0] * a.y + f[1] * d.y;
                have[0] = it.n_tiles > 1 || (g0 & 1) == 0;
                have[1] = it.n_tiles > 1 || (g0 & 1) == 1;
                named_bar_sync(1, S::kSoftmax);   // read, before the staging below writes there
            }
            if (row_valid && wg == 0) p.part_ml[slot] = make_float2(M, l);
            if (ok && warp_live) {
                // O by blocks of 16 columns through shared memory, so that eight rows' 64 bytes go
                // out at a time (stores of 16 bytes from 32 rows each took 3 us of a part)
                uint8_t *stage = smem + warp * 2048;
                long long off[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {   // rows written by this lane: 8 i + lane / 4
                    const int r = (warp % 4) * 32 + 8 * i + lane / 4;
                    off[i] = r < it.rows ? (packed_row(p, it, r) * p.slots + it.c) * HD + lane % 4 * 4 : -1;
                }
#pragma unroll 1
                for (int c0 = wg * (HD / NG); c0 < (wg + 1) * (HD / NG); c0 += 16) {
                    uint32_t r0[16], r1[16];
                    tmem_ld16(lane_base + S::kTmO + c0, r0);
                    if (NG == 2) tmem_ld16(lane_base + S::kTmO + HD + c0, r1);
                    tmem_wait16(r0);
                    if (NG == 2) tmem_wait16(r1);
                    if (NG == 2) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            float x = have[0] && f[0] != 0.f ? f[0] * __uint_as_float(r0[i]) : 0.f;
                            if (have[1] && f[1] != 0.f) x += f[1] * __uint_as_float(r1[i]);
                            r0[i] = __float_as_uint(x);
                        }
                    }
                    __syncwarp();   // the block before has been read
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        *reinterpret_cast<uint4 *>(stage + lane * 64 + ((u ^ (lane >> 1)) & 3) * 16) =
                            make_uint4(r0[4 * u], r0[4 * u + 1], r0[4 * u + 2], r0[4 * u + 3]);
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int row = 8 * i + lane / 4;
                        const uint4 v = *reinterpret_cast<const uint4 *>(stage + row * 64 + (((lane % 4) ^ (row >> 1)) & 3) * 16);
                        if (off[i] >= 0) *reinterpret_cast<uint4 *>(p.part_o + off[i] + c0) = v;
                    }
                }
            }
            tc_fence_before();
            g0 += it.n_tiles;
            ++n_items;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kIssuer) {
        tc_fence_after();
        tmem_dealloc(tmem, S::kTmCols);
    }
}

// ===========================================================================
// split: a sequence's own rows, and prefixes of few packed rows
// ===========================================================================
// CTA = (chunk of keys, KV head and up to 8 of its query heads, sequence), or the same of a
// prefix, where the 8 columns run over its sequences' heads.  Warp 4 streams
// 64-key tiles of K and V through a TMA ring; warps 0-3 take 16 keys of each tile:
//   S^T(16 keys x 8 heads) = K . Q^T,  O^T(hd x 8 heads) += V^T . P^T   (mma.sync)
// so one tile in shared memory serves every query head of the KV head.
constexpr int kKeysPerTile = 64;
constexpr int kConsumerWarps = 4;
constexpr int kSplitThreads = (kConsumerWarps + 1) * 32;
constexpr int kSubtileBytes = kKeysPerTile * 128;
constexpr float kTopLog2 = 15.0f;   // the largest probability so far is 2^15 (fp16 holds 65504): see kHeadLog2

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

template <int HD, int QT>
__global__ void __launch_bounds__(kSplitThreads, 2) split_kernel(const __grid_constant__ SharedParams p)
{
    using S = SplitShape<HD>;
    constexpr int KSTEPS = HD / 16;
    // After a prefix kernel, whose CTAs have all passed their own wait and then triggered when
    // this grid starts, every earlier kernel has completed and nothing here depends on the prefix
    // kernel: the two run side by side.  Its inputs then come from L2 (input(), TMA), where completed
    // kernels have left them, past L1 lines that may be older; its outputs are slots that the prefix
    // kernel does not touch.  This grid may not end before it, as the merge waits for this grid alone: the last CTA waits
    // (if every CTA did, finished ones would hold their SMs until the prefix kernel's end).
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
    if (p.prefix_items == 0) griddep_wait();
    griddep_trigger();
    const bool last_cta =
        p.prefix_items > 0 && blockIdx.x + 1 == gridDim.x && blockIdx.y + 1 == gridDim.y && blockIdx.z + 1 == gridDim.z;
    auto input = [&](auto *at) {   // always past L1: 9 sequences to 2500, 12 heads of 64, 17.5 us against 16.4
        return p.prefix_items > 0 ? __ldcg(at) : *at;
    };
    const int c = blockIdx.x;
    const bool of_prefix = static_cast<int>(blockIdx.z) < p.prefix_units;
    int b, kvh, h_first, nh, key0, n, plen = 0;   // nh head columns; row_of() says whose
    long long seq_row0;
    if (of_prefix) {
        const int u = blockIdx.z / p.prefix_qtiles, t = blockIdx.z % p.prefix_qtiles;
        int s1;
        prefix_range(p, u, b, s1, plen, blockIdx.x + blockIdx.y + t + threadIdx.x == 0);
        kvh = blockIdx.y;
        h_first = t * 8;
        nh = kvh < p.n_kv_heads && c * p.prefix_chunk < plen ? min(8, (s1 - b) * p.group - h_first) : 0;
        seq_row0 = p.prefix_row0[u];
    } else {
        b = blockIdx.z - p.prefix_units;
        kvh = blockIdx.y / p.n_qgroups;
        const int qg = blockIdx.y % p.n_qgroups;
        h_first = kvh * p.group + qg * 8;
        nh = min(8, p.group - qg * 8);
        seq_row0 = input(p.seq_row0 + b);
    }
    // (sequence, query head) of column i; the columns of a prefix run over its sequences' heads
    auto row_of = [&](int i) -> long long {
        const int r = h_first + i;
        return of_prefix ? static_cast<long long>(b + r / p.group) * p.n_heads + kvh * p.group + r % p.group
                         : static_cast<long long>(b) * p.n_heads + r;
    };
    auto first_key = [&](int i) -> int {   // of the prefix that the sequence of column i sees
        int ks, own;
        own_range(p, b + (h_first + i) / p.group, ks, own);
        return max(0, plen + own - p.window);
    };
    if (of_prefix) {   // parts count from the first key any column sees
        int lo = 0;
        if (p.window > 0) {
            lo = plen;
            for (int i = 0; i < nh; ++i) lo = min(lo, first_key(i));
        }
        key0 = lo + c * p.prefix_chunk;
        n = min(plen, key0 + p.prefix_chunk);
        if (key0 >= n && static_cast<int>(threadIdx.x) < nh)
            p.part_ml[row_of(threadIdx.x) * p.slots + c] = make_float2(-INFINITY, 0.f);
    } else {
        int ks;
        own_keys(p, input(p.kv_len + b), ks, n);
        key0 = ks + c * p.chunk;
        n = min(n, key0 + p.chunk);
    }
    if (key0 >= n || nh <= 0) {
        if (last_cta) griddep_wait();
        return;
    }
    const int nkeys = n - key0;
    const int ntiles = (nkeys + kKeysPerTile - 1) / kKeysPerTile;
    const long long row_base = seq_row0 + key0;

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
        for (int v = threadIdx.x; v < nh * HD / 8; v += kConsumerWarps * 32) {
            const int e = v * 8;
            float *dst = qs + (e / HD) * S::kQRowFloats + e % HD;
            const long long off = row_of(e / HD) * HD + e % HD;
            if (p.q_is_bf16) {
                const uint4 w = input(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p.q) + off));
                const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    dst[2 * k] = bf16lo_f32(u[k]);
                    dst[2 * k + 1] = bf16hi_f32(u[k]);
                }
            } else {
                const float4 *src = reinterpret_cast<const float4 *>(static_cast<const float *>(p.q) + off);
                reinterpret_cast<float4 *>(dst)[0] = input(src);
                reinterpret_cast<float4 *>(dst)[1] = input(src + 1);
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
    if (p.scores && !of_prefix && 2 * tq < nh)
        sc_out = p.scores + ((static_cast<long long>(b) * p.n_kv_heads + kvh) * p.score_rows + key0) * p.score_cols +
                 h_first - kvh * p.group + 2 * tq;
    int hidden[2] = {0, 0};   // keys of the chunk before the first that the window shows these heads
    if (of_prefix && p.window > 0)
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (2 * tq + i < nh) hidden[i] = first_key(2 * tq + i) - key0;
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
                const int at = g + (i >> 1) * 8;   // key of the block
                if (at >= nv || kb + at < hidden[i & 1]) x[i] = -INFINITY;
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
            // reference points: the maximum less kTopLog2
            const float mn0 = fmaxf(m_run[0], mb0 - kTopLog2), mn1 = fmaxf(m_run[1], mb1 - kTopLog2);
            // a row whose scores are all -inf so far keeps exponentials of exactly 0
            const float n0 = mn0 == -INFINITY ? 0.f : -mn0, n1 = mn1 == -INFINITY ? 0.f : -mn1;
            const float corr0 = fast_exp2f(m_run[0] + n0), corr1 = fast_exp2f(m_run[1] + n1);
            m_run[0] = mn0;
            m_run[1] = mn1;
            const float p0 = fast_exp2f(x[0] + n0), p1 = fast_exp2f(x[1] + n1);
            const float p2 = fast_exp2f(x[2] + n0), p3 = fast_exp2f(x[3] + n1);
            l_run[0] = l_run[0] * corr0 + (p0 + p2);
            l_run[1] = l_run[1] * corr1 + (p1 + p3);
#pragma unroll
            for (int i = 0; i < KSTEPS; ++i) {
                o[i][0] *= corr0;
                o[i][1] *= corr1;
                o[i][2] *= corr0;
                o[i][3] *= corr1;
            }
            uint32_t pb[2][2];   // P^T as B fragments, keys 0-7 and 8-15: values, remainders
            {
                uint32_t h0, h1, r0, r1;
                split_f16(p0, p1, h0, r0);
                split_f16(p2, p3, h1, r1);
                pb[1][0] = movmatrix_t(r0);
                pb[1][1] = movmatrix_t(r1);
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
                for (int q = 1; q >= 0; --q) mma_f16_16816(o[db], a0, a1, a2, a3, pb[q][0], pb[q][1]);
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
            const float f = mw == -INFINITY ? 0.f : fast_exp2f(mw - M);
            if (f != 0.f) acc += f * red[(w * 8 + h) * kRowF + 2 + d];
            sum += f * red[(w * 8 + h) * kRowF + 1];
        }
        const long long slot = row_of(h) * p.slots + (of_prefix ? 0 : p.prefix_slots) + c;
        p.part_o[slot * HD + d] = acc;
        if (d == 0) p.part_ml[slot] = make_float2(M, sum);
    }
    if (last_cta) griddep_wait();
}

// ===========================================================================
// merge
// ===========================================================================
// Blocks below out_blocks join outputs: kMergeOuts of a query head by `ways` warps that take
// the parts in turn (512 contiguous bytes each) and meet in shared memory.  The others, with
// weights, add the probabilities of kMergeKeys own keys of a KV head each.  A warp finds the
// M and L it needs itself from the (m, l) of the head's parts.
constexpr int kMergeThreads = 256;
constexpr int kMergeWarps = kMergeThreads / 32;
constexpr int kMergeKeys = 1024;
constexpr int kMergeOuts = 128;

// The slots of a sequence that hold parts: [0, np) of its prefix and [own0, own1) of its own rows.
struct Parts {
    int np, own0, own1;
    __device__ __forceinline__ bool has(int slot) const { return slot < np || (slot >= own0 && slot < own1); }
};
// Of sequence b, whose length the caller has loaded; also its visible own keys [ks, n) (the
// whole warp).
__device__ __forceinline__ Parts parts_of(const SharedParams &p, int b, int kv_len, int &ks, int &n)
{
    Parts t;
    t.np = 0;
    for (int g0 = 0; g0 < p.n_prefixes; g0 += 32) {
        const int g = g0 + static_cast<int>(threadIdx.x % 32);
        int mine = 0;
        if (g < p.n_prefixes) {
            int s0, s1, len;
            prefix_range(p, g, s0, s1, len, false);
            if (b >= s0 && b < s1) mine = prefix_parts_of(p, len);
        }
        t.np = max(t.np, __reduce_max_sync(0xffffffffu, mine));
        if (t.np > 0) break;
    }
    own_keys(p, kv_len, ks, n);
    t.own0 = p.prefix_slots;
    t.own1 = p.prefix_slots + (n > ks ? (n - ks + p.chunk - 1) / p.chunk : 0);
    return t;
}

// M and 1/L of a head whose pairs are ml (the whole warp); v: pair `lane`, loaded ahead.
__device__ __forceinline__ void head_sum(const SharedParams &p, const float2 *ml, float2 v, const Parts &t, float &M,
                                         float &inv)
{
    const int lane = threadIdx.x % 32;
    M = -INFINITY;
    float L = 0.f;
    for (int s0 = 0; s0 < t.own1 || s0 < t.np; s0 += 32) {   // one pass: the sum moves with the maximum
        if (s0 > 0) v = t.has(s0 + lane) ? ml[s0 + lane] : make_float2(-INFINITY, 0.f);
        if (!t.has(s0 + lane)) v = make_float2(-INFINITY, 0.f);
        float mx = v.x;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float top = fmaxf(M, mx);
        // without a reference: an empty part (sum 0), or one whose scores are all NaN (sum NaN)
        float s = v.x == -INFINITY ? v.y : fast_exp2f(v.x - top) * v.y;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        L = (M == -INFINITY ? L : L * fast_exp2f(M - top)) + s;
        M = top;
    }
    inv = L != 0.f ? 1.f / L : 0.f;   // NaN stays NaN
}

template <int HD>
__global__ void __launch_bounds__(kMergeThreads, 4) merge_kernel(const __grid_constant__ SharedParams p, int ways, int out_blocks)
{
    griddep_wait();
    griddep_trigger();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (blockIdx.x == 0) {
        for (int g = threadIdx.x; g < p.idle_prefixes; g += kMergeThreads) {
            int s0, s1, len;
            prefix_range(p, g, s0, s1, len, true);
        }
    }
    if (static_cast<int>(blockIdx.x) < out_blocks) {
        // unit u: 128 outputs from element 128 u of the output on (head dim 64: of two heads)
        __shared__ float4 red[kMergeThreads];
        const long long u = static_cast<long long>(blockIdx.x) * (kMergeWarps / ways) + warp / ways;
        const long long row_elems = static_cast<long long>(p.n_heads) * HD;
        const long long e = u * kMergeOuts + lane * 4;      // this lane's first output
        const bool live = e < row_elems * p.n_seqs;
        const int way = warp % ways;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        float inv = 0.f;
        constexpr int kHeads = HD < kMergeOuts ? kMergeOuts / HD : 1;   // heads of a unit
        const long long head0 = u * kMergeOuts / HD;                   // its first (sequence, head)
        constexpr int kLoad = 4;                                       // parts in flight
        // Everything the first parts need is loaded at once: what a slot without a part holds is
        // not used.
        const long long mine = live ? e / HD : 0;   // this lane's (sequence, head)
        const float2 *my_ml = p.part_ml + mine * p.slots;
        const float *src = p.part_o + mine * p.slots * HD + e % HD;
        float r[kLoad];
        float4 v[kLoad];
        auto load_parts = [&](int c0, auto &&wanted) {
#pragma unroll
            for (int k = 0; k < kLoad; ++k) {
                const int c = c0 + k * ways;
                r[k] = -INFINITY;
                v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (live && wanted(c)) {
                    r[k] = my_ml[c].x;
                    v[k] = *reinterpret_cast<const float4 *>(src + static_cast<long long>(c) * HD);
                }
            }
        };
        load_parts(way, [&](int c) { return c < p.slots; });
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            const long long hs = head0 + i;
            if (hs >= static_cast<long long>(p.n_seqs) * p.n_heads) break;
            const int b = static_cast<int>(hs / p.n_heads);
            const float2 *ml = p.part_ml + hs * p.slots;
            const float2 ahead = lane < p.slots ? ml[lane] : make_float2(-INFINITY, 0.f);
            const int kv_len = p.kv_len[b];
            int ks, n;
            const Parts t = parts_of(p, b, kv_len, ks, n);
            if (lane == 0 && way == 0 && hs % p.n_heads == 0 && kv_len != n) atomicOr(p.err, kErrBadArgs);
            float M, my_inv;
            head_sum(p, ml, ahead, t, M, my_inv);
            if (e / HD != hs) continue;   // (a half-warp at head dim 64)
            inv = my_inv;
            for (int c0 = way; c0 < t.own1 || c0 < t.np; c0 += kLoad * ways) {
                if (c0 != way) load_parts(c0, [&](int c) { return t.has(c); });
#pragma unroll
                for (int k = 0; k < kLoad; ++k)
                    if (t.has(c0 + k * ways) && r[k] != -INFINITY) {   // an empty part has no output written
                        const float f = fast_exp2f(r[k] - M);
                        a.x += f * v[k].x, a.y += f * v[k].y, a.z += f * v[k].z, a.w += f * v[k].w;
                    }
            }
        }
        if (ways > 1) {
            red[threadIdx.x] = a;
            __syncthreads();
            if (way != 0) return;
            for (int w = 1; w < ways; ++w) {
                const float4 v = red[threadIdx.x + 32 * w];
                a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
            }
        }
        if (!live) return;
        a.x *= inv, a.y *= inv, a.z *= inv, a.w *= inv;
        if (p.out_is_bf16)
            *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.out) + e) =
                make_uint2(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w));
        else
            *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + e) = a;
        return;
    }
    const int key_blocks = (p.max_kv_len + kMergeKeys - 1) / kMergeKeys;
    const long long wb = blockIdx.x - out_blocks;
    const int j0 = static_cast<int>(wb % key_blocks) * kMergeKeys;
    const long long own = wb / key_blocks;   // (sequence, KV head)
    const int b = static_cast<int>(own / p.n_kv_heads), kvh = static_cast<int>(own % p.n_kv_heads);
    const long long row0 = static_cast<long long>(b) * p.n_heads + kvh * p.group;
    const float2 *ml = p.part_ml + (row0 + warp) * p.slots;   // of the first eight heads
    const float2 ahead = warp < p.group && lane < p.slots ? ml[lane] : make_float2(-INFINITY, 0.f);
    const int kv_len = p.kv_len[b];
    int ks, n;
    const Parts t = parts_of(p, b, kv_len, ks, n);
    if (j0 >= n) return;
    __shared__ float s_M[8], s_inv[8];
    constexpr int kPer = kMergeKeys / kMergeThreads;
    float w[kPer], w_in[kPer];
    auto load_pair = [&](const float *sc, int h, float2 (&x)[kPer]) {   // score_cols is even: 8-byte loads
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int j = j0 + i * kMergeThreads + static_cast<int>(threadIdx.x);
            x[i] = j >= ks && j < n ? *reinterpret_cast<const float2 *>(sc + static_cast<long long>(j) * p.score_cols + h)
                                    : make_float2(-INFINITY, -INFINITY);
        }
    };
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int j = j0 + i * kMergeThreads + static_cast<int>(threadIdx.x);
        w[i] = 0.f;
        w_in[i] = p.weights_in && j < n ? p.weights_in[own * p.weights_stride + j] : 0.f;
    }
    for (int h0 = 0; h0 < p.group; h0 += 8) {
        const int nh = min(8, p.group - h0);
        const float *sc = p.scores + own * p.score_rows * p.score_cols + h0;
        float2 x[kPer];
        load_pair(sc, 0, x);   // in flight while the sums are found
        if (warp < nh) {
            const float2 *mine = ml + static_cast<long long>(h0) * p.slots;
            float M, inv;
            head_sum(p, mine, h0 == 0 ? ahead : lane < p.slots ? mine[lane] : make_float2(-INFINITY, 0.f), t, M, inv);
            if (lane == 0) s_M[warp] = M, s_inv[warp] = inv;
        }
        __syncthreads();
        for (int h = 0; h < nh; h += 2) {
            if (h > 0) load_pair(sc, h, x);
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                if (x[i].x != -INFINITY) w[i] += fast_exp2f(x[i].x - s_M[h]) * s_inv[h];
                if (h + 1 < nh && x[i].y != -INFINITY) w[i] += fast_exp2f(x[i].y - s_M[h + 1]) * s_inv[h + 1];
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
constexpr int kMostLen = 1 << 29;   // of max_kv_len and max_prefix_len: sums of lengths and parts stay within an int
int div_up(long long a, long long b) { return static_cast<int>((a + b - 1) / b); }

// Keys per part for about `per_sm` CTAs per SM, multiples of 64 keys, at most kMostKeys: more
// parts cost their joining, longer ones leave SMs without work where lengths differ (16 sequences
// of 2000 to 8192 keys, 8 KV heads of 128: 65.2 us with 1024, 69.7 with 2048).
constexpr int kMostKeys = 1024;
int part_keys(long long units, int max_len, int per_sm)
{
    long long c = (units * (max_len > 0 ? max_len : 1) + kSms * per_sm - 1) / (kSms * per_sm);
    c = (c + kKeysPerTile - 1) / kKeysPerTile * kKeysPerTile;
    return static_cast<int>(c < kKeysPerTile ? kKeysPerTile : c > kMostKeys ? kMostKeys : c);
}

// Most parts part_keys() makes for any length up to max_len: ceil(L/64) while a part is 64 keys,
// at most ceil(148 per_sm / units) while it grows with the length, ceil(L / kMostKeys) after.
int most_parts(long long units, int max_len, int per_sm)
{
    const int len = max_len > 0 ? max_len : 1;
    int small = div_up(len, kKeysPerTile);
    const int by_work = div_up(kSms * per_sm, units);
    if (small > by_work) small = by_work;
    const int big = div_up(len, kMostKeys);
    return small > big ? small : big;
}
// Own rows, whose lengths differ (us with 8 / 3 / 2: 4 sequences of 2000 to 8192 keys, 8 KV heads
// of 128 19.4 / 14.6 / 15.9; 64 of 300 to 1000, one KV head of 256 31.7 / 18.4 / 20.1; 16 of 300 to
// 1000, 12 KV heads of 64 13.3 / 12.2 / 12.9).
constexpr int kOwnPerSm = 3;
constexpr int kFewPerSm = 2;   // a prefix in the split kernel: one wave (4096 keys, 8 rows: 15.7 us; with 4: 23.6)

// Parts of a prefix: one CTA on each of `sms` SMs over the query tiles and KV heads of all prefixes, no
// part under 128 keys, and none over kMaxPart: the tensor core truncates when it adds to an
// accumulator, which left a part of 6208 keys 1.3e-5 off (1024: 2e-6).
constexpr int kMaxPart = 1024;
int prefix_parts(int n_prefixes, int max_prefix_len, int max_prefix_seqs, int n_heads, int n_kv_heads, int sms)
{
    if (n_prefixes <= 0 || max_prefix_len <= 0 || max_prefix_seqs <= 0) return 0;
    const long long units = static_cast<long long>(n_prefixes) * n_kv_heads *
                            div_up(static_cast<long long>(max_prefix_seqs) * (n_heads / n_kv_heads), kBM);
    int parts = static_cast<int>(sms / units);
    if (parts < 1) parts = 1;
    const int most = div_up(max_prefix_len, 128), least = div_up(max_prefix_len, kMaxPart);
    return parts < least ? least : parts < most ? parts : most;
}

// Packed rows (sequences x group) of a prefix up to which the split kernel takes it too, 8 rows
// at a time: a CTA of the prefix kernel takes as long for one row of its 128-row tile as for all.
// us with the prefix kernel / with the split kernel, 8 KV heads of 128, fp32:
//   rows                  4            8           16           32
//   512 shared keys   15.3 /  8.1  15.8 /  9.8  16.2 / 11.1  15.1 / 16.6
//   4096              18.1 / 12.8  18.6 / 15.7  20.8 / 16.6  21.2 / 22.7
//   32768             63.1 / 31.4  63.6 / 34.5  66.5 / 41.9  54.7 / 67.4
//   8 times 4096      62.3 / 27.2  64.2 / 32.5  66.8 / 44.3  72.7 / 74.2
constexpr int kFewRows = 16;
bool few_rows(int n_seqs, int n_prefixes, int max_prefix_len, int max_prefix_seqs, int n_heads, int n_kv_heads)
{
    const long long rows = static_cast<long long>(max_prefix_seqs) * (n_heads / n_kv_heads);
    return n_prefixes > 0 && max_prefix_len > 0 && rows > 0 && rows <= kFewRows && n_seqs + n_prefixes * ((rows + 7) / 8) <= 65535;
}
long long few_units(int n_prefixes, int max_prefix_seqs, int n_heads, int n_kv_heads)
{
    return static_cast<long long>(n_prefixes) * n_kv_heads * ((max_prefix_seqs * (n_heads / n_kv_heads) + 7) / 8);
}

// CTAs of the prefix kernel, and the SMs its parts are made for.  The CTAs are one per SM, or as
// many as the own rows leave SMs, but no fewer than half: the split kernel keeps HBM busy from
// the others while the prefix kernel, bound by its products and exponentials, works; with all SMs
// the own rows come after it.  Parts are made for the CTAs, except where the own rows take
// longer anyway: then shorter ones.  Estimates in us: own rows at HBM's rate, half of the bound in
// use; an item 5 and 15 for every 1024 keys of 128.  16/8 heads of 128, bf16, us with all SMs /
// with half / so:  64 sequences, 8192 shared and 100 to 1024 own keys 52.9 / 46.5 / 45.3;  20
// sequences, 20000 and 500 to 2000 78.9 / - / 55.8.
struct PrefixGrid {
    int ctas, sms;
};
PrefixGrid prefix_grid(const SharedParams &p, int n_prefixes, int max_prefix_len, int max_prefix_seqs, int hd)
{
    const long long own_ctas = static_cast<long long>(p.n_seqs) * p.n_kv_heads * p.n_qgroups * p.max_chunks;
    const int left = own_ctas < kSms ? kSms - static_cast<int>(own_ctas + 1) / 2 : kSms / 2;   // two of them share an SM
    const double own_us = 0.5 * p.n_seqs * p.max_kv_len * 4.0 * p.n_kv_heads * hd / 6.3e6;
    double prefix_us[2], us[2];
    for (int i = 0; i < 2; ++i) {
        const int sms = i == 0 ? kSms : left;
        const int parts = prefix_parts(n_prefixes, max_prefix_len, max_prefix_seqs, p.n_heads, p.n_kv_heads, sms);
        const long long items = static_cast<long long>(p.prefix_qtiles) * parts * p.n_kv_heads * n_prefixes;
        const double item_us = 5.0 + div_up(max_prefix_len, parts) * (hd < 128 ? 128 : hd) / 131072.0 * 15.0;
        us[i] = prefix_us[i] = static_cast<double>((items + sms - 1) / sms) * item_us;
        if (i == 1) us[i] = us[i] > 1.05 * own_us ? us[i] : 1.05 * own_us;
        else if (items > left) us[i] += own_us > 5.0 ? own_us : 5.0;
    }
    if (us[0] <= us[1]) return {kSms, kSms};
    return {left, own_us > 2.0 * prefix_us[1] ? kSms : left};
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

template <int HD, int QT>
int launch_shared(cudaStream_t st, SharedParams &p, const uint16_t *k_pool, const uint16_t *v_pool, int64_t pool_rows)
{
    const int kv_dim = p.n_kv_heads * HD;
    auto maps = [&](int rows) {
        return make_tmap_2d(&p.tk, k_pool, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, kv_dim, pool_rows, 64, rows) &&
               make_tmap_2d(&p.tv, v_pool, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, kv_dim, pool_rows, 64, rows);
    };
    // Warps per 128 outputs: one where that fills the GPU with warps, up to eight (and a part
    // each) where a row's parts would otherwise be read one after another.
    const long long units = (static_cast<long long>(p.n_seqs) * p.n_heads * HD + kMergeOuts - 1) / kMergeOuts;
    int ways = 1;
    while (ways < kMergeWarps && units * ways < kSms * kMergeWarps && 2 * ways < p.slots) ways *= 2;
    const long long out_blocks = (units * ways + kMergeWarps - 1) / kMergeWarps;
    const long long key_blocks =
        p.scores ? static_cast<long long>(div_up(p.max_kv_len, kMergeKeys)) * p.n_seqs * p.n_kv_heads : 0;
    if (out_blocks + key_blocks > 0x7fffffffLL) return SMOL_B200_ERR_ARGS;
    int box_rows = 0;   // of the maps in p
    if (p.prefix_items > 0) {
        using S = PrefixShape<HD, QT>;
        if (!maps(box_rows = S::kBoxRows) ||
            !allow_smem(reinterpret_cast<const void *>(prefix_kernel<HD, QT>), S::kSmemBytes))
            return SMOL_B200_ERR_CUDA;
        const dim3 grid(static_cast<unsigned>(p.prefix_items < p.prefix_ctas ? p.prefix_items : p.prefix_ctas));
        if (launch_kernel(prefix_kernel<HD, QT>, grid, dim3(S::kThreads), S::kSmemBytes, st, p) != cudaSuccess)
            return SMOL_B200_ERR_CUDA;
    }
    if (p.max_kv_len > 0 || p.prefix_units > 0) {
        using S = SplitShape<HD>;
        if ((box_rows != kKeysPerTile && !maps(kKeysPerTile)) ||
            !allow_smem(reinterpret_cast<const void *>(split_kernel<HD, QT>), S::kSmemBytes))
            return SMOL_B200_ERR_CUDA;
        const int parts = p.prefix_units > 0 && p.prefix_slots > p.max_chunks ? p.prefix_slots : p.max_chunks;
        const dim3 grid(parts, p.n_kv_heads * p.n_qgroups, p.prefix_units + p.n_seqs);
        if (launch_kernel(split_kernel<HD, QT>, grid, dim3(kSplitThreads), S::kSmemBytes, st, p) != cudaSuccess)
            return SMOL_B200_ERR_CUDA;
    }
    if (launch_kernel(merge_kernel<HD>, dim3(static_cast<unsigned>(out_blocks + key_blocks)), dim3(kMergeThreads), 0, st, p,
                      ways, static_cast<int>(out_blocks)) != cudaSuccess)
        return SMOL_B200_ERR_CUDA;
    return SMOL_B200_OK;
}

template <int HD>
int launch_shared_hd(cudaStream_t st, SharedParams &p, const uint16_t *k, const uint16_t *v, int64_t rows)
{
    return p.q_is_bf16 ? launch_shared<HD, 1>(st, p, k, v, rows) : launch_shared<HD, 3>(st, p, k, v, rows);
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
    const int slots =
        most_parts(own_units(n_seqs, n_heads, n_kv_heads), max_kv_len, kOwnPerSm) +
        (few_rows(n_seqs, n_prefixes, max_prefix_len, max_prefix_seqs, n_heads, n_kv_heads)
             ? most_parts(few_units(n_prefixes, max_prefix_seqs, n_heads, n_kv_heads), max_prefix_len, kFewPerSm)
             : prefix_parts(n_prefixes, max_prefix_len, max_prefix_seqs, n_heads, n_kv_heads, kSms));
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
        max_prefix_len < 0 || max_prefix_len > kMostLen || max_kv_len > kMostLen || max_prefix_seqs < 0 || max_prefix_seqs > n_seqs)
        return SMOL_B200_ERR_ARGS;
    if (n_prefixes > 0 && (!prefix_row0 || !prefix_len || !prefix_seq0)) return SMOL_B200_ERR_ARGS;
    if ((reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool) | reinterpret_cast<uintptr_t>(q) |
         reinterpret_cast<uintptr_t>(out)) & 15)
        return SMOL_B200_ERR_ARGS;
    if (!(scale > 0.f)) return SMOL_B200_ERR_ARGS;
    if (weights_in && !weights_out) return SMOL_B200_ERR_ARGS;
    if (weights_out && weights_stride < max_kv_len) return SMOL_B200_ERR_ARGS;
    const int announced = n_prefixes;
    if (max_prefix_len == 0 || max_prefix_seqs == 0) n_prefixes = 0;

    SharedParams p;
    memset(&p, 0, sizeof(p));
    p.n_seqs = n_seqs;
    p.n_heads = n_heads;
    p.n_kv_heads = n_kv_heads;
    p.max_kv_len = max_kv_len;
    const long long units = own_units(n_seqs, n_heads, n_kv_heads);
    // grids; row numbers, and those of a tile times the group, stay within an int
    if (n_kv_heads * ((n_heads / n_kv_heads + 7) / 8) > 65535 || static_cast<long long>(n_seqs) * n_heads > (1 << 30) ||
        n_heads / n_kv_heads > 32768)
        return SMOL_B200_ERR_ARGS;
    p.group = n_heads / n_kv_heads;
    p.n_qgroups = (p.group + 7) / 8;
    p.group_inv = static_cast<unsigned>(((1ll << 31) + p.group - 1) / p.group);
    p.chunk = part_keys(units, max_kv_len, kOwnPerSm);
    p.max_chunks = max_kv_len > 0 ? div_up(max_kv_len, p.chunk) : 0;
    if (few_rows(n_seqs, n_prefixes, max_prefix_len, max_prefix_seqs, n_heads, n_kv_heads)) {
        p.prefix_chunk = part_keys(few_units(n_prefixes, max_prefix_seqs, n_heads, n_kv_heads), max_prefix_len, kFewPerSm);
        p.prefix_slots = div_up(max_prefix_len, p.prefix_chunk);
        p.prefix_qtiles = (max_prefix_seqs * p.group + 7) / 8;
        p.prefix_units = n_prefixes * p.prefix_qtiles;
    } else {
        p.prefix_qtiles = div_up(static_cast<long long>(max_prefix_seqs) * p.group, kBM);
        PrefixGrid grid = {kSms, kSms};
        if (n_prefixes > 0) grid = prefix_grid(p, n_prefixes, max_prefix_len, max_prefix_seqs, head_dim);
        p.prefix_ctas = grid.ctas;
        p.prefix_slots = prefix_parts(n_prefixes, max_prefix_len, max_prefix_seqs, n_heads, n_kv_heads, grid.sms);
        if (p.prefix_slots > 0) p.prefix_chunk = (div_up(max_prefix_len, p.prefix_slots) + 63) / 64 * 64;
        const long long items = static_cast<long long>(p.prefix_qtiles) * p.prefix_slots * n_kv_heads * n_prefixes;
        if (items > 0x7fffff00LL) return SMOL_B200_ERR_ARGS;
        p.prefix_items = static_cast<int>(items);
    }
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
    p.n_prefixes = n_prefixes;
    p.idle_prefixes = announced - n_prefixes;
    p.max_prefix_len = max_prefix_len;
    p.max_prefix_seqs = max_prefix_seqs;
    p.window = window;
    p.scale = scale;
    p.softcap = softcap;
    // every kernel waits for its predecessor before reading anything, but the split kernel after a
    // prefix kernel, which has waited for both
    PdlScope pdl(g_api_pdl);
    switch (head_dim) {
    case 64: return launch_shared_hd<64>(st, p, k_pool, v_pool, pool_rows);
    case 128: return launch_shared_hd<128>(st, p, k_pool, v_pool, pool_rows);
    default: return launch_shared_hd<256>(st, p, k_pool, v_pool, pool_rows);
    }
}

}  // namespace smolb200
