// cache_evict.cu -- brings the caches of a batch to a budget of slots per KV head.
//
// Of the n slots of a (sequence, KV head) the B = min(n, budget) best stay, in the order:
// the first `sink` positions and the most recent `recent` ones, then the running weight,
// equal weights by the lower slot.  What stays ends in slots [0, B): kept slots below B do
// not move, and the i-th dropped slot below B (a hole) takes the row of the i-th kept slot
// from B on (a mover).  Sources lie at B and above, targets below it, so the moves are
// independent of one another and work in place, and no row is moved that need not be:
// attention does not depend on the order of a head's rows.
//
// Select.  The B-th largest of the n 32-bit sort keys is found by bracketing: keys stay in
// registers, a round counts those at or above six candidates -- five around the rank
// interpolated between the bracket's ends, one at its middle, so that it halves at worst.
// It ends when exactly B keys lie at or above a candidate, or when one key value is left,
// whose ties are taken in slot order.  One more ordered count gives holes and movers their
// numbers.  (Two bits a round from the top took 16 rounds of 0.6 us, 1.2 us in a cluster.)
// A (sequence, KV head) is one CTA or, for long caches, one cluster whose CTAs hold a
// segment of the slots each and exchange counts through shared memory.
//
// Bytes: 8 per slot to read (weight, position), as many to write where the outputs are
// other arrays, and K and V of the moved rows.  32 sequences of 1025 slots to 1024, 8 heads of
// 128: 7.6 us, latency (8.3 in place, with the launch that writes the lengths); 8 of 16384 to
// 2048: 52.5 us, 13 of them selection (134 MB: 20 us).
#include <string.h>

#include "b200_common.cuh"
#include "runtime.h"

namespace smolb200 {
namespace {

constexpr int kMaxThreads = 1024;
constexpr int kMaxItems = 32;
constexpr int kMaxCluster = 8;
// Moves whose slots are listed in shared memory; more go through the workspace.
constexpr int kSmemMoves = 2048;

struct EvictParams {
    uint16_t *k, *v;
    long long pool_rows;
    const int64_t *seq_row0;
    const float *weights_in;
    float *weights_out;
    const int *positions_in;
    int *positions_out;
    long long stride;
    const int *kv_len_in;
    int *kv_len_out;
    const int *seq_pos;
    int *lists;      // [n_seqs*n_kv_heads][2*cap]: holes, movers
    int *lengths;    // [n_seqs] new lengths
    unsigned *err;
    int n_kv_heads, hd, max_kv_len, budget, sink, recent, cap;
    int smem_lists, write_len;   // lists in shared memory; this kernel writes kv_len_out
};

// Weight as an unsigned key of the same order: NaN lowest, -0 equal to 0.
__device__ __forceinline__ uint32_t weight_key(float w)
{
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Position of slot j of n: what was recorded, else the slot was appended since the last
// eviction, in order, up to the newest token seen.
__device__ __forceinline__ int slot_position(int recorded, int j, int n, int seen)
{
    return recorded >= 0 ? recorded : seen - n + j;
}

// K and V of the moves of head h, 16 bytes a thread and four pieces in flight, by threads
// first, first + step, ... of `step` (dst_src(r) gives the slots of move r).
template <typename Slots>
__device__ __forceinline__ void move_rows(const EvictParams &p, long long row0, int h, int m, int first, int step,
                                          Slots &&dst_src)
{
    const int vecs = p.hd / 8;   // 16-byte pieces of one head's row
    const long long width = static_cast<long long>(p.n_kv_heads) * p.hd;
    const long long total = static_cast<long long>(m) * 2 * vecs;
    constexpr int kLoad = 4;
    for (long long i0 = first; i0 < total; i0 += static_cast<long long>(step) * kLoad) {
        uint4 v[kLoad];
        uint16_t *to[kLoad];
#pragma unroll
        for (int u = 0; u < kLoad; ++u) {
            const long long i = i0 + static_cast<long long>(u) * step;
            to[u] = nullptr;
            if (i < total) {
                const int r = static_cast<int>(i / (2 * vecs)), e = static_cast<int>(i - static_cast<long long>(r) * 2 * vecs);
                uint16_t *pool = e < vecs ? p.k : p.v;
                const long long col = static_cast<long long>(h) * p.hd + (e < vecs ? e : e - vecs) * 8;
                const int2 ds = dst_src(r);
                to[u] = pool + (row0 + ds.x) * width + col;
                v[u] = *reinterpret_cast<const uint4 *>(pool + (row0 + ds.y) * width + col);
            }
        }
#pragma unroll
        for (int u = 0; u < kLoad; ++u)
            if (to[u]) *reinterpret_cast<uint4 *>(to[u]) = v[u];
    }
}

template <int ITEMS>
__global__ void __launch_bounds__(kMaxThreads) evict_kernel(const __grid_constant__ EvictParams p)
{
    griddep_wait();
    griddep_trigger();
    __shared__ uint32_t s_cnt[8][kMaxThreads / 32];      // every warp's results of a round
    __shared__ uint32_t s_box[2][kMaxCluster][8];        // every CTA's, by round parity
    __shared__ int s_scan[ITEMS][kMaxThreads / 32];      // flags per (item, warp), then those before within the item
    __shared__ int s_item[ITEMS];                        // flags per item
    __shared__ int s_tot_box[2][kMaxCluster];
    __shared__ int s_holes[kSmemMoves], s_movers[kSmemMoves];
    const int C = static_cast<int>(gridDim.x), rank = blockIdx.x;
    const int h = blockIdx.y, b = blockIdx.z;
    const int T = blockDim.x, tid = threadIdx.x, warp = tid / 32, lane = tid % 32, W = T / 32;

    const int length = p.kv_len_in[b];
    const long long row0 = p.seq_row0[b];
    const int seen = p.seq_pos[b];
    const int n = min(max(length, 0), p.max_kv_len);
    // a length or rows that cannot be: the sequence is left as it is
    const bool bad = n != length || (n > p.budget && (row0 < 0 || row0 > p.pool_rows - n));
    const bool keep_all = bad || n <= p.budget;
    const int B = keep_all ? length : p.budget;
    const long long unit = static_cast<long long>(b) * p.n_kv_heads + h;
    if (rank == 0 && tid == 0) {
        if (h == 0) {
            if (bad) atomicOr(p.err, kErrBadArgs);
            p.lengths[b] = B;
            if (p.write_len) p.kv_len_out[b] = B;
        }
    }
    const float *w_in = p.weights_in + unit * p.stride;
    float *w_out = p.weights_out + unit * p.stride;
    const int *pos_in = p.positions_in + unit * p.stride;
    int *pos_out = p.positions_out + unit * p.stride;
    const int j_first = rank * ITEMS * T + tid;   // this thread's slots: j_first + i * T
    if (keep_all) {
#pragma unroll 4
        for (int i = 0; i < ITEMS; ++i) {
            const int j = j_first + i * T;
            if (j < n) {
                if (w_in != w_out) w_out[j] = w_in[j];
                if (pos_in != pos_out) pos_out[j] = pos_in[j];
            }
        }
        return;
    }

    // A CTA's shared memory may be written from another one only once it runs: the first join()
    // waits for every CTA of the cluster, whose arrivals pass while the slots are loaded.
    if (C > 1) cluster_arrive();
    uint32_t key[ITEMS];   // 0 past the last slot: below every candidate
    {
        float w[ITEMS];
        int q[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int j = j_first + i * T;
            w[i] = j < n ? w_in[j] : 0.f;
            q[i] = j < n ? pos_in[j] : 0;
        }
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int j = j_first + i * T;
            const int pos = slot_position(q[i], j, n, seen);
            key[i] = j >= n ? 0u : pos < p.sink || pos >= seen - p.recent ? 0xffffffffu : weight_key(w[i]);
        }
    }
    if (C > 1) cluster_wait();
    // Six sums (and, for `maxima`, two maxima) over all threads of the cluster.  A warp-wide
    // reduction takes a scheduler some 35 cycles, so a warp's six counts go in two of them and
    // one warp each adds up the warps' results.
    int round = 0;
    uint32_t res[8];
    auto join = [&](const uint32_t (&c)[6], bool maxima, uint32_t m0, uint32_t m1) {
        uint32_t sum[6];
        if (ITEMS <= 16) {   // a warp's counts fit 10 bits: three to a reduction
            const uint32_t a = __reduce_add_sync(0xffffffffu, c[0] | (c[1] << 10) | (c[2] << 20));
            const uint32_t b = __reduce_add_sync(0xffffffffu, c[3] | (c[4] << 10) | (c[5] << 20));
#pragma unroll
            for (int k = 0; k < 3; ++k) sum[k] = (a >> (10 * k)) & 1023u, sum[3 + k] = (b >> (10 * k)) & 1023u;
        } else {
#pragma unroll
            for (int k = 0; k < 6; ++k) sum[k] = __reduce_add_sync(0xffffffffu, c[k]);
        }
        if (maxima) {
            m0 = __reduce_max_sync(0xffffffffu, m0);
            m1 = __reduce_max_sync(0xffffffffu, m1);
        }
        if (lane < 8) {
            uint32_t mine = lane == 6 ? m0 : m1;
#pragma unroll
            for (int k = 0; k < 6; ++k)
                if (lane == k) mine = sum[k];
            s_cnt[lane][warp] = mine;
        }
        __syncthreads();
        uint32_t (*box)[8] = s_box[round & 1];
        for (int k = warp; k < (maxima ? 8 : 6); k += W) {
            const uint32_t v = lane < W ? s_cnt[k][lane] : 0;
            const uint32_t all = k < 6 ? __reduce_add_sync(0xffffffffu, v) : __reduce_max_sync(0xffffffffu, v);
            if (C == 1) {
                if (lane == 0) box[0][k] = all;
            } else if (lane < C) {   // to every CTA of the cluster
                const uint32_t dst = map_shared_rank(smem_u32(&box[rank][k]), lane);
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(dst), "r"(all) : "memory");
            }
        }
        if (C > 1) cluster_sync_all();
        else __syncthreads();
#pragma unroll
        for (int k = 0; k < 8; ++k) res[k] = box[0][k];
        for (int r = 1; r < C; ++r) {
#pragma unroll
            for (int k = 0; k < 6; ++k) res[k] += box[r][k];
            res[6] = max(res[6], box[r][6]);
            res[7] = max(res[7], box[r][7]);
        }
        ++round;
    };
    // The bracket [lo, hi) with count(>= lo) = at_lo >= B > at_hi = count(>= hi): at first the
    // smallest key and just above the largest unprotected one.
    uint32_t lo = 0xffffffffu, hi = 0xffffffffu;
    int at_lo = B, at_hi = 0;
    {
        uint32_t c[6] = {0, 0, 0, 0, 0, 0}, top = 0, bottom = 0;   // bottom: largest complement
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const bool in = j_first + i * T < n;
            c[0] += key[i] == 0xffffffffu;
            if (in && key[i] != 0xffffffffu) top = max(top, key[i]), bottom = max(bottom, ~key[i]);
        }
        join(c, true, top, bottom);
        const int safe = static_cast<int>(res[0]);
        if (safe < B) lo = ~res[7], hi = res[6] + 1, at_lo = n, at_hi = safe;
        // safe >= B: exactly the protected ones (at most `budget` of them)
        else at_lo = safe;
    }
    auto narrow = [&](uint32_t c, int k) {
        if (k >= B) {
            if (c > lo) lo = c, at_lo = k;
        } else if (c < hi) {
            hi = c, at_hi = k;
        }
    };
    while (at_lo != B && hi - lo > 1) {
        const uint32_t size = hi - lo;
        const float at = __fdividef(static_cast<float>(at_lo - B) + 0.5f, static_cast<float>(at_lo - at_hi));
        const uint32_t d = size / 8 + 1, e = size / 64 + 1;
        const uint32_t x = lo + min(static_cast<uint32_t>(at * static_cast<float>(size)), size - 1);
        uint32_t cand[6] = {x > lo + d ? x - d : lo + 1, x > lo + e ? x - e : lo + 1, x, hi - x > e ? x + e : hi - 1,
                            hi - x > d ? x + d : hi - 1, lo + size / 2};
        uint32_t c[6] = {0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < 6; ++k) cand[k] = max(cand[k], lo + 1);   // inside (lo, hi)
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int k = 0; k < 6; ++k) c[k] += key[i] >= cand[k];
        join(c, false, 0, 0);
#pragma unroll
        for (int k = 0; k < 6; ++k) narrow(cand[k], static_cast<int>(res[k]));
    }
    const uint32_t t = lo;
    const int at_t = at_lo, above = at_hi;   // keys >= t; keys above t where ties decide

    // Ordered counts: flags in (CTA, item, thread) order = slot order.  Afterwards before_me()
    // gives the flags in front of one of this thread's items; returns their total.
    int scans = 0;
    int item_first[ITEMS];   // flags before this CTA's item i
    auto ordered = [&](uint32_t flags) -> int {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const uint32_t bal = __ballot_sync(0xffffffffu, (flags >> i) & 1u);
            if (lane == 0) s_scan[i][warp] = __popc(bal);
        }
        __syncthreads();
        for (int i = warp; i < ITEMS; i += W) {   // one warp an item: prefix over its W warps
            const int v = lane < W ? s_scan[i][lane] : 0;
            int x = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            if (lane < W) s_scan[i][lane] = x - v;
            if (lane == 31) s_item[i] = x;
        }
        __syncthreads();
        int total = 0;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            item_first[i] = total;
            total += s_item[i];
        }
        if (C > 1) {
            const int box = scans++ & 1;   // at most two scans, a box each
            if (tid < C) {
                const uint32_t dst = map_shared_rank(smem_u32(&s_tot_box[box][rank]), tid);
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(dst), "r"(total) : "memory");
            }
            cluster_sync_all();
            int before = 0;
            total = 0;
            for (int r = 0; r < C; ++r) {
                if (r < rank) before += s_tot_box[box][r];
                total += s_tot_box[box][r];
            }
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) item_first[i] += before;
        }
        return total;
    };
    auto before_me = [&](uint32_t flags, int i) -> int {   // flags before this thread's item i
        const uint32_t bal = __ballot_sync(0xffffffffu, (flags >> i) & 1u);
        return item_first[i] + s_scan[i][warp] + __popc(bal & ((1u << lane) - 1u));
    };

    uint32_t kept = 0, ties = 0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int j = j_first + i * T;
        if (j < n) {
            if (key[i] > t || (at_t == B && key[i] == t)) kept |= 1u << i;
            else if (key[i] == t) ties |= 1u << i;
        }
    }
    if (at_t != B) {   // keys above t number `above`; the first B - above of those equal to t stay
        ordered(ties);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int k = before_me(ties, i);
            if (((ties >> i) & 1u) && k < B - above) kept |= 1u << i;
        }
        __syncthreads();
    }
    uint32_t moved = 0;   // holes below B, movers from B on
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int j = j_first + i * T;
        const bool k = (kept >> i) & 1u;
        if (j < n && (j < B ? !k : k)) moved |= 1u << i;
    }
    const int m = ordered(moved) / 2;   // as many movers as holes
    // The lists: short ones in every CTA's shared memory, long ones in the workspace.
    int *holes = p.smem_lists ? s_holes : p.lists + unit * 2 * p.cap;
    int *movers = p.smem_lists ? s_movers : holes + p.cap;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int j = j_first + i * T;
        const int k = before_me(moved, i);
        if ((moved >> i) & 1u) {
            int *at = j < B ? holes + k : movers + (k - m);
            if (!p.smem_lists || C == 1) *at = j;
            else
                for (int r = 0; r < C; ++r)
                    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(map_shared_rank(smem_u32(at), r)), "r"(j)
                                 : "memory");
        }
    }
    // slots that stay
#pragma unroll 4
    for (int i = 0; i < ITEMS; ++i) {
        const int j = j_first + i * T;
        if (j < B && ((kept >> i) & 1u)) {
            if (w_in != w_out) w_out[j] = w_in[j];
            const int q = pos_in[j];
            if (pos_in != pos_out || q < 0) pos_out[j] = slot_position(q, j, n, seen);
        }
    }
    if (!p.smem_lists) __threadfence();
    __syncthreads();
    if (C > 1) cluster_sync_all();   // the lists are complete
    for (int r = rank * T + tid; r < m; r += C * T) {
        const int dst = holes[r], src = movers[r];
        w_out[dst] = w_in[src];
        pos_out[dst] = slot_position(pos_in[src], src, n, seen);
    }
    __syncthreads();
    if (C > 1) cluster_sync_all();   // every mover's weight and position has been read
#pragma unroll 4
    for (int i = 0; i < ITEMS; ++i) {
        const int j = j_first + i * T;
        if (j >= B && j < n) {
            w_out[j] = 0.f;
            pos_out[j] = -1;
        }
    }
    move_rows(p, row0, h, m, rank * T + tid, C * T, [&](int r) { return make_int2(holes[r], movers[r]); });
}

// kv_len_out is kv_len_in: written once every CTA has read it
__global__ void evict_length_kernel(int *kv_len_out, const int *lengths, int n_seqs)
{
    griddep_wait();
    griddep_trigger();
    const int b = blockIdx.x * blockDim.x + threadIdx.x;
    if (b < n_seqs) kv_len_out[b] = lengths[b];
}

struct EvictLayout {
    size_t lengths, total;
    int cap;
};

EvictLayout evict_layout(int n_seqs, int max_kv_len, int n_kv_heads)
{
    auto al = [](size_t x) { return (x + 255) & ~size_t(255); };
    EvictLayout L;
    const size_t units = static_cast<size_t>(n_seqs) * n_kv_heads;
    L.cap = max_kv_len / 2 + 1;   // min(B, n - B) moves at most
    L.lengths = al(units * 2 * L.cap * 4);
    L.total = L.lengths + al(static_cast<size_t>(n_seqs) * 4);
    return L;
}

template <int ITEMS>
cudaError_t launch_evict(cudaStream_t st, const EvictParams &p, int C, int threads, int n_seqs)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(C, p.n_kv_heads, n_seqs);
    cfg.blockDim = dim3(threads);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = C;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    // the programmatic attribute first, so that either may be left out
    cfg.attrs = g_pdl_scope ? attr : attr + 1;
    cfg.numAttrs = (g_pdl_scope ? 1 : 0) + (C > 1 ? 1 : 0);
    return cudaLaunchKernelEx(&cfg, evict_kernel<ITEMS>, p);
}

}  // namespace

size_t cache_evict_workspace_bytes(int n_seqs, int max_kv_len, int n_kv_heads)
{
    if (n_seqs <= 0 || max_kv_len < 0 || n_kv_heads <= 0) return 0;
    return evict_layout(n_seqs, max_kv_len, n_kv_heads).total;
}

int cache_evict(cudaStream_t st, uint16_t *k_pool, uint16_t *v_pool, int64_t pool_rows, const int64_t *seq_row0,
                const float *weights_in, float *weights_out, const int *positions_in, int *positions_out,
                int64_t stride, const int *kv_len_in, int *kv_len_out, const int *seq_pos, int n_seqs, int max_kv_len,
                int n_kv_heads, int head_dim, int budget, int sink, int recent, void *workspace,
                size_t workspace_bytes)
{
    if (n_seqs <= 0) return SMOL_B200_OK;
    if (!k_pool || !v_pool || !seq_row0 || !weights_in || !weights_out || !positions_in || !positions_out ||
        !kv_len_in || !kv_len_out || !seq_pos || n_seqs > 65535 || n_kv_heads <= 0 || n_kv_heads > 65535 ||
        head_dim <= 0 || head_dim > 256 || head_dim % 8 || pool_rows <= 0 || max_kv_len < 0 ||
        max_kv_len > kMaxCluster * kMaxItems * kMaxThreads || stride < max_kv_len || budget < 1 || sink < 0 ||
        recent < 0 || static_cast<int64_t>(sink) + recent > budget)
        return SMOL_B200_ERR_ARGS;
    if ((reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool)) & 15) return SMOL_B200_ERR_ARGS;
    const EvictLayout L = evict_layout(n_seqs, max_kv_len, n_kv_heads);
    if (!workspace || workspace_bytes < L.total || (reinterpret_cast<uintptr_t>(workspace) & 15))
        return SMOL_B200_ERR_WORKSPACE;
    EvictParams p;
    memset(&p, 0, sizeof(p));
    uint8_t *base = static_cast<uint8_t *>(workspace);
    p.k = k_pool;
    p.v = v_pool;
    p.pool_rows = pool_rows;
    p.seq_row0 = seq_row0;
    p.weights_in = weights_in;
    p.weights_out = weights_out;
    p.positions_in = positions_in;
    p.positions_out = positions_out;
    p.stride = stride;
    p.kv_len_in = kv_len_in;
    p.kv_len_out = kv_len_out;
    p.seq_pos = seq_pos;
    p.lists = reinterpret_cast<int *>(base);
    p.lengths = reinterpret_cast<int *>(base + L.lengths);
    p.err = device_error_word();
    if (!p.err) return SMOL_B200_ERR_CUDA;
    p.n_kv_heads = n_kv_heads;
    p.hd = head_dim;
    p.max_kv_len = max_kv_len;
    p.budget = budget;
    p.sink = sink;
    p.recent = recent;
    p.cap = L.cap;
    const int most = budget < max_kv_len - budget ? budget : max_kv_len - budget;   // moves of one head
    p.smem_lists = most <= kSmemMoves;
    p.write_len = kv_len_out != kv_len_in;
    // One CTA of up to 1024 threads (which fill an SM's registers) per (sequence, KV head), or a
    // cluster: for more slots than it can hold, and while the CTAs still run at once and have
    // more than two slots a thread.
    const long long units = static_cast<long long>(n_seqs) * n_kv_heads;
    int C = 1;
    while (C < kMaxCluster && (max_kv_len > C * kMaxItems * kMaxThreads ||
                               (units * C * 2 <= 148 && max_kv_len > C * 2 * kMaxThreads)))
        C *= 2;
    const int per = (max_kv_len + C - 1) / C;
    int threads = per >= 4 * kMaxThreads ? kMaxThreads : ((per + 3) / 4 + 31) / 32 * 32;
    if (threads < 128) threads = 128;
    const int items = per > 0 ? (per + threads - 1) / threads : 1;
    PdlScope pdl(g_api_pdl);
    cudaError_t e;
    if (items <= 4) e = launch_evict<4>(st, p, C, threads, n_seqs);
    else if (items <= 8) e = launch_evict<8>(st, p, C, threads, n_seqs);
    else if (items <= 16) e = launch_evict<16>(st, p, C, threads, n_seqs);
    else e = launch_evict<32>(st, p, C, threads, n_seqs);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return SMOL_B200_ERR_CUDA;
    }
    if (!p.write_len) {
        if (launch_kernel(evict_length_kernel, dim3((n_seqs + 255) / 256), dim3(256), 0, st, kv_len_out,
                          static_cast<const int *>(p.lengths), n_seqs) != cudaSuccess)
            return SMOL_B200_ERR_CUDA;
    }
    return SMOL_B200_OK;
}

}  // namespace smolb200
