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
// Select.  The B-th largest of the n 32-bit sort keys is found bit by bit, two bits a
// round: keys stay in registers, a round counts those at or above three candidates.  Ties
// at that key are taken in slot order.  One more ordered count gives holes and movers
// their numbers.  A (sequence, KV head) is one CTA or, for long caches, one cluster whose
// CTAs hold a segment of the slots each and exchange counts through shared memory.
//
// Bytes: 8 per slot to read (weight, position), as many to write where the outputs are
// other arrays, and K and V of the moved rows.
#include <string.h>

#include "b200_common.cuh"
#include "runtime.h"

namespace smolb200 {
namespace {

constexpr int kMaxThreads = 1024;
constexpr int kMaxItems = 32;
constexpr int kMaxCluster = 8;
// Moves that the select kernel makes itself; with more possible a second kernel spreads them.
constexpr int kFusedMoves = 64;

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
    int *counts;     // [n_seqs*n_kv_heads] moves
    int *lengths;    // [n_seqs] new lengths
    unsigned *err;
    int n_kv_heads, hd, max_kv_len, budget, sink, recent, cap;
    int fused, write_len;   // this kernel makes the moves / writes kv_len_out
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

// Moves r = first, first + step, ... of (sequence b, head h), one per warp.
__device__ __forceinline__ void move_rows(const EvictParams &p, long long row0, int h, const int *holes,
                                          const int *movers, int m, int first, int step)
{
    const int lane = threadIdx.x % 32;
    const int vecs = p.hd / 8;   // 16-byte pieces of one head's row
    const long long width = static_cast<long long>(p.n_kv_heads) * p.hd;
    for (int r = first; r < m; r += step) {
        const long long dst = (row0 + holes[r]) * width + static_cast<long long>(h) * p.hd;
        const long long src = (row0 + movers[r]) * width + static_cast<long long>(h) * p.hd;
        for (int i = lane; i < 2 * vecs; i += 32) {
            uint16_t *pool = i < vecs ? p.k : p.v;
            const int e = (i < vecs ? i : i - vecs) * 8;
            *reinterpret_cast<uint4 *>(pool + dst + e) = *reinterpret_cast<const uint4 *>(pool + src + e);
        }
    }
}

template <int ITEMS>
__global__ void __launch_bounds__(kMaxThreads) evict_kernel(const __grid_constant__ EvictParams p)
{
    griddep_wait();
    griddep_trigger();
    __shared__ int s_cnt[3][4];                          // counts of a round, three rounds in rotation
    __shared__ int s_box[2][kMaxCluster][3];             // every CTA's counts, by round parity
    __shared__ int s_scan[ITEMS * (kMaxThreads / 32)];   // flags per (item, warp), then their prefix
    __shared__ int s_total, s_tot_box[kMaxCluster];
    const int C = static_cast<int>(gridDim.x), rank = blockIdx.x;
    const int h = blockIdx.y, b = blockIdx.z;
    const int T = blockDim.x, tid = threadIdx.x, warp = tid / 32, lane = tid % 32, W = T / 32;

    const int length = p.kv_len_in[b];
    const long long row0 = p.seq_row0[b];
    const int seen = p.seq_pos[b];
    const int n = min(max(length, 0), p.max_kv_len);
    // a length or rows that cannot be: the sequence is left as it is
    const bool bad = n != length || (n > p.budget && (row0 < 0 || row0 + n > p.pool_rows));
    const bool keep_all = bad || n <= p.budget;
    const int B = keep_all ? length : p.budget;
    const long long unit = static_cast<long long>(b) * p.n_kv_heads + h;
    if (rank == 0 && tid == 0) {
        if (h == 0) {
            if (bad) atomicOr(p.err, kErrBadArgs);
            p.lengths[b] = B;
            if (p.write_len) p.kv_len_out[b] = B;
        }
        if (keep_all) p.counts[unit] = 0;
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

    uint32_t key[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int j = j_first + i * T;
        key[i] = 0u;
        if (j < n) {
            const int pos = slot_position(pos_in[j], j, n, seen);
            key[i] = pos < p.sink || pos >= seen - p.recent ? 0xffffffffu : weight_key(w_in[j]);
        }
    }
    if (tid < 12) s_cnt[tid / 4][tid % 4] = 0;
    __syncthreads();

    // t: the largest key with at least B keys at or above it, two bits a round
    uint32_t t = 0;
    int at_t = n, above = 0;   // keys >= t, keys >= the smallest rejected candidate above t
    for (int round = 0; round < 16; ++round) {
        const int shift = 30 - 2 * round;
        const uint32_t c1 = t | (1u << shift), c2 = t | (2u << shift), c3 = t | (3u << shift);
        int k1 = 0, k2 = 0, k3 = 0;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            k1 += key[i] >= c1;
            k2 += key[i] >= c2;
            k3 += key[i] >= c3;
        }
        k1 = __reduce_add_sync(0xffffffffu, k1);
        k2 = __reduce_add_sync(0xffffffffu, k2);
        k3 = __reduce_add_sync(0xffffffffu, k3);
        int *cnt = s_cnt[round % 3];
        if (lane < 3) atomicAdd(&cnt[lane], lane == 0 ? k1 : lane == 1 ? k2 : k3);
        if (tid < 4) s_cnt[(round + 1) % 3][tid] = 0;   // last read two barriers ago
        __syncthreads();
        int n1 = cnt[0], n2 = cnt[1], n3 = cnt[2];
        if (C > 1) {
            if (tid < C * 3) {   // to every CTA of the cluster
                const uint32_t dst = map_shared_rank(smem_u32(&s_box[round & 1][rank][tid % 3]), tid / 3);
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(dst), "r"(cnt[tid % 3]) : "memory");
            }
            cluster_sync_all();
            n1 = n2 = n3 = 0;
            for (int r = 0; r < C; ++r) {
                n1 += s_box[round & 1][r][0];
                n2 += s_box[round & 1][r][1];
                n3 += s_box[round & 1][r][2];
            }
        }
        if (n3 >= B) t = c3, at_t = n3;
        else if (n2 >= B) t = c2, at_t = n2, above = n3;
        else if (n1 >= B) t = c1, at_t = n1, above = n2;
        else above = n1;
        if (at_t == B) break;   // exactly the keys >= t: no ties to choose from
    }

    // Ordered counts: flags of (CTA, item, thread) order = slot order.  Leaves in s_scan the
    // number of flags before each (item, warp) of the cluster; returns their total.
    auto ordered = [&](uint32_t flags) -> int {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const uint32_t bal = __ballot_sync(0xffffffffu, (flags >> i) & 1u);
            if (lane == 0) s_scan[i * W + warp] = __popc(bal);
        }
        __syncthreads();
        if (warp == 0) {
            int run = 0;
            for (int e0 = 0; e0 < ITEMS * W; e0 += 32) {
                const int e = e0 + lane;
                const int v = e < ITEMS * W ? s_scan[e] : 0;
                int x = v;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, x, o);
                    if (lane >= o) x += y;
                }
                if (e < ITEMS * W) s_scan[e] = run + x - v;
                run += __shfl_sync(0xffffffffu, x, 31);
            }
            if (lane == 0) s_total = run;
        }
        __syncthreads();
        int total = s_total;
        if (C > 1) {
            if (tid < C) {
                const uint32_t dst = map_shared_rank(smem_u32(&s_tot_box[rank]), tid);
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(dst), "r"(total) : "memory");
            }
            cluster_sync_all();
            int before = 0;
            total = 0;
            for (int r = 0; r < C; ++r) {
                if (r < rank) before += s_tot_box[r];
                total += s_tot_box[r];
            }
            cluster_sync_all();   // every CTA has read its box before the next count writes it
            for (int e = tid; e < ITEMS * W; e += T) s_scan[e] += before;
            __syncthreads();
        }
        return total;
    };
    auto before_me = [&](uint32_t flags, int i) -> int {   // flags before this thread's item i
        const uint32_t bal = __ballot_sync(0xffffffffu, (flags >> i) & 1u);
        return s_scan[i * W + warp] + __popc(bal & ((1u << lane) - 1u));
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
    int *holes = p.lists + unit * 2 * p.cap, *movers = holes + p.cap;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int j = j_first + i * T;
        const int k = before_me(moved, i);
        if ((moved >> i) & 1u) {
            if (j < B) holes[k] = j;
            else movers[k - m] = j;
        }
    }
    if (rank == 0 && tid == 0) p.counts[unit] = m;
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
    __threadfence();
    __syncthreads();
    if (C > 1) cluster_sync_all();   // the lists are complete
    for (int r = rank * T + tid; r < m; r += C * T) {
        const int src = movers[r], dst = holes[r];
        w_out[dst] = w_in[src];
        pos_out[dst] = slot_position(pos_in[src], src, n, seen);
    }
    if (p.fused) move_rows(p, row0, h, holes, movers, m, rank * W + warp, C * W);
    __syncthreads();
    if (C > 1) cluster_sync_all();   // every mover has been read
#pragma unroll 4
    for (int i = 0; i < ITEMS; ++i) {
        const int j = j_first + i * T;
        if (j >= B && j < n) {
            w_out[j] = 0.f;
            pos_out[j] = -1;
        }
    }
}

constexpr int kMoveThreads = 256;

__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const __grid_constant__ EvictParams p)
{
    griddep_wait();
    griddep_trigger();
    const int h = blockIdx.y, b = blockIdx.z;
    const long long unit = static_cast<long long>(b) * p.n_kv_heads + h;
    if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) p.kv_len_out[b] = p.lengths[b];
    const int m = p.fused ? 0 : p.counts[unit];
    const int *holes = p.lists + unit * 2 * p.cap;
    const int W = kMoveThreads / 32;
    move_rows(p, p.seq_row0[b], h, holes, holes + p.cap, m, blockIdx.x * W + threadIdx.x / 32, gridDim.x * W);
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
    size_t counts, lengths, total;
    int cap;
};

EvictLayout evict_layout(int n_seqs, int max_kv_len, int n_kv_heads)
{
    auto al = [](size_t x) { return (x + 255) & ~size_t(255); };
    EvictLayout L;
    const size_t units = static_cast<size_t>(n_seqs) * n_kv_heads;
    L.cap = max_kv_len / 2 + 1;   // min(B, n - B) moves at most
    L.counts = al(units * 2 * L.cap * 4);
    L.lengths = L.counts + al(units * 4);
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
    p.counts = reinterpret_cast<int *>(base + L.counts);
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
    p.fused = most <= kFusedMoves;
    p.write_len = p.fused && kv_len_out != kv_len_in;
    // Slots per CTA: one CTA per (sequence, KV head) while there are enough of them, else a
    // cluster; never more than kMaxItems per thread.
    const long long units = static_cast<long long>(n_seqs) * n_kv_heads;
    int C = 1;
    while (C < kMaxCluster && (max_kv_len > C * kMaxItems * kMaxThreads ||
                               (units * C < 148 && max_kv_len > C * 2 * kMaxThreads)))
        C *= 2;
    const int per = (max_kv_len + C - 1) / C;
    int threads = per >= 4 * kMaxThreads ? kMaxThreads : (per / 4 + 31) / 32 * 32;
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
    if (!p.fused) {
        const int per_cta = kMoveThreads / 32 * 4;   // four moves a warp
        int x = (most + per_cta - 1) / per_cta;
        if (x > 256) x = 256;
        if (launch_kernel(evict_move_kernel, dim3(x, n_kv_heads, n_seqs), dim3(kMoveThreads), 0, st, p) !=
            cudaSuccess)
            return SMOL_B200_ERR_CUDA;
    } else if (!p.write_len) {
        if (launch_kernel(evict_length_kernel, dim3((n_seqs + 255) / 256), dim3(256), 0, st, kv_len_out,
                          static_cast<const int *>(p.lengths), n_seqs) != cudaSuccess)
            return SMOL_B200_ERR_CUDA;
    }
    return SMOL_B200_OK;
}

}  // namespace smolb200
