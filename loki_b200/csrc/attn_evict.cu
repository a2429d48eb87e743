// attn_evict.cu -- eviction of cached rows by their accumulated attention weight.
//
// Each row gets a 32-bit key whose unsigned order is the rank: all ones for a protected row, else the mass with its
// bits made monotone (NaN: 0).  The budget-th largest key T is found by a radix selection, most significant 8 bits
// first; rows above T stay, and the first (budget - count) rows equal to it.  The kept rows at or beyond `budget` are
// as many as the dropped ones before it, and the two sets are disjoint: the i-th of the former moves into the i-th of
// the latter, all of them at once, and no other row is touched.
#include "attn_internal.h"

namespace lk {

constexpr int EV_THREADS = 1024;

__device__ __forceinline__ uint32_t evict_key(const EvictParams& p, int slot, int next) {
    if (slot < 0) return 0;
    const int pos = p.kv.pos[slot];
    if (pos < p.sinks || pos >= next - p.recent) return 0xFFFFFFFFu;
    const float m = p.kv.mass[slot] + 0.0f;                      // -0 and 0 are equal
    if (m != m) return 0;
    const uint32_t u = __float_as_uint(m);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// exclusive rank of a predicate over the block, in thread order; total in *sum
__device__ __forceinline__ int block_rank(bool pred, int* warp_sum, int* sum) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t m = __ballot_sync(0xffffffffu, pred);
    __syncthreads();
    if (lane == 0) warp_sum[warp] = __popc(m);
    __syncthreads();
    int before = 0, total = 0;
    for (int w = 0; w < EV_THREADS / 32; ++w) { if (w < warp) before += warp_sum[w]; total += warp_sum[w]; }
    *sum = total;
    return before + __popc(m & ((1u << lane) - 1));
}

__global__ void __launch_bounds__(EV_THREADS) k_evict_select(EvictParams p) {
    __shared__ int hist[256];
    __shared__ int warp_sum[EV_THREADS / 32];
    __shared__ uint32_t s_prefix;
    __shared__ int s_need;
    const int b = blockIdx.x, tid = threadIdx.x;
    const int len = kv_len(p.kv, b, p.err);
    if (len <= p.budget) {
        __syncthreads();
        if (tid == 0) { p.n_moves[b] = 0; p.new_lens[b] = len; }
        return;
    }
    const int next = p.next_pos[b];
    uint32_t prefix = 0;
    int need = p.budget;                                         // rank of the threshold among keys with this prefix
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int i = tid; i < len; i += EV_THREADS) {
            const uint32_t k = evict_key(p, kv_slot(p.kv, b, i, p.err), next);
            if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
        }
        __syncthreads();
        if (tid == 0) {
            int d = 255;
            while (d > 0 && hist[d] < need) need -= hist[d--];
            s_prefix = prefix | (uint32_t)d << shift;
            s_need = need;
        }
        __syncthreads();
        prefix = s_prefix; need = s_need;
    }
    int eq = 0, holes = 0, moved = 0;
    int* src = p.src + b * p.region;
    int* dst = p.dst + b * p.region;
    for (int i0 = 0; i0 < len; i0 += EV_THREADS) {
        const int i = i0 + tid;
        const int slot = i < len ? kv_slot(p.kv, b, i, p.err) : -1;
        const uint32_t k = i < len ? evict_key(p, slot, next) : 0;
        int n;
        const int er = eq + block_rank(i < len && k == prefix, warp_sum, &n);
        eq += n;
        const bool keep = i < len && (k > prefix || (k == prefix && er < need));
        const bool hole = i < p.budget && !keep, tail = i >= p.budget && keep;
        const int hr = holes + block_rank(hole, warp_sum, &n);
        holes += n;
        const int tr = moved + block_rank(tail, warp_sum, &n);
        moved += n;
        if (hole) dst[hr] = slot;
        if (tail) src[tr] = slot;
    }
    if (tid == 0) { p.n_moves[b] = holes; p.new_lens[b] = p.budget; }
}

// one warp per move: the row as 16-byte words, then its mass and position
__global__ void __launch_bounds__(256) k_evict_move(EvictParams p) {
    const int lane = threadIdx.x & 31;
    const int b = blockIdx.y, n = p.n_moves[b];
    for (int m = (blockIdx.x * blockDim.x + threadIdx.x) >> 5; m < n; m += (gridDim.x * blockDim.x) >> 5) {
        const int s = p.src[b * p.region + m], d = p.dst[b * p.region + m];
        if (s < 0 || d < 0) continue;
        const uint4* from = (const uint4*)((const uint16_t*)p.kv.rows + (int64_t)s * p.kv.row_stride);
        uint4* to = (uint4*)((uint16_t*)p.kv.rows + (int64_t)d * p.kv.row_stride);
        for (int c = lane; c < AT_ROW / 8; c += 32) to[c] = from[c];
        if (lane == 0) { p.kv.mass[d] = p.kv.mass[s]; p.kv.pos[d] = p.kv.pos[s]; }
    }
}

cudaError_t launch_evict(const EvictParams& p, int nsm, cudaStream_t st) {
    k_evict_select<<<p.kv.n_seqs, EV_THREADS, 0, st>>>(p);
    const int per = (8 * nsm + p.kv.n_seqs - 1) / p.kv.n_seqs;
    k_evict_move<<<dim3(per, p.kv.n_seqs), 256, 0, st>>>(p);
    return cudaGetLastError();
}

}  // namespace lk
