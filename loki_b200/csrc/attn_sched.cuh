// attn_sched.cuh -- equal cuts of a ragged batch's work, made on the device from the lengths.
//
// Sequence b has ceil(n_b * H / rows per item) items of ceil((len_b + n_b) / TILE) tiles; (item, tile) units are numbered
// sequence by sequence, item by item.  Run q of `used` takes units [W q / used, W (q + 1) / used).
#pragma once
#include "attn_internal.h"

namespace lk {

constexpr int ATT_TILE = 128, ATT_ITEM = 128;

struct TreeWork {
    float4* part;              // [2 per run][512 / 4][128 rows]: O of a run's first and last item where it has only part of it
    float2* ml;                // [2 per run][128 rows]: reference and sum
    int64_t* prefix;           // [n_seqs + 1] units before each sequence
};

struct Segment {
    int b, first, n, len, total;       // sequence, its first drafted token, drafted tokens, context, all rows
    int rt, t0, t1;                    // item of the sequence, tiles
    bool whole;                        // the item's every tile
};

// units before each sequence, prefix[n_seqs] all of them; every thread of the block calls it, the caller synchronises
template <int TILE>
__device__ __forceinline__ void sched_prefix(const TreeParams& p, int64_t* prefix, int tid, int threads) {
    for (int b = tid; b < p.kv.n_seqs; b += threads) {
        const int len = kv_len(p.kv, b, p.err), n = seq_tokens(p.starts, b, p.T, len, p.kv, p.err).y;
        prefix[b + 1] = n ? (int64_t)((n * p.H + ATT_ITEM - 1) / ATT_ITEM) * ((len + n + TILE - 1) / TILE) : 0;
    }
    __syncthreads();
    if (tid < 32) {
        int64_t before = 0;
        for (int b0 = 0; b0 < p.kv.n_seqs; b0 += 32) {
            int64_t v = b0 + tid < p.kv.n_seqs ? prefix[b0 + tid + 1] : 0;
            #pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t w = __shfl_up_sync(0xffffffffu, v, o);
                if (tid >= o) v += w;
            }
            if (b0 + tid < p.kv.n_seqs) prefix[b0 + tid + 1] = before + v;
            before += __shfl_sync(0xffffffffu, v, 31);
        }
        if (tid == 0) prefix[0] = 0;
    }
}

// the next segment of [u, u_end): consecutive tiles of one item
template <int TILE>
__device__ __forceinline__ bool sched_next(const TreeParams& p, const int64_t* prefix, int64_t& u, int64_t u_end, Segment& g) {
    if (u >= u_end) return false;
    int lo = 0, hi = p.kv.n_seqs - 1;                    // the last sequence that starts at or before u and has units
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (prefix[mid] <= u) lo = mid; else hi = mid - 1;
    }
    g.b = lo;
    g.len = kv_len(p.kv, lo, nullptr);
    const int2 sp = seq_tokens(p.starts, lo, p.T, g.len, p.kv, nullptr);
    g.first = sp.x; g.n = sp.y; g.total = g.len + g.n;
    const int tiles = (g.total + TILE - 1) / TILE;
    const int64_t rem = u - prefix[lo];
    g.rt = (int)(rem / tiles);
    g.t0 = (int)(rem % tiles);
    g.t1 = (int)min((int64_t)tiles, g.t0 + (u_end - u));
    g.whole = g.t0 == 0 && g.t1 == tiles;
    u += g.t1 - g.t0;
    return true;
}

// runs that a call is cut into
__host__ __device__ __forceinline__ int sched_pairs(int64_t W, int pairs) { return W < pairs ? (int)W : pairs; }
// the run that has unit u: the last q with W q / used <= u.  A run leaves a part of its first item in slot 2 q and of its
// last in 2 q + 1, so an item that starts inside run q has its first part in 2 q + 1 and the others in even slots
__device__ __forceinline__ int sched_owner(int64_t u, int64_t W, int used) { return (int)(((u + 1) * used + W - 1) / W) - 1; }
template <class T> __device__ __forceinline__ uint32_t nonfinite2(uint32_t v);
template <> __device__ __forceinline__ uint32_t nonfinite2<__half>(uint32_t v) { return (v & 0x7C00u) == 0x7C00u || (v & 0x7C000000u) == 0x7C000000u; }
template <> __device__ __forceinline__ uint32_t nonfinite2<__nv_bfloat16>(uint32_t v) { return (v & 0x7F80u) == 0x7F80u || (v & 0x7F800000u) == 0x7F800000u; }

}  // namespace lk
