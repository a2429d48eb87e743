// attn_sched.cuh -- equal cuts of a ragged batch's work, made on the device from the lengths.
//
// Every sequence has units of about equal cost, numbered sequence by sequence and cut into `runs` of `base` or base + 1 units,
// the longer ones first.  Attention: sequence b has ceil(n_b * H / 128) items of ceil((len_b + n_b) / TILE) tiles, each item's
// after LEAD units that stand for what a further item costs a pair (Q, the output, an empty pipeline).
#pragma once
#include "attn_internal.h"

namespace lk {

constexpr int ATT_TILE = 128, ATT_ITEM = 128;

// a call's sequences, in shared memory
struct Sched {
    int64_t prefix[LK_ATTN_MAX_SEQS + 1];      // units before each sequence, the last: all of them
    int len[LK_ATTN_MAX_SEQS];                 // context rows
    int start[LK_ATTN_MAX_SEQS + 1];           // drafted tokens
    int64_t base; int more, runs;              // units of a run, runs of one unit more, all runs
    __device__ __forceinline__ int64_t run_start(int q) const { return q * base + min(q, more); }
    // the run that has unit u.  A run leaves a part of its first item in slot 2 q and of its last in 2 q + 1, so an item that
    // starts inside run q has its first part in 2 q + 1 and the others in even slots
    __device__ __forceinline__ int owner(int64_t u) const;
    // the sequence that has unit u: the last that starts at or before it
    __device__ __forceinline__ int sequence(int64_t u, int n_seqs) const {
        int lo = 0, hi = n_seqs - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (prefix[mid] <= u) lo = mid; else hi = mid - 1;
        }
        return lo;
    }
};

// 64-bit values that nearly always fit 32 bits, where a division takes a fifth of the instructions
__device__ __forceinline__ int64_t div_small(int64_t a, int64_t b) {
    return (a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}
__device__ __forceinline__ int Sched::owner(int64_t u) const {
    const int64_t longer = more * (base + 1);
    return (int)(u < longer ? div_small(u, base + 1) : more + div_small(u - longer, base));
}

struct Segment {
    int b, first, n, len, total;               // sequence, its first drafted token, drafted tokens, context, all rows
    int rt, t0, t1, tiles;                     // item of the sequence, tiles [t0, t1) of its `tiles`
    int64_t item;                              // the item's first unit
    __device__ __forceinline__ bool whole() const { return t1 - t0 == tiles; }
};

// units(n, tiles): the units of a sequence with n drafted tokens; then(): the whole block again, after the sequences' fields are
// there and before the units are summed (it may change s.prefix[b + 1], still the sequence's own units).
// the whole block calls it (one sequence: its first warp is enough), for at most `pairs` runs and no more than the longest
// run's length needs; the caller synchronises before it reads the runs
template <int TILE, class Units, class Then>
__device__ __forceinline__ void sched_load(const TreeParams& p, Sched& s, int tid, int threads, int pairs, Units units_of, Then then) {
    for (int b = tid; b < p.kv.n_seqs; b += threads) {
        const int len0 = p.kv.lens[b], t0 = p.starts[b], t1 = p.starts[b + 1], cap = p.kv.table_stride << p.kv.page_shift;
        const int len = min(max(len0, 0), cap), n = t1 - t0;
        int64_t units = 0;
        if (len != len0) att_error(p.err, ATT_ERR_LEN);
        if (t0 < 0 || n < 0 || t1 > p.T || n > LK_ATTN_MAX_NODES) att_error(p.err, ATT_ERR_TREE);
        else if (n > cap - len) att_error(p.err, ATT_ERR_LEN);
        else if (n) units = units_of(n, (len + n + TILE - 1) / TILE);
        s.len[b] = len;
        s.start[b] = t0;
        if (b == p.kv.n_seqs - 1) s.start[b + 1] = t1;
        s.prefix[b + 1] = units;
    }
    if (tid == 0) s.prefix[0] = 0;
    if (p.kv.n_seqs > 1) __syncthreads(); else __syncwarp();
    then();
    if (tid < 32) {
        __syncwarp();
        int64_t before = 0;
        for (int b0 = 0; b0 < p.kv.n_seqs; b0 += 32) {
            int64_t v = b0 + tid < p.kv.n_seqs ? s.prefix[b0 + tid + 1] : 0;
            #pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t w = __shfl_up_sync(0xffffffffu, v, o);
                if (tid >= o) v += w;
            }
            if (b0 + tid < p.kv.n_seqs) s.prefix[b0 + tid + 1] = before + v;
            before += __shfl_sync(0xffffffffu, v, 31);
        }
        if (tid == 0) {
            const int64_t per = div_small(before + pairs - 1, pairs);
            s.runs = before ? (int)div_small(before + per - 1, per) : 0;
            s.base = before ? div_small(before, s.runs) : 0;
            s.more = (int)(before - s.runs * s.base);
        }
    }
}

// the next segment of [u, u_end): consecutive tiles of one item
template <int TILE, int LEAD>
__device__ __forceinline__ bool sched_next(const TreeParams& p, const Sched& s, int64_t& u, int64_t u_end, Segment& g) {
    for (;;) {
        if (u >= u_end) return false;
        const int lo = s.sequence(u, p.kv.n_seqs);
        g.b = lo;
        g.len = s.len[lo];
        g.first = s.start[lo];
        g.n = s.start[lo + 1] - g.first;
        g.total = g.len + g.n;
        g.tiles = (g.total + TILE - 1) / TILE;
        const int64_t rem = u - s.prefix[lo];
        g.rt = rem < LEAD + g.tiles ? 0 : (int)div_small(rem, LEAD + g.tiles);
        const int at = (int)(rem - (int64_t)g.rt * (LEAD + g.tiles)), end = (int)min((int64_t)(LEAD + g.tiles), at + (u_end - u));
        g.item = u - at;
        g.t0 = max(0, at - LEAD);
        g.t1 = end - LEAD;
        u += end - at;
        if (g.t1 > g.t0) return true;
    }
}

template <class T> __device__ __forceinline__ uint32_t nonfinite2(uint32_t v);
template <> __device__ __forceinline__ uint32_t nonfinite2<__half>(uint32_t v) { return (v & 0x7C00u) == 0x7C00u || (v & 0x7C000000u) == 0x7C000000u; }
template <> __device__ __forceinline__ uint32_t nonfinite2<__nv_bfloat16>(uint32_t v) { return (v & 0x7F80u) == 0x7F80u || (v & 0x7F800000u) == 0x7F800000u; }

}  // namespace lk
