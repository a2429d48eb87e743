// attn_evict.cu -- eviction of cached rows by their accumulated attention weight.
//
// Each row gets a 32-bit key whose unsigned order is the rank: all ones for a protected row, else the mass with its
// bits made monotone (NaN: 0).  The budget-th largest key T is found by a radix selection, most significant 8 bits
// first; rows above T stay, and the first (budget - count) rows equal to it.  The kept rows at or beyond `budget` are
// as many as the dropped ones before it, and the two sets are disjoint: the i-th of the former moves into the i-th of
// the latter, all of them at once, and no other row is touched.
//
// k_evict_select: a cluster of 8 CTAs per sequence, each with an eighth of its rows in order, whose keys it keeps in shared
// memory (sequences of up to 8 x EV_KEYS rows; beyond, it computes them again in each pass).  Per digit the CTAs' histograms
// are added over distributed shared memory by each CTA alike, so one cluster barrier a digit is all they exchange; ranks come
// from ordered block scans and the CTAs' totals.  It reads 8 bytes a row once and is bound by its ~10 barriers and scans
// (one CTA per sequence took 170 us of a 16-sequence call).
// k_evict_move: 72 threads copy a row's 1152 bytes, two rows in flight; rows lie anywhere in the pool.
// Times a call with mass and pos put back before each (a call leaves nothing for the next on the same cache to move): 1200 rows
// cut to 1024, 167 of them moved, 14.3 us, nearly all of it the selection; 16 sequences of 6000 to 40 000 rows cut to 8192, 74 135
// rows moved, 66: the selection 22, the moves 42 (171 MB read and written, 4.1 TB/s).  The plain forms 305 and 665.
#include "attn_tc.cuh"
#include "moe_internal.h"

namespace lk {

constexpr int EV_THREADS = 1024, EV_CTAS = 8, EV_KEYS = 48 * 1024;
constexpr int EV_WARPS = EV_THREADS / 32;

__device__ __forceinline__ uint32_t evict_key(const EvictParams& p, int slot, int next) {
    if (slot < 0) return 0;
    const int pos = p.kv.pos[slot];
    const float m = p.kv.mass[slot] + 0.0f;                      // -0 and 0 are equal
    if (pos < p.sinks || pos >= next - p.recent) return 0xFFFFFFFFu;
    if (m != m) return 0;
    const uint32_t u = __float_as_uint(m);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// what a CTA shows the others of its cluster
struct EvictShared {
    int hist[2][256];                                            // by digit parity
    int eq, holes, tails;
};

// exclusive prefix of v over the block's threads, and the block's total
__device__ __forceinline__ int block_scan(int v, int* warp_sum, int* total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int x = v;
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x += y; }
    __syncthreads();                                             // warp_sum of the last scan is free
    if (lane == 31) warp_sum[warp] = x;
    __syncthreads();
    int w = warp_sum[lane];
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, w, o); if (lane >= o) w += y; }
    *total = __shfl_sync(0xffffffffu, w, 31);
    const int before = __shfl_sync(0xffffffffu, w, warp ? warp - 1 : 0);
    return x - v + (warp ? before : 0);
}

__device__ __forceinline__ int peer_int(const int* v, uint32_t rank) {
    int r;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(r) : "r"(peer_addr(smem_u32(v), rank)) : "memory");
    return r;
}

__global__ void __cluster_dims__(EV_CTAS, 1, 1) __launch_bounds__(EV_THREADS) k_evict_select(EvictParams p) {
    extern __shared__ uint32_t keys[];
    __shared__ EvictShared sh;
    __shared__ int warp_sum[EV_WARPS];
    __shared__ int s_digit, s_need;
    const int b = blockIdx.x / EV_CTAS, tid = threadIdx.x, lane = tid & 31;
    const uint32_t rank = cluster_rank();
    pdl_wait();
    pdl_trigger();
    const int len = kv_len(p.kv, b, p.err);
    if (len <= p.budget) {                                       // the whole cluster alike
        cluster_sync();                                          // every CTA has read lens before new_lens, which may be the same array, is written
        if (rank == 0 && tid == 0) { p.n_moves[b] = 0; p.new_lens[b] = len; }
        return;
    }
    const int next = p.next_pos[b];
    // this CTA's rows [lo, hi); thread t ranks rows [lo + t * per, ..) of them
    const int share = (len + EV_CTAS - 1) / EV_CTAS, lo = min(len, (int)rank * share), hi = min(len, lo + share), n = hi - lo;
    const bool kept_keys = share <= p.keys;
    auto key_at = [&](int i, int* err = nullptr) { return kept_keys ? keys[i - lo] : evict_key(p, kv_slot(p.kv, b, i, err), next); };
    if (kept_keys) for (int i = tid; i < n; i += EV_THREADS) keys[i] = evict_key(p, kv_slot(p.kv, b, lo + i, p.err), next);
    uint32_t prefix = 0;
    int need = p.budget;                                         // rank of the threshold among keys with this prefix
    for (int d = 0; d < 4; ++d) {
        const int shift = 24 - 8 * d;
        int* hist = sh.hist[d & 1];
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int i0 = 0; i0 < n; i0 += EV_THREADS) {
            const int i = i0 + tid;
            const uint32_t k = i < n ? key_at(lo + i, d ? nullptr : p.err) : 0;      // bad pages are reported once
            const bool in = i < n && (d == 0 || (k >> (shift + 8)) == (prefix >> (shift + 8)));
            // one addition per distinct digit of a warp: masses share their leading digits
            const uint32_t digit = in ? (k >> shift) & 255 : 256, same = __match_any_sync(0xffffffffu, digit);
            if (in && lane == __ffs(same) - 1) atomicAdd(&hist[digit], __popc(same));
        }
        cluster_sync();                                          // all histograms of this digit are made (and read by the next but one)
        // digit thread t of 256 (bin 255 - t): keys in this bin and above
        int c = 0, total;
        if (tid < 256)
            #pragma unroll
            for (int q = 0; q < EV_CTAS; ++q) c += peer_int(&hist[255 - tid], q);
        const int above = block_scan(c, warp_sum, &total);
        if (tid < 256 && above < need && above + c >= need) { s_digit = 255 - tid; s_need = need - above; }
        __syncthreads();
        prefix |= (uint32_t)s_digit << shift;
        need = s_need;
    }
    // the first `need` rows equal to the threshold stay
    const int per = (n + EV_THREADS - 1) / EV_THREADS, i0 = lo + min(n, tid * per), i1 = min(hi, i0 + per);
    int eq = 0, total;
    for (int i = i0; i < i1; ++i) eq += key_at(i) == prefix;
    int eq_at = block_scan(eq, warp_sum, &total);
    if (tid == 0) sh.eq = total;
    cluster_sync();
    for (uint32_t q = 0; q < rank; ++q) eq_at += peer_int(&sh.eq, q);
    int holes = 0, tails = 0;
    {
        int e = eq_at;
        for (int i = i0; i < i1; ++i) {
            const uint32_t k = key_at(i);
            const bool keep = k > prefix || (k == prefix && e < need);
            e += k == prefix;
            holes += i < p.budget && !keep;
            tails += i >= p.budget && keep;
        }
    }
    int n_holes, n_tails;
    int hole_at = block_scan(holes, warp_sum, &n_holes), tail_at = block_scan(tails, warp_sum, &n_tails);
    if (tid == 0) { sh.holes = n_holes; sh.tails = n_tails; }
    cluster_sync();
    int all = 0;
    for (uint32_t q = 0; q < EV_CTAS; ++q) {
        const int h = peer_int(&sh.holes, q);
        all += h;
        if (q < rank) { hole_at += h; tail_at += peer_int(&sh.tails, q); }
    }
    int* src = p.src + b * p.region;
    int* dst = p.dst + b * p.region;
    if (holes || tails)
        for (int i = i0; i < i1; ++i) {
            const uint32_t k = key_at(i);
            const bool keep = k > prefix || (k == prefix && eq_at < need);
            eq_at += k == prefix;
            if (i < p.budget && !keep) dst[hole_at++] = kv_slot(p.kv, b, i, nullptr);
            if (i >= p.budget && keep) src[tail_at++] = kv_slot(p.kv, b, i, nullptr);
        }
    if (rank == 0 && tid == 0) { p.n_moves[b] = all; p.new_lens[b] = p.budget; }
    cluster_sync();                                              // a CTA's shared memory outlives the others' reads of it
}

// 72 threads a row, 4 rows a pass of the block, two passes' loads in flight; then the row's mass and position
constexpr int EM_LANES = AT_ROW / 8, EM_ROWS = 4;

__global__ void __launch_bounds__(EM_LANES * EM_ROWS) k_evict_move(EvictParams p) {
    pdl_wait();
    pdl_trigger();
    const int b = blockIdx.y, n = (int)min((int64_t)p.n_moves[b], p.region), c = threadIdx.x % EM_LANES, r = threadIdx.x / EM_LANES;
    const unsigned pool = (unsigned)p.kv.n_pages << p.kv.page_shift;
    const int* src = p.src + b * p.region;
    const int* dst = p.dst + b * p.region;
    const int step = gridDim.x * EM_ROWS;
    for (int m = blockIdx.x * EM_ROWS + r; m < n; m += 2 * step) {
        const int m2 = m + step;
        const int s0 = src[m], d0 = dst[m], s1 = m2 < n ? src[m2] : -1, d1 = m2 < n ? dst[m2] : -1;
        // a bad page's rows (-1) stay
        const bool go0 = (unsigned)s0 < pool && (unsigned)d0 < pool, go1 = (unsigned)s1 < pool && (unsigned)d1 < pool;
        const uint16_t* rows = (const uint16_t*)p.kv.rows + c * 8;
        uint4 v0, v1;
        if (go0) v0 = __ldcs((const uint4*)(rows + (int64_t)s0 * p.kv.row_stride));
        if (go1) v1 = __ldcs((const uint4*)(rows + (int64_t)s1 * p.kv.row_stride));
        uint16_t* to = (uint16_t*)p.kv.rows + c * 8;
        if (go0) *(uint4*)(to + (int64_t)d0 * p.kv.row_stride) = v0;
        if (go1) *(uint4*)(to + (int64_t)d1 * p.kv.row_stride) = v1;
        if (c == 0 && go0) { p.kv.mass[d0] = p.kv.mass[s0]; p.kv.pos[d0] = p.kv.pos[s0]; }
        if (c == 1 && go1) { p.kv.mass[d1] = p.kv.mass[s1]; p.kv.pos[d1] = p.kv.pos[s1]; }
    }
}

cudaError_t evict_setup() { return cudaFuncSetAttribute(k_evict_select, cudaFuncAttributeMaxDynamicSharedMemorySize, EV_KEYS * 4); }

cudaError_t launch_evict(const EvictParams& p0, int nsm, cudaStream_t st) {
    EvictParams p = p0;
    const int64_t cap = (int64_t)p.kv.table_stride * p.kv.page_size;         // most rows of a sequence
    const int64_t share = (cap + EV_CTAS - 1) / EV_CTAS;
    p.keys = share <= EV_KEYS ? (int)share : EV_KEYS;
    const cudaError_t e = launch_pdl_n(k_evict_select, dim3(p.kv.n_seqs * EV_CTAS), dim3(EV_THREADS), p.keys * 4, st, p);
    if (e != cudaSuccess || p.region == 0) return e;
    // enough blocks for every SM's 7 at a time, and no more than the most rows that can move
    int64_t per = (7 * nsm + p.kv.n_seqs - 1) / p.kv.n_seqs, most = (p.region + EM_ROWS - 1) / EM_ROWS;
    if (per > most) per = most;
    return launch_pdl_n(k_evict_move, dim3((unsigned)per, p.kv.n_seqs), dim3(EM_LANES * EM_ROWS), 0, st, p);
}

}  // namespace lk
