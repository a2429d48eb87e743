// attn_mass.cu -- the attention weight that every cached row received:
//   mass[k] = decay * mass[k] + sum_t w_t sum_h exp(scale q_th . row_k - lse_th).
//
// The sum runs over the rows of the score matrix, so with the lse known each key adds its terms alone.  The products are
// S^T = K Q^T: a pair of CTAs holds 256 keys (M = 256: 128 each, the tensor-memory lanes) and runs over the (token, head) rows
// in blocks of up to 256 (N); a key's scores then lie in one lane, and its sum is a loop over columns without any exchange.
// w exp(s - lse) = 2^(s' - c), c = lse / ln 2 - log2 w; tokens without a positive weight are left out of the rows.  A key's
// terms are added in a fixed order: nothing depends on timing.
//
// Bounds: 2 x 256 x 256 x 576 products of a block take 4608 cycles of both tensor pipes, its 65 536 exponentials 2048 cycles of
// each SM's; Q is re-read per key tile (16 KB per 512 cycles and SM, from L2).  Measured 531 cycles a chunk of 512.  With one
// block (a decoded token) the cache's 1152 bytes a key from HBM are the bound, and below a tile a pair the set-up of 3 us.
// Times a call: 4 sequences x 12 nodes, 128 heads, 10 000 to 30 000 rows, 60 % of the weights positive: 81 to 93 us by the clock
// that the power allows (53 to 61 of products; the plain form 6600); one token over 8191 rows 11.5 with the cache from HBM, 9.7 where it
// is in L2 from the attention before it (819).
//
// The key tile stays in shared memory (9 chunks of 64 values, 144 KB); each chunk is replaced as soon as the last row block has
// read it, so the next tile's loads run under the rest.  Q chunks go through a ring of 4 (16 KB: the CTA's half of the rows x 64
// values), as boxes of `hb` heads of a token: heads are padded to a multiple of 8, which the tensor map fills with zeros, and hb
// is the largest power of two up to 64 that divides that.  (Q by cp.async took 1150 cycles a chunk, of 512 of MMAs.)
// Roles (384 threads): warp 0 loads K, warp 1 of CTA 0 issues the MMAs, warp 2 loads Q, warps 4-11 add.
#include <type_traits>
#include "attn_tc.cuh"
#include "attn_sched.cuh"
#include "moe_internal.h"

namespace lk {

constexpr int MS_THREADS = 384, MS_TILE = 256, MS_ROWS = 256, MS_CHUNK = 16384, MS_RING = 4;
constexpr int MS_Q = 9 * MS_CHUNK, MS_BARS = MS_Q + MS_RING * MS_CHUNK, MS_COL = MS_BARS + 48 * 8;
constexpr int MS_TOK = MS_COL + 2 * MS_ROWS * 4, MS_PART = MS_TOK + 2 * MS_ROWS, MS_ACT = MS_PART + 128 * 4, MS_MASK = MS_ACT + 64 * 4;
constexpr int MS_HALVES = MS_MASK + 64 * 8, MS_SCHED = MS_HALVES + 2 * LK_ATTN_MAX_SEQS;
constexpr int MS_SMEM = MS_SCHED + (int)sizeof(Sched);
static_assert(MS_SMEM <= 232448 && MS_SCHED % 8 == 0, "227 KB a CTA");

struct MassBars {
    uint64_t k_full[9], k_empty[9], q_full[MS_RING], q_empty[MS_RING], d_full[2], d_free[2], drain;
    uint32_t tmem;
    int gave_up, n_act, last;
};
static_assert(sizeof(MassBars) <= 48 * 8, "barrier block");

__host__ __device__ inline int mass_heads(int H) { return (H + 7) & ~7; }            // padded heads
__host__ __device__ inline int mass_box(int H) { const int p = mass_heads(H), b = p & -p; return b < 64 ? b : 64; }
// columns of the MMA for `rows` rows of a block: whole boxes in each CTA's half
__device__ __forceinline__ int mass_cols(int rows, int hb) { const int u = max(32, 2 * hb); return (min(rows, MS_ROWS) + u - 1) / u * u; }

// Units: half a block of rows (128 columns of the MMA) over one key tile, 2304 cycles of products.  A tile has as many as its
// rows need, but at least MS_MIN, the time its 288 KB take from HBM when all pairs load; the work is the last ones, so a
// tile of one half block is never split.  A tile that several runs share is read by each; they leave their sums in `part`
// (run q: slot 2 q for its first tile, 2 q + 1 for its last) and the last to arrive adds them, in the runs' order.  With whole
// tiles as units 4 x 12 nodes are 313 tiles for 74 pairs, and sequences differ in their rows: 111 us to 80 with this and the mask
// of drafted keys taken once a tile.
constexpr int MS_HALF = 128, MS_MIN = 3;

struct MassSegment {
    int b, first, n, len, total;              // sequence, its first drafted token, drafted tokens, context, all rows
    int j, off, per, work;                    // next tile, the next unit of its `per`, of which the last `work` are rows
    int64_t unit, left;                       // unit 0 of that tile, units that remain
    // the next piece of work: half blocks [h0, h1) of a tile
    __device__ __forceinline__ bool next(int& tile, int& h0, int& h1) {
        while (left > 0) {
            const int end = (int)min((int64_t)per, off + left), skip = per - work;
            tile = j; h0 = max(off, skip) - skip; h1 = end - skip;
            left -= end - off; unit += per; ++j; off = 0;
            if (h1 > h0) return true;
        }
        return false;
    }
};

__device__ __forceinline__ bool mass_next(const TreeParams& p, const Sched& s, const uint16_t* halves, int64_t& u, int64_t u_end, MassSegment& g) {
    if (u >= u_end) return false;
    g.b = s.sequence(u, p.kv.n_seqs);
    g.len = s.len[g.b];
    g.first = s.start[g.b];
    g.n = s.start[g.b + 1] - g.first;
    g.total = g.len + g.n;
    g.work = max((int)halves[g.b], 1);
    g.per = max(g.work, MS_MIN);
    const int64_t rem = u - s.prefix[g.b];
    g.j = (int)div_small(rem, g.per);
    g.off = (int)(rem - (int64_t)g.j * g.per);
    g.unit = u - g.off;
    g.left = min(u_end, s.prefix[g.b + 1]) - u;
    u += g.left;
    return true;
}

template <class T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(MS_THREADS, 1)
k_mass(const __grid_constant__ TreeParams p, const __grid_constant__ CUtensorMap kv_map, const __grid_constant__ CUtensorMap q_map,
       const MassWork wk) {
    extern __shared__ __align__(1024) uint8_t sm[];
    MassBars& B = *(MassBars*)(sm + MS_BARS);
    float* col = (float*)(sm + MS_COL);                       // [2][256] c of each row of a block
    uint8_t* tok = sm + MS_TOK;                               // [2][256] its token's place in act
    float* part = (float*)(sm + MS_PART);                     // [128]
    int* act = (int*)(sm + MS_ACT);                           // the segment's tokens of positive weight (within the sequence)
    uint64_t* see = (uint64_t*)(sm + MS_MASK);                // the drafted rows that each of them sees
    uint16_t* halves = (uint16_t*)(sm + MS_HALVES);           // half blocks of rows of each sequence
    Sched& sched = *(Sched*)(sm + MS_SCHED);
    volatile int* gave_up = &B.gave_up;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = cluster_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;

    if (warp == 2 && lane == 0) {
        B.gave_up = 0;
        for (int i = 0; i < 9; ++i) { mbar_init(&B.k_full[i], 2); mbar_init(&B.k_empty[i], 1); }
        for (int i = 0; i < MS_RING; ++i) { mbar_init(&B.q_full[i], 2); mbar_init(&B.q_empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&B.d_full[i], 1); mbar_init(&B.d_free[i], 16); }
        mbar_init(&B.drain, 1);
        fence_mbar_init();
        asm volatile("prefetch.tensormap [%0];" :: "l"(&kv_map) : "memory");
        asm volatile("prefetch.tensormap [%0];" :: "l"(&q_map) : "memory");
    }
    __syncwarp();
    cluster_arrive();                                         // the barriers are there; the wait is below, after the schedule
    if (warp == 3) tmem_alloc2(&B.tmem, 512);
    pdl_wait();
    pdl_trigger();
    if (warp == 0 || p.kv.n_seqs > 1)
        sched_load<MS_TILE>(p, sched, tid, MS_THREADS, pairs, [](int, int tiles) { return (int64_t)tiles; }, [&]() {
            const int warps = p.kv.n_seqs > 1 ? MS_THREADS / 32 : 1;
            for (int b0 = warp; b0 < p.kv.n_seqs; b0 += 4 * warps) {          // four sequences' weights in flight
                int got[4];
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int b = b0 + i * warps, t0 = b < p.kv.n_seqs ? sched.start[b] : 0;
                    const int n = b < p.kv.n_seqs && sched.prefix[b + 1] ? sched.start[b + 1] - t0 : 0;
                    got[i] = 0;
                    if (lane < n) got[i] = !p.weight || p.weight[t0 + lane] > 0.0f;
                    if (lane + 32 < n) got[i] += !p.weight || p.weight[t0 + lane + 32] > 0.0f;
                }
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int b = b0 + i * warps, act_b = __reduce_add_sync(0xffffffffu, got[i]);
                    if (lane == 0 && b < p.kv.n_seqs) {
                        halves[b] = (uint16_t)((act_b * mass_heads(p.H) + MS_HALF - 1) / MS_HALF);
                        sched.prefix[b + 1] *= max((int)halves[b], MS_MIN);
                    }
                }
            }
            if (p.kv.n_seqs > 1) __syncthreads(); else __syncwarp();
        });
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_wait();
    tc_fence_after();
    const uint32_t tmem = B.tmem, smb = smem_u32(sm);
    int64_t u = pair < sched.runs ? sched.run_start(pair) : 0;
    const int64_t u_end = pair < sched.runs ? sched.run_start(pair + 1) : 0;
    uint32_t n_tile = 0, n_q = 0, n_d = 0;                    // this role's key tiles, Q chunks and row blocks so far
    bool ok = true;
    const int Hp = mass_heads(p.H), hb = mass_box(p.H);

    for (MassSegment g; mass_next(p, sched, halves, u, u_end, g);) {
        if (warp != 0) asm volatile("bar.sync 2, %0;" :: "n"(MS_THREADS - 32) : "memory");      // act of the last segment is free
        if (warp == 2) {
            int n = 0;
            for (int j0 = 0; j0 < g.n; j0 += 32) {
                const int j = j0 + lane;
                const bool in = j < g.n && (!p.weight || p.weight[g.first + j] > 0.0f);
                const uint32_t m = __ballot_sync(0xffffffffu, in);
                const int at = n + __popc(m & ((1u << lane) - 1));
                if (in) { act[at] = j; see[at] = node_mask(p.tree, g.first + j, j, g.n); }
                n += __popc(m);
            }
            if (lane == 0) B.n_act = n;
        }
        if (warp != 0) asm volatile("bar.sync 2, %0;" :: "n"(MS_THREADS - 32) : "memory");
        const int rows = B.n_act * Hp;                        // not for warp 0, which loads K meanwhile
        int j, h0, h1;

        if (warp == 0) {
            // ---------------------------------------------------------------- K: 128 keys of this CTA, 9 chunks a tile
            if (halves[g.b] && elect_one()) {
                const uint32_t full0 = peer_addr(smem_u32(&B.k_full[0]), 0);
                const int box = min(p.kv.page_size, 64);
                for (; ok && g.next(j, h0, h1); ++n_tile) {
                    int row[8];                               // pool rows of the boxes; those beyond the drafts read the last page again
                    #pragma unroll
                    for (int x = 0; x < 8; ++x)
                        row[x] = (x * 16 & (box - 1)) == 0 ? max(0, kv_slot(p.kv, g.b, min(j * MS_TILE + (int)rank * 128 + x * 16, (g.total - 1) & ~15), p.err)) : 0;
                    for (int c = 0; c < 9; ++c) {
                        if (!(ok = wait_phase(&B.k_empty[c], (n_tile & 1) ^ 1, gave_up, p.err))) break;
                        arrive_expect_at(full0 + 8 * c, MS_CHUNK);
                        #pragma unroll
                        for (int x = 0; x < 8; ++x)
                            if ((x * 16 & (box - 1)) == 0) tma_2d_pair(smb + c * MS_CHUNK + x * 2048, &kv_map, c * 64, row[x], full0 + 8 * c);
                    }
                }
                if (!ok) __nanosleep(1000000);                // given up: the loads in flight land before the CTA ends
            }
        } else if (warp == 1) {
            // ---------------------------------------------------------------- MMAs, issued by CTA 0 for both
            if (rows && rank == 0 && elect_one()) {
                auto wait = [&](uint64_t* bar, uint32_t parity) { return ok = wait_phase(bar, parity, gave_up, p.err); };
                for (; ok && g.next(j, h0, h1); ++n_tile) {
                    const int end = min(h1 * MS_HALF, rows);
                    for (int r = h0 * MS_HALF; ok && r < end; r += MS_ROWS, ++n_d) {
                        const bool first = r == h0 * MS_HALF, last = r + MS_ROWS >= end;
                        const uint32_t buf = n_d & 1, d = tmem + buf * 256;
                        const uint32_t idesc = att_idesc(256, 0, BF, false) | ((uint32_t)(mass_cols(end - r, hb) >> 3) << 17);
                        if (!wait(&B.d_free[buf], ((n_d >> 1) & 1) ^ 1)) break;
                        tc_fence_after();
                        for (int c = 0; c < 9; ++c, ++n_q) {
                            const uint32_t st = n_q % MS_RING;
                            if (first && !wait(&B.k_full[c], n_tile & 1)) break;
                            if (!wait(&B.q_full[st], (n_q / MS_RING) & 1)) break;
                            umma2_x4_n(d, sw128_lo(smb + c * MS_CHUNK, 16), sw128_lo(smb + MS_Q + st * MS_CHUNK, 16), idesc, c != 0);
                            commit2(&B.q_empty[st]);
                            if (last) commit2(&B.k_empty[c]);
                        }
                        if (!ok) break;
                        commit2(&B.d_full[buf]);
                    }
                }
                if (!ok) { commit2(&B.drain); mbar_wait(&B.drain, 0, nullptr, 0); }
            }
        } else if (warp == 2) {
            // ---------------------------------------------------------------- Q: this CTA's half of a block's rows, 64 values a stage
            if (rows && elect_one()) {
                const uint32_t full0 = peer_addr(smem_u32(&B.q_full[0]), 0);
                auto load = [&](auto head_major) {            // the order of the map's dimensions, settled outside the loops
                    while (ok && g.next(j, h0, h1)) {
                        const int end = min(h1 * MS_HALF, rows);
                        for (int r1 = h0 * MS_HALF; ok && r1 < end; r1 += MS_ROWS) {
                            const int half = mass_cols(end - r1, hb) / 2, r0 = r1 + (int)rank * half;
                            const int a0 = r0 / Hp, hd0 = r0 - a0 * Hp;
                            for (int c = 0; c < 9; ++c, ++n_q) {
                                const uint32_t st = n_q % MS_RING, bar = full0 + 8 * st;
                                if (!(ok = wait_phase(&B.q_empty[st], ((n_q / MS_RING) & 1) ^ 1, gave_up, p.err))) break;
                                arrive_expect_at(bar, half * 128);
                                uint32_t to = smb + MS_Q + st * MS_CHUNK;
                                for (int r = 0, a = a0, h = hd0; r < half; r += hb, to += hb * 128) {
                                    // rows beyond the last token's: that token's again (their c is infinite)
                                    const int t = g.first + act[min(a, rows / Hp - 1)];
                                    if (decltype(head_major)::value) tma_3d_pair(to, &q_map, c * 64, t, h, bar);
                                    else tma_3d_pair(to, &q_map, c * 64, h, t, bar);
                                    if ((h += hb) == Hp) { h = 0; ++a; }
                                }
                            }
                        }
                    }
                };
                if (p.q_head_major) load(std::true_type()); else load(std::false_type());
                if (!ok) __nanosleep(1000000);
            }
        } else if (warp >= 4) {
            // ---------------------------------------------------------------- sums: lane = key; the two groups of four warps take
            // every other 32 columns.  A wait that gives up is not acted on: the loops end.
            const int t8 = tid - 128, L = t8 & 127, grp = t8 >> 7;
            const uint32_t lane_base = (uint32_t)(32 * (warp & 3)) << 16;
            const uint32_t d_free0 = peer_addr(smem_u32(&B.d_free[0]), 0);
            const float scale2 = p.scale * 1.4426950408889634f;
            while (g.next(j, h0, h1)) {
                const int end = min(h1 * MS_HALF, rows);
                const int key = j * MS_TILE + (int)rank * 128 + L, node = key - g.len;
                const bool tail = j * MS_TILE + (int)rank * 128 + 127 >= g.len, careful = tail || Hp != p.H;
                uint64_t seen = node < 0 ? ~0ull : 0;         // the tokens that see this key (read where `tail`)
                if (node >= 0 && node < 64)
                    for (int a = 0; a < B.n_act; ++a) seen |= ((see[a] >> node) & 1) << a;
                float acc[4] = { 0, 0, 0, 0 };
                for (int r = h0 * MS_HALF; r < end; r += MS_ROWS, ++n_d) {
                    const uint32_t buf = n_d & 1;
                    {                                         // c of column t8
                        const int gr = r + t8, a = gr / Hp, h = gr - a * Hp;
                        float c = INFINITY;                   // no row: 2^-inf
                        if (gr < rows && h < p.H) {
                            const int t = g.first + act[a];
                            const float lse = p.lse[(int64_t)t * p.H + h];
                            if (lse != -INFINITY) c = lse * 1.4426950408889634f - (p.weight ? log2f(p.weight[t]) : 0.0f);
                        }
                        col[buf * MS_ROWS + t8] = c;
                        tok[buf * MS_ROWS + t8] = (uint8_t)min(a, 63);
                    }
                    group_sync();
                    warp_wait_phase(&B.d_full[buf], (n_d >> 1) & 1, gave_up, p.err);
                    tc_fence_after();
                    const int cols = mass_cols(end - r, hb);
                    for (int c0 = grp * 32; c0 < cols; c0 += 64) {
                        uint32_t s[32];
                        tmem_ld32(tmem + lane_base + buf * 256 + c0, s);
                        tmem_wait_ld();
                        const float4* c4 = (const float4*)(col + buf * MS_ROWS + c0);
                        if (careful) {
                            // a term that does not count is taken out by its exponent and not by its score or its c: a token's lse may
                            // be NaN, and the zeros of padded heads times an infinite key are
                            const uint8_t* tk = tok + buf * MS_ROWS + c0;
                            #pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const bool sees = !tail | ((seen >> tk[i / 2 * 8]) & 1);       // eight columns are heads of one token
                                const float4 v = c4[i];
                                const float c[4] = { v.x, v.y, v.z, v.w };
                                #pragma unroll
                                for (int x = 0; x < 4; ++x) {
                                    const float e = fmaf(__uint_as_float(s[4 * i + x]), scale2, -c[x]);
                                    acc[x] += exp2_approx(sees & (c[x] != INFINITY) ? e : -INFINITY);
                                }
                            }
                            continue;
                        }
                        #pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float4 c = c4[i];
                            acc[0] += exp2_approx(fmaf(__uint_as_float(s[4 * i]), scale2, -c.x));
                            acc[1] += exp2_approx(fmaf(__uint_as_float(s[4 * i + 1]), scale2, -c.y));
                            acc[2] += exp2_approx(fmaf(__uint_as_float(s[4 * i + 2]), scale2, -c.z));
                            acc[3] += exp2_approx(fmaf(__uint_as_float(s[4 * i + 3]), scale2, -c.w));
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_at(d_free0 + 8 * buf);
                }
                float a = (acc[0] + acc[1]) + (acc[2] + acc[3]);
                if (grp) part[L] = a;
                group_sync();
                a += part[L];
                if (h1 - h0 < g.work) {                       // others have rows of this tile too
                    const int64_t lo = g.unit - g.work, hi = g.unit - 1;      // its first and last unit of work
                    const int q0 = sched.owner(lo), q1 = sched.owner(hi);
                    float* mine = wk.part + (int)rank * 128 + L;
                    if (!grp) __stcg(mine + (int64_t)(pair == q0 ? 2 * pair + 1 : 2 * pair) * MS_TILE, a);
                    group_sync();
                    if (t8 == 0) {                            // back to 0 with the last
                        uint32_t before;
                        asm volatile("atom.acq_rel.gpu.global.inc.u32 %0, [%1], %2;"
                                     : "=r"(before) : "l"(wk.arrived + 2 * q0 + rank), "r"(q1 - q0) : "memory");
                        B.last = before == (uint32_t)(q1 - q0);
                    }
                    group_sync();
                    if (B.last && !grp) {
                        a = 0;
                        for (int q = q0; q <= q1; ++q) a += __ldcg(mine + (int64_t)(q == q0 ? 2 * q + 1 : 2 * q) * MS_TILE);
                    }
                }
                if (!grp && key < g.total && (h1 - h0 == g.work || B.last)) {
                    const int slot = kv_slot(p.kv, g.b, key, p.err);
                    if (slot >= 0) p.kv.mass[slot] = p.decay * p.kv.mass[slot] + a;
                }
                group_sync();                                 // part is free again
            }
        }
        __syncwarp();                                         // the single-thread roles' warps
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    if (warp == 3) { tc_fence_after(); tmem_dealloc2(tmem, 512); }
}

template <class T>
static cudaError_t mass_go(const TreeParams& p, const CUtensorMap& map, const CUtensorMap& q_map, const MassWork& wk, int pairs, cudaStream_t st) {
    return launch_pdl_n(k_mass<T>, dim3(2 * pairs), dim3(MS_THREADS), MS_SMEM, st, p, map, q_map, wk);
}

cudaError_t mass_setup() {
    const cudaError_t e = cudaFuncSetAttribute(k_mass<__half>, cudaFuncAttributeMaxDynamicSharedMemorySize, MS_SMEM);
    return e != cudaSuccess ? e : cudaFuncSetAttribute(k_mass<__nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize, MS_SMEM);
}
int mass_q_box(int H) { return mass_box(H); }

cudaError_t launch_mass(const TreeParams& p, int dtype, const CUtensorMap& map, const CUtensorMap& q_map, const MassWork& wk, int pairs, cudaStream_t st) {
    return dtype == LK_DT_F16 ? mass_go<__half>(p, map, q_map, wk, pairs, st) : mass_go<__nv_bfloat16>(p, map, q_map, wk, pairs, st);
}

}  // namespace lk
