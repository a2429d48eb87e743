// attn_tree.cu -- attention of drafted token trees over the paged latent cache.
//
// S = scale * Q K^T with K the 576-wide rows, P = softmax(S) over the rows that a token sees, O = P C with C the first
// 512 values of the same rows.  One pass over the cache with a running reference m and sum l per row: P = 2^(S' - m + 7)
// (S' in units of log 2), and where a tile's maximum exceeds m by more than 8, m moves there and O and l are scaled.
//
// Work.  A row is one (token, head); 128 rows of one sequence are an item, 128 cached rows a tile, and (item, tile) a
// unit of work: 35.7 M products, 147 KB of cache.  All units, numbered item by item, are cut into equal runs, one per
// pair of CTAs, whatever the batch's lengths; an item that lies in several runs leaves partial O, m and l for k_merge.
// Lengths are read on the device, so a captured call follows them.
//
// Why a pair.  fp32 O is 128 x 512: all of one SM's tensor memory.  A pair halves the rows (2-CTA tcgen05.mma, M = 128:
// 64 rows of each CTA in all 128 lanes), so O takes 256 columns and two S buffers 128, and Q 72 KB of shared memory.  Each
// CTA loads half of a tile's rows for S (64 x 576) and half of the latent columns of all of them for O (128 x 256).
// Measured on a B200, 2-CTA M = 128 runs at the full 4096 products per cycle and SM for N = 128 and 256 (one CTA with
// M = 128, N = 128 reaches 2925), so a unit costs 2176 cycles of tensor pipe.  A unit takes about 3000: the thread that issues S
// waits at five stages of K a tile.  L2 is not what bounds it (136 KB a CTA; leaving V's loads out gains under 5 %).
// Times a call: 64 nodes over 65 000 rows 1050 us in a long run (1.10 PFLOP/s at the 1.49 GHz that 1 kW allows; 915 to 920 in the first
// ten calls after a rest), 8 nodes over 16 384 rows 49.7, one token over 30 011 rows 27.6 (of them 8 the tiles and 10 the parts and
// their merge; the same whether the cache lies in L2 or not), 16 sequences of 3 to 17 nodes on 32 heads 95, one tile 12 (14 where the
// pages could hold more and the merge is launched); the plain forms: 25 000, 1470, 837, 6250, 699.
//
// P is rounded to the cache's type before its product, because an MMA takes 16-bit operands of one type (in tf32 it would run at half
// the rate or less, on a copy of C in 32 bits).  The rounding is relative, 2^-9 (bf16) or 2^-12 (fp16) of each weight at most, and the sum l
// takes the weights unrounded: against 64 bits out is off by 1.7 to 2.0e-3 in bf16, where the rounding of out alone gives 1.66e-3, and
// by 2.2 to 2.6e-4 in fp16 (2.07e-4); lse by 1 to 4e-7.
//
// Roles (384 threads a CTA): warp 0 loads (TMA, ring of 8 x 16 KB), warps 1 and 2 of CTA 0 issue the MMAs of S and of O,
// warp 3 repairs tail tiles, warps 4-11 do softmax, O's scaling and the output (two threads per tensor-memory lane, four per
// row: with one per lane V waits twice as long in the ring for P).  Order of the ring: K(0), K(1), V(0),
// K(2), V(1), ..: softmax j runs under S(j + 1).  Two issuing threads because a satisfied barrier wait between two MMAs
// leaves the tensor pipe empty for ~50 cycles, 11 times a unit: while one thread waits the other's MMAs run.  A stage has one
// "full" barrier for K and one for V: a parity wait is only right for a barrier's next phase, and with a shared one the thread
// of O, which can reach a stage while the K before it is still on its way (V is in L2 by then), would take that phase for its own.
//
// Rows that must not matter: a tile's rows beyond the drafts, and drafted rows that a token does not see, get P = 0; but
// 0 * NaN is NaN, so the former are loaded as zeros from outside the pool (the last 16 rows' rest is zeroed by warp 3), and warp 3
// zeroes every drafted row of the O operand that holds a non-finite value (a token that does see it gets its NaN through S and P; where
// its score is -infinity, the row has no weight).
#include <type_traits>
#include "attn_tc.cuh"
#include "attn_sched.cuh"
#include "moe_internal.h"

namespace lk {

constexpr int TR_THREADS = 384, TR_STAGES = 8, TR_STAGE = 16384, TR_CHUNK = 8192;
constexpr int TR_Q = 0, TR_P = 9 * TR_CHUNK, TR_RING = TR_P + TR_STAGE, TR_BARS = TR_RING + TR_STAGES * TR_STAGE;
constexpr int TR_XCH = TR_BARS + 44 * 8, TR_SCHED = TR_XCH + 256 * 4;
constexpr int TR_SMEM = TR_SCHED + (int)sizeof(Sched);
static_assert(TR_SMEM <= 232448, "227 KB a CTA");
constexpr int TR_LEAD = 3;                            // a further item of a run costs about as much as three tiles (4 us)
constexpr uint32_t TR_S_COL = 256, TR_TMEM = 512;
constexpr float TR_SHIFT = 7.0f, TR_JUMP = 8.0f;      // P <= 2^15 fits fp16; its smallest normal is 2^-21 of the reference

struct TreeBars {
    uint64_t k_full[TR_STAGES], v_full[TR_STAGES], land[TR_STAGES], empty[TR_STAGES];
    uint64_t s_full[2], s_free[2], p_full, o_done, q_full, drain[2];
    uint32_t tmem;
    int gave_up;
};
static_assert(sizeof(TreeBars) <= 44 * 8, "barrier block");

// whether rows i0 .. i0 + 63 hold drafted ones: warp 3 looks them over before the MMAs do
__device__ __forceinline__ bool tail_rows(const Segment& g, int i0) { return i0 + 64 > g.len && i0 < g.total; }

// the load role of one CTA, one thread: boxes of BOX rows x 64 values.  Its instructions are the loop's length (a loaded
// stage feeds 512 cycles of MMAs), so the page lookups are made a tile ahead and nothing is computed per box.
template <int BOX>
__device__ __forceinline__ bool tree_load(const TreeParams& p, const Sched& sched, int64_t u, int64_t u_end, const CUtensorMap* map,
                                          const CUtensorMap* map16, TreeBars& B, uint32_t smb, uint32_t rank) {
    constexpr int NB = 64 / BOX;                          // boxes of 64 rows
    constexpr uint32_t V = sizeof(B.k_full);              // from a stage's k_full to its v_full
    const uint32_t full0 = peer_addr(smem_u32(&B.k_full[0]), 0);
    uint32_t st = 0, ph = 1, dst = smb + TR_RING, bar = full0;
    auto advance = [&]() {
        dst += TR_STAGE; bar += 8;
        if (++st == TR_STAGES) { st = 0; ph ^= 1; dst = smb + TR_RING; bar = full0; }
    };
    for (Segment g; sched_next<ATT_TILE, TR_LEAD>(p, sched, u, u_end, g);) {
        int next[2 * NB], k[2 * NB], v[2 * NB];           // pool rows of the boxes of tiles j + 1, j and j - 1
        // boxes beyond the drafts read the last 16 rows' page again
        auto rows_of = [&](int j) {
            #pragma unroll
            for (int x = 0; x < 2 * NB; ++x) next[x] = max(0, kv_slot(p.kv, g.b, min(j * ATT_TILE + x * BOX, (g.total - 1) & ~15), p.err));
        };
        rows_of(g.t0);
        for (int j = g.t0; j <= g.t1; ++j) {              // K of tile j, then V of tile j - 1
            #pragma unroll
            for (int x = 0; x < 2 * NB; ++x) { v[x] = k[x]; k[x] = next[x]; }
            if (j + 1 < g.t1) rows_of(j + 1);
            if (j < g.t1) {
                int mine[NB];
                #pragma unroll
                for (int x = 0; x < NB; ++x) mine[x] = rank ? k[NB + x] : k[x];
                #pragma unroll
                for (int s = 0; s < 5; ++s) {
                    if (!wait_phase(&B.empty[st], ph, &B.gave_up, p.err)) return false;
                    arrive_expect_at(bar, (s < 4 ? 2 : 1) * TR_CHUNK);
                    #pragma unroll
                    for (int c = 0; c < (s < 4 ? 2 : 1); ++c)
                        #pragma unroll
                        for (int x = 0; x < NB; ++x) tma_2d_pair(dst + c * TR_CHUNK + x * BOX * 128, map, (2 * s + c) * 64, mine[x], bar);
                    advance();
                }
            }
            if (j > g.t0) {
                #pragma unroll
                for (int s = 0; s < 4; ++s) {             // column group s / 2, row half s % 2
                    if (!wait_phase(&B.empty[st], ph, &B.gave_up, p.err)) return false;
                    const int i0 = (j - 1) * ATT_TILE + (s & 1) * 64, col = (s >> 1) * 256 + (int)rank * 128;
                    uint32_t to = bar + V;
                    if (tail_rows(g, i0)) { to = smem_u32(&B.land[st]); mbar_arrive_expect_tx(&B.land[st], TR_STAGE); }
                    else arrive_expect_at(to, TR_STAGE);
                    if (i0 + 64 <= g.len) {
                        #pragma unroll
                        for (int c = 0; c < 2; ++c)
                            #pragma unroll
                            for (int x = 0; x < NB; ++x) tma_2d_pair(dst + c * TR_CHUNK + x * BOX * 128, map, col + c * 64, v[(s & 1) * NB + x], to);
                    } else                                // 16 rows at a time; beyond the drafts from outside the pool: zeros
                        for (int x = 0; x < 4; ++x) {
                            int row = p.kv.n_pages << p.kv.page_shift;
                            #pragma unroll
                            for (int y = 0; y < NB; ++y) if (x * 16 / BOX == y && i0 + x * 16 < g.total) row = v[(s & 1) * NB + y] + x * 16 % BOX;
                            for (int c = 0; c < 2; ++c) tma_2d_pair(dst + c * TR_CHUNK + x * 2048, map16, col + c * 64, row, to);
                        }
                    advance();
                }
            }
        }
    }
    return true;
}

template <class T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(TR_THREADS, 1)
k_tree(const __grid_constant__ TreeParams p, const __grid_constant__ CUtensorMap kv_map, const __grid_constant__ CUtensorMap kv_map16,
       const __grid_constant__ CUtensorMap q_map, TreeWork wk) {
    extern __shared__ __align__(1024) uint8_t sm[];
    TreeBars& B = *(TreeBars*)(sm + TR_BARS);
    float* xch = (float*)(sm + TR_XCH);
    Sched& sched = *(Sched*)(sm + TR_SCHED);
    volatile int* gave_up = &B.gave_up;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = cluster_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;

    if (warp == 2 && lane == 0) {
        B.gave_up = 0;
        for (int s = 0; s < TR_STAGES; ++s) { mbar_init(&B.k_full[s], 2); mbar_init(&B.v_full[s], 2); mbar_init(&B.land[s], 1); mbar_init(&B.empty[s], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&B.s_full[i], 1); mbar_init(&B.s_free[i], 16); mbar_init(&B.drain[i], 1); }
        mbar_init(&B.p_full, 16); mbar_init(&B.o_done, 1); mbar_init(&B.q_full, p.q_flat ? 2 : 16);
        fence_mbar_init();
        asm volatile("prefetch.tensormap [%0];" :: "l"(&kv_map) : "memory");
        asm volatile("prefetch.tensormap [%0];" :: "l"(&q_map) : "memory");
    }
    cluster_arrive();                                     // the barriers are there; the wait comes with a role's first use of the other CTA
    if (warp == 3) tmem_alloc2(&B.tmem, TR_TMEM);
    pdl_wait();
    pdl_trigger();
    if (warp == 0 || p.kv.n_seqs > 1) sched_load<ATT_TILE>(p, sched, tid, TR_THREADS, pairs,
        [&](int n, int tiles) { return (int64_t)((n * p.H + ATT_ITEM - 1) / ATT_ITEM) * (TR_LEAD + tiles); }, []() {});
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (rank == 0 && tid == 128) wk.split[2 * pair].info = wk.split[2 * pair + 1].info = 0;
    int64_t u = pair < sched.runs ? sched.run_start(pair) : 0;
    const int64_t u_end = pair < sched.runs ? sched.run_start(pair + 1) : 0;
    const uint32_t smb = smem_u32(sm);

    if (warp < 4) cluster_wait();                         // the softmax warps may start Q first
    tc_fence_after();
    const uint32_t tmem = B.tmem;
    if (warp == 0) {
        // ---------------------------------------------------------------- loads
        if (elect_one()) {
            const bool ok = p.kv.page_size >= 64 ? tree_load<64>(p, sched, u, u_end, &kv_map, &kv_map16, B, smb, rank)
                          : p.kv.page_size == 32 ? tree_load<32>(p, sched, u, u_end, &kv_map, &kv_map16, B, smb, rank)
                                                 : tree_load<16>(p, sched, u, u_end, &kv_map, &kv_map16, B, smb, rank);
            if (!ok) __nanosleep(1000000);                // given up: the loads in flight land before the CTA ends
        }
    } else if (warp < 3) {
        // ---------------------------------------------------------------- MMAs, issued by CTA 0 for both: S and O by a thread each
        if (rank == 0 && elect_one()) {
            constexpr uint32_t id_s = att_idesc(128, 128, BF, false), id_o = att_idesc(128, 256, BF, true);
            uint32_t st = 0, uses = 0, n = 0, n_q = 0;    // ring place; parity of this thread's uses of each stage; tiles, segments
            bool ok = true;
            auto wait = [&](uint64_t* bar, uint32_t parity) { return ok = wait_phase(bar, parity, gave_up, p.err); };
            auto advance = [&](uint32_t k) { st = (st + k) % TR_STAGES; };
            auto wait_stage = [&](uint64_t* full) { const bool got = wait(&full[st], (uses >> st) & 1); uses ^= 1u << st; return got; };
            if (warp == 1) {
                for (Segment g; ok && sched_next<ATT_TILE, TR_LEAD>(p, sched, u, u_end, g);) {
                    if (!wait(&B.q_full, n_q++ & 1)) break;
                    for (int j = g.t0; ok && j < g.t1; ++j, ++n) {
                        const uint32_t buf = n & 1, d = tmem + TR_S_COL + buf * 64;
                        if (!wait(&B.s_free[buf], ((n >> 1) & 1) ^ 1)) break;
                        tc_fence_after();
                        for (int s = 0; s < 5; ++s) {
                            if (!wait_stage(B.k_full)) break;
                            const uint32_t kb = smb + TR_RING + st * TR_STAGE, qb = smb + TR_Q + 2 * s * TR_CHUNK;
                            umma2_x4<id_s, 32, 32>(d, sw128_lo(qb, 16), sw128_lo(kb, 16), s != 0);
                            if (s < 4) umma2_x4<id_s, 32, 32>(d, sw128_lo(qb + TR_CHUNK, 16), sw128_lo(kb + TR_CHUNK, 16), 1);
                            commit2(&B.empty[st]);
                            advance(1);
                        }
                        if (!ok) break;
                        commit2(&B.s_full[buf]);
                        if (j > g.t0) advance(4);         // V of tile j - 1
                    }
                    advance(4);                           // V of the last tile
                }
            } else {
                for (Segment g; ok && sched_next<ATT_TILE, TR_LEAD>(p, sched, u, u_end, g);) {
                    advance(5);                           // K of the first tile
                    for (int j = g.t0; ok && j < g.t1; ++j, ++n) {
                        if (j + 1 < g.t1) advance(5);     // K of tile j + 1
                        if (!wait(&B.p_full, n & 1)) break;
                        tc_fence_after();
                        for (int s = 0; s < 4; ++s) {
                            if (!wait_stage(B.v_full)) break;
                            const uint32_t vb = smb + TR_RING + st * TR_STAGE, pb = smb + TR_P + (s & 1) * TR_CHUNK;
                            umma2_x4<id_o, 32, 2048>(tmem + (s >> 1) * 128, sw128_lo(pb, 16), sw128_lo(vb, TR_CHUNK), j > g.t0 || (s & 1));
                            commit2(&B.empty[st]);
                            advance(1);
                        }
                        if (!ok) break;
                        commit2(&B.o_done);
                    }
                }
            }
            if (!ok) {                                    // given up: this thread's MMAs complete before the CTA ends
                uint64_t* drain = &B.drain[warp - 1];
                commit2(drain);
                mbar_wait(drain, 0, nullptr, 0);
            }
        }
    } else if (warp < 4) {
        // ---------------------------------------------------------------- repair of the O operand's tail tiles
        const uint32_t full0 = peer_addr(smem_u32(&B.v_full[0]), 0);
        uint32_t st = 0, uses = 0;                        // bit s: parity of the uses of land[s]
        auto advance = [&](int n) { st = (st + n) % TR_STAGES; };
        for (Segment g; sched_next<ATT_TILE, TR_LEAD>(p, sched, u, u_end, g);) {
            for (int j = g.t0; j <= g.t1; ++j) {
                if (j < g.t1) advance(5);
                if (j == g.t0) continue;
                for (int s = 0; s < 4; ++s, advance(1)) {
                    const int i0 = (j - 1) * ATT_TILE + (s & 1) * 64;
                    if (!tail_rows(g, i0)) continue;
                    warp_wait_phase(&B.land[st], (uses >> st) & 1, gave_up, p.err);
                    uses ^= 1u << st;
                    // rows (s % 2) * 64 .. + 63 of the tile, 2 x 128 bytes each: eight lanes a row.  Each row's part is judged by
                    // itself: all that matters is that nothing non-finite is multiplied by 0
                    for (int r = max(0, g.len - i0) & ~3; r < min(64, (g.total - i0 + 15) & ~15); r += 4) {
                        const int i = i0 + r + (lane >> 3);
                        uint4* v = (uint4*)(sm + TR_RING + st * TR_STAGE + (r + (lane >> 3)) * 128) + (lane & 7);
                        bool bad = i >= g.total;
                        if (i0 + r < g.total) {           // a 16-bit value whose exponent bits are all ones
                            const uint4 a = v[0], c = v[TR_CHUNK / 16];
                            const uint32_t hit = nonfinite2<T>(a.x) | nonfinite2<T>(a.y) | nonfinite2<T>(a.z) | nonfinite2<T>(a.w) |
                                                 nonfinite2<T>(c.x) | nonfinite2<T>(c.y) | nonfinite2<T>(c.z) | nonfinite2<T>(c.w);
                            const uint32_t rows = __ballot_sync(0xffffffffu, hit);
                            bad |= i >= g.len && ((rows >> (lane & 24)) & 0xff);
                        }
                        if (bad) v[0] = v[TR_CHUNK / 16] = make_uint4(0, 0, 0, 0);
                    }
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) arrive_at(full0 + 8 * st);
                }
            }
        }
    } else {
        // ---------------------------------------------------------------- softmax, O's scaling, output
        // Thread (lane L, column half ch): row L % 64, keys 64 (L / 64) + 32 ch .. + 31 of a tile, O columns 128 ch .. + 127 of
        // the lane.  A wait that gives up is not acted on here: every later one then returns at once, and the loops end.
        const int L = (tid - 128) & 127, ch = (tid - 128) >> 7, row = L & 63, half = L >> 6, part = 2 * half + ch;
        const uint32_t lane_base = (uint32_t)(32 * (warp & 3)) << 16, o_base = tmem + lane_base + ch * 128;
        const uint32_t s_free0 = peer_addr(smem_u32(&B.s_free[0]), 0), p_full0 = peer_addr(smem_u32(&B.p_full), 0),
                       q_full0 = peer_addr(smem_u32(&B.q_full), 0);
        const float scale2 = p.scale * 1.4426950408889634f;
        uint32_t n = 0;                                   // tiles so far
        auto wait = [&](uint64_t* bar, uint32_t parity) { warp_wait_phase(bar, parity, gave_up, p.err); tc_fence_after(); };
        // Q of a segment: this CTA's 64 rows of the item, 9 swizzled chunks of 64 values.  Rows in equal steps through q, whatever
        // the heads, are nine boxes (rows beyond the sequence's are another's or zeros, and are not used); where a token's step is
        // not its heads', 8 rows a warp by 16-byte copies, their places in q from the lanes that own the rows (4000 cycles).
        auto box_q = [&](const Segment& g) {
            if (warp == 4 && elect_one()) {
                arrive_expect_at(q_full0, 9 * TR_CHUNK);
                #pragma unroll
                for (int c = 0; c < 9; ++c) tma_2d_pair(smb + TR_Q + c * TR_CHUNK, &q_map, c * 64, g.first * p.H + g.rt * ATT_ITEM + (int)rank * 64, q_full0);
            }
            __syncwarp();
        };
        auto start_q = [&](const Segment& g) {
            const int gr = g.rt * ATT_ITEM + (int)rank * 64 + row, tj = gr / p.H;
            const int64_t q_at = gr < g.n * p.H ? (g.first + tj) * p.q_token + (gr - tj * p.H) * p.q_head : -1;
            const int w0 = ((warp - 4) >> 1) * 8;
            #pragma unroll 2
            for (int i = 0; i < 8; ++i) {
                const int64_t at = __shfl_sync(0xffffffffu, q_at, w0 + i);
                const int r = (warp & 1) * 32 + w0 + i;
                const T* src = (const T*)p.q + max(at, (int64_t)0);
                #pragma unroll
                for (int c = lane; c < 72; c += 32)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                                 :: "r"(smb + TR_Q + (c >> 3) * TR_CHUNK + r * 128 + (((c & 7) ^ (r & 7)) << 4)), "l"(src + c * 8), "r"(at < 0 ? 0 : 16) : "memory");
            }
        };
        auto finish_q = [&]() {
            asm volatile("cp.async.wait_all;" ::: "memory");
            fence_async_smem();
            __syncwarp();
            if (lane == 0) arrive_at(q_full0);
        };
        Segment g, next;
        bool more = sched_next<ATT_TILE, TR_LEAD>(p, sched, u, u_end, g);
        if (more && !p.q_flat) start_q(g);
        cluster_wait();
        if (more) { if (p.q_flat) box_q(g); else finish_q(); }
        while (more) {
            const int gr = g.rt * ATT_ITEM + (int)rank * 64 + row, tj = gr / p.H, h = gr - tj * p.H, t = g.first + tj;
            const bool live = gr < g.n * p.H;
            const uint64_t mask = live ? node_mask(p.tree, t, tj, g.n) : 0;
            float m = -INFINITY, l = 0.0f;
            for (int j = g.t0; j < g.t1; ++j, ++n) {
                const uint32_t buf = n & 1;
                wait(&B.s_full[buf], (n >> 1) & 1);
                float s[32];
                {
                    uint32_t a[32];
                    tmem_ld32(tmem + lane_base + TR_S_COL + buf * 64 + ch * 32, a);
                    tmem_wait_ld();
                    #pragma unroll
                    for (int i = 0; i < 32; ++i) s[i] = __uint_as_float(a[i]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_at(s_free0 + 8 * buf);
                const int base = j * ATT_TILE + half * 64 + ch * 32 - g.len;        // drafted node of the first column
                if (base > -32) {
                    const uint32_t see = base >= 64 ? 0 : base >= 0 ? (uint32_t)(mask >> base) : (uint32_t)(mask << -base) | ((1u << -base) - 1);
                    #pragma unroll
                    for (int i = 0; i < 32; ++i) if (!((see >> i) & 1)) s[i] = -INFINITY;
                }
                float mx[4] = { s[0], s[1], s[2], s[3] };
                #pragma unroll
                for (int i = 4; i < 32; ++i) mx[i & 3] = fmaxf(mx[i & 3], s[i]);
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale2;
                if (group_or(top > m + TR_JUMP)) {
                    xch[part * 64 + row] = top;
                    group_sync();
                    const float m1 = fmaxf(fmaxf(m, fmaxf(xch[row], xch[64 + row])), fmaxf(xch[128 + row], xch[192 + row]));
                    const float f = m1 == m ? 1.0f : exp2_approx(m - m1);  // m = -inf: 0
                    l *= f;
                    m = m1;
                    if (j > g.t0) {                       // O(j - 1) is complete: scale its columns
                        wait(&B.o_done, (n - 1) & 1);
                        for (int c = 0; c < 128; c += 32) {
                            uint32_t o[32];
                            tmem_ld32(o_base + c, o);
                            tmem_wait_ld();
                            #pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            tmem_st32(o_base + c, o);
                        }
                        tmem_wait_st();
                        tc_fence_before();
                    }
                    group_sync();               // xch is free again
                }
                const float ref = (m == -INFINITY ? 0.0f : m) - TR_SHIFT;
                uint32_t e2[16];
                float sum[4] = { 0, 0, 0, 0 };
                #pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const float e0 = exp2_approx(fmaf(s[i], scale2, -ref)), e1 = exp2_approx(fmaf(s[i + 1], scale2, -ref));
                    sum[i & 2] += e0;
                    sum[(i & 2) + 1] += e1;
                    e2[i / 2] = pack2<T>(e0, e1);
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                if (j > g.t0) wait(&B.o_done, (n - 1) & 1);        // O(j - 1) has read P
                uint8_t* pr = sm + TR_P + half * TR_CHUNK + row * 128;
                #pragma unroll
                for (int c = 0; c < 4; ++c)
                    *(uint4*)(pr + (((4 * ch + c) ^ (row & 7)) << 4)) = make_uint4(e2[4 * c], e2[4 * c + 1], e2[4 * c + 2], e2[4 * c + 3]);
                fence_async_smem();
                __syncwarp();
                if (lane == 0) arrive_at(p_full0);
            }
            // ---- output: all of O, then the row's four sums; the next segment's Q and first S under them (this one's S are done)
            more = sched_next<ATT_TILE, TR_LEAD>(p, sched, u, u_end, next);
            if (more) { if (p.q_flat) box_q(next); else start_q(next); }
            wait(&B.o_done, (n - 1) & 1);
            if (more && !p.q_flat) finish_q();
            xch[part * 64 + row] = l;
            group_sync();
            l = (xch[row] + xch[64 + row]) + (xch[128 + row] + xch[192 + row]);
            group_sync();
            const float ref = (m == -INFINITY ? 0.0f : m) - TR_SHIFT;
            if (g.whole()) {
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                T* out = (T*)p.out + (int64_t)t * p.out_token + (int64_t)h * p.out_head + ch * 256 + half * 128;
                for (int c = 0; c < 128; c += 32) {
                    uint32_t o[32];
                    tmem_ld32(o_base + c, o);
                    tmem_wait_ld();
                    if (live)
                        #pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            uint4 v;
                            v.x = pack2<T>(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv);
                            v.y = pack2<T>(__uint_as_float(o[i + 2]) * inv, __uint_as_float(o[i + 3]) * inv);
                            v.z = pack2<T>(__uint_as_float(o[i + 4]) * inv, __uint_as_float(o[i + 5]) * inv);
                            v.w = pack2<T>(__uint_as_float(o[i + 6]) * inv, __uint_as_float(o[i + 7]) * inv);
                            *(uint4*)(out + c + i) = v;
                        }
                }
                if (live && part == 0 && p.lse) p.lse[(int64_t)t * p.H + h] = l == 0.0f ? -INFINITY : (ref + log2f(l)) * 0.6931471805599453f;
            } else {
                // a part: 8-row groups of 128-byte lines
                const int slot = 2 * pair + (g.item > sched.run_start(pair)), pr = (int)rank * 64 + row;
                float4* to = wk.part + (int64_t)slot * (128 * 128) + (pr >> 3) * 1024 + (ch * 64 + half * 32) * 8 + (pr & 7);
                for (int c = 0; c < 128; c += 32) {
                    uint32_t o[32];
                    tmem_ld32(o_base + c, o);
                    tmem_wait_ld();
                    if (live)
                        #pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            to[(c + i) * 2] = make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]), __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
                }
                if (live && part == 0) wk.ml[slot * 128 + pr] = make_float2(m, l);
                if (rank == 0 && tid == 128) {
                    const int64_t first = g.item + TR_LEAD;       // the units of the item's tiles; those of its start leave no part
                    const int q0 = sched.owner(first), n_parts = sched.owner(first + g.tiles - 1) - q0 + 1;
                    wk.split[slot] = TreeSplit{ n_parts | (pair - q0) << 8 | min(ATT_ITEM, g.n * p.H - g.rt * ATT_ITEM) << 16,
                                                2 * q0 + (g.item > sched.run_start(q0)), g.rt * ATT_ITEM, g.first };
                }
            }
            tc_fence_before();
            g = next;
        }
    }
    __syncwarp();                                         // the single-thread roles' warps
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    if (warp == 3) { tc_fence_after(); tmem_dealloc2(tmem, TR_TMEM); }
}

// ---------------------------------------------------------------- joining split items
// out = sum_q f_q O_q / sum_q f_q l_q with f_q = 2^(m_q - max m) over an item's parts q, added in a fixed order.  The runs that
// worked on an item share its rows out: MG_BLOCKS blocks for each of them, which read that run's record alone (one list that all
// blocks searched took 3 us more, most of it waiting for the same few lines).  A task is 8 rows (a part's 128-byte lines) x 128
// latent values, or x 32 for items of 24 parts and more (a decoded token's), where 4 groups of 64 threads then take every fourth
// part.  A task's first 8 parts a thread are on their way before its factors are known, since its time is that of the loads one
// after another.  Items of 60 parts: 29.4 us a call so, 32.7 with 8 groups and all parts at once; 4 blocks a run 1 us more.
constexpr int MG_ROWS = 8, MG_THREADS = 256, MG_PARTS = 128, MG_DEEP = 8, MG_BLOCKS = 8, MG_MANY = 24;

__device__ __forceinline__ float4 load_cg(const float4* p) {      // volatile: not moved behind a test of its weight
    float4 v;
    asm volatile("ld.global.cg.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p) : "memory");
    return v;
}

template <class T>
__global__ void __launch_bounds__(MG_THREADS) k_merge(const __grid_constant__ TreeParams p, TreeWork wk, int pairs) {
    __shared__ float4 acc[MG_THREADS];
    __shared__ float f[MG_PARTS][MG_ROWS];
    __shared__ float ref[MG_ROWS], sum[MG_ROWS];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int own = blockIdx.x / MG_BLOCKS, sub = blockIdx.x % MG_BLOCKS;
    pdl_wait();
    pdl_trigger();
    const int4 s = __ldcg((const int4*)wk.split + own);
    const int n = s.x & 0xff, rank = s.x >> 8 & 0xff, rows = s.x >> 16;
    if (!n) return;
    const int lg = n < MG_MANY ? 0 : 2, G = 1 << lg;
    const int e = tid & (MG_THREADS / G - 1), grp = tid >> (8 - lg), r = e % MG_ROWS;
    auto slot = [&](int i) { return i ? (s.y & ~1) + 2 * i : s.y; };
    for (int at = rank * MG_BLOCKS + sub; at < (rows + MG_ROWS - 1) / MG_ROWS << (2 + lg); at += n * MG_BLOCKS) {
        const int pr0 = (at >> (2 + lg)) * MG_ROWS, nr = min(MG_ROWS, rows - pr0);
        const int c4 = ((at & ((4 << lg) - 1)) << (5 - lg)) + e / MG_ROWS;
        const float4* src = wk.part + pr0 / MG_ROWS * 1024 + c4 * 8 + r;
        float4 v[MG_DEEP];
        auto fetch = [&](int i0) {
            #pragma unroll
            for (int k = 0; k < MG_DEEP; ++k) if (i0 + k * G < n) v[k] = load_cg(src + (int64_t)slot(i0 + k * G) * (128 * 128));
        };
        fetch(grp);
        if (warp < nr) {                                          // the factors of one row
            float2 ml[MG_PARTS / 32];
            float m = -INFINITY, l = 0.0f;
            #pragma unroll
            for (int k = 0; k < MG_PARTS / 32; ++k)
                if (32 * k < n) {
                    const int i = 32 * k + lane;
                    ml[k] = i < n ? __ldcg(&wk.ml[slot(i) * 128 + pr0 + warp]) : make_float2(-INFINITY, 0.0f);
                }
            #pragma unroll
            for (int k = 0; k < MG_PARTS / 32; ++k) if (32 * k < n) m = fmaxf(m, ml[k].x);
            #pragma unroll
            for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            const float rf = m == -INFINITY ? 0.0f : m;
            #pragma unroll
            for (int k = 0; k < MG_PARTS / 32; ++k)
                if (32 * k < n) {
                    // a part that saw nothing has sum 0; one that saw a NaN score has a NaN sum, which must reach the row however
                    // small the part's maximum is against the others' (or with none, where all its scores are NaN)
                    const float w = ml[k].y == 0.0f ? 0.0f : ml[k].y != ml[k].y ? ml[k].y : exp2_approx(ml[k].x - rf);
                    if (32 * k + lane < n) f[32 * k + lane][warp] = w;
                    l += w == 0.0f ? 0.0f : w * ml[k].y;
                }
            #pragma unroll
            for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
            if (lane == 0) { ref[warp] = rf; sum[warp] = l; }
        }
        __syncthreads();
        float4 a = make_float4(0, 0, 0, 0);
        for (int i0 = grp; i0 < n; i0 += MG_DEEP * G) {
            if (i0 != grp) fetch(i0);
            #pragma unroll
            for (int k = 0; k < MG_DEEP; ++k)
                if (i0 + k * G < n && r < nr) {
                    const float w = f[i0 + k * G][r];
                    if (w != 0.0f) { a.x += w * v[k].x; a.y += w * v[k].y; a.z += w * v[k].z; a.w += w * v[k].w; }
                }
        }
        if (G > 1) {
            acc[tid] = a;
            __syncthreads();
            if (grp == 0)
                for (int k = 1; k < G; ++k) {
                    const float4 w = acc[k * (MG_THREADS / G) + e];
                    a.x += w.x; a.y += w.y; a.z += w.z; a.w += w.w;
                }
        }
        if (grp == 0 && r < nr) {
            const int gr = s.z + pr0 + r, tj = gr / p.H, h = gr - tj * p.H, t = s.w + tj;
            const float l = sum[r], inv = l == 0.0f ? 0.0f : 1.0f / l;
            *(uint2*)((T*)p.out + (int64_t)t * p.out_token + (int64_t)h * p.out_head + 4 * c4) =
                make_uint2(pack2<T>(a.x * inv, a.y * inv), pack2<T>(a.z * inv, a.w * inv));
            if (c4 == 0 && p.lse) p.lse[(int64_t)t * p.H + h] = l == 0.0f ? -INFINITY : (ref[r] - TR_SHIFT + log2f(l)) * 0.6931471805599453f;
        }
        __syncthreads();
    }
}

int tree_pairs(int nsm) { return nsm / 2 < MG_PARTS ? nsm / 2 : MG_PARTS; }

cudaError_t tree_setup() {
    const cudaError_t e = cudaFuncSetAttribute(k_tree<__half>, cudaFuncAttributeMaxDynamicSharedMemorySize, TR_SMEM);
    return e != cudaSuccess ? e : cudaFuncSetAttribute(k_tree<__nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize, TR_SMEM);
}

template <class T>
static cudaError_t tree_go(const TreeParams& p, const CUtensorMap& map, const CUtensorMap& map16, const CUtensorMap& q_map, const TreeWork& wk, int pairs, cudaStream_t st) {
    const cudaError_t e = launch_pdl_n(k_tree<T>, dim3(2 * pairs), dim3(TR_THREADS), TR_SMEM, st, p, map, map16, q_map, wk);
    // no item is split where a sequence's pages hold one tile at most: a launch less (one tile 2 us less a call)
    if (e != cudaSuccess || p.kv.table_stride << p.kv.page_shift <= ATT_TILE) return e;
    return launch_pdl_n(k_merge<T>, dim3(2 * pairs * MG_BLOCKS), dim3(MG_THREADS), 0, st, p, wk, pairs);
}

cudaError_t launch_tree(const TreeParams& p, int dtype, const CUtensorMap& map, const CUtensorMap& map16, const CUtensorMap& q_map, const TreeWork& wk, int pairs, cudaStream_t st) {
    return dtype == LK_DT_F16 ? tree_go<__half>(p, map, map16, q_map, wk, pairs, st) : tree_go<__nv_bfloat16>(p, map, map16, q_map, wk, pairs, st);
}

}  // namespace lk
