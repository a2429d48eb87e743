// attn_tree.cu -- attention of drafted token trees over the paged latent cache.
//
// S = scale * Q K^T with K the 576-wide rows, P = softmax(S) over the rows that a token sees, O = P C with C the first
// 512 values of the same rows.  One pass over the cache with a running reference m and sum l per row: P = 2^(S' - m + 7)
// (S' in units of log 2), and where a tile's maximum exceeds m by more than 8, m moves there and O and l are scaled.
//
// Work.  A row is one (token, head); 128 rows of one sequence are an item, 128 cached rows a tile, and (item, tile) a
// unit of work: 35.7 M products, 147 KB of cache.  All units, numbered item by item, are cut into equal runs, one per
// pair of CTAs, whatever the batch's lengths; of an item that lies in several runs each leaves its O, m and l, and joins a share of them.
// Lengths are read on the device, so a captured call follows them.
//
// Why a pair.  fp32 O is 128 x 512: all of one SM's tensor memory.  A pair halves the rows (2-CTA tcgen05.mma, M = 128:
// 64 rows of each CTA in all 128 lanes), so O takes 256 columns and two S buffers 128, and Q 72 KB of shared memory.  Each
// CTA loads half of a tile's rows for S (64 x 576) and half of the latent columns of all of them for O (128 x 256).
// Measured on a B200, 2-CTA M = 128 runs at the full 4096 products per cycle and SM for N = 128 and 256 (one CTA with
// M = 128, N = 128 reaches 2925), so a unit costs 2176 cycles of tensor pipe; 45 bytes per cycle and SM from L2 into all
// SMs at once makes the 136 KB a CTA loads for it about 3100, which bounds calls with many rows.  Few rows are bound by
// HBM: 74 pairs at 3100 cycles ask for 6.7 TB/s.
//
// Roles (384 threads a CTA): warp 0 loads (TMA, ring of 8 x 16 KB), warps 1 and 2 of CTA 0 issue the MMAs of S and of O,
// warp 3 repairs tail tiles, warps 4-11 do softmax, O's scaling and the output (two threads per tensor-memory lane, four per
// row: with one per lane V waits twice as long in the ring for P).  Order of the ring: K(0), K(1), V(0),
// K(2), V(1), ..: softmax j runs under S(j + 1).  Two issuing threads because a satisfied barrier wait between two MMAs
// leaves the tensor pipe empty for ~50 cycles, 11 times a unit: while one thread waits the other's MMAs run.
//
// Rows that must not matter: a tile's rows beyond the drafts, and drafted rows that a token does not see, get P = 0; but
// 0 * NaN is NaN, so warp 3 zeroes the former in the O operand, and every drafted row there that holds a non-finite
// value (a token that does see it gets its NaN through S and P).
#include <type_traits>
#include "attn_tc.cuh"
#include "attn_sched.cuh"

namespace lk {

constexpr int TR_THREADS = 384, TR_STAGES = 8, TR_STAGE = 16384, TR_CHUNK = 8192;
constexpr int TR_Q = 0, TR_P = 9 * TR_CHUNK, TR_RING = TR_P + TR_STAGE, TR_BARS = TR_RING + TR_STAGES * TR_STAGE;
constexpr int TR_XCH = TR_BARS + 48 * 8, TR_SCHED = TR_XCH + 256 * 4;
constexpr int TR_SMEM = TR_SCHED + (int)sizeof(Sched);
static_assert(TR_SMEM <= 232448, "227 KB a CTA");
constexpr uint32_t TR_S_COL = 256, TR_TMEM = 512;
constexpr float TR_SHIFT = 7.0f, TR_JUMP = 8.0f;      // P <= 2^15 fits fp16; its smallest normal is 2^-21 of the reference

// a split item that this CTA left a part of
struct TreeJoin { int q0, parts, slot0, rows, row0, first; };       // first run, runs, the first part's slot, rows, first row, first token

struct TreeBars {
    uint64_t full[TR_STAGES], empty[TR_STAGES], land[TR_STAGES];
    uint64_t s_full[2], s_free[2], p_full, o_done, q_full, joined, drain[2];
    uint32_t tmem;
    int gave_up;
    TreeJoin join[2];
};
static_assert(sizeof(TreeBars) <= 48 * 8, "barrier block");

// ---------------------------------------------------------------- joining the parts of an item
// out = sum_q f_q O_q / sum_q f_q l_q with f_q = 2^(m_q - max m) over the item's parts q.  Every CTA that left a part takes an
// equal share of the item's (8-row group, 4 latent values, row) elements once all parts are there: 128 KB in all, whatever the
// number of parts, fetched by one bulk copy a part into the memory that Q and the ring had.  They are added in the parts'
// order, so the result does not depend on who was first.
constexpr int JN_PARTS = 128, JN_STAGE = 8192;

template <class T>
__device__ __forceinline__ void tree_join(const TreeParams& p, const TreeWork& wk, const TreeJoin& jn, int cta, int pairs, uint8_t* sm, int tid,
                                          uint64_t* bar, uint32_t parity, volatile int* gave_up) {
    const int warp = tid >> 5, lane = tid & 31, n = jn.parts, ctas = 2 * n;
    float* ref = (float*)sm; float* sum = ref + 128; float* f = sum + 128;      // of the share's rows; f [part][row]
    const float4* stage = (const float4*)(sm + JN_STAGE);                       // [part][element]
    auto slot = [&](int i) { return i ? (jn.slot0 & ~1) + 2 * i : jn.slot0; };
    // this CTA's elements e: row group e / 1024, values 4 (e / 8 % 128), row e % 8
    const int mine = cta - 2 * jn.q0, all = (jn.rows + 7) / 8 * 1024;
    const int e0 = (int)((uint32_t)(all * mine) / (uint32_t)ctas), e1 = (int)((uint32_t)(all * (mine + 1)) / (uint32_t)ctas), ne = e1 - e0;
    const int r0 = e0 >> 10 << 3, nr = ne ? min(jn.rows, ((e1 - 1) >> 10 << 3) + 8) - r0 : 0;
    if (warp == 0) {
        if (lane == 0) {
            const unsigned long long t0 = globaltimer_ns();
            int seen;
            do {
                asm volatile("ld.acquire.gpu.s32 %0, [%1];" : "=r"(seen) : "l"(wk.sync + jn.q0) : "memory");
                if (seen < ctas && (*gave_up || globaltimer_ns() - t0 > WAIT_LIMIT_NS)) { att_error(p.err, DEV_ERR_TIMEOUT_FULL); *gave_up = 1; break; }
            } while (seen < ctas);
            asm volatile("fence.proxy.async;" ::: "memory");                    // the parts were written by ordinary stores
            mbar_arrive_expect_tx(bar, (uint32_t)(n * ne) * 16);
        }
        __syncwarp();
        if (ne) for (int i = lane; i < n; i += 32) bulk_g2s((void*)(stage + i * ne), wk.part + (int64_t)slot(i) * (128 * 128) + e0, ne * 16, bar);
    }
    named_bar_sync(1, 256);
    for (int r = warp; r < nr; r += 8) {
        float m = -INFINITY, l = 0.0f;
        for (int i = lane; i < n; i += 32) m = fmaxf(m, __ldcg(&wk.ml[slot(i) * 128 + r0 + r]).x);
        #pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float rf = m == -INFINITY ? 0.0f : m;
        for (int i = lane; i < n; i += 32) {
            const float2 ml = __ldcg(&wk.ml[slot(i) * 128 + r0 + r]);
            // a part that saw nothing has sum 0; one of NaN scores alone has no maximum, and a NaN sum
            const float v = ml.y == 0.0f ? 0.0f : exp2_approx((ml.x == -INFINITY ? 0.0f : ml.x) - rf);
            f[i * nr + r] = v;
            l += v == 0.0f ? 0.0f : v * ml.y;
        }
        #pragma unroll
        for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if (lane == 0) { ref[r] = rf; sum[r] = l; }
    }
    named_bar_sync(1, 256);
    wait_phase(bar, parity, gave_up, p.err);
    for (int x = tid; x < ne; x += 256) {
        const int e = e0 + x, r = (e >> 10 << 3) + (e & 7), c4 = (e >> 3) & 127;
        if (r >= jn.rows) continue;
        float4 s = make_float4(0, 0, 0, 0);
        #pragma unroll 4
        for (int i = 0; i < n; ++i) {
            const float4 v = stage[i * ne + x];
            const float w = f[i * nr + r - r0];
            s.x += w == 0.0f ? 0.0f : w * v.x;
            s.y += w == 0.0f ? 0.0f : w * v.y;
            s.z += w == 0.0f ? 0.0f : w * v.z;
            s.w += w == 0.0f ? 0.0f : w * v.w;
        }
        const int gr = jn.row0 + r, tj = gr / p.H, h = gr - tj * p.H, t = jn.first + tj;
        const float l = sum[r - r0], inv = l == 0.0f ? 0.0f : 1.0f / l;
        *(uint2*)((T*)p.out + (int64_t)t * p.out_token + (int64_t)h * p.out_head + 4 * c4) =
            make_uint2(pack2<T>(s.x * inv, s.y * inv), pack2<T>(s.z * inv, s.w * inv));
        if (c4 == 0 && p.lse) p.lse[(int64_t)t * p.H + h] = l == 0.0f ? -INFINITY : (ref[r - r0] - TR_SHIFT + log2f(l)) * 0.6931471805599453f;
    }
    if (tid == 0 && atomicAdd(wk.sync + pairs + jn.q0, 1) == ctas - 1) { wk.sync[jn.q0] = 0; wk.sync[pairs + jn.q0] = 0; }
    fence_async_smem();                                // the next join's copies come after these reads
    named_bar_sync(1, 256);
}

// the load role of one CTA, one thread: boxes of BOX rows x 64 values.  Its instructions are the loop's length (a loaded
// stage feeds 512 cycles of MMAs), so the page lookups are made a tile ahead and nothing is computed per box.
template <int BOX>
__device__ __forceinline__ bool tree_load(const TreeParams& p, const Sched& sched, int64_t u, int64_t u_end, const CUtensorMap* map,
                                          TreeBars& B, uint32_t smb, uint32_t rank) {
    constexpr int NB = 64 / BOX;                          // boxes of 64 rows
    const uint32_t full0 = peer_addr(smem_u32(&B.full[0]), 0);
    uint32_t st = 0, ph = 1, dst = smb + TR_RING, bar = full0;
    auto advance = [&]() {
        dst += TR_STAGE; bar += 8;
        if (++st == TR_STAGES) { st = 0; ph ^= 1; dst = smb + TR_RING; bar = full0; }
    };
    for (Segment g; sched_next<ATT_TILE>(p, sched, u, u_end, g);) {
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
                const bool tail = j * ATT_TILE > g.len;   // tile j - 1 reaches beyond the context: warp 3 passes it on
                #pragma unroll
                for (int s = 0; s < 4; ++s) {             // column group s / 2, row half s % 2
                    if (!wait_phase(&B.empty[st], ph, &B.gave_up, p.err)) return false;
                    uint32_t to = bar;
                    if (tail) { to = smem_u32(&B.land[st]); mbar_arrive_expect_tx(&B.land[st], TR_STAGE); }
                    else arrive_expect_at(bar, TR_STAGE);
                    const int col = (s >> 1) * 256 + (int)rank * 128;
                    #pragma unroll
                    for (int c = 0; c < 2; ++c)
                        #pragma unroll
                        for (int x = 0; x < NB; ++x) tma_2d_pair(dst + c * TR_CHUNK + x * BOX * 128, map, col + c * 64, v[(s & 1) * NB + x], to);
                    advance();
                }
            }
        }
    }
    return true;
}

template <class T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(TR_THREADS, 1)
k_tree(const __grid_constant__ TreeParams p, const __grid_constant__ CUtensorMap kv_map, TreeWork wk) {
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
        for (int s = 0; s < TR_STAGES; ++s) { mbar_init(&B.full[s], 2); mbar_init(&B.empty[s], 1); mbar_init(&B.land[s], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&B.s_full[i], 1); mbar_init(&B.s_free[i], 16); mbar_init(&B.drain[i], 1); }
        mbar_init(&B.p_full, 16); mbar_init(&B.o_done, 1); mbar_init(&B.q_full, 16); mbar_init(&B.joined, 1);
        fence_mbar_init();
        asm volatile("prefetch.tensormap [%0];" :: "l"(&kv_map) : "memory");
    }
    if (warp == 3) tmem_alloc2(&B.tmem, TR_TMEM);
    if (warp == 0 || p.kv.n_seqs > 1) sched_load<ATT_TILE>(p, sched, tid, TR_THREADS, pairs);
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = B.tmem;
    int64_t u = pair < sched.runs ? sched.run_start(pair) : 0;
    const int64_t u_end = pair < sched.runs ? sched.run_start(pair + 1) : 0;
    const uint32_t smb = smem_u32(sm);

    if (warp == 0) {
        // ---------------------------------------------------------------- loads
        if (elect_one()) {
            const bool ok = p.kv.page_size >= 64 ? tree_load<64>(p, sched, u, u_end, &kv_map, B, smb, rank)
                          : p.kv.page_size == 32 ? tree_load<32>(p, sched, u, u_end, &kv_map, B, smb, rank)
                                                 : tree_load<16>(p, sched, u, u_end, &kv_map, B, smb, rank);
            if (!ok) __nanosleep(1000000);                // given up: the loads in flight land before the CTA ends
        }
    } else if (warp < 3) {
        // ---------------------------------------------------------------- MMAs, issued by CTA 0 for both: S and O by a thread each
        if (rank == 0 && elect_one()) {
            constexpr uint32_t id_s = att_idesc(128, 128, BF, false), id_o = att_idesc(128, 256, BF, true);
            uint32_t st = 0, ph = 0, n = 0, n_q = 0;      // ring place; tiles and segments so far
            bool ok = true;
            auto wait = [&](uint64_t* bar, uint32_t parity) { return ok = wait_phase(bar, parity, gave_up, p.err); };
            auto advance = [&](uint32_t k) { st += k; if (st >= TR_STAGES) { st -= TR_STAGES; ph ^= 1; } };
            if (warp == 1) {
                for (Segment g; ok && sched_next<ATT_TILE>(p, sched, u, u_end, g);) {
                    if (!wait(&B.q_full, n_q++ & 1)) break;
                    for (int j = g.t0; ok && j < g.t1; ++j, ++n) {
                        const uint32_t buf = n & 1, d = tmem + TR_S_COL + buf * 64;
                        if (!wait(&B.s_free[buf], ((n >> 1) & 1) ^ 1)) break;
                        tc_fence_after();
                        for (int s = 0; s < 5; ++s) {
                            if (!wait(&B.full[st], ph)) break;
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
                for (Segment g; ok && sched_next<ATT_TILE>(p, sched, u, u_end, g);) {
                    advance(5);                           // K of the first tile
                    for (int j = g.t0; ok && j < g.t1; ++j, ++n) {
                        if (j + 1 < g.t1) advance(5);     // K of tile j + 1
                        if (!wait(&B.p_full, n & 1)) break;
                        tc_fence_after();
                        for (int s = 0; s < 4; ++s) {
                            if (!wait(&B.full[st], ph)) break;
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
        const uint32_t full0 = peer_addr(smem_u32(&B.full[0]), 0);
        uint32_t st = 0, uses = 0;                        // bit s: parity of the uses of land[s]
        auto advance = [&](int n) { st = (st + n) % TR_STAGES; };
        for (Segment g; sched_next<ATT_TILE>(p, sched, u, u_end, g);) {
            for (int j = g.t0; j <= g.t1; ++j) {
                if (j < g.t1) advance(5);
                if (j == g.t0) continue;
                if (j * ATT_TILE <= g.len) { advance(4); continue; }
                for (int s = 0; s < 4; ++s, advance(1)) {
                    wait_phase(&B.land[st], (uses >> st) & 1, gave_up, p.err);
                    uses ^= 1u << st;
                    // rows (s % 2) * 64 .. + 63 of the tile, 2 x 128 bytes each: eight lanes a row.  Each row's part is judged by
                    // itself: all that matters is that nothing non-finite is multiplied by 0
                    const int i0 = (j - 1) * ATT_TILE + (s & 1) * 64;
                    for (int r = max(0, g.len - i0) & ~3; r < 64; r += 4) {
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
        int parts = 0;                                    // split items so far
        auto wait = [&](uint64_t* bar, uint32_t parity) { wait_phase(bar, parity, gave_up, p.err); tc_fence_after(); };
        // Q of a segment: this CTA's 64 rows of the item, 9 swizzled chunks of 64 values; 8 rows a warp, whose places in q
        // the lanes that own the rows know
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
        bool more = sched_next<ATT_TILE>(p, sched, u, u_end, g);
        if (more) { start_q(g); finish_q(); }
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
                if (named_bar_or(1, 256, top > m + TR_JUMP)) {
                    xch[part * 64 + row] = top;
                    named_bar_sync(1, 256);
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
                    named_bar_sync(1, 256);               // xch is free again
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
            more = sched_next<ATT_TILE>(p, sched, u, u_end, next);
            if (more) start_q(next);
            wait(&B.o_done, (n - 1) & 1);
            if (more) finish_q();
            xch[part * 64 + row] = l;
            named_bar_sync(1, 256);
            l = (xch[row] + xch[64 + row]) + (xch[128 + row] + xch[192 + row]);
            named_bar_sync(1, 256);
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
                const int q0 = sched.owner(g.item);
                if (tid == 128) {
                    TreeJoin& jn = B.join[parts];
                    jn.q0 = q0;
                    jn.parts = sched.owner(g.item + g.tiles - 1) - q0 + 1;
                    jn.slot0 = 2 * q0 + (g.item > sched.run_start(q0));
                    jn.rows = min(ATT_ITEM, g.n * p.H - g.rt * ATT_ITEM);
                    jn.row0 = g.rt * ATT_ITEM;
                    jn.first = g.first;
                }
                ++parts;
                __threadfence();
                named_bar_sync(1, 256);
                if (tid == 128) atomicAdd(wk.sync + q0, 1);
            }
            tc_fence_before();
            g = next;
        }
        for (int i = 0; i < parts; ++i) tree_join<T>(p, wk, B.join[i], 2 * pair + (int)rank, pairs, sm, tid - 128, &B.joined, i, gave_up);
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    if (warp == 3) { tc_fence_after(); tmem_dealloc2(tmem, TR_TMEM); }
}

int tree_pairs(int nsm) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.gridDim = nsm / 2 * 2; cfg.blockDim = TR_THREADS; cfg.dynamicSmemBytes = TR_SMEM; cfg.attrs = attr; cfg.numAttrs = 1;
    int n = 0;
    if (cudaFuncSetAttribute(k_tree<__half>, cudaFuncAttributeMaxDynamicSharedMemorySize, TR_SMEM) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, k_tree<__half>, &cfg) != cudaSuccess) { cudaGetLastError(); return 0; }
    n = n < nsm / 2 ? n : nsm / 2;
    return n < JN_PARTS ? n : JN_PARTS;
}

template <class T>
static cudaError_t tree_go(const TreeParams& p, const CUtensorMap& map, const TreeWork& wk, int pairs, cudaStream_t st) {
    cudaError_t e = cudaFuncSetAttribute(k_tree<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, TR_SMEM);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeCooperative;      // pairs wait for one another's parts: all of them run at once
    attr[0].val.cooperative = 1;
    cfg.gridDim = 2 * pairs; cfg.blockDim = TR_THREADS; cfg.dynamicSmemBytes = TR_SMEM; cfg.stream = st; cfg.attrs = attr; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_tree<T>, p, map, wk);
}

cudaError_t launch_tree(const TreeParams& p, int dtype, const CUtensorMap& map, const TreeWork& wk, int pairs, cudaStream_t st) {
    return dtype == LK_DT_F16 ? tree_go<__half>(p, map, wk, pairs, st) : tree_go<__nv_bfloat16>(p, map, wk, pairs, st);
}

}  // namespace lk
