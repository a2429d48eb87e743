// attn_api.cu -- the lk_attn_* C ABI (include/loki_attn.h): context, workspaces, argument checks and launches.
#include <cstdio>
#include <cstdarg>
#include <new>
#include "attn_internal.h"

using namespace lk;

struct LkAttnCtx {
    LkAttnConfig cfg;
    int device = 0, nsm = 0;
    int* err = nullptr;
    int* n_moves = nullptr;
    // eviction: [2][n_seqs][region] of the last of `moves`.  A captured graph keeps the address that its call had, so a list that
    // became too small stays until the context ends; sizes are powers of two, so the ones before take no more than the last.
    int* moves[64] = {}; int n_lists = 0; int64_t moves_cap = 0;
    TreeWork work{}; int pairs = 0;                                           // lk_attn_tree: parts of split items
    MassWork mass{};
    char msg[256] = {0};
};

static int set_err(LkAttnCtx* c, int code, const char* fmt, ...) {
    if (c) { va_list ap; va_start(ap, fmt); vsnprintf(c->msg, sizeof(c->msg), fmt, ap); va_end(ap); }
    return code;
}
// a failed call is reported once: the runtime's last error would come out again of the next launch that asks for it
static int cuda_err(LkAttnCtx* c, const char* call, cudaError_t e) {
    cudaGetLastError();
    return set_err(c, LK_ERR_CUDA, "%s: %s", call, cudaGetErrorString(e));
}
#define LK_CU(call) do { cudaError_t e_ = (call); if (e_ != cudaSuccess) return cuda_err(c, #call, e_); } while (0)

namespace {
// the context's device for the length of a call; the caller's is put back
struct OnDevice {
    int prev = -1;
    explicit OnDevice(int device) { if (cudaGetDevice(&prev) == cudaSuccess && prev != device) cudaSetDevice(device); else prev = -1; }
    ~OnDevice() { if (prev >= 0) cudaSetDevice(prev); }
};
}

static bool is16(const void* p) { return p && !((uintptr_t)p & 15); }

// rows of 64-value columns as a tensor map: dims[0] values of a row, the outer strides in elements, boxes of 64 values x `rows` of
// dimension `along`, 128-byte swizzle, zeros outside
static int encode_map(LkAttnCtx* c, CUtensorMap* map, int dtype, const void* base, int rank, const int64_t* dims, const int64_t* strides, int rows,
                      int along = 1) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        const bool ok = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess;
        return ok ? (Encode)f : nullptr;
    }();
    if (!encode) return set_err(c, LK_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
    cuuint64_t d[3], s[2];
    for (int i = 0; i < rank; ++i) d[i] = (cuuint64_t)dims[i];
    for (int i = 0; i + 1 < rank; ++i) s[i] = (cuuint64_t)strides[i] * 2;
    const cuuint32_t box[3] = { 64, along == 1 ? (cuuint32_t)rows : 1, along == 2 ? (cuuint32_t)rows : 1 }, step[3] = { 1, 1, 1 };
    const CUresult r = encode(map, dtype == LK_DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), d, s,
                              box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? LK_OK : set_err(c, LK_ERR_CUDA, "cuTensorMapEncodeTiled: %d", (int)r);
}
// the cache: boxes of up to `most` rows of one page
static int kv_map(LkAttnCtx* c, const LkKvCache* k, CUtensorMap* map, int most = 64) {
    const int64_t dims[2] = { AT_ROW, (int64_t)k->n_pages * k->page_size }, strides[1] = { k->row_stride };
    return encode_map(c, map, k->dtype, k->rows, 2, dims, strides, k->page_size < most ? k->page_size : most);
}

// a workspace that is made on the first call that needs it; not inside a stream capture
static int may_allocate(LkAttnCtx* c, cudaStream_t st) {
    cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
    LK_CU(cudaStreamIsCapturing(st, &cs));
    return cs == cudaStreamCaptureStatusNone ? LK_OK : set_err(c, LK_ERR_CAPACITY, "the first call makes its workspace: call once before the capture");
}

// the cache's fields, and what the kernels see of it
static int check_cache(LkAttnCtx* c, const LkKvCache* k, KvView* v) {
    if (!k) return set_err(c, LK_ERR_ARG, "null cache");
    if (k->dtype != LK_DT_F16 && k->dtype != LK_DT_BF16) return set_err(c, LK_ERR_UNSUPPORTED, "cache dtype %d: fp16 (1) or bf16 (2)", k->dtype);
    if (!is16(k->rows)) return set_err(c, LK_ERR_ARG, "cache rows null or not 16-byte aligned");
    if (k->row_stride < AT_ROW || k->row_stride % 8) return set_err(c, LK_ERR_ARG, "row stride %lld: at least 576 and a multiple of 8", (long long)k->row_stride);
    int shift = 4;
    while (shift < 8 && (1 << shift) != k->page_size) ++shift;
    if ((1 << shift) != k->page_size) return set_err(c, LK_ERR_UNSUPPORTED, "page size %d: 16, 32, 64, 128 or 256", k->page_size);
    if (k->n_pages < 1 || (int64_t)k->n_pages * k->page_size > 0x7fffffff) return set_err(c, LK_ERR_ARG, "%d pages of %d rows", k->n_pages, k->page_size);
    if (k->n_seqs < 1 || k->n_seqs > c->cfg.max_seqs) return set_err(c, LK_ERR_CAPACITY, "%d sequences, context capacity %d", k->n_seqs, c->cfg.max_seqs);
    if (!k->block_table || !k->lens) return set_err(c, LK_ERR_ARG, "null block table or lens");
    if (k->table_stride < 1 || (int64_t)k->table_stride * k->page_size > 0x7fffff00) return set_err(c, LK_ERR_ARG, "table stride %d", k->table_stride);
    *v = KvView{ k->rows, k->row_stride, k->page_size, shift, k->n_pages, k->table_stride, k->n_seqs, k->block_table, k->lens, k->mass, k->pos };
    return LK_OK;
}

static int check_rows(LkAttnCtx* c, const char* name, const void* p, int64_t token, int64_t head) {
    if (!is16(p)) return set_err(c, LK_ERR_ARG, "%s null or not 16-byte aligned", name);
    if (token % 8 || head % 8) return set_err(c, LK_ERR_ARG, "%s strides must be multiples of 8", name);
    return LK_OK;
}

extern "C" {

int lk_attn_create(const LkAttnConfig* cfg, int device, LkAttnCtx** out) {
    if (!cfg || !out) return LK_ERR_ARG;
    *out = nullptr;
    if (cfg->max_seqs < 1 || cfg->max_seqs > LK_ATTN_MAX_SEQS || cfg->max_tokens < 1 || cfg->max_tokens > LK_ATTN_MAX_SEQS * LK_ATTN_MAX_NODES)
        return LK_ERR_UNSUPPORTED;
    LkAttnCtx* c = new (std::nothrow) LkAttnCtx();
    if (!c) return LK_ERR_CAPACITY;
    c->cfg = *cfg;
    c->device = device;
    int prev = 0;
    cudaError_t e = cudaGetDevice(&prev);
    if (e == cudaSuccess) e = cudaSetDevice(device);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&c->nsm, cudaDevAttrMultiProcessorCount, device);
    if (e == cudaSuccess) e = cudaMalloc((void**)&c->err, sizeof(int));
    if (e == cudaSuccess) e = cudaMemset(c->err, 0, sizeof(int));
    if (e == cudaSuccess) e = cudaMalloc((void**)&c->n_moves, (size_t)cfg->max_seqs * sizeof(int));
    const size_t sums = (size_t)(c->nsm / 2) * 2 * 256 * sizeof(float), counts = (size_t)(c->nsm / 2) * 2 * sizeof(unsigned);
    if (e == cudaSuccess) e = cudaMalloc((void**)&c->mass.part, sums + counts);
    if (e == cudaSuccess) e = cudaMemset(c->mass.part, 0, sums + counts);
    c->mass.arrived = (unsigned*)((char*)c->mass.part + sums);
    if (e == cudaSuccess) e = tree_setup();
    if (e == cudaSuccess) e = mass_setup();
    if (e == cudaSuccess) e = evict_setup();
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    cudaSetDevice(prev);
    if (e != cudaSuccess) { lk_attn_destroy(c); cudaGetLastError(); return LK_ERR_CUDA; }
    *out = c;
    return LK_OK;
}

void lk_attn_destroy(LkAttnCtx* c) {
    if (!c) return;
    OnDevice on(c->device);
    void* ptrs[] = { c->err, c->n_moves, c->work.part, c->mass.part };
    for (void* p : ptrs) if (p) cudaFree(p);
    for (int i = 0; i < c->n_lists; ++i) cudaFree(c->moves[i]);
    delete c;
}

int lk_attn_get_error(LkAttnCtx* c, lk_stream_t stream) {
    if (!c) return LK_ERR_ARG;
    OnDevice on(c->device);
    // all of it in the stream's own order: the default stream would wait for others, and its memset could run behind a later call
    const cudaStream_t st = (cudaStream_t)stream;
    int e = 0;
    LK_CU(cudaMemcpyAsync(&e, c->err, sizeof(int), cudaMemcpyDeviceToHost, st));
    LK_CU(cudaStreamSynchronize(st));
    if (!e) return LK_OK;
    LK_CU(cudaMemsetAsync(c->err, 0, sizeof(int), st));
    LK_CU(cudaStreamSynchronize(st));
    const char* what = e == ATT_ERR_PAGE ? "a page id outside the pool" : e == ATT_ERR_POS ? "a position outside the rope table"
                     : e == ATT_ERR_LEN ? "a length outside its pages" : e == ATT_ERR_TREE ? "token ranges out of order or too long"
                     : "a bounded wait ran out";
    return set_err(c, LK_ERR_DEVICE, "device error code %d: %s", e, what);
}

const char* lk_attn_last_error(LkAttnCtx* c) { return c ? c->msg : "null context"; }

int lk_attn_rope_table(LkAttnCtx* c, const LkRopeConfig* cfg, int max_pos, float* table, lk_stream_t stream) {
    if (!cfg || !table || ((uintptr_t)table & 7)) return set_err(c, LK_ERR_ARG, "null config, or table null or not 8-byte aligned");
    if (cfg->rot_dim < 2 || cfg->rot_dim % 2 || cfg->rot_dim > 4096 || max_pos < 1 || max_pos > (1 << 26)) return set_err(c, LK_ERR_ARG, "rot_dim %d, max_pos %d", cfg->rot_dim, max_pos);
    if (!(cfg->base > 1.0) || !(cfg->factor >= 1.0) || !(cfg->mscale > 0.0)) return set_err(c, LK_ERR_ARG, "base must exceed 1, factor be at least 1, mscale positive");
    if (cfg->factor > 1.0 && (cfg->orig_ctx < 1 || !(cfg->beta_slow > 0.0) || !(cfg->beta_fast >= cfg->beta_slow)))
        return set_err(c, LK_ERR_ARG, "a stretched context needs orig_ctx and beta_fast >= beta_slow > 0");
    LK_CU(launch_rope_table(*cfg, max_pos, (float2*)table, (cudaStream_t)stream));
    return LK_OK;
}

int lk_attn_rope(LkAttnCtx* c, int dtype, const void* x, int64_t x_token, int64_t x_head, void* y, int64_t y_token, int64_t y_head,
                 int T, int H, int head_dim, int rot_offset, int rot_dim, int layout, int grad, const int* pos, const float* table,
                 int max_pos, lk_stream_t stream) {
    if (!c) return LK_ERR_ARG;
    if (dtype < LK_DT_F32 || dtype > LK_DT_BF16 || layout < LK_ROPE_INTERLEAVED || layout > LK_ROPE_HALF)
        return set_err(c, LK_ERR_UNSUPPORTED, "dtype %d, layout %d", dtype, layout);
    if (T < 0 || H < 1 || H > 65536 || head_dim < 1 || head_dim > 65536 || rot_dim < 2 || rot_dim % 2 || rot_offset < 0 || rot_offset > head_dim - rot_dim || max_pos < 1)
        return set_err(c, LK_ERR_ARG, "T %d, H %d, head_dim %d, rotated part [%d, %d)", T, H, head_dim, rot_offset, rot_offset + rot_dim);
    if (T == 0) return LK_OK;
    const int es = dtype == LK_DT_F32 ? 4 : 2;
    if (!x || !y || !pos || !table || ((uintptr_t)x | (uintptr_t)y) % es || ((uintptr_t)table & 7)) return set_err(c, LK_ERR_ARG, "null or misaligned pointer");
    if (x == y && (x_token != y_token || x_head != y_head)) return set_err(c, LK_ERR_ARG, "in place needs equal strides");
    // a token's units are counted in 32 bits, as are the blocks
    if ((int64_t)H * head_dim > (1 << 30) || (int64_t)T * (((int64_t)H * head_dim + 31) / 32) > 0x7fffffff) return set_err(c, LK_ERR_CAPACITY, "T %d x H %d x %d", T, H, head_dim);
    OnDevice on(c->device);
    RopeParams p{ x, x_token, x_head, y, y_token, y_head, T, H, head_dim, rot_offset, rot_dim, grad != 0, x != y, pos, (const float2*)table, max_pos, c->err };
    LK_CU(launch_rope(p, dtype, layout, (cudaStream_t)stream));
    return LK_OK;
}

int lk_attn_append(LkAttnCtx* c, const LkKvCache* cache, int in_dtype, const void* latent, int64_t latent_ld, const void* k_rope,
                   int64_t rope_ld, int T, const int* starts, const int* pos, const float* table, int max_pos, int layout,
                   lk_stream_t stream) {
    if (!c) return LK_ERR_ARG;
    AppendParams p{};
    if (int rc = check_cache(c, cache, &p.kv)) return rc;
    if (in_dtype != LK_DT_F32 && in_dtype != cache->dtype) return set_err(c, LK_ERR_UNSUPPORTED, "input dtype %d: fp32 or the cache's", in_dtype);
    if (layout < LK_ROPE_INTERLEAVED || layout > LK_ROPE_HALF) return set_err(c, LK_ERR_UNSUPPORTED, "layout %d", layout);
    if (T < 0 || T > 0x7fffffff / 256 || max_pos < 1) return set_err(c, LK_ERR_ARG, "T %d, max_pos %d", T, max_pos);
    if (T == 0) return LK_OK;
    if (int rc = check_rows(c, "latent", latent, latent_ld, 0)) return rc;
    if (int rc = check_rows(c, "k_rope", k_rope, rope_ld, 0)) return rc;
    if (!starts || !pos || !table || ((uintptr_t)table & 7)) return set_err(c, LK_ERR_ARG, "null or misaligned pointer");
    OnDevice on(c->device);
    p.latent = latent; p.latent_ld = latent_ld; p.k_rope = k_rope; p.rope_ld = rope_ld; p.T = T; p.starts = starts; p.pos = pos;
    p.table = (const float2*)table; p.max_pos = max_pos; p.err = c->err;
    LK_CU(launch_append(p, in_dtype, cache->dtype, layout, (cudaStream_t)stream));
    return LK_OK;
}

// what lk_attn_tree and lk_attn_mass check alike
static int tree_params(LkAttnCtx* c, const LkKvCache* cache, const void* q, int64_t q_token, int64_t q_head, int T, int H,
                       const int* starts, const uint64_t* tree, float scale, TreeParams* p) {
    if (int rc = check_cache(c, cache, &p->kv)) return rc;
    if (T < 0 || H < 1 || H > LK_ATTN_MAX_HEADS) return set_err(c, LK_ERR_ARG, "T %d, H %d (at most %d heads)", T, H, LK_ATTN_MAX_HEADS);
    if (T > c->cfg.max_tokens) return set_err(c, LK_ERR_CAPACITY, "T %d > capacity %d", T, c->cfg.max_tokens);
    if (!(scale > 0.0f) || scale > 3.0e38f) return set_err(c, LK_ERR_ARG, "scale must be positive and finite");
    if (T == 0) return LK_OK;
    if (int rc = check_rows(c, "q", q, q_token, q_head)) return rc;
    if (!starts || ((uintptr_t)tree & 7)) return set_err(c, LK_ERR_ARG, "null starts or misaligned tree");
    p->q = q; p->q_token = q_token; p->q_head = q_head; p->T = T; p->H = H; p->starts = starts; p->tree = tree; p->scale = scale;
    p->err = c->err;
    return LK_OK;
}

int lk_attn_tree(LkAttnCtx* c, const LkKvCache* cache, const void* q, int64_t q_token, int64_t q_head, int T, int H, const int* starts,
                 const uint64_t* tree, float scale, void* out, int64_t out_token, int64_t out_head, float* lse, lk_stream_t stream) {
    if (!c) return LK_ERR_ARG;
    TreeParams p{};
    if (int rc = tree_params(c, cache, q, q_token, q_head, T, H, starts, tree, scale, &p)) return rc;
    if (T == 0) return LK_OK;
    if (int rc = check_rows(c, "out", out, out_token, out_head)) return rc;
    OnDevice on(c->device);
    p.out = out; p.out_token = out_token; p.out_head = out_head; p.lse = lse;
    CUtensorMap map, map16, q_map{};
    if (int rc = kv_map(c, cache, &map)) return rc;
    if (int rc = kv_map(c, cache, &map16, 16)) return rc;
    const int64_t step = H > 1 ? q_head : q_token;       // from one (token, head) row to the next
    p.q_flat = (H == 1 || T == 1 || q_token == H * q_head) && step >= AT_ROW;
    if (p.q_flat) {
        const int64_t dims[2] = { AT_ROW, (int64_t)T * H };
        if (int rc = encode_map(c, &q_map, cache->dtype, q, 2, dims, &step, 64)) return rc;
    }
    if (!c->work.part) {                              // parts of at most two items per pair of SMs: 0.5 MB a pair
        if (int rc = may_allocate(c, (cudaStream_t)stream)) return rc;
        c->pairs = tree_pairs(c->nsm);
        const size_t part = (size_t)c->pairs * 2 * 128 * AT_LATENT * 4, ml = (size_t)c->pairs * 2 * 128 * 8;
        char* w = nullptr;
        LK_CU(cudaMalloc((void**)&w, part + ml + 2 * c->pairs * sizeof(TreeSplit)));
        c->work = TreeWork{ (float4*)w, (float2*)(w + part), (TreeSplit*)(w + part + ml) };
    }
    LK_CU(launch_tree(p, cache->dtype, map, map16, q_map, c->work, c->pairs, (cudaStream_t)stream));
    return LK_OK;
}

int lk_attn_mass(LkAttnCtx* c, const LkKvCache* cache, const void* q, int64_t q_token, int64_t q_head, int T, int H, const int* starts,
                 const uint64_t* tree, float scale, const float* lse, const float* weight, float decay, lk_stream_t stream) {
    if (!c) return LK_ERR_ARG;
    TreeParams p{};
    if (int rc = tree_params(c, cache, q, q_token, q_head, T, H, starts, tree, scale, &p)) return rc;
    if (!p.kv.mass) return set_err(c, LK_ERR_ARG, "the cache has no mass array");
    if (!(decay >= 0.0f && decay <= 1.0f)) return set_err(c, LK_ERR_ARG, "decay must be in [0, 1]");
    if (T == 0) return LK_OK;
    if (!lse) return set_err(c, LK_ERR_ARG, "null lse");
    OnDevice on(c->device);
    p.lse = const_cast<float*>(lse); p.weight = weight; p.decay = decay;
    CUtensorMap map, q_map;
    if (int rc = kv_map(c, cache, &map)) return rc;
    // dimensions from the smaller stride to the larger; one of a single entry has no stride of its own
    const int64_t head = H > 1 ? q_head : AT_ROW, token = T > 1 ? q_token : head * H;
    if (head <= 0 || token <= 0) return set_err(c, LK_ERR_UNSUPPORTED, "q strides (%lld, %lld) must be positive", (long long)q_token, (long long)q_head);
    p.q_head_major = token < head;
    const int64_t dims[3] = { AT_ROW, p.q_head_major ? T : H, p.q_head_major ? H : T }, strides[2] = { p.q_head_major ? token : head, p.q_head_major ? head : token };
    if (int rc = encode_map(c, &q_map, cache->dtype, q, 3, dims, strides, mass_q_box(H), p.q_head_major ? 2 : 1)) return rc;
    LK_CU(launch_mass(p, cache->dtype, map, q_map, c->mass, c->nsm / 2, (cudaStream_t)stream));
    return LK_OK;
}

int lk_attn_evict(LkAttnCtx* c, const LkKvCache* cache, int budget, int sinks, int recent, const int* next_pos, int* new_lens,
                  lk_stream_t stream) {
    if (!c) return LK_ERR_ARG;
    EvictParams p{};
    if (int rc = check_cache(c, cache, &p.kv)) return rc;
    if (!p.kv.mass || !p.kv.pos) return set_err(c, LK_ERR_ARG, "eviction needs the cache's mass and pos");
    if (budget < 1 || sinks < 0 || recent < 0) return set_err(c, LK_ERR_ARG, "budget %d, sinks %d, recent %d", budget, sinks, recent);
    if (!next_pos || !new_lens) return set_err(c, LK_ERR_ARG, "null next_pos or new_lens");
    OnDevice on(c->device);
    const int64_t cap = (int64_t)p.kv.table_stride * p.kv.page_size;
    p.region = cap > budget ? (cap - budget < budget ? cap - budget : budget) : 0;      // most rows that one sequence can move
    const int64_t need = 2 * p.region * p.kv.n_seqs;
    if (need > c->moves_cap) {
        if (int rc = may_allocate(c, (cudaStream_t)stream)) return rc;
        int64_t cap2 = 1024;
        while (cap2 < need) cap2 *= 2;
        LK_CU(cudaMalloc((void**)&c->moves[c->n_lists], cap2 * sizeof(int)));
        ++c->n_lists;
        c->moves_cap = cap2;
    }
    p.budget = budget; p.sinks = sinks; p.recent = recent; p.next_pos = next_pos; p.new_lens = new_lens;
    p.src = c->n_lists ? c->moves[c->n_lists - 1] : nullptr; p.dst = p.src + p.region * p.kv.n_seqs; p.n_moves = c->n_moves; p.err = c->err;
    LK_CU(launch_evict(p, c->nsm, (cudaStream_t)stream));
    return LK_OK;
}

}  // extern "C"
