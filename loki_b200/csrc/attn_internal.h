// attn_internal.h -- parameter blocks, launchers and device helpers of the latent-cache attention operators.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <stdint.h>
#include "../../include/loki_attn.h"

namespace lk {

constexpr int AT_LATENT = LK_ATTN_LATENT, AT_ROPE = LK_ATTN_ROPE, AT_ROW = LK_ATTN_ROW;

// device error codes (beside the DEV_* of moe_device.cuh; first writer wins)
enum { ATT_ERR_PAGE = 16, ATT_ERR_POS = 17, ATT_ERR_LEN = 18, ATT_ERR_TREE = 19 };

// the cache as the kernels see it
struct KvView {
    void* rows; int64_t row_stride;
    int page_size, page_shift, n_pages, table_stride, n_seqs;
    const int* block_table; const int* lens;
    float* mass; int* pos;
};

// Launches.  Every kernel here is set up while the one before it in the stream ends (launch_pdl_n): it waits for that one before
// its first access to memory (pdl_wait), and only then lets the next be set up (pdl_trigger), so that a kernel never runs beside
// one two places before it.  2 us less a call of 10 to 100 us in a stream (append of 8 x 1024 rows 10.2 -> 8.3 us).
struct RopeParams {
    const void* x; int64_t x_token, x_head;
    void* y; int64_t y_token, y_head;
    int T, H, head_dim, off, rot, grad, copy;
    const int* pos; const float2* table; int max_pos;
    int* err;
};
cudaError_t launch_rope(const RopeParams& p, int dtype, int layout, cudaStream_t st);
cudaError_t launch_rope_table(const LkRopeConfig& c, int max_pos, float2* table, cudaStream_t st);

struct AppendParams {
    KvView kv;
    const void* latent; int64_t latent_ld;
    const void* k_rope; int64_t rope_ld;
    int T; const int* starts; const int* pos; const float2* table; int max_pos;
    int* err;
};
cudaError_t launch_append(const AppendParams& p, int in_dtype, int kv_dtype, int layout, cudaStream_t st);

struct TreeParams {
    KvView kv;
    const void* q; int64_t q_token, q_head;
    int T, H;
    const int* starts; const uint64_t* tree;
    float scale;                                   // score scale, natural units
    void* out; int64_t out_token, out_head;
    float* lse;                                    // tree: out; mass: in
    const float* weight; float decay;              // mass
    int q_flat;                                    // tree: q's rows (t, h) lie at equal distances
    int q_head_major;                              // mass: the dimensions of q's tensor map are (576, T, H), else (576, H, T)
    int* err;
};
// parts of items that more than one pair of CTAs works on (attn_tree.cu)
struct alignas(16) TreeSplit { int info, slot0, row0, first; };      // parts + 256 x this one's place among them + 65536 x rows; slot of the first part; first row, first token
struct TreeWork {
    float4* part;              // [2 per pair][16 groups of 8 rows][512 / 4][8 rows]: O, not yet divided by the sum
    float2* ml;                // [2 per pair][128 rows]: reference and sum
    TreeSplit* split;          // [2 per pair] the item that a part belongs to (info 0: no part)
};
int tree_pairs(int nsm);       // pairs of CTAs of a launch
// what a device needs once before the launches below (shared-memory sizes)
cudaError_t tree_setup();
cudaError_t mass_setup();
cudaError_t evict_setup();
// map, map16: the cache in boxes of up to 64 rows of a page, and of 16; q_map: q's T * H rows in boxes of 64, where p.q_flat
cudaError_t launch_tree(const TreeParams& p, int dtype, const CUtensorMap& map, const CUtensorMap& map16, const CUtensorMap& q_map, const TreeWork& wk, int pairs, cudaStream_t st);
int mass_q_box(int H);         // heads of a box of q's tensor map
// sums of key tiles that more than one pair of CTAs works on (attn_mass.cu): [2 per pair][256 keys], and for the tile that
// starts in a run the parts that have arrived, one counter a CTA, 0 between calls
struct MassWork { float* part; unsigned* arrived; };
cudaError_t launch_mass(const TreeParams& p, int dtype, const CUtensorMap& map, const CUtensorMap& q_map, const MassWork& wk, int pairs, cudaStream_t st);

struct EvictParams {
    KvView kv;
    int budget, sinks, recent;
    const int* next_pos; int* new_lens;
    int* src; int* dst; int* n_moves;              // [n_seqs][region] pool rows, [n_seqs]
    int64_t region;
    int keys;                                      // keys that a CTA of the selection keeps
    int* err;
};
cudaError_t launch_evict(const EvictParams& p, int nsm, cudaStream_t st);

// ---- device helpers
__device__ __forceinline__ void att_error(int* err, int code) { if (err) atomicCAS(err, 0, code); }

// rows of context of sequence b, refused values clamped (negative, or more than its pages hold)
__device__ __forceinline__ int kv_len(const KvView& kv, int b, int* err) {
    const int n = kv.lens[b], cap = kv.table_stride << kv.page_shift;
    if (n < 0 || n > cap) { att_error(err, ATT_ERR_LEN); return n < 0 ? 0 : cap; }
    return n;
}
// pool row of row i of sequence b; -1 (recorded) where its page id is not one of the pool's
__device__ __forceinline__ int kv_slot(const KvView& kv, int b, int i, int* err) {
    const int pi = i >> kv.page_shift;
    if ((unsigned)pi >= (unsigned)kv.table_stride) { att_error(err, ATT_ERR_LEN); return -1; }
    const int page = kv.block_table[(int64_t)b * kv.table_stride + pi];
    if ((unsigned)page >= (unsigned)kv.n_pages) { att_error(err, ATT_ERR_PAGE); return -1; }
    return (page << kv.page_shift) + (i & (kv.page_size - 1));
}
// the drafted tokens of sequence b: first token and count, refused ranges clamped to none
__device__ __forceinline__ int2 seq_tokens(const int* starts, int b, int T, int len, const KvView& kv, int* err) {
    const int s = starts[b], e = starts[b + 1];
    if (s < 0 || e < s || e > T || e - s > LK_ATTN_MAX_NODES) { att_error(err, ATT_ERR_TREE); return make_int2(0, 0); }
    if (e - s > (kv.table_stride << kv.page_shift) - len) { att_error(err, ATT_ERR_LEN); return make_int2(0, 0); }
    return make_int2(s, e - s);
}
// which drafted rows token j (of n) of a sequence sees
__device__ __forceinline__ uint64_t node_mask(const uint64_t* tree, int t, int j, int n) {
    const uint64_t all = n >= 64 ? ~0ull : (1ull << n) - 1;
    return all & (tree ? tree[t] : (j >= 63 ? ~0ull : (2ull << j) - 1));
}

template <class T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

}  // namespace lk
