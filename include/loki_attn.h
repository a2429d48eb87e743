/* loki_attn.h -- the latent-cache side of a DeepSeek-R1 attention layer next to the MoE half: rotary positions,
 * the paged latent cache, attention of drafted token trees over it, the attention weight that each cached row
 * has received, and eviction by that weight.  Device-pointer C ABI of libloki_moe.so.
 *
 * Every pointer argument is a device pointer unless stated otherwise; work is queued on the caller's stream and
 * the calls do not synchronise (lk_attn_get_error does).  Return values are the LK_* status codes of loki_moe.h;
 * no call exits the process.  A context belongs to one device, as do all pointers of its calls, and holds the workspaces of
 * its calls, so calls on one context are issued to one stream at a time (or ordered by events); contexts are independent.
 * A captured call keeps the workspaces that it was captured with: the context outlives the graph, and later calls of any size
 * leave them as they are.
 *
 * One cached row is 576 values: the 512-wide latent c, which is the key's first part and the value, and 64
 * rotated key values.  The query of one (token, head) row has the same 576 values (the head's query already
 * multiplied into the latent space, then its rotated part).  The reference keeps the same row and computes the
 * same products one token at a time (src/fused_layer.cu:277-308, src/attn_core_tc.cuh:17-76); the tree, the
 * pages, the accumulated weight and the eviction have no counterpart there.
 */
#ifndef LOKI_ATTN_H
#define LOKI_ATTN_H
#include "loki_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

#define LK_ATTN_LATENT 512
#define LK_ATTN_ROPE 64
#define LK_ATTN_ROW 576
#define LK_ATTN_MAX_HEADS 128
#define LK_ATTN_MAX_NODES 64       /* drafted tokens per sequence and call */
#define LK_ATTN_MAX_SEQS 512

enum { LK_DT_F32 = 0, LK_DT_F16 = 1, LK_DT_BF16 = 2 };
enum { LK_ROPE_INTERLEAVED = 0, LK_ROPE_HALF = 1 };     /* pairs (2i, 2i+1), or (i, i + rot_dim/2) */

typedef struct LkAttnCtx LkAttnCtx;

typedef struct LkAttnConfig {
    int max_seqs;       /* sequences per call, <= LK_ATTN_MAX_SEQS */
    int max_tokens;     /* drafted tokens per lk_attn_tree / lk_attn_mass call, all sequences together */
} LkAttnConfig;

/* Rotation frequencies base^(-2i/rot_dim).  factor > 1 stretches the context factor-fold: frequency i keeps its
 * value where it makes more than beta_fast turns over orig_ctx positions, is divided by factor where it makes
 * fewer than beta_slow, and is a linear mix (in i) between.  cos and sin are multiplied by mscale. */
typedef struct LkRopeConfig {
    int rot_dim;                       /* even */
    double base, factor;               /* factor 1: no stretching (the fields below are not read) */
    int orig_ctx;
    double beta_fast, beta_slow;
    double mscale;
} LkRopeConfig;

/* The paged cache of n_seqs sequences.  Row i of sequence b is pool row
 * block_table[b * table_stride + i / page_size] * page_size + i % page_size.  Sequences may share pages where a call only
 * reads rows (lk_attn_tree); lk_attn_append, lk_attn_mass and lk_attn_evict write what their sequences' pages hold.  With the
 * heads shared out over GPUs, lk_attn_mass gives a GPU the share of its heads: sum mass over the GPUs before lk_attn_evict, or
 * each keeps other rows. */
typedef struct LkKvCache {
    void* rows;                        /* [n_pages * page_size] rows, 16-byte aligned */
    int64_t row_stride;                /* elements from one row to the next: >= 576 and a multiple of 8 */
    int dtype;                         /* LK_DT_F16 or LK_DT_BF16 */
    int page_size;                     /* 16, 32, 64, 128 or 256 */
    int n_pages;
    const int* block_table;            /* [n_seqs][table_stride] page ids */
    int table_stride;
    int n_seqs;
    const int* lens;                   /* [n_seqs] rows of context (drafted rows follow them and are not counted) */
    float* mass;                       /* optional [n_pages * page_size]: accumulated attention weight per pool row */
    int* pos;                          /* optional [n_pages * page_size]: position of the token in each pool row */
} LkKvCache;

LK_API int  lk_attn_create(const LkAttnConfig* cfg, int device, LkAttnCtx** out);
LK_API void lk_attn_destroy(LkAttnCtx* ctx);
/* synchronise `stream`, then read and clear the context's device error word (a bad page id, position, length or
 * tree, or a bounded wait that ran out; the kernels skip or clamp what they refuse, and never read out of range) */
LK_API int  lk_attn_get_error(LkAttnCtx* ctx, lk_stream_t stream);
LK_API const char* lk_attn_last_error(LkAttnCtx* ctx);

/* cos and sin of positions 0 .. max_pos-1 into table [max_pos][rot_dim/2][2] fp32; the angles are computed in 64
 * bits (an fp32 angle at position 1e5 is off by 4e-3) and reduced there.  On the current device; ctx may be null (it
 * only takes the message of a refusal) */
LK_API int lk_attn_rope_table(LkAttnCtx* ctx, const LkRopeConfig* cfg, int max_pos, float* table, lk_stream_t stream);

/* y = x [T][H][head_dim] with elements [rot_offset, rot_offset + rot_dim) of every head rotated to position
 * pos[t]; the other elements are copied (y == x rotates in place).  grad != 0 applies the transpose: the gradient
 * of x from the gradient of y.  Strides in elements; dtype of x and y: any LK_DT_*, the rotation is fp32. */
LK_API int lk_attn_rope(LkAttnCtx* ctx, int dtype, const void* x, int64_t x_token, int64_t x_head, void* y, int64_t y_token,
                        int64_t y_head, int T, int H, int head_dim, int rot_offset, int rot_dim, int layout, int grad,
                        const int* pos, const float* table, int max_pos, lk_stream_t stream);

/* New rows: tokens starts[b] .. starts[b+1]-1 of latent [T][512] (row stride latent_ld) and k_rope [T][64] (not yet
 * rotated, row stride rope_ld), both in_dtype, become rows lens[b], lens[b]+1, .. of sequence b: the latent, then
 * k_rope rotated to pos[t].  cache->pos receives the positions and cache->mass zeros, where given.  The table is
 * for rot_dim 64.  lens is not advanced: the caller does that once the rows are accepted. */
LK_API int lk_attn_append(LkAttnCtx* ctx, const LkKvCache* cache, int in_dtype, const void* latent, int64_t latent_ld,
                          const void* k_rope, int64_t rope_ld, int T, const int* starts, const int* pos, const float* table,
                          int max_pos, int layout, lk_stream_t stream);

/* Attention of the drafted tokens starts[b] .. starts[b+1]-1 (n_b <= LK_ATTN_MAX_NODES) of every sequence b, whose rows
 * follow its context (lk_attn_append): token t, head h of q [T][H][576] (cache->dtype) attends to the lens[b] context
 * rows and to drafted row j where bit j of tree[t] is set.
 *   out[t][h] = sum_k p_k c_k,  p = softmax(scale * q . row_k),  lse[t][h] = ln sum_k exp(scale * q . row_k)
 * A row that sees nothing gives out = 0, lse = -inf; a row that it does not see never reaches it, whatever it holds.
 * Tokens that are in no sequence's range (before starts[0], or from starts[n_seqs] on) have their out and lse left as they are.
 * tree null: every token sees the drafted rows up to its own (a plain chain).  One token per sequence and tree null is
 * ordinary decoding.  out [T][H][512] in cache->dtype, lse [T][H] fp32 (optional).  Strides in elements, multiples of 8. */
LK_API int lk_attn_tree(LkAttnCtx* ctx, const LkKvCache* cache, const void* q, int64_t q_token, int64_t q_head, int T, int H,
                        const int* starts, const uint64_t* tree, float scale, void* out, int64_t out_token, int64_t out_head,
                        float* lse, lk_stream_t stream);

/* cache->mass[row k] = decay * mass + sum_t weight[t] * sum_h exp(scale * q . row_k - lse[t][h]) for every row of every
 * sequence (context and drafted), over the tokens that see it: the attention weight that lk_attn_tree gave it (sequences
 * without tokens keep theirs).  weight [T] (null: all 1; 0 for rejected drafts: only tokens of positive weight count).
 * Each row's terms are added in a fixed order, so results repeat.  q's strides must be positive here (heads or tokens that a
 * stride of 0 repeats are refused; lk_attn_tree takes them). */
LK_API int lk_attn_mass(LkAttnCtx* ctx, const LkKvCache* cache, const void* q, int64_t q_token, int64_t q_head, int T, int H,
                        const int* starts, const uint64_t* tree, float scale, const float* lse, const float* weight,
                        float decay, lk_stream_t stream);

/* Cuts every sequence longer than `budget` rows to its `budget` best: first the protected rows (position < sinks, or
 * position >= next_pos[b] - recent), then those of the largest mass; equal ones in row order, a NaN mass last.  The kept
 * rows at or beyond `budget` move, in order, into the holes before it (row, mass and pos); nothing else is written.
 * new_lens [n_seqs] receives min(lens, budget) and may be the cache's lens array itself.  Needs cache->mass and pos.
 * Rows need no order: each key carries its position in its rotated part, and pos tells it.
 * The move lists are made on the first call that needs ones of their size, so not under capture; a captured call keeps its own. */
LK_API int lk_attn_evict(LkAttnCtx* ctx, const LkKvCache* cache, int budget, int sinks, int recent, const int* next_pos,
                         int* new_lens, lk_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif
