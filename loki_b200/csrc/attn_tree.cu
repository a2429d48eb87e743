// attn_tree.cu -- attention of drafted token trees over the paged latent cache.
//
// S = scale * Q K^T with K the 576-wide rows, P = softmax(S) over the rows a token sees, O = P C with C the first 512
// values of the same rows.  One pass over the cache with a running maximum m and sum l per row: on a new tile
// m' = max(m, max S), O and l scale by exp(m - m'), P = exp(S - m').
//
// One CTA per (token, 16 heads): the rows of one token share its cache rows and its mask.  Keys in tiles of 32.
#include "attn_internal.h"

namespace lk {

constexpr int TS_H = 16, TS_K = 32, TS_THREADS = 256;
constexpr int TS_SMEM = TS_H * AT_ROW * 4 + TS_K * (AT_ROW + 2) * 4 + TS_H * (TS_K + 1) * 4 + 3 * TS_H * 4 + TS_K * 4;

template <class T>
__global__ void __launch_bounds__(TS_THREADS) k_tree(TreeParams p) {
    extern __shared__ float sm[];
    float* Q = sm;                                   // [16][576]
    float* K = Q + TS_H * AT_ROW;                    // [32][578]
    float* P = K + TS_K * (AT_ROW + 2);              // [16][33]
    float* M = P + TS_H * (TS_K + 1);                // running maximum, sum, and this tile's rescale
    float* L = M + TS_H;
    float* F = L + TS_H;
    int* slot = (int*)(F + TS_H);
    const int t = blockIdx.x, h0 = blockIdx.y * TS_H, tid = threadIdx.x;
    int b = -1, len = 0, j = 0, n = 0;
    for (int s = 0; s < p.kv.n_seqs; ++s) {
        if (t < p.starts[s] || t >= p.starts[s + 1]) continue;
        len = kv_len(p.kv, s, p.err);
        const int2 sp = seq_tokens(p.starts, s, p.T, len, p.kv, p.err);
        if (sp.y) { b = s; j = t - sp.x; n = sp.y; }
        break;
    }
    if (b < 0 && tid == 0) att_error(p.err, ATT_ERR_TREE);
    const uint64_t mask = b >= 0 ? node_mask(p.tree, t, j, n) : 0;
    const int total = b >= 0 ? len + n : 0;
    for (int i = tid; i < TS_H * AT_ROW; i += TS_THREADS) {
        const int h = h0 + i / AT_ROW;
        Q[i] = h < p.H ? to_f<T>(((const T*)p.q)[t * p.q_token + h * p.q_head + i % AT_ROW]) : 0.0f;
    }
    if (tid < TS_H) { M[tid] = -INFINITY; L[tid] = 0.0f; }
    float o[TS_H][2];
    #pragma unroll
    for (int h = 0; h < TS_H; ++h) o[h][0] = o[h][1] = 0.0f;
    for (int k0 = 0; k0 < total; k0 += TS_K) {
        __syncthreads();
        if (tid < TS_K) {
            const int i = k0 + tid;
            const bool see = i < len || (i < total && ((mask >> (i - len)) & 1));
            slot[tid] = see ? kv_slot(p.kv, b, i, p.err) : -1;
        }
        __syncthreads();
        for (int i = tid; i < TS_K * AT_ROW; i += TS_THREADS) {
            const int r = i / AT_ROW, c = i % AT_ROW;
            K[r * (AT_ROW + 2) + c] = slot[r] < 0 ? 0.0f : to_f<T>(((const T*)p.kv.rows)[(int64_t)slot[r] * p.kv.row_stride + c]);
        }
        __syncthreads();
        for (int i = tid; i < TS_H * TS_K; i += TS_THREADS) {
            const int h = i / TS_K, r = i % TS_K;
            float s = 0.0f;
            for (int c = 0; c < AT_ROW; ++c) s += Q[h * AT_ROW + c] * K[r * (AT_ROW + 2) + c];
            P[h * (TS_K + 1) + r] = slot[r] < 0 ? -INFINITY : s * p.scale;
        }
        __syncthreads();
        if (tid < TS_H) {
            float m = M[tid];
            for (int r = 0; r < TS_K; ++r) m = fmaxf(m, P[tid * (TS_K + 1) + r]);
            const float f = m == -INFINITY ? 1.0f : expf(M[tid] - m);
            float l = L[tid] * f;
            for (int r = 0; r < TS_K; ++r) {
                const float s = P[tid * (TS_K + 1) + r], e = s == -INFINITY ? 0.0f : expf(s - m);
                P[tid * (TS_K + 1) + r] = e;
                l += e;
            }
            M[tid] = m; L[tid] = l; F[tid] = f;
        }
        __syncthreads();
        #pragma unroll
        for (int h = 0; h < TS_H; ++h) { o[h][0] *= F[h]; o[h][1] *= F[h]; }
        for (int r = 0; r < TS_K; ++r) {
            const float c0 = K[r * (AT_ROW + 2) + 2 * tid], c1 = K[r * (AT_ROW + 2) + 2 * tid + 1];
            #pragma unroll
            for (int h = 0; h < TS_H; ++h) { o[h][0] += P[h * (TS_K + 1) + r] * c0; o[h][1] += P[h * (TS_K + 1) + r] * c1; }
        }
    }
    __syncthreads();
    for (int h = 0; h < TS_H && h0 + h < p.H; ++h) {
        const float l = L[h], inv = l == 0.0f ? 0.0f : 1.0f / l;
        T* out = (T*)p.out + t * p.out_token + (h0 + h) * p.out_head;
        out[2 * tid] = from_f<T>(o[h][0] * inv);
        out[2 * tid + 1] = from_f<T>(o[h][1] * inv);
        if (tid == 0 && p.lse) p.lse[(int64_t)t * p.H + h0 + h] = l == 0.0f ? -INFINITY : M[h] + logf(l);
    }
}

template <class T>
static cudaError_t tree_go(const TreeParams& p, cudaStream_t st) {
    cudaError_t e = cudaFuncSetAttribute(k_tree<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, TS_SMEM);
    if (e != cudaSuccess) return e;
    k_tree<T><<<dim3(p.T, (p.H + TS_H - 1) / TS_H), TS_THREADS, TS_SMEM, st>>>(p);
    return cudaGetLastError();
}

cudaError_t launch_tree(const TreeParams& p, int dtype, int, cudaStream_t st) {
    return dtype == LK_DT_F16 ? tree_go<__half>(p, st) : tree_go<__nv_bfloat16>(p, st);
}

}  // namespace lk
