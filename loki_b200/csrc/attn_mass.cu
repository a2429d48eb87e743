// attn_mass.cu -- the attention weight that every cached row received:
//   mass[k] = decay * mass[k] + sum_t w_t sum_h exp(scale q_th . row_k - lse_th).
// The sum runs over the rows of the score matrix, so the known lse lets each key add its terms alone: a CTA owns 32
// keys (one per lane), its warps share out the (token, head) rows, and the partial sums are added in a fixed order.
#include "attn_internal.h"

namespace lk {

constexpr int MS_K = 32, MS_WARPS = 8;
constexpr int MS_LD = AT_ROW + 1;

template <class T>
__global__ void __launch_bounds__(MS_WARPS * 32) k_mass(TreeParams p) {
    extern __shared__ float sm[];
    float* K = sm;                                  // [32][577]: lanes read one column of 32 rows without conflicts
    float* part = K + MS_K * MS_LD;                 // [8][32]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int item = blockIdx.x;                          // tiles of all sequences, numbered in order
    for (int b = 0; b < p.kv.n_seqs; ++b) {
        const int len = kv_len(p.kv, b, p.err);
        const int2 sp = seq_tokens(p.starts, b, p.T, len, p.kv, p.err);
        const int total = sp.y ? len + sp.y : 0, tiles = (total + MS_K - 1) / MS_K;
        for (; item < tiles; item += gridDim.x) {
            const int k0 = item * MS_K;
            __syncthreads();
            for (int r = warp; r < MS_K; r += MS_WARPS) {
                const int slot = k0 + r < total ? kv_slot(p.kv, b, k0 + r, p.err) : -1;
                for (int c = lane; c < AT_ROW; c += 32)
                    K[r * MS_LD + c] = slot < 0 ? 0.0f : to_f<T>(((const T*)p.kv.rows)[(int64_t)slot * p.kv.row_stride + c]);
            }
            __syncthreads();
            const int i = k0 + lane;
            float acc = 0.0f;
            for (int j = 0; j < sp.y; ++j) {
                const int t = sp.x + j;
                const float w = p.weight ? p.weight[t] : 1.0f;
                if (w == 0.0f) continue;
                const uint64_t mask = node_mask(p.tree, t, j, sp.y);
                const bool see = i < len || (i < total && ((mask >> (i - len)) & 1));
                float sum = 0.0f;
                for (int h = warp; h < p.H; h += MS_WARPS) {
                    const T* q = (const T*)p.q + t * p.q_token + h * p.q_head;
                    float s = 0.0f;
                    for (int c = 0; c < AT_ROW; ++c) s += to_f<T>(q[c]) * K[lane * MS_LD + c];
                    if (see) sum += expf(s * p.scale - p.lse[(int64_t)t * p.H + h]);
                }
                acc += w * sum;
            }
            part[warp * 32 + lane] = acc;
            __syncthreads();
            if (warp == 0 && i < total) {
                float a = 0.0f;
                for (int w = 0; w < MS_WARPS; ++w) a += part[w * 32 + lane];
                const int slot = kv_slot(p.kv, b, i, p.err);
                if (slot >= 0) p.kv.mass[slot] = p.decay * p.kv.mass[slot] + a;
            }
        }
        item -= tiles;
    }
}

template <class T>
static cudaError_t mass_go(const TreeParams& p, int nsm, cudaStream_t st) {
    constexpr int smem = (MS_K * MS_LD + MS_WARPS * 32) * 4;
    cudaError_t e = cudaFuncSetAttribute(k_mass<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    k_mass<T><<<2 * nsm, MS_WARPS * 32, smem, st>>>(p);
    return cudaGetLastError();
}

cudaError_t launch_mass(const TreeParams& p, int dtype, int nsm, cudaStream_t st) {
    return dtype == LK_DT_F16 ? mass_go<__half>(p, nsm, st) : mass_go<__nv_bfloat16>(p, nsm, st);
}

}  // namespace lk
