// attn_rope.cu -- rotary positions on part of a head, and the rotate-and-append of new rows to the paged latent cache.
//
// y_a = m (cos t x_a - sin t x_b), y_b = m (sin t x_a + cos t x_b) for the pair (a, b) = (2i, 2i+1) (interleaved) or
// (i, i + R/2) (half), t = pos * f_i; the transpose (the gradient) negates sin.  Both only move data: 3 operations
// per rotated value against one load and one store, so HBM (or, for a decode step's few KB, the launch) bounds them.
// cos and sin come from a table made once in 64 bits: an fp32 product pos * f_i is off by half an ulp of the angle,
// 4e-3 at position 1e5, and sin/cos in the kernel would cost more than the rotation.
#include <math.h>
#include "attn_internal.h"
#include "attn_tc.cuh"
#include "moe_internal.h"

namespace lk {

// N elements of T moved as one 4-, 8- or 16-byte access
template <class T, int N> struct alignas(sizeof(T) * N) Vec { T v[N]; };

// ---------------------------------------------------------------- table
__global__ void __launch_bounds__(256) k_rope_table(LkRopeConfig c, double lo, double hi, int max_pos, float2* __restrict__ table) {
    const int half = c.rot_dim / 2;
    const int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (idx >= (int64_t)max_pos * half) return;
    const int i = (int)(idx % half);
    double f = pow(c.base, -2.0 * i / c.rot_dim);
    if (c.factor > 1.0) {
        const double r = fmin(fmax((i - lo) / fmax(hi - lo, 1e-3), 0.0), 1.0);
        f = f * (1.0 - r) + f / c.factor * r;
    }
    double s, co;
    sincos((double)(idx / half) * f, &s, &co);
    table[idx] = make_float2((float)(co * c.mscale), (float)(s * c.mscale));
}

cudaError_t launch_rope_table(const LkRopeConfig& c, int max_pos, float2* table, cudaStream_t st) {
    double lo = 0, hi = 0;
    if (c.factor > 1.0) {       // the (real) frequency index that makes `turns` turns over the original context
        auto at = [&](double turns) { return c.rot_dim * log(c.orig_ctx / (turns * 2 * M_PI)) / (2 * log(c.base)); };
        lo = fmax(0.0, floor(at(c.beta_fast)));
        hi = fmin(c.rot_dim - 1.0, ceil(at(c.beta_slow)));
    }
    const int64_t n = (int64_t)max_pos * (c.rot_dim / 2);
    k_rope_table<<<(unsigned)((n + 255) / 256), 256, 0, st>>>(c, lo, hi, max_pos, table);
    return cudaGetLastError();
}

__device__ __forceinline__ int checked_pos(int pos, int max_pos, int* err) {
    if ((unsigned)pos < (unsigned)max_pos) return pos;
    att_error(err, ATT_ERR_POS);
    return pos < 0 ? 0 : max_pos - 1;
}

// V pairs: interleaved, a holds the first V elements of 2V consecutive ones and b the rest; half, a and b are the
// pairs' two sides
template <int V, int LAYOUT>
__device__ __forceinline__ void rotate(float (&a)[V], float (&b)[V], const float2* __restrict__ cs, float sign) {
    #pragma unroll
    for (int i = 0; i < V; ++i) {
        const float2 t = __ldg(cs + i);
        const float s = sign * t.y;
        if (LAYOUT == LK_ROPE_HALF) {
            const float x = a[i], y = b[i];
            a[i] = t.x * x - s * y;
            b[i] = s * x + t.x * y;
        } else {
            float& p = 2 * i < V ? a[2 * i] : b[2 * i - V];
            float& q = 2 * i + 1 < V ? a[2 * i + 1] : b[2 * i + 1 - V];
            const float x = p, y = q;
            p = t.x * x - s * y;
            q = s * x + t.x * y;
        }
    }
}

// ---------------------------------------------------------------- rope
// A unit is V pairs of the rotated part, or V copied elements; V elements are one 16-byte access (V = 1 where the
// head's geometry, a stride or a pointer is not a multiple of that).  A thread takes N units a block apart and loads them all
// before it stores: 805 MB (fp32, 4096 tokens x 128 heads x 192, half pairs) take 130 us a call among others (6.2 TB/s, 95 % of a
// copy's rate), 124 in a graph.
template <class T, int V, int LAYOUT, int N>
__global__ void __launch_bounds__(256) k_rope(RopeParams p, int units, int blocks_per_token) {
    const int t = blockIdx.x / blocks_per_token, rot_units = p.rot / 2 / V;
    const int idx0 = (blockIdx.x - t * blocks_per_token) * (blockDim.x * N) + threadIdx.x;
    using Vt = Vec<T, V>;
    const T* x = (const T*)p.x + t * p.x_token;
    T* y = (T*)p.y + t * p.y_token;
    Vt va[N], vb[N];
    int h[N], ea[N], u[N];
    pdl_wait();
    pdl_trigger();
    #pragma unroll
    for (int k = 0; k < N; ++k) {
        const int idx = idx0 + k * blockDim.x;
        h[k] = idx / units;
        u[k] = idx - h[k] * units;
        if (h[k] >= p.H) continue;
        const T* xh = x + h[k] * p.x_head;
        if (u[k] < rot_units) {
            ea[k] = p.off + (LAYOUT == LK_ROPE_HALF ? u[k] * V : 2 * u[k] * V);
            vb[k] = *(const Vt*)(xh + ea[k] + (LAYOUT == LK_ROPE_HALF ? p.rot / 2 : V));
        } else {
            ea[k] = (u[k] - rot_units) * V;
            if (ea[k] >= p.off) ea[k] += p.rot;
        }
        va[k] = *(const Vt*)(xh + ea[k]);
    }
    const float2* cs = p.table + (int64_t)checked_pos(p.pos[t], p.max_pos, p.err) * (p.rot / 2);
    #pragma unroll
    for (int k = 0; k < N; ++k) {
        if (h[k] >= p.H) continue;
        T* yh = y + h[k] * p.y_head;
        if (u[k] < rot_units) {
            float a[V], b[V];
            #pragma unroll
            for (int i = 0; i < V; ++i) { a[i] = to_f<T>(va[k].v[i]); b[i] = to_f<T>(vb[k].v[i]); }
            rotate<V, LAYOUT>(a, b, cs + u[k] * V, p.grad ? -1.0f : 1.0f);
            #pragma unroll
            for (int i = 0; i < V; ++i) { va[k].v[i] = from_f<T>(a[i]); vb[k].v[i] = from_f<T>(b[i]); }
            *(Vt*)(yh + ea[k] + (LAYOUT == LK_ROPE_HALF ? p.rot / 2 : V)) = vb[k];
        }
        *(Vt*)(yh + ea[k]) = va[k];
    }
}

template <class T, int V, int N>
static cudaError_t rope_n(const RopeParams& p, int layout, cudaStream_t st) {
    const int units = p.rot / 2 / V + (p.copy ? (p.head_dim - p.rot) / V : 0), all = p.H * units;
    const int threads = all >= 256 * N ? 256 : ((all + N - 1) / N + 31) / 32 * 32;
    const int bpt = (all + threads * N - 1) / (threads * N);
    if (layout == LK_ROPE_HALF) return launch_pdl_n(k_rope<T, V, LK_ROPE_HALF, N>, dim3(p.T * bpt), dim3(threads), 0, st, p, units, bpt);
    return launch_pdl_n(k_rope<T, V, LK_ROPE_INTERLEAVED, N>, dim3(p.T * bpt), dim3(threads), 0, st, p, units, bpt);
}

// Units a thread, both sides measured (interleaved / half pairs, 192-wide heads of which 64 rotate, a call in a graph):
// 16-byte units of 16-bit types: one, at every size (4096 x 128 heads 98 / 109 us, with four 175 / 179; 64 x 128 3.7 / 3.3, 5.5 / 5.6).
// Others: four from 64 tokens on.  fp32 142 / 124 us for 4096 x 128 (one: 146 / 147), 12.3 / 11.3 for 1024 x 32 (10.3 / 10.3), 4.2 / 4.3 for
// 64 x 128 (3.9 / 3.9); single elements (heads of 193) 277 / 272 for 4096 x 128 in bf16 (375 / 383), 6.2 / 6.3 for 64 x 128 (7.3 / 7.4).
template <class T, int V>
static cudaError_t rope_go(const RopeParams& p, int layout, cudaStream_t st) {
    if constexpr (V == 8) return rope_n<T, V, 1>(p, layout, st);
    else return p.T < 64 ? rope_n<T, V, 1>(p, layout, st) : rope_n<T, V, 4>(p, layout, st);
}

template <class T>
static cudaError_t rope_type(const RopeParams& p, int layout, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const bool wide = p.off % V == 0 && p.rot % (2 * V) == 0 && p.head_dim % V == 0 && p.x_token % V == 0 && p.x_head % V == 0 &&
                      p.y_token % V == 0 && p.y_head % V == 0 && !(((uintptr_t)p.x | (uintptr_t)p.y) & 15);
    return wide ? rope_go<T, V>(p, layout, st) : rope_go<T, 1>(p, layout, st);
}

cudaError_t launch_rope(const RopeParams& p, int dtype, int layout, cudaStream_t st) {
    switch (dtype) {
        case LK_DT_F32: return rope_type<float>(p, layout, st);
        case LK_DT_F16: return rope_type<__half>(p, layout, st);
        default: return rope_type<__nv_bfloat16>(p, layout, st);
    }
}

// ---------------------------------------------------------------- append
// One thread per 8 latent values (64 of them) or 8 rotated pairs (4): 68 units a token.  8 x 1024 bf16 rows take 7.2 us a call,
// 3.2 of them the bytes: the launch and the chain of loads from starts to page are the rest (8.3 with the values loaded after it).
// fp32 rows 9.5, 4.6 of them the bytes; up to 64 rows 2.7 in a graph.
constexpr int AP_UNITS = AT_LATENT / 8 + AT_ROPE / 16;

template <class T> __device__ __forceinline__ void store8(T* dst, const float (&v)[8]) {
    Vec<T, 8> w;
    #pragma unroll
    for (int i = 0; i < 8; ++i) w.v[i] = from_f<T>(v[i]);
    *(Vec<T, 8>*)dst = w;
}

template <class TI, class TO, int LAYOUT>
__global__ void __launch_bounds__(256) k_append(AppendParams p) {
    const int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int t = (int)(idx / AP_UNITS), u = (int)(idx % AP_UNITS);
    if (t >= p.T) return;
    pdl_wait();
    pdl_trigger();
    // the values first: their loads run under the search for their place.  u < 64: 8 of the latent in x; else 8 pairs in x and y
    const int r = u - AT_LATENT / 8;
    const int ea = LAYOUT == LK_ROPE_HALF ? 8 * r : 16 * r, eb = ea + (LAYOUT == LK_ROPE_HALF ? AT_ROPE / 2 : 8);
    const TI* src = r < 0 ? (const TI*)p.latent + t * p.latent_ld + u * 8 : (const TI*)p.k_rope + t * p.rope_ld + ea;
    constexpr int N = 16 / sizeof(TI);
    Vec<TI, N> x[8 / N], y[8 / N];
    #pragma unroll
    for (int k = 0; k < 8 / N; ++k) x[k] = ((const Vec<TI, N>*)src)[k];
    if (r >= 0)
        #pragma unroll
        for (int k = 0; k < 8 / N; ++k) y[k] = ((const Vec<TI, N>*)(src + (eb - ea)))[k];
    const int pos = p.pos[t];
    int b = 0;                                   // the sequence: last b with starts[b] <= t
    for (int lo = 0, hi = p.kv.n_seqs - 1; lo <= hi;) {
        const int mid = (lo + hi) >> 1;
        if (p.starts[mid] <= t) { b = mid; lo = mid + 1; } else hi = mid - 1;
    }
    const int i = t - p.starts[b];
    if (i < 0 || t >= p.starts[b + 1]) { if (u == 0) att_error(p.err, ATT_ERR_TREE); return; }
    // a row beyond 2^31 wraps to a negative one, which no page holds
    const int slot = kv_slot(p.kv, b, (int)((unsigned)kv_len(p.kv, b, p.err) + (unsigned)i), p.err);
    if (slot < 0) return;
    TO* row = (TO*)p.kv.rows + (int64_t)slot * p.kv.row_stride;
    float v[8];
    #pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = to_f<TI>(x[k / N].v[k % N]);
    if (r < 0) {
        store8<TO>(row + u * 8, v);
        if (u == 0) {
            if (p.kv.pos) p.kv.pos[slot] = pos;
            if (p.kv.mass) p.kv.mass[slot] = 0.0f;
        }
        return;
    }
    float c[8];
    #pragma unroll
    for (int k = 0; k < 8; ++k) c[k] = to_f<TI>(y[k / N].v[k % N]);
    rotate<8, LAYOUT>(v, c, p.table + (int64_t)checked_pos(pos, p.max_pos, p.err) * (AT_ROPE / 2) + 8 * r, 1.0f);
    store8<TO>(row + AT_LATENT + ea, v);
    store8<TO>(row + AT_LATENT + eb, c);
}

template <class TI, class TO>
static cudaError_t append_go(const AppendParams& p, int layout, cudaStream_t st) {
    const unsigned grid = (unsigned)(((int64_t)p.T * AP_UNITS + 255) / 256);
    if (layout == LK_ROPE_HALF) return launch_pdl_n(k_append<TI, TO, LK_ROPE_HALF>, dim3(grid), dim3(256), 0, st, p);
    return launch_pdl_n(k_append<TI, TO, LK_ROPE_INTERLEAVED>, dim3(grid), dim3(256), 0, st, p);
}

cudaError_t launch_append(const AppendParams& p, int in_dtype, int kv_dtype, int layout, cudaStream_t st) {
    if (kv_dtype == LK_DT_F16)
        return in_dtype == LK_DT_F32 ? append_go<float, __half>(p, layout, st) : append_go<__half, __half>(p, layout, st);
    return in_dtype == LK_DT_F32 ? append_go<float, __nv_bfloat16>(p, layout, st)
                                 : append_go<__nv_bfloat16, __nv_bfloat16>(p, layout, st);
}

}  // namespace lk
