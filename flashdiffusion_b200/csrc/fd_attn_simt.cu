// Softmax attention on the CUDA cores: every type, stride, head size up to 256
// and length.  One warp owns one query row (forward, dq) or one key row of one
// key head (dk, dv) and walks over the other side 32 rows at a time: lane l
// evaluates the score of row l, then the 32 weights are broadcast and lane l
// accumulates coordinates l, l + 32, ... in fp32.  Masked pairs are skipped
// before their values are touched, so nothing in their memory matters.
#include "fd_attn.cuh"

namespace fd {
namespace attn {
namespace simt {

constexpr int WARPS = 4;
constexpr int MAXC = 8;   // coordinates per lane: dim <= 256

template <class T> __device__ __forceinline__ float up(T x);
template <> __device__ __forceinline__ float up<float>(float x) { return x; }
template <> __device__ __forceinline__ float up<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float up<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T> __device__ __forceinline__ T down(float x);
template <> __device__ __forceinline__ float down<float>(float x) { return x; }
template <> __device__ __forceinline__ __half down<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 down<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <class T>
__device__ __forceinline__ const T* row(const View& v, int b, int64_t s, int h) {
    return (const T*)v.p + b * v.sb + s * v.ss + h * v.sh;
}

template <class T>
__device__ __forceinline__ float dot(const float* a, const T* x, int dim) {
    float d = 0.f;
    for (int c = 0; c < dim; ++c) d = fmaf(a[c], up<T>(x[c]), d);
    return d;
}

// score and, for the gradient, d score / d (q.k) without the scale
__device__ __forceinline__ float score(const Prob& a, float d, float slope, int pos, int j, float* bend) {
    float s = a.scale * d;
    if (a.cap > 0.f) {
        const float t = tanhf(s / a.cap);
        s = a.cap * t;
        if (bend) *bend = 1.f - t * t;
    } else if (bend) {
        *bend = 1.f;
    }
    return s - slope * fabsf((float)(pos - j));
}

__device__ __forceinline__ float warp_max(float x) {
    for (int o = 16; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(~0u, x, o));
    return x;
}
__device__ __forceinline__ float warp_sum(float x) {
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
    return x;
}

template <class T>
__global__ void __launch_bounds__(WARPS * 32) forward_kernel(const Prob a) {
    __shared__ float sq[WARPS][256];
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t i = (int64_t)blockIdx.x * WARPS + w;
    const int h = blockIdx.y % a.heads, b = blockIdx.y / a.heads, hk = h / a.group;
    if (i >= a.q_len) return;
    const T* q = row<T>(a.q, b, i, h);
    for (int c = lane; c < a.dim; c += 32) sq[w][c] = up<T>(q[c]);
    __syncwarp();
    const int n = keys_of(a, b);
    const int2 sp = row_span(a, b, (int)i, n);
    const int pos = n - a.q_len + (int)i;
    const float slope = a.slopes ? a.slopes[h] : 0.f;
    float m = -INFINITY, l = 0.f, acc[MAXC] = {};
    for (int j0 = sp.x; j0 < sp.y; j0 += 32) {
        const int j = j0 + lane;
        const float s = j < sp.y ? score(a, dot(sq[w], row<T>(a.k, b, j, hk), a.dim), slope, pos, j, nullptr) : -INFINITY;
        const float mn = fmaxf(m, warp_max(s));
        const float base = mn == -INFINITY ? 0.f : mn;
        const float fix = expf(m - base), p = j < sp.y ? expf(s - base) : 0.f;
        m = mn;
        l = l * fix + p;
        const int most = min(32, sp.y - j0);
#pragma unroll
        for (int c = 0; c < MAXC; ++c) acc[c] *= fix;
        for (int t = 0; t < most; ++t) {
            const float pt = __shfl_sync(~0u, p, t);
            const T* v = row<T>(a.v, b, j0 + t, hk);
#pragma unroll
            for (int c = 0; c < MAXC; ++c)
                if (lane + 32 * c < a.dim) acc[c] = fmaf(pt, up<T>(v[lane + 32 * c]), acc[c]);
        }
    }
    l = warp_sum(l);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* o = (T*)row<T>(a.o, b, i, h);
#pragma unroll
    for (int c = 0; c < MAXC; ++c)
        if (lane + 32 * c < a.dim) o[lane + 32 * c] = down<T>(acc[c] * inv);
    if (a.lse && lane == 0) a.lse[((int64_t)b * a.heads + h) * a.q_len + i] = l == 0.f ? -INFINITY : m + logf(l);
}

template <class T>
__global__ void __launch_bounds__(WARPS * 32) delta_kernel(const Prob a, float* __restrict__ delta) {
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t i = (int64_t)blockIdx.x * WARPS + w;
    const int h = blockIdx.y % a.heads, b = blockIdx.y / a.heads;
    if (i >= a.q_len) return;
    const T *g = row<T>(a.d_o, b, i, h), *o = row<T>(a.o, b, i, h);
    float d = 0.f;
    for (int c = lane; c < a.dim; c += 32) d = fmaf(up<T>(g[c]), up<T>(o[c]), d);
    d = warp_sum(d);
    if (lane == 0) delta[((int64_t)b * a.heads + h) * a.q_len + i] = d;
}

template <class T>
__global__ void __launch_bounds__(WARPS * 32) dq_kernel(const Prob a, const float* __restrict__ delta) {
    __shared__ float sq[WARPS][256], sg[WARPS][256];
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t i = (int64_t)blockIdx.x * WARPS + w;
    const int h = blockIdx.y % a.heads, b = blockIdx.y / a.heads, hk = h / a.group;
    if (i >= a.q_len) return;
    const T *q = row<T>(a.q, b, i, h), *g = row<T>(a.d_o, b, i, h);
    for (int c = lane; c < a.dim; c += 32) {
        sq[w][c] = up<T>(q[c]);
        sg[w][c] = up<T>(g[c]);
    }
    __syncwarp();
    const int n = keys_of(a, b);
    const int2 sp = row_span(a, b, (int)i, n);
    const int pos = n - a.q_len + (int)i;
    const float slope = a.slopes ? a.slopes[h] : 0.f;
    const int64_t at = ((int64_t)b * a.heads + h) * a.q_len + i;
    const float lse = a.lse[at], dl = delta[at];
    float acc[MAXC] = {};
    for (int j0 = sp.x; j0 < sp.y && lse != -INFINITY; j0 += 32) {
        const int j = j0 + lane;
        float ds = 0.f;
        if (j < sp.y) {
            float bend;
            const float s = score(a, dot(sq[w], row<T>(a.k, b, j, hk), a.dim), slope, pos, j, &bend);
            ds = expf(s - lse) * (dot(sg[w], row<T>(a.v, b, j, hk), a.dim) - dl) * bend * a.scale;
        }
        const int most = min(32, sp.y - j0);
        for (int t = 0; t < most; ++t) {
            const float dt = __shfl_sync(~0u, ds, t);
            const T* k = row<T>(a.k, b, j0 + t, hk);
#pragma unroll
            for (int c = 0; c < MAXC; ++c)
                if (lane + 32 * c < a.dim) acc[c] = fmaf(dt, up<T>(k[lane + 32 * c]), acc[c]);
        }
    }
    T* o = (T*)row<T>(a.dq, b, i, h);
#pragma unroll
    for (int c = 0; c < MAXC; ++c)
        if (lane + 32 * c < a.dim) o[lane + 32 * c] = down<T>(acc[c]);
}

template <class T>
__global__ void __launch_bounds__(WARPS * 32) dkv_kernel(const Prob a, const float* __restrict__ delta) {
    __shared__ float sk[WARPS][256], sv[WARPS][256];
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t j = (int64_t)blockIdx.x * WARPS + w;
    const int hk = blockIdx.y % a.kv_heads, b = blockIdx.y / a.kv_heads;
    if (j >= a.k_len) return;
    const T *k = row<T>(a.k, b, j, hk), *v = row<T>(a.v, b, j, hk);
    for (int c = lane; c < a.dim; c += 32) {
        sk[w][c] = up<T>(k[c]);
        sv[w][c] = up<T>(v[c]);
    }
    __syncwarp();
    const int n = keys_of(a, b);
    float ak[MAXC] = {}, av[MAXC] = {};
    for (int i0 = 0; i0 < a.q_len; i0 += 32) {
        const int i = i0 + lane;
        bool see = false;
        if (i < a.q_len) {
            const int2 sp = row_span(a, b, i, n);
            see = j >= sp.x && j < sp.y;
        }
        const unsigned any = __ballot_sync(~0u, see);
        if (!any) continue;
        for (int g = 0; g < a.group; ++g) {
            const int h = hk * a.group + g;
            const float slope = a.slopes ? a.slopes[h] : 0.f;
            const int64_t at = ((int64_t)b * a.heads + h) * a.q_len + i;
            float p = 0.f, ds = 0.f;
            if (see && a.lse[at] != -INFINITY) {
                float bend;
                const float s = score(a, dot(sk[w], row<T>(a.q, b, i, h), a.dim), slope, n - a.q_len + i, (int)j, &bend);
                p = expf(s - a.lse[at]);
                ds = p * (dot(sv[w], row<T>(a.d_o, b, i, h), a.dim) - delta[at]) * bend * a.scale;
            }
            for (unsigned left = any; left; left &= left - 1) {
                const int t = __ffs(left) - 1;
                const float pt = __shfl_sync(~0u, p, t), dt = __shfl_sync(~0u, ds, t);
                const T *q = row<T>(a.q, b, i0 + t, h), *go = row<T>(a.d_o, b, i0 + t, h);
#pragma unroll
                for (int c = 0; c < MAXC; ++c)
                    if (lane + 32 * c < a.dim) {
                        ak[c] = fmaf(dt, up<T>(q[lane + 32 * c]), ak[c]);
                        av[c] = fmaf(pt, up<T>(go[lane + 32 * c]), av[c]);
                    }
            }
        }
    }
    T *dk = (T*)row<T>(a.dk, b, j, hk), *dv = (T*)row<T>(a.dv, b, j, hk);
#pragma unroll
    for (int c = 0; c < MAXC; ++c)
        if (lane + 32 * c < a.dim) {
            dk[lane + 32 * c] = down<T>(ak[c]);
            dv[lane + 32 * c] = down<T>(av[c]);
        }
}

inline dim3 grid_of(int rows, int heads, int batch) {
    return dim3((unsigned)cdiv(rows, WARPS), (unsigned)(heads * batch));
}

}  // namespace simt

#define FD_ATTN_TYPES(dtype, NAME, ...)                                        \
    switch (dtype) {                                                           \
        case FD_DTYPE_F16: { using T = __half; NAME(__VA_ARGS__); break; }       \
        case FD_DTYPE_BF16: { using T = __nv_bfloat16; NAME(__VA_ARGS__); break; } \
        default: { using T = float; NAME(__VA_ARGS__); }                         \
    }

int simt_forward(const Prob& a, int dtype, cudaStream_t s) {
#define GO() simt::forward_kernel<T><<<simt::grid_of(a.q_len, a.heads, a.batch), simt::WARPS * 32, 0, s>>>(a)
    FD_ATTN_TYPES(dtype, GO)
#undef GO
    FD_CUDA_TRY(cudaGetLastError());
    return FD_OK;
}

int launch_delta(const Prob& a, int dtype, float* delta, cudaStream_t s) {
#define GO() simt::delta_kernel<T><<<simt::grid_of(a.q_len, a.heads, a.batch), simt::WARPS * 32, 0, s>>>(a, delta)
    FD_ATTN_TYPES(dtype, GO)
#undef GO
    FD_CUDA_TRY(cudaGetLastError());
    return FD_OK;
}

int simt_backward(const Prob& a, int dtype, float* delta, cudaStream_t s) {
    if (a.q_len > 0) {
        FD_TRY(launch_delta(a, dtype, delta, s));
#define GO() simt::dq_kernel<T><<<simt::grid_of(a.q_len, a.heads, a.batch), simt::WARPS * 32, 0, s>>>(a, delta)
        FD_ATTN_TYPES(dtype, GO)
#undef GO
        FD_CUDA_TRY(cudaGetLastError());
    }
    if (a.k_len > 0) {
#define GO() simt::dkv_kernel<T><<<simt::grid_of(a.k_len, a.kv_heads, a.batch), simt::WARPS * 32, 0, s>>>(a, delta)
        FD_ATTN_TYPES(dtype, GO)
#undef GO
        FD_CUDA_TRY(cudaGetLastError());
    }
    return FD_OK;
}

}  // namespace attn
}  // namespace fd
