// Softmax attention on the CUDA cores: every type, stride, head size up to 256
// and length, in fp32.  The tensor-core kernels take 16-bit heads of a multiple of
// 8 coordinates, up to 256 forward and 128 backward; what is left comes here.
//
// A block of 256 threads holds a tile of rows of one side and walks over tiles of
// the other, both as fp32 in shared memory.  Thread (ty, tx) owns M x M scores,
// rows ty M .. and columns tx, tx + 16, ... , and of the output tile the same rows
// and columns 4 tx .. 4 tx + 3 of every 64: both products then read 16 bytes at a
// time, rows padded by 16 bytes, without bank conflicts, and are bound by the
// multiply-adds.  Forward and dq own query rows, dk and dv own key rows of one key
// head and sum over the query heads that share it: every sum has one owner and a
// fixed order.
//
// Measured, fp32, 2 x 2048 rows of 8 / 4 heads, causal: D = 64 360 us forward and 1490 us backward, D = 128 592 us
// (29 TFLOP/s) and 2600 us; the copies into shared memory are not overlapped with the products of the same block.
// One warp for each row without shared tiles took 10 and 37 ms, 18 and 70 ms.
//
// Masked places have the weight zero.  Zero times a NaN or an infinity there would
// reach the row, so a tile that holds one takes the product that asks for each
// pair whether it is seen.
#include <cooperative_groups.h>

#include <type_traits>

#include "fd_attn.cuh"
#include "fd_tc_common.cuh"

namespace fd {
namespace attn {
namespace simt {

namespace cg = cooperative_groups;

constexpr int THREADS = 256;
constexpr int WARPS = 8;
constexpr int MAXC = 8;   // coordinates per lane of a warp: dim <= 256

template <class T> __device__ __forceinline__ float up(T x);
template <> __device__ __forceinline__ float up<float>(float x) { return x; }
template <> __device__ __forceinline__ float up<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float up<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T> __device__ __forceinline__ T down(float x);
template <> __device__ __forceinline__ float down<float>(float x) { return x; }
template <> __device__ __forceinline__ __half down<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 down<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// four values at an address that is a multiple of four of them
__device__ __forceinline__ float4 up4(const float* p) { return *(const float4*)p; }
template <class T>
__device__ __forceinline__ float4 up4(const T* p) {
    const uint2 w = *(const uint2*)p;
    T v[4];
    memcpy(v, &w, 8);
    return make_float4(up<T>(v[0]), up<T>(v[1]), up<T>(v[2]), up<T>(v[3]));
}

template <class T>
__device__ __forceinline__ T* row(const View& v, int b, int64_t s, int h) {
    return (T*)v.p + b * v.sb + s * v.ss + h * v.sh;
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

__device__ __forceinline__ float warp_max(float x, int from = 16) {
    for (int o = from; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(~0u, x, o));
    return x;
}
__device__ __forceinline__ float warp_sum(float x, int from = 16) {
    for (int o = from; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
    return x;
}

// ---- tiles ------------------------------------------------------------------------------------------------------

template <int DP> constexpr int LD = DP + 4;          // floats of a tile row
template <int N> constexpr int LW = N + 4;            // floats of a row of N weights

// Rows r0 .. r0 + ROWS of one head as fp32, zeros behind row `rows` and coordinate dim; true if a value is not finite.
template <class T, int ROWS, int DP>
__device__ __forceinline__ bool load_tile(float* dst, const View& v, int b, int h, int r0, int rows, int dim, bool vec) {
    constexpr int PIECES = ROWS * DP / 4 / THREADS, AHEAD = 8;   // loads in flight
    static_assert(PIECES * THREADS * 4 == ROWS * DP && (PIECES % AHEAD == 0 || PIECES < AHEAD), "whole turns");
    constexpr int TURN = PIECES < AHEAD ? PIECES : AHEAD;
    bool bad = false;
#pragma unroll 1
    for (int x0 = threadIdx.x; x0 < ROWS * DP / 4; x0 += TURN * THREADS) {
        float4 f[TURN];
#pragma unroll
        for (int y = 0; y < TURN; ++y) {
            const int x = x0 + y * THREADS, r = x / (DP / 4), c = x % (DP / 4) * 4;
            f[y] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r0 + r >= rows || c >= dim) continue;
            const T* p = row<T>(v, b, r0 + r, h) + c;
            if (vec) {
                f[y] = up4(p);
            } else {
                f[y].x = up<T>(p[0]);
                if (c + 1 < dim) f[y].y = up<T>(p[1]);
                if (c + 2 < dim) f[y].z = up<T>(p[2]);
                if (c + 3 < dim) f[y].w = up<T>(p[3]);
            }
        }
#pragma unroll
        for (int y = 0; y < TURN; ++y) {
            const int x = x0 + y * THREADS, r = x / (DP / 4), c = x % (DP / 4) * 4;
            // 0 f is a NaN where f is not finite
            bad = bad || fmaf(0.f, f[y].x, 0.f * f[y].y) + fmaf(0.f, f[y].z, 0.f * f[y].w) != 0.f;
            *(float4*)(dst + r * LD<DP> + c) = f[y];
        }
    }
    return bad;
}

// s[i][j] = A[ty M + i] . B[tx + 16 j]
template <int M, int DP>
__device__ __forceinline__ void products(const float* A, const float* B, int dim, float (&s)[M][M]) {
    const float* pa = A + (threadIdx.x / 16) * M * LD<DP>;
    const float* pb = B + (threadIdx.x % 16) * LD<DP>;
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
        for (int j = 0; j < M; ++j) s[i][j] = 0.f;
#pragma unroll 4
    for (int d = 0; d < dim; d += 4) {
        float4 x[M], y[M];
#pragma unroll
        for (int i = 0; i < M; ++i) {
            x[i] = *(const float4*)(pa + i * LD<DP> + d);
            y[i] = *(const float4*)(pb + i * 16 * LD<DP> + d);
        }
#pragma unroll
        for (int i = 0; i < M; ++i)
#pragma unroll
            for (int j = 0; j < M; ++j)
                s[i][j] = fmaf(x[i].x, y[j].x, fmaf(x[i].y, y[j].y, fmaf(x[i].z, y[j].z, fmaf(x[i].w, y[j].w, s[i][j]))));
    }
}

// acc[i][c] += sum_j W[ty M + i][j] B[j][64 c + 4 tx ..]; `seen`(row, j) is asked only if `ask`
template <int M, int DP, class Seen>
__device__ __forceinline__ void accumulate(const float* W, const float* B, float4 (&acc)[M][DP / 64], bool ask, Seen seen) {
    constexpr int N = 16 * M;
    const float* pw = W + (threadIdx.x / 16) * M * LW<N>;
    const float* pb = B + (threadIdx.x % 16) * 4;
    auto add = [](float4& o, float w, const float4& v) {
        o.x = fmaf(w, v.x, o.x);
        o.y = fmaf(w, v.y, o.y);
        o.z = fmaf(w, v.z, o.z);
        o.w = fmaf(w, v.w, o.w);
    };
    if (ask) {
#pragma unroll 1
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int i = 0; i < M; ++i) {
                if (!seen((int)threadIdx.x / 16 * M + i, j)) continue;
#pragma unroll
                for (int c = 0; c < DP / 64; ++c) add(acc[i][c], pw[i * LW<N> + j], *(const float4*)(pb + j * LD<DP> + 64 * c));
            }
        return;
    }
#pragma unroll 2
    for (int j = 0; j < N; j += 4) {
        float w[M][4];
#pragma unroll
        for (int i = 0; i < M; ++i) {
            const float4 x = *(const float4*)(pw + i * LW<N> + j);
            w[i][0] = x.x;
            w[i][1] = x.y;
            w[i][2] = x.z;
            w[i][3] = x.w;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int c = 0; c < DP / 64; ++c) {
                const float4 v = *(const float4*)(pb + (j + e) * LD<DP> + 64 * c);
#pragma unroll
                for (int i = 0; i < M; ++i) add(acc[i][c], w[i][e], v);
            }
    }
}

template <class T>
__device__ __forceinline__ void store4(T* out, const float4& f, float by, int c, int dim) {
    const float v[4] = {f.x * by, f.y * by, f.z * by, f.w * by};
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (c + e < dim) out[c + e] = down<T>(v[e]);
}

// Spans of the N query rows from q0 on, and the keys [lo, hi) that any of them sees.
template <int N>
struct Rows {
    int first[N], end[N];
    int lo, hi;
    __device__ void fill(const Prob& a, int b, int q0, int n) {
        if (threadIdx.x == 0) {
            lo = 0x7fffffff;
            hi = 0;
        }
        __syncthreads();
        if (threadIdx.x < N) {
            const int i = q0 + (int)threadIdx.x;
            const int2 sp = i < a.q_len ? row_span(a, b, i, n) : make_int2(0, 0);
            first[threadIdx.x] = sp.x;
            end[threadIdx.x] = sp.y;
            if (sp.y > sp.x) {
                atomicMin(&lo, sp.x);
                atomicMax(&hi, sp.y);
            }
        }
        __syncthreads();
    }
    __device__ bool sees(int r, int key) const { return key >= first[r] && key < end[r]; }
};

struct Place {
    int tile, b, h;
    // the last tile first: it sees most keys under a causal mask
    __device__ Place(int heads, int batch) {
        const int nh = heads * batch, x = blockIdx.x % nh;
        tile = (int)(gridDim.x / nh) - 1 - blockIdx.x / nh;
        b = x / heads;
        h = x - b * heads;
    }
};

// Forward.  K and V of a tile take turns in one buffer, so that two blocks fit on an SM at D = 128.
template <class T, int DP>
__global__ void __launch_bounds__(THREADS, DP <= 128 ? 2 : 1) forward_kernel(const __grid_constant__ Prob a, bool vec) {
    constexpr int M = 4, N = 16 * M;
    extern __shared__ __align__(16) float smem[];
    float *sq = smem, *sk = sq + N * LD<DP>, *sp = sk + N * LD<DP>;
    __shared__ Rows<N> rows;
    const Place at(a.heads, a.batch);
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    const int b = at.b, h = at.h, hk = h / a.group, q0 = at.tile * N, n = keys_of(a, b);
    rows.fill(a, b, q0, n);
    load_tile<T, N, DP>(sq, a.q, b, h, q0, a.q_len, a.dim, vec);
    const float slope = a.slopes ? a.slopes[h] : 0.f;
    float m[M], l[M];
    float4 acc[M][DP / 64];
#pragma unroll
    for (int i = 0; i < M; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) acc[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int k0 = rows.lo & ~(N - 1); k0 < rows.hi; k0 += N) {
        load_tile<T, N, DP>(sk, a.k, b, hk, k0, n, a.dim, vec);
        __syncthreads();
        float s[M][M];
        products<M, DP>(sq, sk, a.dim, s);
        __syncthreads();
        const bool bad = load_tile<T, N, DP>(sk, a.v, b, hk, k0, n, a.dim, vec);
#pragma unroll
        for (int i = 0; i < M; ++i) {
            const int r = ty * M + i, pos = n - a.q_len + q0 + r;
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < M; ++j) {
                const int key = k0 + tx + 16 * j;
                s[i][j] = rows.sees(r, key) ? score(a, s[i][j], slope, pos, key, nullptr) : -INFINITY;
                top = fmaxf(top, s[i][j]);
            }
            const float mn = fmaxf(m[i], warp_max(top, 8)), base = mn == -INFINITY ? 0.f : mn;
            const float fix = expf(m[i] - base);
            m[i] = mn;
            l[i] *= fix;
#pragma unroll
            for (int c = 0; c < DP / 64; ++c) {
                acc[i][c].x *= fix;
                acc[i][c].y *= fix;
                acc[i][c].z *= fix;
                acc[i][c].w *= fix;
            }
#pragma unroll
            for (int j = 0; j < M; ++j) {
                const float p = rows.sees(r, k0 + tx + 16 * j) ? expf(s[i][j] - base) : 0.f;
                l[i] += p;
                sp[r * LW<N> + tx + 16 * j] = p;
            }
        }
        const bool ask = __syncthreads_or(bad);
        accumulate<M, DP>(sp, sk, acc, ask, [&](int r, int j) { return rows.sees(r, k0 + j); });
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < M; ++i) {
        const int q = q0 + ty * M + i;
        float sum = warp_sum(l[i], 8);
        if (q >= a.q_len) continue;
        sum = sum_or_nan(sum, rows.end[ty * M + i] > rows.first[ty * M + i]);
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        T* o = row<T>(a.o, b, q, h);
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) store4(o, acc[i][c], inv, 64 * c + 4 * tx, a.dim);
        if (a.lse && tx == 0) a.lse[((int64_t)b * a.heads + h) * a.q_len + q] = sum == 0.f ? -INFINITY : m[i] + logf(sum);
    }
}

// Forward of few query rows: a cluster of blocks for each row, whose warps take blocks of 32 keys in turn.  Lane l
// evaluates the score of key l; then the 32 weights are broadcast and lane l sums coordinates l, l + 32, ...  The
// first block joins the sums of all warps, in order, out of the others' shared memory.
template <class T>
__global__ void __launch_bounds__(THREADS) few_kernel(const __grid_constant__ Prob a, bool vec) {
    __shared__ __align__(16) float sq[256];
    __shared__ float so[WARPS][256], sm[WARPS], sl[WARPS];
    cg::cluster_group cluster = cg::this_cluster();
    const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row_at = blockIdx.x / parts, nh = a.heads * a.batch, i = row_at / nh;
    const int b = (row_at - i * nh) / a.heads, h = row_at - i * nh - b * a.heads, hk = h / a.group;
    if ((int)threadIdx.x < a.dim) sq[threadIdx.x] = up<T>(row<T>(a.q, b, i, h)[threadIdx.x]);
    __syncthreads();
    const int n = keys_of(a, b), pos = n - a.q_len + i;
    const int2 sp = row_span(a, b, i, n);
    const float slope = a.slopes ? a.slopes[h] : 0.f;
    float m = -INFINITY, l = 0.f, acc[MAXC] = {};
    for (int64_t j0 = sp.x + (part * WARPS + w) * 32; j0 < sp.y; j0 += parts * WARPS * 32) {
        const int j = (int)j0 + lane;
        float s = -INFINITY;
        if (j < sp.y) {
            const T* k = row<T>(a.k, b, j, hk);
            float d = 0.f;
            if (vec)
#pragma unroll 8
                for (int c = 0; c < a.dim; c += 4) {
                    const float4 x = up4(k + c), y = *(const float4*)(sq + c);
                    d = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, d))));
                }
            else
                for (int c = 0; c < a.dim; ++c) d = fmaf(sq[c], up<T>(k[c]), d);
            s = score(a, d, slope, pos, j, nullptr);
        }
        const float mn = fmaxf(m, warp_max(s)), base = mn == -INFINITY ? 0.f : mn;
        const float fix = expf(m - base), p = j < sp.y ? expf(s - base) : 0.f;
        m = mn;
        l = l * fix + p;
        const int most = (int)min((int64_t)32, sp.y - j0);
#pragma unroll
        for (int c = 0; c < MAXC; ++c) acc[c] *= fix;
#pragma unroll 8
        for (int t = 0; t < most; ++t) {
            const float pt = __shfl_sync(~0u, p, t);
            const T* v = row<T>(a.v, b, j0 + t, hk);
#pragma unroll
            for (int c = 0; c < MAXC; ++c)
                if (lane + 32 * c < a.dim) acc[c] = fmaf(pt, up<T>(v[lane + 32 * c]), acc[c]);
        }
    }
    l = warp_sum(l);
#pragma unroll
    for (int c = 0; c < MAXC; ++c) so[w][lane + 32 * c] = acc[c];
    if (lane == 0) {
        sm[w] = m;
        sl[w] = l;
    }
    cluster.sync();
    if (part == 0) {
        m = -INFINITY;
        for (int y = 0; y < parts; ++y) {
            const float* om = cluster.map_shared_rank(sm, y);
            for (int x = 0; x < WARPS; ++x) m = fmaxf(m, om[x]);
        }
        const float base = m == -INFINITY ? 0.f : m;
        float sum = 0.f, o = 0.f;
        for (int y = 0; y < parts; ++y) {
            const float *om = cluster.map_shared_rank(sm, y), *ol = cluster.map_shared_rank(sl, y);
            const float* oo = cluster.map_shared_rank(&so[0][0], y);
            for (int x = 0; x < WARPS; ++x) {
                const float f = expf(om[x] - base);
                sum = fmaf(f, ol[x], sum);
                o = fmaf(f, oo[x * 256 + threadIdx.x], o);
            }
        }
        sum = sum_or_nan(sum, sp.y > sp.x);
        if ((int)threadIdx.x < a.dim) row<T>(a.o, b, i, h)[threadIdx.x] = down<T>(sum == 0.f ? 0.f : o / sum);
        if (a.lse && threadIdx.x == 0)
            a.lse[((int64_t)b * a.heads + h) * a.q_len + i] = sum == 0.f ? -INFINITY : m + logf(sum);
    }
    cluster.sync();   // nobody leaves while its shared memory is read
}

// delta[b, h, i] = dO . o, with the low bits of o where the forward pass kept them; a warp a row
template <class T>
__global__ void __launch_bounds__(THREADS) delta_kernel(const __grid_constant__ Prob a, float* __restrict__ delta) {
    const int lane = threadIdx.x & 31;
    const int64_t x = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5);
    if (x >= (int64_t)a.batch * a.heads * a.q_len) return;
    const int64_t bh = x / a.q_len;
    const int i = (int)(x - bh * a.q_len), b = (int)(bh / a.heads), h = (int)(bh - (int64_t)b * a.heads);
    const T *g = row<T>(a.d_o, b, i, h), *o = row<T>(a.o, b, i, h);
    const int8_t* low = a.o_low ? a.o_low + (((int64_t)b * a.q_len + i) * a.heads + h) * a.dim : nullptr;
    float d = 0.f;
    for (int c = lane; c < a.dim; c += 32) {
        float f = up<T>(o[c]);
        if (sizeof(T) == 2 && low) f = with_low<std::is_same<T, __half>::value>(f, low[c]);
        d = fmaf(up<T>(g[c]), f, d);
    }
    d = warp_sum(d);
    if (lane == 0) delta[x] = d;
}

// Rows and columns of a backward tile: 16 M; D = 256 has room for 32 only.
template <int DP> constexpr int BM = DP <= 128 ? 4 : 2;

// dq = sum_j dS_j k_j, dS = P (dP - delta) bend scale
template <class T, int DP>
__global__ void __launch_bounds__(THREADS, DP <= 64 ? 2 : 1) dq_kernel(const __grid_constant__ Prob a, const float* __restrict__ delta,
                                                     bool vec) {
    constexpr int M = BM<DP>, N = 16 * M;
    extern __shared__ __align__(16) float smem[];
    float *sq = smem, *sg = sq + N * LD<DP>, *sk = sg + N * LD<DP>, *sv = sk + N * LD<DP>, *ss = sv + N * LD<DP>;
    __shared__ Rows<N> rows;
    const Place at(a.heads, a.batch);
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    const int b = at.b, h = at.h, hk = h / a.group, q0 = at.tile * N, n = keys_of(a, b);
    rows.fill(a, b, q0, n);
    load_tile<T, N, DP>(sq, a.q, b, h, q0, a.q_len, a.dim, vec);
    load_tile<T, N, DP>(sg, a.d_o, b, h, q0, a.q_len, a.dim, vec);
    const float slope = a.slopes ? a.slopes[h] : 0.f;
    float lse[M], dl[M];
    float4 acc[M][DP / 64];
#pragma unroll
    for (int i = 0; i < M; ++i) {
        const int q = q0 + ty * M + i;
        const int64_t x = ((int64_t)b * a.heads + h) * a.q_len + q;
        lse[i] = q < a.q_len ? a.lse[x] : -INFINITY;
        dl[i] = q < a.q_len ? delta[x] : 0.f;
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) acc[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int k0 = rows.lo & ~(N - 1); k0 < rows.hi; k0 += N) {
        const bool bad = load_tile<T, N, DP>(sk, a.k, b, hk, k0, n, a.dim, vec);
        load_tile<T, N, DP>(sv, a.v, b, hk, k0, n, a.dim, vec);
        const bool ask = __syncthreads_or(bad);
        float s[M][M], dp[M][M];
        products<M, DP>(sq, sk, a.dim, s);
        products<M, DP>(sg, sv, a.dim, dp);
#pragma unroll
        for (int i = 0; i < M; ++i)
#pragma unroll
            for (int j = 0; j < M; ++j) {
                const int r = ty * M + i, key = k0 + tx + 16 * j;
                float ds = 0.f, bend;
                if (rows.sees(r, key) && lse[i] != -INFINITY) {
                    const float x = score(a, s[i][j], slope, n - a.q_len + q0 + r, key, &bend);
                    ds = expf(x - lse[i]) * (dp[i][j] - dl[i]) * bend * a.scale;
                }
                ss[r * LW<N> + tx + 16 * j] = ds;
            }
        __syncthreads();
        accumulate<M, DP>(ss, sk, acc, ask, [&](int r, int j) { return rows.sees(r, k0 + j); });
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < M; ++i) {
        const int q = q0 + ty * M + i;
        if (q >= a.q_len) continue;
        T* o = row<T>(a.dq, b, q, h);
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) store4(o, acc[i][c], 1.f, 64 * c + 4 * tx, a.dim);
    }
}

// dv = sum_i P_i dO_i, dk = sum_i dS_i q_i over the query rows and heads that see the keys
template <class T, int DP>
__global__ void __launch_bounds__(THREADS, DP <= 64 ? 2 : 1) dkv_kernel(const __grid_constant__ Prob a, const float* __restrict__ delta,
                                                      bool vec) {
    constexpr int M = BM<DP>, N = 16 * M;
    extern __shared__ __align__(16) float smem[];
    float *sk = smem, *sv = sk + N * LD<DP>, *sq = sv + N * LD<DP>, *sg = sq + N * LD<DP>;
    float *sp = sg + N * LD<DP>, *ss = sp + N * LW<N>;
    __shared__ Rows<N> rows;
    __shared__ float lse[N], dl[N];
    const Place at(a.kv_heads, a.batch);
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    const int b = at.b, hk = at.h, k0 = at.tile * N, n = keys_of(a, b);
    load_tile<T, N, DP>(sk, a.k, b, hk, k0, n, a.dim, vec);
    load_tile<T, N, DP>(sv, a.v, b, hk, k0, n, a.dim, vec);
    float4 ak[M][DP / 64], av[M][DP / 64];
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) ak[i][c] = av[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int q0 = 0; q0 < a.q_len; q0 += N) {
        rows.fill(a, b, q0, n);
        if (rows.hi <= k0 || rows.lo >= k0 + N) {
            __syncthreads();                      // all have looked before the next tile's rows are written
            continue;
        }
        for (int g = 0; g < a.group; ++g) {
            const int h = hk * a.group + g;
            const float slope = a.slopes ? a.slopes[h] : 0.f;
            bool bad = load_tile<T, N, DP>(sq, a.q, b, h, q0, a.q_len, a.dim, vec);
            bad |= load_tile<T, N, DP>(sg, a.d_o, b, h, q0, a.q_len, a.dim, vec);
            if (threadIdx.x < N) {
                const int q = q0 + (int)threadIdx.x;
                const int64_t x = ((int64_t)b * a.heads + h) * a.q_len + q;
                lse[threadIdx.x] = q < a.q_len ? a.lse[x] : -INFINITY;
                dl[threadIdx.x] = q < a.q_len ? delta[x] : 0.f;
            }
            const bool ask = __syncthreads_or(bad);
            float s[M][M], dp[M][M];
            products<M, DP>(sk, sq, a.dim, s);
            products<M, DP>(sv, sg, a.dim, dp);
#pragma unroll
            for (int i = 0; i < M; ++i)
#pragma unroll
                for (int j = 0; j < M; ++j) {
                    const int r = tx + 16 * j, key = k0 + ty * M + i;
                    float p = 0.f, ds = 0.f, bend;
                    if (rows.sees(r, key) && lse[r] != -INFINITY) {
                        p = expf(score(a, s[i][j], slope, n - a.q_len + q0 + r, key, &bend) - lse[r]);
                        ds = p * (dp[i][j] - dl[r]) * bend * a.scale;
                    }
                    sp[(ty * M + i) * LW<N> + r] = p;
                    ss[(ty * M + i) * LW<N> + r] = ds;
                }
            __syncthreads();
            auto seen = [&](int key, int r) { return rows.sees(r, k0 + key); };
            accumulate<M, DP>(sp, sg, av, ask, seen);
            accumulate<M, DP>(ss, sq, ak, ask, seen);
            __syncthreads();
        }
    }
#pragma unroll
    for (int i = 0; i < M; ++i) {
        const int key = k0 + ty * M + i;
        if (key >= a.k_len) continue;
        T *dk = row<T>(a.dk, b, key, hk), *dv = row<T>(a.dv, b, key, hk);
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
            store4(dk, ak[i][c], 1.f, 64 * c + 4 * tx, a.dim);
            store4(dv, av[i][c], 1.f, 64 * c + 4 * tx, a.dim);
        }
    }
}

// Four coordinates at a time can be read at once.
inline bool vectors(const Prob& a, const View& v, size_t type) {
    return a.dim % 4 == 0 && (uintptr_t)v.p % (4 * type) == 0 && v.sb % 4 == 0 && v.ss % 4 == 0 && v.sh % 4 == 0;
}

// Blocks of `rows` rows for all heads of the batch.
inline int blocks_of(int64_t rows, int per, int64_t heads, int batch, unsigned* out) {
    const int64_t blocks = cdiv(rows, (int64_t)per) * heads * batch;
    FD_CHECK_ARG(blocks <= 0x7fffffff, "fd_attention: too many rows and heads");
    *out = (unsigned)blocks;
    return FD_OK;
}

// The forward pass takes a cluster for each query row (few_kernel) while rows times its time for a key, 0.26 ns, stay
// below the tiles' waves times theirs, 250 ns for each of 64 keys wherever only some rows of a tile are real (fp32
// heads of 128: 8 rows of 8 heads against 8192 keys 165 us by rows, 1630 us by tiles; 8 rows of 256 heads 4290 us by
// rows, 2600 us by tiles).
inline bool by_rows(const Prob& a) {
    const int64_t heads = (int64_t)a.heads * a.batch;
    return a.q_len * heads <= 1000 * cdiv(cdiv(a.q_len, 64) * heads, 2 * num_sms());
}

template <class T, int DP>
int forward(const Prob& a, bool vec, cudaStream_t s) {
    constexpr int N = 64;
    constexpr uint32_t bytes = 4 * (2 * N * LD<DP> + N * LW<N>);
    unsigned blocks;
    FD_TRY(blocks_of(a.q_len, N, a.heads, a.batch, &blocks));
    FD_TRY((allow_smem<forward_kernel<T, DP>>(bytes)));
    forward_kernel<T, DP><<<blocks, THREADS, bytes, s>>>(a, vec);
    FD_CUDA_TRY(cudaGetLastError());
    return FD_OK;
}

template <class T, int DP>
int backward(const Prob& a, float* delta, bool vec, cudaStream_t s) {
    constexpr int N = 16 * BM<DP>;
    constexpr uint32_t tiles = 4 * 4 * N * LD<DP>, weights = 4 * N * LW<N>;
    unsigned blocks;
    if (a.q_len > 0) {
        FD_TRY(blocks_of((int64_t)a.q_len * a.heads * a.batch, WARPS, 1, 1, &blocks));
        delta_kernel<T><<<blocks, THREADS, 0, s>>>(a, delta);
        FD_TRY(blocks_of(a.q_len, N, a.heads, a.batch, &blocks));
        FD_TRY((allow_smem<dq_kernel<T, DP>>(tiles + weights)));
        dq_kernel<T, DP><<<blocks, THREADS, tiles + weights, s>>>(a, delta, vec);
        FD_CUDA_TRY(cudaGetLastError());
    }
    if (a.k_len > 0) {
        FD_TRY(blocks_of(a.k_len, N, a.kv_heads, a.batch, &blocks));
        FD_TRY((allow_smem<dkv_kernel<T, DP>>(tiles + 2 * weights)));
        dkv_kernel<T, DP><<<blocks, THREADS, tiles + 2 * weights, s>>>(a, delta, vec);
        FD_CUDA_TRY(cudaGetLastError());
    }
    return FD_OK;
}

template <class T>
int forward_of(const Prob& a, cudaStream_t s) {
    const bool vec = vectors(a, a.q, sizeof(T)) && vectors(a, a.k, sizeof(T)) && vectors(a, a.v, sizeof(T));
    if (by_rows(a)) {
        // blocks for each row: enough to fill the SMs, none without a block of keys for each warp
        int parts = 1;
        const int64_t rows = (int64_t)a.q_len * a.heads * a.batch;
        while (parts < 8 && rows * parts < 2 * num_sms() && (int64_t)parts * WARPS * 32 < a.k_len) parts *= 2;
        unsigned blocks;
        FD_TRY(blocks_of(rows, 1, parts, 1, &blocks));
        cudaLaunchAttribute size{};
        size.id = cudaLaunchAttributeClusterDimension;
        size.val.clusterDim.x = parts;
        size.val.clusterDim.y = size.val.clusterDim.z = 1;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(blocks);
        cfg.blockDim = dim3(THREADS);
        cfg.stream = s;
        cfg.attrs = &size;
        cfg.numAttrs = 1;
        FD_CUDA_TRY(cudaLaunchKernelEx(&cfg, few_kernel<T>, a, vec));
        FD_CUDA_TRY(cudaGetLastError());
        return FD_OK;
    }
    if (a.dim <= 64) return forward<T, 64>(a, vec, s);
    return a.dim <= 128 ? forward<T, 128>(a, vec, s) : forward<T, 256>(a, vec, s);
}

template <class T>
int backward_of(const Prob& a, float* delta, cudaStream_t s) {
    const bool vec = vectors(a, a.q, sizeof(T)) && vectors(a, a.k, sizeof(T)) && vectors(a, a.v, sizeof(T)) &&
                     vectors(a, a.d_o, sizeof(T));
    if (a.dim <= 64) return backward<T, 64>(a, delta, vec, s);
    return a.dim <= 128 ? backward<T, 128>(a, delta, vec, s) : backward<T, 256>(a, delta, vec, s);
}

}  // namespace simt

int simt_forward(const Prob& a, int dtype, cudaStream_t s) {
    if (dtype == FD_DTYPE_F16) return simt::forward_of<__half>(a, s);
    if (dtype == FD_DTYPE_BF16) return simt::forward_of<__nv_bfloat16>(a, s);
    return simt::forward_of<float>(a, s);
}

int simt_backward(const Prob& a, int dtype, float* delta, cudaStream_t s) {
    if (dtype == FD_DTYPE_F16) return simt::backward_of<__half>(a, delta, s);
    if (dtype == FD_DTYPE_BF16) return simt::backward_of<__nv_bfloat16>(a, delta, s);
    return simt::backward_of<float>(a, delta, s);
}

}  // namespace attn
}  // namespace fd
