// Rotary positions of query and key heads, forward and inverse (= gradient).
//
//   pair (a, b) of a head turns by t = pos * f_p:
//   a' = m (a cos t - b sin t),   b' = m (a sin t + b cos t)
//
// Bandwidth-bound: each element is read and written once.  The angle belongs to
// a (token, pair), not to a head, so a block makes the angles of a few tokens
// once, in shared memory, and then streams over the heads of q and k, which lie
// together in memory, one chunk a thread and as many threads as the SMs hold.
// One thread walking the heads of a token with its angles in registers
// kept too little in flight and scattered it (8192 tokens of 32 + 8 bf16 heads of
// 128: 40 us against 31, 5.4 TB/s).
#include "fd_tc_common.cuh"

namespace fd {
namespace rotary {

struct Side {
    const void* x;
    void* y;
    int64_t xs[3], ys[3];
    int heads;
};

struct Args {
    Side side[2];
    const void* pos;
    int64_t ps[2];
    const double* freqs;
    float magnitude;
    int pos_dtype, inverse;
    int64_t tokens, total;   // tokens per batch entry; batch * tokens
    int dim, rot;
    int rot_units, units;    // chunks of pairs; chunks of pairs and of copied coordinates
    int block_tokens;
};

template <class T> struct Cvt;
template <> struct Cvt<float> {
    __device__ static float up(float x) { return x; }
    __device__ static float down(float x) { return x; }
};
template <> struct Cvt<__half> {
    __device__ static float up(__half x) { return __half2float(x); }
    __device__ static __half down(float x) { return __float2half_rn(x); }
};
template <> struct Cvt<__nv_bfloat16> {
    __device__ static float up(__nv_bfloat16 x) { return __bfloat162float(x); }
    __device__ static __nv_bfloat16 down(float x) { return __float2bfloat16_rn(x); }
};

template <class T, int N>
struct alignas(sizeof(T) * N) Vec {
    T v[N];
};

__device__ __forceinline__ int64_t batch_of(const Args& a, int64_t t) {
    if (a.tokens == a.total) return 0;
    return (uint64_t)(t | a.tokens) >> 32 ? t / a.tokens : (uint32_t)t / (uint32_t)a.tokens;
}

__device__ __forceinline__ double position(const Args& a, int64_t t) {
    const int64_t b = batch_of(a, t), i = b * a.ps[0] + (t - b * a.tokens) * a.ps[1];
    switch (a.pos_dtype) {
        case FD_DTYPE_I32: return (double)((const int32_t*)a.pos)[i];
        case FD_DTYPE_I64: return (double)((const int64_t*)a.pos)[i];
        case FD_DTYPE_F32: return (double)((const float*)a.pos)[i];
        default: return ((const double*)a.pos)[i];
    }
}

// cos and sin of pos * f.  Positions reach 1e6 and more, where an fp32 product
// keeps no digit of the fraction: the quarter turns pos * f * 2 / pi are formed in
// fp64, rounded to a whole number there (by adding and taking away 1.5 * 2^52,
// whose low bits then hold the quadrant), and the rest h, |h| <= 1/2 and exact to
// 2^-26, goes through polynomials of degree 7 and 6 in fp32 (fitted on Chebyshev
// nodes; absolute error 1.1e-7 at most and 3e-8 in the mean, h's rounding and
// every fp32 step included).  Some 20 instructions an angle: the general
// sincospi's 45 made a call with few heads issue-bound.
__device__ __forceinline__ void angle_of(double pos, double f, float& cs, float& sn) {
    const double t = pos * (f * 0.63661977236758134308);
    const double near = t + 6755399441055744.0;
    const int k = __double2loint(near);
    const float h = (float)(t - (near - 6755399441055744.0)), y = h * h;
    const float s = h * fmaf(fmaf(fmaf(-0.004602163f, y, 0.07968022f), y, -0.6459635f), y, 1.5707964f);
    const float c = fmaf(fmaf(fmaf(-0.020408256f, y, 0.2535986f), y, -1.233697f), y, 1.0f);
    const float a = k & 1 ? s : c, b = k & 1 ? c : s;
    cs = (k + 1) & 2 ? -a : a;
    sn = k & 2 ? -b : b;
}

// N floats from shared memory, 16 bytes at a time where they allow it.
template <int N>
__device__ __forceinline__ void table(const float* p, float (&v)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 x = *(const float4*)(p + i);
            v[i] = x.x;
            v[i + 1] = x.y;
            v[i + 2] = x.z;
            v[i + 3] = x.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = p[i];
    }
}

// One chunk turned: V pairs in two vectors (half layout, or single elements), or V / 2 adjacent pairs in one.
template <class T, int V, bool TWO, int P>
__device__ __forceinline__ void turn_chunk(Vec<T, V>& lo, Vec<T, V>& hi, const float (&c)[P], const float (&s)[P]) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
        T& x = TWO ? lo.v[p] : lo.v[2 * p];
        T& y = TWO ? hi.v[p] : lo.v[V > 1 ? 2 * p + 1 : 0];
        const float f0 = Cvt<T>::up(x), f1 = Cvt<T>::up(y);
        x = Cvt<T>::down(f0 * c[p] - f1 * s[p]);
        y = Cvt<T>::down(f0 * s[p] + f1 * c[p]);
    }
}

// V: elements per vector access.  A chunk is V pairs in the half layout (two
// vectors) and V / 2 pairs in the interleaved one (one vector; V = 1 there
// means one pair read as two scalars).  Thread (u, y) of a block takes chunk u of
// the (token, head) rows y, y + blockDim.y, ...
template <class T, int V, bool HALF>
__global__ void __launch_bounds__(256) rotary_kernel(const __grid_constant__ Args a) {
    constexpr int P = HALF ? V : (V > 1 ? V / 2 : 1);
    constexpr bool TWO = HALF || V == 1;       // a chunk's pairs lie in two vectors
    extern __shared__ __align__(16) char smem[];
    const int pairs = a.rot / 2, tid = threadIdx.y * blockDim.x + threadIdx.x, threads = blockDim.x * blockDim.y;
    const int64_t t0 = (int64_t)blockIdx.x * a.block_tokens;
    const int nt = (int)min((int64_t)a.block_tokens, a.total - t0);
    int64_t(*off)[4] = (int64_t(*)[4])smem;    // of a token's first head: x and y of q, x and y of k
    float* cs = (float*)(smem + a.block_tokens * 32);
    float* sn = cs + a.block_tokens * pairs;
    for (int i = tid; i < nt; i += threads) {
        const int64_t t = t0 + i, b = batch_of(a, t), s = t - b * a.tokens;
        for (int z = 0; z < 2; ++z) {
            off[i][2 * z] = b * a.side[z].xs[0] + s * a.side[z].xs[1];
            off[i][2 * z + 1] = b * a.side[z].ys[0] + s * a.side[z].ys[1];
        }
    }
    for (int i = tid; i < nt * pairs; i += threads) {
        const int k = i / pairs, p = i - k * pairs;
        float x, y;
        angle_of(position(a, t0 + k), a.freqs[p], x, y);
        cs[i] = a.magnitude * x;
        sn[i] = a.magnitude * (a.inverse ? -y : y);
    }
    __syncthreads();
    const int nq = a.side[0].heads, n = nq + a.side[1].heads, far = HALF ? pairs : 1;
    for (int u = threadIdx.x; u < a.units; u += blockDim.x) {
        const bool turn = u < a.rot_units;
        const int at = turn ? (HALF ? u * V : u * 2 * P) : a.rot + (u - a.rot_units) * V;
        int k = (int)threadIdx.y / n, h = (int)threadIdx.y - k * n;     // this thread's next row
        while (k < nt) {
            const bool q = h < nq;
            const Side& sd = a.side[q ? 0 : 1];
            const int64_t* o = off[k] + (q ? 0 : 2);
            const int64_t hh = q ? h : h - nq;
            const T* src = (const T*)sd.x + o[0] + hh * sd.xs[2] + at;
            T* dst = (T*)sd.y + o[1] + hh * sd.ys[2] + at;
            Vec<T, V> lo = *(const Vec<T, V>*)src, hi;
            if (TWO && turn) hi = *(const Vec<T, V>*)(src + far);
            const int tok = k;
            for (h += blockDim.y; h >= n; h -= n) ++k;
            if (turn) {
                float c[P], s[P];
                table<P>(cs + tok * pairs + u * P, c);
                table<P>(sn + tok * pairs + u * P, s);
                turn_chunk<T, V, TWO, P>(lo, hi, c, s);
                if (TWO) *(Vec<T, V>*)(dst + far) = hi;
            }
            *(Vec<T, V>*)dst = lo;
        }
    }
}

// The same for few heads, where no angle is worth sharing: thread (u, y) takes
// chunk u of one token, and its first load is under way while its angles are made.
template <class T, int V, bool HALF>
__global__ void __launch_bounds__(256) rotary_few_kernel(const __grid_constant__ Args a) {
    constexpr int P = HALF ? V : (V > 1 ? V / 2 : 1);
    constexpr bool TWO = HALF || V == 1;
    const int64_t t = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (t >= a.total) return;
    const int64_t b = batch_of(a, t), st = t - b * a.tokens;
    const int far = HALF ? a.rot / 2 : 1;
    for (int u = threadIdx.x; u < a.units; u += blockDim.x) {
        const bool turn = u < a.rot_units;
        const int at = turn ? (HALF ? u * V : u * 2 * P) : a.rot + (u - a.rot_units) * V;
        float c[P], s[P];
        bool made = false;
#pragma unroll 1
        for (int z = 0; z < 2; ++z) {
            const Side& sd = a.side[z];
            if (!sd.heads) continue;
            const T* src = (const T*)sd.x + b * sd.xs[0] + st * sd.xs[1] + at;
            T* dst = (T*)sd.y + b * sd.ys[0] + st * sd.ys[1] + at;
            for (int h = 0; h < sd.heads; ++h, src += sd.xs[2], dst += sd.ys[2]) {
                Vec<T, V> lo = *(const Vec<T, V>*)src, hi;
                if (turn) {
                    if (TWO) hi = *(const Vec<T, V>*)(src + far);
                    if (!made) {
                        const double pos = position(a, t);
#pragma unroll
                        for (int p = 0; p < P; ++p) {
                            float x, y;
                            angle_of(pos, a.freqs[u * P + p], x, y);
                            c[p] = a.magnitude * x;
                            s[p] = a.magnitude * (a.inverse ? -y : y);
                        }
                        made = true;
                    }
                    turn_chunk<T, V, TWO, P>(lo, hi, c, s);
                    if (TWO) *(Vec<T, V>*)(dst + far) = hi;
                }
                *(Vec<T, V>*)dst = lo;
            }
        }
    }
}

// Heads up to which each thread makes its own angles.
constexpr int FEW = 2;

template <class T, int V>
int launch(Args& a, int layout, cudaStream_t s) {
    const bool half = layout == FD_ROTARY_HALF;
    const int pairs = half ? V : (V > 1 ? V / 2 : 1);
    a.rot_units = a.rot / 2 / pairs;
    a.units = a.rot_units + (a.dim - a.rot) / V;
    const dim3 block((unsigned)(a.units < 128 ? a.units : 128), (unsigned)(a.units < 128 ? 256 / a.units : 2));
    // As many tokens to a block as give each of its threads an angle, while that leaves every SM several blocks.
    const int64_t fit = 512 / a.rot < 1 ? 1 : 512 / a.rot, spread = a.total / (num_sms() * 4);
    a.block_tokens = (int)(spread < 1 ? 1 : spread < fit ? spread : fit);
    const int64_t blocks = cdiv(a.total, a.block_tokens);
    const size_t smem = a.block_tokens * (32 + (size_t)a.rot * 4);
    FD_CHECK_ARG(blocks <= 0x7fffffff, "fd_rotary: %lld tokens are too many for one call", (long long)a.total);
    if (a.side[0].heads + a.side[1].heads <= FEW) {
        const int64_t few = cdiv(a.total, block.y);
        FD_CHECK_ARG(few <= 0x7fffffff, "fd_rotary: %lld tokens are too many for one call", (long long)a.total);
        if (half) rotary_few_kernel<T, V, true><<<(unsigned)few, block, 0, s>>>(a);
        else rotary_few_kernel<T, V, false><<<(unsigned)few, block, 0, s>>>(a);
    } else if (half) {
        rotary_kernel<T, V, true><<<(unsigned)blocks, block, smem, s>>>(a);
    } else {
        rotary_kernel<T, V, false><<<(unsigned)blocks, block, smem, s>>>(a);
    }
    FD_CUDA_TRY(cudaGetLastError());
    return FD_OK;
}

template <class T>
int dispatch(Args& a, int layout, cudaStream_t s) {
    // 16-byte chunks when every address they touch is 16-byte aligned
    constexpr int V = 16 / sizeof(T);
    const int64_t step = layout == FD_ROTARY_HALF ? 2 * V : V;
    bool wide = a.rot % step == 0 && a.dim % V == 0;
    for (int z = 0; z < 2; ++z) {
        const Side& sd = a.side[z];
        if (!sd.heads) continue;
        wide = wide && ((uintptr_t)sd.x & 15) == 0 && ((uintptr_t)sd.y & 15) == 0;
        for (int i = 0; i < 3; ++i) wide = wide && sd.xs[i] % V == 0 && sd.ys[i] % V == 0;
    }
    return wide ? launch<T, V>(a, layout, s) : launch<T, 1>(a, layout, s);
}

}  // namespace rotary
}  // namespace fd

extern "C" int fd_rotary(const fd_rotary_args* r, void* stream) {
    using namespace fd;
    FD_CHECK_ARG(r, "fd_rotary: null arguments");
    FD_CHECK_ARG(r->batch >= 0 && r->tokens >= 0 && r->heads >= 0 && r->kv_heads >= 0, "fd_rotary: negative size");
    FD_CHECK_ARG(r->dim <= 4096, "fd_rotary: dim=%d above 4096", r->dim);
    FD_CHECK_ARG(r->dim >= 1 && r->rot >= 2 && r->rot <= r->dim && r->rot % 2 == 0,
                 "fd_rotary: rot=%d must be even, at least 2 and at most dim=%d", r->rot, r->dim);
    FD_CHECK_ARG(r->layout == FD_ROTARY_HALF || r->layout == FD_ROTARY_INTERLEAVED, "fd_rotary: layout %d", r->layout);
    FD_CHECK_ARG(r->position_dtype == FD_DTYPE_I32 || r->position_dtype == FD_DTYPE_I64 ||
                     r->position_dtype == FD_DTYPE_F32 || r->position_dtype == FD_DTYPE_F64,
                 "fd_rotary: position dtype %d", r->position_dtype);
    FD_CHECK_ARG(r->dtype == FD_DTYPE_F32 || r->dtype == FD_DTYPE_F16 || r->dtype == FD_DTYPE_BF16,
                 "fd_rotary: dtype %d", r->dtype);
    if (r->batch * r->tokens == 0 || r->heads + r->kv_heads == 0) return FD_OK;
    FD_CHECK_ARG((r->heads == 0 || (r->q && r->qo)) && (r->kv_heads == 0 || (r->k && r->ko)) && r->positions && r->freqs,
                 "fd_rotary: null pointer");
    rotary::Args a{};
    a.side[0] = {r->q, r->qo, {}, {}, r->heads};
    a.side[1] = {r->k, r->ko, {}, {}, r->kv_heads};
    // a stride that is never taken (extent 1) may be anything: it becomes 0
    for (int i = 0; i < 3; ++i) {
        const bool lone = (i == 0 && r->batch == 1) || (i == 1 && r->tokens == 1);
        const bool q1 = lone || (i == 2 && r->heads == 1), k1 = lone || (i == 2 && r->kv_heads == 1);
        a.side[0].xs[i] = q1 ? 0 : r->q_stride[i];
        a.side[0].ys[i] = q1 ? 0 : r->qo_stride[i];
        a.side[1].xs[i] = k1 ? 0 : r->k_stride[i];
        a.side[1].ys[i] = k1 ? 0 : r->ko_stride[i];
    }
    a.pos = r->positions;
    a.ps[0] = r->position_stride[0];
    a.ps[1] = r->position_stride[1];
    a.freqs = r->freqs;
    a.magnitude = (float)r->magnitude;
    a.pos_dtype = r->position_dtype;
    a.inverse = r->inverse != 0;
    a.tokens = r->tokens;
    a.total = r->batch * r->tokens;
    a.dim = r->dim;
    a.rot = r->rot;
    switch (r->dtype) {
        case FD_DTYPE_F16: return rotary::dispatch<__half>(a, r->layout, (cudaStream_t)stream);
        case FD_DTYPE_BF16: return rotary::dispatch<__nv_bfloat16>(a, r->layout, (cudaStream_t)stream);
        default: return rotary::dispatch<float>(a, r->layout, (cudaStream_t)stream);
    }
}
