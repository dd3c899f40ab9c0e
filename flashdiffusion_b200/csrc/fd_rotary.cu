// Rotary positions of query and key heads, forward and inverse (= gradient).
//
//   pair (a, b) of a head turns by t = pos * f_p:
//   a' = m (a cos t - b sin t),   b' = m (a sin t + b cos t)
//
// Bandwidth-bound: each element is read and written once.  The angle belongs to
// a (token, pair), not to a head, so a thread takes one chunk of pairs of one
// token, reduces its angles once and walks over the heads of q and then of k.
// Angles: positions reach 1e6 and more, where an fp32 product keeps no digit of
// the fraction; pos * f / 2pi is formed in fp64 turns, its integer part dropped
// there, and the remaining fraction (|r| <= 1/2, exact to 2^-25) goes through
// fp32 sincospi.
#include "fd_common.cuh"

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
    int split;               // threads that share the heads of one chunk
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

__device__ __forceinline__ double position(const Args& a, int64_t b, int64_t s) {
    const int64_t i = b * a.ps[0] + s * a.ps[1];
    switch (a.pos_dtype) {
        case FD_DTYPE_I32: return (double)((const int32_t*)a.pos)[i];
        case FD_DTYPE_I64: return (double)((const int64_t*)a.pos)[i];
        case FD_DTYPE_F32: return (double)((const float*)a.pos)[i];
        default: return ((const double*)a.pos)[i];
    }
}

// V: elements per vector access.  A chunk is V pairs in the half layout (two
// vectors) and V / 2 pairs in the interleaved one (one vector; V = 1 there
// means one pair read as two scalars).
template <class T, int V, bool HALF>
__global__ void __launch_bounds__(256) rotary_kernel(const Args a) {
    constexpr int P = HALF ? V : (V > 1 ? V / 2 : 1);
    const int64_t g = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (g >= a.total * a.split * a.units) return;
    const int u = (int)(g % a.units);
    const int64_t ts = g / a.units;
    const int hs = (int)(ts % a.split);
    const int64_t t = ts / a.split;
    const int64_t b = t / a.tokens, s = t - b * a.tokens;
    const bool turn = u < a.rot_units;
    float c[P], n[P];
    int at0, at1 = 0;
    if (turn) {
        const double pos = position(a, b, s);
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const double turns = pos * a.freqs[u * P + p] * 0.15915494309189533577;
            float sn, cs;
            sincospif(2.0f * (float)(turns - rint(turns)), &sn, &cs);
            c[p] = a.magnitude * cs;
            n[p] = a.magnitude * (a.inverse ? -sn : sn);
        }
        at0 = HALF ? u * V : u * 2 * P;
        at1 = a.rot / 2 + u * V;
    } else {
        at0 = a.rot + (u - a.rot_units) * V;
    }
#pragma unroll
    for (int z = 0; z < 2; ++z) {
        const Side& sd = a.side[z];
        const T* x = (const T*)sd.x + b * sd.xs[0] + s * sd.xs[1] + at0;
        T* y = (T*)sd.y + b * sd.ys[0] + s * sd.ys[1] + at0;
#pragma unroll 4
        for (int h = hs; h < sd.heads; h += a.split) {
            const T* xh = x + h * sd.xs[2];
            T* yh = y + h * sd.ys[2];
            if (!turn) {
                *(Vec<T, V>*)yh = *(const Vec<T, V>*)xh;
            } else if constexpr (HALF) {
                const Vec<T, V> lo = *(const Vec<T, V>*)xh, hi = *(const Vec<T, V>*)(xh + (at1 - at0));
                Vec<T, V> lo2, hi2;
#pragma unroll
                for (int p = 0; p < V; ++p) {
                    const float f0 = Cvt<T>::up(lo.v[p]), f1 = Cvt<T>::up(hi.v[p]);
                    lo2.v[p] = Cvt<T>::down(f0 * c[p] - f1 * n[p]);
                    hi2.v[p] = Cvt<T>::down(f0 * n[p] + f1 * c[p]);
                }
                *(Vec<T, V>*)yh = lo2;
                *(Vec<T, V>*)(yh + (at1 - at0)) = hi2;
            } else if constexpr (V > 1) {
                const Vec<T, V> v = *(const Vec<T, V>*)xh;
                Vec<T, V> w;
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    const float f0 = Cvt<T>::up(v.v[2 * p]), f1 = Cvt<T>::up(v.v[2 * p + 1]);
                    w.v[2 * p] = Cvt<T>::down(f0 * c[p] - f1 * n[p]);
                    w.v[2 * p + 1] = Cvt<T>::down(f0 * n[p] + f1 * c[p]);
                }
                *(Vec<T, V>*)yh = w;
            } else {
                const float f0 = Cvt<T>::up(xh[0]), f1 = Cvt<T>::up(xh[1]);
                yh[0] = Cvt<T>::down(f0 * c[0] - f1 * n[0]);
                yh[1] = Cvt<T>::down(f0 * n[0] + f1 * c[0]);
            }
        }
    }
}

template <class T, int V>
int launch(Args& a, int layout, cudaStream_t s) {
    const bool half = layout == FD_ROTARY_HALF;
    const int pairs = half ? V : (V > 1 ? V / 2 : 1);
    a.rot_units = a.rot / 2 / pairs;
    a.units = a.rot_units + (a.dim - a.rot) / V;
    // Few tokens: the heads of a chunk are shared by up to `heads` threads, until
    // the launch fills the SMs' thread slots; many tokens: one thread walks all
    // heads and pays for its angles once.
    const int most = a.side[0].heads > a.side[1].heads ? a.side[0].heads : a.side[1].heads;
    const int64_t want = cdiv((int64_t)148 * 2048, a.total * a.units);
    a.split = (int)(want < 1 ? 1 : want > most ? most : want);
    const int64_t threads = a.total * a.units * a.split;
    const int64_t blocks = cdiv(threads, 256);
    FD_CHECK_ARG(blocks <= 0x7fffffff, "fd_rotary: %lld tokens are too many for one call", (long long)a.total);
    if (half) rotary_kernel<T, V, true><<<(unsigned)blocks, 256, 0, s>>>(a);
    else rotary_kernel<T, V, false><<<(unsigned)blocks, 256, 0, s>>>(a);
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
