// Softmax attention over key spans: what the kernels of fd_attn_*.cu share.
#pragma once
#include <atomic>

#include "fd_common.cuh"

namespace fd {
namespace attn {

// Allow kernel FN `bytes` of dynamic shared memory on the current device: set once
// for each device (the call costs a microsecond and more).
template <auto FN>
inline int allow_smem(uint32_t bytes) {
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    FD_CUDA_TRY(cudaGetDevice(&dev));
    const uint64_t bit = 1ull << (dev & 63);
    if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return FD_OK;
    FD_CUDA_TRY(cudaFuncSetAttribute(FN, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    done.fetch_or(bit, std::memory_order_relaxed);
    return FD_OK;
}

struct View {
    void* p;
    int64_t sb, ss, sh;   // batch, token, head strides in elements
};

struct Prob {
    View q, k, v, o, d_o, dq, dk, dv;
    float* lse;
    int8_t* o_low;
    const int32_t *first, *end;
    int64_t span_stride;
    const int32_t* lengths;
    const float* slopes;
    float scale, cap;
    int causal, window;
    int batch, q_len, k_len, heads, kv_heads, dim, group;
};

// Keys in use by batch entry b.
__device__ __forceinline__ int keys_of(const Prob& a, int b) {
    if (!a.lengths) return a.k_len;
    return min(max(a.lengths[b], 0), a.k_len);
}

// Span [x, y) of keys that row i of batch entry b (n keys in use) sees; empty spans come out as x = y.
__device__ __forceinline__ int2 row_span(const Prob& a, int b, int i, int n) {
    int lo, hi;
    if (a.first) {
        const int64_t at = b * a.span_stride + i;
        lo = max(a.first[at], 0);
        hi = min(a.end[at], n);
    } else {
        const int pos = n - a.q_len + i;
        hi = a.causal ? min(pos + 1, n) : n;
        lo = a.window > 0 ? max(pos - a.window + 1, 0) : 0;
    }
    hi = max(hi, 0);
    return make_int2(min(lo, hi), hi);
}

// A row that sees keys but none above a score of -infinity has no softmax and is NaN; a row that sees nothing is zeros.
// Kernels that join parts of a row tell the two by the maximum of an unfinished row: LOWEST, or -infinity for a row
// that sees nothing.  Both have a sum of zero.
constexpr float LOWEST = -3.402823466e38f;
__device__ __forceinline__ float not_a_number() { return __int_as_float(0x7fffffff); }
__device__ __forceinline__ float sum_or_nan(float l, bool sees) { return l == 0.f && sees ? not_a_number() : l; }

// A rounded output with the eight bits kept below it, in units of 2^8 (bf16) or 2^5 (fp16) last places of fp32.
// delta = d_o . o summed from rounded outputs would be the largest error of dq and dk after their own rounding and
// that of dS.
template <bool F16>
__device__ __forceinline__ float with_low(float back, int low) {
    return __int_as_float(__float_as_int(back) + low * (F16 ? 32 : 256));
}

// Launchers (fd_attn_simt.cu).
int simt_forward(const Prob& a, int dtype, cudaStream_t s);
int simt_backward(const Prob& a, int dtype, float* delta, cudaStream_t s);   // delta: batch * heads * q_len floats

}  // namespace attn
}  // namespace fd
