// Tensor-core attention kernels: what fd_attn_fwd.cu and fd_attn_bwd.cu share.
#pragma once
#include "fd_attn.cuh"
#include "fd_tc_common.cuh"

namespace fd {
namespace attn {

constexpr int T = 128;                          // rows of a tile, on both sides
constexpr uint32_t BOX_BYTES = T * 128;         // one TMA box: 128 rows of 64 16-bit coordinates, 128-byte swizzle
constexpr uint64_t WAIT_NS = 2000000000ull;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

// Tensor-core kernels take 16-bit heads of a multiple of 8 coordinates up to
// 128 whose rows start on 16-byte boundaries (TMA's rule); the rest runs on the
// CUDA cores.
inline bool tma_view(const View& v, const int64_t (&extent)[3]) {
    if ((uintptr_t)v.p & 15) return false;
    const int64_t st[3] = {v.sb, v.ss, v.sh};
    for (int i = 0; i < 3; ++i)
        if (extent[i] > 1 && (st[i] <= 0 || st[i] % 8 || st[i] >= ((int64_t)1 << 38))) return false;
    return true;
}

// 4-D map (coordinate, row, head, batch) of one operand, boxes of 64 x 128 x 1 x 1.
int make_head_map(CUtensorMap* map, const View& v, int64_t rows, int heads, int batch, int dim, bool f16);

__device__ __forceinline__ uint64_t kmajor(uint32_t base, int ks) {
    return ptx::sw128_kmajor_desc(base + (uint32_t)(ks >> 2) * BOX_BYTES + (uint32_t)(ks & 3) * 32);
}
// The same tile with its rows as the contracted index: step ks covers rows 16 ks .. 16 ks + 15.
__device__ __forceinline__ uint64_t mnmajor(uint32_t base, int ks) {
    return ptx::sw128_mnmajor_desc(base + (uint32_t)ks * 2048, BOX_BYTES);
}

// Scores in base 2 from the raw products: x = c s, or with a cap
// x = cap log2(e) tanh(s scale / cap), minus slope log2(e) |distance|.
struct Score {
    float c;            // scale log2(e); with a cap: scale / cap
    float cap2;         // cap log2(e), 0 without a cap
    float slope2;       // slope log2(e)
};

// tanh of N arguments.  |u| <= 0.6 for all 32 lanes (scores well inside their cap,
// the usual case): an odd degree-9 polynomial on the FMA pipe in packed pairs,
// absolute error 8.5e-8 (least-squares fit on Chebyshev nodes).  Otherwise
// 1 - 2 / (1 + e^2u) with two MUFU operations, absolute error 2e-7: three MUFU
// operations per pair with the softmax's own would make MUFU the bound.
template <int N>
__device__ __forceinline__ void tanh_n(float (&u)[N]) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, fabsf(u[i]));
    if (__all_sync(~0u, top <= 0.6f)) {
        const uint64_t c4 = ptx::pack2(0.01548669f, 0.01548669f), c3 = ptx::pack2(-0.052109625f, -0.052109625f);
        const uint64_t c2 = ptx::pack2(0.13310358f, 0.13310358f), c1 = ptx::pack2(-0.33332324f, -0.33332324f);
        const uint64_t c0 = ptx::pack2(0.99999994f, 0.99999994f), zero = ptx::pack2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const uint64_t x = ptx::pack2(u[i], u[i + 1]);
            const uint64_t y = ptx::fma2(x, x, zero);
            uint64_t p = ptx::fma2(c4, y, c3);
            p = ptx::fma2(p, y, c2);
            p = ptx::fma2(p, y, c1);
            p = ptx::fma2(p, y, c0);
            p = ptx::fma2(p, x, zero);
            uint32_t a, b;
            ptx::unpack2(p, a, b);
            u[i] = __uint_as_float(a);
            u[i + 1] = __uint_as_float(b);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            // e^2u overflows to infinity (tanh 1) and underflows to 0 (tanh -1); NaN stays NaN
            const float e = ptx::ex2_mufu(u[i] * (2.f * LOG2E));
            u[i] = fmaf(-2.f, ptx::rcp_mufu(1.f + e), 1.f);
        }
    }
}

// Wait that goes on after an abort: for copies in flight that must land before the block ends.
__device__ __forceinline__ void wait_landed(uint64_t* b, uint32_t parity) {
    const uint64_t t0 = ptx::globaltimer();
    while (!ptx::mbar_try_wait(b, parity) && ptx::globaltimer() - t0 < WAIT_NS) {
    }
}

__device__ __forceinline__ int warp_min(int x) { return __reduce_min_sync(~0u, x); }
__device__ __forceinline__ int warp_max(int x) { return __reduce_max_sync(~0u, x); }

// Launchers of the tensor-core kernels.
bool tc_applies(const Prob& a, int dtype, bool backward);
int tc_forward(const Prob& a, int dtype, cudaStream_t s);
// Few rows against many keys (fd_attn_rows.cu), where tc_applies: up to MAX_ROWS query rows per key head; above,
// the 128-row tcgen05 tiles are full enough.
constexpr int MAX_ROWS = 64;
bool rows_applies(const Prob& a);
size_t rows_bytes(int dim);
int rows_forward(const Prob& a, int dtype, void* workspace, cudaStream_t s);
size_t tc_backward_bytes(int64_t batch, int64_t heads, int64_t q_len);
int tc_backward(const Prob& a, int dtype, void* workspace, cudaStream_t s);

}  // namespace attn
}  // namespace fd
