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

// Tensor-core kernels take 16-bit heads of a multiple of 8 coordinates, up to 256
// forward and 128 in the gradients, whose rows start on 16-byte boundaries (TMA's
// rule); the rest runs on the CUDA cores.
inline bool tma_view(const View& v, const int64_t (&extent)[3]) {
    if ((uintptr_t)v.p & 15) return false;
    const int64_t st[3] = {v.sb, v.ss, v.sh};
    for (int i = 0; i < 3; ++i)
        if (extent[i] > 1 && (st[i] <= 0 || st[i] % 8 || st[i] >= ((int64_t)1 << 38))) return false;
    return true;
}

// 4-D map (coordinate, row, head, batch) of one operand, boxes of 64 x 128 x 1 x 1.
int make_head_map(CUtensorMap* map, const View& v, int64_t rows, int heads, int batch, int dim, bool f16);

// ---- tensor-core products, issued by a whole warp with one elected lane.
// Everything but the instruction itself is the same in all 32 lanes and stays in
// uniform registers, where tcgen05.mma wants its operands: under `if (lane == 0)`
// every descriptor word is moved there first, and issuing cost about 115 cycles an
// instruction (3,700 of the 4,800 cycles of a gradient tile) against the 64 that
// the tensor core needs for it.
__device__ __forceinline__ uint32_t elect_lane() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p;
}
__device__ __forceinline__ void mma_ss(uint32_t lead, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t more) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(more), "r"(lead)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t more) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(more), "r"(lead)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t lead, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(ptx::smem_u32(bar)), "r"(lead)
        : "memory");
}
// A wait of the whole warp, with an answer that is the same in all lanes.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort, int* status) {
    return __all_sync(~0u, ptx::wait_bounded(bar, parity, abort, status, WAIT_NS));
}

// D[128 x 128] = A B^T over DP coordinates (`kd` steps of 16 are not zero), both tiles as TMA left them.
template <int DP>
__device__ __forceinline__ void product_rows(uint32_t lead, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, int kd) {
    const uint64_t da = ptx::sw128_kmajor_desc(a), db = ptx::sw128_kmajor_desc(b);
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
        const uint32_t off = ((ks >> 2) * BOX_BYTES + (ks & 3) * 32) >> 4;
        if (ks < kd) mma_ss(lead, d, da + off, db + off, idesc, ks > 0);
    }
}
// D[128 x N] (+)= P B: P 16-bit in TMEM, the words of keys 32 x .. 32 x + 31 at p + (x / PER) * STEP + (x % PER) * 16;
// the rows of B, as TMA left them, are the contracted index.
template <int PER, int STEP>
__device__ __forceinline__ void product_sum(uint32_t lead, uint32_t d, uint32_t p, uint32_t b, uint32_t idesc, bool more) {
    const uint64_t db = ptx::sw128_mnmajor_desc(b, BOX_BYTES);
#pragma unroll
    for (int ks = 0; ks < T / 16; ++ks)
        mma_ts(lead, d, p + (ks / 2 / PER) * STEP + (ks / 2 % PER) * 16 + (ks & 1) * 8, db + ks * (2048 >> 4), idesc, more || ks > 0);
}

// Scores in base 2 from the raw products, 32 columns of a row as 16 packed pairs:
//   x = c s + add                       (no cap; c = scale log2(e))
//   x = cap2 tanh(c s) + add            (c = scale / cap, cap2 = cap log2(e))
// minus slope2 |distance| (slope2 = slope log2(e)).
//
// The tanh has two forms.  |c s| <= 0.45 (scores well inside their cap, the usual
// case): an odd degree-7 polynomial in the raw product, with c and cap2 in its
// coefficients, on the FMA pipe in packed pairs (absolute error of the tanh 9e-8;
// weighted least squares on Chebyshev nodes).  Otherwise 1 - 2 / (1 + e^2u) with
// two MUFU operations, absolute error 2e-7: with the softmax's own that makes
// three MUFU operations a pair, and MUFU the bound.
struct Score {
    uint64_t c, cap2;            // both halves the same
    uint64_t b0, b1, b2, b3;     // cap2 tanh(c s) = s (b0 + b1 s^2 + b2 s^4 + b3 s^6)
    uint64_t shrink;             // -1 / cap2^2: 1 - tanh^2 = 1 + shrink x^2
    float limit;                 // |s| up to which it holds
    bool capped;
    __device__ explicit Score(const Prob& a) {
        capped = a.cap > 0.f;
        const float f = capped ? a.scale / a.cap : a.scale * LOG2E, top = a.cap * LOG2E;
        c = ptx::both2(f);
        cap2 = ptx::both2(top);
        b0 = ptx::both2(0.99999905f * f * top);
        b1 = ptx::both2(-0.33326662f * f * f * f * top);
        b2 = ptx::both2(0.13208261f * f * f * f * f * f * top);
        b3 = ptx::both2(-0.04522878f * f * f * f * f * f * f * f * top);
        shrink = ptx::both2(capped ? -1.f / (top * top) : 0.f);
        // Steep enough for a coefficient to overflow: the polynomial is never taken.  So flat that b3, b2 or b1 leaves
        // the normal numbers (caps are 1e-3 and more): it is taken as far as what is left of it is good to 1e-8.
        // s^2 must not overflow either.
        const float flat = fabsf(f), upto = flat >= 2e-5f ? 0.45f : flat >= 2e-7f ? 0.1f : flat >= 1e-11f ? 0.037f : 0.003f;
        limit = !(fabsf(ptx::lo2(b3)) < INFINITY) ? -1.f : flat > 0.f ? fminf(upto / flat, 1e18f) : 1e18f;
    }
    // the factor of s in the polynomial
    __device__ __forceinline__ uint64_t ratio(uint64_t s) const {
        const uint64_t y = ptx::mul2(s, s);
        return ptx::fma2(ptx::fma2(ptx::fma2(b3, y, b2), y, b1), y, b0);
    }
};

__device__ __forceinline__ bool inside32(const uint64_t (&s)[16], float limit) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, fmaxf(fabsf(ptx::lo2(s[i])), fabsf(ptx::hi2(s[i]))));
    return __all_sync(~0u, top <= limit);
}
// x = cap2 tanh(c x).  Each score is a function of its own product alone, and so what lies in masked places, or in
// another row, changes no bit of it: the vote only leaves out the form that no score of the warp takes.
__device__ __forceinline__ void cap32(uint64_t (&x)[16], const Score& sc) {
    if (inside32(x, sc.limit)) {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = ptx::mul2(sc.ratio(x[i]), x[i]);
    } else {
        // e^2u overflows to infinity (tanh 1) and underflows to 0 (tanh -1); NaN stays NaN
        const float c = ptx::lo2(sc.c) * (2.f * LOG2E), top = ptx::lo2(sc.cap2);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float s0 = ptx::lo2(x[i]), s1 = ptx::hi2(x[i]);
            const uint64_t near = ptx::mul2(sc.ratio(x[i]), x[i]);
            const float e0 = ptx::ex2_mufu(s0 * c), e1 = ptx::ex2_mufu(s1 * c);
            const float far0 = fmaf(-2.f * top, ptx::rcp_mufu(1.f + e0), top), far1 = fmaf(-2.f * top, ptx::rcp_mufu(1.f + e1), top);
            x[i] = ptx::pack2(fabsf(s0) <= sc.limit ? ptx::lo2(near) : far0, fabsf(s1) <= sc.limit ? ptx::hi2(near) : far1);
        }
    }
}

// x[i] += from + by * (2 i, 2 i + 1), four independent chains
__device__ __forceinline__ void add_line(uint64_t (&x)[16], float from, float by) {
    uint64_t l[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) l[j] = ptx::pack2(fmaf(by, (float)(2 * j), from), fmaf(by, (float)(2 * j + 1), from));
    const uint64_t step = ptx::both2(8.f * by);
#pragma unroll
    for (int i = 0; i < 16; i += 4)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[i + j] = ptx::add2(x[i + j], l[j]);
            if (i < 12) l[j] = ptx::add2(l[j], step);
        }
}

// x[i] -= slope2 |dist + by * (2 i, 2 i + 1)|, by = 1 or -1: the distances of 32
// pairs.  `side` says what is known of their sign in the whole tile: 1 none is
// negative where it matters, -1 none positive, 0 both.
__device__ __forceinline__ void add_bias(uint64_t (&x)[16], float slope2, float dist, float by, int side) {
    if (side != 0) {
        const float f = side > 0 ? -slope2 : slope2;
        add_line(x, f * dist, f * by);
        return;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float d0 = fabsf(fmaf(by, (float)(2 * i), dist)), d1 = fabsf(fmaf(by, (float)(2 * i + 1), dist));
        x[i] = ptx::pack2(fmaf(-slope2, d0, ptx::lo2(x[i])), fmaf(-slope2, d1, ptx::hi2(x[i])));
    }
}

// Sign of pos - key over positions [p0, p0 + T) and keys [k0, k0 + T), as add_bias takes it.
__device__ __forceinline__ int side_of(const Prob& a, int p0, int k0) {
    if (a.causal || p0 >= k0 + T - 1) return 1;   // causal: pairs with a negative distance are masked
    return p0 + T - 1 <= k0 ? -1 : 0;
}

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// 2^x of a pair on the FMA pipe, as exp2_poly2 of the tile kernels has it (2^j 2^f,
// degree-4 polynomial, relative error 3.6e-6, never below 2^-125), but a NaN does
// not come out as a number that could pass for a weight.
__device__ __forceinline__ uint64_t exp2_fma2(uint64_t x) {
    const uint64_t X = ptx::pack2(max_nan(ptx::lo2(x), -125.f), max_nan(ptx::hi2(x), -125.f));
    const uint64_t SH = ptx::both2(12582912.0f);
    const uint64_t T = ptx::add2(X, SH);
    const uint64_t F = ptx::sub2(X, ptx::sub2(T, SH));
    uint64_t P = ptx::fma2(ptx::both2(0.009782912f), F, ptx::both2(0.055976883f));
    P = ptx::fma2(P, F, ptx::both2(0.2402071f));
    P = ptx::fma2(P, F, ptx::both2(0.6931136f));
    P = ptx::fma2(P, F, ptx::both2(1.0f));
    uint32_t p0, p1, t0, t1;
    ptx::unpack2(P, p0, p1);
    ptx::unpack2(T, t0, t1);
    return ptx::pack2(__uint_as_float(p0 + (t0 << 23)), __uint_as_float(p1 + (t1 << 23)));
}

// 2^x of 16 pairs; POLY of every 4 go to the FMA pipe: MUFU, 16 exponentials a
// clock and SM, is the bound of the softmax.  POLY = 0 where zeros must be zeros.
template <int POLY>
__device__ __forceinline__ void exp32(uint64_t (&x)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        if (i % 4 >= 4 - POLY) x[i] = exp2_fma2(x[i]);
        else x[i] = ptx::pack2(ptx::ex2_mufu(ptx::lo2(x[i])), ptx::ex2_mufu(ptx::hi2(x[i])));
    }
}

// A row's 32 TMEM columns as pairs.
__device__ __forceinline__ void pairs32(const uint32_t (&r)[32], uint64_t (&x)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = ptx::pack2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
}
template <bool F16>
__device__ __forceinline__ void round32(const uint64_t (&x)[16], uint32_t (&p)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] = ptx::pack16<F16>(ptx::lo2(x[i]), ptx::hi2(x[i]));
}
// Pairs outside columns [lo, lo + len) become `value`.
__device__ __forceinline__ void mask32(uint64_t (&x)[16], int lo, uint32_t len, float value) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const bool a = (uint32_t)(2 * i - lo) < len, b = (uint32_t)(2 * i + 1 - lo) < len;
        x[i] = ptx::pack2(a ? ptx::lo2(x[i]) : value, b ? ptx::hi2(x[i]) : value);
    }
}

// Wait that goes on after an abort: for copies in flight that must land before the block ends.
__device__ __forceinline__ void wait_landed(uint64_t* b, uint32_t parity) {
    const uint64_t t0 = ptx::globaltimer();
    while (!ptx::mbar_try_wait(b, parity) && ptx::globaltimer() - t0 < WAIT_NS) {
    }
}

// A tile in shared memory: elements that are NaN or infinite become zeros; true (in all lanes) if there were any.
template <bool F16>
__device__ __forceinline__ bool clear_bad(uint8_t* tile, int bytes, int lane) {
    constexpr uint32_t EXP = F16 ? 0x7c00u : 0x7f80u;
    // zero times x is NaN for a NaN or an infinity and zero for a number: one packed multiply-add for two elements
    float seen = 0.f;
    if (F16) {
        __half2 z[4] = {};
#pragma unroll 8
        for (int i = lane; i < bytes / 16; i += 32) {
            const uint4 x = ((uint4*)tile)[i];
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) z[e] = __hfma2(*(__half2*)&w[e], __half2half2(__ushort_as_half(0)), z[e]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) seen += __low2float(z[e]) + __high2float(z[e]);
    } else {
        __nv_bfloat162 z[4] = {};
#pragma unroll 8
        for (int i = lane; i < bytes / 16; i += 32) {
            const uint4 x = ((uint4*)tile)[i];
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                z[e] = __hfma2(*(__nv_bfloat162*)&w[e], __bfloat162bfloat162(__ushort_as_bfloat16(0)), z[e]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) seen += __low2float(z[e]) + __high2float(z[e]);
    }
    bool bad = seen != 0.f;      // NaN differs from everything
    bad = __any_sync(~0u, bad);
    if (bad) {
        for (int i = lane; i < bytes / 4; i += 32) {
            uint32_t x = ((uint32_t*)tile)[i];
            if ((x & EXP) == EXP) x &= 0xffff0000u;
            if (((x >> 16) & EXP) == EXP) x &= 0xffffu;
            ((uint32_t*)tile)[i] = x;
        }
        ptx::fence_async_shared();
        __syncwarp();
    }
    return bad;
}

__device__ __forceinline__ int warp_min(int x) { return __reduce_min_sync(~0u, x); }
__device__ __forceinline__ int warp_max(int x) { return __reduce_max_sync(~0u, x); }

// The eight bits below a rounded output (with_low reads them): `f` is the unrounded value, `back` the rounded one.
template <bool F16>
__device__ __forceinline__ int low_bits(float f, float back) {
    constexpr int SH = F16 ? 5 : 8;
    if (!(fabsf(back) < INFINITY)) return 0;
    return min(max((__float_as_int(f) - __float_as_int(back) + (1 << (SH - 1))) >> SH, -128), 127);
}
template <bool F16>
__device__ __forceinline__ float2 pair_of(uint32_t w) {
    if (F16) return __half22float2(*(__half2*)&w);
    return __bfloat1622float2(*(__nv_bfloat162*)&w);
}
// Eight outputs, 16-bit to `out` and their low bits to `low` (unless it is null).
template <bool F16>
__device__ __forceinline__ void store8(void* out, int8_t* low, const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = ptx::pack16<F16>(f[2 * i], f[2 * i + 1]);
    *(uint4*)out = make_uint4(w[0], w[1], w[2], w[3]);
    if (low) {
        uint32_t v[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 b = pair_of<F16>(w[i]);
            v[i / 2] |= ((uint32_t)low_bits<F16>(f[2 * i], b.x) & 255) << (i % 2 * 16);
            v[i / 2] |= ((uint32_t)low_bits<F16>(f[2 * i + 1], b.y) & 255) << (i % 2 * 16 + 8);
        }
        *(uint2*)low = make_uint2(v[0], v[1]);
    }
}

// Launchers of the tensor-core kernels.
bool tc_applies(const Prob& a, int dtype, bool backward);
size_t tc_forward_bytes(const Prob& a);   // these two read the sizes and switches of a call only
int tc_forward(const Prob& a, int dtype, void* workspace, cudaStream_t s);
// Few rows against many keys (fd_attn_rows.cu), where tc_applies: up to MAX_ROWS query rows per key head; above,
// the 128-row tcgen05 tiles are full enough.
constexpr int MAX_ROWS = 64;
bool rows_applies(const Prob& a);
size_t rows_bytes(int dim);
int rows_forward(const Prob& a, int dtype, void* workspace, cudaStream_t s);
size_t tc_backward_bytes(const Prob& a);
int tc_backward(const Prob& a, int dtype, void* workspace, cudaStream_t s);

}  // namespace attn
}  // namespace fd
