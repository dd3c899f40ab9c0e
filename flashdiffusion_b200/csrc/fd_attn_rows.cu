// Softmax attention of few query rows against many keys: the newest tokens of
// each sequence and a cache, and any call of at most MAX_ROWS query rows per key
// head.  Bandwidth-bound: every visible key and value is read once, and the
// arithmetic of up to 16 rows (the query heads that share a key head, times the
// new tokens) rides on one mma.sync tile, whose 16 rows would leave 112 of a
// tcgen05 tile empty.
//
// Work split: the keys in use come from device memory, so the split is made on
// the device.  All (sequence, key head, row tile) pairs are cut into units of 64
// keys, laid end to end, and every CTA of a fixed grid takes an equal run of
// units; lengths from 1 to the longest fill the SMs evenly.  A pair cut between
// CTAs leaves (m, l, O) partials that join_kernel sums in CTA order (the same
// bits at every call); a pair inside one CTA is finished there.
//
// Loads go from global memory to registers in 16-byte pieces and are MMA
// fragments as they are: the order of the contracted coordinate in Q K^T is free
// (Q is loaded the same way), and so is the order of output coordinates in P V;
// the pairs of keys that a P V fragment wants are put together by byte
// permutes.  No shared memory, no barrier in the loop.  P is split in two
// 16-bit parts, so that it adds no rounding of its own: the second product is
// hidden behind the loads.
#include <algorithm>

#include "fd_attn_tc.cuh"

namespace fd {
namespace attn {
namespace rows {

constexpr int WARPS = 4;
constexpr int UNIT = 16 * WARPS;      // keys of a unit: 16 per warp
constexpr int CTAS_PER_SM = 2;

struct Range {
    int lo, hi;   // keys seen by any row of the sequence, lo on a multiple of 16
};

__device__ __forceinline__ Range key_range(const Prob& a, int b) {
    const int n = keys_of(a, b);
    int lo = 0x7fffffff, hi = 0;
    if (a.first) {
        for (int i = 0; i < a.q_len; ++i) {
            const int2 s = row_span(a, b, i, n);
            if (s.y > s.x) {
                lo = min(lo, s.x);
                hi = max(hi, s.y);
            }
        }
    } else {   // both ends grow with the row
        hi = row_span(a, b, a.q_len - 1, n).y;
        lo = row_span(a, b, 0, n).x;
    }
    if (hi <= lo) return {0, 0};
    return {lo & ~15, hi};
}

__device__ __forceinline__ int64_t units_of(const Prob& a, int b) {
    const Range r = key_range(a, b);
    return (r.hi - r.lo + UNIT - 1) / UNIT;
}

struct Plan {
    int pairs;        // (key head, row tile) pairs of a sequence
    int row_tiles, rows;
    int ctas;
};

__device__ __forceinline__ int64_t cut(int64_t total, int ctas, int c) { return total * c / ctas; }

struct Place {
    int b;             // sequence
    int64_t before;    // units of the sequences before it
    int64_t total;
};

// Sum of the units of all sequences, and either the sequence that holds CTA c's
// first unit (c >= 0) or the units before sequence b (c < 0).  Every warp does it
// for itself: no barrier.
__device__ Place find(const Prob& a, const Plan& p, int c, int b) {
    const int lane = threadIdx.x & 31;
    const int per = (a.batch + 31) / 32, b0 = min(lane * per, a.batch), b1 = min(b0 + per, a.batch);
    int64_t sum = 0, part = 0;
    for (int i = b0; i < b1; ++i) {
        const int64_t u = units_of(a, i) * p.pairs;
        sum += u;
        if (i < b) part += u;
    }
    int64_t incl = sum;
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(~0u, incl, o);
        if (lane >= o) incl += x;
    }
    Place r;
    r.total = __shfl_sync(~0u, incl, 31);
    if (c < 0) {
        for (int o = 16; o; o >>= 1) part += __shfl_xor_sync(~0u, part, o);
        r.b = b;
        r.before = part;
        return r;
    }
    const int64_t u = cut(r.total, p.ctas, c);
    int64_t before = incl - sum;
    const bool mine = u >= before && u < incl;
    int at = b0;
    if (mine)
        for (;; ++at) {
            const int64_t x = units_of(a, at) * p.pairs;
            if (u < before + x) break;
            before += x;
        }
    const int src = __ffs(__ballot_sync(~0u, mine)) - 1;
    r.b = src < 0 ? a.batch : __shfl_sync(~0u, at, src);
    r.before = src < 0 ? r.total : __shfl_sync(~0u, before, src);
    return r;
}

template <bool F16>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    if (F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <bool F16>
__device__ __forceinline__ float2 unpack16(uint32_t w) {
    if (F16) return __half22float2(*(__half2*)&w);
    return __bfloat1622float2(*(__nv_bfloat162*)&w);
}

template <bool F16>
__device__ __forceinline__ float one16(uint16_t w) {
    return F16 ? __half2float(__ushort_as_half(w)) : __bfloat162float(__ushort_as_bfloat16(w));
}

__device__ __forceinline__ uint4 load16(const uint16_t* p, bool there) {
    return there ? __ldg((const uint4*)p) : make_uint4(0, 0, 0, 0);
}

// Floats of one partial: O of 16 rows, then their m and l.
template <int DP>
constexpr int PART = 16 * DP + 32;

// out[gr, d .. d + 8) = acc / l, and the row's lse with its first piece
template <bool F16>
__device__ __forceinline__ void store_row(const Prob& a, int b, int hk, int gr, int d, const float (&acc)[8], float m,
                                          float l) {
    const int i = gr / a.group, h = hk * a.group + gr % a.group;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (d < a.dim) {
        uint4 w;
        w.x = ptx::pack16<F16>(acc[0] * inv, acc[1] * inv);
        w.y = ptx::pack16<F16>(acc[2] * inv, acc[3] * inv);
        w.z = ptx::pack16<F16>(acc[4] * inv, acc[5] * inv);
        w.w = ptx::pack16<F16>(acc[6] * inv, acc[7] * inv);
        *(uint4*)((uint16_t*)a.o.p + b * a.o.sb + (int64_t)i * a.o.ss + h * a.o.sh + d) = w;
    }
    if (d == 0 && a.lse) a.lse[((int64_t)b * a.heads + h) * a.q_len + i] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
}

// Row r of a pair: query i = r / group, head hk * group + r % group.
template <int DP, bool F16>
__global__ void __launch_bounds__(WARPS * 32, CTAS_PER_SM)
rows_kernel(const __grid_constant__ Prob a, const __grid_constant__ Plan p, float* __restrict__ parts) {
    constexpr int KI = DP / 32, VB = DP / 64;
    __shared__ float so[WARPS][16][DP + 4];
    __shared__ float sm[WARPS][16], sl[WARPS][16];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    Place at = find(a, p, blockIdx.x, 0);
    int64_t u = cut(at.total, p.ctas, blockIdx.x);
    const int64_t u0 = u, u1 = cut(at.total, p.ctas, blockIdx.x + 1);
    const float c = a.cap > 0.f ? a.scale / a.cap : a.scale * LOG2E, cap2 = a.cap * LOG2E;
    while (u < u1 && at.b < a.batch) {
        const int b = at.b;
        const Range kr = key_range(a, b);
        const int64_t ub = (kr.hi - kr.lo + UNIT - 1) / UNIT;
        if (u >= at.before + ub * p.pairs) {
            at.before += ub * p.pairs;
            ++at.b;
            continue;
        }
        const int pair = (int)((u - at.before) / ub);
        const int blk = (int)((u - at.before) - (int64_t)pair * ub);
        const int take = (int)min(ub - blk, u1 - u);
        const bool whole = blk == 0 && take == ub;
        const int hk = pair / p.row_tiles, rt = pair - hk * p.row_tiles;
        const int n = keys_of(a, b);

        // this thread's rows: g and g + 8 of the tile
        uint32_t q[2][KI][4];
        int2 sp[2];
        int pos[2];
        float slope2[2], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            const int r = rt * 16 + g + 8 * z;
            const bool real = r < p.rows;
            const int i = real ? r / a.group : 0, h = hk * a.group + (real ? r % a.group : 0);
            sp[z] = real ? row_span(a, b, i, n) : make_int2(0, 0);
            pos[z] = n - a.q_len + i;
            slope2[z] = a.slopes ? a.slopes[h] * LOG2E : 0.f;
            const uint16_t* qr = (const uint16_t*)a.q.p + b * a.q.sb + i * a.q.ss + h * a.q.sh;
#pragma unroll
            for (int k = 0; k < KI; ++k) {
                const int d = 32 * k + 8 * t;
                const uint4 x = load16(qr + d, real && d < a.dim);
                q[z][k][0] = x.x;
                q[z][k][1] = x.y;
                q[z][k][2] = x.z;
                q[z][k][3] = x.w;
            }
        }
        // keys that every real row sees: [flo, fhi)
        int flo = max(sp[0].y > sp[0].x ? sp[0].x : 0, sp[1].y > sp[1].x ? sp[1].x : 0);
        int fhi = 0x7fffffff;
        bool hole = false;
#pragma unroll
        for (int z = 0; z < 2; ++z)
            if (rt * 16 + g + 8 * z < p.rows) {
                fhi = min(fhi, sp[z].y);
                hole = hole || sp[z].y <= sp[z].x;
            }
        flo = warp_max(flo);
        fhi = warp_min(fhi);
        hole = __any_sync(~0u, hole);

        const uint16_t* kb = (const uint16_t*)a.k.p + b * a.k.sb + hk * a.k.sh;
        const uint16_t* vb = (const uint16_t*)a.v.p + b * a.v.sb + hk * a.v.sh;
        float o[VB][8][4];
#pragma unroll
        for (int i = 0; i < VB; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int z = 0; z < 4; ++z) o[i][e][z] = 0.f;

        const int k_begin = kr.lo + blk * UNIT + warp * 16, k_end = min(kr.hi, kr.lo + (blk + take) * UNIT);
        uint4 kx[2][KI];
        auto load_k = [&](int k0) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int key = k0 + 8 * j + g;
#pragma unroll
                for (int k = 0; k < KI; ++k)
                    kx[j][k] = load16(kb + (int64_t)key * a.k.ss + 32 * k + 8 * t, key < k_end && 32 * k + 8 * t < a.dim);
            }
        };
        if (k_begin < k_end) load_k(k_begin);
#pragma unroll 1
        for (int k0 = k_begin; k0 < k_end; k0 += UNIT) {
            uint4 vx[4][VB];
#pragma unroll
            for (int z = 0; z < 4; ++z) {
                const int key = k0 + 2 * t + (z & 1) + 8 * (z >> 1);
#pragma unroll
                for (int i = 0; i < VB; ++i)
                    vx[z][i] = load16(vb + (int64_t)key * a.v.ss + 64 * i + 8 * g, key < k_end && 64 * i + 8 * g < a.dim);
            }
            float s[2][4];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int z = 0; z < 4; ++z) s[j][z] = 0.f;
#pragma unroll
                for (int k = 0; k < KI; ++k) {
                    mma<F16>(s[j], q[0][k][0], q[1][k][0], q[0][k][1], q[1][k][1], kx[j][k].x, kx[j][k].y);
                    mma<F16>(s[j], q[0][k][2], q[1][k][2], q[0][k][3], q[1][k][3], kx[j][k].z, kx[j][k].w);
                }
            }
            if (k0 + UNIT < k_end) load_k(k0 + UNIT);
            const bool edge = k0 < flo || k0 + 16 > fhi || hole;
            // s[j][z]: row g + 8 (z / 2), key k0 + 8 j + 2 t + z % 2
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    const int key = k0 + 8 * j + 2 * t + (z & 1);
                    float x = s[j][z] * c;
                    if (cap2 > 0.f) {
                        const float e = ptx::ex2_mufu(x * (2.f * LOG2E));
                        x = cap2 * fmaf(-2.f, ptx::rcp_mufu(1.f + e), 1.f);
                    }
                    x = fmaf(-slope2[z >> 1], fabsf((float)(pos[z >> 1] - key)), x);
                    if (edge && (key < sp[z >> 1].x || key >= sp[z >> 1].y)) x = -INFINITY;
                    s[j][z] = x;
                }
            uint32_t ph[2][2], pl[2][2];   // [row g / g + 8][key block]
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                float top = fmaxf(fmaxf(s[0][2 * z], s[0][2 * z + 1]), fmaxf(s[1][2 * z], s[1][2 * z + 1]));
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
                const float mn = fmaxf(m[z], top), base = mn == -INFINITY ? 0.f : mn;
                const float fix = ptx::ex2_mufu(m[z] - base);
                if (__any_sync(~0u, top > m[z])) {
#pragma unroll
                    for (int i = 0; i < VB; ++i)
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            o[i][e][2 * z] *= fix;
                            o[i][e][2 * z + 1] *= fix;
                        }
                }
                m[z] = mn;
                l[z] *= fix;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float e0 = ptx::ex2_mufu(s[j][2 * z] - base), e1 = ptx::ex2_mufu(s[j][2 * z + 1] - base);
                    l[z] += e0 + e1;
                    ph[z][j] = ptx::pack16<F16>(e0, e1);
                    const float2 hi = unpack16<F16>(ph[z][j]);
                    pl[z][j] = ptx::pack16<F16>(e0 - hi.x, e1 - hi.y);
                }
            }
            bool bad = false;
            if (edge) {
                // zero times a NaN or an infinity of a masked place would reach the row: such elements of V
                // become zeros here and are given back below to the rows that see them
                constexpr uint32_t EXP = F16 ? 0x7c00u : 0x7f80u;
#pragma unroll
                for (int z = 0; z < 4; ++z)
#pragma unroll
                    for (int i = 0; i < VB; ++i) {
                        uint32_t(&w)[4] = reinterpret_cast<uint32_t(&)[4]>(vx[z][i]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if ((w[e] & EXP) == EXP) { w[e] &= 0xffff0000u; bad = true; }
                            if (((w[e] >> 16) & EXP) == EXP) { w[e] &= 0xffffu; bad = true; }
                        }
                    }
                bad = __any_sync(~0u, bad);
            }
#pragma unroll
            for (int i = 0; i < VB; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t w0 = reinterpret_cast<uint32_t(&)[4]>(vx[0][i])[e], w1 = reinterpret_cast<uint32_t(&)[4]>(vx[1][i])[e];
                    const uint32_t w2 = reinterpret_cast<uint32_t(&)[4]>(vx[2][i])[e], w3 = reinterpret_cast<uint32_t(&)[4]>(vx[3][i])[e];
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const uint32_t b0 = __byte_perm(w0, w1, y ? 0x7632 : 0x5410), b1 = __byte_perm(w2, w3, y ? 0x7632 : 0x5410);
                        mma<F16>(o[i][2 * e + y], ph[0][0], ph[1][0], ph[0][1], ph[1][1], b0, b1);
                        mma<F16>(o[i][2 * e + y], pl[0][0], pl[1][0], pl[0][1], pl[1][1], b0, b1);
                    }
                }
            if (bad) {
                for (int key = k0; key < min(k0 + 16, k_end); ++key) {
                    const uint16_t* vr = vb + (int64_t)key * a.v.ss;
#pragma unroll
                    for (int i = 0; i < VB; ++i)
#pragma unroll
                        for (int e = 0; e < 8; ++e)
#pragma unroll
                            for (int y = 0; y < 2; ++y) {
                                const int d = 64 * i + 16 * t + 8 * y + e;
                                if (d >= a.dim) continue;
                                constexpr uint16_t EXP = F16 ? 0x7c00 : 0x7f80;
                                const uint16_t w = vr[d];
                                if ((w & EXP) != EXP) continue;
                                if (key >= sp[0].x && key < sp[0].y) o[i][e][y] += one16<F16>(w);
                                if (key >= sp[1].x && key < sp[1].y) o[i][e][2 + y] += one16<F16>(w);
                            }
                }
            }
        }
        // ---- the four warps' sums meet
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            l[z] += __shfl_xor_sync(~0u, l[z], 1);
            l[z] += __shfl_xor_sync(~0u, l[z], 2);
            if (t == 0) {
                sm[warp][g + 8 * z] = m[z];
                sl[warp][g + 8 * z] = l[z];
            }
#pragma unroll
            for (int i = 0; i < VB; ++i)
#pragma unroll
                for (int y = 0; y < 2; ++y)
#pragma unroll
                    for (int e = 0; e < 8; e += 4)
                        *(float4*)&so[warp][g + 8 * z][64 * i + 16 * t + 8 * y + e] =
                            make_float4(o[i][e][2 * z + y], o[i][e + 1][2 * z + y], o[i][e + 2][2 * z + y], o[i][e + 3][2 * z + y]);
        }
        __syncthreads();
        float* part = parts + ((int64_t)blockIdx.x * 2 + (u == u0 ? 0 : 1)) * PART<DP>;
        for (int x = threadIdx.x; x < 16 * (DP / 8); x += WARPS * 32) {
            const int r = x / (DP / 8), d = x % (DP / 8) * 8, gr = rt * 16 + r;
            if (gr >= p.rows) continue;
            float top = sm[0][r];
#pragma unroll
            for (int w = 1; w < WARPS; ++w) top = fmaxf(top, sm[w][r]);
            const float base = top == -INFINITY ? 0.f : top;
            float acc[8] = {}, lsum = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float f = ptx::ex2_mufu(sm[w][r] - base);
                lsum = fmaf(f, sl[w][r], lsum);
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[e] = fmaf(f, so[w][r][d + e], acc[e]);
            }
            if (!whole) {
                *(float4*)(part + r * DP + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
                *(float4*)(part + r * DP + d + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
                if (d == 0) {
                    part[16 * DP + r] = top;
                    part[16 * DP + 16 + r] = lsum;
                }
                continue;
            }
            store_row<F16>(a, b, hk, gr, d, acc, top, lsum);
        }
        __syncthreads();
        u += take;
    }
}

// Pairs that were cut: their partials in CTA order.  Pairs that see no key: zeros.
template <int DP, bool F16>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ Prob a, const __grid_constant__ Plan p,
                                                   const float* __restrict__ parts, int64_t per_block) {
    const int64_t all = (int64_t)a.batch * p.pairs;
    const int64_t p0 = min(blockIdx.x * per_block, all), p1 = min(p0 + per_block, all);
    if (p0 >= p1) return;
    Place at = find(a, p, -1, (int)(p0 / p.pairs));
    auto owner = [&](int64_t u) {
        int c = (int)min((int64_t)p.ctas - 1, u * p.ctas / at.total);
        while (c + 1 < p.ctas && cut(at.total, p.ctas, c + 1) <= u) ++c;
        while (c > 0 && cut(at.total, p.ctas, c) > u) --c;
        return c;
    };
    for (int64_t x = p0; x < p1; ++x) {
        const int b = (int)(x / p.pairs), pair = (int)(x - (int64_t)b * p.pairs);
        const int64_t ub = units_of(a, b);
        if (b != at.b) {
            at.before += units_of(a, at.b) * p.pairs;
            at.b = b;
        }
        const int hk = pair / p.row_tiles, rt = pair - hk * p.row_tiles;
        const int64_t ua = at.before + pair * ub, uz = ua + ub;
        const int c0 = ub ? owner(ua) : 0, c1 = ub ? owner(uz - 1) : 0;
        if (ub && c0 == c1) continue;
        for (int y = threadIdx.x; y < 16 * (DP / 8); y += 128) {
            const int r = y / (DP / 8), d = y % (DP / 8) * 8, gr = rt * 16 + r;
            if (gr >= p.rows) continue;
            float acc[8] = {}, m = -INFINITY, l = 0.f;
            for (int cc = c0; ub && cc <= c1; ++cc) {
                const int64_t start = cut(at.total, p.ctas, cc);
                if (start == cut(at.total, p.ctas, cc + 1)) continue;
                const float* part = parts + ((int64_t)cc * 2 + (start >= ua ? 0 : 1)) * PART<DP>;
                const float pm = part[16 * DP + r], pl = part[16 * DP + 16 + r];
                const float4 v0 = *(const float4*)(part + r * DP + d), v1 = *(const float4*)(part + r * DP + d + 4);
                const float mn = fmaxf(m, pm), base = mn == -INFINITY ? 0.f : mn;
                const float f0 = ptx::ex2_mufu(m - base), f1 = ptx::ex2_mufu(pm - base);
                m = mn;
                l = fmaf(l, f0, pl * f1);
                const float v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[e] = fmaf(acc[e], f0, v[e] * f1);
            }
            store_row<F16>(a, b, hk, gr, d, acc, m, l);
        }
    }
}

template <int DP, bool F16>
int launch(const Prob& a, float* parts, cudaStream_t s) {
    Plan p;
    p.rows = a.group * a.q_len;
    p.row_tiles = (int)cdiv(p.rows, 16);
    p.pairs = a.kv_heads * p.row_tiles;
    p.ctas = num_sms() * CTAS_PER_SM;
    rows_kernel<DP, F16><<<p.ctas, WARPS * 32, 0, s>>>(a, p, parts);
    FD_CUDA_TRY(cudaGetLastError());
    const int64_t all = (int64_t)a.batch * p.pairs, blocks = std::min<int64_t>(all, 8 * num_sms());
    join_kernel<DP, F16><<<(unsigned)blocks, 128, 0, s>>>(a, p, parts, cdiv(all, blocks));
    FD_CUDA_TRY(cudaGetLastError());
    return FD_OK;
}

}  // namespace rows

bool rows_applies(const Prob& a) { return (int64_t)a.group * a.q_len <= MAX_ROWS; }

size_t rows_bytes(int dim) {
    return sizeof(float) * 2 * (size_t)num_sms() * rows::CTAS_PER_SM * (dim <= 64 ? rows::PART<64> : rows::PART<128>);
}

int rows_forward(const Prob& a, int dtype, void* workspace, cudaStream_t s) {
    float* parts = (float*)workspace;
    if (dtype == FD_DTYPE_F16)
        return a.dim <= 64 ? rows::launch<64, true>(a, parts, s) : rows::launch<128, true>(a, parts, s);
    return a.dim <= 64 ? rows::launch<64, false>(a, parts, s) : rows::launch<128, false>(a, parts, s);
}

}  // namespace attn
}  // namespace fd
