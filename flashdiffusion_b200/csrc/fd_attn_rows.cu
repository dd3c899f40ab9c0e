// Softmax attention of few query rows against many keys: the newest tokens of
// each sequence and a cache, and any call of at most MAX_ROWS query rows per key
// head.  Bandwidth-bound: every visible key and value is read once, and the
// arithmetic of up to 16 or 32 rows (the query heads that share a key head, times
// the new tokens) rides on mma.sync tiles of 16 rows; a tcgen05 tile has 128.
//
// Work split: the keys in use come from device memory, so the split is made on
// the device.  The keys of all (sequence, key head, row tile) pairs are cut into
// units of 64, laid end to end with SETUP units more for each pair (what its
// start and end cost), and every CTA of a fixed grid takes an equal run: lengths
// from 1 to the longest fill the SMs evenly.  A pair cut between CTAs leaves
// (m, l, O) partials that join_kernel sums in CTA order (the same bits at every
// call); a pair inside one CTA is finished there.
//
// Each warp copies its own 16-key blocks with cp.async into a ring of its own,
// STAGES - 1 blocks ahead and across the ends of pairs, and reads MMA fragments
// from it in 16-byte pieces: the order of the contracted coordinate in Q K^T is
// free (Q is loaded the same way), and so is the order of output coordinates in
// P V; the pairs of keys that a P V fragment wants are put together by byte
// permutes.  P is split in two 16-bit parts, so that it adds no rounding of its
// own: the second product hides behind the loads.
#include <algorithm>

#include "fd_attn_tc.cuh"

namespace fd {
namespace attn {
namespace rows {

constexpr int WARPS = 4;
constexpr int UNIT = 16 * WARPS;      // keys of a unit: 16 per warp
constexpr int CTAS_PER_SM = 2;
constexpr int STAGES = 3;
constexpr int SETUP = 2;

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

// Units of one pair of this range, its SETUP included; 0 for an empty range.
__device__ __forceinline__ int units_of(const Range& r) {
    return r.hi > r.lo ? (r.hi - r.lo + UNIT - 1) / UNIT + SETUP : 0;
}

struct Plan {
    int pairs;        // (key head, row tile) pairs of a sequence
    int row_tiles, rows;
    int ctas;
};

// Equal runs of `total` units for `ctas` CTAs: the first `more` take one more than `each`.
struct Cut {
    int64_t total, each, more;
    int ctas;          // CTAs that have work
    __device__ Cut(int64_t t, int n) : total(t), ctas((int)min((int64_t)n, t)) {
        each = ctas ? t / ctas : 0;
        more = ctas ? t - each * ctas : 0;
    }
    __device__ int64_t start(int c) const { return c >= ctas ? total : each * c + min((int64_t)c, more); }
    __device__ int owner(int64_t u) const {
        const int64_t wide = more * (each + 1);
        return (int)(u < wide ? u / (each + 1) : more + (u - wide) / each);
    }
};

struct Place {
    int b;             // sequence
    int64_t before;    // units of the sequences before it
};

// The units of all sequences and, by `c`, where CTA c's run starts (c >= 0) or
// the units before sequence b (c < 0).  Every warp does it for itself: no barrier.
__device__ Cut find(const Prob& a, const Plan& p, int c, int b, Place& at) {
    const int lane = threadIdx.x & 31;
    const int per = (a.batch + 31) / 32, b0 = min(lane * per, a.batch), b1 = min(b0 + per, a.batch);
    int64_t sum = 0, part = 0;
    for (int i = b0; i < b1; ++i) {
        const int64_t u = (int64_t)units_of(key_range(a, i)) * p.pairs;
        sum += u;
        if (i < b) part += u;
    }
    int64_t incl = sum;
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(~0u, incl, o);
        if (lane >= o) incl += x;
    }
    const Cut cut(__shfl_sync(~0u, incl, 31), p.ctas);
    if (c < 0) {
        for (int o = 16; o; o >>= 1) part += __shfl_xor_sync(~0u, part, o);
        at = {b, part};
        return cut;
    }
    const int64_t u = cut.start(c);
    int64_t before = incl - sum;
    const bool mine = u >= before && u < incl;
    int x = b0;
    if (mine)
        for (;; ++x) {
            const int64_t n = (int64_t)units_of(key_range(a, x)) * p.pairs;
            if (u < before + n) break;
            before += n;
        }
    const int src = __ffs(__ballot_sync(~0u, mine)) - 1;
    at.b = src < 0 ? a.batch : __shfl_sync(~0u, x, src);
    at.before = src < 0 ? cut.total : __shfl_sync(~0u, before, src);
    return cut;
}

// A CTA's run, pair by pair.
struct Walk {
    Place at;
    int64_t u, u1;     // next unit, end of the run
    int b, pair;       // the current pair and its keys [k0, k1) in this run
    int k0, k1;
    bool whole, front; // all of the pair; at the front of the run
    __device__ bool next(const Prob& a, const Plan& p, int64_t u0) {
        while (u < u1 && at.b < a.batch) {
            const Range r = key_range(a, at.b);
            const int ub = units_of(r);
            const int64_t here = (int64_t)ub * p.pairs, off = u - at.before;
            if (off >= here) {
                at.before += here;
                ++at.b;
                continue;
            }
            pair = (uint64_t)off >> 32 ? (int)(off / ub) : (int)((uint32_t)off / (uint32_t)ub);
            const int blk = (int)(off - (int64_t)pair * ub);
            const int take = (int)min((int64_t)(ub - blk), u1 - u);
            b = at.b;
            k0 = r.lo + max(blk - SETUP, 0) * UNIT;
            k1 = min(r.hi, r.lo + max(blk + take - SETUP, 0) * UNIT);
            whole = blk == 0 && take == ub;
            front = u == u0;
            u += take;
            if (k1 > k0) return true;   // else the run ends inside the pair's SETUP units
        }
        return false;
    }
};

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

// 16 bytes to shared memory, zeros where `there` is false (nothing is read then)
__device__ __forceinline__ void copy16(uint32_t dst, const uint16_t* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}

// Floats of one partial: O of 16 MT rows, then their m and l.
template <int DP, int MT>
constexpr int PART = 16 * MT * (DP + 2);

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

template <int DP>
struct Smem {
    static constexpr uint32_t HALF = 16 * DP * 2;                 // K or V of a block
    static constexpr uint32_t RING = WARPS * STAGES * 2 * HALF;
    static constexpr int PIECES = DP / 8 + 1;                     // 16-byte pieces of one lane's sums: O, and m and l
    static constexpr uint32_t BYTES = RING + 2 * PIECES * 32 * 16;
    // two CTAs to an SM: 228 KB, of which each takes 1 KB for itself
    static_assert(CTAS_PER_SM * (BYTES + 1024) <= 228 * 1024, "shared memory budget");
};

// Row r of a pair: query i = r / group, head hk * group + r % group.
template <int DP, bool F16, int MT>
__global__ void __launch_bounds__(WARPS * 32, CTAS_PER_SM)
rows_kernel(const __grid_constant__ Prob a, const __grid_constant__ Plan p, float* __restrict__ parts) {
    using S = Smem<DP>;
    constexpr int KI = DP / 32, VB = DP / 64, CH = DP / 8;   // 16-byte pieces of a row: CH
    extern __shared__ __align__(16) uint8_t smem[];
    float4* meet = (float4*)(smem + S::RING);                 // [2][PIECES][lane]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    asm volatile("griddepcontrol.launch_dependents;");
    Walk w;
    const Cut cut = find(a, p, blockIdx.x, 0, w.at);
    if ((int)blockIdx.x >= cut.ctas) return;
    const int64_t u0 = cut.start(blockIdx.x);
    w.u = u0;
    w.u1 = cut.start(blockIdx.x + 1);
    const float c = a.cap > 0.f ? a.scale / a.cap : a.scale * LOG2E, cap2 = a.cap * LOG2E;
    const uint32_t ring = ptx::smem_u32(smem) + warp * STAGES * 2 * S::HALF;

    // ---- the copies run ahead: block `ahead` of pair `f`
    Walk f = w;
    int fk = 0, fend = 0, wr = 0;
    const uint16_t *fkp = nullptr, *fvp = nullptr;
    auto fetch = [&]() {
        while (fk >= fend) {
            if (!f.next(a, p, u0)) {
                fk = 0x7fffffff;
                fend = 0x7fffffff;
                break;
            }
            const int hk = f.pair / p.row_tiles;
            fk = f.k0 + warp * 16;
            fend = f.k1;
            fkp = (const uint16_t*)a.k.p + f.b * a.k.sb + hk * a.k.sh;
            fvp = (const uint16_t*)a.v.p + f.b * a.v.sb + hk * a.v.sh;
        }
        if (fk < fend) {
            const uint32_t dst = ring + wr * 2 * S::HALF;
#pragma unroll
            for (int x = 0; x < 16 * CH / 32; ++x) {
                const int at = x * 32 + lane, r = at / CH, ch = at % CH, key = fk + r;
                const bool there = key < fend && ch * 8 < a.dim;
                const int64_t kk = there ? key : fk, cc = there ? ch * 8 : 0;
                // pieces are swapped within 128 bytes so that the fragment reads below hit every bank once
                copy16(dst + (r * CH + (ch ^ ((r & 1) << 2))) * 16, fkp + kk * a.k.ss + cc, there);
                copy16(dst + S::HALF + (r * CH + (ch ^ (r & 6))) * 16, fvp + kk * a.v.ss + cc, there);
            }
            fk += UNIT;
            wr = wr + 1 == STAGES ? 0 : wr + 1;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int x = 0; x < STAGES - 1; ++x) fetch();
    int rd = 0;

    while (w.next(a, p, u0)) {
        const int b = w.b, hk = w.pair / p.row_tiles, rt = w.pair - hk * p.row_tiles;
        const int n = keys_of(a, b);
        // this thread's rows: g and g + 8 of each 16-row tile
        uint32_t q[MT][2][KI][4];
        int2 sp[MT][2];
        int pos[MT][2];
        float slope2[MT][2], m[MT][2], l[MT][2];
        int flo = 0, fhi = 0x7fffffff;   // keys that every row sees: [flo, fhi)
        bool hole = false;
#pragma unroll
        for (int y = 0; y < MT; ++y)
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                const int r = (rt * MT + y) * 16 + g + 8 * z;
                const bool real = r < p.rows;
                const int i = real ? r / a.group : 0, h = hk * a.group + (real ? r % a.group : 0);
                sp[y][z] = real ? row_span(a, b, i, n) : make_int2(0, 0);
                pos[y][z] = n - a.q_len + i;
                slope2[y][z] = a.slopes ? a.slopes[h] * LOG2E : 0.f;
                m[y][z] = -INFINITY;
                l[y][z] = 0.f;
                const uint16_t* qr = (const uint16_t*)a.q.p + b * a.q.sb + i * a.q.ss + h * a.q.sh;
#pragma unroll
                for (int k = 0; k < KI; ++k) {
                    const int d = 32 * k + 8 * t;
                    const uint4 x = load16(qr + d, real && d < a.dim);
                    q[y][z][k][0] = x.x;
                    q[y][z][k][1] = x.y;
                    q[y][z][k][2] = x.z;
                    q[y][z][k][3] = x.w;
                }
                if (real) {
                    if (sp[y][z].y > sp[y][z].x) flo = max(flo, sp[y][z].x);
                    else hole = true;
                    fhi = min(fhi, sp[y][z].y);
                }
            }
        flo = warp_max(flo);
        fhi = warp_min(fhi);
        hole = __any_sync(~0u, hole);
        float o[MT][VB][8][4];
#pragma unroll
        for (int y = 0; y < MT; ++y)
#pragma unroll
            for (int i = 0; i < VB; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e)
#pragma unroll
                    for (int z = 0; z < 4; ++z) o[y][i][e][z] = 0.f;

#pragma unroll 1
        for (int k0 = w.k0 + warp * 16; k0 < w.k1; k0 += UNIT) {
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
            __syncwarp();
            const uint32_t sk = ring + rd * 2 * S::HALF, sv = sk + S::HALF;
            rd = rd + 1 == STAGES ? 0 : rd + 1;
            float s[MT][2][4];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int y = 0; y < MT; ++y)
#pragma unroll
                    for (int z = 0; z < 4; ++z) s[y][j][z] = 0.f;
#pragma unroll
                for (int k = 0; k < KI; ++k) {
                    const int r = 8 * j + g;
                    const uint4 x = lds16(sk + (r * CH + ((4 * k + t) ^ ((r & 1) << 2))) * 16);
#pragma unroll
                    for (int y = 0; y < MT; ++y) {
                        mma<F16>(s[y][j], q[y][0][k][0], q[y][1][k][0], q[y][0][k][1], q[y][1][k][1], x.x, x.y);
                        mma<F16>(s[y][j], q[y][0][k][2], q[y][1][k][2], q[y][0][k][3], q[y][1][k][3], x.z, x.w);
                    }
                }
            }
            fetch();
            const bool edge = k0 < flo || k0 + 16 > fhi || hole;
            uint32_t ph[MT][2][2], pl[MT][2][2];   // [row g / g + 8][key block]
#pragma unroll
            for (int y = 0; y < MT; ++y) {
                // s[y][j][z]: row g + 8 (z / 2), key k0 + 8 j + 2 t + z % 2
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        const int key = k0 + 8 * j + 2 * t + (z & 1);
                        float x = s[y][j][z] * c;
                        if (cap2 > 0.f) {
                            const float e = ptx::ex2_mufu(x * (2.f * LOG2E));
                            x = cap2 * fmaf(-2.f, ptx::rcp_mufu(1.f + e), 1.f);
                        }
                        x = fmaf(-slope2[y][z >> 1], fabsf((float)(pos[y][z >> 1] - key)), x);
                        if (edge && (key < sp[y][z >> 1].x || key >= sp[y][z >> 1].y)) x = -INFINITY;
                        s[y][j][z] = x;
                    }
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    float top = fmaxf(fmaxf(s[y][0][2 * z], s[y][0][2 * z + 1]), fmaxf(s[y][1][2 * z], s[y][1][2 * z + 1]));
                    top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
                    if (__any_sync(~0u, top > m[y][z])) {
                        const float mn = fmaxf(m[y][z], top);
                        const float fix = mn == -INFINITY ? 0.f : ptx::ex2_mufu(m[y][z] - mn);
                        m[y][z] = mn;
                        l[y][z] *= fix;
#pragma unroll
                        for (int i = 0; i < VB; ++i)
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                o[y][i][e][2 * z] *= fix;
                                o[y][i][e][2 * z + 1] *= fix;
                            }
                    }
                    const float base = m[y][z] == -INFINITY ? 0.f : m[y][z];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float e0 = ptx::ex2_mufu(s[y][j][2 * z] - base), e1 = ptx::ex2_mufu(s[y][j][2 * z + 1] - base);
                        l[y][z] += e0 + e1;
                        ph[y][z][j] = ptx::pack16<F16>(e0, e1);
                        const float2 hi = unpack16<F16>(ph[y][z][j]);
                        pl[y][z][j] = ptx::pack16<F16>(e0 - hi.x, e1 - hi.y);
                    }
                }
            }
            bool bad = false;
#pragma unroll
            for (int i = 0; i < VB; ++i) {
                uint32_t v[4][4];
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    const int r = 2 * t + (z & 1) + 8 * (z >> 1);
                    const uint4 x = lds16(sv + (r * CH + ((8 * i + g) ^ (r & 6))) * 16);
                    v[z][0] = x.x;
                    v[z][1] = x.y;
                    v[z][2] = x.z;
                    v[z][3] = x.w;
                }
                if (edge) {
                    // zero times a NaN or an infinity of a masked place would reach the row: such elements
                    // of V become zeros here and are given back below to the rows that see them
                    constexpr uint32_t EXP = F16 ? 0x7c00u : 0x7f80u;
#pragma unroll
                    for (int z = 0; z < 4; ++z)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if ((v[z][e] & EXP) == EXP) { v[z][e] &= 0xffff0000u; bad = true; }
                            if (((v[z][e] >> 16) & EXP) == EXP) { v[z][e] &= 0xffffu; bad = true; }
                        }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t b0 = __byte_perm(v[0][e], v[1][e], x ? 0x7632 : 0x5410);
                        const uint32_t b1 = __byte_perm(v[2][e], v[3][e], x ? 0x7632 : 0x5410);
#pragma unroll
                        for (int y = 0; y < MT; ++y) {
                            mma<F16>(o[y][i][2 * e + x], ph[y][0][0], ph[y][1][0], ph[y][0][1], ph[y][1][1], b0, b1);
                            mma<F16>(o[y][i][2 * e + x], pl[y][0][0], pl[y][1][0], pl[y][0][1], pl[y][1][1], b0, b1);
                        }
                    }
            }
            if (__any_sync(~0u, bad)) {
                const uint16_t* vb = (const uint16_t*)a.v.p + b * a.v.sb + hk * a.v.sh;
                for (int key = k0; key < min(k0 + 16, w.k1); ++key) {
                    const uint16_t* vr = vb + (int64_t)key * a.v.ss;
#pragma unroll
                    for (int i = 0; i < VB; ++i)
#pragma unroll
                        for (int e = 0; e < 8; ++e)
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                const int d = 64 * i + 16 * t + 8 * x + e;
                                if (d >= a.dim) continue;
                                constexpr uint16_t EXP = F16 ? 0x7c00 : 0x7f80;
                                const uint16_t h = vr[d];
                                if ((h & EXP) != EXP) continue;
#pragma unroll
                                for (int y = 0; y < MT; ++y) {
                                    if (key >= sp[y][0].x && key < sp[y][0].y) o[y][i][e][x] += one16<F16>(h);
                                    if (key >= sp[y][1].x && key < sp[y][1].y) o[y][i][e][2 + x] += one16<F16>(h);
                                }
                            }
                }
            }
        }
        // ---- the four warps' sums meet: 2 and 3 hand theirs to 0 and 1, then 1 to 0
        float* part = parts + ((int64_t)blockIdx.x * 2 + (w.front ? 0 : 1)) * PART<DP, MT>;
#pragma unroll
        for (int y = 0; y < MT; ++y) {
#pragma unroll
            for (int from = 2; from; from >>= 1) {
                if (warp >= from && warp < 2 * from) {
                    float4* to = meet + (warp - from) * S::PIECES * 32 + lane;
#pragma unroll
                    for (int i = 0; i < VB; ++i)
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            to[(i * 8 + e) * 32] = make_float4(o[y][i][e][0], o[y][i][e][1], o[y][i][e][2], o[y][i][e][3]);
                    to[VB * 8 * 32] = make_float4(m[y][0], m[y][1], l[y][0], l[y][1]);
                }
                __syncthreads();
                if (warp < from) {
                    const float4* in = meet + warp * S::PIECES * 32 + lane;
                    const float4 ml = in[VB * 8 * 32];
                    const float mo[2] = {ml.x, ml.y}, lo[2] = {ml.z, ml.w};
                    float f0[2], f1[2];
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        const float mn = fmaxf(m[y][z], mo[z]), base = mn == -INFINITY ? 0.f : mn;
                        f0[z] = ptx::ex2_mufu(m[y][z] - base);
                        f1[z] = ptx::ex2_mufu(mo[z] - base);
                        m[y][z] = mn;
                        l[y][z] = l[y][z] * f0[z] + lo[z] * f1[z];
                    }
#pragma unroll
                    for (int i = 0; i < VB; ++i)
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const float4 v = in[(i * 8 + e) * 32];
                            o[y][i][e][0] = o[y][i][e][0] * f0[0] + v.x * f1[0];
                            o[y][i][e][1] = o[y][i][e][1] * f0[0] + v.y * f1[0];
                            o[y][i][e][2] = o[y][i][e][2] * f0[1] + v.z * f1[1];
                            o[y][i][e][3] = o[y][i][e][3] * f0[1] + v.w * f1[1];
                        }
                }
                __syncthreads();
            }
            if (warp == 0) {
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    const int pr = y * 16 + g + 8 * z, gr = rt * MT * 16 + pr;
                    float ls = l[y][z];
                    ls += __shfl_xor_sync(~0u, ls, 1);
                    ls += __shfl_xor_sync(~0u, ls, 2);
                    if (gr >= p.rows) continue;
#pragma unroll
                    for (int i = 0; i < VB; ++i)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const int d = 64 * i + 16 * t + 8 * x;
                            float acc[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) acc[e] = o[y][i][e][2 * z + x];
                            if (w.whole) {
                                store_row<F16>(a, b, hk, gr, d, acc, m[y][z], ls);
                            } else {
                                *(float4*)(part + pr * DP + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
                                *(float4*)(part + pr * DP + d + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
                            }
                        }
                    if (!w.whole && t == 0) {
                        part[16 * MT * DP + pr] = m[y][z];
                        part[16 * MT * (DP + 1) + pr] = ls;
                    }
                }
            }
        }
    }
}

// Pairs that were cut: their partials, in CTA order.  Pairs that see no key: zeros.
// Block: one pair after another; up to 256 threads share the (row, 8 coordinates)
// pieces of it, and where those are fewer the partials too (summed in group order).
template <int DP, bool F16, int MT>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Prob a, const __grid_constant__ Plan p,
                                                   const float* __restrict__ parts, int64_t per_block) {
    constexpr int CH = DP / 8;
    __shared__ float sacc[256][9];
    __shared__ float sml[256][2];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t all = (int64_t)a.batch * p.pairs;
    const int64_t p0 = min(blockIdx.x * per_block, all), p1 = min(p0 + per_block, all);
    if (p0 >= p1) return;
    Place at;
    const Cut cut = find(a, p, -1, (int)(p0 / p.pairs), at);
    for (int64_t x = p0; x < p1; ++x) {
        const int b = (int)(x / p.pairs), pair = (int)(x - (int64_t)b * p.pairs);
        if (b != at.b) {
            at.before += (int64_t)units_of(key_range(a, at.b)) * p.pairs;
            at.b = b;
        }
        const int ub = units_of(key_range(a, b));
        const int hk = pair / p.row_tiles, rt = pair - hk * p.row_tiles;
        const int64_t ua = at.before + (int64_t)pair * ub;
        int c0 = 0, nc = 0;
        bool first_behind = false;   // the first CTA's run began before this pair
        if (ub) {
            c0 = cut.owner(ua + SETUP);
            nc = cut.owner(ua + ub - 1) - c0 + 1;
            first_behind = cut.start(c0) < ua;
            // one CTA has it all and finished it, unless it began inside the pair's SETUP units
            if (nc == 1 && cut.start(c0) <= ua) continue;
        }
        const int live = min(p.rows - rt * 16 * MT, 16 * MT), pieces = live * CH;
        const int groups = max(1, 256 / pieces);
        for (int y0 = 0; y0 < pieces; y0 += 256) {
            const int y = y0 + (groups > 1 ? threadIdx.x % pieces : threadIdx.x);
            const int grp = groups > 1 ? threadIdx.x / pieces : 0;
            const int r = y / CH, d = y % CH * 8;
            const bool busy = y < pieces && grp < groups;
            float acc[8] = {}, m = -INFINITY, l = 0.f;
            if (busy) {
                auto part_of = [&](int i) {
                    return parts + ((int64_t)(c0 + i) * 2 + (i == 0 && first_behind ? 1 : 0)) * PART<DP, MT>;
                };
#pragma unroll 4
                for (int i = grp; i < nc; i += groups) m = fmaxf(m, part_of(i)[16 * MT * DP + r]);
                const float base = m == -INFINITY ? 0.f : m;
#pragma unroll 4
                for (int i = grp; i < nc; i += groups) {
                    const float* pt = part_of(i);
                    const float fx = ptx::ex2_mufu(pt[16 * MT * DP + r] - base);
                    l = fmaf(fx, pt[16 * MT * (DP + 1) + r], l);
                    const float4 v0 = *(const float4*)(pt + r * DP + d), v1 = *(const float4*)(pt + r * DP + d + 4);
                    const float v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
                    for (int e = 0; e < 8; ++e) acc[e] = fmaf(fx, v[e], acc[e]);
                }
            }
            if (groups > 1) {
#pragma unroll
                for (int e = 0; e < 8; ++e) sacc[threadIdx.x][e] = acc[e];
                sml[threadIdx.x][0] = m;
                sml[threadIdx.x][1] = l;
                __syncthreads();
                if (busy && grp == 0) {
                    for (int i = 1; i < groups; ++i) m = fmaxf(m, sml[threadIdx.x + i * pieces][0]);
                    const float base = m == -INFINITY ? 0.f : m;
                    l = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
                    for (int i = 0; i < groups; ++i) {
                        const int s = threadIdx.x + i * pieces;
                        const float fx = ptx::ex2_mufu(sml[s][0] - base);
                        l = fmaf(fx, sml[s][1], l);
#pragma unroll
                        for (int e = 0; e < 8; ++e) acc[e] = fmaf(fx, sacc[s][e], acc[e]);
                    }
                }
                __syncthreads();
            }
            if (busy && grp == 0) store_row<F16>(a, b, hk, rt * 16 * MT + r, d, acc, m, l);
        }
    }
}

template <int DP, bool F16, int MT>
int launch(const Prob& a, float* parts, cudaStream_t s) {
    Plan p;
    p.rows = a.group * a.q_len;
    p.row_tiles = (int)cdiv(p.rows, 16 * MT);
    p.pairs = a.kv_heads * p.row_tiles;
    p.ctas = num_sms() * CTAS_PER_SM;
    using S = Smem<DP>;
    auto fn = rows_kernel<DP, F16, MT>;
    FD_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, S::BYTES));
    fn<<<p.ctas, WARPS * 32, S::BYTES, s>>>(a, p, parts);
    FD_CUDA_TRY(cudaGetLastError());
    const int64_t all = (int64_t)a.batch * p.pairs, blocks = std::min<int64_t>(all, 4 * num_sms());
    // launched while the rows kernel runs; it waits (griddepcontrol) for that grid's end before it reads
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    const float* in = parts;
    FD_CUDA_TRY(cudaLaunchKernelEx(&cfg, join_kernel<DP, F16, MT>, a, p, in, cdiv(all, blocks)));
    return FD_OK;
}

template <int DP, bool F16>
int by_rows(const Prob& a, float* parts, cudaStream_t s) {
    return a.group * a.q_len <= 16 ? launch<DP, F16, 1>(a, parts, s) : launch<DP, F16, 2>(a, parts, s);
}

}  // namespace rows

bool rows_applies(const Prob& a) { return (int64_t)a.group * a.q_len <= MAX_ROWS; }

size_t rows_bytes(int dim) {
    return sizeof(float) * 2 * (size_t)num_sms() * rows::CTAS_PER_SM * (dim <= 64 ? rows::PART<64, 2> : rows::PART<128, 2>);
}

int rows_forward(const Prob& a, int dtype, void* workspace, cudaStream_t s) {
    float* parts = (float*)workspace;
    if (dtype == FD_DTYPE_F16)
        return a.dim <= 64 ? rows::by_rows<64, true>(a, parts, s) : rows::by_rows<128, true>(a, parts, s);
    return a.dim <= 64 ? rows::by_rows<64, false>(a, parts, s) : rows::by_rows<128, false>(a, parts, s);
}

}  // namespace attn
}  // namespace fd
