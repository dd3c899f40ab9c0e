// Softmax attention of few query rows against many keys: the newest tokens of
// each sequence and a cache, and any call of at most MAX_ROWS query rows per key
// head.  Bandwidth-bound: every visible key and value is read once, and the
// arithmetic of 8, 16 or 32 rows (the query heads that share a key head, times
// the new tokens) rides on mma.sync tiles with keys as their 16 rows and queries
// as their 8 columns; a tcgen05 tile would have 128 rows.
//
//   S^T = K Q^T,  P^T = 2^(x - m),  O^T += V^T P^T
//
// Work split: the keys in use come from device memory, so the split is made on
// the device.  The keys of all (sequence, key head, row tile) pairs are cut into
// units, laid end to end with SETUP units more for each pair (what its start and
// end cost), and every CTA of a fixed grid takes an equal run: lengths from 1 to
// the longest fill the SMs evenly.  A pair cut between CTAs leaves (m, l, O)
// partials that join_kernel sums in CTA order (the same bits at every call); a
// pair inside one CTA is finished there.
//
// Each warp copies its own blocks of keys with cp.async into a ring of its own,
// one or two blocks ahead and across the ends of pairs, and reads MMA fragments
// from it in 16-byte pieces: the order of the contracted coordinate in K Q^T is
// free (Q is loaded the same way), and so is the order of output coordinates in
// V^T P^T; the pairs of keys that a V^T fragment wants are put together by byte
// permutes, and P^T is turned from accumulator to operand by movmatrix.  P is
// split in two 16-bit parts, good to 2^-17 (bf16) and 2^-22 (fp16) of a weight, so
// that it adds next to no rounding of its own.  fp16 ends at 2^-24: P is held times
// 2^7 there, and weights down to 2^-31 of the largest keep a bit.  m is raised only
// when a score exceeds it by more than 8 (P then stays below 2^8, fp16 2^15), so
// the usual block needs no exchange between lanes.
#include <algorithm>

#include "fd_attn_tc.cuh"

namespace fd {
namespace attn {
namespace rows {

constexpr int WARPS = 4;
constexpr int SETUP = 3;
// CTAs to an SM and blocks of a warp's ring, by column tiles: registers allow three CTAs for up to 8 rows, shared
// memory then two blocks for each warp (48 ragged lengths to 8192 of 32 / 8 heads of 128: 50 us with two CTAs and
// three blocks, 44 so), else two.
__host__ __device__ constexpr int ctas_per_sm(int nt) { return nt == 1 ? 3 : 2; }
__host__ __device__ constexpr int stages(int nt) { return nt == 1 ? 2 : 3; }

// How far m is set below a row's maximum: log2 of what P, and with it l and O, are held times.
template <bool F16> constexpr float P_SHIFT = F16 ? 7.f : 0.f;

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

struct Plan {
    int pairs;        // (key head, row tile) pairs of a sequence
    int row_tiles, rows;
    int ctas;
    int unit;         // log2 of the keys of a unit: a block for each warp
    int magic;        // r / group = r magic >> 16 for the rows of a pair (r, group <= 64: off by less than 1 / 600)
    __device__ int query(int r) const { return r * magic >> 16; }
    __device__ int head(int pair) const { return row_tiles == 1 ? pair : pair / row_tiles; }
};

// Units of one pair of this range, its SETUP included; 0 for an empty range.
__device__ __forceinline__ int units_of(const Range& r, const Plan& p) {
    return r.hi > r.lo ? ((r.hi - r.lo - 1) >> p.unit) + 1 + SETUP : 0;
}

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
        const int64_t u = (int64_t)units_of(key_range(a, i), p) * p.pairs;
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
            const int64_t n = (int64_t)units_of(key_range(a, x), p) * p.pairs;
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
            const int ub = units_of(r, p);
            const int64_t here = (int64_t)ub * p.pairs, off = u - at.before;
            if (off >= here) {
                at.before += here;
                ++at.b;
                continue;
            }
            pair = off < ub ? 0 : (uint64_t)off >> 32 ? (int)(off / ub) : (int)((uint32_t)off / (uint32_t)ub);
            const int blk = (int)(off - (int64_t)pair * ub);
            const int take = (int)min((int64_t)(ub - blk), u1 - u);
            b = at.b;
            k0 = r.lo + (max(blk - SETUP, 0) << p.unit);
            k1 = (int)min((int64_t)r.hi, r.lo + ((int64_t)max(blk + take - SETUP, 0) << p.unit));
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
// 8 x 8 16-bit matrix, rows over the lanes' quads -> its transpose in the same places
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}

// Floats of one partial: O of 8 NT rows, then their m and l.
template <int DP, int NT>
constexpr int PART = 8 * NT * (DP + 2);

// out[gr, d .. d + 8) = acc / l, and the row's lse with its first piece
template <bool F16>
__device__ __forceinline__ void store_row(const Prob& a, const Plan& p, int b, int hk, int gr, int d,
                                          const float (&acc)[8], float m, float l) {
    const int i = p.query(gr), h = hk * a.group + gr - i * a.group;
    l = sum_or_nan(l, m == LOWEST);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (d < a.dim) {
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = acc[e] * inv;
        store8<F16>((uint16_t*)a.o.p + b * a.o.sb + (int64_t)i * a.o.ss + h * a.o.sh + d,
                    a.o_low ? a.o_low + (((int64_t)b * a.q_len + i) * a.heads + h) * a.dim + d : nullptr, f);
    }
    if (d == 0 && a.lse) a.lse[((int64_t)b * a.heads + h) * a.q_len + i] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
}

template <int DP, int NT>
struct Smem {
    static constexpr int STAGES = stages(NT), CTAS = ctas_per_sm(NT);
    static constexpr int KEYS = 2048 / DP;                        // keys of a block: 16 or 32
    static constexpr uint32_t HALF = KEYS * DP * 2;               // K or V of a block, 4 KB
    static constexpr uint32_t RING = WARPS * STAGES * 2 * HALF;
    static constexpr int PIECES = DP / 16 + 1;                    // 16-byte pieces of one lane's sums: O, and m and l
    static constexpr uint32_t CAP_OFF = RING + 2 * PIECES * 32 * 16;   // the tanh's coefficients and their limit
    static constexpr uint32_t BYTES = CAP_OFF + 32;
    // 228 KB to an SM, of which each CTA takes 1 KB for itself
    static_assert(CTAS * (BYTES + 1024) <= 228 * 1024, "shared memory budget");
};

// Row r of a pair: query i = r / group, head hk * group + r % group.
template <int DP, bool F16, int NT>
__global__ void __launch_bounds__(WARPS * 32, ctas_per_sm(NT))
rows_kernel(const __grid_constant__ Prob a, const __grid_constant__ Plan p, float* __restrict__ parts) {
    using S = Smem<DP, NT>;
    constexpr int STAGES = S::STAGES;
    constexpr int KEYS = S::KEYS, KT = KEYS / 16, UNIT = KEYS * WARPS;
    constexpr int KI = DP / 32, VB = DP / 64, CH = DP / 8;   // 16-byte pieces of a row: CH
    extern __shared__ __align__(128) uint8_t smem[];
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
    if (cap2 > 0.f) {
        // in shared memory, for registers are short and only a cap wants them.  All warps write the same.
        if (lane == 0) {
            const Score sc(a);
            float* to = (float*)(smem + S::CAP_OFF);
            *(float4*)to = make_float4(ptx::lo2(sc.b0), ptx::lo2(sc.b1), ptx::lo2(sc.b2), ptx::lo2(sc.b3));
            to[4] = sc.limit;
        }
        __syncwarp();
    }
    const uint32_t ring = ptx::smem_u32(smem) + warp * STAGES * 2 * S::HALF;

    // ---- the copies run ahead: lane (lr, ch) copies piece ch of rows lr, lr + RP, ... of each block
    constexpr int RP = 32 / CH;
    const int lr = lane / CH, ch = lane % CH;
    const bool col = ch * 8 < a.dim;
    Walk f = w;
    // blocks flast, flast + UNIT, ... below fend, the last first: the nearest keys have the largest scores
    // where a bias falls with distance, and m then rises once
    auto last_block = [](int lo, int end) { return end > lo ? lo + (end - lo - 1) / UNIT * UNIT : lo - UNIT; };
    int fk = -1, flast = 0, fend = 0, wr = 0;
    const uint16_t *pk = nullptr, *pv = nullptr;
    auto fetch = [&]() {
        while (fk < flast) {
            if (!f.next(a, p, u0)) break;
            const int hk = p.head(f.pair);
            flast = f.k0 + warp * KEYS;
            fend = f.k1;
            fk = last_block(flast, fend);
            pk = (const uint16_t*)a.k.p + f.b * a.k.sb + hk * a.k.sh + (int64_t)(fk + lr) * a.k.ss + (col ? ch * 8 : 0);
            pv = (const uint16_t*)a.v.p + f.b * a.v.sb + hk * a.v.sh + (int64_t)(fk + lr) * a.v.ss + (col ? ch * 8 : 0);
        }
        if (fk >= flast) {
            // pieces are swapped within 128 bytes (by bit 0 of the row for K, bits 1 and 2 for V) so that the
            // fragment reads below hit every bank once
            const uint32_t dst = ring + wr * 2 * S::HALF + lr * CH * 16;
            const uint32_t dk = dst + (ch ^ ((lr & 1) << 2)) * 16, dv = dst + S::HALF + (ch ^ (lr & 6)) * 16;
            const int left = fend - fk - lr;     // this lane's rows before the end
#pragma unroll
            for (int x = 0; x < KEYS / RP; ++x) {
                const bool there = x * RP < left && col;
                copy16(dk + x * RP * CH * 16, there ? pk + x * RP * a.k.ss : (const uint16_t*)a.k.p, there);
                copy16((dv ^ (((x * RP) & 6) << 4)) + x * RP * CH * 16, there ? pv + x * RP * a.v.ss : (const uint16_t*)a.v.p,
                       there);
            }
            fk -= UNIT;
            pk -= UNIT * a.k.ss;
            pv -= UNIT * a.v.ss;
            wr = wr + 1 == STAGES ? 0 : wr + 1;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int x = 0; x < STAGES - 1; ++x) fetch();
    int rd = 0;

    while (w.next(a, p, u0)) {
        const int b = w.b, hk = p.head(w.pair), r0 = (w.pair - hk * p.row_tiles) * NT * 8;
        const int n = keys_of(a, b);
        // operand rows: query r0 + 8 y + g; accumulator columns: queries r0 + 8 y + 2 t + z
        uint32_t q[NT][KI][4];
        float at[NT][2], slope2[NT][2], m[NT][2], l[NT][2];
        auto span_of = [&](int y, int z) {       // of this lane's column, made again where a block is not wholly seen
            const int r = r0 + 8 * y + 2 * t + z;
            return r < p.rows ? row_span(a, b, p.query(r), n) : make_int2(0, 0);
        };
        int flo = 0, fhi = 0x7fffffff;   // keys that every row sees: [flo, fhi)
        bool hole = false;
#pragma unroll
        for (int y = 0; y < NT; ++y) {
            const int rq = r0 + 8 * y + g;
            const int qi = rq < p.rows ? p.query(rq) : 0, qh = rq < p.rows ? rq - qi * a.group : 0;
            const uint16_t* qr = (const uint16_t*)a.q.p + b * a.q.sb + qi * a.q.ss + (hk * a.group + qh) * a.q.sh;
#pragma unroll
            for (int k = 0; k < KI; ++k) {
                const int d = 32 * k + 8 * t;
                const uint4 x = load16(qr + d, rq < p.rows && d < a.dim);
                q[y][k][0] = x.x;
                q[y][k][1] = x.y;
                q[y][k][2] = x.z;
                q[y][k][3] = x.w;
            }
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                const int r = r0 + 8 * y + 2 * t + z;
                const bool real = r < p.rows;
                const int i = real ? p.query(r) : 0, h = hk * a.group + (real ? r - i * a.group : 0);
                at[y][z] = (float)(n - a.q_len + i - g - w.k0 - warp * KEYS);   // distance to this lane's first key
                slope2[y][z] = a.slopes ? a.slopes[h] * LOG2E : 0.f;
                m[y][z] = -INFINITY;
                l[y][z] = 0.f;
                if (real) {
                    const int2 sp = row_span(a, b, i, n);
                    if (sp.y > sp.x) {
                        flo = max(flo, sp.x);
                        m[y][z] = LOWEST;
                    } else {
                        hole = true;
                    }
                    fhi = min(fhi, sp.y);
                }
            }
        }
        flo = warp_max(flo);
        fhi = warp_min(fhi);
        hole = __any_sync(~0u, hole);
        float o[NT][VB * 4][4];
#pragma unroll
        for (int y = 0; y < NT; ++y)
#pragma unroll
            for (int e = 0; e < VB * 4; ++e)
#pragma unroll
                for (int z = 0; z < 4; ++z) o[y][e][z] = 0.f;

        const int kfirst = w.k0 + warp * KEYS;
#pragma unroll 1
        for (int k0 = last_block(kfirst, w.k1); k0 >= kfirst; k0 -= UNIT) {
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
            __syncwarp();
            const uint32_t sk = ring + rd * 2 * S::HALF, sv = sk + S::HALF;
            rd = rd + 1 == STAGES ? 0 : rd + 1;
            // s[y][k][z]: query 2 t + z % 2 of column tile y, key k0 + 16 k + g + 8 (z / 2)
            float s[NT][KT][4];
#pragma unroll
            for (int k = 0; k < KT; ++k) {
#pragma unroll
                for (int y = 0; y < NT; ++y)
#pragma unroll
                    for (int z = 0; z < 4; ++z) s[y][k][z] = 0.f;
#pragma unroll
                for (int i = 0; i < KI; ++i) {
                    const uint32_t at_k = sk + ((16 * k + g) * CH + ((4 * i + t) ^ ((g & 1) << 2))) * 16;
                    const uint4 x0 = lds16(at_k), x1 = lds16(at_k + 8 * CH * 16);
#pragma unroll
                    for (int y = 0; y < NT; ++y) {
                        mma<F16>(s[y][k], x0.x, x1.x, x0.y, x1.y, q[y][i][0], q[y][i][1]);
                        mma<F16>(s[y][k], x0.z, x1.z, x0.w, x1.w, q[y][i][2], q[y][i][3]);
                    }
                }
            }
            fetch();
            const bool edge = k0 < flo || k0 + KEYS > fhi || hole;
            const float step = (float)(k0 - kfirst);
            if (cap2 > 0.f) {
                // the two forms of the tanh, as cap32 has them: each score from its own product alone
                float big = 0.f;
#pragma unroll
                for (int y = 0; y < NT; ++y)
#pragma unroll
                    for (int k = 0; k < KT; ++k)
#pragma unroll
                        for (int z = 0; z < 4; ++z) big = fmaxf(big, fabsf(s[y][k][z]));
                const uint4 bw = lds16(ptx::smem_u32(smem) + S::CAP_OFF);
                const float limit = *(volatile float*)(smem + S::CAP_OFF + 16);
                const bool inside = __all_sync(~0u, big <= limit);
                const float b0 = __uint_as_float(bw.x), b1 = __uint_as_float(bw.y), b2 = __uint_as_float(bw.z), b3 = __uint_as_float(bw.w);
#pragma unroll
                for (int y = 0; y < NT; ++y)
#pragma unroll
                    for (int k = 0; k < KT; ++k)
#pragma unroll
                        for (int z = 0; z < 4; ++z) {
                            const float v = s[y][k][z], w2 = v * v, near = fmaf(fmaf(fmaf(b3, w2, b2), w2, b1), w2, b0) * v;
                            if (inside) {
                                s[y][k][z] = near;
                                continue;
                            }
                            const float e = ptx::ex2_mufu(v * (c * 2.f * LOG2E));
                            s[y][k][z] = fabsf(v) <= limit ? near : fmaf(-2.f * cap2, ptx::rcp_mufu(1.f + e), cap2);
                        }
            }
            // s becomes score - m (score itself while m is not yet a number)
            constexpr float SH = P_SHIFT<F16>;
            const float mul = cap2 > 0.f ? 1.f : c;
            float top[NT][2];
            bool raise = false;
#pragma unroll
            for (int y = 0; y < NT; ++y)
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    const float nb = m[y][z] <= LOWEST ? 0.f : -m[y][z];
                    const float sl = slope2[y][z], far = at[y][z] - step, from = fmaf(-sl, far, nb);
#pragma unroll
                    for (int k = 0; k < KT; ++k)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const float off = (float)(16 * k + 8 * x);
                            // causal: the key is never ahead of the query, but where it is masked
                            const float add = !a.slopes ? nb : a.causal ? fmaf(sl, off, from) : fmaf(-sl, fabsf(far - off), nb);
                            s[y][k][2 * x + z] = fmaf(s[y][k][2 * x + z], mul, add);
                        }
                    if (edge) {
                        const int2 sp = span_of(y, z);
#pragma unroll
                        for (int k = 0; k < KT; ++k)
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                const int key = k0 + 16 * k + g + 8 * x;
                                if (key < sp.x || key >= sp.y) s[y][k][2 * x + z] = -INFINITY;
                            }
                    }
                    top[y][z] = fmaxf(s[y][0][z], s[y][0][2 + z]);
#pragma unroll
                    for (int k = 1; k < KT; ++k) top[y][z] = fmaxf(top[y][z], fmaxf(s[y][k][z], s[y][k][2 + z]));
                    raise = raise || top[y][z] > (m[y][z] <= LOWEST ? -INFINITY : 8.f + SH);
                }
            if (__any_sync(~0u, raise)) {
#pragma unroll
                for (int y = 0; y < NT; ++y)
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        float tp = top[y][z];
                        tp = fmaxf(tp, __shfl_xor_sync(~0u, tp, 4));
                        tp = fmaxf(tp, __shfl_xor_sync(~0u, tp, 8));
                        tp = fmaxf(tp, __shfl_xor_sync(~0u, tp, 16));
                        const bool fresh = m[y][z] <= LOWEST;
                        // nothing seen yet, or no need: what another row of the warp sees moves no bit of this one
                        if (!(tp > (fresh ? -INFINITY : 8.f + SH))) continue;
                        tp -= SH;                                 // by how much m rises, or its first value
                        const float fix = fresh ? 0.f : ptx::ex2_mufu(-tp);
                        m[y][z] = fresh ? tp : m[y][z] + tp;
                        l[y][z] *= fix;
#pragma unroll
                        for (int k = 0; k < KT; ++k) {
                            s[y][k][z] -= tp;
                            s[y][k][2 + z] -= tp;
                        }
#pragma unroll
                        for (int e = 0; e < VB * 4; ++e) {
                            o[y][e][z] *= fix;
                            o[y][e][2 + z] *= fix;
                        }
                    }
            }
            // P^T as B operand: keys along the contracted index
            uint32_t ph[NT][KT][2], pl[NT][KT][2];
#pragma unroll
            for (int y = 0; y < NT; ++y)
#pragma unroll
                for (int k = 0; k < KT; ++k)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const float e0 = ptx::ex2_mufu(s[y][k][2 * x]), e1 = ptx::ex2_mufu(s[y][k][2 * x + 1]);
                        l[y][0] += e0;
                        l[y][1] += e1;
                        const uint32_t hi = ptx::pack16<F16>(e0, e1);
                        const float2 hf = unpack16<F16>(hi);
                        ph[y][k][x] = transpose8x8(hi);
                        pl[y][k][x] = transpose8x8(ptx::pack16<F16>(e0 - hf.x, e1 - hf.y));
                    }
            bool bad = false;
#pragma unroll
            for (int k = 0; k < KT; ++k)
#pragma unroll
                for (int i = 0; i < VB; ++i) {
                    uint32_t v[4][4];
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        const int r = 16 * k + 2 * t + (z & 1) + 8 * (z >> 1);
                        const uint4 x = lds16(sv + (r * CH + ((8 * i + g) ^ (2 * t))) * 16);
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
                    for (int e = 0; e < 4; ++e) {
                        // rows g and g + 8 of the tile: coordinates 64 i + 8 g + 2 e and the next one
                        const uint32_t a0 = __byte_perm(v[0][e], v[1][e], 0x5410), a1 = __byte_perm(v[0][e], v[1][e], 0x7632);
                        const uint32_t a2 = __byte_perm(v[2][e], v[3][e], 0x5410), a3 = __byte_perm(v[2][e], v[3][e], 0x7632);
#pragma unroll
                        for (int y = 0; y < NT; ++y) {
                            mma<F16>(o[y][i * 4 + e], a0, a1, a2, a3, ph[y][k][0], ph[y][k][1]);
                            mma<F16>(o[y][i * 4 + e], a0, a1, a2, a3, pl[y][k][0], pl[y][k][1]);
                        }
                    }
                }
            if (__any_sync(~0u, bad)) {
                const uint16_t* vb = (const uint16_t*)a.v.p + b * a.v.sb + hk * a.v.sh;
                for (int key = k0; key < min(k0 + KEYS, w.k1); ++key) {
                    const uint16_t* vr = vb + (int64_t)key * a.v.ss;
#pragma unroll
                    for (int e = 0; e < VB * 4; ++e)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const int d = 64 * (e / 4) + 8 * g + 2 * (e % 4) + x;
                            if (d >= a.dim) continue;
                            constexpr uint16_t EXP = F16 ? 0x7c00 : 0x7f80;
                            const uint16_t h = vr[d];
                            if ((h & EXP) != EXP) continue;
#pragma unroll
                            for (int y = 0; y < NT; ++y)
#pragma unroll
                                for (int z = 0; z < 2; ++z) {
                                    const int2 sp = span_of(y, z);
                                    if (key >= sp.x && key < sp.y) o[y][e][2 * x + z] += one16<F16>(h);
                                }
                        }
                }
            }
        }
        // ---- the four warps' sums meet: 2 and 3 hand theirs to 0 and 1, then 1 to 0
        float* part = parts + ((int64_t)blockIdx.x * 2 + (w.front ? 0 : 1)) * PART<DP, NT>;
#pragma unroll
        for (int y = 0; y < NT; ++y) {
#pragma unroll
            for (int from = 2; from; from >>= 1) {
                if (warp >= from && warp < 2 * from) {
                    float4* to = meet + (warp - from) * S::PIECES * 32 + lane;
#pragma unroll
                    for (int e = 0; e < VB * 4; ++e) to[e * 32] = make_float4(o[y][e][0], o[y][e][1], o[y][e][2], o[y][e][3]);
                    to[VB * 4 * 32] = make_float4(m[y][0], m[y][1], l[y][0], l[y][1]);
                }
                __syncthreads();
                if (warp < from) {
                    const float4* in = meet + warp * S::PIECES * 32 + lane;
                    const float4 ml = in[VB * 4 * 32];
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
                    for (int e = 0; e < VB * 4; ++e) {
                        const float4 v = in[e * 32];
                        o[y][e][0] = o[y][e][0] * f0[0] + v.x * f1[0];
                        o[y][e][1] = o[y][e][1] * f0[1] + v.y * f1[1];
                        o[y][e][2] = o[y][e][2] * f0[0] + v.z * f1[0];
                        o[y][e][3] = o[y][e][3] * f0[1] + v.w * f1[1];
                    }
                }
                __syncthreads();
            }
            if (warp == 0) {
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    const int pr = 8 * y + 2 * t + z, gr = r0 + pr;
                    float ls = l[y][z];
                    ls += __shfl_xor_sync(~0u, ls, 4);
                    ls += __shfl_xor_sync(~0u, ls, 8);
                    ls += __shfl_xor_sync(~0u, ls, 16);
                    if (gr >= p.rows) continue;
#pragma unroll
                    for (int i = 0; i < VB; ++i) {
                        const int d = 64 * i + 8 * g;
                        float acc[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) acc[e] = o[y][i * 4 + e / 2][2 * (e & 1) + z];
                        if (w.whole) {
                            store_row<F16>(a, p, b, hk, gr, d, acc, m[y][z], ls);
                        } else {
                            *(float4*)(part + pr * DP + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
                            *(float4*)(part + pr * DP + d + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
                        }
                    }
                    if (!w.whole && g == 0) {
                        part[8 * NT * DP + pr] = m[y][z];
                        part[8 * NT * (DP + 1) + pr] = ls;
                    }
                }
            }
        }
    }
}

// Pairs that were cut: their partials, in CTA order.  Pairs that see no key: zeros.
// A block takes one slice of a pair, 32 pieces of a row and 8 coordinates; its
// eight warps share the partials (warp v takes v, v + 8, ...), and their sums are
// added in warp order.
template <int DP, bool F16, int NT>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Prob a, const __grid_constant__ Plan p,
                                                   const float* __restrict__ parts) {
    constexpr int CH = DP / 8, SLICES = 8 * NT * CH / 32;
    __shared__ float sacc[8][8][32];
    __shared__ float sml[8][2][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int slice = blockIdx.x % SLICES;
    const int64_t all = (int64_t)a.batch * p.pairs, blocks = gridDim.x / SLICES;
    const int64_t per_block = (all + blocks - 1) / blocks;
    const int64_t p0 = min(blockIdx.x / SLICES * per_block, all), p1 = min(p0 + per_block, all);
    Place at;
    // only lengths and spans are read before the rows kernel is known to have ended
    const Cut cut = find(a, p, -1, (int)(p0 / p.pairs), at);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int y = slice * 32 + lane, r = y / CH, d = y % CH * 8;
    for (int64_t x = p0; x < p1; ++x) {
        const int b = (int)(x / p.pairs), pair = (int)(x - (int64_t)b * p.pairs);
        if (b != at.b) {
            at.before += (int64_t)units_of(key_range(a, at.b), p) * p.pairs;
            at.b = b;
        }
        const int ub = units_of(key_range(a, b), p);
        const int hk = p.head(pair), gr = (pair - hk * p.row_tiles) * 8 * NT + r;
        if (__all_sync(~0u, gr >= p.rows)) continue;        // the same for all warps: no barrier is missed
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
        float acc[8] = {}, m = -INFINITY, l = 0.f;
        const float* first = parts + ((int64_t)c0 * 2 + (first_behind ? 1 : 0)) * PART<DP, NT>;
        const float* rest = parts + (int64_t)c0 * 2 * PART<DP, NT>;
        if (gr < p.rows) {
#pragma unroll 4
            for (int i = warp; i < nc; i += 8) {
                const float* pt = i ? rest + (int64_t)i * 2 * PART<DP, NT> : first;
                const float pm = pt[8 * NT * DP + r], pl = pt[8 * NT * (DP + 1) + r];
                const float4 v0 = *(const float4*)(pt + r * DP + d), v1 = *(const float4*)(pt + r * DP + d + 4);
                const float mn = fmaxf(m, pm), base = mn == -INFINITY ? 0.f : mn;
                const float f0 = ptx::ex2_mufu(m - base), f1 = ptx::ex2_mufu(pm - base);
                m = mn;
                l = l * f0 + pl * f1;
                const float v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[e] = acc[e] * f0 + v[e] * f1;
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) sacc[warp][e][lane] = acc[e];
        sml[warp][0][lane] = m;
        sml[warp][1][lane] = l;
        __syncthreads();
        if (warp == 0) {
#pragma unroll
            for (int i = 1; i < 8; ++i) m = fmaxf(m, sml[i][0][lane]);
            const float base = m == -INFINITY ? 0.f : m;
            l = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float fx = ptx::ex2_mufu(sml[i][0][lane] - base);
                l = fmaf(fx, sml[i][1][lane], l);
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[e] = fmaf(fx, sacc[i][e][lane], acc[e]);
            }
            if (gr < p.rows) store_row<F16>(a, p, b, hk, gr, d, acc, m, l);
        }
        __syncthreads();
    }
}

template <int DP, bool F16, int NT>
int launch(const Prob& a, float* parts, cudaStream_t s) {
    Plan p;
    p.rows = a.group * a.q_len;
    p.row_tiles = (int)cdiv(p.rows, 8 * NT);
    p.pairs = a.kv_heads * p.row_tiles;
    p.ctas = num_sms() * ctas_per_sm(NT);
    p.unit = DP == 64 ? 7 : 6;
    static_assert(Smem<DP, NT>::KEYS * WARPS == (DP == 64 ? 128 : 64), "unit");
    p.magic = (65536 + a.group - 1) / a.group;
    using S = Smem<DP, NT>;
    FD_TRY((allow_smem<rows_kernel<DP, F16, NT>>(S::BYTES)));
    rows_kernel<DP, F16, NT><<<p.ctas, WARPS * 32, S::BYTES, s>>>(a, p, parts);
    FD_CUDA_TRY(cudaGetLastError());
    constexpr int slices = 8 * NT * DP / 8 / 32;
    const int64_t blocks = std::min<int64_t>((int64_t)a.batch * p.pairs, 4 * num_sms()) * slices;
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
    FD_CUDA_TRY(cudaLaunchKernelEx(&cfg, join_kernel<DP, F16, NT>, a, p, in));
    return FD_OK;
}

template <int DP, bool F16>
int by_rows(const Prob& a, float* parts, cudaStream_t s) {
    const int rows = a.group * a.q_len;
    return rows <= 8    ? launch<DP, F16, 1>(a, parts, s)
           : rows <= 16 ? launch<DP, F16, 2>(a, parts, s)
                        : launch<DP, F16, 4>(a, parts, s);
}

}  // namespace rows

bool rows_applies(const Prob& a) { return a.dim <= 128 && (int64_t)a.group * a.q_len <= MAX_ROWS; }

size_t rows_bytes(int dim) {
    static_assert(rows::ctas_per_sm(4) * 4 >= rows::ctas_per_sm(1), "the widest kernel has the largest partials");
    return sizeof(float) * 2 * (size_t)num_sms() * rows::ctas_per_sm(4) * (dim <= 64 ? rows::PART<64, 4> : rows::PART<128, 4>);
}

int rows_forward(const Prob& a, int dtype, void* workspace, cudaStream_t s) {
    float* parts = (float*)workspace;
    if (dtype == FD_DTYPE_F16)
        return a.dim <= 64 ? rows::by_rows<64, true>(a, parts, s) : rows::by_rows<128, true>(a, parts, s);
    return a.dim <= 64 ? rows::by_rows<64, false>(a, parts, s) : rows::by_rows<128, false>(a, parts, s);
}

}  // namespace attn
}  // namespace fd
