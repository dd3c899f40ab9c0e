// Gradients of softmax attention on the tensor cores.
//
//   P = 2^(x - lse2),  dP = dO V^T,  delta_i = dO_i . o_i
//   dS = P (dP - delta) (1 - tanh^2 with a cap)
//   dV = P^T dO,   dK = scale dS^T Q,   dQ = scale dS K
//
// Scores are made again from Q and K.  dK and dV of a key tile are summed by one
// CTA over all query tiles and heads that share the key head, dQ of a query tile
// by another over its key tiles: seven products in the place of five, but every
// sum has one owner and a fixed order (the same bits at every call), and no
// fp32 gradient passes through memory.  Both kinds of CTA are one launch, the
// longest first, so that the short ones fill the SMs at its end.  Where there are
// too few for that (few key heads, few query rows), a CTA's tiles are shared
// between several, whose fp32 sums sum_kernel adds up in their order.
//
// Measured, bf16: 2 x 4096 rows of 16 / 4 heads of 128 688 us, 999 TFLOP/s of the
// five products, causal 401 us, 857, with a cap 647 us (881 where most blocks of
// scores reach beyond 0.45 of it); the tensor pipe is busy 66 % of the time, S and
// dP being bound by the shared memory they read both operands from (128 bytes a
// clock).  A CTA's start and end take about 8 us.
//
// CTA: two compute warpgroups that share the 128 rows of the accumulators (64
// columns of each score tile apiece), and a warpgroup with a TMA producer, an
// MMA issuer and a guard.
//   key side    rows = keys.  TMEM: S^T | dP^T | dV | dK.  P^T and dS^T go back to
//               TMEM over the scores they came from and are the A operands.  The
//               tensor core runs dV(i) and S(i + 1) while dS(i) is made, dK(i) and
//               dP(i + 1) while P(i + 1) is.
//   query side  rows = queries.  TMEM: S | dP, dP | dQ (dP in two buffers, so that
//               the next tile's products do not wait for dS).
#include <algorithm>
#include <climits>
#include <cmath>

#include "fd_attn_tc.cuh"

namespace fd {
namespace attn {
namespace bwd {

constexpr int TMA_WARP = 8, MMA_WARP = 9, GUARD_WARP = 10;
constexpr int NTHREADS = 12 * 32;
// 168 registers a thread at launch (64512 in all): 256 * 208 + 128 * 80 = 63488
constexpr int COMPUTE_REGS = 208, OTHER_REGS = 80;
constexpr uint32_t TMEM_COLS = 512;
// fp16 is normal from 2^-14 up, and a key far from every query has nothing but weights below that: P <= 1 is
// held times 2^14 (by way of lse2, so that it costs nothing) and dV scaled back at the end.
constexpr float P_SHIFT_F16 = 14.f;

struct Bounds {
    int lo, hi;     // keys seen by any row of a query tile
    int flo, fhi;   // keys seen by every row
};

// What prep_kernel leaves for the gradient kernel.
struct Work {
    float* delta;        // -delta, [batch * heads][rows padded to 128]
    float* lse2;         // -lse in base 2 (plus P_SHIFT_F16 for fp16); -inf for rows that see nothing and for the padding
    int2* spans;         // [batch][rows padded to 128]
    Bounds* bounds;      // [batch][query tiles]
    unsigned* top;       // fp16: bits of the largest |dO row|^2 and |V row|^2 that take part, [batch][key heads][2]
    float *dq, *dk, *dv; // fp32 sums of each part, [part][batch][row][head][dim], where there are parts
};

// What the sizes of a call say about its work.
struct Shape {
    int64_t batch, heads, kv_heads, q_len, k_len, dim, window;
    bool causal, spans;
    explicit Shape(const Prob& a)
        : batch(a.batch), heads(a.heads), kv_heads(a.kv_heads), q_len(a.q_len), k_len(a.k_len), dim(a.dim),
          window(a.window), causal(a.causal != 0), spans(a.first != nullptr) {}
    int key_parts() const { return parts(tiles(q_len, k_len) * (heads / kv_heads)); }
    int query_parts() const { return parts(tiles(k_len, q_len)); }
    // tiles of one side that a tile of the other sees
    int64_t tiles(int64_t of, int64_t by) const {
        return window > 0 ? std::min(cdiv(of, T), window / T + 2) : cdiv(of, T);
    }
    // The share of score tiles that hold a visible pair; of spans, which lie in device memory, half is taken.  Whole, with
    // half counted and with all, bf16: 4 x 1531 rows with prefixes, 8 / 2 heads of 128, bias 217, 175 and 221 us; 4 / 1
    // heads of 128, one document of 8192 causal 399, 233 and 399, all of it visible 430, 370 and 432, nine documents of
    // 7001 rows causal 137, 84 and 137, all visible 237, 118 and 238, but 16 documents of 512 rows 59, 66 and 59: parts
    // that a packed batch leaves nearly empty.  12 heads of 64 are not cut by any of the three.
    double visible() const {
        if (q_len < 1 || k_len < 1) return 1.0;
        if (spans) return 0.5;
        if (window > 0) return (window / T + 1.0) / (window / T + 2.0);
        return !causal ? 1.0 : q_len <= k_len ? 1.0 - 0.5 * q_len / k_len : 0.5 * k_len / q_len;
    }
    // A CTA of `items` score tiles is cut where it would outlast an SM's equal share of them all by more than a third,
    // but into parts of no fewer than MIN_ITEMS, which cost about what a part's start, its fp32 rows and their join do.
    // Whole and cut, causal, bf16: 7900 rows of 4 / 1 heads of 64 348 and 156 us; 1000 rows of 4 / 1 heads of 128 70 and
    // 37 us; 512 rows of 8 / 2 heads against 16384 keys 178 and 119 us; 1000 rows of 4 / 4 heads, not cut, 29 us, 33 us
    // in parts of four.
    int parts(int64_t items) const {
        const double share = 2 * visible() * cdiv(q_len, T) * heads * batch * tiles(k_len, q_len) / num_sms();
        return (int)std::min(std::max(std::ceil(items / std::max(share, (double)MIN_ITEMS) - 0.35), 1.0), 64.0);
    }
    static constexpr int MIN_ITEMS = 8;
};

inline size_t work_layout(Work* w, void* base, const Shape& z) {
    const int64_t bh = z.batch * z.heads, batch = z.batch, n_qt = cdiv(z.q_len, T);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) & ~(size_t)255;
        return (char*)base + here;
    };
    char* a = take(sizeof(float) * bh * n_qt * T);
    char* b = take(sizeof(float) * bh * n_qt * T);
    char* c = take(sizeof(int2) * batch * n_qt * T);
    char* d = take(sizeof(Bounds) * batch * n_qt);
    char* e = take(2 * sizeof(unsigned) * batch * z.kv_heads);
    auto sums = [&](int parts, int64_t rows) { return parts > 1 ? sizeof(float) * parts * batch * rows * z.dim : 0; };
    char* f = take(sums(z.query_parts(), z.q_len * z.heads));
    char* g = take(sums(z.key_parts(), z.k_len * z.kv_heads));
    char* h = take(sums(z.key_parts(), z.k_len * z.kv_heads));
    if (w) *w = {(float*)a, (float*)b, (int2*)c, (Bounds*)d, (unsigned*)e, (float*)f, (float*)g, (float*)h};
    return at;
}

// Which of the keys k0 .. k0 + 127 some query row sees, as 128 bits.  All threads of a block of 256; the answer is the
// same in all.  Causal rows and windows move on by one key a row, so their union is one run.  Of spans those about the
// keys' own positions are read first: they show the keys of most masks, and nothing is left to look for in the others.
__device__ __forceinline__ uint4 keys_seen(const Prob& a, int b, int n, int k0, uint32_t (&bits)[4]) {
    auto run = [&](int w, int lo, int hi) {   // bits of word w within [lo, hi)
        const int x = max(lo - k0 - 32 * w, 0), y = min(hi - k0 - 32 * w, 32);
        return y > x ? ~0u >> (32 - (y - x)) << x : 0u;
    };
    if (!a.first) {
        const int lo = row_span(a, b, 0, n).x, hi = row_span(a, b, a.q_len - 1, n).y;
        return make_uint4(run(0, lo, hi), run(1, lo, hi), run(2, lo, hi), run(3, lo, hi));
    }
    if (threadIdx.x < 4) bits[threadIdx.x] = 0;
    __syncthreads();
    auto rows = [&](int lo, int hi) {
        uint32_t m[4] = {};
        constexpr int AHEAD = 8;   // spans in flight
        for (int i0 = lo + (int)threadIdx.x; i0 < hi; i0 += AHEAD * 256) {
            int2 sp[AHEAD];
#pragma unroll
            for (int y = 0; y < AHEAD; ++y) sp[y] = i0 + 256 * y < hi ? row_span(a, b, i0 + 256 * y, n) : make_int2(0, 0);
#pragma unroll
            for (int y = 0; y < AHEAD; ++y)
#pragma unroll
                for (int w = 0; w < 4; ++w) m[w] |= run(w, sp[y].x, sp[y].y);
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            m[w] = __reduce_or_sync(~0u, m[w]);
            if ((threadIdx.x & 31) == 0 && m[w]) atomicOr(&bits[w], m[w]);
        }
        __syncthreads();
    };
    // the row that stands at the tile's first key is lo + 64
    const int lo = min(max(k0 - (n - a.q_len) - 64, 0), a.q_len), hi = min(lo + 256, a.q_len);
    rows(lo, hi);
    bool all = true;
#pragma unroll
    for (int w = 0; w < 4; ++w) all = all && (~bits[w] & run(w, 0, n)) == 0;
    if (!__syncthreads_and(all)) rows(0, a.q_len);
    return make_uint4(bits[0], bits[1], bits[2], bits[3]);
}

// Block (t, h, b): delta and lse2 of 128 rows, 16 lanes a row (one 16-byte piece
// each); head 0 also makes the tile's bounds.  fp16: the largest row norms of dO
// and, in the blocks behind the query tiles, of V, for each sequence and key head;
// of V only the rows that some query sees, for the others may hold anything.
// Bandwidth-bound: dO and o are read once.
template <bool F16>
__global__ void __launch_bounds__(256) prep_kernel(const __grid_constant__ Prob a, const __grid_constant__ Work w, int n_qt) {
    // V's blocks first: theirs is the longer chain where spans have to be read
    const int h = blockIdx.y, b = blockIdx.z, t = (int)(gridDim.x - 1 - blockIdx.x);
    const int piece = threadIdx.x & 15, r0 = threadIdx.x >> 4;
    float top = 0.f;
    asm volatile("griddepcontrol.launch_dependents;");   // the gradient kernel sets itself up and waits
    if (t >= n_qt) {
        if (h >= a.kv_heads) return;
        __shared__ uint32_t bits[4];
        const int k0 = (t - n_qt) * T;
        uint4 x[T / 16];         // on their way while the spans are looked at
#pragma unroll
        for (int r8 = 0; r8 < T / 16; ++r8) {
            const int64_t j = k0 + r0 + 16 * r8;
            x[r8] = make_uint4(0, 0, 0, 0);
            if (j < a.k_len && piece * 8 < a.dim)
                x[r8] = *(const uint4*)((const uint16_t*)a.v.p + b * a.v.sb + j * a.v.ss + h * a.v.sh + piece * 8);
        }
        const uint4 seen = keys_seen(a, b, keys_of(a, b), k0, bits);
        const uint32_t word[4] = {seen.x, seen.y, seen.z, seen.w};
#pragma unroll
        for (int r8 = 0; r8 < T / 16; ++r8) {
            float s = 0.f;
            if (word[r8 / 2] >> ((r0 + 16 * r8) & 31) & 1) {
                const uint32_t xs[4] = {x[r8].x, x[r8].y, x[r8].z, x[r8].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = pair_of<F16>(xs[i]);
                    s = fmaf(f.x, f.x, fmaf(f.y, f.y, s));
                }
            }
            for (int o = 8; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
            if (s < INFINITY) top = fmaxf(top, s);
        }
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
        if ((threadIdx.x & 31) == 0 && top > 0.f) atomicMax(&w.top[2 * (b * a.kv_heads + h) + 1], __float_as_uint(top));
        return;
    }
    __shared__ int sb[4];
    const int n = keys_of(a, b);
    if (h == 0) {
        if (threadIdx.x == 0) {
            sb[0] = sb[2] = 0x7fffffff;
            sb[1] = sb[3] = 0;
        }
        __syncthreads();
        if (threadIdx.x < T) {
            const int i = t * T + threadIdx.x;
            const bool real = i < a.q_len;
            const int2 sp = real ? row_span(a, b, i, n) : make_int2(0, 0);
            w.spans[((int64_t)b * n_qt + t) * T + threadIdx.x] = sp;
            const bool some = sp.y > sp.x;
            if (some) {
                atomicMin(&sb[0], sp.x);
                atomicMax(&sb[1], sp.y);
            }
            if (real) {
                atomicMax(&sb[3], some ? sp.x : 0x7fffffff);
                atomicMin(&sb[2], some ? sp.y : 0);
            }
        }
        __syncthreads();
        if (threadIdx.x == 0) w.bounds[(int64_t)b * n_qt + t] = {sb[0], sb[1], sb[3], sb[2]};
    }
    const int64_t base = ((int64_t)b * a.heads + h) * n_qt * T;
    uint4 x[8], y[8];
    uint2 low[8];
    float lse[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int64_t i = (int64_t)t * T + r0 + 16 * j;
        const bool real = i < a.q_len;
        x[j] = y[j] = make_uint4(0, 0, 0, 0);
        low[j] = make_uint2(0, 0);
        if (real && piece * 8 < a.dim) {
            x[j] = *(const uint4*)((const uint16_t*)a.d_o.p + b * a.d_o.sb + i * a.d_o.ss + h * a.d_o.sh + piece * 8);
            y[j] = *(const uint4*)((const uint16_t*)a.o.p + b * a.o.sb + i * a.o.ss + h * a.o.sh + piece * 8);
            if (a.o_low) low[j] = *(const uint2*)(a.o_low + (((int64_t)b * a.q_len + i) * a.heads + h) * a.dim + piece * 8);
        }
        lse[j] = real ? a.lse[((int64_t)b * a.heads + h) * a.q_len + i] : -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float d = 0.f, s = 0.f;
        const uint32_t xs[4] = {x[j].x, x[j].y, x[j].z, x[j].w}, ys[4] = {y[j].x, y[j].y, y[j].z, y[j].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 f = pair_of<F16>(xs[e]), g = pair_of<F16>(ys[e]);
            const uint32_t l = e < 2 ? low[j].x : low[j].y;
            const float g0 = with_low<F16>(g.x, (int8_t)(l >> (e % 2 * 16))), g1 = with_low<F16>(g.y, (int8_t)(l >> (e % 2 * 16 + 8)));
            d = fmaf(f.x, g0, fmaf(f.y, g1, d));
            if (F16) s = fmaf(f.x, f.x, fmaf(f.y, f.y, s));
        }
        for (int o = 8; o; o >>= 1) {
            d += __shfl_xor_sync(~0u, d, o);
            if (F16) s += __shfl_xor_sync(~0u, s, o);
        }
        const bool some = lse[j] != -INFINITY;
        if (F16 && some && s < INFINITY) top = fmaxf(top, s);
        if (piece == 0) {
            const int64_t at = base + (int64_t)t * T + r0 + 16 * j;
            w.delta[at] = some ? -d : 0.f;
            w.lse2[at] = some ? (F16 ? P_SHIFT_F16 : 0.f) - lse[j] * LOG2E : -INFINITY;
        }
    }
    if (F16) {
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
        if ((threadIdx.x & 31) == 0 && top > 0.f) atomicMax(&w.top[2 * (b * a.kv_heads + h / a.group)], __float_as_uint(top));
    }
}

template <int DP>
struct Cfg {
    static constexpr int BOXES = DP / 64;
    static constexpr uint32_t TILE = BOXES * BOX_BYTES;
    // ring A: Q (key side) or K (query side), needed until the last product of a tile; ring B: dO or V, needed
    // for less long, with lse2 and delta on the key side
    static constexpr int SA = DP == 128 ? 3 : 4, SB = DP == 128 ? 2 : 4;
    static constexpr uint32_t A_OFF = 2 * TILE;                       // behind the resident pair
    static constexpr uint32_t B_OFF = A_OFF + SA * TILE;
    static constexpr uint32_t VEC_OFF = B_OFF + SB * TILE;
    static constexpr uint32_t BAR_OFF = VEC_OFF + SB * 2 * T * 4;
    // opfull, afull[SA], aempty[SA], bfull[SB], bempty[SB], sfull, sread, pfull, dpfull[2], dsfull[2], accfull,
    // toguard, guarded
    static constexpr int NBARS = 1 + 2 * SA + 2 * SB + 10;
    static constexpr uint32_t MISC_OFF = BAR_OFF + NBARS * 8;
    static constexpr uint32_t SMEM = MISC_OFF + 32;                   // 1024-byte aligned: nothing lies before it
    static_assert(SMEM <= 227 * 1024, "shared memory budget");
};

struct Misc {
    uint32_t tmem;
    int abort;
    int poison;
    int lo, hi;      // key side: query tiles [lo, hi)
};

struct Args {
    Prob a;
    Work w;
    int n_qt;                   // query tiles
    int first, keys_first;      // CTAs of the side that starts first: the one with the longer CTAs
    int key_parts, query_parts; // CTAs that share a key tile's, a query tile's items
};

// Store N columns of one accumulator row, times f, behind column c0: as 16-bit values of `out`, or as fp32 of `sums`.
template <int N, bool F16>
__device__ __forceinline__ void store_cols(uint32_t taddr, float f, uint8_t* out, float* sums, int c0, int dim, bool live,
                                           bool have) {
#pragma unroll 1
    for (int g = 0; g < N; g += 32) {
        uint32_t o[32];
        if (have) {
            ptx::tmem_ld32(taddr + g, o);
            ptx::tmem_wait_ld(o);
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0;
        }
        if (!live) continue;
        if (sums) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
                if (c0 + g + i < dim)
                    *(float4*)(sums + c0 + g + i) =
                        make_float4(__uint_as_float(o[i]) * f, __uint_as_float(o[i + 1]) * f, __uint_as_float(o[i + 2]) * f,
                                    __uint_as_float(o[i + 3]) * f);
            continue;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (c0 + g + i * 8 >= dim) continue;
            uint32_t p[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                p[e] = ptx::pack16<F16>(__uint_as_float(o[8 * i + 2 * e]) * f, __uint_as_float(o[8 * i + 2 * e + 1]) * f);
            *(uint4*)(out + 2 * (c0 + g + i * 8)) = make_uint4(p[0], p[1], p[2], p[3]);
        }
    }
}

// What every role of a CTA knows.
struct Cta {
    const Prob& a;
    const Work& w;
    bool key_side;
    int tile, b, h;        // h: key head on the key side, query head on the query side
    int r0, n, n_qt;       // first row of this CTA, keys in use, query tiles
    int t0, nt;            // the other side's tiles t0 .. t0 + nt, walked once for each head of the group on the key side
    int skip, items;       // this CTA's items of that walk
    Bounds own;            // query side: this tile's bounds
    const Bounds* bounds;
};

// Item i of a CTA: its tile, and the query head on the key side.
struct Item {
    int i, t, head;
    __device__ explicit Item(const Cta& c) : i(0), t(c.t0 + c.skip), head(c.key_side ? c.h * c.a.group : c.h) {
        if (c.skip >= c.nt && c.nt > 0) {
            t = c.t0 + c.skip % c.nt;
            head += c.skip / c.nt;
        }
    }
    __device__ void next(const Cta& c) {
        ++i;
        if (++t == c.t0 + c.nt) {
            t = c.t0;
            ++head;
        }
    }
    // some pair of the tile is masked
    __device__ bool partial(const Cta& c) const {
        if (!c.key_side) return t * T < c.own.flo || (t + 1) * T > c.own.fhi;
        const Bounds o = c.bounds[t];
        return c.r0 < o.flo || c.r0 + T > o.fhi;
    }
};

struct Bars {
    uint64_t *opfull, *afull, *aempty, *bfull, *bempty, *sfull, *sread, *pfull, *dpfull, *dsfull, *accfull, *toguard, *guarded;
};

// Stage and phase of a ring of N slots.
template <int N>
struct Slot {
    int at = 0;
    uint32_t ph = 0;
    __device__ void next() {
        if (++at == N) {
            at = 0;
            ph ^= 1;
        }
    }
};

template <int DP>
__device__ __forceinline__ void load_box(const Cta& c, uint8_t* dst, const CUtensorMap* m, uint64_t* bar, int t, int head) {
    for (int x = 0; x < Cfg<DP>::BOXES; ++x) ptx::tma_load_4d(dst + x * BOX_BYTES, m, bar, x * 64, t * T, head, c.b);
}

// This CTA's own pair of tiles: on its way before anything is known of the other side (a microsecond of each CTA's ten).
template <int DP>
__device__ __forceinline__ void load_resident(const Cta& c, const Bars& br, uint8_t* base, const CUtensorMap* tmq,
                                              const CUtensorMap* tmk, const CUtensorMap* tmv, const CUtensorMap* tmdo) {
    ptx::mbar_expect_tx(br.opfull, 2 * Cfg<DP>::TILE);
    load_box<DP>(c, base, c.key_side ? tmk : tmq, br.opfull, c.tile, c.h);
    load_box<DP>(c, base + Cfg<DP>::TILE, c.key_side ? tmv : tmdo, br.opfull, c.tile, c.h);
}

template <int DP, bool F16>
__device__ __forceinline__ void produce(const Cta& c, const Bars& br, uint8_t* base, const CUtensorMap* tmq,
                                        const CUtensorMap* tmk, const CUtensorMap* tmv, const CUtensorMap* tmdo,
                                        volatile int* abort, int* status) {
    using C = Cfg<DP>;
    const int hk = c.h / c.a.group;      // query side
    Slot<C::SA> sa;
    Slot<C::SB> sb;
    int na = 0, nb = 0;
    for (Item it(c); it.i < c.items; it.next(c)) {
        const int hh = c.key_side ? it.head : hk;
        if (!ptx::wait_bounded(&br.aempty[sa.at], sa.ph ^ 1, abort, status, WAIT_NS)) break;
        ptx::mbar_expect_tx(&br.afull[sa.at], C::TILE);
        load_box<DP>(c, base + C::A_OFF + sa.at * C::TILE, c.key_side ? tmq : tmk, &br.afull[sa.at], it.t, hh);
        sa.next();
        ++na;
        if (!ptx::wait_bounded(&br.bempty[sb.at], sb.ph ^ 1, abort, status, WAIT_NS)) break;
        ptx::mbar_expect_tx(&br.bfull[sb.at], C::TILE + (c.key_side ? 2 * T * 4 : 0));
        load_box<DP>(c, base + C::B_OFF + sb.at * C::TILE, c.key_side ? tmdo : tmv, &br.bfull[sb.at], it.t, hh);
        if (c.key_side) {
            float* vec = (float*)(base + C::VEC_OFF) + sb.at * 2 * T;
            const int64_t at = (((int64_t)c.b * c.a.heads + hh) * c.n_qt + it.t) * T;
            ptx::bulk_load(vec, c.w.lse2 + at, T * 4, &br.bfull[sb.at]);
            ptx::bulk_load(vec + T, c.w.delta + at, T * 4, &br.bfull[sb.at]);
        }
        sb.next();
        ++nb;
    }
    if (*abort) {   // the copies in flight still write into this block's memory
        wait_landed(br.opfull, 0);
        for (int z = max(0, na - C::SA); z < na; ++z) wait_landed(&br.afull[z % C::SA], (z / C::SA) & 1);
        for (int z = max(0, nb - C::SB); z < nb; ++z) wait_landed(&br.bfull[z % C::SB], (z / C::SB) & 1);
    }
}

template <int DP, bool F16>
__device__ __forceinline__ void issue(const Cta& c, const Bars& br, uint8_t* base, uint32_t tmem, volatile int* abort,
                                      int* status) {
    using C = Cfg<DP>;
    const uint32_t lead = elect_lane();
    const int kd = (c.a.dim + 15) / 16;
    const uint32_t id_s = ptx::idesc_f32acc(T, T, F16);
    const uint32_t id_acc = ptx::idesc_f32acc(T, kd * 16, F16) | ptx::IDESC_B_MN;
    const uint32_t op0 = ptx::smem_u32(base), op1 = op0 + C::TILE, ra = op0 + C::A_OFF, rb = op0 + C::B_OFF;
    auto wait = [&](uint64_t* bar, uint32_t ph) { return wait_warp(bar, ph & 1, abort, status); };
    auto commit = [&](uint64_t* bar) { mma_commit(lead, bar); };
    // D[128 x 128] = resident operand . ring operand^T
    auto scores = [&](uint32_t d, uint32_t op, uint32_t rg) {
        ptx::tc_fence_after();
        product_rows<DP>(lead, d, op, rg, id_s, kd);
    };
    // acc[128 x dim] += (16-bit tile in TMEM, 64 columns of it at `src`, 64 at `src` + 64) . ring tile
    auto sum = [&](uint32_t acc, uint32_t src, uint32_t rg, bool more) {
        ptx::tc_fence_after();
        product_sum<2, 64>(lead, acc, src, rg, id_acc, more);
    };
    uint32_t ng = 0;
    bool ok = wait(br.opfull, 0);
    if (c.key_side) {
        const uint32_t S = tmem, DPT = tmem + 128, DV = tmem + 256, DK = tmem + 384;
        Slot<C::SA> sa, da;      // next S, current dK
        Slot<C::SB> sb, db;      // next dP, current dV
        Item ahead(c);           // tile of the next dP
        bool look = false;
        auto first = [&]() {     // S^T
            if (!wait(&br.afull[sa.at], sa.ph)) return false;
            scores(S, op0, ra + sa.at * C::TILE);
            commit(br.sfull);
            sa.next();
            return true;
        };
        auto second = [&]() {    // dP^T
            if (!wait(&br.bfull[sb.at], sb.ph)) return false;
            scores(DPT, op1, rb + sb.at * C::TILE);
            commit(&br.dpfull[0]);
            look = ahead.partial(c);
            if (look && lead) ptx::mbar_arrive(br.toguard);
            sb.next();
            ahead.next(c);
            return true;
        };
        ok = ok && first() && second();
        for (int i = 0; i < c.items && ok; ++i) {
            if (!(ok = wait(br.pfull, i))) break;
            if (look) {
                if (!(ok = wait(br.guarded, ng))) break;
                ++ng;
            }
            sum(DV, S, rb + db.at * C::TILE, i > 0);
            commit(&br.bempty[db.at]);
            db.next();
            if (i + 1 < c.items && !(ok = first())) break;
            if (!(ok = wait(&br.dsfull[0], i))) break;
            sum(DK, DPT, ra + da.at * C::TILE, i > 0);
            commit(&br.aempty[da.at]);
            da.next();
            if (i + 1 < c.items) ok = second();
        }
    } else {
        const uint32_t S = tmem, DQ = tmem + 384;
        Slot<C::SA> sa, da;
        Slot<C::SB> sb;
        int made = 0;
        auto both = [&]() {       // S and dP of the next tile
            if (!wait(&br.afull[sa.at], sa.ph)) return false;
            scores(S, op0, ra + sa.at * C::TILE);
            commit(br.sfull);
            if (!wait(&br.bfull[sb.at], sb.ph)) return false;
            scores(tmem + 128 + (made & 1) * 128, op1, rb + sb.at * C::TILE);
            commit(&br.dpfull[made & 1]);
            commit(&br.bempty[sb.at]);
            sa.next();
            sb.next();
            ++made;
            return true;
        };
        ok = ok && both();
        for (Item it(c); it.i < c.items && ok; it.next(c)) {
            const bool look = it.partial(c);
            if (look && lead) ptx::mbar_arrive(br.toguard);
            if (it.i + 1 < c.items) {
                if (!(ok = wait(br.sread, it.i))) break;
                if (!(ok = both())) break;
            }
            // one barrier for each dP buffer: a warp may be a tile ahead of another, and its arrival for the
            // next tile must not stand in for the other's for this one
            if (!(ok = wait(&br.dsfull[it.i & 1], it.i >> 1))) break;
            if (look) {
                if (!(ok = wait(br.guarded, ng))) break;
                ++ng;
            }
            sum(DQ, tmem + 128 + (it.i & 1) * 128, ra + da.at * C::TILE, it.i > 0);
            commit(&br.aempty[da.at]);
            da.next();
        }
    }
    commit(br.accfull);
    if (!ok) wait_landed(br.accfull, 0);
}

// Masked pairs have P = dS = 0, and zero times a NaN or an infinity of the other operand would reach the sum: in
// partly visible tiles such elements become zeros before the product.  What a visible pair loses with them is NaN
// already through lse (Q, K) or delta (dO) of its row, except for dV, where a visible row's bad dO elements are put
// back at the end (`poison`).
template <int DP, bool F16>
__device__ __forceinline__ void watch(const Cta& c, const Bars& br, uint8_t* base, int lane, int* poison,
                                      volatile int* abort, int* status) {
    using C = Cfg<DP>;
    uint32_t ng = 0;
    Slot<C::SA> sa;
    Slot<C::SB> sb;
    for (Item it(c); it.i < c.items; it.next(c), sa.next(), sb.next()) {
        if (!it.partial(c)) continue;
        // not before the issuer has seen the tile: see the forward kernel's guard
        if (!ptx::wait_bounded(br.toguard, ng & 1, abort, status, WAIT_NS)) return;
        ++ng;
        if (!ptx::wait_bounded(&br.afull[sa.at], sa.ph, abort, status, WAIT_NS)) return;
        clear_bad<F16>(base + C::A_OFF + sa.at * C::TILE, C::TILE, lane);
        if (c.key_side) {
            if (!ptx::wait_bounded(&br.bfull[sb.at], sb.ph, abort, status, WAIT_NS)) return;
            if (clear_bad<F16>(base + C::B_OFF + sb.at * C::TILE, C::TILE, lane) && lane == 0) *poison = 1;
            __syncwarp();
        }
        if (lane == 0) ptx::mbar_arrive(br.guarded);
    }
}

// Raw products of one row, 32 columns, to weights: x = 2^(score + add); with a cap, bend = 1 - tanh^2.
template <bool GEN>
__device__ __forceinline__ void weights32(uint64_t (&x)[16], const uint64_t (&add)[16], const Score& sc, float slope2,
                                          float dist, float by, int side, uint64_t (&bend)[GEN ? 16 : 1]) {
    if (GEN && sc.capped) {
        cap32(x, sc);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            bend[e] = ptx::fma2(ptx::mul2(x[e], sc.shrink), x[e], ptx::both2(1.f));
            x[e] = ptx::add2(x[e], add[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = ptx::fma2(x[e], sc.c, add[e]);
    }
    if (GEN && slope2 != 0.f) add_bias(x, slope2, dist, by, side);
    if (GEN && sc.capped) exp32<0>(x);     // a cap keeps the FMA pipe busy enough
    else exp32<1>(x);
}

// Keep the places of x whose bit is set.
__device__ __forceinline__ void keep32(uint64_t (&x)[16], uint32_t bits) {
#pragma unroll
    for (int e = 0; e < 16; ++e)
        x[e] = ptx::pack2(bits >> (2 * e) & 1 ? ptx::lo2(x[e]) : 0.f, bits >> (2 * e + 1) & 1 ? ptx::hi2(x[e]) : 0.f);
}

// Which of 32 queries see which of the warp's 32 keys from `k0` on: lane e brings query e's span; bit e of the answer
// of lane l: query e sees key k0 + l.
__device__ __forceinline__ uint32_t seen32(int2 span, int k0, int lane) {
    if (__all_sync(~0u, span.x <= k0 && span.y >= k0 + 32)) return ~0u;
    if (!__any_sync(~0u, span.x < k0 + 32 && span.y > k0)) return 0;
    uint32_t bits = 0;
#pragma unroll
    for (int l = 0; l < 32; ++l) {
        const uint32_t b = __ballot_sync(~0u, span.x <= k0 + l && span.y > k0 + l);
        if (lane == l) bits = b;
    }
    return bits;
}

template <int DP, bool F16, bool GEN>
__device__ __forceinline__ bool compute_key(const Cta& c, const Bars& br, const uint8_t* base, uint32_t lanes, int half,
                                            int row, float up_p, volatile int* abort, int* status) {
    using C = Cfg<DP>;
    const Prob& a = c.a;
    const int lane = threadIdx.x & 31;
    const Score sc(a);
    const int shift = c.n - a.q_len;              // position of query i: shift + i
    const int2* spans = c.w.spans + (int64_t)c.b * c.n_qt * T;
    Slot<C::SB> sb;
    float slope2 = 0.f;
    int head = -1;
    Item it(c);
    bool masked = it.i < c.items && it.partial(c);
    for (; it.i < c.items;) {
        const int t = it.t, q0 = t * T + half * 64;          // this thread's first column
        if (GEN && a.slopes && head != it.head) {
            head = it.head;
            slope2 = a.slopes[head] * LOG2E;
        }
        const int side = GEN ? side_of(a, shift + t * T, c.r0) : 1;
        const uint32_t i = it.i;
        const float* vec = (const float*)(base + C::VEC_OFF) + sb.at * 2 * T + half * 64;
        int2 see[2] = {};
        if (masked && a.first) {
            see[0] = spans[q0 + lane];
            see[1] = spans[q0 + 32 + lane];
        }
        if (!ptx::wait_bounded(&br.bfull[sb.at], sb.ph, abort, status, WAIT_NS)) return false;
        uint64_t add[2][16];
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int e = 0; e < 16; e += 2) ptx::lds_pairs(vec + g * 32 + 2 * e, add[g][e], add[g][e + 1]);
        if (!ptx::wait_bounded(br.sfull, i & 1, abort, status, WAIT_NS)) return false;
        ptx::tc_fence_after();
        uint64_t x[2][16];
        {
            uint32_t r[2][32];
            ptx::tmem_ld32(lanes + half * 64, r[0]);
            ptx::tmem_ld32(lanes + half * 64 + 32, r[1]);
            ptx::tmem_wait_ld(r[0]);
            ptx::tmem_wait_ld(r[1]);
            pairs32(r[0], x[0]);
            pairs32(r[1], x[1]);
        }
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            uint64_t bend[GEN ? 16 : 1];
            weights32<GEN>(x[g], add[g], sc, slope2, (float)(shift + q0 + g * 32 - row), 1.f, side, bend);
            if (masked) {
                if (!a.first) {
                    // the queries that see this key are a run: i >= row - shift, and i < that + window
                    const int lo = a.causal ? row - shift : row < c.n ? INT_MIN / 2 : INT_MAX / 2;
                    const int64_t hi = row >= c.n ? lo : a.window ? (int64_t)row - shift + a.window : a.q_len;
                    const int l0 = max(lo, 0) - (q0 + g * 32), l1 = (int)min(hi, (int64_t)a.q_len) - (q0 + g * 32);
                    if (!__all_sync(~0u, l0 <= 0 && l1 >= 32)) mask32(x[g], l0, (uint32_t)max(l1 - l0, 0), 0.f);
                } else {
                    const uint32_t bits = seen32(see[g], row - lane, lane);
                    if (!__all_sync(~0u, bits == ~0u)) keep32(x[g], bits);
                }
            }
            uint32_t p[16];
            round32<F16>(x[g], p);
            ptx::tmem_st16(lanes + half * 64 + g * 16, p);
            if (GEN && sc.capped) {
                if (masked) {   // a masked pair's bend may be a NaN: the maximum takes the number
#pragma unroll
                    for (int e = 0; e < 16; ++e) bend[e] = ptx::pack2(fmaxf(ptx::lo2(bend[e]), 0.f), fmaxf(ptx::hi2(bend[e]), 0.f));
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) x[g][e] = ptx::mul2(x[g][e], bend[e]);
            }
        }
        // delta leaves the stage before it may be refilled (after dV of this tile)
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int e = 0; e < 16; e += 2) ptx::lds_pairs(vec + T + g * 32 + 2 * e, add[g][e], add[g][e + 1]);
        ptx::tmem_wait_st();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(br.pfull);
        sb.next();
        it.next(c);
        const bool next_masked = it.i < c.items && it.partial(c);
        if (!ptx::wait_bounded(&br.dpfull[0], i & 1, abort, status, WAIT_NS)) return false;
        ptx::tc_fence_after();
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            uint32_t r[32];
            ptx::tmem_ld32(lanes + 128 + half * 64 + g * 32, r);
            ptx::tmem_wait_ld(r);
            uint64_t d[16];
            pairs32(r, d);
#pragma unroll
            for (int e = 0; e < 16; ++e) d[e] = ptx::mul2(x[g][e], ptx::add2(d[e], add[g][e]));
            if (masked) {   // zero, whatever dP of a masked pair holds
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    d[e] = ptx::pack2(ptx::lo2(x[g][e]) == 0.f ? 0.f : ptx::lo2(d[e]), ptx::hi2(x[g][e]) == 0.f ? 0.f : ptx::hi2(d[e]));
            }
            if (F16) {
#pragma unroll
                for (int e = 0; e < 16; ++e) d[e] = ptx::mul2(d[e], ptx::both2(up_p));
            }
            uint32_t p[16];
            round32<F16>(d, p);
            ptx::tmem_st16(lanes + 128 + half * 64 + g * 16, p);
        }
        ptx::tmem_wait_st();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&br.dsfull[0]);
        masked = next_masked;
    }
    return true;
}

template <int DP, bool F16, bool GEN>
__device__ __forceinline__ bool compute_query(const Cta& c, const Bars& br, uint32_t lanes, int half, int row, float up_p,
                                              volatile int* abort, int* status) {
    const Prob& a = c.a;
    const int lane = threadIdx.x & 31;
    const Score sc(a);
    const int64_t at = (((int64_t)c.b * a.heads + c.h) * c.n_qt) * T + row;
    const uint64_t nlse = ptx::both2(c.w.lse2[at]), ndelta = ptx::both2(c.w.delta[at]);
    // rows behind the last query have no weight, and are not stored
    const int2 span = row < a.q_len ? c.w.spans[(int64_t)c.b * c.n_qt * T + row] : make_int2(0, INT_MAX);
    const float slope2 = GEN && a.slopes ? a.slopes[c.h] * LOG2E : 0.f;
    const int shift = c.n - a.q_len;
    uint64_t add[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) add[e] = nlse;
    for (Item it(c); it.i < c.items; it.next(c)) {
        const int k0 = it.t * T + half * 64;                 // this thread's first column
        const uint32_t i = it.i, buf = i & 1;
        const bool masked = it.partial(c);
        const int side = GEN ? side_of(a, shift + c.r0, it.t * T) : 1;
        if (!ptx::wait_bounded(br.sfull, i & 1, abort, status, WAIT_NS)) return false;
        ptx::tc_fence_after();
        uint64_t x[2][16];
        {
            uint32_t r[2][32];
            ptx::tmem_ld32(lanes + half * 64, r[0]);
            ptx::tmem_ld32(lanes + half * 64 + 32, r[1]);
            ptx::tmem_wait_ld(r[0]);
            ptx::tmem_wait_ld(r[1]);
            pairs32(r[0], x[0]);
            pairs32(r[1], x[1]);
        }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(br.sread);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            uint64_t bend[GEN ? 16 : 1];
            weights32<GEN>(x[g], add, sc, slope2, (float)(shift + row - k0 - g * 32), -1.f, side, bend);
            if (GEN && sc.capped) {   // before the mask: a masked pair's bend may be a NaN
#pragma unroll
                for (int e = 0; e < 16; ++e) x[g][e] = ptx::mul2(x[g][e], bend[e]);
            }
            if (masked) {
                const int lo = span.x - k0 - g * 32;
                if (!__all_sync(~0u, lo <= 0 && (int64_t)lo + (span.y - span.x) >= 32))
                    mask32(x[g], lo, (uint32_t)(span.y - span.x), 0.f);
            }
        }
        const uint32_t dp = lanes + 128 + buf * 128 + half * 64;
        if (!ptx::wait_bounded(&br.dpfull[buf], (i >> 1) & 1, abort, status, WAIT_NS)) return false;
        ptx::tc_fence_after();
        uint32_t r[2][32];
        ptx::tmem_ld32(dp, r[0]);
        ptx::tmem_ld32(dp + 32, r[1]);
        ptx::tmem_wait_ld(r[0]);
        ptx::tmem_wait_ld(r[1]);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            uint64_t d[16];
            pairs32(r[g], d);
#pragma unroll
            for (int e = 0; e < 16; ++e) d[e] = ptx::mul2(x[g][e], ptx::add2(d[e], ndelta));
            if (masked) {   // zero, whatever dP of a masked pair holds
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    d[e] = ptx::pack2(ptx::lo2(x[g][e]) == 0.f ? 0.f : ptx::lo2(d[e]), ptx::hi2(x[g][e]) == 0.f ? 0.f : ptx::hi2(d[e]));
            }
            if (F16) {
#pragma unroll
                for (int e = 0; e < 16; ++e) d[e] = ptx::mul2(d[e], ptx::both2(up_p));
            }
            uint32_t p[16];
            round32<F16>(d, p);
            ptx::tmem_st16(dp + g * 16, p);
        }
        ptx::tmem_wait_st();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&br.dsfull[buf]);
    }
    return true;
}

// dV row `out` (or this part's `sums`): the NaN and infinite dO elements that the guard took out, of the queries that
// see this key.
template <bool F16>
__device__ void put_back(const Cta& c, uint8_t* out, float* sums, int row) {
    const Prob& a = c.a;
    for (Item it(c); it.i < c.items; it.next(c)) {
        if (!it.partial(c)) continue;
        const int q1 = min((it.t + 1) * T, a.q_len);
        for (int q = it.t * T; q < q1; ++q) {
            const int2 sp = row_span(a, c.b, q, c.n);
            if (row < sp.x || row >= sp.y) continue;
            const uint16_t* g = (const uint16_t*)a.d_o.p + c.b * a.d_o.sb + (int64_t)q * a.d_o.ss + it.head * a.d_o.sh;
            constexpr uint16_t EXP = F16 ? 0x7c00 : 0x7f80;
            for (int d = 0; d < a.dim; ++d)
                if ((g[d] & EXP) == EXP) {
                    if (sums) {
                        sums[d] += pair_of<F16>(g[d]).x;
                        continue;
                    }
                    uint16_t* o = (uint16_t*)out + d;
                    const float2 f = pair_of<F16>((uint32_t)*o | ((uint32_t)g[d] << 16));
                    *o = (uint16_t)ptx::pack16<F16>(f.x + f.y, 0.f);
                }
        }
    }
}

template <int DP, bool F16, bool GEN>
__global__ void __launch_bounds__(NTHREADS, 1)
gradient_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                const __grid_constant__ CUtensorMap tmv, const __grid_constant__ CUtensorMap tmdo,
                const __grid_constant__ Args args, int* __restrict__ status) {
    using C = Cfg<DP>;
    extern __shared__ __align__(1024) uint8_t base[];
    if (ptx::smem_u32(base) & 1023) {   // the swizzled tiles need it, and there is no room to round up
        if (threadIdx.x == 0) atomicExch(status, FD_ERR_UNSUPPORTED);
        return;
    }
    Bars br;
    br.opfull = (uint64_t*)(base + C::BAR_OFF);
    br.afull = br.opfull + 1;
    br.aempty = br.afull + C::SA;
    br.bfull = br.aempty + C::SA;
    br.bempty = br.bfull + C::SB;
    br.sfull = br.bempty + C::SB;
    br.sread = br.sfull + 1;
    br.pfull = br.sread + 1;
    br.dpfull = br.pfull + 1;
    br.dsfull = br.dpfull + 2;
    br.accfull = br.dsfull + 2;
    br.toguard = br.accfull + 1;
    br.guarded = br.toguard + 1;
    Misc& ms = *(Misc*)(base + C::MISC_OFF);
    volatile int* abort = &ms.abort;
    const Prob& a = args.a;
    const Work& w = args.w;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Cta c{a, w};
    int parts, part;
    const int x = (int)blockIdx.x < args.first ? blockIdx.x : blockIdx.x - args.first;
    c.key_side = ((int)blockIdx.x < args.first) == (args.keys_first != 0);
    if (c.key_side) {
        // earlier key tiles are seen by more queries under a causal mask: they start first
        const int nh = a.kv_heads * a.batch;
        parts = args.key_parts;
        part = x / nh % parts;
        c.tile = x / (nh * parts);
        c.b = x % nh / a.kv_heads;
        c.h = x % nh % a.kv_heads;
    } else {
        const int nh = a.heads * a.batch;
        parts = args.query_parts;
        part = x / nh % parts;
        c.tile = args.n_qt - 1 - x / (nh * parts);
        c.b = x % nh / a.heads;
        c.h = x % nh % a.heads;
    }
    c.r0 = c.tile * T;
    c.n = keys_of(a, c.b);
    c.n_qt = args.n_qt;
    c.bounds = w.bounds + (int64_t)c.b * args.n_qt;

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::NBARS; ++i) {
            uint64_t* bar = br.opfull + i;
            ptx::mbar_init(bar, bar == br.sread || bar == br.pfull || (bar >= br.dsfull && bar < br.dsfull + 2) ? 8 : 1);
        }
        ms.abort = 0;
        ms.poison = 0;
        ms.lo = 0x7fffffff;
        ms.hi = 0;
        ptx::fence_mbar_init();
    }
    if (warp == MMA_WARP) {
        ptx::tmem_alloc(&ms.tmem, TMEM_COLS);
        ptx::tmem_relinquish();
    }
    if (warp == TMA_WARP && lane == 0) {
        ptx::prefetch_tmap(&tmq);
        ptx::prefetch_tmap(&tmk);
        ptx::prefetch_tmap(&tmv);
        ptx::prefetch_tmap(&tmdo);
    }
    __syncthreads();
    if (warp == TMA_WARP && lane == 0) load_resident<DP>(c, br, base, &tmq, &tmk, &tmv, &tmdo);
    __syncwarp();
    asm volatile("griddepcontrol.wait;" ::: "memory");   // prep_kernel's results from here on
    if (c.key_side) {
        int lo = 0x7fffffff, hi = 0;
        for (int t = threadIdx.x; t < args.n_qt; t += NTHREADS)
            if (c.bounds[t].hi > c.r0 && c.bounds[t].lo < c.r0 + T) {
                lo = min(lo, t);
                hi = max(hi, t + 1);
            }
        lo = warp_min(lo);
        hi = warp_max(hi);
        if (lane == 0) {
            atomicMin(&ms.lo, lo);
            atomicMax(&ms.hi, hi);
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = ms.tmem;
    c.own = {0, 0, 0, 0};
    if (c.key_side) {
        c.t0 = ms.lo;
        c.nt = ms.hi > ms.lo ? ms.hi - ms.lo : 0;
    } else {
        c.own = c.bounds[c.tile];
        c.t0 = c.own.lo / T;
        c.nt = c.own.hi > c.own.lo ? (c.own.hi + T - 1) / T - c.t0 : 0;
    }
    c.items = c.key_side ? c.nt * a.group : c.nt;
    c.skip = 0;
    if (parts > 1) {
        c.skip = (int)((int64_t)c.items * part / parts);
        c.items = (int)((int64_t)c.items * (part + 1) / parts) - c.skip;
    }

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
        if (warp == TMA_WARP) {
            if (lane == 0 && c.items > 0) produce<DP, F16>(c, br, base, &tmq, &tmk, &tmv, &tmdo, abort, status);
            if (lane == 0 && c.items == 0) wait_landed(br.opfull, 0);
        } else if (warp == MMA_WARP) {
            if (c.items > 0) issue<DP, F16>(c, br, base, tmem, abort, status);
        } else if (warp == GUARD_WARP) {
            watch<DP, F16>(c, br, base, lane, &ms.poison, abort, status);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(COMPUTE_REGS));
        const int half = warp >> 2;                 // columns 64 half .. of each score tile
        const int row = c.r0 + (threadIdx.x & 127); // this thread's key (key side) or query
        const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);
        // fp16 keeps 2^-14 .. 65504: dS is scaled by a power of two that brings its bound 2 |dO| |V|, over the rows of
        // this sequence and key head that take part, to 2^14 .. 2^15, and the accumulator is scaled back at the end
        float up = 1.f, p_back = 1.f;
        if (F16) {
            const unsigned* top = w.top + 2 * (c.b * a.kv_heads + (c.key_side ? c.h : c.h / a.group));
            const float m2 = __uint_as_float(top[0]) * __uint_as_float(top[1]);
            if (m2 > 0.f && m2 < INFINITY) up = exp2f(14.f - ceilf(0.5f * log2f(m2)));
            up = fminf(fmaxf(up, 0x1p-60f), 0x1p60f);
            p_back = exp2f(-P_SHIFT_F16);
        }
        const bool ok = c.key_side ? compute_key<DP, F16, GEN>(c, br, base, lanes, half, row, up * p_back, abort, status)
                                   : compute_query<DP, F16, GEN>(c, br, lanes, half, row, up * p_back, abort, status);
        const bool have = c.items > 0 && ok && ptx::wait_bounded(br.accfull, 0, abort, status, WAIT_NS);
        ptx::tc_fence_after();
        // gave up: NaN, not numbers that could pass for the sums (store_cols has zeros in their place)
        const float given = c.items > 0 && !have ? __int_as_float(0x7fffffff) : 1.f;
        const float back = given * a.scale / up;
        // this row's sums of this part, if there are parts
        auto sums = [&](float* to, int rows, int heads) {
            return parts > 1 ? to + ((((int64_t)part * a.batch + c.b) * rows + row) * heads + c.h) * a.dim : nullptr;
        };
        if (!c.key_side) {
            uint8_t* out = (uint8_t*)a.dq.p + 2 * (c.b * a.dq.sb + (int64_t)row * a.dq.ss + c.h * a.dq.sh);
            store_cols<DP / 2, F16>(lanes + 384 + half * (DP / 2), back, out, sums(w.dq, a.q_len, a.heads), half * (DP / 2),
                                    a.dim, row < a.q_len, have);
        } else if (half == 0) {
            uint8_t* out = (uint8_t*)a.dv.p + 2 * (c.b * a.dv.sb + (int64_t)row * a.dv.ss + c.h * a.dv.sh);
            float* to = sums(w.dv, a.k_len, a.kv_heads);
            store_cols<DP, F16>(lanes + 256, given * p_back, out, to, 0, a.dim, row < a.k_len, have);
            if (have && row < a.k_len && *(volatile int*)&ms.poison) put_back<F16>(c, out, to, row);
        } else {
            uint8_t* out = (uint8_t*)a.dk.p + 2 * (c.b * a.dk.sb + (int64_t)row * a.dk.ss + c.h * a.dk.sh);
            store_cols<DP, F16>(lanes + 384, back, out, sums(w.dk, a.k_len, a.kv_heads), 0, a.dim, row < a.k_len, have);
        }
        ptx::tc_fence_before();
    }
    __syncthreads();
    if (warp == MMA_WARP) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, TMEM_COLS);
    }
}

// One gradient's parts, in order.
struct Sums {
    const float* parts;
    View out;
    int n, rows, heads;
};

// Thread: eight coordinates of a row of dq, dk or dv.
template <bool F16>
__global__ void __launch_bounds__(256) sum_kernel(const __grid_constant__ Sums dq, const __grid_constant__ Sums dk,
                                                  const __grid_constant__ Sums dv, int batch, int dim) {
    int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int pieces = dim / 8;
    for (int g = 0; g < 3; ++g) {
        const Sums& z = g == 0 ? dq : g == 1 ? dk : dv;
        const int64_t rows = z.n > 1 ? (int64_t)batch * z.rows * z.heads : 0;
        if (x >= rows * pieces) {
            x -= rows * pieces;
            continue;
        }
        const int64_t r = x / pieces, t = r / z.heads, b = t / z.rows;
        const int d = (int)(x - r * pieces) * 8, h = (int)(r - t * z.heads);
        float f[8] = {};
#pragma unroll 4
        for (int p = 0; p < z.n; ++p) {
            const float* o = z.parts + (p * rows + r) * dim + d;
            const float4 u = *(const float4*)o, v = *(const float4*)(o + 4);
            const float e[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] += e[i];
        }
        store8<F16>((uint16_t*)z.out.p + b * z.out.sb + (t - b * z.rows) * z.out.ss + h * z.out.sh + d, nullptr, f);
        return;
    }
}

template <int DP, bool F16, bool GEN>
int launch(const Prob& a, const Work& w, const Shape& z, cudaStream_t s) {
    CUtensorMap q, k, v, g;
    FD_TRY(make_head_map(&q, a.q, a.q_len, a.heads, a.batch, a.dim, F16));
    FD_TRY(make_head_map(&k, a.k, a.k_len, a.kv_heads, a.batch, a.dim, F16));
    FD_TRY(make_head_map(&v, a.v, a.k_len, a.kv_heads, a.batch, a.dim, F16));
    FD_TRY(make_head_map(&g, a.d_o, a.q_len, a.heads, a.batch, a.dim, F16));
    int* status = nullptr;
    FD_TRY(status_word(&status));
    Args args;
    args.a = a;
    args.w = w;
    args.n_qt = (int)cdiv(a.q_len, T);
    const int n_kt = (int)cdiv(a.k_len, T);
    args.key_parts = z.key_parts();
    args.query_parts = z.query_parts();
    const int64_t keys = (int64_t)n_kt * a.kv_heads * a.batch * args.key_parts;
    const int64_t queries = (int64_t)args.n_qt * a.heads * a.batch * args.query_parts, blocks = keys + queries;
    args.keys_first = z.tiles(a.q_len, a.k_len) * a.group * args.query_parts >= z.tiles(a.k_len, a.q_len) * args.key_parts;
    FD_CHECK_ARG(blocks <= 0x7fffffff && cdiv(a.q_len, T) + cdiv(a.k_len, T) <= 0x7fffffff, "fd_attention: too many tiles");
    args.first = (int)(args.keys_first ? keys : queries);
    const int v_blocks = F16 ? n_kt : 0;
    if (F16) FD_CUDA_TRY(cudaMemsetAsync(w.top, 0, 2 * sizeof(unsigned) * a.batch * a.kv_heads, s));
    prep_kernel<F16><<<dim3(args.n_qt + v_blocks, a.heads, a.batch), 256, 0, s>>>(a, w, args.n_qt);
    FD_CUDA_TRY(cudaGetLastError());
    FD_TRY((allow_smem<gradient_kernel<DP, F16, GEN>>(Cfg<DP>::SMEM)));
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(NTHREADS);
    cfg.dynamicSmemBytes = Cfg<DP>::SMEM;
    cfg.stream = s;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    FD_CUDA_TRY(cudaLaunchKernelEx(&cfg, gradient_kernel<DP, F16, GEN>, q, k, v, g, args, status));
    const int64_t joined = (args.query_parts > 1 ? (int64_t)a.q_len * a.heads : 0) +
                           (args.key_parts > 1 ? 2 * (int64_t)a.k_len * a.kv_heads : 0);
    if (joined > 0) {
        const Sums dq{w.dq, a.dq, args.query_parts, a.q_len, a.heads}, dk{w.dk, a.dk, args.key_parts, a.k_len, a.kv_heads},
            dv{w.dv, a.dv, args.key_parts, a.k_len, a.kv_heads};
        sum_kernel<F16><<<(unsigned)cdiv(joined * a.batch * (a.dim / 8), 256), 256, 0, s>>>(dq, dk, dv, a.batch, a.dim);
    }
    FD_CUDA_TRY(cudaGetLastError());
    return FD_OK;
}

template <int DP>
int by_type(const Prob& a, int dtype, const Work& w, const Shape& z, cudaStream_t s) {
    const bool gen = a.cap > 0.f || a.slopes;
    if (dtype == FD_DTYPE_F16) return gen ? launch<DP, true, true>(a, w, z, s) : launch<DP, true, false>(a, w, z, s);
    return gen ? launch<DP, false, true>(a, w, z, s) : launch<DP, false, false>(a, w, z, s);
}

}  // namespace bwd

size_t tc_backward_bytes(const Prob& a) { return bwd::work_layout(nullptr, nullptr, bwd::Shape(a)); }

int tc_backward(const Prob& a, int dtype, void* workspace, cudaStream_t s) {
    const bwd::Shape z(a);
    bwd::Work w;
    bwd::work_layout(&w, workspace, z);
    return a.dim <= 64 ? bwd::by_type<64>(a, dtype, w, z, s) : bwd::by_type<128>(a, dtype, w, z, s);
}

}  // namespace attn
}  // namespace fd
