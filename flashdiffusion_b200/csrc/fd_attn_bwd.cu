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
// longest first, so that the short ones fill the SMs at its end.
//
// CTA: two compute warpgroups that share the 128 rows of the accumulators (64
// columns of each score tile apiece), and a warpgroup with a TMA producer, an
// MMA issuer and a guard.
//   key side    rows = keys.  TMEM: S^T | dP^T | dV | dK.  While the exponentials
//               of tile i + 1 wait for S^T, the tensor core runs dV(i), S(i+1),
//               and while dS(i) is made ... : P^T and dS^T go back to TMEM over
//               the scores they came from and are the A operands.
//   query side  rows = queries.  TMEM: S | dP, dP | dQ (dP in two buffers, so that
//               the next tile's products do not wait for dS).
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
    float* delta;        // [batch * heads][rows padded to 128]
    float* lse2;         // the same, base 2 (less P_SHIFT_F16 for fp16); +inf for rows that see nothing and for the padding
    Bounds* bounds;      // [batch][query tiles]
    unsigned* top;       // fp16: bits of the largest |dO row|^2 and |V row|^2
};

__host__ __device__ inline size_t work_layout(Work* w, void* base, int64_t bh, int64_t batch, int64_t n_qt) {
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) & ~(size_t)255;
        return (char*)base + here;
    };
    char* a = take(sizeof(float) * bh * n_qt * T);
    char* b = take(sizeof(float) * bh * n_qt * T);
    char* c = take(sizeof(Bounds) * batch * n_qt);
    char* d = take(2 * sizeof(unsigned));
    if (w) *w = {(float*)a, (float*)b, (Bounds*)c, (unsigned*)d};
    return at;
}

template <bool F16>
__device__ __forceinline__ float2 pair_of(uint32_t w) {
    if (F16) return __half22float2(*(__half2*)&w);
    return __bfloat1622float2(*(__nv_bfloat162*)&w);
}

// Block (t, h, b): delta and lse2 of 128 rows, 16 lanes a row (one 16-byte piece
// each); head 0 also makes the tile's bounds.  fp16: the largest row norms of dO
// and, in the blocks behind the query tiles, of V.  Bandwidth-bound: dO and o are
// read once.
template <bool F16>
__global__ void __launch_bounds__(256) prep_kernel(const __grid_constant__ Prob a, const __grid_constant__ Work w, int n_qt) {
    const int h = blockIdx.y, b = blockIdx.z, t = blockIdx.x;
    const int piece = threadIdx.x & 15, r0 = threadIdx.x >> 4;
    float top = 0.f;
    if (t >= n_qt) {
        if (h >= a.kv_heads) return;
        for (int r = r0; r < T; r += 16) {
            const int64_t j = (int64_t)(t - n_qt) * T + r;
            float s = 0.f;
            if (j < a.k_len && piece * 8 < a.dim) {
                const uint4 x = *(const uint4*)((const uint16_t*)a.v.p + b * a.v.sb + j * a.v.ss + h * a.v.sh + piece * 8);
                const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
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
        if ((threadIdx.x & 31) == 0 && top > 0.f) atomicMax(&w.top[1], __float_as_uint(top));
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
    for (int r = r0; r < T; r += 16) {
        const int64_t i = (int64_t)t * T + r;
        float d = 0.f, s = 0.f;
        const bool real = i < a.q_len;
        if (real && piece * 8 < a.dim) {
            const uint4 x = *(const uint4*)((const uint16_t*)a.d_o.p + b * a.d_o.sb + i * a.d_o.ss + h * a.d_o.sh + piece * 8);
            const uint4 y = *(const uint4*)((const uint16_t*)a.o.p + b * a.o.sb + i * a.o.ss + h * a.o.sh + piece * 8);
            const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 f = pair_of<F16>(xs[e]), g = pair_of<F16>(ys[e]);
                d = fmaf(f.x, g.x, fmaf(f.y, g.y, d));
                if (F16) s = fmaf(f.x, f.x, fmaf(f.y, f.y, s));
            }
        }
        for (int o = 8; o; o >>= 1) {
            d += __shfl_xor_sync(~0u, d, o);
            if (F16) s += __shfl_xor_sync(~0u, s, o);
        }
        const float lse = real ? a.lse[((int64_t)b * a.heads + h) * a.q_len + i] : -INFINITY;
        const bool some = lse != -INFINITY;
        if (F16 && some && s < INFINITY) top = fmaxf(top, s);
        if (piece == 0) {
            w.delta[base + i] = some ? d : 0.f;
            w.lse2[base + i] = some ? lse * LOG2E - (F16 ? P_SHIFT_F16 : 0.f) : INFINITY;
        }
    }
    if (F16) {
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
        if ((threadIdx.x & 31) == 0 && top > 0.f) atomicMax(&w.top[0], __float_as_uint(top));
    }
}

template <int DP>
struct Cfg {
    static constexpr int BOXES = DP / 64;
    static constexpr uint32_t TILE = BOXES * BOX_BYTES;
    static constexpr int STAGES = 2;
    static constexpr uint32_t RING_OFF = 2 * TILE;                       // behind the resident pair
    static constexpr uint32_t VEC_OFF = RING_OFF + 2 * STAGES * TILE;    // lse2 and delta of each stage
    static constexpr uint32_t BAR_OFF = VEC_OFF + STAGES * 2 * T * 4;
    static constexpr int NBARS = 32;
    static constexpr uint32_t MISC_OFF = BAR_OFF + NBARS * 8;
    static constexpr uint32_t SMEM = MISC_OFF + 64 + 1024;
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
    int n_qt, n_kt, n_key;   // query tiles, key tiles, CTAs of the key side
};

// A tile in shared memory: elements that are NaN or infinite become zeros; true if there were any.
template <bool F16>
__device__ __forceinline__ bool clear_bad(uint8_t* tile, int bytes, int lane) {
    constexpr uint32_t EXP = F16 ? 0x7c00u : 0x7f80u;
    bool bad = false;
#pragma unroll 8
    for (int i = lane; i < bytes / 16; i += 32) {
        const uint4 x = ((uint4*)tile)[i];
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) bad = bad || (w[e] & EXP) == EXP || ((w[e] >> 16) & EXP) == EXP;
    }
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

// Store N columns of one accumulator row, times f, as 16-bit values behind column c0 of `out`.
template <int N, bool F16>
__device__ __forceinline__ void store_cols(uint32_t taddr, float f, uint8_t* out, int c0, int dim, bool live, bool have) {
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

template <int DP, bool F16, bool GEN>
__global__ void __launch_bounds__(NTHREADS, 1)
gradient_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                const __grid_constant__ CUtensorMap tmv, const __grid_constant__ CUtensorMap tmdo,
                const __grid_constant__ Args args, int* __restrict__ status) {
    using C = Cfg<DP>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* bars = (uint64_t*)(base + C::BAR_OFF);
    // ring A: Q (key side) or K (query side), needed until the last product of a tile;
    // ring B: dO or V
    uint64_t *opfull = bars, *afull = bars + 1, *aempty = afull + C::STAGES, *bfull = aempty + C::STAGES,
             *bempty = bfull + C::STAGES, *sfull = bempty + C::STAGES, *sread = sfull + 1, *pfull = sread + 1,
             *dpfull = pfull + 1, *dsfull = dpfull + 2, *accfull = dsfull + 2, *toguard = accfull + 1,
             *guarded = toguard + 1;
    Misc& ms = *(Misc*)(base + C::MISC_OFF);
    volatile int* abort = &ms.abort;
    const Prob& a = args.a;
    const Work& w = args.w;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool key_side = (int)blockIdx.x < args.n_key;
    int tile, b, h;     // h: key head on the key side, query head on the query side
    if (key_side) {
        // earlier key tiles are seen by more queries under a causal mask: they start first
        const int nh = a.kv_heads * a.batch;
        tile = blockIdx.x / nh;
        b = blockIdx.x % nh / a.kv_heads;
        h = blockIdx.x % nh % a.kv_heads;
    } else {
        const int nh = a.heads * a.batch, u = blockIdx.x - args.n_key;
        tile = args.n_qt - 1 - u / nh;
        b = u % nh / a.heads;
        h = u % nh % a.heads;
    }
    const int r0 = tile * T;                     // first row of this CTA
    const int n = keys_of(a, b);
    const Bounds* bounds = w.bounds + (int64_t)b * args.n_qt;

    if (threadIdx.x == 0) {
        ptx::mbar_init(opfull, 1);
        for (int i = 0; i < C::STAGES; ++i) {
            ptx::mbar_init(&afull[i], 1);
            ptx::mbar_init(&aempty[i], 1);
            ptx::mbar_init(&bfull[i], 1);
            ptx::mbar_init(&bempty[i], 1);
        }
        ptx::mbar_init(sfull, 1);
        ptx::mbar_init(sread, 8);
        ptx::mbar_init(pfull, 8);
        ptx::mbar_init(&dpfull[0], 1);
        ptx::mbar_init(&dpfull[1], 1);
        ptx::mbar_init(&dsfull[0], 8);
        ptx::mbar_init(&dsfull[1], 8);
        ptx::mbar_init(accfull, 1);
        ptx::mbar_init(toguard, 1);
        ptx::mbar_init(guarded, 1);
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
    if (key_side) {
        int lo = 0x7fffffff, hi = 0;
        for (int t = threadIdx.x; t < args.n_qt; t += NTHREADS)
            if (bounds[t].hi > r0 && bounds[t].lo < r0 + T) {
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
    // the other side's tiles, t0 .. t0 + nt, walked `items / nt` times (once for each head of the group)
    int t0, nt;
    Bounds own = {0, 0, 0, 0};
    if (key_side) {
        t0 = ms.lo;
        nt = ms.hi > ms.lo ? ms.hi - ms.lo : 0;
    } else {
        own = bounds[tile];
        t0 = own.lo / T;
        nt = own.hi > own.lo ? (own.hi + T - 1) / T - t0 : 0;
    }
    const int items = key_side ? nt * a.group : nt;
    auto tile_of = [&](int i) { return t0 + (key_side ? i % nt : i); };
    auto head_of = [&](int i) { return h * a.group + i / nt; };
    // some pair of the tile is masked
    auto partial = [&](int i) {
        const int t = tile_of(i);
        if (!key_side) return t * T < own.flo || (t + 1) * T > own.fhi;
        const Bounds o = bounds[t];
        return r0 < o.flo || r0 + T > o.fhi;
    };

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
        uint8_t* ring_a = base + C::RING_OFF;
        uint8_t* ring_b = ring_a + C::STAGES * C::TILE;
        if (warp == TMA_WARP) {
            if (lane == 0 && items > 0) {
                auto load = [&](uint8_t* dst, const CUtensorMap* m, uint64_t* bar, int t, int hh) {
                    for (int c = 0; c < C::BOXES; ++c) ptx::tma_load_4d(dst + c * BOX_BYTES, m, bar, c * 64, t * T, hh, b);
                };
                ptx::mbar_expect_tx(opfull, 2 * C::TILE);
                const int hk = key_side ? h : h / a.group;
                load(base, key_side ? &tmk : &tmq, opfull, tile, h);
                load(base + C::TILE, key_side ? &tmv : &tmdo, opfull, tile, h);
                int i = 0, ib = 0;
                for (; i < items; ++i, ++ib) {
                    const int st = i % C::STAGES, ph = (i / C::STAGES) & 1;
                    const int t = tile_of(i), hh = key_side ? head_of(i) : hk;
                    if (!ptx::wait_bounded(&aempty[st], ph ^ 1, abort, status, WAIT_NS)) break;
                    ptx::mbar_expect_tx(&afull[st], C::TILE + (key_side ? 2 * T * 4 : 0));
                    load(ring_a + st * C::TILE, key_side ? &tmq : &tmk, &afull[st], t, hh);
                    if (key_side) {
                        float* vec = (float*)(base + C::VEC_OFF) + st * 2 * T;
                        const int64_t at = (((int64_t)b * a.heads + hh) * args.n_qt + t) * T;
                        ptx::bulk_load(vec, w.lse2 + at, T * 4, &afull[st]);
                        ptx::bulk_load(vec + T, w.delta + at, T * 4, &afull[st]);
                    }
                    if (!ptx::wait_bounded(&bempty[st], ph ^ 1, abort, status, WAIT_NS)) { ++i; break; }
                    ptx::mbar_expect_tx(&bfull[st], C::TILE);
                    load(ring_b + st * C::TILE, key_side ? &tmdo : &tmv, &bfull[st], t, hh);
                }
                if (*abort) {   // the copies in flight still write into this block's memory
                    wait_landed(opfull, 0);
                    for (int z = max(0, i - C::STAGES); z < i; ++z) wait_landed(&afull[z % C::STAGES], (z / C::STAGES) & 1);
                    for (int z = max(0, ib - C::STAGES); z < ib; ++z) wait_landed(&bfull[z % C::STAGES], (z / C::STAGES) & 1);
                }
            }
        } else if (warp == MMA_WARP) {
            if (lane == 0 && items > 0) {
                const int kd = (a.dim + 15) / 16;
                const uint32_t id_s = ptx::idesc_f32acc(T, T, F16);
                const uint32_t id_acc = ptx::idesc_f32acc(T, kd * 16, F16) | ptx::IDESC_B_MN;
                const uint32_t op0 = ptx::smem_u32(base), op1 = op0 + C::TILE;
                const uint32_t ra = ptx::smem_u32(ring_a), rb = ptx::smem_u32(ring_b);
                auto wait = [&](uint64_t* bar, int ph) { return ptx::wait_bounded(bar, ph & 1, abort, status, WAIT_NS); };
                // D[128 x 128] = resident operand . ring operand^T
                auto scores = [&](uint32_t d, uint32_t op, uint32_t rg, int st) {
                    ptx::tc_fence_after();
                    for (int ks = 0; ks < kd; ++ks)
                        ptx::umma_ss(d, kmajor(op, ks), kmajor(rg + st * C::TILE, ks), id_s, ks > 0);
                };
                // acc[128 x dim] += (16-bit tile in TMEM, 64 columns of it at `src`, 64 at `src` + 64) . ring tile
                auto sum = [&](uint32_t acc, uint32_t src, uint32_t rg, int st, bool more) {
                    ptx::tc_fence_after();
#pragma unroll
                    for (int ks = 0; ks < T / 16; ++ks)
                        ptx::umma_ts(acc, src + (ks >> 2) * 64 + (ks & 3) * 8, mnmajor(rg + st * C::TILE, ks), id_acc,
                                     more || ks > 0);
                };
                uint32_t ng = 0;
                bool ok = wait(opfull, 0);
                if (key_side) {
                    const uint32_t S = tmem, DPT = tmem + 128, DV = tmem + 256, DK = tmem + 384;
                    bool look = false;
                    auto first = [&](int i) {      // S^T(i)
                        const int st = i % C::STAGES;
                        if (!wait(&afull[st], i / C::STAGES)) return false;
                        scores(S, op0, ra, st);
                        ptx::umma_commit(sfull);
                        return true;
                    };
                    auto second = [&](int i) {     // dP^T(i)
                        const int st = i % C::STAGES;
                        if (!wait(&bfull[st], i / C::STAGES)) return false;
                        scores(DPT, op1, rb, st);
                        ptx::umma_commit(&dpfull[0]);
                        look = partial(i);
                        if (look) ptx::mbar_arrive(toguard);
                        return true;
                    };
                    ok = ok && first(0) && second(0);
                    for (int i = 0; i < items && ok; ++i) {
                        const int st = i % C::STAGES;
                        if (!(ok = wait(pfull, i))) break;
                        if (look) {
                            if (!(ok = wait(guarded, ng))) break;
                            ++ng;
                        }
                        sum(DV, S, rb, st, i > 0);
                        ptx::umma_commit(&bempty[st]);
                        if (i + 1 < items && !(ok = first(i + 1))) break;
                        if (!(ok = wait(&dsfull[0], i))) break;
                        sum(DK, DPT, ra, st, i > 0);
                        ptx::umma_commit(&aempty[st]);
                        if (i + 1 < items) ok = second(i + 1);
                    }
                } else {
                    const uint32_t S = tmem, DQ = tmem + 384;
                    auto both = [&](int i) {       // S(i), dP(i)
                        const int st = i % C::STAGES;
                        if (!wait(&afull[st], i / C::STAGES)) return false;
                        scores(S, op0, ra, st);
                        ptx::umma_commit(sfull);
                        if (!wait(&bfull[st], i / C::STAGES)) return false;
                        scores(tmem + 128 + (i & 1) * 128, op1, rb, st);
                        ptx::umma_commit(&dpfull[i & 1]);
                        ptx::umma_commit(&bempty[st]);
                        return true;
                    };
                    ok = ok && both(0);
                    for (int i = 0; i < items && ok; ++i) {
                        const int st = i % C::STAGES;
                        const bool look = partial(i);
                        if (look) ptx::mbar_arrive(toguard);
                        if (i + 1 < items) {
                            if (!(ok = wait(sread, i))) break;
                            if (!(ok = both(i + 1))) break;
                        }
                        // one barrier for each dP buffer: a warp may be a tile ahead of another, and its
                        // arrival for i + 1 must not stand in for the other's for i
                        if (!(ok = wait(&dsfull[i & 1], i >> 1))) break;
                        if (look) {
                            if (!(ok = wait(guarded, ng))) break;
                            ++ng;
                        }
                        sum(DQ, tmem + 128 + (i & 1) * 128, ra, st, i > 0);
                        ptx::umma_commit(&aempty[st]);
                    }
                }
                ptx::umma_commit(accfull);
                if (!ok) wait_landed(accfull, 0);
            }
        } else if (warp == GUARD_WARP) {
            // Masked pairs have P = dS = 0, and zero times a NaN or an infinity of the other operand would
            // reach the sum: in partly visible tiles such elements become zeros before the product.  What a
            // visible pair loses with them is NaN already through lse (Q, K) or delta (dO) of its row, except
            // for dV, where a visible row's bad dO elements are put back at the end.
            uint32_t ng = 0;
            for (int i = 0; i < items; ++i) {
                if (!partial(i)) continue;
                const int st = i % C::STAGES, ph = (i / C::STAGES) & 1;
                // not before the issuer has seen the tile: see the forward kernel's guard
                if (!ptx::wait_bounded(toguard, ng & 1, abort, status, WAIT_NS)) break;
                ++ng;
                if (!ptx::wait_bounded(&afull[st], ph, abort, status, WAIT_NS)) break;
                clear_bad<F16>(ring_a + st * C::TILE, C::TILE, lane);
                if (key_side) {
                    if (!ptx::wait_bounded(&bfull[st], ph, abort, status, WAIT_NS)) break;
                    if (clear_bad<F16>(ring_b + st * C::TILE, C::TILE, lane) && lane == 0) ms.poison = 1;
                    __syncwarp();
                }
                if (lane == 0) ptx::mbar_arrive(guarded);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(COMPUTE_REGS));
        const int half = warp >> 2;                 // columns 64 half .. of each score tile
        const int lrow = threadIdx.x & 127;
        const int row = r0 + lrow;                  // this thread's key (key side) or query
        const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);
        Score sc;
        sc.cap2 = a.cap * LOG2E;
        sc.c = a.cap > 0.f ? a.scale / a.cap : a.scale * LOG2E;
        sc.slope2 = 0.f;
        const bool sloped = GEN && a.slopes;
        // fp16 keeps 2^-14 .. 65504: dS is scaled by a power of two that brings its bound 2 |dO| |V| to
        // 2^14 .. 2^15, and the accumulator is scaled back at the end
        float up = 1.f, up_p = 1.f, p_back = 1.f;
        if (F16) {
            const float m2 = __uint_as_float(w.top[0]) * __uint_as_float(w.top[1]);
            if (m2 > 0.f && m2 < INFINITY) up = exp2f(14.f - ceilf(0.5f * log2f(m2)));
            up = fminf(fmaxf(up, 0x1p-60f), 0x1p60f);
            p_back = exp2f(-P_SHIFT_F16);
            up_p = up * p_back;
        }
        int2 span = make_int2(0, 0x7fffffff);
        float my_lse2 = 0.f, my_delta = 0.f;
        if (!key_side) {
            const int64_t at = (((int64_t)b * a.heads + h) * args.n_qt + tile) * T + lrow;
            my_lse2 = w.lse2[at];
            my_delta = w.delta[at];
            if (row < a.q_len) span = row_span(a, b, row, n);
            if (sloped) sc.slope2 = a.slopes[h] * LOG2E;
        }
        const int shift = n - a.q_len;              // position of query i: shift + i
        bool ok = true;
        for (int i = 0; i < items; ++i) {
            const int t = tile_of(i);
            const float* vec = (const float*)(base + C::VEC_OFF) + (i % C::STAGES) * 2 * T + half * 64;
            if (key_side && sloped) sc.slope2 = a.slopes[head_of(i)] * LOG2E;
            const bool masked = partial(i);
            if (!ptx::wait_bounded(sfull, i & 1, abort, status, WAIT_NS)) { ok = false; break; }
            // the stage's lse2 and delta came with Q: sfull implies it
            ptx::tc_fence_after();
            uint32_t x[2][32];
            ptx::tmem_ld32(lanes + half * 64, x[0]);
            ptx::tmem_ld32(lanes + half * 64 + 32, x[1]);
            ptx::tmem_wait_ld(x[0]);
            ptx::tmem_wait_ld(x[1]);
            float(&v)[2][32] = reinterpret_cast<float(&)[2][32]>(x);
            if (!key_side) {
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(sread);
            }
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const int c0 = half * 64 + g * 32;   // column of v[g][0]
                float bend[GEN ? 32 : 1];
                if (GEN) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) v[g][e] *= sc.c;
                    if (sc.cap2 > 0.f) {
                        tanh_n(v[g]);
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            bend[e] = fmaf(-v[g][e], v[g][e], 1.f);
                            v[g][e] *= sc.cap2;
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) bend[e] = 1.f;
                    }
                    if (sc.slope2 != 0.f) {
                        // distance of column e from this row, as |at -+ e|: symmetric, one form for both sides
                        const float at = key_side ? (float)(row - shift - t * T - c0) : (float)(shift + row - t * T - c0);
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[g][e] = fmaf(-sc.slope2, fabsf(at - (float)e), v[g][e]);
                    }
                }
                const float c = GEN ? 1.f : sc.c;
                if (key_side) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        const float4 l4 = *(const float4*)(vec + g * 32 + e);
                        v[g][e] = ptx::ex2_mufu(fmaf(v[g][e], c, -l4.x));
                        v[g][e + 1] = ptx::ex2_mufu(fmaf(v[g][e + 1], c, -l4.y));
                        v[g][e + 2] = ptx::ex2_mufu(fmaf(v[g][e + 2], c, -l4.z));
                        v[g][e + 3] = ptx::ex2_mufu(fmaf(v[g][e + 3], c, -l4.w));
                    }
                    if (masked) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            const int q = t * T + c0 + e;
                            const int2 sp = q < a.q_len ? row_span(a, b, q, n) : make_int2(0, 0);
                            if (row < sp.x || row >= sp.y) v[g][e] = 0.f;
                        }
                    }
                    uint32_t p[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) p[e] = ptx::pack16<F16>(v[g][2 * e], v[g][2 * e + 1]);
                    ptx::tmem_st16(lanes + half * 64 + g * 16, p);
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) v[g][e] = ptx::ex2_mufu(fmaf(v[g][e], c, -my_lse2));
                    if (masked) {
                        const int lo = span.x - t * T - c0;
                        const uint32_t len = (uint32_t)(span.y - span.x);
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if ((uint32_t)(e - lo) >= len) v[g][e] = 0.f;
                    }
                }
                if (GEN) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) v[g][e] *= bend[e];
                }
            }
            if (key_side) {
                ptx::tmem_wait_st();
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(pfull);
            }
            const int buf = key_side ? 0 : i & 1;
            const uint32_t dp_addr = lanes + 128 + buf * 128 + half * 64;
            if (!ptx::wait_bounded(&dpfull[buf], key_side ? i & 1 : (i >> 1) & 1, abort, status, WAIT_NS)) { ok = false; break; }
            ptx::tc_fence_after();
            uint32_t y[2][32];
            ptx::tmem_ld32(dp_addr, y[0]);
            ptx::tmem_ld32(dp_addr + 32, y[1]);
            ptx::tmem_wait_ld(y[0]);
            ptx::tmem_wait_ld(y[1]);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                float(&d)[32] = reinterpret_cast<float(&)[32]>(y[g]);
                if (key_side) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        const float4 d4 = *(const float4*)(vec + T + g * 32 + e);
                        d[e] = v[g][e] * (d[e] - d4.x);
                        d[e + 1] = v[g][e + 1] * (d[e + 1] - d4.y);
                        d[e + 2] = v[g][e + 2] * (d[e + 2] - d4.z);
                        d[e + 3] = v[g][e + 3] * (d[e + 3] - d4.w);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) d[e] = v[g][e] * (d[e] - my_delta);
                }
                if (masked) {   // zero, whatever dP of a masked pair holds
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (v[g][e] == 0.f) d[e] = 0.f;
                }
                uint32_t p[16];
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    p[e] = F16 ? ptx::pack16<F16>(d[2 * e] * up_p, d[2 * e + 1] * up_p) : ptx::pack16<F16>(d[2 * e], d[2 * e + 1]);
                ptx::tmem_st16(dp_addr + g * 16, p);
            }
            ptx::tmem_wait_st();
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&dsfull[buf]);
        }
        bool have = items > 0 && ok;
        if (have) have = ptx::wait_bounded(accfull, 0, abort, status, WAIT_NS);
        ptx::tc_fence_after();
        const float back = a.scale / up;
        if (key_side) {
            const bool live = row < a.k_len;
            if (half == 0) {
                uint8_t* out = (uint8_t*)a.dv.p + 2 * (b * a.dv.sb + (int64_t)row * a.dv.ss + h * a.dv.sh);
                store_cols<DP, F16>(lanes + 256, p_back, out, 0, a.dim, live, have);
                if (have && live && *(volatile int*)&ms.poison) {
                    for (int i = 0; i < items; ++i) {
                        if (!partial(i)) continue;
                        const int q1 = min((tile_of(i) + 1) * T, a.q_len);
                        for (int q = tile_of(i) * T; q < q1; ++q) {
                            const int2 sp = row_span(a, b, q, n);
                            if (row < sp.x || row >= sp.y) continue;
                            const uint16_t* g = (const uint16_t*)a.d_o.p + b * a.d_o.sb + (int64_t)q * a.d_o.ss + head_of(i) * a.d_o.sh;
                            constexpr uint16_t EXP = F16 ? 0x7c00 : 0x7f80;
                            for (int c = 0; c < a.dim; ++c)
                                if ((g[c] & EXP) == EXP) {
                                    uint16_t* o = (uint16_t*)out + c;
                                    const uint32_t pr = (uint32_t)*o | ((uint32_t)g[c] << 16);
                                    const float2 f = pair_of<F16>(pr);
                                    *o = (uint16_t)ptx::pack16<F16>(f.x + f.y, 0.f);
                                }
                        }
                    }
                }
            } else {
                uint8_t* out = (uint8_t*)a.dk.p + 2 * (b * a.dk.sb + (int64_t)row * a.dk.ss + h * a.dk.sh);
                store_cols<DP, F16>(lanes + 384, back, out, 0, a.dim, live, have);
            }
        } else {
            uint8_t* out = (uint8_t*)a.dq.p + 2 * (b * a.dq.sb + (int64_t)row * a.dq.ss + h * a.dq.sh);
            store_cols<DP / 2, F16>(lanes + 384 + half * (DP / 2), back, out, half * (DP / 2), a.dim, row < a.q_len, have);
        }
        ptx::tc_fence_before();
    }
    __syncthreads();
    if (warp == MMA_WARP) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, TMEM_COLS);
    }
}

template <int DP, bool F16, bool GEN>
int launch(const Prob& a, const Work& w, cudaStream_t s) {
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
    args.n_kt = (int)cdiv(a.k_len, T);
    const int64_t keys = (int64_t)args.n_kt * a.kv_heads * a.batch;
    const int64_t blocks = keys + (int64_t)args.n_qt * a.heads * a.batch;
    FD_CHECK_ARG(blocks <= 0x7fffffff && cdiv(a.q_len, T) + cdiv(a.k_len, T) <= 0x7fffffff, "fd_attention: too many tiles");
    args.n_key = (int)keys;
    const int v_blocks = F16 ? args.n_kt : 0;
    if (F16) FD_CUDA_TRY(cudaMemsetAsync(w.top, 0, 2 * sizeof(unsigned), s));
    prep_kernel<F16><<<dim3(args.n_qt + v_blocks, a.heads, a.batch), 256, 0, s>>>(a, w, args.n_qt);
    FD_CUDA_TRY(cudaGetLastError());
    auto fn = gradient_kernel<DP, F16, GEN>;
    FD_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<DP>::SMEM));
    fn<<<(unsigned)blocks, NTHREADS, Cfg<DP>::SMEM, s>>>(q, k, v, g, args, status);
    FD_CUDA_TRY(cudaGetLastError());
    return FD_OK;
}

template <int DP>
int by_type(const Prob& a, int dtype, const Work& w, cudaStream_t s) {
    const bool gen = a.cap > 0.f || a.slopes;
    if (dtype == FD_DTYPE_F16) return gen ? launch<DP, true, true>(a, w, s) : launch<DP, true, false>(a, w, s);
    return gen ? launch<DP, false, true>(a, w, s) : launch<DP, false, false>(a, w, s);
}

}  // namespace bwd

size_t tc_backward_bytes(int64_t batch, int64_t heads, int64_t q_len) {
    return bwd::work_layout(nullptr, nullptr, batch * heads, batch, cdiv(q_len, T));
}

int tc_backward(const Prob& a, int dtype, void* workspace, cudaStream_t s) {
    bwd::Work w;
    bwd::work_layout(&w, workspace, (int64_t)a.batch * a.heads, a.batch, cdiv(a.q_len, T));
    return a.dim <= 64 ? bwd::by_type<64>(a, dtype, w, s) : bwd::by_type<128>(a, dtype, w, s);
}

}  // namespace attn
}  // namespace fd
