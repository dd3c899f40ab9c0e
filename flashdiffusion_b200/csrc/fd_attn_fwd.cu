// Forward softmax attention on the tensor cores.
//
//   S = Q K^T           tcgen05.mma, both operands from shared memory, fp32 in TMEM
//   P = 2^(x - m)       x the base-2 score, m a running bound of the row (below)
//   O += P V            P 16-bit in TMEM over S's columns, V as it lies (MN-major)
//   o = O / l, lse = ln2 (m + log2 l),   l the fp32 sum of the unrounded P
//
// One pass over the keys.  m is raised only when a row's new maximum exceeds it
// by more than 8 (a factor 256): P then stays below 2^8 (fp16: times 2^7, so that
// weights down to 2^-21 of the largest stay normal and the largest fit), and the O columns of a row are rescaled a few times per
// row instead of at every tile, by the softmax threads themselves.
//
// CTA = 256 query rows of one head (two subtiles of 128) against a stream of
// 128-key tiles; both subtiles use a K/V tile while it is in shared memory, and
// the tensor core works on one subtile's products while the other's
// exponentials are made.  Five warpgroups: four for the softmax, one with a TMA
// producer, an MMA issuer and a guard that looks at the V tiles of which some row
// sees only a part (see `guard`).  Two softmax threads share a row, 64 columns
// each, and exchange their maxima through shared memory: with one thread a row
// (8 warps) the SM issued an instruction in 0.35 of its cycles, two warps a
// scheduler being too few for the latencies of TMEM, MUFU and FMA chains.  Heads
// of 129 to 256 coordinates leave room for one subtile.
//
// Measured, bf16: 2 x 4096 rows of 16 / 4 heads of 128 298 us, 922 TFLOP/s, causal
// 164 us, 840; 16384 causal rows of 8 / 2 heads 504 us, 1091, with a cap and a
// window of 4096 (fp16) 351 us, 685; 8192 causal rows of 8 / 4 heads of 256 328 us,
// 839.  No pipe is full (2 x 4096 causal rows: tensor 41 %, issue slots 46 %, MUFU
// 32 %): a subtile's next scores wait for its own P V and that for its
// exponentials, and two subtiles hide only a part of the chain.
#include <algorithm>

#include "fd_attn_tc.cuh"

namespace fd {
namespace attn {
namespace fwd {

constexpr int TMA_WARP = 16, MMA_WARP = 17, GUARD_WARP = 18;
constexpr int NTHREADS = 20 * 32;
// Registers: 96 a thread at launch (61440 in all); the softmax threads hold 64 scores each and take 104, the others
// give up what they do not use: 512 * 104 + 128 * 56 = 60416.
constexpr int SOFTMAX_REGS = 104, OTHER_REGS = 56;
constexpr uint32_t TMEM_COLS = 512;

template <int DP>
struct Cfg {
    static constexpr int BOXES = DP / 64;
    static constexpr uint32_t TILE = BOXES * BOX_BYTES;
    // D = 256 fills TMEM (O) and shared memory (K and V take turns in a slot each) with one subtile; the warps of
    // the other then have nothing to do
    static constexpr int SUBTILES = DP <= 128 ? 2 : 1;
    static constexpr uint32_t Q_BYTES = SUBTILES * TILE;
    static constexpr int SLOTS = DP == 64 ? 8 : DP == 128 ? 5 : 2;
    static constexpr uint32_t BAR_OFF = Q_BYTES + SLOTS * TILE;
    // qfull, full[SLOTS], empty[SLOTS], sfull[2], pfull[2], ofull[2], toguard, guarded, rest
    static constexpr int NBARS = 1 + 2 * SLOTS + 6 + 3;
    static constexpr uint32_t MISC_OFF = BAR_OFF + NBARS * 8;
    // maxima and, at the end, sums of a row's two threads: [2 subtiles][2 halves][128]
    static constexpr uint32_t MEET_OFF = (MISC_OFF + 64 + 15) / 16 * 16;
    static constexpr uint32_t SMEM = MEET_OFF + 4 * T * 4;            // 1024-byte aligned: nothing lies before it
    static constexpr uint32_t O_COL = 256;
    static_assert(SMEM <= 227 * 1024, "shared memory budget");
    static_assert(O_COL + SUBTILES * DP <= TMEM_COLS, "TMEM budget");
};

struct Misc {
    uint32_t tmem;
    int abort;
    int poison;          // a partly visible V tile held a NaN or an infinity
    int lo[2], hi[2];    // keys seen by any row of the subtile: [lo, hi)
    int flo[2], fhi[2];  // keys seen by every row: [flo, fhi)
};

// Keys cut into parts (parts > 1): each CTA leaves its normalised rows and their lse2 for join_kernel.
struct Split {
    int parts;
    float* o;        // [part][batch][query][head][dim]
    float* lse2;     // [part][batch][query][head], base 2
};

template <int DP, bool F16, bool GEN>
__global__ void __launch_bounds__(NTHREADS, 1)
forward_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
               const __grid_constant__ CUtensorMap tmv, const __grid_constant__ Prob a, const __grid_constant__ Split sp,
               int n_qt, int* __restrict__ status) {
    using C = Cfg<DP>;
    constexpr float P_SHIFT = F16 ? 7.f : 0.f;
    extern __shared__ __align__(1024) uint8_t base[];
    if (ptx::smem_u32(base) & 1023) {   // the swizzled tiles need it, and there is no room to round up
        if (threadIdx.x == 0) atomicExch(status, FD_ERR_UNSUPPORTED);
        return;
    }
    uint8_t* sQ = base;
    uint8_t* ring = base + C::Q_BYTES;
    uint64_t* qfull = (uint64_t*)(base + C::BAR_OFF);
    uint64_t* full = qfull + 1;
    uint64_t* empty = full + C::SLOTS;
    uint64_t* sfull = empty + C::SLOTS;
    uint64_t* pfull = sfull + 2;
    uint64_t* ofull = pfull + 2;
    uint64_t* toguard = ofull + 2;
    uint64_t* guarded = toguard + 1;
    uint64_t* rest = guarded + 1;
    Misc& ms = *(Misc*)(base + C::MISC_OFF);
    volatile int* abort = &ms.abort;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // later query tiles see more keys under a causal mask: they start first
    const int nh = a.heads * a.batch;
    const int qt = n_qt - 1 - blockIdx.x / (nh * sp.parts);
    const int part = blockIdx.x / nh % sp.parts, bh = blockIdx.x % nh;
    const int b = bh / a.heads, h = bh - b * a.heads, hk = h / a.group;
    const int q0 = qt * C::SUBTILES * T;
    const int n = keys_of(a, b);

    if (threadIdx.x == 0) {
        ptx::mbar_init(qfull, 1);
        for (int i = 0; i < C::SLOTS; ++i) {
            ptx::mbar_init(&full[i], 1);
            ptx::mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(&sfull[i], 1);
            ptx::mbar_init(&pfull[i], 8);
            ptx::mbar_init(&ofull[i], 1);
            ms.lo[i] = 0x7fffffff;
            ms.hi[i] = 0;
            ms.flo[i] = 0;
            ms.fhi[i] = 0x7fffffff;
        }
        ptx::mbar_init(toguard, 1);
        ptx::mbar_init(guarded, 1);
        ptx::mbar_init(rest, 1);
        ms.abort = 0;
        ms.poison = 0;
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
    }
    __syncthreads();

    if (warp == TMA_WARP && lane == 0) {   // on their way before the spans are known
        ptx::mbar_expect_tx(qfull, C::Q_BYTES);
        for (int s = 0; s < C::SUBTILES; ++s)
            for (int c = 0; c < C::BOXES; ++c)
                ptx::tma_load_4d(sQ + s * C::TILE + c * BOX_BYTES, &tmq, qfull, c * 64, q0 + s * T, h, b);
    }
    __syncwarp();
    const int sub = warp >> 3, half = (warp >> 2) & 1;   // softmax warps: query subtile, columns 64 half ..
    const int lrow = threadIdx.x & 127, row = q0 + sub * T + lrow;
    int2 span = make_int2(0, 0);
    if (sub < 2) {
        const bool real = sub < C::SUBTILES && row < a.q_len;
        if (real) span = row_span(a, b, row, n);
        const bool some = span.y > span.x;
        const int lo = warp_min(some ? span.x : 0x7fffffff), hi = warp_max(some ? span.y : 0);
        // rows behind the last query are never stored: they need no mask
        const int flo = warp_max(!real ? 0 : some ? span.x : 0x7fffffff);
        const int fhi = warp_min(!real ? 0x7fffffff : some ? span.y : 0);
        if (!real) span = make_int2(0, 0x7fffffff);
        if (lane == 0) {
            atomicMin(&ms.lo[sub], lo);
            atomicMax(&ms.hi[sub], hi);
            atomicMax(&ms.flo[sub], flo);
            atomicMin(&ms.fhi[sub], fhi);
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = ms.tmem;
    int ta[2], tb[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const bool some = ms.hi[s] > ms.lo[s];
        ta[s] = some ? ms.lo[s] / T : 0;
        tb[s] = some ? (ms.hi[s] + T - 1) / T : 0;
    }
    // tiles of either subtile; an empty subtile takes no part
    int t0 = tb[0] == 0 ? ta[1] : tb[1] == 0 ? ta[0] : min(ta[0], ta[1]);
    int t1 = max(tb[0], tb[1]);
    if (sp.parts > 1) {
        const int n = t1 - t0, from = t0 + n * part / sp.parts, to = t0 + n * (part + 1) / sp.parts;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            ta[s] = max(ta[s], from);
            tb[s] = min(tb[s], to);
            if (ta[s] >= tb[s]) ta[s] = tb[s] = 0;
        }
        t0 = tb[0] == 0 ? ta[1] : tb[1] == 0 ? ta[0] : min(ta[0], ta[1]);
        t1 = max(tb[0], tb[1]);
    }
    auto active = [&](int s, int j) { return j >= ta[s] && j < tb[s]; };
    // some row of an active subtile sees only a part of tile j
    auto partial = [&](int j) {
        bool p = false;
        for (int s = 0; s < 2; ++s) p = p || (active(s, j) && (j * T < ms.flo[s] || (j + 1) * T > ms.fhi[s]));
        return p;
    };

    if (sub == 2) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
    if (warp == TMA_WARP) {
        if (lane == 0 && t1 > t0) {
            const int items = 2 * (t1 - t0);
            int i = 0;
            for (; i < items; ++i) {
                const int slot = i % C::SLOTS, round = i / C::SLOTS;
                if (!ptx::wait_bounded(&empty[slot], (round & 1) ^ 1, abort, status, WAIT_NS)) break;
                ptx::mbar_expect_tx(&full[slot], C::TILE);
                for (int c = 0; c < C::BOXES; ++c)
                    ptx::tma_load_4d(ring + slot * C::TILE + c * BOX_BYTES, (i & 1) ? &tmv : &tmk, &full[slot], c * 64,
                                     (t0 + i / 2) * T, hk, b);
            }
            if (i < items) {   // gave up: the copies in flight still write into this block's memory
                wait_landed(qfull, 0);
                for (int z = max(0, i - C::SLOTS); z < i; ++z) wait_landed(&full[z % C::SLOTS], (z / C::SLOTS) & 1);
            }
        } else if (lane == 0) {
            wait_landed(qfull, 0);   // nothing to do, but the copy is still under way
        }
    } else if (warp == MMA_WARP) {
        if (t1 > t0) {
            const uint32_t lead = elect_lane();
            const int ks_qk = (a.dim + 15) / 16;
            const uint32_t id_qk = ptx::idesc_f32acc(T, T, F16);
            const uint32_t id_pv = ptx::idesc_f32acc(T, ks_qk * 16, F16) | ptx::IDESC_B_MN;
            const uint32_t q_base = ptx::smem_u32(sQ), r_base = ptx::smem_u32(ring);
            auto slot_of = [&](int item) { return item % C::SLOTS; };
            auto wait_full = [&](int item) {
                return wait_warp(&full[slot_of(item)], (item / C::SLOTS) & 1, abort, status);
            };
            auto issue_qk = [&](int s, int item) {
                ptx::tc_fence_after();
                product_rows<DP>(lead, tmem + s * T, q_base + s * C::TILE, r_base + slot_of(item) * C::TILE, id_qk, ks_qk);
                mma_commit(lead, &sfull[s]);
            };
            bool ok = wait_warp(qfull, 0, abort, status) && wait_full(0);
            if (ok) {
                for (int s = 0; s < 2; ++s)
                    if (active(s, t0)) issue_qk(s, 0);
                mma_commit(lead, &empty[0]);
            }
            uint32_t np[2] = {0, 0}, ng = 0;
            for (int j = t0; j < t1 && ok; ++j) {
                const int iv = 2 * (j - t0) + 1, ik = iv + 1;
                ok = wait_full(iv) && (j + 1 == t1 || wait_full(ik));
                bool look = ok && partial(j);
                if (look && lead) ptx::mbar_arrive(toguard);
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    if (!ok) break;
                    if (active(s, j)) {
                        ok = wait_warp(&pfull[s], np[s] & 1, abort, status);
                        if (!ok) break;
                        ++np[s];
                        if (look) {
                            ok = wait_warp(guarded, ng & 1, abort, status);
                            if (!ok) break;
                            ++ng;
                            look = false;
                        }
                        ptx::tc_fence_after();
                        product_sum<1, 32>(lead, tmem + C::O_COL + s * DP, tmem + s * T, r_base + slot_of(iv) * C::TILE, id_pv,
                                        j > ta[s]);
                        if (j + 1 == tb[s]) mma_commit(lead, &ofull[s]);
                    }
                    if (j + 1 < t1 && active(s, j + 1)) issue_qk(s, ik);
                }
                mma_commit(lead, &empty[slot_of(iv)]);
                if (j + 1 < t1) mma_commit(lead, &empty[slot_of(ik)]);
            }
            if (!ok) {   // gave up: products in flight still read this block's memory and write its columns
                mma_commit(lead, rest);
                wait_landed(rest, 0);
            }
        }
    } else if (warp == GUARD_WARP) {
        // ---- guard: where some row sees only a part of a tile, its P is zero in
        //      the masked places, and 0 times a NaN or an infinity in V would reach
        //      the row all the same.  Such elements become zeros in shared memory
        //      before the product; the rows that do see them get them back at the
        //      end (`poison`).  Partly visible tiles are the few at the ends of the
        //      rows' spans, and the scan runs while their scores are made.
        uint32_t ng = 0;
        for (int j = t0; j < t1; ++j) {
            if (!partial(j)) continue;
            const int item = 2 * (j - t0) + 1, slot = item % C::SLOTS;
            // the issuer says when the tile is there (and holds it until the guard answers): waiting for
            // `full` alone, rounds ahead of the ring, would match an older phase of the same parity
            if (!ptx::wait_bounded(toguard, ng & 1, abort, status, WAIT_NS)) break;
            ++ng;
            if (!ptx::wait_bounded(&full[slot], (item / C::SLOTS) & 1, abort, status, WAIT_NS)) break;
            if (clear_bad<F16>(ring + slot * C::TILE, C::TILE, lane) && lane == 0) ms.poison = 1;
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(guarded);
        }
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFTMAX_REGS));
        // ---- softmax: two threads a query row
        const uint32_t s_addr = tmem + ((uint32_t)(warp & 3) << 21) + sub * T + half * 64;
        const uint32_t o_addr = tmem + ((uint32_t)(warp & 3) << 21) + C::O_COL + sub * DP + half * (DP / 2);
        float* meet = (float*)(base + C::MEET_OFF) + (sub * 2 + half) * T + lrow;
        const float* other = (const float*)(base + C::MEET_OFF) + (sub * 2 + (half ^ 1)) * T + lrow;
        // the threads of a subtile meet; true if `good` is true in all of them, so that they leave the loop together
        auto both_here = [&](bool good) {
            uint32_t all;
            asm volatile(
                "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.cta.red.and.pred q, %2, 256, p;\n\t"
                "selp.u32 %0, 1, 0, q;\n\t}" : "=r"(all) : "r"((uint32_t)good), "r"(1 + sub) : "memory");
            return all != 0;
        };
        const Score sc(a);
        const float slope2 = GEN && a.slopes ? a.slopes[h] * LOG2E : 0.f;
        // plain scores stay raw until the exponential's own multiply-add
        const float c = GEN ? 1.f : ptx::lo2(sc.c);
        const float room = GEN ? 8.f : 8.f / c;
        const int pos = n - a.q_len + row;
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        int it = 0;
        for (int j = ta[sub]; j < tb[sub]; ++j, ++it) {
            ok = ptx::wait_bounded(&sfull[sub], it & 1, abort, status, WAIT_NS);
            ptx::tc_fence_after();
            uint64_t x[2][16];
            {
                uint32_t r[2][32];
                ptx::tmem_ld32(s_addr, r[0]);
                ptx::tmem_ld32(s_addr + 32, r[1]);
                ptx::tmem_wait_ld(r[0]);
                ptx::tmem_wait_ld(r[1]);
                pairs32(r[0], x[0]);
                pairs32(r[1], x[1]);
            }
            const int k0 = j * T + half * 64;
            const int lo = span.x - k0, len = span.y - span.x;
            const bool masked = !__all_sync(~0u, lo <= 0 && (int64_t)lo + len >= 64);
            // A cap alone, well inside its range: it is monotone, so the largest score comes from the largest (or
            // smallest) raw product, and the polynomial goes straight into the exponential's argument.
            bool direct = GEN && sc.capped && slope2 == 0.f && !masked;
            // a NaN among the visible scores becomes the row's m, and with it the whole row NaN
            float mt;
            if (direct) {
                float hi[2], bo[2];
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    hi[g] = max_nan(ptx::lo2(x[g][0]), ptx::hi2(x[g][0]));
                    bo[g] = fminf(ptx::lo2(x[g][0]), ptx::hi2(x[g][0]));
#pragma unroll
                    for (int i = 1; i < 16; ++i) {
                        hi[g] = max_nan(hi[g], max_nan(ptx::lo2(x[g][i]), ptx::hi2(x[g][i])));
                        bo[g] = fminf(bo[g], fminf(ptx::lo2(x[g][i]), ptx::hi2(x[g][i])));
                    }
                }
                mt = max_nan(hi[0], hi[1]);
                const float mb = fminf(bo[0], bo[1]);
                direct = __all_sync(~0u, mt <= sc.limit && mb >= -sc.limit);
                if (direct) {
                    const float end = ptx::lo2(sc.c) > 0.f ? mt : mb;
                    mt = end * ptx::lo2(sc.ratio(ptx::both2(end)));
                }
            }
            if (!direct) {
                if (GEN) {
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        if (sc.capped) {
                            cap32(x[g], sc);
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; ++i) x[g][i] = ptx::mul2(x[g][i], sc.c);
                        }
                        if (slope2 != 0.f)
                            add_bias(x[g], slope2, (float)(pos - k0 - g * 32), -1.f,
                                     side_of(a, n - a.q_len + q0 + sub * T, j * T));
                    }
                }
                if (masked) {
#pragma unroll
                    for (int g = 0; g < 2; ++g) mask32(x[g], lo - g * 32, (uint32_t)len, -INFINITY);
                }
                float top[4];
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    top[g] = max_nan(ptx::lo2(x[g / 2][g % 2 * 8]), ptx::hi2(x[g / 2][g % 2 * 8]));
#pragma unroll
                    for (int i = 1; i < 8; ++i)
                        top[g] = max_nan(top[g], max_nan(ptx::lo2(x[g / 2][g % 2 * 8 + i]), ptx::hi2(x[g / 2][g % 2 * 8 + i])));
                }
                mt = max_nan(max_nan(top[0], top[1]), max_nan(top[2], top[3]));
            }
            // the next tile's scores come only after every thread here has read this and handed over its P
            meet[0] = mt;
            ok = both_here(ok);
            if (!ok) break;
            mt = max_nan(mt, other[0]);
            const bool raise = !(mt <= m + room);
            if (__any_sync(~0u, raise)) {
                const float mn = raise ? mt : m;
                const float fix = m == -INFINITY ? 0.f : ptx::ex2_mufu((m - mn) * c);
                m = mn;
                l *= fix;
                if (it > 0) {
                    // S's commit also covered the previous P V, so O is at rest; each thread takes half its columns
#pragma unroll 1
                    for (int g = 0; g < DP / 2; g += 16) {
                        uint32_t o[16];
                        ptx::tmem_ld16(o_addr + g, o);
                        ptx::tmem_wait_ld16(o);
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * fix);
                        ptx::tmem_st16(o_addr + g, o);
                    }
                }
            }
            const uint64_t off = ptx::both2(m == -INFINITY ? 0.f : fmaf(-m, c, P_SHIFT));
            const uint64_t c2 = ptx::both2(c);
            uint64_t part[2] = {0, 0};
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                if (direct) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[g][i] = ptx::fma2(sc.ratio(x[g][i]), x[g][i], off);
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[g][i] = GEN ? ptx::add2(x[g][i], off) : ptx::fma2(x[g][i], c2, off);
                }
                // masked places must be zeros; a cap keeps the FMA pipe busy enough
                if (masked || direct) exp32<0>(x[g]);
                else exp32<1>(x[g]);
#pragma unroll
                for (int i = 0; i < 16; ++i) part[i & 1] = ptx::add2(part[i & 1], x[g][i]);
                uint32_t p[16];
                round32<F16>(x[g], p);
                ptx::tmem_st16(s_addr + g * 32, p);
            }
            part[0] = ptx::add2(part[0], part[1]);
            l += ptx::lo2(part[0]) + ptx::hi2(part[0]);
            ptx::tmem_wait_st();
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&pfull[sub]);
        }
        if (it > 0 && ok) ok = ptx::wait_bounded(&ofull[sub], 0, abort, status, WAIT_NS);
        ptx::tc_fence_after();
        both_here(ok);
        meet[0] = l;
        both_here(ok);
        l += other[0];
        const bool real = sub < C::SUBTILES && row < a.q_len;
        if (m == -INFINITY) l = 0.f;               // exponentials on the FMA pipe end at 2^-125, above zero
        const bool sees = real && span.y > span.x;
        if (sp.parts == 1) l = sum_or_nan(l, sees);
        if (!ok) l = not_a_number();               // gave up: NaN, not numbers that could pass for the rows
        const float inv = l == 0.f ? 0.f : 1.f / l;
        uint8_t* out = (uint8_t*)a.o.p + 2 * (b * a.o.sb + (int64_t)row * a.o.ss + h * a.o.sh);
        int8_t* low = a.o_low ? a.o_low + (((int64_t)b * a.q_len + row) * a.heads + h) * a.dim : nullptr;
        const bool poison = it > 0 && *(volatile int*)&ms.poison;
#pragma unroll 1
        for (int g = 0; g < DP / 2; g += 16) {
            const int c0 = half * (DP / 2) + g;
            uint32_t o[16];
            if (it > 0 && ok) {
                ptx::tmem_ld16(o_addr + g, o);
                ptx::tmem_wait_ld16(o);
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = 0;
            }
            float(&f)[16] = reinterpret_cast<float(&)[16]>(o);
#pragma unroll
            for (int i = 0; i < 16; ++i) f[i] = l == 0.f ? 0.f : f[i] * inv;
            if (poison && real && l != 0.f) {
                // put back what the guard took out, for the keys that this row sees
                for (int j = ta[sub]; j < tb[sub]; ++j) {
                    if (!partial(j)) continue;
                    for (int k = max(span.x, j * T); k < min(span.y, (j + 1) * T); ++k) {
                        const uint16_t* vr = (const uint16_t*)a.v.p + b * a.v.sb + (int64_t)k * a.v.ss + hk * a.v.sh + c0;
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            if (c0 + i >= a.dim) continue;
                            const uint16_t w = vr[i];
                            constexpr uint16_t EXP = F16 ? 0x7c00 : 0x7f80;
                            if ((w & EXP) == EXP) f[i] += F16 ? __half2float(__ushort_as_half(w))
                                                              : __bfloat162float(__ushort_as_bfloat16(w));
                        }
                    }
                }
            }
            if (real && sp.parts > 1) {
                float* to = sp.o + ((((int64_t)part * a.batch + b) * a.q_len + row) * a.heads + h) * a.dim + c0;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (c0 + i * 4 < a.dim) *(float4*)(to + 4 * i) = make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
            } else if (real) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (c0 + i * 8 >= a.dim) continue;
                    store8<F16>(out + 2 * (c0 + i * 8), low ? low + c0 + i * 8 : nullptr, f + 8 * i);
                }
            }
        }
        if (half == 0 && real) {
            const float lse2 = l == 0.f ? (sees ? LOWEST : -INFINITY) : m * c + (log2f(l) - P_SHIFT);
            if (sp.parts > 1) sp.lse2[(((int64_t)part * a.batch + b) * a.q_len + row) * a.heads + h] = lse2;
            else if (a.lse) a.lse[((int64_t)b * a.heads + h) * a.q_len + row] = lse2 * LN2;
        }
        ptx::tc_fence_before();
    }
    __syncthreads();
    if (warp == MMA_WARP) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, TMEM_COLS);
    }
}

// The parts of a row, in order: o = sum_p 2^(lse2_p - lse2) o_p.  Thread: eight coordinates.
template <bool F16>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Prob a, const __grid_constant__ Split sp) {
    const int pieces = a.dim / 8;
    const int64_t rows = (int64_t)a.batch * a.q_len * a.heads, x = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (x >= rows * pieces) return;
    const int64_t r = x / pieces;
    const int d = (int)(x - r * pieces) * 8;
    float m = -INFINITY;
    for (int p = 0; p < sp.parts; ++p) m = fmaxf(m, sp.lse2[p * rows + r]);
    const float base = m == -INFINITY ? 0.f : m;
    float sum = m == LOWEST ? not_a_number() : 0.f, acc[8] = {};
#pragma unroll 4
    for (int p = 0; p < sp.parts; ++p) {
        const float w = exp2f(sp.lse2[p * rows + r] - base);
        const float* o = sp.o + (p * rows + r) * a.dim + d;
        const float4 u = *(const float4*)o, v = *(const float4*)(o + 4);
        const float f[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
        sum += w;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = fmaf(w, f[e], acc[e]);
    }
    const int64_t t = r / a.heads, b = t / a.q_len, row = t - b * a.q_len;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= inv;
    const int h = (int)(r - t * a.heads);
    store8<F16>((uint16_t*)a.o.p + b * a.o.sb + row * a.o.ss + h * a.o.sh + d, a.o_low ? a.o_low + r * a.dim + d : nullptr, acc);
    if (d == 0 && a.lse)
        a.lse[(b * a.heads + h) * a.q_len + row] = sum == 0.f ? -INFINITY : (base + log2f(sum)) * LN2;
}

template <int DP, bool F16, bool GEN>
int launch(const Prob& a, const Split& sp, cudaStream_t s) {
    CUtensorMap q, k, v;
    FD_TRY(make_head_map(&q, a.q, a.q_len, a.heads, a.batch, a.dim, F16));
    FD_TRY(make_head_map(&k, a.k, a.k_len, a.kv_heads, a.batch, a.dim, F16));
    FD_TRY(make_head_map(&v, a.v, a.k_len, a.kv_heads, a.batch, a.dim, F16));
    int* status = nullptr;
    FD_TRY(status_word(&status));
    FD_TRY((allow_smem<forward_kernel<DP, F16, GEN>>(Cfg<DP>::SMEM)));
    const int n_qt = (int)cdiv(a.q_len, Cfg<DP>::SUBTILES * T);
    const int64_t blocks = (int64_t)n_qt * a.heads * a.batch * sp.parts;
    FD_CHECK_ARG(blocks <= 0x7fffffff, "fd_attention: too many query tiles");
    forward_kernel<DP, F16, GEN><<<(unsigned)blocks, NTHREADS, Cfg<DP>::SMEM, s>>>(q, k, v, a, sp, n_qt, status);
    FD_CUDA_TRY(cudaGetLastError());
    if (sp.parts > 1) {
        const int64_t threads = (int64_t)a.batch * a.q_len * a.heads * (a.dim / 8);
        join_kernel<F16><<<(unsigned)cdiv(threads, 256), 256, 0, s>>>(a, sp);
        FD_CUDA_TRY(cudaGetLastError());
    }
    return FD_OK;
}

template <int DP>
int by_type(const Prob& a, int dtype, const Split& sp, cudaStream_t s) {
    // the plain kernel keeps raw scores and needs them to grow with the products
    const bool gen = a.cap > 0.f || a.slopes || !(a.scale > 0.f);
    if (dtype == FD_DTYPE_F16) return gen ? launch<DP, true, true>(a, sp, s) : launch<DP, true, false>(a, sp, s);
    return gen ? launch<DP, false, true>(a, sp, s) : launch<DP, false, false>(a, sp, s);
}

}  // namespace fwd

int make_head_map(CUtensorMap* map, const View& v, int64_t rows, int heads, int batch, int dim, bool f16) {
    EncodeTiledFn enc;
    FD_TRY(get_encode(&enc));
    const cuuint64_t dims[4] = {(cuuint64_t)dim, (cuuint64_t)rows, (cuuint64_t)heads, (cuuint64_t)batch};
    // an extent of 1 never takes its stride; the map still wants a multiple of 16 bytes
    auto bytes = [&](int64_t stride, int64_t extent) { return (cuuint64_t)(extent > 1 ? stride * 2 : 16 * cdiv(dim, 8)); };
    const cuuint64_t strides[3] = {bytes(v.ss, rows), bytes(v.sh, heads), bytes(v.sb, batch)};
    const cuuint32_t box[4] = {64, (cuuint32_t)T, 1, 1}, one[4] = {1, 1, 1, 1};
    const CUresult r = enc(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, v.p, dims,
                           strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(FD_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return FD_OK;
}

bool tc_applies(const Prob& a, int dtype, bool backward) {
    if (dtype != FD_DTYPE_F16 && dtype != FD_DTYPE_BF16) return false;
    if (a.dim % 8 || a.dim > (backward ? 128 : 256) || a.q_len == 0 || a.k_len == 0) return false;
    const int64_t qe[3] = {a.batch, a.q_len, a.heads}, ke[3] = {a.batch, a.k_len, a.kv_heads};
    if (!tma_view(a.q, qe) || !tma_view(a.k, ke) || !tma_view(a.v, ke) || !tma_view(a.o, qe)) return false;
    if (!backward) return true;
    return tma_view(a.d_o, qe) && tma_view(a.dq, qe) && tma_view(a.dk, ke) && tma_view(a.dv, ke);
}

// Parts of the key axis for each query tile: as many as the SMs hold, none with fewer than four key tiles, which cost
// about what a part's start, its fp32 rows and the join do (8 / 2 bf16 heads of 128, 512 causal rows: against 16384
// keys 267 us whole, 59 us in 9 parts; against 4096 keys 79 and 35 us; two heads of 128 rows against 640 keys are as
// fast whole, 20.5 us, as in two parts).
static int split_parts(const Prob& a) {
    const int64_t ctas = cdiv(a.q_len, (a.dim <= 128 ? 2 : 1) * T) * a.heads * a.batch;
    const int64_t keys = a.window > 0 ? std::min<int64_t>(a.k_len, (int64_t)a.window + 2 * T) : a.k_len;
    return (int)std::max<int64_t>(1, std::min<int64_t>(num_sms() / std::max<int64_t>(ctas, 1), cdiv(keys, T) / 4));
}

size_t tc_forward_bytes(const Prob& a) {
    const int64_t parts = split_parts(a);
    return parts > 1 ? align256(sizeof(float) * parts * a.batch * a.q_len * a.heads * (a.dim + 1)) : 0;
}

int tc_forward(const Prob& a, int dtype, void* workspace, cudaStream_t s) {
    fwd::Split sp{};
    sp.parts = split_parts(a);
    sp.o = (float*)workspace;
    sp.lse2 = sp.o + (int64_t)sp.parts * a.batch * a.q_len * a.heads * a.dim;
    if (a.dim <= 64) return fwd::by_type<64>(a, dtype, sp, s);
    return a.dim <= 128 ? fwd::by_type<128>(a, dtype, sp, s) : fwd::by_type<256>(a, dtype, sp, s);
}

}  // namespace attn
}  // namespace fd
