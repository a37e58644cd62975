// Gradients of window attention (window_attn_fwd.hip) for f16 / bf16 / float32 on the matrix cores.
//
//     P = exp(scale Q K^T - lse) where seen, else 0          dV = P^T dO
//     dP = dO V^T,  delta = rowsum(dO o O),  dS = P o (dP - delta)
//     dQ = scale dS K,   dK = scale dS^T Q                   dK, dV summed over the query heads that share them
//
// Two kernels and, where keys are split, a third; no atomics, so results do not depend on timing.
//   dQ      workgroup = 128 query rows (4 waves x 32) and the key tiles they see, as in the forward:
//           S^T = K Q^T and dP^T = V dO^T put the query on the lane; dS^T is in place the B operand of
//           dQ^T += K^T dS^T.  Its prologue has the rows of dO at hand, reads those of O and leaves -delta and
//           lse * log2(e) of every row for the second kernel.
//   dK, dV  workgroup = 128 keys (4 waves x 32) of one key/value head and, head after head of its group,
//           the query tiles that see some of them: S = Q K^T and dP = dO V^T put the key on the lane; P and
//           dS are in place the B operands of dV^T += dO^T P and dK^T += Q^T dS.  The sums over the group
//           happen in the accumulators.
//   join    The first `sinks` keys are seen by every later query, the others by about `window`: key blocks
//           with sinks are split over several workgroups by queries, their float32 parts added here in order.
// Beyond 128 columns a workgroup of dK, dV keeps 128 columns of both (the accumulators and the fragments of
// its keys fill the registers) and forms S and dP for each half again.
// Measured, bf16, B 4, 32 heads on 8 of 4096 positions, d 128, window 1024, 4 sinks: dQ 404 us, dK, dV 551, join 5.5; that is
// 895 and 875 TFLOP/s of the three and four products (those of S and dP are formed twice; one kernel for all would have
// to add dQ up with atomics, in no fixed order).  Matrix pipe busy 50 % and 51 % of the cycles, at the clock that the power
// limit leaves on random operands.
// P and dS are rounded to the element type as operands; everything else is float32.  Rows and keys that
// have no visible partner in the workgroup are fetched as zeros, so whatever stands there stays out; what some of its
// rows see and others do not: window_attn_exact.h.
#include "attn_bwd_plan.h"
#include "window_attn_exact.h"

namespace myfa {
namespace {

template <typename T, int D> constexpr int bwd_tile() { return D * (int)sizeof(T) <= 256 ? 64 : 32; }
constexpr int kStatPad = 64;                         // rows of the statistics per head: a multiple of this

// ---------------------------------------------------------------- row statistics
// A lane's query row of dO and O (chunks 2 ks + h): -delta and lse * log2(e) of the row, which the dK, dV kernel reads
// from `st` (two arrays of `rows`, nqp a head).  Every row up to nqp is written; those that see nothing get
// lse = +inf (P = 0) and delta = 0.  All lanes of the wave take part.
struct RowStat { float lse2, ndelta; };
template <typename T, int KS, typename Frag>
__device__ __forceinline__ RowStat row_stat(const Frag (&of)[KS], const T* out_row, const float* lse_at, bool live, int d, int h,
                                            float* st, int64_t rows, int64_t srow, bool store) {
    constexpr int EPC = 16 / (int)sizeof(T);
    typedef T vec __attribute__((ext_vector_type(EPC)));
    float acc = 0.f;
    if (live) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int c = (2 * ks + h) * EPC;
            if (c < d) {
                const vec x = *reinterpret_cast<const vec*>(out_row + c), y = __builtin_bit_cast(vec, of[ks]);
#pragma unroll
                for (int j = 0; j < EPC; ++j) acc += (float)x[j] * (float)y[j];
            }
        }
    }
    acc = half_exchange_sum(acc);
    const RowStat s{live ? *lse_at * kLog2eW : INFINITY, live ? -acc : 0.f};
    if (store && h == 0) {
        st[srow] = s.lse2;
        st[rows + srow] = s.ndelta;
    }
    return s;
}

// ---------------------------------------------------------------- dQ
template <typename T, int D>
__global__ void __launch_bounds__(256, D * sizeof(T) <= 256 ? 2 : 1)
window_bwd_dq_kernel(const T* __restrict__ Qg, const T* __restrict__ Kg, const T* __restrict__ Vg,
                     const T* __restrict__ dOg, const T* __restrict__ Og, const float* __restrict__ LSEg, float* __restrict__ st, T* __restrict__ dQg,
                     WindowShape w, int nqp, int64_t rows, int nqblk) {
    using R = TileReader<T, D>;
    constexpr int BN = bwd_tile<T, D>(), NB = BN / 32, TILE_B = BN * R::RB;
    __shared__ __attribute__((aligned(1024))) char lds[4 * TILE_B];   // K0 K1 V0 V1

    const Ranked at_ = ranked(blockIdx.x, w.B * w.H);
    const int bh = at_.head, q0 = (nqblk - 1 - at_.rank) * 128;      // the last block of a head sees the most keys
    const int b = bh / w.H, head = bh - b * w.H, kvh = head / (w.H / w.Hkv);

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, h = lane >> 5;
    const KeyTiles<BN> kt(w, b, q0, 128);
    const int ntiles = kt.ntiles;

    const int qrow = q0 + 32 * wave + r;
    const int p_own = qrow + kt.shift;
    const bool live = qrow < w.Nq && p_own < kt.len;
    const RowSees sees{p_own - w.window + 1, live ? p_own : -1};
    const int wave_lo = q0 + 32 * wave + kt.shift, wave_hi = min(wave_lo + 32, kt.pz) - 1;

    const T* Kh = Kg + b * w.ks[0] + kvh * w.ks[1];
    const T* Vh = Vg + b * w.vs[0] + kvh * w.vs[1];
    constexpr int EPC = 16 / (int)sizeof(T);
    typename R::frag qf[R::KS], of[R::KS];
    {
        const int row = min(qrow, w.Nq - 1);
        const T* qp = Qg + b * w.qs[0] + head * w.qs[1] + (int64_t)row * w.qs[2];
        const T* op = dOg + ((int64_t)bh * w.Nq + row) * w.d;
#pragma unroll
        for (int ks = 0; ks < R::KS; ++ks) {
            const int c = (2 * ks + h) * EPC;
            qf[ks] = typename R::frag{};
            of[ks] = typename R::frag{};
            if (c < w.d) {
                qf[ks] = *reinterpret_cast<const typename R::frag*>(qp + c);
                of[ks] = *reinterpret_cast<const typename R::frag*>(op + c);
            }
        }
    }
    const int64_t orow = (int64_t)bh * w.Nq + min(qrow, w.Nq - 1);
    const RowStat stat = row_stat<T>(of, Og + orow * w.d, LSEg + orow, live, w.d, h, st, rows, (int64_t)bh * nqp + qrow, qrow < nqp);
    const float lse2 = stat.lse2, ndelta = stat.ndelta;
    const float sl2 = w.scale * kLog2eW;

    const R rd(lane);
    const TileFetch<T, D, BN, 256> kfetch(tid, w.ks[2], w.d), vfetch(tid, w.vs[2], w.d);
    auto fetch = [&](int t, int buf) __attribute__((always_inline)) {
        const int k0 = kt.first_key(t);
        const bool all = kt.all(k0, w.sinks);
        auto keep = [&](int row) { return kt.one(k0 + row, w.sinks); };
        kfetch.fetch(Kh + (int64_t)k0 * w.ks[2], lds + buf * TILE_B, all, keep);
        vfetch.fetch(Vh + (int64_t)k0 * w.vs[2], lds + (2 + buf) * TILE_B, all, keep);
    };

    f32x16 dq[R::DB];
#pragma unroll
    for (int db = 0; db < R::DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) dq[db][i] = 0.f;

    if (ntiles > 0) fetch(0, 0);
    for (int t = 0; t < ntiles; ++t) {
        const int buf = t & 1, k0 = kt.first_key(t);
        tile_ready();
        if (t + 1 < ntiles) fetch(t + 1, buf ^ 1);
        if (k0 > wave_hi || (k0 + BN <= wave_lo - w.window + 1 && k0 >= w.sinks)) continue;
        const char* Kb = lds + buf * TILE_B;
        const char* Vb = lds + (2 + buf) * TILE_B;
        const bool edge = !(k0 + BN - 1 <= wave_lo && wave_lo + 31 < kt.pz && (k0 >= wave_lo + 31 - w.window + 1 || k0 + BN <= w.sinks));
#pragma unroll
        for (int kb = 0; kb < NB; ++kb) {
            f32x16 s, dp;
#pragma unroll
            for (int i = 0; i < 16; ++i) { s[i] = 0.f; dp[i] = ndelta; }
#pragma unroll
            for (int ks = 0; ks < R::KS; ++ks) s = mma_chunk<T>(rd.row(Kb, kb, ks), qf[ks], s);
#pragma unroll
            for (int ks = 0; ks < R::KS; ++ks) dp = mma_chunk<T>(rd.row(Vb, kb, ks), of[ks], dp);
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], sl2, -lse2)) * dp[i];
            if (edge) sees.hide(s, kt, t, k0, k0 + 32 * kb + 4 * h, w.sinks, 0.f);
            rd.add_transposed(Kb, kb, s, dq);
        }
    }

    // (hidden dS are set to 0 behind the product with dP: hidden keys reach dQ, hidden values do not)
    const uint32_t redo = not_finite_rows(dq, live && finite(lse2) && finite(ndelta));
    if (qrow < w.Nq) {
        T* row = dQg + ((int64_t)bh * w.Nq + qrow) * w.d;
        typedef T vec4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int db = 0; db < R::DB; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = 32 * db + 8 * g + 4 * h;
                vec4 x;
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = live ? (T)(dq[db][4 * g + j] * w.scale) : (T)0.f;
                if (c < w.d) *reinterpret_cast<vec4*>(row + c) = x;
            }
    }
    if (redo != 0) {                                        // (window_attn_exact.h)
        const uint32_t cols = hidden_keys<T, D>(kt, w, q0 + 32 * wave + kt.shift, Kh, w.ks[2], lane);
        stored();
        for (uint32_t left = any_lane(cols != 0) ? redo : 0; left != 0; left &= left - 1) {
            const int x = __builtin_ctz(left), i = q0 + 32 * wave + x;
            const int64_t at = ((int64_t)bh * w.Nq + i) * w.d;
            exact_dq_row<T, D>(Qg + b * w.qs[0] + head * w.qs[1] + i * w.qs[2], dOg + at, Kh, Vh, read_lane(lse2, x), read_lane(ndelta, x), dQg + at,
                               w, i + kt.shift, cols, lane);
        }
    }
}

// dQ for 16-bit elements and up to 128 columns.  The tile's 64 keys are two blocks of 32, staggered so that
// the vector part of one block runs in the shadow of the other's matrix products:
//     S0, dP0 | S1, dP1 with dS0 | barrier | dQ += block 0 with dS1 | dQ += block 1
// K in a ring of three, V in one of two: behind the tile's last transposing read (which waits for every
// LDS-DMA load in flight) K(t + 2) and V(t + 2) are requested; the barrier of tile t + 1 finds them complete.
// Two workgroups a CU (160 KiB of LDS between them).
template <typename T, int D>
__global__ void __launch_bounds__(256, 2)
window_bwd_dq16_kernel(const T* __restrict__ Qg, const T* __restrict__ Kg, const T* __restrict__ Vg,
                       const T* __restrict__ dOg, const T* __restrict__ Og, const float* __restrict__ LSEg, float* __restrict__ st, T* __restrict__ dQg,
                       WindowShape w, int nqp, int64_t rows, int nqblk) {
    using M = Mma<T>;
    using R = TileReader<T, D>;
    constexpr int BN = 64, KS = R::KS, DB = R::DB, TILE_B = BN * R::RB, FW = 4;
    __shared__ __attribute__((aligned(1024))) char lds[5 * TILE_B];   // K0 K1 K2 V0 V1

    const Ranked at_ = ranked(blockIdx.x, w.B * w.H);
    const int bh = at_.head, q0 = (nqblk - 1 - at_.rank) * 128;      // the last block of a head sees the most keys
    const int b = bh / w.H, head = bh - b * w.H, kvh = head / (w.H / w.Hkv);

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, h = lane >> 5;
    const KeyTiles<BN> kt(w, b, q0, 128);
    const int ntiles = kt.ntiles;

    const int qrow = q0 + 32 * wave + r;
    const int p_own = qrow + kt.shift;
    const bool live = qrow < w.Nq && p_own < kt.len;
    const RowSees sees{p_own - w.window + 1, live ? p_own : -1};
    const int wave_lo = q0 + 32 * wave + kt.shift, wave_hi = min(wave_lo + 32, kt.pz) - 1;

    const T* Kh = Kg + b * w.ks[0] + kvh * w.ks[1];
    const T* Vh = Vg + b * w.vs[0] + kvh * w.vs[1];
    const R rd(lane);
    const TileFetch<T, D, BN, 256> kfetch(tid, w.ks[2], w.d), vfetch(tid, w.vs[2], w.d);
    auto fetch = [&](int t, int kslot) __attribute__((always_inline)) {
        if (t >= ntiles) return;
        const int k0 = kt.first_key(t);
        char* kd = lds + kslot * TILE_B;
        char* vd = lds + (3 + (t & 1)) * TILE_B;
        if (kt.all(k0, w.sinks)) {
            kfetch.fetch(Kh + (int64_t)k0 * w.ks[2], kd, true, [](int) { return true; });
            vfetch.fetch(Vh + (int64_t)k0 * w.vs[2], vd, true, [](int) { return true; });
        } else {
            auto keep = [&](int row) { return kt.one(k0 + row, w.sinks); };
            kfetch.fetch(Kh + (int64_t)k0 * w.ks[2], kd, false, keep);
            vfetch.fetch(Vh + (int64_t)k0 * w.vs[2], vd, false, keep);
        }
    };
    fetch(0, 0);
    fetch(1, 1);

    s16x8 qf[KS], of[KS];
    {
        const int row = min(qrow, w.Nq - 1);
        const T* qp = Qg + b * w.qs[0] + head * w.qs[1] + (int64_t)row * w.qs[2];
        const T* op = dOg + ((int64_t)bh * w.Nq + row) * w.d;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int c = (2 * ks + h) * 8;
            qf[ks] = s16x8{};
            of[ks] = s16x8{};
            if (c < w.d) {
                qf[ks] = *reinterpret_cast<const s16x8*>(qp + c);
                of[ks] = *reinterpret_cast<const s16x8*>(op + c);
            }
        }
    }
    const int64_t orow = (int64_t)bh * w.Nq + min(qrow, w.Nq - 1);
    const RowStat stat = row_stat<T>(of, Og + orow * w.d, LSEg + orow, live, w.d, h, st, rows, (int64_t)bh * nqp + qrow, qrow < nqp);
    const float lse2 = stat.lse2, ndelta = stat.ndelta;
    const float sl2 = w.scale * kLog2eW;

    f32x16 dq[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) dq[db][i] = 0.f;
    tile_ready();

    int cur = 0, nxt = 1, fre = 2;                 // K slots of tiles t, t + 1, t + 2
    // One tile: MASKED, or seen whole by all rows; `some`: the wave's rows see something of it; behind(): requests tile t + 2.
    auto tile = [&](int t, int k0, bool some, auto masked_, auto&& behind) __attribute__((always_inline)) {
        constexpr bool MASKED = decltype(masked_)::value != 0;
        const char* Kb = lds + cur * TILE_B;
        const char* Vb = lds + (3 + (t & 1)) * TILE_B;
        f32x16 s[2], dp[2];
        typename M::vec8 sb[4];
        auto pds = [&](int kb, int i) __attribute__((always_inline)) {
            s[kb][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][i], sl2, -lse2)) * dp[kb][i];
        };
        auto finish = [&](int kb) __attribute__((always_inline)) {
            if constexpr (MASKED) sees.hide(s[kb], kt, t, k0, k0 + 32 * kb + 4 * h, w.sinks, 0.f);
#pragma unroll
            for (int i = 0; i < 16; ++i) sb[2 * kb + (i >> 3)][i & 7] = (T)s[kb][i];
        };
        if (!MASKED || some) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i) { s[kb][i] = 0.f; dp[kb][i] = ndelta; }
            auto block = [&](auto kb_, auto&& after) __attribute__((always_inline)) {
                constexpr int kb = decltype(kb_)::value;
                mma_stream<2 * KS, FW>([&](auto ic) __attribute__((always_inline)) {
                                           constexpr int i = decltype(ic)::value;
                                           return rd.row(i / KS ? Vb : Kb, kb, i % KS);
                                       },
                                       [&](auto ic, s16x8 a) __attribute__((always_inline)) {
                                           constexpr int i = decltype(ic)::value;
                                           if constexpr (i / KS) dp[kb] = mma_chunk<T>(a, of[i % KS], dp[kb]);
                                           else s[kb] = mma_chunk<T>(a, qf[i % KS], s[kb]);
                                       }, after);
            };
            constexpr int EP = 16 / (2 * KS);
            block(IC<0>{}, [](auto) {});
            block(IC<1>{}, [&](auto ic) __attribute__((always_inline)) {
#pragma unroll
                for (int e = 0; e < EP; ++e) pds(0, EP * decltype(ic)::value + e);
            });
            finish(0);
        }
        tile_ready();
        if (!MASKED || some) {
            auto add = [&](auto kb_, auto&& after) __attribute__((always_inline)) {
                constexpr int kb = decltype(kb_)::value;
                mma_stream<2 * DB, FW>([&](auto ic) __attribute__((always_inline)) {
                                           constexpr int i = decltype(ic)::value;
                                           return rd.transposed(Kb, kb, i / DB, i % DB);
                                       },
                                       [&](auto ic, s16x8 a) __attribute__((always_inline)) {
                                           constexpr int i = decltype(ic)::value;
                                           dq[i % DB] = M::run(a, sb[2 * kb + i / DB], dq[i % DB]);
                                       }, after);
            };
            constexpr int EP = 16 / (2 * DB);
            add(IC<0>{}, [&](auto ic) __attribute__((always_inline)) {
#pragma unroll
                for (int e = 0; e < EP; ++e) pds(1, EP * decltype(ic)::value + e);
            });
            finish(1);
            add(IC<1>{}, [&](auto ic) __attribute__((always_inline)) {
                constexpr int from = 2 * DB > FW ? 2 * DB - FW : 0;              // behind the last transposing read
                if constexpr (decltype(ic)::value >= from) behind(IC<decltype(ic)::value - from>{});
            });
        } else {
            behind(IC<0>{});
        }
        const int was = cur;
        cur = nxt; nxt = fre; fre = was;
    };
    auto masked_tiles = [&](int t0, int t1) __attribute__((always_inline)) {
        for (int t = t0; t < t1; ++t) {
            const int k0 = kt.first_key(t);
            tile(t, k0, !(k0 > wave_hi || (k0 + BN <= wave_lo - w.window + 1 && k0 >= w.sinks)), IC<1>{},
                 [&](auto ic) __attribute__((always_inline)) { if constexpr (decltype(ic)::value == 0) fetch(t + 2, fre); });
        }
    };
    const int f0 = kt.whole_from(w.window, 128), f1 = kt.whole_to(128);      // tiles that all rows see whole
    masked_tiles(0, min(f0, ntiles));
    if (f0 < f1) {
        const T* kp = Kh + (int64_t)kt.first_key(f0 + 2) * w.ks[2];
        const T* vp = Vh + (int64_t)kt.first_key(f0 + 2) * w.vs[2];
        const int64_t kstep = BN * w.ks[2], vstep = BN * w.vs[2];
        // (pieces: tile t + 2 is whole too, and is requested two pieces at a step)
        auto whole_tiles = [&](int t0, int t1, auto pieces) __attribute__((always_inline)) {
            for (int t = t0; t < t1; ++t) {
                tile(t, 0, true, IC<0>{}, [&](auto ic) __attribute__((always_inline)) {
                    constexpr int i = decltype(ic)::value, LPT = TileFetch<T, D, BN, 256>::LPT;
                    static_assert(LPT <= (2 * DB < FW ? 2 * DB : FW), "two pieces a step");
                    if constexpr (decltype(pieces)::value) {
                        if constexpr (i < LPT) {
                            kfetch.template piece<i>(kp, lds + fre * TILE_B);
                            vfetch.template piece<i>(vp, lds + (3 + (t & 1)) * TILE_B);
                        }
                    } else if constexpr (i == 0) {
                        fetch(t + 2, fre);
                    }
                });
                kp += kstep;
                vp += vstep;
            }
        };
        whole_tiles(f0, f1 - 2, IC<1>{});
        whole_tiles(max(f0, f1 - 2), f1, IC<0>{});
    }
    masked_tiles(min(max(f0, f1), ntiles), ntiles);

    // (hidden dS are set to 0 behind the product with dP: hidden keys reach dQ, hidden values do not)
    const uint32_t redo = not_finite_rows(dq, live && finite(lse2) && finite(ndelta));
    if (qrow < w.Nq) {
        T* row = dQg + ((int64_t)bh * w.Nq + qrow) * w.d;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = 32 * db + 8 * g + 4 * h;
                typename M::vec4 x;
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = live ? (T)(dq[db][4 * g + j] * w.scale) : (T)0.f;
                if (c < w.d) *reinterpret_cast<typename M::vec4*>(row + c) = x;
            }
    }
    if (redo != 0) {                                        // (window_attn_exact.h)
        const uint32_t cols = hidden_keys<T, D>(kt, w, q0 + 32 * wave + kt.shift, Kh, w.ks[2], lane);
        stored();
        for (uint32_t left = any_lane(cols != 0) ? redo : 0; left != 0; left &= left - 1) {
            const int x = __builtin_ctz(left), i = q0 + 32 * wave + x;
            const int64_t at = ((int64_t)bh * w.Nq + i) * w.d;
            exact_dq_row<T, D>(Qg + b * w.qs[0] + head * w.qs[1] + i * w.qs[2], dOg + at, Kh, Vh, read_lane(lse2, x), read_lane(ndelta, x), dQg + at,
                               w, i + kt.shift, cols, lane);
        }
    }
}

// Few rows (see window_attn_common.h): 32 rows a workgroup, wave x takes tiles x, x + 4, ... of 32 keys.
template <typename T, int D>
__global__ void __launch_bounds__(256, D * sizeof(T) <= 256 ? 2 : 1)
window_bwd_dq_few_kernel(const T* __restrict__ Qg, const T* __restrict__ Kg, const T* __restrict__ Vg,
                         const T* __restrict__ dOg, const T* __restrict__ Og, const float* __restrict__ LSEg, float* __restrict__ st, T* __restrict__ dQg,
                         WindowShape w, int nqp, int64_t rows, int nqblk) {
    using R = TileReader<T, D>;
    constexpr int BN = 32, TILE_B = BN * R::RB, WAVE_B = 2 * TILE_B;
    static_assert(WAVE_B >= 32 * D * 4, "a wave's sums fit its tiles");
    __shared__ __attribute__((aligned(1024))) char lds[4 * WAVE_B];
    __shared__ uint32_t redo_of[4];

    const Ranked at_ = ranked(blockIdx.x, w.B * w.H);
    const int bh = at_.head, q0 = (nqblk - 1 - at_.rank) * 32;
    const int b = bh / w.H, head = bh - b * w.H, kvh = head / (w.H / w.Hkv);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, h = lane >> 5;
    const KeyTiles<BN> kt(w, b, q0, 32);
    const int ntiles = kt.ntiles;
    const int qrow = q0 + r, p_own = qrow + kt.shift;
    const bool live = qrow < w.Nq && p_own < kt.len;
    const RowSees sees{p_own - w.window + 1, live ? p_own : -1};

    const T* Kh = Kg + b * w.ks[0] + kvh * w.ks[1];
    const T* Vh = Vg + b * w.vs[0] + kvh * w.vs[1];
    const R rd(lane);
    const TileFetch<T, D, BN, 64> kfetch(lane, w.ks[2], w.d), vfetch(lane, w.vs[2], w.d);
    char* own = lds + wave * WAVE_B;
    auto fetch = [&](int t, char* to) __attribute__((always_inline)) {
        if (t >= ntiles) return;
        const int k0 = kt.first_key(t);
        const bool all = kt.all(k0, w.sinks);
        auto keep = [&](int row) { return kt.one(k0 + row, w.sinks); };
        kfetch.fetch(Kh + (int64_t)k0 * w.ks[2], to, all, keep);
        vfetch.fetch(Vh + (int64_t)k0 * w.vs[2], to + TILE_B, all, keep);
    };
    fetch(wave, own);

    typename R::frag qf[R::KS], of[R::KS];
    const int row = min(qrow, w.Nq - 1);
    {
        constexpr int EPC = 16 / (int)sizeof(T);
        const T* qp = Qg + b * w.qs[0] + head * w.qs[1] + (int64_t)row * w.qs[2];
        const T* op = dOg + ((int64_t)bh * w.Nq + row) * w.d;
#pragma unroll
        for (int ks = 0; ks < R::KS; ++ks) {
            const int c = (2 * ks + h) * EPC;
            qf[ks] = typename R::frag{};
            of[ks] = typename R::frag{};
            if (c < w.d) {
                qf[ks] = *reinterpret_cast<const typename R::frag*>(qp + c);
                of[ks] = *reinterpret_cast<const typename R::frag*>(op + c);
            }
        }
    }
    const int64_t orow = (int64_t)bh * w.Nq + row;
    const RowStat stat = row_stat<T>(of, Og + orow * w.d, LSEg + orow, live, w.d, h, st, rows, (int64_t)bh * nqp + qrow, wave == 0 && qrow < nqp);
    // the rows between the last workgroup's 32 and nqp are nobody's else: dK, dV reads 64 at a time
    if (wave == 0 && h == 0 && q0 + 32 >= w.Nq && qrow + 32 < nqp) {
        st[(int64_t)bh * nqp + qrow + 32] = INFINITY;
        st[rows + (int64_t)bh * nqp + qrow + 32] = 0.f;
    }
    const float sl2 = w.scale * kLog2eW;

    f32x16 dq[R::DB];
#pragma unroll
    for (int db = 0; db < R::DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) dq[db][i] = 0.f;

    for (int t = wave; t < ntiles; t += 4) {
        const int k0 = kt.first_key(t);
        const char* Kb = own;
        wave_fetched();
        f32x16 s, dp;
#pragma unroll
        for (int i = 0; i < 16; ++i) { s[i] = 0.f; dp[i] = stat.ndelta; }
#pragma unroll
        for (int ks = 0; ks < R::KS; ++ks) s = mma_chunk<T>(rd.row(Kb, 0, ks), qf[ks], s);
#pragma unroll
        for (int ks = 0; ks < R::KS; ++ks) dp = mma_chunk<T>(rd.row(Kb + TILE_B, 0, ks), of[ks], dp);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], sl2, -stat.lse2)) * dp[i];
        if (!(k0 + BN - 1 <= kt.pa && kt.pz == kt.pa + 32 && (k0 >= kt.pa + 32 - w.window || k0 + BN <= w.sinks)))
            sees.hide(s, kt, t, k0, k0 + 4 * h, w.sinks, 0.f);
        rd.add_transposed(Kb, 0, s, dq);
        wave_read();
        fetch(t + 4, own);
    }

    put_sums(reinterpret_cast<float*>(own), dq, r, h);
    {                                                       // (hidden values do not reach dQ, as above)
        const uint32_t bad = not_finite_rows(dq, live && finite(stat.lse2) && finite(stat.ndelta));
        if (lane == 0) redo_of[wave] = bad;
    }
    __syncthreads();
    const uint32_t redo = __builtin_amdgcn_readfirstlane(redo_of[0] | redo_of[1] | redo_of[2] | redo_of[3]);
    typedef T vec4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int e = tid; e < 32 * D / 4; e += 256) {
        const int rw = e / (D / 4), col = (e - rw * (D / 4)) * 4;
        if (q0 + rw >= w.Nq) break;
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < 4; ++x) sum += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + x * WAVE_B) + sum_at<D>(rw, col));
        const bool sees_any = q0 + rw + kt.shift < kt.len;
        vec4 y;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = sees_any ? (T)(sum[j] * w.scale) : (T)0.f;
        if (col < w.d) *reinterpret_cast<vec4*>(dQg + ((int64_t)bh * w.Nq + q0 + rw) * w.d + col) = y;
    }
    if (redo != 0) {                                        // (window_attn_exact.h)
        const uint32_t cols = hidden_keys<T, D>(kt, w, q0 + kt.shift, Kh, w.ks[2], lane);
        stored();
        __syncthreads();
        int turn = 0;
        for (uint32_t left = any_lane(cols != 0) ? redo : 0; left != 0; left &= left - 1, ++turn) {
            if ((turn & 3) != wave) continue;
            const int x = __builtin_ctz(left);
            const int64_t at = ((int64_t)bh * w.Nq + q0 + x) * w.d;
            exact_dq_row<T, D>(Qg + b * w.qs[0] + head * w.qs[1] + (q0 + x) * w.qs[2], dOg + at, Kh, Vh, read_lane(stat.lse2, x),
                               read_lane(stat.ndelta, x), dQg + at, w, q0 + x + kt.shift, cols, lane);
        }
    }
}

// ---------------------------------------------------------------- dK, dV
// Where a workgroup of keys writes: the gradients, or, where its block is split, its part of them.
template <typename T> struct KeyOut {
    T *dk, *dv;                       // of the block's first key
    float *pk, *pv;                   // null: not split
};

// The second look (window_attn_exact.h) of a wave at its keys first .. first + 31, rows base .. of the block: those of `left`, bit x: key
// first + x, of every `turns` of them the ones with turn `mine`; columns [c0, c1).  The workgroup's tiles are [j0, j1), of BQ
// queries, nt a head from tile tq0 on; their queries at positions outside [pa, pz) were fetched as zeros.
template <typename T, int D>
__device__ __forceinline__ void exact_keys(uint32_t left, int turns, int mine, int first, int base, const WindowShape& w, int b, int kvh, int len,
                                           int pa, int pz, int j0, int j1, int nt, int tq0, int BQ, const T* Qg, const T* Kg, const T* Vg,
                                           const T* dOg, const float* st, int nqp, int64_t rows, const KeyOut<T>& to, int c0, int c1, int lane) {
    using L = LaneRow<T, D>;
    const int shift = w.Nk - w.Nq, group = w.H / w.Hkv, last = first + 31;
    // columns that hidden queries reach: of dV where dO is not finite; of dK where Q is not, and all where dO or delta is not
    uint32_t ck = 0, cv = 0;
    for (int j = j0; j < j1; ++j) {
        const int g = j / nt, i0 = (tq0 + j - g * nt) * BQ, head = kvh * group + g, pt = i0 + shift;
        const int64_t bh = (int64_t)b * w.H + head;
        if (pt >= last && pt + BQ <= len && last < w.Nk && (last < w.sinks || pt + BQ - 1 < first + w.window)) continue;
        for (int i = i0; i < i0 + BQ; ++i) {
            if (!finite(st[rows + bh * nqp + i])) ck = L::all(w.d, lane);
            if (i + shift < pa || i + shift >= pz) continue;
            const uint32_t bad = L(dOg + (bh * w.Nq + i) * w.d, w.d, lane).not_finite();
            cv |= bad;
            ck |= any_lane(bad != 0) ? L::all(w.d, lane) : L(Qg + b * w.qs[0] + head * w.qs[1] + i * w.qs[2], w.d, lane).not_finite();
        }
    }
    if (!any_lane((ck | cv) != 0)) return;
    for (int turn = 0; left != 0; left &= left - 1, ++turn) {
        if (turn % turns != mine) continue;
        const int x = __builtin_ctz(left), key = first + x;
        const int p_hi = key < w.sinks ? len - 1 : min(len - 1, key + w.window - 1);
        ExactKey<T, D> e(Kg + b * w.ks[0] + kvh * w.ks[1] + key * w.ks[2], Vg + b * w.vs[0] + kvh * w.vs[1] + key * w.vs[2], w, lane);
        bool more = true;
        for (int j = j0; j < j1 && more; ++j) {
            const int g = j / nt, i0 = (tq0 + j - g * nt) * BQ, head = kvh * group + g;
            const int64_t bh = (int64_t)b * w.H + head;
            const int from = max(i0, key - shift), to_i = min(i0 + BQ - 1, p_hi - shift);
            for (int i = max(from, 0); i <= to_i && more; i += kAtOnce) {
                e.add(Qg + b * w.qs[0] + head * w.qs[1] + i * w.qs[2], w.qs[2], dOg + (bh * w.Nq + i) * w.d, st + bh * nqp + i,
                      st + rows + bh * nqp + i, min(kAtOnce, to_i + 1 - i));
                more = any_lane(((ck & ~e.dk.not_finite()) | (cv & ~e.dv.not_finite())) != 0);
            }
        }
        const int64_t at = (int64_t)(base + x) * w.d;
        if (to.pk) {
            e.dk.store(to.pk + at, w.scale, ck, c0, c1, lane);
            e.dv.store(to.pv + at, 1.f, cv, c0, c1, lane);
        } else {
            e.dk.store(to.dk + at, w.scale, ck, c0, c1, lane);
            e.dv.store(to.dv + at, 1.f, cv, c0, c1, lane);
        }
    }
}
template <typename T, int D>
__global__ void __launch_bounds__(256, D * sizeof(T) <= 128 ? 2 : 1)
window_bwd_dkv_kernel(const T* __restrict__ Qg, const T* __restrict__ Kg, const T* __restrict__ Vg,
                      const T* __restrict__ dOg, const float* __restrict__ st, T* __restrict__ dKg, T* __restrict__ dVg,
                      float* __restrict__ parts, WindowShape w, int nqp, int64_t rows, int nsb, int ns) {
    using R = TileReader<T, D>;
    constexpr int BQ = bwd_tile<T, D>(), NB = BQ / 32, TILE_B = BQ * R::RB;
    constexpr int ODB = R::DB < 4 ? R::DB : 4, NC = R::DB / ODB;             // column blocks kept, workgroups per key block
    __shared__ __attribute__((aligned(1024))) char lds[4 * TILE_B + 4 * 64 * 4];   // Q0 Q1 dO0 dO1 [buf][lse2 | -delta][64]
    float* stat = reinterpret_cast<float*>(lds + 4 * TILE_B);

    // a head's units: the split sink blocks first, then the other key blocks; the last ones see the fewest queries
    const int lid = blockIdx.x / NC, col0 = ((int)blockIdx.x - lid * NC) * ODB * 32;
    const Ranked at_ = ranked(lid, w.B * w.Hkv);
    const int bg = at_.head, unit = at_.rank;
    const bool split = unit < nsb * ns;
    const int kblk = split ? unit / ns : unit - nsb * ns + nsb, part = split ? unit - kblk * ns : 0, nparts = split ? ns : 1;
    const int b = bg / w.Hkv, kvh = bg - b * w.Hkv, group = w.H / w.Hkv;
    const int k0 = kblk * 128;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, h = lane >> 5;
    const int len = w.lens ? min(max(w.lens[b], 0), w.Nk) : w.Nk;
    const int shift = w.Nk - w.Nq;
    // positions that see some key of the block: [pa, pz)
    const int pa = max(k0, shift), pz = k0 < w.sinks ? len : min(len, k0 + 127 + w.window);
    const int tq0 = (pa - shift) / BQ, nt = pz > pa ? (pz - shift + BQ - 1) / BQ - tq0 : 0;
    const int total = nt * group;
    const int j0 = (int)((int64_t)total * part / nparts), j1 = (int)((int64_t)total * (part + 1) / nparts);

    const int krow = k0 + 32 * wave + r;
    // positions that see the lane's key
    const int p_lo = krow, p_hi = krow >= w.Nk ? -1 : krow < w.sinks ? len - 1 : min(len - 1, krow + w.window - 1);
    const bool seen = max(p_lo, shift) <= p_hi;      // a key that no query sees counts as zeros, whatever stands there
    const int key_a = k0 + 32 * wave, key_z = key_a + 31;                 // the wave's keys

    constexpr int EPC = 16 / (int)sizeof(T);
    typename R::frag kf[R::KS], vf[R::KS];
    {
        const int row = min(krow, w.Nk - 1);
        const T* kp = Kg + b * w.ks[0] + kvh * w.ks[1] + (int64_t)row * w.ks[2];
        const T* vp = Vg + b * w.vs[0] + kvh * w.vs[1] + (int64_t)row * w.vs[2];
#pragma unroll
        for (int ks = 0; ks < R::KS; ++ks) {
            const int c = (2 * ks + h) * EPC;
            kf[ks] = typename R::frag{};
            vf[ks] = typename R::frag{};
            if (c < w.d && seen) {
                kf[ks] = *reinterpret_cast<const typename R::frag*>(kp + c);
                vf[ks] = *reinterpret_cast<const typename R::frag*>(vp + c);
            }
        }
    }
    const float sl2 = w.scale * kLog2eW;

    const R rd(lane);
    const TileFetch<T, D, BQ, 256> qfetch(tid, w.qs[2], w.d), ofetch(tid, w.d, w.d);
    auto fetch = [&](int j, int buf) __attribute__((always_inline)) {
        const int g = j / nt, i0 = (tq0 + j - g * nt) * BQ;
        const int head = kvh * group + g;
        const int64_t bh = (int64_t)b * w.H + head;
        const bool all = i0 + shift >= pa && i0 + BQ + shift <= pz;
        auto keep = [&](int row) { const int p = i0 + row + shift; return (p >= pa) & (p < pz); };
        qfetch.fetch(Qg + b * w.qs[0] + head * w.qs[1] + (int64_t)i0 * w.qs[2], lds + buf * TILE_B, all, keep);
        ofetch.fetch(dOg + (bh * w.Nq + i0) * w.d, lds + (2 + buf) * TILE_B, all, keep);
#if defined(__HIP_DEVICE_COMPILE__)
        if (wave < 2) {
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)(st + wave * rows + bh * nqp + i0), 0, BQ * 4, 0x00020000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(stat + (2 * buf + wave) * 64), 4, lane * 4, 0, 0, 0);
        }
#endif
    };

    f32x16 dk[ODB], dv[ODB];
#pragma unroll
    for (int db = 0; db < ODB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) { dk[db][i] = 0.f; dv[db][i] = 0.f; }

    if (j0 < j1) fetch(j0, 0);
    for (int j = j0; j < j1; ++j) {
        const int buf = (j - j0) & 1;
        tile_ready();
        if (j + 1 < j1) fetch(j + 1, buf ^ 1);
        const int g = j / nt, pt = (tq0 + j - g * nt) * BQ + shift;              // position of the tile's first row
        if (pt + BQ <= key_a || (key_a >= w.sinks && pt > key_z + w.window - 1)) continue;
        const char* Qb = lds + buf * TILE_B;
        const char* Ob = lds + (2 + buf) * TILE_B;
        const float* lse2b = stat + 2 * buf * 64;
        const bool edge = !(pt >= key_z && pt + BQ <= len && key_z < w.Nk && (key_z < w.sinks || pt + BQ - 1 < key_a + w.window));
#pragma unroll
        for (int qb = 0; qb < NB; ++qb) {
            f32x16 s, dp;
            f32x4 l4[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                l4[q] = *reinterpret_cast<const f32x4*>(lse2b + 32 * qb + 8 * q + 4 * h);
                const f32x4 nd = *reinterpret_cast<const f32x4*>(lse2b + 64 + 32 * qb + 8 * q + 4 * h);
#pragma unroll
                for (int e = 0; e < 4; ++e) { s[4 * q + e] = 0.f; dp[4 * q + e] = nd[e]; }
            }
#pragma unroll
            for (int ks = 0; ks < R::KS; ++ks) s = mma_chunk<T>(rd.row(Qb, qb, ks), kf[ks], s);
#pragma unroll
            for (int ks = 0; ks < R::KS; ++ks) dp = mma_chunk<T>(rd.row(Ob, qb, ks), vf[ks], dp);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], sl2, -l4[i >> 2][i & 3]));
                dp[i] *= s[i];
            }
            if (edge) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int p = pt + 32 * qb + 8 * (i >> 2) + 4 * h + (i & 3);
                    if ((p < p_lo) | (p > p_hi)) { s[i] = 0.f; dp[i] = 0.f; }
                }
            }
            rd.add_transposed(Ob + R::COLB * (col0 / 32), qb, s, dv);
            rd.add_transposed(Qb + R::COLB * (col0 / 32), qb, dp, dk);
        }
    }

    const uint32_t redo = not_finite_rows(dk, krow < w.Nk) | not_finite_rows(dv, krow < w.Nk);
    if (krow < w.Nk) {
        typedef T vec4 __attribute__((ext_vector_type(4)));
        const int64_t at = ((int64_t)bg * w.Nk + krow) * w.d;
        float* pk = parts + (((int64_t)(bg * nsb + kblk) * ns + part) * 2 * 128 + (krow - k0)) * w.d;
#pragma unroll
        for (int db = 0; db < ODB; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = col0 + 32 * db + 8 * g + 4 * h;
                if (c >= w.d) continue;
                f32x4 xk, xv;
#pragma unroll
                for (int e = 0; e < 4; ++e) { xk[e] = dk[db][4 * g + e] * w.scale; xv[e] = dv[db][4 * g + e]; }
                if (split && ns > 1) {
                    *reinterpret_cast<f32x4*>(pk + c) = xk;
                    *reinterpret_cast<f32x4*>(pk + (int64_t)128 * w.d + c) = xv;
                } else {
                    vec4 yk, yv;
#pragma unroll
                    for (int e = 0; e < 4; ++e) { yk[e] = (T)xk[e]; yv[e] = (T)xv[e]; }
                    *reinterpret_cast<vec4*>(dKg + at + c) = yk;
                    *reinterpret_cast<vec4*>(dVg + at + c) = yv;
                }
            }
    }
    if (redo != 0) {                                        // (window_attn_exact.h)
        const KeyOut<T> to{dKg + ((int64_t)bg * w.Nk + k0) * w.d, dVg + ((int64_t)bg * w.Nk + k0) * w.d,
                           split && ns > 1 ? parts + ((int64_t)(bg * nsb + kblk) * ns + part) * 2 * 128 * w.d : nullptr,
                           split && ns > 1 ? parts + (((int64_t)(bg * nsb + kblk) * ns + part) * 2 + 1) * 128 * w.d : nullptr};
        stored();
        exact_keys<T, D>(redo, 1, 0, k0 + 32 * wave, 32 * wave, w, b, kvh, len, pa, pz, j0, j1, nt, tq0, BQ, Qg, Kg, Vg, dOg, st, nqp, rows, to,
                         col0, min(w.d, col0 + 32 * ODB), lane);
    }
}

// dK, dV for 16-bit elements and up to 128 columns: one wave per SIMD with the keys' fragments and both
// accumulators in its 512 registers, the tile one pinned stream of 8 KS MFMAs whose shadows take the
// vector work in the order that attn_bwd_plan.h plans.  S and dP are pinned to vector registers (Mma::acc_v),
// with the distance to their readers that this asks for; dK and dV to the accumulator registers by use.  Three
// buffers of Q and dO: tile j + 2 is requested in the last steps of tile j, behind its last transposing read.
// The tiles of a query head in which every row sees every key of the workgroup carry no mask code.
template <typename T, int D>
__global__ void __launch_bounds__(256, 1)
window_bwd_dkv16_kernel(const T* __restrict__ Qg, const T* __restrict__ Kg, const T* __restrict__ Vg,
                        const T* __restrict__ dOg, const float* __restrict__ st, T* __restrict__ dKg, T* __restrict__ dVg,
                        float* __restrict__ parts, WindowShape w, int nqp, int64_t rows, int nsb, int ns) {
    using M = Mma<T>;
    using vec8 = typename M::vec8;
    using vec4 = typename M::vec4;
    using R = TileReader<T, D>;
    constexpr int BQ = 64, KS = R::KS, DB = R::DB, TILE_B = BQ * R::RB;
    using F = TileFetch<T, D, BQ, 256>;
    constexpr int LPT = F::LPT;
    __shared__ __attribute__((aligned(1024))) char lds[6 * TILE_B + 6 * BQ * 4];    // Q0 Q1 Q2 dO0 dO1 dO2, [buf][lse2 | -delta][64]
    float* stat = reinterpret_cast<float*>(lds + 6 * TILE_B);

    const Ranked at_ = ranked(blockIdx.x, w.B * w.Hkv);
    const int bg = at_.head, unit = at_.rank;
    const bool split = unit < nsb * ns;
    const int kblk = split ? unit / ns : unit - nsb * ns + nsb, part = split ? unit - kblk * ns : 0, nparts = split ? ns : 1;
    const int b = bg / w.Hkv, kvh = bg - b * w.Hkv, group = w.H / w.Hkv;
    const int k0 = kblk * 128;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, h = lane >> 5;
    const int len = w.lens ? min(max(w.lens[b], 0), w.Nk) : w.Nk;
    const int shift = w.Nk - w.Nq;
    // positions that see some key of the block: [pa, pz); tiles of a head: nt from tq0 on
    const int pa = max(k0, shift), pz = k0 < w.sinks ? len : min(len, k0 + 127 + w.window);
    const int tq0 = (pa - shift) / BQ, nt = pz > pa ? (pz - shift + BQ - 1) / BQ - tq0 : 0;
    const int total = nt * group;
    const int j0 = (int)((int64_t)total * part / nparts), j1 = (int)((int64_t)total * (part + 1) / nparts);
    // tiles [m0, m1) of a head are whole: positions at or behind the block's last key, inside the length, and
    // inside the window of its first key unless all of it are sinks
    const int whole_end = k0 + 127 >= w.Nk ? 0 : k0 + 128 <= w.sinks ? len : min(len, k0 + w.window);
    const int m0 = max(k0 + 127 - shift - tq0 * BQ + BQ - 1, 0) / BQ, m1 = max(whole_end - shift - tq0 * BQ, 0) / BQ;

    const int krow = k0 + 32 * wave + r;
    const int p_lo = krow, p_hi = krow >= w.Nk ? -1 : krow < w.sinks ? len - 1 : min(len - 1, krow + w.window - 1);
    const bool seen = max(p_lo, shift) <= p_hi;      // a key that no query sees counts as zeros, whatever stands there

    s16x8 kf_[KS], vf_[KS];
    {
        const int row = min(krow, w.Nk - 1);
        const T* kp = Kg + b * w.ks[0] + kvh * w.ks[1] + (int64_t)row * w.ks[2];
        const T* vp = Vg + b * w.vs[0] + kvh * w.vs[1] + (int64_t)row * w.vs[2];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int c = (2 * ks + h) * 8;
            kf_[ks] = s16x8{};
            vf_[ks] = s16x8{};
            if (c < w.d && seen) {
                kf_[ks] = *reinterpret_cast<const s16x8*>(kp + c);
                vf_[ks] = *reinterpret_cast<const s16x8*>(vp + c);
            }
        }
    }
    vec8 kf[KS], vf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) { kf[ks] = __builtin_bit_cast(vec8, kf_[ks]); vf[ks] = __builtin_bit_cast(vec8, vf_[ks]); }
    const float sl2 = w.scale * kLog2eW;

    const R rd(lane);
    const F qfetch(tid, w.qs[2], w.d), ofetch(tid, w.d, w.d);
    // A place in the flat list of tiles, head after head: tile x of head g, and where its rows begin.
    struct At { const T *q, *o; const float* s; int p, x; };
    const int64_t qstep = BQ * w.qs[2], ostep = (int64_t)BQ * w.d;
    const int64_t qhead = w.qs[1] - (nt - 1) * qstep, ohead = (int64_t)w.Nq * w.d - (nt - 1) * ostep, shead = nqp - (nt - 1) * BQ;
    auto next_of = [&](At& a) __attribute__((always_inline)) {
        const bool wrap = a.x + 1 == nt;
        a.q += wrap ? qhead : qstep;
        a.o += wrap ? ohead : ostep;
        a.s += wrap ? shead : (int64_t)BQ;
        a.p = wrap ? tq0 * BQ + shift : a.p + BQ;
        a.x = wrap ? 0 : a.x + 1;
    };
    // piece p of a tile's fetch: even p chunk set p / 2 of Q, odd p that of dO (p < 2 LPT), then the row statistics (wave 0).
    // Rows that see no key of the block read as zeros.
    auto fetch_piece = [&](const At& a, int buf, auto p_) __attribute__((always_inline)) {
#if defined(__HIP_DEVICE_COMPILE__)
        constexpr int p = decltype(p_)::value;
        if constexpr (p < 2 * LPT) {
            const F& f = p % 2 ? ofetch : qfetch;
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)(p % 2 ? a.o : a.q), 0, kTileBytesMax, 0x00020000);
            const int off = (unsigned)(a.p + f.row[p / 2] - pa) < (unsigned)(pz - pa) ? f.off[p / 2] : kOffPast;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(lds + ((p % 2) * 3 + buf) * TILE_B + 1024 * (wave * LPT + p / 2)), 16, off, 0, 0, 0);
        } else if (wave == 0) {
            const __amdgpu_buffer_rsrc_t rl = __builtin_amdgcn_make_buffer_rsrc((void*)a.s, 0, BQ * 4, 0x00020000);
            const __amdgpu_buffer_rsrc_t rdl = __builtin_amdgcn_make_buffer_rsrc((void*)(a.s + rows), 0, BQ * 4, 0x00020000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rl, (lds_void*)(stat + buf * 2 * BQ), 4, lane * 4, 0, 0, 0);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rdl, (lds_void*)(stat + buf * 2 * BQ + BQ), 4, lane * 4, 0, 0, 0);
        }
#endif
    };
    auto fetch_tile = [&](const At& a, int buf) __attribute__((always_inline)) {
        static_for<2 * LPT + 1>([&](auto ic) __attribute__((always_inline)) { fetch_piece(a, buf, ic); });
    };

    f32x16 dk[DB], dv[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) { dk[db][i] = 0.f; dv[db][i] = 0.f; }

    using Plan = DkvPlanFor<KS>;
    static_assert(Plan::plan.ok && 4 * DB == 2 * KS, "every vector operation placed before its deadline");
    constexpr int NSTEP = 8 * KS, FW = 8, PSTEP = FW / (2 * LPT);
    static_assert(PSTEP >= 1 && PSTEP * 2 * LPT == FW, "the tile's loads fill its last FW steps");
    int cur = 0, nxt = 1, fre = 2;
    At ahead{};                                    // tile j + 2, or the last one
    int pt = 0, left = 0;                          // the position tile j begins at; tiles behind `ahead`

    auto tile = [&](auto edge_) __attribute__((always_inline)) {
        constexpr bool EDGE = decltype(edge_)::value != 0;
        const char* Qb = lds + cur * TILE_B;
        const char* dOb = lds + (3 + cur) * TILE_B;
        const float* lse2b = stat + cur * 2 * BQ;
        f32x16 s[2], dp[2];
        f32x4 l4[2][4];
        vec8 pb[4], sb[4];
#pragma unroll
        for (int qb = 0; qb < 2; ++qb)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                l4[qb][g] = *reinterpret_cast<const f32x4*>(lse2b + 32 * qb + 8 * g + 4 * h);
                const f32x4 nd = *reinterpret_cast<const f32x4*>(lse2b + BQ + 32 * qb + 8 * g + 4 * h);
                dp[qb][4 * g] = nd[0]; dp[qb][4 * g + 1] = nd[1]; dp[qb][4 * g + 2] = nd[2]; dp[qb][4 * g + 3] = nd[3];
            }
        // element c = 32 qb + 8 (i >> 2) + (i & 3) of this lane is seen iff c_lo <= c <= c_lo + c_span
        [[maybe_unused]] const int c_lo = p_hi < p_lo ? 1 << 30 : p_lo - (pt + 4 * h);
        [[maybe_unused]] const unsigned c_span = p_hi < p_lo ? 0u : (unsigned)(p_hi - p_lo);

        auto frag = [&](auto gc) __attribute__((always_inline)) -> s16x8 {
            constexpr int g = decltype(gc)::value;
            if constexpr (g < 4 * KS) {
                constexpr int qb = g / (2 * KS), which = (g / KS) & 1, ks = g % KS;
                return rd.row(which ? dOb : Qb, qb, ks);
            } else {
                constexpr int qb = (g - 4 * KS) / (2 * KS), i = g % (2 * KS);
                constexpr int sx = i / (2 * DB), db = (i / 2) % DB, which = i & 1;
                return rd.transposed(which ? Qb : dOb, qb, sx, db);
            }
        };
        auto mma = [&](auto gc, s16x8 a) __attribute__((always_inline)) {
            constexpr int g = decltype(gc)::value;
            if constexpr (g < 4 * KS) {
                constexpr int qb = g / (2 * KS), which = (g / KS) & 1, ks = g % KS;
                if constexpr (which) M::acc_v(a, vf[ks], dp[qb]);
                else if constexpr (ks == 0) M::first_v(a, kf[0], s[qb]);
                else M::acc_v(a, kf[ks], s[qb]);
            } else {
                constexpr int qb = (g - 4 * KS) / (2 * KS), i = g % (2 * KS);
                constexpr int sx = i / (2 * DB), db = (i / 2) % DB, which = i & 1;
                if constexpr (which) dk[db] = M::run(a, sb[2 * qb + sx], dk[db]);
                else dv[db] = M::run(a, pb[2 * qb + sx], dv[db]);
            }
        };
        auto vop = [&](auto op_) __attribute__((always_inline)) {
            constexpr int o = decltype(op_)::value;
            constexpr int qb = Plan::plan.op[o].blk, kind = Plan::plan.op[o].kind, e = Plan::plan.op[o].e;
            [[maybe_unused]] constexpr int c = 32 * qb + 8 * (e >> 2) + (e & 3);
            if constexpr (kind == 0) {
                s[qb][e] = __builtin_fmaf(s[qb][e], sl2, -l4[qb][e >> 2][e & 3]);
            } else if constexpr (kind == 1) {
                const float pe = __builtin_amdgcn_exp2f(s[qb][e]);
                if constexpr (EDGE) s[qb][e] = (unsigned)(c - c_lo) > c_span ? 0.f : pe;
                else s[qb][e] = pe;
            } else if constexpr (kind == 2) {
                dp[qb][e] *= s[qb][e];
            } else if constexpr (kind == 3) {
                pb[2 * qb + (e >> 2)][(2 * e) & 7] = (T)s[qb][2 * e];
                pb[2 * qb + (e >> 2)][((2 * e) & 7) + 1] = (T)s[qb][2 * e + 1];
            } else {
                sb[2 * qb + (e >> 2)][(2 * e) & 7] = (T)dp[qb][2 * e];
                sb[2 * qb + (e >> 2)][((2 * e) & 7) + 1] = (T)dp[qb][2 * e + 1];
            }
        };
        mma_stream<NSTEP, FW>(frag, mma, [&](auto gc) __attribute__((always_inline)) {
            constexpr int g = decltype(gc)::value;
            // this wave's pieces of tile j + 1, requested a tile ago, are confirmed before those of j + 2 go out
            if constexpr (g == NSTEP - FW) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if constexpr (g >= NSTEP - FW && (g - (NSTEP - FW)) % PSTEP == 0) fetch_piece(ahead, fre, IC<(g - (NSTEP - FW)) / PSTEP>{});
            if constexpr (g == NSTEP - 1) fetch_piece(ahead, fre, IC<2 * LPT>{});
            constexpr int o0 = Plan::plan.start[g], o1 = Plan::plan.start[g + 1];
            static_for<o1 - o0>([&](auto oc) __attribute__((always_inline)) { vop(IC<o0 + decltype(oc)::value>{}); });
        });
        // tile j + 1 complete, tile j released (the bare barrier: the loads just issued stay in flight)
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const int was = cur;
        cur = nxt; nxt = fre; fre = was;
    };

    if (j0 < j1) {
        {
            const int g = j0 / nt, x = j0 - g * nt, i0 = (tq0 + x) * BQ, head = kvh * group + g;
            const int64_t bh = (int64_t)b * w.H + head;
            ahead = At{Qg + b * w.qs[0] + head * w.qs[1] + (int64_t)i0 * w.qs[2], dOg + (bh * w.Nq + i0) * w.d, st + bh * nqp + i0, i0 + shift, x};
        }
        int x = ahead.x;
        pt = ahead.p;
        left = j1 - 1 - j0;
        auto step = [&]() __attribute__((always_inline)) { if (left > 0) { next_of(ahead); --left; } };
        fetch_tile(ahead, 0);
        step();
        fetch_tile(ahead, 1);
        step();
        tile_ready();
        auto run = [&](int n, auto edge_) __attribute__((always_inline)) {
            for (; n > 0; --n) {
                tile(edge_);
                step();
                pt += BQ;
            }
        };
        for (int todo = j1 - j0; todo > 0;) {
            // a head's tiles: masked ones, whole ones, masked ones
            const bool edge = x < m0 || x >= m1;
            const int end = x < m0 ? min(m0, nt) : edge ? nt : m1, n = min(todo, end - x);
            if (edge) run(n, IC<1>{});
            else run(n, IC<0>{});
            todo -= n;
            x += n;
            if (x == nt) { x = 0; pt = tq0 * BQ + shift; }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // nothing in flight into an LDS that is given up
    }

    const uint32_t redo = not_finite_rows(dk, krow < w.Nk) | not_finite_rows(dv, krow < w.Nk);
    if (krow < w.Nk) {
        const int64_t out = ((int64_t)bg * w.Nk + krow) * w.d;
        float* pk = parts + (((int64_t)(bg * nsb + kblk) * ns + part) * 2 * 128 + (krow - k0)) * w.d;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = 32 * db + 8 * g + 4 * h;
                if (c >= w.d) continue;
                f32x4 xk, xv;
#pragma unroll
                for (int e = 0; e < 4; ++e) { xk[e] = dk[db][4 * g + e] * w.scale; xv[e] = dv[db][4 * g + e]; }
                if (split && ns > 1) {
                    *reinterpret_cast<f32x4*>(pk + c) = xk;
                    *reinterpret_cast<f32x4*>(pk + (int64_t)128 * w.d + c) = xv;
                } else {
                    vec4 yk, yv;
#pragma unroll
                    for (int e = 0; e < 4; ++e) { yk[e] = (T)xk[e]; yv[e] = (T)xv[e]; }
                    *reinterpret_cast<vec4*>(dKg + out + c) = yk;
                    *reinterpret_cast<vec4*>(dVg + out + c) = yv;
                }
            }
    }
    if (redo != 0) {                                        // (window_attn_exact.h)
        const KeyOut<T> to{dKg + ((int64_t)bg * w.Nk + k0) * w.d, dVg + ((int64_t)bg * w.Nk + k0) * w.d,
                           split && ns > 1 ? parts + ((int64_t)(bg * nsb + kblk) * ns + part) * 2 * 128 * w.d : nullptr,
                           split && ns > 1 ? parts + (((int64_t)(bg * nsb + kblk) * ns + part) * 2 + 1) * 128 * w.d : nullptr};
        stored();
        exact_keys<T, D>(redo, 1, 0, k0 + 32 * wave, 32 * wave, w, b, kvh, len, pa, pz, j0, j1, nt, tq0, BQ, Qg, Kg, Vg, dOg, st, nqp, rows, to,
                         0, w.d, lane);
    }
}

// Few rows (see window_attn_common.h): 32 keys a workgroup, wave x takes every fourth of the query tiles of 32.
template <typename T, int D>
__global__ void __launch_bounds__(256, 1)
window_bwd_dkv_few_kernel(const T* __restrict__ Qg, const T* __restrict__ Kg, const T* __restrict__ Vg,
                          const T* __restrict__ dOg, const float* __restrict__ st, T* __restrict__ dKg, T* __restrict__ dVg,
                          float* __restrict__ parts, WindowShape w, int nqp, int64_t rows, int nsb, int ns) {
    using R = TileReader<T, D>;
    constexpr int BQ = 32, NBUF = R::RB <= 256 ? 2 : 1, TILE_B = BQ * R::RB, WAVE_B = NBUF * 2 * TILE_B;
    constexpr int ODB = R::DB < 4 ? R::DB : 4, NC = R::DB / ODB, C = 32 * ODB;
    static_assert(WAVE_B >= 2 * 32 * C * 4, "a wave's sums fit its tiles");
    __shared__ __attribute__((aligned(1024))) char lds[4 * WAVE_B];
    __shared__ __attribute__((aligned(16))) float stats[4][NBUF][2][32];
    __shared__ uint32_t redo_of[4];

    const int lid = blockIdx.x / NC, col0 = ((int)blockIdx.x - lid * NC) * C;
    const Ranked at_ = ranked(lid, w.B * w.Hkv);
    const int bg = at_.head, unit = at_.rank;
    const bool split = unit < nsb * ns;
    const int kblk = split ? unit / ns : unit - nsb * ns + nsb, part = split ? unit - kblk * ns : 0, nparts = split ? ns : 1;
    const int b = bg / w.Hkv, kvh = bg - b * w.Hkv, group = w.H / w.Hkv;
    const int k0 = kblk * 32;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, h = lane >> 5;
    const int len = w.lens ? min(max(w.lens[b], 0), w.Nk) : w.Nk;
    const int shift = w.Nk - w.Nq;
    const int pa = max(k0, shift), pz = k0 < w.sinks ? len : min(len, k0 + 31 + w.window);
    const int tq0 = (pa - shift) / BQ, nt = pz > pa ? (pz - shift + BQ - 1) / BQ - tq0 : 0;
    const int total = nt * group;
    const int j0 = (int)((int64_t)total * part / nparts), j1 = (int)((int64_t)total * (part + 1) / nparts);

    const int krow = k0 + r;
    const int p_lo = krow, p_hi = krow >= w.Nk ? -1 : krow < w.sinks ? len - 1 : min(len - 1, krow + w.window - 1);
    const bool seen = max(p_lo, shift) <= p_hi;      // a key that no query sees counts as zeros, whatever stands there

    const R rd(lane);
    const TileFetch<T, D, BQ, 64> qfetch(lane, w.qs[2], w.d), ofetch(lane, w.d, w.d);
    char* own = lds + wave * WAVE_B;
    auto fetch = [&](int j, int buf) __attribute__((always_inline)) {
        if (j >= j1) return;
        const int g = j / nt, i0 = (tq0 + j - g * nt) * BQ;
        const int head = kvh * group + g;
        const int64_t bh = (int64_t)b * w.H + head;
        char* to = own + buf * 2 * TILE_B;
        const bool all = i0 + shift >= pa && i0 + BQ + shift <= pz;
        auto keep = [&](int row) { const int p = i0 + row + shift; return (p >= pa) & (p < pz); };
        qfetch.fetch(Qg + b * w.qs[0] + head * w.qs[1] + (int64_t)i0 * w.qs[2], to, all, keep);
        ofetch.fetch(dOg + (bh * w.Nq + i0) * w.d, to + TILE_B, all, keep);
#if defined(__HIP_DEVICE_COMPILE__)
        if (lane < BQ) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)(st + x * rows + bh * nqp + i0), 0, BQ * 4, 0x00020000);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)&stats[wave][buf][x][0], 4, lane * 4, 0, 0, 0);
            }
        }
#endif
    };
#pragma unroll
    for (int i = 0; i < NBUF; ++i) fetch(j0 + wave + 4 * i, i);

    constexpr int EPC = 16 / (int)sizeof(T);
    typename R::frag kf[R::KS], vf[R::KS];
    {
        const int row = min(krow, w.Nk - 1);
        const T* kp = Kg + b * w.ks[0] + kvh * w.ks[1] + (int64_t)row * w.ks[2];
        const T* vp = Vg + b * w.vs[0] + kvh * w.vs[1] + (int64_t)row * w.vs[2];
#pragma unroll
        for (int ks = 0; ks < R::KS; ++ks) {
            const int c = (2 * ks + h) * EPC;
            kf[ks] = typename R::frag{};
            vf[ks] = typename R::frag{};
            if (c < w.d && seen) {
                kf[ks] = *reinterpret_cast<const typename R::frag*>(kp + c);
                vf[ks] = *reinterpret_cast<const typename R::frag*>(vp + c);
            }
        }
    }
    const float sl2 = w.scale * kLog2eW;
    f32x16 dk[ODB], dv[ODB];
#pragma unroll
    for (int db = 0; db < ODB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) { dk[db][i] = 0.f; dv[db][i] = 0.f; }

    int buf = 0;
    for (int j = j0 + wave; j < j1; j += 4) {
        const int g = j / nt, pt = (tq0 + j - g * nt) * BQ + shift;
        const char* Qb = own + buf * 2 * TILE_B;
        const char* Ob = Qb + TILE_B;
        wave_fetched();
        f32x16 s, dp;
        f32x4 l4[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            l4[q] = *reinterpret_cast<const f32x4*>(&stats[wave][buf][0][8 * q + 4 * h]);
            const f32x4 nd = *reinterpret_cast<const f32x4*>(&stats[wave][buf][1][8 * q + 4 * h]);
#pragma unroll
            for (int e = 0; e < 4; ++e) { s[4 * q + e] = 0.f; dp[4 * q + e] = nd[e]; }
        }
#pragma unroll
        for (int ks = 0; ks < R::KS; ++ks) s = mma_chunk<T>(rd.row(Qb, 0, ks), kf[ks], s);
#pragma unroll
        for (int ks = 0; ks < R::KS; ++ks) dp = mma_chunk<T>(rd.row(Ob, 0, ks), vf[ks], dp);
        const bool edge = !(pt >= k0 + 31 && pt + BQ <= len && k0 + 31 < w.Nk && (k0 + 31 < w.sinks || pt + BQ - 1 < k0 + w.window));
        const int c_lo = p_hi < p_lo ? 1 << 30 : p_lo - (pt + 4 * h);
        const unsigned c_span = p_hi < p_lo ? 0u : (unsigned)(p_hi - p_lo);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], sl2, -l4[i >> 2][i & 3]));
            if (edge && (unsigned)(8 * (i >> 2) + (i & 3) - c_lo) > c_span) s[i] = 0.f;
            dp[i] *= s[i];
        }
        rd.add_transposed(Ob + R::COLB * (col0 / 32), 0, s, dv);
        rd.add_transposed(Qb + R::COLB * (col0 / 32), 0, dp, dk);
        wave_read();
        fetch(j + 4 * NBUF, buf);
        buf = NBUF == 2 ? buf ^ 1 : 0;
    }

    put_sums(reinterpret_cast<float*>(own), dk, r, h);
    put_sums(reinterpret_cast<float*>(own) + 32 * C, dv, r, h);
    {
        const uint32_t bad = not_finite_rows(dk, krow < w.Nk) | not_finite_rows(dv, krow < w.Nk);
        if (lane == 0) redo_of[wave] = bad;
    }
    __syncthreads();
    const uint32_t redo = __builtin_amdgcn_readfirstlane(redo_of[0] | redo_of[1] | redo_of[2] | redo_of[3]);
    typedef T vec4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int e = tid; e < 2 * 32 * C / 4; e += 256) {
        const int which = e / (32 * C / 4), rw = (e / (C / 4)) & 31, col = (e & (C / 4 - 1)) * 4, c = col0 + col;
        if (k0 + rw >= w.Nk || c >= w.d) continue;
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < 4; ++x) sum += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + x * WAVE_B) + which * 32 * C + sum_at<C>(rw, col));
        if (!which) sum *= w.scale;
        if (split && ns > 1) {
            *reinterpret_cast<f32x4*>(parts + ((((int64_t)(bg * nsb + kblk) * ns + part) * 2 + which) * 32 + rw) * w.d + c) = sum;
        } else {
            vec4 y;
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = (T)sum[j];
            *reinterpret_cast<vec4*>((which ? dVg : dKg) + ((int64_t)bg * w.Nk + k0 + rw) * w.d + c) = y;
        }
    }
    if (redo != 0) {                                        // (window_attn_exact.h)
        const KeyOut<T> to{dKg + ((int64_t)bg * w.Nk + k0) * w.d, dVg + ((int64_t)bg * w.Nk + k0) * w.d,
                           split && ns > 1 ? parts + ((int64_t)(bg * nsb + kblk) * ns + part) * 2 * 32 * w.d : nullptr,
                           split && ns > 1 ? parts + (((int64_t)(bg * nsb + kblk) * ns + part) * 2 + 1) * 32 * w.d : nullptr};
        stored();
        __syncthreads();
        exact_keys<T, D>(redo, 4, wave, k0, 0, w, b, kvh, len, pa, pz, j0, j1, nt, tq0, BQ, Qg, Kg, Vg, dOg, st, nqp, rows, to, col0, min(w.d, col0 + C),
                         lane);
    }
}

// ---------------------------------------------------------------- the split key blocks' parts, in order
template <typename T>
__global__ void __launch_bounds__(256)
window_bwd_join_kernel(const float* __restrict__ parts, T* __restrict__ dKg, T* __restrict__ dVg, int Nk, int d, int bk, int nsb, int ns, int64_t n4) {
    typedef T vec4 __attribute__((ext_vector_type(4)));
    const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (u >= n4) return;
    const int per_row = d / 4;
    const int c = (int)(u % per_row) * 4;
    int64_t x = u / per_row;
    const int row = (int)(x % bk); x /= bk;
    const int which = (int)(x % 2); x /= 2;
    const int kblk = (int)(x % nsb);
    const int64_t bg = x / nsb;
    const int krow = kblk * bk + row;
    if (krow >= Nk) return;
    const float* p = parts + (((bg * nsb + kblk) * ns * 2 + which) * bk + row) * (int64_t)d + c;
    f32x4 sum = *reinterpret_cast<const f32x4*>(p);
    for (int i = 1; i < ns; ++i) sum += *reinterpret_cast<const f32x4*>(p + (int64_t)i * 2 * bk * d);
    vec4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (T)sum[e];
    *reinterpret_cast<vec4*>((which ? dVg : dKg) + (bg * Nk + krow) * (int64_t)d + c) = y;
}

// ---------------------------------------------------------------- host
// The kernels for many rows: 16-bit elements up to 128 columns have their own.
template <typename T, int D> struct Large {
    static constexpr auto dq() { if constexpr (sizeof(T) == 2 && D <= 128) return window_bwd_dq16_kernel<T, D>; else return window_bwd_dq_kernel<T, D>; }
    static constexpr auto dkv() { if constexpr (sizeof(T) == 2 && D <= 128) return window_bwd_dkv16_kernel<T, D>; else return window_bwd_dkv_kernel<T, D>; }
};

struct BwdPlan { bool few_q, few_k; int bk, nqp, nkblk, nsb, ns; int64_t rows, stat_floats, part_floats; };

// How many workgroups share a key block with sinks: enough that none has more than about a plain block's
// queries, at most 32 (the parts are written and read once more).  Where many blocks hold sinks there is less to even out, and
// the parts are bounded: they hold as many rows as there are keys, or come from at most 1024 workgroups (four a CU).  Measured, bf16,
// d 128, window 256, without the bound / with: B 4, 32 heads on 8 of 16384 positions, 8192 sinks 27.5 ms and 8.6 GB of workspace / 21.1 ms
// and 554 MB; B 1, 8 heads of 8192, 1024 sinks 268 us, 185 MB / 239 us, 135 MB; one head of 16384, 4000 sinks 210 us both.
constexpr int64_t kSplitUnits = 1024;
BwdPlan bwd_plan(const WindowShape& w, int elem_size) {
    BwdPlan p;
    p.few_q = few_queries(w);
    p.few_k = few_keys(w, elem_size);
    p.bk = p.few_k ? 32 : 128;
    p.nqp = (int)cdiv(w.Nq, kStatPad) * kStatPad;
    p.rows = (int64_t)w.B * w.H * p.nqp;
    p.nkblk = (int)cdiv(w.Nk, p.bk);
    const bool uneven = w.sinks > 0 && w.window + p.bk < w.Nk;
    p.nsb = uneven ? (int)cdiv(w.sinks, p.bk) : 0;
    const int64_t each = cdiv(w.Nk, (int64_t)w.window + p.bk);
    int64_t most = 32;
    if (p.nsb > 0) {
        const int64_t rows = p.nkblk / p.nsb, units = kSplitUnits / ((int64_t)w.B * w.Hkv * p.nsb), bound = rows > units ? rows : units;
        if (bound < most) most = bound > 1 ? bound : 1;
    }
    p.ns = p.nsb > 0 ? (int)(each < most ? each : most) : 1;
    p.stat_floats = 2 * p.rows;
    p.part_floats = p.ns > 1 ? (int64_t)w.B * w.Hkv * p.nsb * p.ns * 2 * p.bk * w.d : 0;
    return p;
}

template <typename T>
int launch_bwd(const void* q, const void* k, const void* v, const void* o, const float* lse, const void* dout,
               void* dq, void* dk, void* dv, float* ws, const WindowShape& w, hipStream_t s) {
    const BwdPlan p = bwd_plan(w, (int)sizeof(T));
    float* st = ws;
    float* parts = ws + p.stat_floats;
    const int nqblk = (int)cdiv(w.Nq, p.few_q ? 32 : 128);
    const int64_t nq = (int64_t)w.B * w.H * nqblk, nkv = (int64_t)w.B * w.Hkv * (p.nsb * (int64_t)p.ns + p.nkblk - p.nsb) * (w.d > 128 ? 2 : 1);
    if (nq > 0x7fffffff || nkv > 0x7fffffff)
        return fail(MYFA_E_UNSUPPORTED, "window attention backward: too many blocks");
    auto go_q = [&](auto kern) {
        if (nq > 0)
            launch_kernel(kern, dim3((unsigned)nq), dim3(256), 0, s, static_cast<const T*>(q), static_cast<const T*>(k),
                          static_cast<const T*>(v), static_cast<const T*>(dout), static_cast<const T*>(o), lse, st, static_cast<T*>(dq),
                          w, p.nqp, p.rows, nqblk);
    };
    auto go_kv = [&](auto kern) {
        launch_kernel(kern, dim3((unsigned)nkv), dim3(256), 0, s, static_cast<const T*>(q), static_cast<const T*>(k),
                      static_cast<const T*>(v), static_cast<const T*>(dout), st, static_cast<T*>(dk), static_cast<T*>(dv), parts,
                      w, p.nqp, p.rows, p.nsb, p.ns);
    };
    // (dQ first: it leaves the row statistics that dK, dV reads)
    if (w.d <= 64) {
        go_q(p.few_q ? window_bwd_dq_few_kernel<T, 64> : Large<T, 64>::dq());
        go_kv(p.few_k ? window_bwd_dkv_few_kernel<T, 64> : Large<T, 64>::dkv());
    } else if (w.d <= 128) {
        go_q(p.few_q ? window_bwd_dq_few_kernel<T, 128> : Large<T, 128>::dq());
        go_kv(p.few_k ? window_bwd_dkv_few_kernel<T, 128> : Large<T, 128>::dkv());
    } else if constexpr (sizeof(T) == 2) {
        go_q(p.few_q ? window_bwd_dq_few_kernel<T, 256> : Large<T, 256>::dq());
        go_kv(p.few_k ? window_bwd_dkv_few_kernel<T, 256> : Large<T, 256>::dkv());
    }
    if (p.ns > 1) {
        const int64_t n4 = (int64_t)w.B * w.Hkv * p.nsb * 2 * p.bk * (w.d / 4);
        launch_kernel(window_bwd_join_kernel<T>, dim3((unsigned)cdiv(n4, 256)), dim3(256), 0, s, parts, static_cast<T*>(dk),
                      static_cast<T*>(dv), w.Nk, w.d, p.bk, p.nsb, p.ns, n4);
    }
    return check_launch("window attention backward");
}

}  // namespace

int64_t window_attn_bwd_ws_bytes(const WindowShape& w, int elem_size) {
    const BwdPlan p = bwd_plan(w, elem_size);
    return (p.stat_floats + p.part_floats) * 4;
}

int window_attn_bwd(const void* q, const void* k, const void* v, const void* o, const float* lse, const void* dout,
                    void* dq, void* dk, void* dv, float* ws, const WindowShape& w, int dtype, hipStream_t s) {
    if (dtype == MYFA_F32) return launch_bwd<float>(q, k, v, o, lse, dout, dq, dk, dv, ws, w, s);
    if (dtype == MYFA_F16) return launch_bwd<_Float16>(q, k, v, o, lse, dout, dq, dk, dv, ws, w, s);
    return launch_bwd<__bf16>(q, k, v, o, lse, dout, dq, dk, dv, ws, w, s);
}

}  // namespace myfa
