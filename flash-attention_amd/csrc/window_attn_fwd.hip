// Attention in which a query sees the last `window` keys up to its own position and the first `sinks`
// keys, forward: O = softmax(scale Q K^T over what is seen) V, for f16 / bf16 / float32 on the matrix cores.
//
// One workgroup = 128 query rows of one head (4 waves x 32), which walks the key tiles that some of its
// rows see: the tiles of the first `sinks` keys, then those from its first row's window start to its last
// row's position.  Running maximum m and sum l per row (float32, base 2); P is rounded to the element type
// before P V (the matrix cores take operands of one type), m, l, S and O are float32 throughout.
//   S^T = K Q^T puts the query on the lane, so that m, l and the rescale are per-lane scalars and P, formed
//   in the accumulator, is in place the B operand of O^T += V^T P^T.
// The tiles go HBM/L2 -> LDS directly, double buffered, one barrier a tile; with 16-bit elements and up to
// 128 columns two workgroups share a CU and run out of step, so that one's exponentials hide behind the
// other's matrix products.
// Keys that no row of the workgroup sees (behind the sequence's length, before the window) are fetched as
// zeros: whatever stands there, NaN and infinities too, does not reach the products.  What some rows see and others
// do not: window_attn_exact.h.
#include "window_attn_exact.h"

namespace myfa {
namespace {

// keys per tile: what two buffers of K and V leave room for, twice per CU where the registers allow it
template <typename T, int D> constexpr int win_tile() { return D * (int)sizeof(T) <= 256 ? 64 : 32; }

template <typename T, int D>
__global__ void __launch_bounds__(256, D * sizeof(T) <= 256 ? 2 : 1)
window_attn_fwd_kernel(const T* __restrict__ Qg, const T* __restrict__ Kg, const T* __restrict__ Vg,
                       T* __restrict__ Og, float* __restrict__ LSEg, WindowShape w, int nqblk) {
    using R = TileReader<T, D>;
    constexpr int BN = win_tile<T, D>(), NB = BN / 32, TILE_B = BN * R::RB;
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
    const int wave_lo = q0 + 32 * wave + kt.shift, wave_hi = min(wave_lo + 32, kt.pz) - 1;    // positions of the wave's live rows

    const T* Kh = Kg + b * w.ks[0] + kvh * w.ks[1];
    const T* Vh = Vg + b * w.vs[0] + kvh * w.vs[1];

    typename R::frag qf[R::KS];
    {
        const T* qp = Qg + b * w.qs[0] + head * w.qs[1] + (int64_t)min(qrow, w.Nq - 1) * w.qs[2];
        constexpr int EPC = 16 / (int)sizeof(T);
#pragma unroll
        for (int ks = 0; ks < R::KS; ++ks) {
            const int c = (2 * ks + h) * EPC;
            if (c < w.d) qf[ks] = *reinterpret_cast<const typename R::frag*>(qp + c);
            else qf[ks] = typename R::frag{};
        }
    }

    const R rd(lane);
    const TileFetch<T, D, BN, 256> kfetch(tid, w.ks[2], w.d), vfetch(tid, w.vs[2], w.d);
    auto fetch = [&](int t, int buf) __attribute__((always_inline)) {
        const int k0 = kt.first_key(t);
        const bool all = kt.all(k0, w.sinks);
        auto keep = [&](int row) { return kt.one(k0 + row, w.sinks); };
        kfetch.fetch(Kh + (int64_t)k0 * w.ks[2], lds + buf * TILE_B, all, keep);
        vfetch.fetch(Vh + (int64_t)k0 * w.vs[2], lds + (2 + buf) * TILE_B, all, keep);
    };

    f32x16 o[R::DB];
#pragma unroll
    for (int db = 0; db < R::DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
    float m = -INFINITY, l = 0.f;
    const float sl2 = w.scale * kLog2eW;

    if (ntiles > 0) fetch(0, 0);
    for (int t = 0; t < ntiles; ++t) {
        const int buf = t & 1, k0 = kt.first_key(t);
        tile_ready();
        if (t + 1 < ntiles) fetch(t + 1, buf ^ 1);
        // nothing of this tile is seen by the wave's rows
        if (k0 > wave_hi || (k0 + BN <= wave_lo - w.window + 1 && k0 >= w.sinks)) continue;
        const char* Kb = lds + buf * TILE_B;
        const char* Vb = lds + (2 + buf) * TILE_B;

        f32x16 s[NB];
#pragma unroll
        for (int kb = 0; kb < NB; ++kb) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[kb][i] = 0.f;
#pragma unroll
            for (int ks = 0; ks < R::KS; ++ks) s[kb] = mma_chunk<T>(rd.row(Kb, kb, ks), qf[ks], s[kb]);
        }
        // every row of the wave sees every key of the tile, or a select per element
        if (!(k0 + BN - 1 <= wave_lo && wave_lo + 31 < kt.pz && (k0 >= wave_lo + 31 - w.window + 1 || k0 + BN <= w.sinks))) {
#pragma unroll
            for (int kb = 0; kb < NB; ++kb) sees.hide(s[kb], kt, t, k0, k0 + 32 * kb + 4 * h, w.sinks, -INFINITY);
        }

        float tmax = s[0][0];
#pragma unroll
        for (int kb = 0; kb < NB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) tmax = fmaxf(tmax, s[kb][i]);
        tmax = half_exchange_max(tmax);
        const float m_new = fmaxf(m, tmax * sl2);
        const float ref = m_new == -INFINITY ? 0.f : m_new;          // a row that has seen nothing yet: all weights 0
        const float alpha = __builtin_amdgcn_exp2f(m - ref);
        m = m_new;
        float psum = 0.f;
#pragma unroll
        for (int kb = 0; kb < NB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[kb][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][i], sl2, -ref));
                psum += s[kb][i];
            }
        l = l * alpha + psum;
#pragma unroll
        for (int db = 0; db < R::DB; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[db][i] *= alpha;
#pragma unroll
        for (int kb = 0; kb < NB; ++kb) rd.add_transposed(Vb, kb, s[kb], o);
    }

    // lane (r, h) holds columns 32 db + 8 g + 4 h + 0..3 of its query in registers 4g..4g+3 of block db
    const float total = half_exchange_sum(l);
    const uint32_t redo = not_finite_rows(o, live && finite(total));
    if (qrow < w.Nq) {
        const float inv = live ? 1.0f / total : 0.f;
        T* orow = Og + ((int64_t)bh * w.Nq + qrow) * w.d;
        typedef T vec4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int db = 0; db < R::DB; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = 32 * db + 8 * g + 4 * h;
                vec4 x;
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = live ? (T)(o[db][4 * g + j] * inv) : (T)0.f;
                if (c < w.d) *reinterpret_cast<vec4*>(orow + c) = x;
            }
        if (LSEg != nullptr && h == 0)
            LSEg[(int64_t)bh * w.Nq + qrow] = live ? (m + __builtin_amdgcn_logf(total)) * kLn2W : -INFINITY;
    }
    if (redo != 0) {                                        // (window_attn_exact.h)
        const uint32_t cols = hidden_keys<T, D>(kt, w, q0 + 32 * wave + kt.shift, Vh, w.vs[2], lane);
        stored();
        for (uint32_t left = any_lane(cols != 0) ? redo : 0; left != 0; left &= left - 1) {
            const int x = q0 + 32 * wave + __builtin_ctz(left);
            exact_fwd_row<T, D>(Qg + b * w.qs[0] + head * w.qs[1] + x * w.qs[2], Kh, Vh, Og + ((int64_t)bh * w.Nq + x) * w.d, w, x + kt.shift, cols, lane);
        }
    }
}

// The kernel for 16-bit elements and up to 128 columns: the same work, arranged for the matrix cores.
//   One barrier a tile, between the softmax and P V: it makes V(t) and K(t + 1) visible and frees K(t) and
//   V(t - 1), so that two buffers of each do.  Their successors, V(t + 1) and K(t + 2), are requested behind the
//   tile's last transposing read: hipcc makes such a read wait for every LDS-DMA load in flight, and so they have
//   the whole of the next S and softmax to arrive in.
//   Both products run as pinned streams (mma_stream).  The weights of a tile are formed against the running maximum
//   as it stands; only when a lane's sum passes 2^8 (a vote of the wave; its first keys always do) is the tile's
//   maximum looked for, the running one moved, O and l rescaled and the weights formed again from the logits.
//   Weights up to 2^8 are rounded with the same relative error, and neither the search for the maximum nor the
//   rescale of O, 64 multiplications a lane, is in most tiles.
//   Rows that see nothing (behind the length) have no vote, and waves of nothing but such rows no products: 16 heads of batches of 16,
//   lengths 185 to 1100 of 1100, 110 us against 119 with them; lengths of whole blocks take the same time.
//   The tiles that every row of the workgroup sees whole run in a loop without masks, bounds or tile arithmetic.
// Measured (bf16, d 128): 16 heads of 16384 positions, window 4096: 452 us, 1065 TFLOP/s of what is seen, where a
// library product of 8192^3 reaches 1194; B 4, 32 heads of 4096 positions, window 1024: 290 us, 832 (a tenth of the work
// is in tiles that the masks halve).  Bound by the matrix pipe at the clock that the power limit leaves it: on operands
// that are all ones the first takes 335 us.  With the next tiles' requests in a row instead of one to a step: 490 against 478
// us on one card, all ones 358 against 335.  Forming each half of a tile's weights beside the products of the other half: no
// faster (458 against 453, all ones 339 against 334), the two workgroups of a CU do that already.
template <typename T, int D>
__global__ void __launch_bounds__(256, 2)
window_attn_fwd16_kernel(const T* __restrict__ Qg, const T* __restrict__ Kg, const T* __restrict__ Vg,
                         T* __restrict__ Og, float* __restrict__ LSEg, WindowShape w, int nqblk) {
    using M = Mma<T>;
    using R = TileReader<T, D>;
    constexpr int BN = 64, KS = R::KS, DB = R::DB, TILE_B = BN * R::RB, FW = D == 128 ? 8 : 4;
    __shared__ __attribute__((aligned(1024))) char lds[4 * TILE_B];   // K0 K1 V0 V1

    const Ranked at_ = ranked(blockIdx.x, w.B * w.H);
    const int bh = at_.head, q0 = (nqblk - 1 - at_.rank) * 128;      // the last block of a head sees the most keys
    const int b = bh / w.H, head = bh - b * w.H, kvh = head / (w.H / w.Hkv);

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, h = lane >> 5;
    const KeyTiles<BN> kt(w, b, q0, 128);
    const int ntiles = kt.ntiles;
    const int f0 = kt.whole_from(w.window, 128), f1 = kt.whole_to(128);      // tiles that all rows see whole

    const int qrow = q0 + 32 * wave + r;
    const int p_own = qrow + kt.shift;
    const bool live = qrow < w.Nq && p_own < kt.len;
    const RowSees sees{p_own - w.window + 1, live ? p_own : -1};
    const int wave_lo = q0 + 32 * wave + kt.shift, wave_hi = min(wave_lo + 32, kt.pz) - 1;

    const T* Kh = Kg + b * w.ks[0] + kvh * w.ks[1];
    const T* Vh = Vg + b * w.vs[0] + kvh * w.vs[1];
    const R rd(lane);
    const TileFetch<T, D, BN, 256> kfetch(tid, w.ks[2], w.d), vfetch(tid, w.vs[2], w.d);
    auto fetch = [&](const auto& f, const T* base, int64_t stride, int t, char* to) __attribute__((always_inline)) {
        const int k0 = kt.first_key(t);
        const bool all = kt.all(k0, w.sinks);
        if (all) f.fetch(base + (int64_t)k0 * stride, to, true, [](int) { return true; });
        else f.fetch(base + (int64_t)k0 * stride, to, false, [&](int row) { return kt.one(k0 + row, w.sinks); });
    };
    auto fetch_k = [&](int t) __attribute__((always_inline)) { if (t < ntiles) fetch(kfetch, Kh, w.ks[2], t, lds + (t & 1) * TILE_B); };
    auto fetch_v = [&](int t) __attribute__((always_inline)) { if (t < ntiles) fetch(vfetch, Vh, w.vs[2], t, lds + (2 + (t & 1)) * TILE_B); };
    fetch_k(0);
    fetch_v(0);
    fetch_k(1);

    s16x8 qf[KS];
    {
        const T* qp = Qg + b * w.qs[0] + head * w.qs[1] + (int64_t)min(qrow, w.Nq - 1) * w.qs[2];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int c = (2 * ks + h) * 8;
            qf[ks] = s16x8{};
            if (c < w.d) qf[ks] = *reinterpret_cast<const s16x8*>(qp + c);
        }
    }
    f32x16 o[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
    float m = -INFINITY, l = 0.f;
    const float sl2 = w.scale * kLog2eW;
    typename M::vec8 pb[4];

    auto logits = [&](const char* Kb, f32x16 (&s)[2]) __attribute__((always_inline)) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[kb][i] = 0.f;
        mma_stream<2 * KS, FW>([&](auto ic) __attribute__((always_inline)) { constexpr int i = decltype(ic)::value; return rd.row(Kb, i / KS, i % KS); },
                               [&](auto ic, s16x8 a) __attribute__((always_inline)) {
                                   constexpr int i = decltype(ic)::value;
                                   s[i / KS] = mma_chunk<T>(a, qf[i % KS], s[i / KS]);
                               }, [](auto) {});
    };
    // votes: the lane's row sees something (rows that never do have no maximum to come)
    auto softmax = [&](f32x16 (&s)[2], bool votes) __attribute__((always_inline)) {
        float sum[2];
        auto weights = [&](float ref) __attribute__((always_inline)) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][i], sl2, -ref));
                    sum[kb] = i == 0 ? p : sum[kb] + p;
                    pb[2 * kb + (i >> 3)][i & 7] = (T)p;
                }
        };
        weights(m == -INFINITY ? 0.f : m);
        // (negated: a NaN or an infinite sum goes back too)
        if (__builtin_amdgcn_ballot_w64(votes && (!(sum[0] + sum[1] <= 256.f) || m == -INFINITY)) != 0) {
            float a = vmax3(s[0][0], s[0][1], s[0][2]), c = vmax3(s[1][0], s[1][1], s[1][2]);
#pragma unroll
            for (int i = 3; i < 15; i += 2) { a = vmax3(a, s[0][i], s[0][i + 1]); c = vmax3(c, s[1][i], s[1][i + 1]); }
            const float m_new = fmaxf(m, half_exchange_max(vmax3(a, c, vmax2(s[0][15], s[1][15]))) * sl2);
            const float alpha = m_new == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);    // (nothing seen yet: all is 0)
            m = m_new;
            l *= alpha;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[db][i] *= alpha;
            weights(m == -INFINITY ? 0.f : m);
        }
        l += sum[0] + sum[1];
    };
    constexpr int NP = 4 * DB;
    auto add_pv = [&](const char* Vb, auto&& behind) __attribute__((always_inline)) {
        mma_stream<NP, FW>([&](auto ic) __attribute__((always_inline)) {
                               constexpr int i = decltype(ic)::value, st = i / DB;
                               return rd.transposed(Vb, st >> 1, st & 1, i % DB);
                           },
                           [&](auto ic, s16x8 a) __attribute__((always_inline)) {
                               constexpr int i = decltype(ic)::value;
                               o[i % DB] = M::run(a, pb[i / DB], o[i % DB]);
                           },
                           [&](auto ic) __attribute__((always_inline)) {
                               if constexpr (decltype(ic)::value >= NP - FW) behind(IC<decltype(ic)::value - (NP - FW)>{});
                           });
    };
    tile_ready();

    auto masked_tiles = [&](int t0, int t1) __attribute__((always_inline)) {
        for (int t = t0; t < t1; ++t) {
            const int k0 = kt.first_key(t);
            // something of this tile is seen by the wave's rows (and some of them see anything)
            const bool some = wave_lo < kt.pz && !(k0 > wave_hi || (k0 + BN <= wave_lo - w.window + 1 && k0 >= w.sinks));
            if (some) {
                f32x16 s[2];
                logits(lds + (t & 1) * TILE_B, s);
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) sees.hide(s[kb], kt, t, k0, k0 + 32 * kb + 4 * h, w.sinks, -INFINITY);
                softmax(s, live);
            }
            tile_ready();
            auto ahead = [&](auto ic) __attribute__((always_inline)) { if constexpr (decltype(ic)::value == 0) { fetch_v(t + 1); fetch_k(t + 2); } };
            if (some) add_pv(lds + (2 + (t & 1)) * TILE_B, ahead);
            else ahead(IC<0>{});
        }
    };
    masked_tiles(0, min(f0, ntiles));
    const int first_after = max(f0, f1);
    if (f0 < f1) {
        const T* kp = Kh + (int64_t)kt.first_key(f0 + 2) * w.ks[2];
        const T* vp = Vh + (int64_t)kt.first_key(f0 + 1) * w.vs[2];
        const int64_t kstep = BN * w.ks[2], vstep = BN * w.vs[2];
        int buf = f0 & 1;
        // (pieces: tiles t + 1 and t + 2 are whole too, and are requested a piece at a step)
        auto whole_tiles = [&](int t0, int t1, auto pieces) __attribute__((always_inline)) {
            for (int t = t0; t < t1; ++t) {
                f32x16 s[2];
                logits(lds + buf * TILE_B, s);
                softmax(s, true);
                tile_ready();
                add_pv(lds + (2 + buf) * TILE_B, [&](auto ic) __attribute__((always_inline)) {
                    constexpr int i = decltype(ic)::value, LPT = TileFetch<T, D, BN, 256>::LPT;
                    static_assert(2 * LPT <= FW, "a piece a step");
                    if constexpr (decltype(pieces)::value) {
                        if constexpr (i < LPT) vfetch.template piece<i>(vp, lds + (3 - buf) * TILE_B);
                        else if constexpr (i < 2 * LPT) kfetch.template piece<i - LPT>(kp, lds + buf * TILE_B);
                    } else if constexpr (i == 0) {
                        fetch_v(t + 1);
                        fetch_k(t + 2);
                    }
                });
                kp += kstep;
                vp += vstep;
                buf ^= 1;
            }
        };
        whole_tiles(f0, f1 - 2, IC<1>{});
        whole_tiles(max(f0, f1 - 2), f1, IC<0>{});
    }
    masked_tiles(min(first_after, ntiles), ntiles);

    const float total = half_exchange_sum(l);
    const uint32_t redo = not_finite_rows(o, live && finite(total));
    if (qrow < w.Nq) {
        const float inv = live ? 1.0f / total : 0.f;
        T* orow = Og + ((int64_t)bh * w.Nq + qrow) * w.d;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = 32 * db + 8 * g + 4 * h;
                typename M::vec4 x;
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = live ? (T)(o[db][4 * g + j] * inv) : (T)0.f;
                if (c < w.d) *reinterpret_cast<typename M::vec4*>(orow + c) = x;
            }
        if (LSEg != nullptr && h == 0)
            LSEg[(int64_t)bh * w.Nq + qrow] = live ? (m + __builtin_amdgcn_logf(total)) * kLn2W : -INFINITY;
    }
    if (redo != 0) {                                        // (window_attn_exact.h)
        const uint32_t cols = hidden_keys<T, D>(kt, w, q0 + 32 * wave + kt.shift, Vh, w.vs[2], lane);
        stored();
        for (uint32_t left = any_lane(cols != 0) ? redo : 0; left != 0; left &= left - 1) {
            const int x = q0 + 32 * wave + __builtin_ctz(left);
            exact_fwd_row<T, D>(Qg + b * w.qs[0] + head * w.qs[1] + x * w.qs[2], Kh, Vh, Og + ((int64_t)bh * w.Nq + x) * w.d, w, x + kt.shift, cols, lane);
        }
    }
}

// Few rows (see window_attn_common.h): 32 rows a workgroup, wave x takes tiles x, x + 4, ... of 32 keys.
template <typename T, int D>
__global__ void __launch_bounds__(256, D * sizeof(T) <= 256 ? 2 : 1)
window_attn_fwd_few_kernel(const T* __restrict__ Qg, const T* __restrict__ Kg, const T* __restrict__ Vg,
                           T* __restrict__ Og, float* __restrict__ LSEg, WindowShape w, int nqblk) {
    using R = TileReader<T, D>;
    constexpr int BN = 32, TILE_B = BN * R::RB, WAVE_B = 2 * TILE_B;
    static_assert(WAVE_B >= 32 * D * 4, "a wave's sums fit its tiles");
    __shared__ __attribute__((aligned(1024))) char lds[4 * WAVE_B];
    __shared__ float ml[4][2][32];
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

    typename R::frag qf[R::KS];
    {
        const T* qp = Qg + b * w.qs[0] + head * w.qs[1] + (int64_t)min(qrow, w.Nq - 1) * w.qs[2];
        constexpr int EPC = 16 / (int)sizeof(T);
#pragma unroll
        for (int ks = 0; ks < R::KS; ++ks) {
            const int c = (2 * ks + h) * EPC;
            qf[ks] = typename R::frag{};
            if (c < w.d) qf[ks] = *reinterpret_cast<const typename R::frag*>(qp + c);
        }
    }
    f32x16 o[R::DB];
#pragma unroll
    for (int db = 0; db < R::DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
    float m = -INFINITY, l = 0.f;
    const float sl2 = w.scale * kLog2eW;

    for (int t = wave; t < ntiles; t += 4) {
        const int k0 = kt.first_key(t);
        const char* Kb = own;
        wave_fetched();
        f32x16 s;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < R::KS; ++ks) s = mma_chunk<T>(rd.row(Kb, 0, ks), qf[ks], s);
        if (!(k0 + BN - 1 <= kt.pa && kt.pz == kt.pa + 32 && (k0 >= kt.pa + 32 - w.window || k0 + BN <= w.sinks)))
            sees.hide(s, kt, t, k0, k0 + 4 * h, w.sinks, -INFINITY);
        float tmax = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) tmax = fmaxf(tmax, s[i]);
        const float m_new = fmaxf(m, half_exchange_max(tmax) * sl2);
        const float ref = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = __builtin_amdgcn_exp2f(m - ref);
        m = m_new;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], sl2, -ref));
            sum += s[i];
        }
        l = l * alpha + sum;
#pragma unroll
        for (int db = 0; db < R::DB; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[db][i] *= alpha;
        rd.add_transposed(Kb + TILE_B, 0, s, o);
        wave_read();
        fetch(t + 4, own);
    }

    l = half_exchange_sum(l);
    if (h == 0) { ml[wave][0][r] = m; ml[wave][1][r] = l; }
    put_sums(reinterpret_cast<float*>(own), o, r, h);
    {
        const uint32_t bad = not_finite_rows(o, live && finite(l));
        if (lane == 0) redo_of[wave] = bad;
    }
    __syncthreads();
    const uint32_t redo = __builtin_amdgcn_readfirstlane(redo_of[0] | redo_of[1] | redo_of[2] | redo_of[3]);
    typedef T vec4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int e = tid; e < 32 * D / 4; e += 256) {
        const int row = e / (D / 4), col = (e - row * (D / 4)) * 4;
        if (q0 + row >= w.Nq) break;
        const bool sees_any = q0 + row + kt.shift < kt.len;
        float top = ml[0][0][row];
#pragma unroll
        for (int x = 1; x < 4; ++x) top = fmaxf(top, ml[x][0][row]);
        const float ref = top == -INFINITY ? 0.f : top;
        float total = 0.f;
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const float f = __builtin_amdgcn_exp2f(ml[x][0][row] - ref);
            total += f * ml[x][1][row];
            sum += f * *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + x * WAVE_B) + sum_at<D>(row, col));
        }
        const float inv = 1.f / total;
        vec4 y;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = sees_any ? (T)(sum[j] * inv) : (T)0.f;
        const int64_t at = (int64_t)bh * w.Nq + q0 + row;
        if (col < w.d) *reinterpret_cast<vec4*>(Og + at * w.d + col) = y;
        if (col == 0 && LSEg != nullptr) LSEg[at] = sees_any ? (top + __builtin_amdgcn_logf(total)) * kLn2W : -INFINITY;
    }
    if (redo != 0) {                                        // (window_attn_exact.h)
        const uint32_t cols = hidden_keys<T, D>(kt, w, q0 + kt.shift, Vh, w.vs[2], lane);
        stored();
        __syncthreads();
        int turn = 0;
        for (uint32_t left = any_lane(cols != 0) ? redo : 0; left != 0; left &= left - 1, ++turn) {
            if ((turn & 3) != wave) continue;
            const int x = q0 + __builtin_ctz(left);
            exact_fwd_row<T, D>(Qg + b * w.qs[0] + head * w.qs[1] + x * w.qs[2], Kh, Vh, Og + ((int64_t)bh * w.Nq + x) * w.d, w, x + kt.shift, cols, lane);
        }
    }
}

template <typename T>
int launch_fwd(const void* q, const void* k, const void* v, void* o, float* lse, const WindowShape& w, hipStream_t s) {
    const bool few = few_queries(w);
    const int nqblk = (int)cdiv(w.Nq, few ? 32 : 128);
    const int64_t nwg = (int64_t)w.B * w.H * nqblk;
    if (nwg > 0x7fffffff) return fail(MYFA_E_UNSUPPORTED, "window attention: %lld query blocks", (long long)nwg);
    auto go = [&](auto kern) {
        launch_kernel(kern, dim3((unsigned)nwg), dim3(256), 0, s, static_cast<const T*>(q), static_cast<const T*>(k),
                      static_cast<const T*>(v), static_cast<T*>(o), lse, w, nqblk);
    };
    if constexpr (sizeof(T) == 2) {
        if (w.d <= 64) few ? go(window_attn_fwd_few_kernel<T, 64>) : go(window_attn_fwd16_kernel<T, 64>);
        else if (w.d <= 128) few ? go(window_attn_fwd_few_kernel<T, 128>) : go(window_attn_fwd16_kernel<T, 128>);
        else few ? go(window_attn_fwd_few_kernel<T, 256>) : go(window_attn_fwd_kernel<T, 256>);
    } else {
        if (w.d <= 64) few ? go(window_attn_fwd_few_kernel<T, 64>) : go(window_attn_fwd_kernel<T, 64>);
        else few ? go(window_attn_fwd_few_kernel<T, 128>) : go(window_attn_fwd_kernel<T, 128>);
    }
    return check_launch("window attention");
}

}  // namespace

int window_attn_fwd(const void* q, const void* k, const void* v, void* o, float* lse, const WindowShape& w, int dtype, hipStream_t s) {
    if (dtype == MYFA_F32) return launch_fwd<float>(q, k, v, o, lse, w, s);
    if (dtype == MYFA_F16) return launch_fwd<_Float16>(q, k, v, o, lse, w, s);
    return launch_fwd<__bf16>(q, k, v, o, lse, w, s);
}

}  // namespace myfa
