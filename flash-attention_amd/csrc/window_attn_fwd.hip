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
// zeros: whatever stands there, NaN and infinities too, does not reach the products.
#include "window_attn_common.h"

namespace myfa {
namespace {

// keys per tile: what two buffers of K and V leave room for, twice per CU where the registers allow it
template <typename T, int D> constexpr int win_tile() { return D * (int)sizeof(T) <= 256 ? 64 : 32; }

template <typename T, int D>
__global__ void __launch_bounds__(256, D * sizeof(T) <= 256 ? 2 : 1)
window_attn_fwd_kernel(const T* __restrict__ Qg, const T* __restrict__ Kg, const T* __restrict__ Vg,
                       T* __restrict__ Og, float* __restrict__ LSEg, WindowShape w, int nqblk, int nwg) {
    using R = TileReader<T, D>;
    constexpr int BN = win_tile<T, D>(), NB = BN / 32, TILE_B = BN * R::RB;
    __shared__ __attribute__((aligned(1024))) char lds[4 * TILE_B];   // K0 K1 V0 V1

    const int lid = xcd_range_id(blockIdx.x, nwg);
    const int bh = lid / nqblk;
    const int b = bh / w.H, head = bh - b * w.H, kvh = head / (w.H / w.Hkv);
    const int q0 = (lid - bh * nqblk) * 128;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, h = lane >> 5;
    const int len = w.lens ? min(max(w.lens[b], 0), w.Nk) : w.Nk;
    const int shift = w.Nk - w.Nq;

    // positions of the workgroup's rows that see anything: [pa, pz)
    const int pa = q0 + shift, pz = min(min(q0 + 128, w.Nq) + shift, len);
    const int lo = max(0, pa - w.window + 1);                       // first key of the block's windows
    const int t_win = lo / BN, t_end = pz > pa ? (pz + BN - 1) / BN : t_win;
    const int n_sink = pz > pa ? min((min(w.sinks, pz) + BN - 1) / BN, t_win) : 0;
    const int ntiles = n_sink + (t_end - t_win);

    const int qrow = q0 + 32 * wave + r;
    const int p_own = qrow + shift;
    const bool live = qrow < w.Nq && p_own < len;
    const int p_hi = live ? p_own : -1, p_lo = p_own - w.window + 1;
    const int wave_lo = q0 + 32 * wave + shift, wave_hi = min(wave_lo + 32, pz) - 1;    // positions of the wave's live rows

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
    auto first_key = [&](int t) __attribute__((always_inline)) { return (t < n_sink ? t : t - n_sink + t_win) * BN; };
    auto fetch = [&](int t, int buf) __attribute__((always_inline)) {
        const int k0 = first_key(t);
        const bool all = k0 + BN <= pz && (k0 >= lo || k0 + BN <= w.sinks);
        auto keep = [&](int row) { const int k = k0 + row; return (k < pz) & ((k >= lo) | (k < w.sinks)); };
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
        const int buf = t & 1, k0 = first_key(t);
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
        if (!(k0 + BN - 1 <= wave_lo && wave_lo + 31 < len && wave_lo + 31 - shift < w.Nq &&
              (k0 >= wave_lo + 31 - w.window + 1 || k0 + BN <= w.sinks))) {
#pragma unroll
            for (int kb = 0; kb < NB; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int key = k0 + 32 * kb + 8 * (i >> 2) + 4 * h + (i & 3);
                    if (!((key <= p_hi) & ((key >= p_lo) | (key < w.sinks)))) s[kb][i] = -INFINITY;
                }
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
}

// The kernel for 16-bit elements and up to 128 columns: the same work, arranged for the matrix cores.
//   One barrier a tile, between the softmax and P V: it makes V(t) and K(t + 1) visible and frees K(t) and
//   V(t - 1), so that two buffers of each do.  Their successors, V(t + 1) and K(t + 2), are requested behind the
//   tile's last transposing read: hipcc makes such a read wait for every LDS-DMA load in flight, and so they have
//   the whole of the next S and softmax to arrive in.
//   Both products run as pinned streams (mma_stream).  The running maximum moves only when some row's grows by
//   more than 2^8 (a vote of the wave): until then weights up to 2^8 stand in P, rounded with the same relative
//   error, and the rescale of O, 64 multiplications a lane, stays out of most tiles.
template <typename T, int D>
__global__ void __launch_bounds__(256, 2)
window_attn_fwd16_kernel(const T* __restrict__ Qg, const T* __restrict__ Kg, const T* __restrict__ Vg,
                         T* __restrict__ Og, float* __restrict__ LSEg, WindowShape w, int nqblk, int nwg) {
    using M = Mma<T>;
    using R = TileReader<T, D>;
    constexpr int BN = 64, KS = R::KS, DB = R::DB, TILE_B = BN * R::RB, FW = D == 128 ? 8 : 4;
    __shared__ __attribute__((aligned(1024))) char lds[4 * TILE_B];   // K0 K1 V0 V1

    const int lid = xcd_range_id(blockIdx.x, nwg);
    const int bh = lid / nqblk;
    const int b = bh / w.H, head = bh - b * w.H, kvh = head / (w.H / w.Hkv);
    const int q0 = (lid - bh * nqblk) * 128;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, h = lane >> 5;
    const int len = w.lens ? min(max(w.lens[b], 0), w.Nk) : w.Nk;
    const int shift = w.Nk - w.Nq;
    const int pa = q0 + shift, pz = min(min(q0 + 128, w.Nq) + shift, len);
    const int lo = max(0, pa - w.window + 1);
    const int t_win = lo / BN, t_end = pz > pa ? (pz + BN - 1) / BN : t_win;
    const int n_sink = pz > pa ? min((min(w.sinks, pz) + BN - 1) / BN, t_win) : 0;
    const int ntiles = n_sink + (t_end - t_win);

    const int qrow = q0 + 32 * wave + r;
    const int p_own = qrow + shift;
    const bool live = qrow < w.Nq && p_own < len;
    const int p_hi = live ? p_own : -1, p_lo = p_own - w.window + 1;
    const int wave_lo = q0 + 32 * wave + shift, wave_hi = min(wave_lo + 32, pz) - 1;

    const T* Kh = Kg + b * w.ks[0] + kvh * w.ks[1];
    const T* Vh = Vg + b * w.vs[0] + kvh * w.vs[1];
    const R rd(lane);
    const TileFetch<T, D, BN, 256> kfetch(tid, w.ks[2], w.d), vfetch(tid, w.vs[2], w.d);
    auto first_key = [&](int t) __attribute__((always_inline)) { return (t < n_sink ? t : t - n_sink + t_win) * BN; };
    auto fetch = [&](const auto& f, const T* base, int64_t stride, int t, char* to) __attribute__((always_inline)) {
        const int k0 = first_key(t);
        const bool all = k0 + BN <= pz && (k0 >= lo || k0 + BN <= w.sinks);
        if (all) f.fetch(base + (int64_t)k0 * stride, to, true, [](int) { return true; });
        else f.fetch(base + (int64_t)k0 * stride, to, false, [&](int row) { const int k = k0 + row; return (k < pz) & ((k >= lo) | (k < w.sinks)); });
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
    tile_ready();

    for (int t = 0; t < ntiles; ++t) {
        const int k0 = first_key(t);
        const char* Kb = lds + (t & 1) * TILE_B;
        const char* Vb = lds + (2 + (t & 1)) * TILE_B;
        // something of this tile is seen by the wave's rows
        const bool some = !(k0 > wave_hi || (k0 + BN <= wave_lo - w.window + 1 && k0 >= w.sinks));
        typename M::vec8 pb[4];
        if (some) {
            f32x16 s[2];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[kb][i] = 0.f;
            mma_stream<2 * KS, FW>([&](auto ic) __attribute__((always_inline)) { constexpr int i = decltype(ic)::value; return rd.row(Kb, i / KS, i % KS); },
                                   [&](auto ic, s16x8 a) __attribute__((always_inline)) {
                                       constexpr int i = decltype(ic)::value;
                                       s[i / KS] = mma_chunk<T>(a, qf[i % KS], s[i / KS]);
                                   }, [](auto) {});
            if (!(k0 + BN - 1 <= wave_lo && wave_lo + 31 < len && wave_lo + 31 - shift < w.Nq &&
                  (k0 >= wave_lo + 31 - w.window + 1 || k0 + BN <= w.sinks))) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int key = k0 + 32 * kb + 8 * (i >> 2) + 4 * h + (i & 3);
                        if (!((key <= p_hi) & ((key >= p_lo) | (key < w.sinks)))) s[kb][i] = -INFINITY;
                    }
            }
            float a = vmax3(s[0][0], s[0][1], s[0][2]), c = vmax3(s[1][0], s[1][1], s[1][2]);
#pragma unroll
            for (int i = 3; i < 15; i += 2) { a = vmax3(a, s[0][i], s[0][i + 1]); c = vmax3(c, s[1][i], s[1][i + 1]); }
            const float tmax = half_exchange_max(vmax3(a, c, vmax2(s[0][15], s[1][15]))) * sl2;
            // (a row that has seen nothing has m = -inf: any key it sees moves it)
            if (__builtin_amdgcn_ballot_w64(tmax - m > 8.f) != 0) {
                const float m_new = fmaxf(m, tmax);
                const float alpha = m_new == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
                m = m_new;
                l *= alpha;
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[db][i] *= alpha;
            }
            const float ref = m == -INFINITY ? 0.f : m;
            float sum[2] = {0.f, 0.f};
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][i], sl2, -ref));
                    sum[kb] += p;
                    pb[2 * kb + (i >> 3)][i & 7] = (T)p;
                }
            l += sum[0] + sum[1];
        }
        tile_ready();
        constexpr int NP = 4 * DB;
        if (some) {
            mma_stream<NP, FW>([&](auto ic) __attribute__((always_inline)) {
                                   constexpr int i = decltype(ic)::value, st = i / DB;
                                   return rd.transposed(Vb, st >> 1, st & 1, i % DB);
                               },
                               [&](auto ic, s16x8 a) __attribute__((always_inline)) {
                                   constexpr int i = decltype(ic)::value;
                                   o[i % DB] = M::run(a, pb[i / DB], o[i % DB]);
                               },
                               [&](auto ic) __attribute__((always_inline)) {
                                   if constexpr (decltype(ic)::value == NP - FW) { fetch_v(t + 1); fetch_k(t + 2); }
                               });
        } else {
            fetch_v(t + 1);
            fetch_k(t + 2);
        }
    }

    const float total = half_exchange_sum(l);
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
}

template <typename T>
int launch_fwd(const void* q, const void* k, const void* v, void* o, float* lse, const WindowShape& w, hipStream_t s) {
    const int nqblk = (int)cdiv(w.Nq, 128);
    const int64_t nwg = (int64_t)w.B * w.H * nqblk;
    if (nwg > 0x7fffffff) return fail(MYFA_E_UNSUPPORTED, "window attention: %lld query blocks", (long long)nwg);
    auto go = [&](auto kern) {
        launch_kernel(kern, dim3((unsigned)nwg), dim3(256), 0, s, static_cast<const T*>(q), static_cast<const T*>(k),
                      static_cast<const T*>(v), static_cast<T*>(o), lse, w, nqblk, (int)nwg);
    };
    if constexpr (sizeof(T) == 2) {
        if (w.d <= 64) go(window_attn_fwd16_kernel<T, 64>);
        else if (w.d <= 128) go(window_attn_fwd16_kernel<T, 128>);
        else go(window_attn_fwd_kernel<T, 256>);
    } else {
        if (w.d <= 64) go(window_attn_fwd_kernel<T, 64>);
        else go(window_attn_fwd_kernel<T, 128>);
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
