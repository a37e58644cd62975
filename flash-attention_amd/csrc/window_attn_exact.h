// The way out for rows whose tiles hold infinities or NaN that the rows themselves do not see.
//
// In the tiled kernels a hidden pair has weight 0, and 0 times a NaN or an infinity is NaN: a value that one row
// sees would reach the others of its tile.  Nothing in the loops looks for that.  Where at the end a wave's float32 sums
// are not finite, it looks through what its tiles held hidden (the tiles at the edges of what its rows see, no more) for
// columns that are not finite; in those alone its rows are formed again, key by key (or its keys query by query) over
// what they see and nothing else, with the columns on the lanes and until nothing finite is left in them (a column that is infinite
// by then stays so, though a later key would make it NaN: which of the two a row gets that sees both infinities is not pinned).
// The forward looks at hidden values, dQ at hidden keys (hidden values reach hidden dS alone, which are set to 0 behind
// them), dK and dV at hidden queries, output gradients and statistics.
// In the ordinary case it is a ballot per 32 rows, which costs nothing that shows: 452 us for 16 heads of 16384 positions with
// a window of 4096, with and without.  There, a value row of infinities halfway takes the forward to 22 ms and the backward to
// 176 (one wave forms 32 rows of 4096 keys); one that every later row sees costs the look, 0.7 and 9.5 ms.
#ifndef MYFA_WINDOW_ATTN_EXACT_H_
#define MYFA_WINDOW_ATTN_EXACT_H_
#include "window_attn_common.h"

namespace myfa {
namespace {

// The rows (columns of the accumulator, lane & 31) that hold a value that is not finite, among lanes with `count`.
template <int NDB>
__device__ __forceinline__ uint32_t not_finite_rows(const f32x16 (&acc)[NDB], bool count) {
    float x = 0.f;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) x = __builtin_fmaf(acc[db][i], 0.f, x);
    const uint64_t b = __builtin_amdgcn_ballot_w64(count && !(x == 0.f));
    return (uint32_t)(b | b >> 32);
}
__device__ __forceinline__ bool finite(float x) { return x - x == 0.f; }
__device__ __forceinline__ bool any_lane(bool x) { return __builtin_amdgcn_ballot_w64(x) != 0; }

template <typename T, int D> struct LaneRow {
    static constexpr int N = D / 64;
    float x[N];
    __device__ __forceinline__ LaneRow() {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = 0.f;
    }
    __device__ __forceinline__ LaneRow(const T* p, int d, int lane) {
#pragma unroll
        for (int i = 0; i < N; ++i) {                 // (no branch around the load: one would wait for it there)
            const float y = (float)p[min(64 * i + lane, d - 1)];
            x[i] = 64 * i + lane < d ? y : 0.f;
        }
    }
    __device__ __forceinline__ float dot(const LaneRow& y) const {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) s = __builtin_fmaf(x[i], y.x[i], s);
        return wave_sum(s);
    }
    __device__ __forceinline__ void add(float f, const LaneRow& y) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = __builtin_fmaf(f, y.x[i], x[i]);
    }
    __device__ __forceinline__ void scale(float f) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] *= f;
    }
    // bit i: column 64 i + lane
    static __device__ __forceinline__ uint32_t all(int d, int lane) {
        uint32_t cols = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) cols |= (uint32_t)(64 * i + lane < d) << i;
        return cols;
    }
    __device__ __forceinline__ uint32_t not_finite() const {
        uint32_t bad = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) bad |= (uint32_t)!finite(x[i]) << i;
        return bad;
    }
    // the columns of `cols` within [c0, c1)
    template <typename O> __device__ __forceinline__ void store(O* p, float f, uint32_t cols, int c0, int c1, int lane) const {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if ((cols >> i & 1) && 64 * i + lane >= c0 && 64 * i + lane < c1) p[64 * i + lane] = (O)(x[i] * f);
    }
};

// Columns that are not finite in keys of `base` which the wave with rows at positions p0 .. p0 + 31 goes through and some
// of these rows do not see.
template <typename T, int D, int BN>
__device__ __forceinline__ uint32_t hidden_keys(const KeyTiles<BN>& kt, const WindowShape& w, int p0, const T* base, int64_t stride, int lane) {
    uint32_t bad = 0;
    for (int t = 0; t < kt.ntiles; ++t) {
        const int k0 = kt.first_key(t);
        if (k0 > p0 + 31 || (k0 + BN <= p0 - w.window + 1 && k0 >= w.sinks)) continue;                          // nothing of it is seen
        if (k0 + BN - 1 <= p0 && (k0 > p0 + 31 - w.window || k0 + BN <= w.sinks)) continue;                     // all of it is
        for (int key = k0; key < k0 + BN; ++key)
            if (kt.one(key, w.sinks)) bad |= LaneRow<T, D>(base + key * stride, w.d, lane).not_finite();
    }
    return bad;
}

constexpr int kAtOnce = 4;             // rows of an exact sum whose loads and reductions overlap

// f(key, n): keys key .. key + n - 1, over the keys that position p sees, while it returns true
template <class F> __device__ __forceinline__ void for_seen_keys(const WindowShape& w, int p, F&& f) {
    const int lo = max(0, p - w.window + 1), sinks = min(w.sinks, lo);
    for (int j = 0; j < sinks; j += kAtOnce)
        if (!f(j, min(kAtOnce, sinks - j))) return;
    for (int j = lo; j <= p; j += kAtOnce)
        if (!f(j, min(kAtOnce, p + 1 - j))) return;
}

// What has been stored is stored: nothing of the wave's comes after what it stores next.
__device__ __forceinline__ void stored() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

template <typename T, int D>
__device__ __forceinline__ void exact_fwd_row(const T* q, const T* Kh, const T* Vh, T* out, const WindowShape& w, int p, uint32_t cols, int lane) {
    using L = LaneRow<T, D>;
    const L qr(q, w.d, lane);
    L o;
    float m = -INFINITY, l = 0.f;
    for_seen_keys(w, p, [&](int j, int n) {
        float s[kAtOnce], m_new = m;
        L v[kAtOnce];
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x) {
            const int key = j + min(x, n - 1);
            s[x] = qr.dot(L(Kh + key * w.ks[2], w.d, lane)) * (w.scale * kLog2eW);
            v[x] = L(Vh + key * w.vs[2], w.d, lane);
            m_new = fmaxf(m_new, s[x]);
        }
        const float ref = m_new == -INFINITY ? 0.f : m_new, alpha = __builtin_amdgcn_exp2f(m - ref);
        if (m_new > m) o.scale(alpha);
        l *= alpha;
        m = m_new;
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x)
            if (x < n) {
                const float pj = __builtin_amdgcn_exp2f(s[x] - ref);
                l += pj;
                o.add(pj, v[x]);
            }
        return any_lane((cols & ~o.not_finite()) != 0);
    });
    o.store(out, 1.f / l, cols, 0, w.d, lane);
}

template <typename T, int D>
__device__ __forceinline__ void exact_dq_row(const T* q, const T* dout, const T* Kh, const T* Vh, float lse2, float ndelta, T* out,
                                             const WindowShape& w, int p, uint32_t cols, int lane) {
    using L = LaneRow<T, D>;
    const L qr(q, w.d, lane), dr(dout, w.d, lane);
    L dq;
    for_seen_keys(w, p, [&](int j, int n) {
        float ds[kAtOnce];
        L k[kAtOnce];
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x) {
            const int key = j + min(x, n - 1);
            k[x] = L(Kh + key * w.ks[2], w.d, lane);
            const float pj = __builtin_amdgcn_exp2f(__builtin_fmaf(qr.dot(k[x]), w.scale * kLog2eW, -lse2));
            ds[x] = pj * (dr.dot(L(Vh + key * w.vs[2], w.d, lane)) + ndelta);
        }
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x)
            if (x < n) dq.add(ds[x], k[x]);
        return any_lane((cols & ~dq.not_finite()) != 0);
    });
    dq.store(out, w.scale, cols, 0, w.d, lane);
}

// dK and dV of a key, a few queries at a time: rows q + x qs, dout + x d, statistics lse2[x], ndelta[x] for x < n
template <typename T, int D> struct ExactKey {
    using L = LaneRow<T, D>;
    L k, v, dk, dv;
    float sl2;
    int d, lane;
    __device__ __forceinline__ ExactKey(const T* kr, const T* vr, const WindowShape& w, int ln)
        : k(kr, w.d, ln), v(vr, w.d, ln), sl2(w.scale * kLog2eW), d(w.d), lane(ln) {}
    __device__ __forceinline__ void add(const T* q, int64_t qs, const T* dout, const float* lse2, const float* ndelta, int n) {
        float p[kAtOnce], ds[kAtOnce];
        L qr[kAtOnce], dr[kAtOnce];
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x) {
            const int i = min(x, n - 1);
            qr[x] = L(q + i * qs, d, lane);
            dr[x] = L(dout + (int64_t)i * d, d, lane);
            p[x] = __builtin_amdgcn_exp2f(__builtin_fmaf(qr[x].dot(k), sl2, -lse2[i]));
            ds[x] = p[x] * (dr[x].dot(v) + ndelta[i]);
        }
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x)
            if (x < n) {
                dv.add(p[x], dr[x]);
                dk.add(ds[x], qr[x]);
            }
    }
};

}  // namespace
}  // namespace myfa
#endif  // MYFA_WINDOW_ATTN_EXACT_H_
