// The way out for rows whose tiles hold infinities or NaN that the rows themselves do not see.
//
// In the tiled kernels a hidden pair has weight 0, and 0 times a NaN or an infinity is NaN: a value that one row
// sees would reach the others of its tile.  Nothing in the loops looks for that; at the end a row whose float32 sums
// are not finite although its statistics are is computed again here, key by key (or query by query) over what it
// sees and nothing else, by one wave with the columns on its lanes.  Slow (about a microsecond per two keys), taken
// only when such values are there; a row whose statistics are NaN is NaN by definition and is left.  The looks themselves
// (a ballot per 32 rows, once) cost nothing that shows: 452 us for 16 heads of 16384 positions with a window of 4096, with and without.
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
template <typename T, int KS, typename Frag> __device__ __forceinline__ bool finite_chunks(const Frag (&f)[KS]) {
    constexpr int EPC = 16 / (int)sizeof(T);
    typedef T vec __attribute__((ext_vector_type(EPC)));
    float x = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int j = 0; j < EPC; ++j) x = __builtin_fmaf((float)__builtin_bit_cast(vec, f[ks])[j], 0.f, x);
    return x == 0.f;
}

template <typename T, int D> struct LaneRow {
    static constexpr int N = D / 64;
    float x[N];
    __device__ __forceinline__ LaneRow() {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = 0.f;
    }
    __device__ __forceinline__ LaneRow(const T* p, int d, int lane) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = 64 * i + lane < d ? (float)p[64 * i + lane] : 0.f;
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
    // columns [c0, c1)
    template <typename O> __device__ __forceinline__ void store(O* p, float f, int c0, int c1, int lane) const {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (64 * i + lane >= c0 && 64 * i + lane < c1) p[64 * i + lane] = (O)(x[i] * f);
    }
};

// f(key) over the keys that position p sees
template <class F> __device__ __forceinline__ void for_seen_keys(const WindowShape& w, int p, F&& f) {
    const int lo = max(0, p - w.window + 1);
    for (int j = 0; j < min(w.sinks, lo); ++j) f(j);
    for (int j = lo; j <= p; ++j) f(j);
}

template <typename T, int D>
__device__ __forceinline__ void exact_fwd_row(const T* q, const T* Kh, const T* Vh, T* out, const WindowShape& w, int p, int lane) {
    using L = LaneRow<T, D>;
    const L qr(q, w.d, lane);
    L o;
    float m = -INFINITY, l = 0.f;
    for_seen_keys(w, p, [&](int j) {
        const float s = qr.dot(L(Kh + j * w.ks[2], w.d, lane)) * (w.scale * kLog2eW);
        const float m_new = fmaxf(m, s), ref = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = __builtin_amdgcn_exp2f(m - ref), pj = __builtin_amdgcn_exp2f(s - ref);
        if (m_new > m) o.scale(alpha);
        l = l * alpha + pj;
        m = m_new;
        o.add(pj, L(Vh + j * w.vs[2], w.d, lane));
    });
    o.store(out, 1.f / l, 0, w.d, lane);
}

template <typename T, int D>
__device__ __forceinline__ void exact_dq_row(const T* q, const T* dout, const T* Kh, const T* Vh, float lse2, float ndelta, T* out,
                                             const WindowShape& w, int p, int lane) {
    using L = LaneRow<T, D>;
    const L qr(q, w.d, lane), dr(dout, w.d, lane);
    L dq;
    for_seen_keys(w, p, [&](int j) {
        const L k(Kh + j * w.ks[2], w.d, lane);
        const float pj = __builtin_amdgcn_exp2f(__builtin_fmaf(qr.dot(k), w.scale * kLog2eW, -lse2));
        dq.add(pj * (dr.dot(L(Vh + j * w.vs[2], w.d, lane)) + ndelta), k);
    });
    dq.store(out, w.scale, 0, w.d, lane);
}

// dK and dV of a key: f_query(add) calls add(q row, dout row, lse2, -delta) for every query of the workgroup's tiles that
// sees the key.
template <typename T, int D> struct ExactKey {
    using L = LaneRow<T, D>;
    L k, v, dk, dv;
    float sl2;
    int d, lane;
    __device__ __forceinline__ ExactKey(const T* kr, const T* vr, const WindowShape& w, int ln)
        : k(kr, w.d, ln), v(vr, w.d, ln), sl2(w.scale * kLog2eW), d(w.d), lane(ln) {}
    __device__ __forceinline__ void add(const T* q, const T* dout, float lse2, float ndelta) {
        const L qr(q, d, lane), dr(dout, d, lane);
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(qr.dot(k), sl2, -lse2));
        dv.add(p, dr);
        dk.add(p * (dr.dot(v) + ndelta), qr);
    }
};

}  // namespace
}  // namespace myfa
#endif  // MYFA_WINDOW_ATTN_EXACT_H_
