// Attention of one new token per sequence over a paged key/value cache, and the append that fills it.
//
//     out[b, h] = softmax_j( scale q[b, h] . K[b, h / G, j] ) V[b, h / G, j]     over the keys j < len[b] that
//     the window leaves: len[b] - 1 - j < window or j < sinks.   G = query heads per key/value head.
//
// HBM-bound: a key costs 2 d elements read and 4 G d flops.  One workgroup takes one key/value head of one
// sequence and a share of its keys, and serves up to 16 query heads with every byte it reads; further query
// heads of the group, and further shares, are other workgroups.  A wave takes tiles of 32 keys:
//   S^T[32 keys x 16 heads] = K Q^T on v_mfma 16x16 (16x16x32 16-bit, 16x16x4 float32), K chunks straight from
//   memory to registers as the A operand; running maximum and sum per head (float32, base 2); P^T is in place
//   the B operand of O^T[d x 16 heads] += V^T P^T, V^T coming through a wave-private LDS tile by transposing
//   reads.  P is rounded to the element type there (the matrix cores take operands of one type, and 16-bit ones at sixteen
//   times float32's rate); logits, maxima, sums, parts and the weights that are added up are float32.
//   The next tile's K and V are requested before the exponentials of this one.
// The waves of a workgroup are joined through LDS; with more than one share per head a second launch joins the
// shares' unnormalised sums, in order.  With `weight_sum`, the logits are kept in the workspace (4 bytes per
// head and key against 4 d read) and the second launch adds exp(logit - lse), summed over the group's heads in
// order, to the running sum of each key.
// Measured, 32 heads on 8, d 128: 8 sequences of up to 131072 keys (f16, 2.7 GB) 476 us = 5.76 TB/s, where a
// product of a matrix and a vector of that size reaches 6.1; 64 of up to 4096 with weights (bf16, 615 MB) 157 us = 3.9 TB/s.  There
// the weights are 20 of it (and the join's launch 13), and unequal lengths little: all of one length 155, sorted 148.  The rest
// is that shares are short: a wave has four tiles in the longest sequence and one or none in a short one, and its first loads and the
// joins in LDS and memory stand beside them.  One sequence of 1024 keys 12.1 us: two launches, 9.4 us of dependent loads (table,
// keys, values) and 2.5 us of join.
// Append: 64 tokens 4.2 us (a launch); 8 prompts of 4096 (268 MB) 55 us = 4.9 TB/s.
#include "paged_common.h"

namespace myfa {

namespace {

constexpr float kLog2eP = 1.4426950408889634f;
constexpr float kLn2P = 0.6931471805599453f;
constexpr int kKeys = 32;             // keys of a wave's tile

// The keys a sequence's new token sees, as tiles of 32: first those of the sinks, then those of the window.
struct Seen {
    int len, lo, n_sink, t_win, ntiles;
    bool past;                        // the given length is beyond the table
};
__device__ __forceinline__ Seen seen_of(int len, int cap, int window, int sinks) {
    Seen s;
    s.past = len > cap;
    s.len = min(max(len, 0), cap);
    s.lo = max(0, s.len - window);
    s.t_win = s.lo / kKeys;
    s.n_sink = min((min(sinks, s.len) + kKeys - 1) / kKeys, s.t_win);
    s.ntiles = s.n_sink + (s.len + kKeys - 1) / kKeys - s.t_win;
    return s;
}

template <typename T> struct DFrag { using type = s16x8; };
template <> struct DFrag<float> { using type = f32x4; };

template <typename T>
__device__ __forceinline__ f32x4 mma16_chunk(typename DFrag<T>::type a, typename DFrag<T>::type b, f32x4 c) {
    if constexpr (sizeof(T) == 2) {
        return Mma16<T>::run(a, __builtin_bit_cast(typename Mma16<T>::vec8, b), c);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
}

// swizzle of a V row's 16-byte chunks: eight rows of the same two columns of chunks on different banks
template <int RB> __device__ __forceinline__ int v_swz(int row) { return RB == 128 ? ((row >> 1) & 3) << 5 : (row & 7) << 5; }

// The sequence that is `slot`-th in length, so that the launch does not end with long ones.
__device__ __forceinline__ int longest_first(const DecodeShape& w, int slot, int lane) {
    const int len = lane < w.B ? max(w.lens[lane], 0) : -1;
    int before = 0;
    for (int x = 0; x < w.B; ++x) {
        const int other = __builtin_amdgcn_readlane(len, x);
        before += (other > len) | ((other == len) & (x < lane));
    }
    return (int)__builtin_ctzll(__builtin_amdgcn_ballot_w64(before == slot && lane < w.B));
}

template <typename T, int D>
__global__ void __launch_bounds__(256, D * sizeof(T) <= 256 ? 3 : 1)
paged_decode_kernel(const T* __restrict__ Qg, PagedCache c, T* __restrict__ Og, float* __restrict__ LSEg, DecodeShape w,
                    int qtiles, int ns, bool ranked, float* __restrict__ part_o, float* __restrict__ part_ml,
                    float* __restrict__ scores, int64_t score_row) {
    using frag = typename DFrag<T>::type;
    constexpr int RB = D * (int)sizeof(T), KS = RB / 64, DB = D / 16, EPC = 16 / (int)sizeof(T);
    constexpr int WAVE_B = kKeys * RB;
    static_assert(WAVE_B >= 16 * D * 4, "a wave's sums fit its tile");
    __shared__ __attribute__((aligned(16))) char lds[4 * WAVE_B];
    __shared__ float ml[4][2][16];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int i = lane & 15, g = lane >> 4;
    const int part = blockIdx.x % ns;
    int u = blockIdx.x / ns;
    const int qt = u % qtiles; u /= qtiles;
    const int kvh = u % w.Hkv, b = ranked ? longest_first(w, u / w.Hkv, lane) : u / w.Hkv, group = w.H / w.Hkv;
    const int heads = min(16, group - 16 * qt);                       // query heads of this workgroup
    const int head0 = kvh * group + 16 * qt;

    const Seen sn = seen_of(w.lens[b], c.width * (int)c.page.d, w.window, w.sinks);
    const int per = sn.ntiles / ns, more = sn.ntiles - per * ns;       // the first `more` shares have a tile more
    const int t0 = per * part + min(part, more), t1 = t0 + per + (part < more ? 1 : 0);

    frag qf[KS];
    {
        const T* qp = Qg + b * w.qs[0] + (int64_t)(head0 + min(i, heads - 1)) * w.qs[1];
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int col = (4 * s + g) * EPC;
            qf[s] = frag{};
            if (col < w.d && i < heads) qf[s] = *reinterpret_cast<const frag*>(qp + col);
        }
    }
    const float sl2 = w.scale * kLog2eP;
    const int* row_table = c.table + (int64_t)b * c.width;
    char* vt = lds + wave * WAVE_B;

    // Where keys i and 16 + i of a tile stand: looked up one tile ahead of the loads that need it, so that a tile's
    // time does not hold the table's latency and then the cache's.
    int page[2], slot[2];                       // page -1: a key that is not seen
    auto look_up = [&](int t) __attribute__((always_inline)) {
        const int k0 = (t < sn.n_sink ? t : t - sn.n_sink + sn.t_win) * kKeys;
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
            const int key = k0 + 16 * blk + i;
            page[blk] = -1;
            if ((key < sn.len) & ((key >= sn.lo) | (key < w.sinks))) {
                const int pi = (int)c.page.div((uint32_t)key);
                slot[blk] = key - pi * (int)c.page.d;
                const int at = row_table[pi];
                page[blk] = at == -1 ? -2 : at;
            }
        }
    };
    // K and V rows i and 16 + i of the tile looked up, chunks 4 s + g.  Keys that are not seen are zeros (V) and
    // masked below (K); a key whose page number is not of the pool is NaN, so that its sequence's result is.
    u32x4 kr[2][KS], vr[2][KS];
    auto load = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
            const bool ok = (page[blk] >= 0) & (page[blk] < c.num_pages);
            const char* kp = c.k + page[blk] * c.kst[0] + kvh * c.kst[1] + slot[blk] * c.kst[2];
            const char* vp = c.v + page[blk] * c.vst[0] + kvh * c.vst[1] + slot[blk] * c.vst[2];
            const unsigned fill = page[blk] != -1 && !ok ? 0x7FFF7FFFu : 0u;      // a NaN in all three types
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int at = (4 * s + g) * 16;
                kr[blk][s] = u32x4{fill, fill, fill, fill};
                vr[blk][s] = u32x4{0, 0, 0, 0};
                if (ok && at < c.row_bytes) {
                    kr[blk][s] = *reinterpret_cast<const u32x4*>(kp + at);
                    vr[blk][s] = *reinterpret_cast<const u32x4*>(vp + at);
                }
            }
        }
    };

    f32x4 o[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    const int tq = (lane & 15) >> 2, tp = lane & 3;

    int t = t0 + wave;
    if (t < t1) { look_up(t); load(); }
    if (t + 4 < t1) look_up(t + 4);
    for (; t < t1; t += 4) {
        const int k0 = (t < sn.n_sink ? t : t - sn.n_sink + sn.t_win) * kKeys;
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int row = 16 * blk + i;
                *reinterpret_cast<u32x4*>(vt + row * RB + ((64 * s + 16 * g) ^ v_swz<RB>(row))) = vr[blk][s];
            }
        f32x4 sc[2];
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
            sc[blk] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < KS; ++s) sc[blk] = mma16_chunk<T>(__builtin_bit_cast(frag, kr[blk][s]), qf[s], sc[blk]);
        }
        if (t + 4 < t1) load();
        if (t + 8 < t1) look_up(t + 8);

        // lane (i, g): head i, keys k0 + 16 blk + 4 g + r
        const bool edge = k0 + kKeys > sn.len || (k0 < sn.lo && k0 + kKeys > w.sinks);
        float mx = -INFINITY;
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int key = k0 + 16 * blk + 4 * g + r;
                float x = sc[blk][r] * sl2;
                if (edge && !((key < sn.len) & ((key >= sn.lo) | (key < w.sinks)))) x = -INFINITY;
                sc[blk][r] = x;
                mx = fmaxf(mx, x);
            }
        if (scores != nullptr && i < heads) {
            float* sp = scores + ((int64_t)b * w.H + head0 + i) * score_row + k0 + 4 * g;
            *reinterpret_cast<f32x4*>(sp) = sc[0];
            *reinterpret_cast<f32x4*>(sp + 16) = sc[1];
        }
        mx = four_rows_allreduce(mx, MaxOp{});
        const float m_new = fmaxf(m, mx);
        const float ref = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = __builtin_amdgcn_exp2f(m - ref);
        m = m_new;
        float ps = 0.f;
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                sc[blk][r] = __builtin_amdgcn_exp2f(sc[blk][r] - ref);
                ps += sc[blk][r];
            }
        l = l * alpha + ps;
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db] *= alpha;

        asm volatile("" ::: "memory");
        if constexpr (sizeof(T) == 2) {
            typename Mma16<T>::vec8 p;
#pragma unroll
            for (int r = 0; r < 4; ++r) { p[r] = (T)sc[0][r]; p[4 + r] = (T)sc[1][r]; }
            const int row = 4 * g + tq, swz = v_swz<RB>(row);
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                const char* at = vt + row * RB + ((32 * db + 16 * (tp >> 1)) ^ swz) + 8 * (tp & 1);
                const s16x4 x = lds_read_tr(at), y = lds_read_tr(at + 16 * RB);
                s16x8 a;
                a[0] = x[0]; a[1] = x[1]; a[2] = x[2]; a[3] = x[3];
                a[4] = y[0]; a[5] = y[1]; a[6] = y[2]; a[7] = y[3];
                o[db] = Mma16<T>::run(a, p, o[db]);
            }
        } else {
#pragma unroll
            for (int blk = 0; blk < 2; ++blk)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 16 * blk + 4 * g + r, swz = v_swz<RB>(row);
#pragma unroll
                    for (int db = 0; db < DB; ++db) {
                        const float a = *reinterpret_cast<const float*>(vt + row * RB + ((64 * db + 16 * (i >> 2)) ^ swz) + 4 * (i & 3));
                        o[db] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, sc[blk][r], o[db], 0, 0, 0);
                    }
                }
        }
        asm volatile("" ::: "memory");
    }

    // ---- the four waves' sums: lane (i, g) holds columns 16 db + 4 g + r of head i
    l = four_rows_allreduce(l, SumOp{});
    if (sn.past) l = __builtin_nanf("");
    if (g == 0) { ml[wave][0][i] = m; ml[wave][1][i] = l; }
    float* ot = reinterpret_cast<float*>(vt);
#pragma unroll
    for (int db = 0; db < DB; ++db) *reinterpret_cast<f32x4*>(ot + i * D + 16 * db + 4 * g) = o[db];
    __syncthreads();
    for (int e = tid; e < heads * (D / 4); e += 256) {
        const int hd = e / (D / 4), col = (e - hd * (D / 4)) * 4;
        float top = ml[0][0][hd];
#pragma unroll
        for (int x = 1; x < 4; ++x) top = fmaxf(top, ml[x][0][hd]);
        const float ref = top == -INFINITY ? 0.f : top;
        float total = 0.f;
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const float f = __builtin_amdgcn_exp2f(ml[x][0][hd] - ref);
            total += f * ml[x][1][hd];
            sum += f * *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + x * WAVE_B) + hd * D + col);
        }
        const int64_t bh = (int64_t)b * w.H + head0 + hd;
        if (col == 0 && part_ml != nullptr) {
            part_ml[(bh * ns + part) * 2] = top;
            part_ml[(bh * ns + part) * 2 + 1] = total;
        }
        if (ns > 1) {
            *reinterpret_cast<f32x4*>(part_o + (bh * ns + part) * D + col) = sum;
        } else {
            const bool any = (sn.len > 0) | sn.past;             // (past: NaN, with a table of no pages too)
            const float inv = any ? 1.f / total : 0.f;
            typedef T vec4 __attribute__((ext_vector_type(4)));
            vec4 y;
#pragma unroll
            for (int r = 0; r < 4; ++r) y[r] = any ? (T)(sum[r] * inv) : (T)0.f;
            if (col < w.d) *reinterpret_cast<vec4*>(Og + bh * w.d + col) = y;
            if (col == 0 && LSEg != nullptr) LSEg[bh] = any ? (top + __builtin_amdgcn_logf(total)) * kLn2P : -INFINITY;
        }
    }
}

// Maximum and sum of a head over its ns shares; the lanes of a wave take them in turn and all get the result.
struct TopSum { float top, ref, total; };
__device__ __forceinline__ TopSum join_ml(const float* ml, int ns, int lane) {
    TopSum j{-INFINITY, 0.f, 0.f};
    for (int s = lane; s < ns; s += 64) j.top = fmaxf(j.top, ml[2 * s]);
    j.top = wave_max(j.top);
    j.ref = j.top == -INFINITY ? 0.f : j.top;
    for (int s = lane; s < ns; s += 64) j.total += __builtin_amdgcn_exp2f(ml[2 * s] - j.ref) * ml[2 * s + 1];
    j.total = wave_sum(j.total);
    return j;
}

// Workgroups [0, njoin): one query head each (none where every head had one share); D / 4 threads take a share's
// columns, the workgroup's groups of so many every share in turn, and their sums meet in LDS in order.  The others:
// 1024 keys of one key/value head, four per thread.
template <typename T>
__global__ void __launch_bounds__(256)
paged_join_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml, const float* __restrict__ scores,
                  T* __restrict__ Og, float* __restrict__ LSEg, float* __restrict__ weight_sum, DecodeShape w,
                  int cap, int ns, int D, int njoin, int nchunk, int64_t score_row) {
    __shared__ __attribute__((aligned(16))) float lds[1024];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if ((int)blockIdx.x < njoin) {
        const int64_t bh = blockIdx.x;
        const int len = w.lens[bh / w.H];
        const float* ml = part_ml + bh * ns * 2;
        const TopSum j = join_ml(ml, ns, lane);
        const int tpg = D / 4, grp = tid / tpg, groups = 256 / tpg, col = 4 * (tid - grp * tpg);
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int s = grp; s < ns; s += groups)
            sum += __builtin_amdgcn_exp2f(ml[2 * s] - j.ref) * *reinterpret_cast<const f32x4*>(part_o + (bh * ns + s) * D + col);
        *reinterpret_cast<f32x4*>(lds + 4 * tid) = sum;
        __syncthreads();
        if (grp == 0 && col < w.d) {
            for (int g = 1; g < groups; ++g) sum += *reinterpret_cast<const f32x4*>(lds + 4 * (tid + g * tpg));
            const float inv = 1.f / j.total;
            typedef T vec4 __attribute__((ext_vector_type(4)));
            vec4 y;
#pragma unroll
            for (int r = 0; r < 4; ++r) y[r] = len > 0 ? (T)(sum[r] * inv) : (T)0.f;
            *reinterpret_cast<vec4*>(Og + bh * w.d + col) = y;
            if (col == 0 && LSEg != nullptr) LSEg[bh] = len > 0 ? (j.top + __builtin_amdgcn_logf(j.total)) * kLn2P : -INFINITY;
        }
        return;
    }
    const int u = blockIdx.x - njoin;
    const int chunk = u % nchunk, bg = u / nchunk;
    const int b = bg / w.Hkv, kvh = bg - b * w.Hkv, group = w.H / w.Hkv;
    const Seen sn = seen_of(w.lens[b], cap, w.window, w.sinks);
    // chunks of the tiles that the first launch went through, as they follow each other there
    const int vt = chunk * 32 + (tid >> 3);
    if (chunk * 32 >= sn.ntiles) return;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    const int key = (vt < sn.n_sink ? vt : vt - sn.n_sink + sn.t_win) * kKeys + (tid & 7) * 4;
    for (int h0 = 0; h0 < group; h0 += 64) {
        const int n = min(64, group - h0);
        __syncthreads();
        for (int x = wave; x < n; x += 4) {
            const TopSum j = join_ml(part_ml + ((int64_t)b * w.H + kvh * group + h0 + x) * ns * 2, ns, lane);
            if (lane == 0) lds[x] = j.top + __builtin_amdgcn_logf(j.total);
        }
        __syncthreads();
        if (vt < sn.ntiles)
#pragma unroll 4
            for (int x = 0; x < n; ++x) {
                const f32x4 s = *reinterpret_cast<const f32x4*>(scores + ((int64_t)b * w.H + kvh * group + h0 + x) * score_row + key);
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] += __builtin_amdgcn_exp2f(s[e] - lds[x]);
            }
    }
    if (vt < sn.ntiles) {
        float* out = weight_sum + (int64_t)bg * cap;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (key + e < sn.len && (key + e >= sn.lo || key + e < w.sinks)) out[key + e] += sum[e];
    }
}

// ---------------------------------------------------------------- append
// One thread per 16-byte chunk of a new key and the same chunk of its value.
__global__ void __launch_bounds__(256)
paged_append_kernel(const char* __restrict__ kn, const char* __restrict__ vn, char* __restrict__ kc, char* __restrict__ vc,
                    PagedCache c, AppendShape a, FastDiv cpr, FastDiv tokens, FastDiv heads, uint32_t total) {
    const uint32_t u = blockIdx.x * 256u + threadIdx.x;
    if (u >= total) return;
    const uint32_t row = cpr.div(u), ch = u - row * cpr.d;
    const uint32_t bh = tokens.div(row), x = row - bh * tokens.d;
    const uint32_t b = heads.div(bh), h = bh - b * heads.d;
    const int64_t at = (int64_t)a.lens[b] + x;
    if (a.counts != nullptr && (int)x >= a.counts[b]) return;
    if (at < 0 || at >= (int64_t)c.width * c.page.d) return;
    const uint32_t pi = c.page.div((uint32_t)at), slot = (uint32_t)at - pi * c.page.d;
    const int page = c.table[(int64_t)b * c.width + pi];
    if (page < 0 || page >= c.num_pages) return;
    const u32x4 kx = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kn + b * a.ks[0] + h * a.ks[1] + x * a.ks[2] + ch * 16));
    const u32x4 vx = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(vn + b * a.vs[0] + h * a.vs[1] + x * a.vs[2] + ch * 16));
    *reinterpret_cast<u32x4*>(kc + page * c.kst[0] + h * c.kst[1] + slot * c.kst[2] + ch * 16) = kx;
    *reinterpret_cast<u32x4*>(vc + page * c.vst[0] + h * c.vst[1] + slot * c.vst[2] + ch * 16) = vx;
}

// ---------------------------------------------------------------- host
int pad_dim(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

struct DecodePlan { int ns, D, qtiles; bool ranked; int64_t score_row, ml_floats, o_floats, score_floats; };

// Shares per head: enough workgroups that the chip is full several times over (the lengths are on the device, and
// sequences differ), as long as every wave of a share has two tiles of the longest possible sequence; one share where
// its waves have four tiles or fewer, which saves the second launch.  Measured (us, workgroups aimed at 1024 / 2048 /
// 4096 / 8192): 8 sequences up to 131072 keys 499 / 505 / 485 / 503, 64 up to 4096 171 / 157 / 153 / 157; tiles per
// wave 1 / 2 / 4 / 8: one sequence of 1024 keys 12.3 / 12.7 / 17.1 / 23.2; at most 300 keys, split / not: 12.7 / 10.3.
// Sequences go longest first (batches of up to a wave's lanes) where a share of the longest possible one is long: measured, as they
// come / longest first, tiles a share: 16 sequences of up to 32768 keys 235 / 220 (32), 64 of 8192 212 / 202 (32), 32 of 16384
// 219 / 209 (32), 8 of 131072 484 / 476 (64); 64 of 4096 with weights 157 / 160 (16), 32 of 4096 52 / 59 (8: a tail of short ones).
DecodePlan decode_plan(const DecodeShape& w, int64_t cap, bool weights) {
    DecodePlan p;
    p.D = pad_dim(w.d);
    p.qtiles = (int)cdiv(w.H / w.Hkv, 16);
    const int64_t base = (int64_t)w.B * w.Hkv * p.qtiles;
    int64_t seen = cap;
    if ((int64_t)w.window + w.sinks < cap) seen = (int64_t)w.window + w.sinks;
    const int64_t tiles = cdiv(seen, kKeys), most = tiles <= 16 ? 1 : cdiv(tiles, 8);
    int64_t ns = cdiv(4096, base > 0 ? base : 1);
    if (ns > most) ns = most;
    if (ns > 128) ns = 128;
    p.ns = (int)(ns < 1 ? 1 : ns);
    p.ranked = w.B > 1 && w.B <= 64 && tiles / p.ns >= 32;
    const int64_t bh = (int64_t)w.B * w.H;
    p.score_row = weights ? cdiv(cap, kKeys) * kKeys : 0;
    p.ml_floats = p.ns > 1 || weights ? cdiv(bh * p.ns * 2, 4) * 4 : 0;
    p.o_floats = p.ns > 1 ? bh * p.ns * p.D : 0;
    p.score_floats = bh * p.score_row;
    return p;
}

template <typename T>
int launch_decode(const void* q, const PagedCache& c, void* o, float* lse, float* weight_sum, float* ws, const DecodeShape& w, hipStream_t s) {
    const int cap = c.width * (int)c.page.d;
    const DecodePlan p = decode_plan(w, cap, weight_sum != nullptr);
    const int64_t nwg = (int64_t)w.B * w.Hkv * p.qtiles * p.ns;
    const int nchunk = weight_sum ? (int)cdiv(cdiv(cap, kKeys) + 1, 32) : 0;
    const int64_t njoin = p.ns > 1 ? (int64_t)w.B * w.H : 0, nw = (int64_t)w.B * w.Hkv * nchunk;
    if (nwg > 0x7fffffff || njoin + nw > 0x7fffffff) return fail(MYFA_E_UNSUPPORTED, "paged attention: too many workgroups");
    float* ml = p.ml_floats ? ws + p.o_floats : nullptr;
    float* scores = weight_sum ? ws + p.o_floats + p.ml_floats : nullptr;
    auto go = [&](auto kern) {
        launch_kernel(kern, dim3((unsigned)nwg), dim3(256), 0, s, static_cast<const T*>(q), c, static_cast<T*>(o), lse, w,
                      p.qtiles, p.ns, p.ranked, ws, ml, scores, p.score_row);
    };
    if (p.D == 64) go(paged_decode_kernel<T, 64>);
    else if (p.D == 128) go(paged_decode_kernel<T, 128>);
    else if constexpr (sizeof(T) == 2) go(paged_decode_kernel<T, 256>);
    if (njoin + nw > 0)
        launch_kernel(paged_join_kernel<T>, dim3((unsigned)(njoin + nw)), dim3(256), 0, s, ws, ml, scores, static_cast<T*>(o), lse,
                      weight_sum, w, cap, p.ns, p.D, (int)njoin, nchunk, p.score_row);
    return check_launch("paged attention");
}

}  // namespace

int64_t paged_decode_ws_bytes(const DecodeShape& w, int64_t cap, bool weights) {
    const DecodePlan p = decode_plan(w, cap, weights);
    return (p.o_floats + p.ml_floats + p.score_floats) * 4;
}

int paged_decode(const void* q, const PagedCache& c, void* o, float* lse, float* weight_sum, float* ws, const DecodeShape& w,
                 int dtype, hipStream_t s) {
    if (dtype == MYFA_F32) return launch_decode<float>(q, c, o, lse, weight_sum, ws, w, s);
    if (dtype == MYFA_F16) return launch_decode<_Float16>(q, c, o, lse, weight_sum, ws, w, s);
    return launch_decode<__bf16>(q, c, o, lse, weight_sum, ws, w, s);
}

int paged_append(const void* k, const void* v, const PagedCache& c, const AppendShape& a, hipStream_t s) {
    const int64_t total = (int64_t)a.B * a.Hkv * a.n * (c.row_bytes / 16);
    if (total > 0x7fffff00) return fail(MYFA_E_UNSUPPORTED, "paged append: %lld chunks of 16 bytes in one call", (long long)total);
    launch_kernel(paged_append_kernel, dim3((unsigned)cdiv(total, 256)), dim3(256), 0, s, static_cast<const char*>(k),
                  static_cast<const char*>(v), const_cast<char*>(c.k), const_cast<char*>(c.v), c, a,
                  FastDiv((uint32_t)(c.row_bytes / 16)), FastDiv((uint32_t)a.n), FastDiv((uint32_t)a.Hkv), (uint32_t)total);
    return check_launch("paged append");
}

}  // namespace myfa
