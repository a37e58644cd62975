// Pieces shared by the window attention kernels (forward and backward): the shape record, what a query
// sees, and the products of a 32-row block with an LDS tile, for 16-bit and float32 elements alike.
//
// What a query sees.  Query i of a sequence stands at position p = i + Nk - Nq.  It sees key j when
//     j <= p  and  p < len  and  ( p - j < window  or  j < sinks ),
// len being the sequence's length (Nk where the caller gives none).  A position p >= len sees nothing.
//
// Fragments.  Both element types move through the matrix cores in 16-byte chunks: a lane's chunk is the
// A or B operand of one v_mfma_f32_32x32x16 (16-bit) or of four v_mfma_f32_32x32x2_f32, one per element,
// where the two lane halves hold chunk 2s and 2s + 1 of the row, i.e. the k index of MFMA e of step s is
// column 8s + 4h + e on both operands.  The accumulator layout is the same: lane (r = l & 31, h = l >> 5)
// holds column r and rows 8 (i >> 2) + 4 h + (i & 3), i = 0..15.
#ifndef MYFA_WINDOW_ATTN_COMMON_H_
#define MYFA_WINDOW_ATTN_COMMON_H_
#include "attn_mfma_common.h"

namespace myfa {

struct WindowShape {
    int B, H, Hkv, Nq, Nk, d;
    int window, sinks;                 // both clamped to Nk
    float scale;
    const int* lens;                   // [B] or null
    int64_t qs[3], ks[3], vs[3];       // strides of batch, head, row, in elements
};

namespace {

constexpr float kLog2eW = 1.4426950408889634f;
constexpr float kLn2W = 0.6931471805599453f;
// Fetches of rows or columns that are not there use this offset: behind every buffer's end, answered
// with zeros without touching memory.  In-tile offsets stay below kTileBytesMax (checked by the host).
constexpr int kOffPast = 0x7FFF0000;
constexpr int kTileBytesMax = 0x7FFE0000;

template <typename T> struct Frag16 { using type = s16x8; };
template <> struct Frag16<float> { using type = f32x4; };

// c += a b over one 16-byte chunk per lane
template <typename T>
__device__ __forceinline__ f32x16 mma_chunk(typename Frag16<T>::type a, typename Frag16<T>::type b, f32x16 c) {
    if constexpr (sizeof(T) == 2) {
        return Mma<T>::run(a, __builtin_bit_cast(typename Mma<T>::vec8, b), c);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
}

// The per-lane bases of the reads from a [rows][D] tile image (8-row x 64-byte subtiles, see img_off):
// row chunks, and the transposed operand whose k index runs over the tile's rows.
template <typename T, int D> struct TileReader {
    static constexpr int RB = D * (int)sizeof(T);      // bytes of a row
    static constexpr int SUB = 8 * RB;                 // bytes of 8 rows
    static constexpr int KS = RB / 32;                 // chunk pairs of a row
    static constexpr int DB = D / 32;
    static constexpr int COLB = sizeof(T) == 2 ? 512 : 1024;   // image bytes between 32-column blocks
    using frag = typename Frag16<T>::type;
    int rb[2], tb[2];

    __device__ __forceinline__ TileReader(int lane) {
        const int r = lane & 31, h = lane >> 5;
        const int tq = (lane & 15) >> 2, tp = lane & 3, tg1 = (lane >> 4) & 1;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            rb[e] = SUB * (r >> 3) + 64 * (r & 7) + 16 * ((2 * e + h) ^ ((r >> 2) & 3));
            if constexpr (sizeof(T) == 2)
                tb[e] = 64 * (4 * h + tq) + 16 * ((2 * tg1 + (tp >> 1)) ^ (2 * e + h)) + 8 * (tp & 1) + SUB * e;
            else
                tb[e] = 512 * (r >> 4) + 256 * h + 16 * (((r >> 2) & 3) ^ (2 * e + h)) + 4 * (r & 3);
        }
    }
    // chunk 2 ks + h of row 32 blk + r
    __device__ __forceinline__ frag row(const char* tile, int blk, int ks) const {
        return *reinterpret_cast<const frag*>(tile + rb[ks & 1] + SUB * 4 * blk + 512 * (ks >> 1));
    }
    // 16-bit: the A operand of k-step st of block blk (rows 32 blk + 16 st + ...) and columns 32 db ..
    __device__ __forceinline__ s16x8 transposed(const char* tile, int blk, int st, int db) const {
        const int imm = SUB * 2 * (2 * blk + st) + COLB * db;
        const s16x4 lo = lds_read_tr(tile + tb[0] + imm);
        const s16x4 hi = lds_read_tr(tile + tb[1] + imm);
        s16x8 a;
        a[0] = lo[0]; a[1] = lo[1]; a[2] = lo[2]; a[3] = lo[3];
        a[4] = hi[0]; a[5] = hi[1]; a[6] = hi[2]; a[7] = hi[3];
        return a;
    }
    // acc[db] += tile[rows of blk][32 columns of db]^T x[rows of blk], x an accumulator-shaped block
    // (rounded to T): the accumulator's row index is this product's k index, in place.  `tile` may point
    // at a later column block (COLB bytes each): acc then holds the columns from there on.
    template <int NDB>
    __device__ __forceinline__ void add_transposed(const char* tile, int blk, const f32x16& x, f32x16 (&acc)[NDB]) const {
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                typename Mma<T>::vec8 b;
#pragma unroll
                for (int j = 0; j < 8; ++j) b[j] = (T)x[8 * st + j];
#pragma unroll
                for (int db = 0; db < NDB; ++db) {
                    acc[db] = Mma<T>::run(transposed(tile, blk, st, db), b, acc[db]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
#pragma unroll
                for (int db = 0; db < NDB; ++db) {
                    const float a = *reinterpret_cast<const float*>(tile + tb[(i >> 2) & 1] + SUB * (4 * blk + (i >> 2)) +
                                                                    COLB * db + 64 * (i & 3));
                    acc[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, x[i], acc[db], 0, 0, 0);
                }
        }
    }
};

// Fetches [ROWS][D] tiles straight into LDS (one wave instruction fills 1 KiB of the image, so the image
// is produced by choosing each lane's source chunk).  Columns from d on read as zeros.
template <typename T, int D, int ROWS, int THREADS> struct TileFetch {
    static constexpr int RB = D * (int)sizeof(T), CPR = RB / 16, LPT = ROWS * CPR / THREADS;
    static_assert(LPT >= 1 && ROWS * CPR % THREADS == 0, "every thread fetches whole chunks");
    int off[LPT], row[LPT];
    int wave;
    __device__ __forceinline__ TileFetch(int tid, int64_t row_stride, int d) : wave(__builtin_amdgcn_readfirstlane(tid >> 6)) {
        const int lane = tid & 63;
#pragma unroll
        for (int i = 0; i < LPT; ++i) {
            const int u = 64 * (wave * LPT + i) + lane;
            const int grp8 = u / (RB / 2), within = u % (RB / 2);
            row[i] = 8 * grp8 + ((within & 31) >> 2);
            const int ch = 4 * (within >> 5) + ((within & 3) ^ ((row[i] >> 2) & 3));
            off[i] = ch * (16 / (int)sizeof(T)) < d ? (row[i] * (int)row_stride + ch * (16 / (int)sizeof(T))) * (int)sizeof(T) : kOffPast;
        }
    }
    // piece I of a whole tile: an LDS-DMA instruction takes its wave about 40 cycles to issue, so that pieces dealt one
    // to an MFMA are hidden and several in a row are not
    template <int I> __device__ __forceinline__ void piece(const T* base, char* lds) const {
#if defined(__HIP_DEVICE_COMPILE__)
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, kTileBytesMax, 0x00020000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(lds + 1024 * (wave * LPT + I)), 16, off[I], 0, 0, 0);
#endif
    }
    // rows of the tile for which keep(row) does not hold read as zeros
    template <class Keep>
    __device__ __forceinline__ void fetch(const T* base, char* lds, bool all, Keep&& keep) const {
#if defined(__HIP_DEVICE_COMPILE__)
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, kTileBytesMax, 0x00020000);
#pragma unroll
        for (int i = 0; i < LPT; ++i) {
            const int o = (int)all | (int)keep(row[i]) ? off[i] : kOffPast;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(lds + 1024 * (wave * LPT + i)), 16, o, 0, 0, 0);
        }
#endif
    }
};

// A sequence of MFMAs as one software-pipelined stream: the LDS fragment of step i + FW is requested when
// step i issues (left alone, the scheduler sinks every read to just in front of its MFMA), after(i) runs in
// that MFMA's shadow, and the order is pinned.
template <int N, int FW, class Frag, class Mm, class After>
__device__ __forceinline__ void mma_stream(Frag&& frag, Mm&& mm, After&& after) {
    decltype(frag(IC<0>{})) win[FW];
    static_for<(FW < N ? FW : N)>([&](auto ic) __attribute__((always_inline)) { win[decltype(ic)::value] = frag(ic); });
    __builtin_amdgcn_s_setprio(1);      // the matrix pipe first: 3 % on the forward, 1 % on the backward
    static_for<N>([&](auto ic) __attribute__((always_inline)) {
        constexpr int i = decltype(ic)::value;
        const auto a = win[i % FW];
        mm(ic, a);
        if constexpr (i + FW < N) win[i % FW] = frag(IC<i + FW>{});
        after(ic);
        __builtin_amdgcn_sched_barrier(0);
    });
    __builtin_amdgcn_s_setprio(0);
}

// The wave's own fetches so far are complete / its reads so far are (what it reads may be fetched over).
__device__ __forceinline__ void wave_fetched() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void wave_read() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// Few rows: a workgroup's four waves share 32 rows and deal the tiles among themselves, so that a launch has four
// times the workgroups and each a quarter of the serial work; their float32 sums meet in LDS at the end.  A wave's
// part of LDS holds a pair of 32-row tiles (dK, dV: two pairs where rows are up to 256 bytes), and then its sums
// [32][C], 16-byte chunks swizzled so that eight rows' chunks of one column lie on different banks.  One pair
// leaves room for a second workgroup on the CU, which hides more than a prefetch does (forward bf16 d 128, 128 blocks
// of 128 rows: 11.9 us against 18.0 with two pairs).
template <int C> __device__ __forceinline__ int sum_at(int row, int col) { return row * C + ((col >> 2) ^ (row & 7)) * 4; }
template <int NDB> __device__ __forceinline__ void put_sums(float* to, const f32x16 (&acc)[NDB], int r, int h) {
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<f32x4*>(to + sum_at<32 * NDB>(r, 32 * db + 8 * g + 4 * h)) =
                f32x4{acc[db][4 * g], acc[db][4 * g + 1], acc[db][4 * g + 2], acc[db][4 * g + 3]};
}

// Everyone's fetches so far are complete and everyone has left the tile read before.
__device__ __forceinline__ void tile_ready() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Which query block or unit of keys, and which head, a workgroup takes: rank 0 of every head first.  The launchers
// rank by length, so the short ones fill the end of the launch.  Workgroups go to the XCDs round robin (id mod 8);
// the heads are dealt such that neighbouring ones, which share keys and values, land on one XCD's L2.  Speed only.
struct Ranked { int head, rank; };
__device__ __forceinline__ Ranked ranked(int bid, int heads) {
    const int rank = bid / heads, j = bid - rank * heads;
    return {heads % 8 == 0 ? (j & 7) * (heads >> 3) + (j >> 3) : j, rank};
}

// The keys that `rows` query rows from q0 on see, as tiles of BN keys: n_sink tiles that hold sinks and nothing of any
// window, then those from t_win on.
template <int BN> struct KeyTiles {
    int len, shift, pa, pz, lo, t_win, n_sink, ntiles;      // [pa, pz): the positions of rows that see anything
    __device__ __forceinline__ KeyTiles(const WindowShape& w, int b, int q0, int rows) {
        len = w.lens ? min(max(w.lens[b], 0), w.Nk) : w.Nk;
        shift = w.Nk - w.Nq;
        pa = q0 + shift;
        pz = min(min(q0 + rows, w.Nq) + shift, len);
        lo = max(0, pa - w.window + 1);
        t_win = lo / BN;
        const int t_end = pz > pa ? (pz + BN - 1) / BN : t_win;
        n_sink = pz > pa ? min((min(w.sinks, pz) + BN - 1) / BN, t_win) : 0;
        ntiles = n_sink + (t_end - t_win);
    }
    __device__ __forceinline__ int first_key(int t) const { return (t < n_sink ? t : t - n_sink + t_win) * BN; }
    // every key of the tile is seen by some row (for the fetch), or key k is
    __device__ __forceinline__ bool all(int k0, int sinks) const { return k0 + BN <= pz && (k0 >= lo || k0 + BN <= sinks); }
    __device__ __forceinline__ bool one(int k, int sinks) const { return (k < pz) & ((k >= lo) | (k < sinks)); }
    // the tiles [f0, f1) are seen whole by all `rows` rows
    __device__ __forceinline__ int whole_from(int window, int rows) const {
        return max(n_sink + (max(pa + rows - window, 0) + BN - 1) / BN - t_win, n_sink);
    }
    __device__ __forceinline__ int whole_to(int rows) const { return pz == pa + rows ? n_sink + (pa + 1) / BN - t_win : 0; }
};

// Hides from a lane's row what it does not see of a 32-key block whose accumulator element i is key
// base + 8 (i >> 2) + (i & 3) (base: the block's first key + 4 h).  In a tile that holds only sinks, only keys behind
// them, or one whose row's window reaches the sinks, what it sees is one range: a subtraction, a comparison and
// a select per element.
struct RowSees {
    int p_lo, p_hi;                                          // the row's window; p_hi = -1: a row that sees nothing
    template <int BN>
    __device__ __forceinline__ void hide(f32x16& s, const KeyTiles<BN>& kt, int t, int k0, int base, int sinks, float fill) const {
        const bool sink_tile = t < kt.n_sink;
        if (sink_tile || k0 >= sinks) {
            const int lo = sink_tile ? 0 : p_lo, hi = sink_tile ? min(p_hi, sinks - 1) : p_hi;
            const int from = hi < 0 ? 1 << 30 : lo - base;
            const unsigned span = hi < 0 ? 0u : (unsigned)(hi - lo);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if ((unsigned)(8 * (i >> 2) + (i & 3) - from) > span) s[i] = fill;
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int key = base + 8 * (i >> 2) + (i & 3);
                if (!((key <= p_hi) & ((key >= p_lo) | (key < sinks)))) s[i] = fill;
            }
        }
    }
};

// Whether a launch takes the few-rows kernels: while blocks of 128 rows leave CUs empty; dK, dV fewer of them where
// one of its workgroups fills a CU's LDS (16-bit rows of 256 bytes).  Measured, many / few, in us:
//   forward, bf16 d 64    128 blocks 15.7 / 7.9   192 15.5 / 11.6   256 15.7 / 13.4   512 18.2 / 22.1
//            bf16 d 128    64 blocks 18.9 / 8.7   128 19.6 / 11.9   192 19.7 / 17.7   256 19.9 / 20.6
//            float32 d 64 128 blocks 43.1 / 25.3  192 43.1 / 36.6   256 43.8 / 48.0          dQ: alike
//   dK, dV: what few saves of a whole backward, against blocks of 128 keys
//            bf16 d 64     64 blocks 21 of 61     256 -35 to +61    512 3 of 65      1008 -3 of 138
//            bf16 d 128    64 blocks 20 of 84     128 -3 of 76, -28 of 286           512 -27 of 105
//            float32 d 64  64 blocks 168 of 310   256 200 of 1815   512 26 of 298    1008 -6 of 731
// (float32 keeps gaining because the large kernel walks a whole group of heads in one workgroup.)
inline bool few_queries(const WindowShape& w) { return (int64_t)w.B * w.H * cdiv(w.Nq, 128) <= 192; }
inline bool few_keys(const WindowShape& w, int elem_size) {
    return (int64_t)w.B * w.Hkv * cdiv(w.Nk, 128) <= (elem_size == 4 ? 512 : w.d > 64 ? 64 : 192);
}

}  // namespace
}  // namespace myfa
#endif  // MYFA_WINDOW_ATTN_COMMON_H_
