// Eviction from a paged cache by accumulated attention weight.
//
// Of a sequence longer than the budget every key/value head keeps its first `sinks` keys, its last `recent`
// keys and, of those between, the ones with the largest sums of attention weights (what paged attention adds
// up per key; equal sums: the lowest index; NaN counts as larger than everything).  The kept keys, values and
// sums go, in the order they had, to the pages of another table.  Shorter sequences are copied whole.
//
// Two launches.  The first finds, per head, the m-th largest sum exactly by a radix selection over the
// ordered bit patterns (digits of 11, 11 and 10 bits: the first holds sign, exponent and two bits of the
// mantissa, which spreads the counts of real sums over many bins), then walks the keys once in order and
// gives each kept one its place by a prefix sum.  Reading the sums is its floor, 4 bytes a key, and with one
// workgroup per head its passes are bound by latency.  The second copies rows in 16-byte chunks, as many
// threads as chunks: bound by memory, 2 d elements read and written a key.  With few kept keys the first does it all.
// Measured, d 128, bf16: 16 sequences of up to 8192 keys and 8 heads to 2048 keys 70 us: selection 14 (128 workgroups, no more
// work than that to share out), copy 52 (268 MB, 5.1 TB/s); one sequence of 1024 keys to 256, d 64: 8.3 us, one launch.
#include "paged_common.h"

namespace myfa {
namespace {

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64, kBins = 2048, kPer = 4;
constexpr int kMoveChunks = 2048;      // chunks of a head's kept keys that the selecting workgroup moves itself

// Order-preserving map of float32 to uint32; the zeros are one value, NaN is the largest.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) return 0xFFFFFFFFu;
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);        // -0 + 0 = +0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Inclusive prefix sum over the workgroup's threads; `total` is everyone's.  A barrier first and last.
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t* waves, uint32_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t y = __shfl_up(x, d);
        if (lane >= d) x += y;
    }
    __syncthreads();
    if (lane == 63) waves[wave] = x;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < kSelWaves; ++i) {
        if (i < wave) before += waves[i];
        total += waves[i];
    }
    return x + before;
}

// Chunk `ch` of a kept key and of its value: from its old place to its new one.  A kept key whose old page number is not of
// the pool becomes NaN; one whose new page number is not is dropped.
__device__ __forceinline__ void move_chunk(const PagedCache& c, const EvictShape& e, uint32_t b, uint32_t h, uint32_t from, uint32_t to, uint32_t ch) {
    const uint32_t po = c.page.div(from), so = from - po * c.page.d;
    const uint32_t pn = c.page.div(to), sn = to - pn * c.page.d;
    const int old_page = c.table[(int64_t)b * c.width + po];
    const int new_page = e.new_table[(int64_t)b * (e.new_cap / (int)c.page.d) + pn];
    if (new_page < 0 || new_page >= c.num_pages) return;
    u32x4 kx = {0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu}, vx = kx;
    if (old_page >= 0 && old_page < c.num_pages) {
        kx = *reinterpret_cast<const u32x4*>(c.k + old_page * c.kst[0] + h * c.kst[1] + so * c.kst[2] + ch * 16);
        vx = *reinterpret_cast<const u32x4*>(c.v + old_page * c.vst[0] + h * c.vst[1] + so * c.vst[2] + ch * 16);
    }
    *reinterpret_cast<u32x4*>(const_cast<char*>(c.k) + new_page * c.kst[0] + h * c.kst[1] + sn * c.kst[2] + ch * 16) = kx;
    *reinterpret_cast<u32x4*>(const_cast<char*>(c.v) + new_page * c.vst[0] + h * c.vst[1] + sn * c.vst[2] + ch * 16) = vx;
}

// PER > 0: a thread holds up to PER consecutive sums of the row in registers (rows of up to PER * 1024 keys); PER = 0: the
// row is read again in every pass.  MOVE: the kept keys are few and go to their new places here.
template <int PER, bool MOVE>
__global__ void __launch_bounds__(kSelThreads)
paged_evict_select_kernel(EvictShape e, PagedCache c, FastDiv cpr) {
    __shared__ uint32_t hist[kBins], waves[kSelWaves], found[3];
    __shared__ uint32_t places[MOVE ? kMoveChunks : 1];
    const int bg = blockIdx.x, b = bg / e.Hkv, tid = threadIdx.x;
    const int len = min(max(e.lens[b], 0), e.cap), keep = min(len, e.budget);
    const float* sums = e.sums + (int64_t)bg * e.cap;
    float* new_sums = e.new_sums + (int64_t)bg * e.new_cap;
    int* kept = e.kept + (int64_t)bg * e.budget;

    constexpr int HELD = PER > 0 ? PER : kPer;
    const int per = PER > 0 ? (len + kSelThreads - 1) / kSelThreads : kPer;       // consecutive keys of a thread
    float x[HELD];
    auto read = [&](int i0) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < HELD; ++j) {
            const int i = i0 + tid * per + j;
            x[j] = j < per && i < len ? sums[i] : 0.f;
        }
    };
    if constexpr (PER > 0) read(0);

    // the middle's m largest: keys above `limit`, and the first `quota` that equal it
    const bool all = len <= e.budget;
    const int first = e.sinks, last = len - e.recent;
    uint32_t quota = all ? 0 : e.budget - e.sinks - e.recent, limit = 0;
    if (!all && quota > 0) {
        int shift = 32;
#pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
            const int bits = pass < 2 ? 11 : 10;
            const uint32_t above = limit;                              // the digits found so far
            shift -= bits;
            for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
            __syncthreads();
            auto count = [&](float v) __attribute__((always_inline)) {
                const uint32_t k = order_key(v);
                if (pass == 0 || (k >> (shift + bits)) == above) atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1)], 1u);
            };
            if constexpr (PER > 0) {
#pragma unroll
                for (int j = 0; j < HELD; ++j) {
                    const int i = tid * per + j;
                    if (j < per && i >= first && i < last) count(x[j]);
                }
            } else {
                for (int i = first + tid; i < last; i += kSelThreads) count(sums[i]);
            }
            __syncthreads();
            // from the largest digit down: the digit in which the count reaches the quota
            const int hi = kBins - 1 - 2 * tid;
            const uint32_t c0 = hist[hi], c1 = hist[hi - 1];
            uint32_t total;
            const uint32_t upto = block_scan(c0 + c1, waves, total), before = upto - c0 - c1;
            if (before < quota && quota <= upto) {
                const bool second = before + c0 < quota;
                found[0] = (uint32_t)(second ? hi - 1 : hi);
                found[1] = quota - before - (second ? c0 : 0u);
                found[2] = second ? c1 : c0;
            }
            __syncthreads();
            limit = (above << bits) | found[0];
            quota = found[1];
            const bool whole = quota == found[2];                      // the digit's keys are all among them: no more digits
            __syncthreads();
            if (whole) {                                               // (the least key is -infinity's 0x007FFFFF: no wrap)
                limit = (limit << shift) - 1;
                quota = 0;
                break;
            }
        }
    }
    const bool none = !all && e.budget - e.sinks - e.recent == 0;

    // places, in order: `sure` keys and equal keys counted together, 16 bits each
    uint32_t base_sure = 0, base_tie = 0;
    for (int i0 = 0; i0 < len; i0 += kSelThreads * per) {
        if constexpr (PER == 0) read(i0);
        uint32_t sure = 0, tie = 0, mine = 0;
#pragma unroll
        for (int j = 0; j < HELD; ++j) {
            const int i = i0 + tid * per + j;
            bool s = j < per && i < len, t = false;
            if (s && !all && i >= first && i < last) {
                const uint32_t k = order_key(x[j]);
                s = !none && k > limit;
                t = !none && k == limit;
            }
            sure |= (uint32_t)s << j;
            tie |= (uint32_t)t << j;
            mine += (uint32_t)s + ((uint32_t)t << 16);
        }
        uint32_t total;
        const uint32_t before = block_scan(mine, waves, total) - mine;
        uint32_t ns = base_sure + (before & 0xFFFFu), nt = base_tie + (before >> 16);
#pragma unroll
        for (int j = 0; j < HELD; ++j) {
            const bool s = (sure >> j) & 1, t = (tie >> j) & 1;
            if (s || (t && nt < quota)) {
                const uint32_t at = ns + min(nt, quota);
                kept[at] = i0 + tid * per + j;
                new_sums[at] = x[j];
                if constexpr (MOVE) places[at] = i0 + tid * per + j;
            }
            ns += s;
            nt += t;
        }
        base_sure += total & 0xFFFFu;
        base_tie += total >> 16;
    }
    for (int i = keep + tid; i < e.budget; i += kSelThreads) kept[i] = -1;
    for (int i = keep + tid; i < e.new_cap; i += kSelThreads) new_sums[i] = 0.f;
    if (tid == 0 && bg % e.Hkv == 0) e.new_lens[b] = keep;
    if constexpr (MOVE) {
        __syncthreads();
        for (uint32_t u = tid; u < keep * cpr.d; u += kSelThreads) {
            const uint32_t to = cpr.div(u);
            move_chunk(c, e, b, bg - b * e.Hkv, places[to], to, u - to * cpr.d);
        }
    }
}

// One thread per 16-byte chunk of a kept key and the same chunk of its value.
__global__ void __launch_bounds__(256)
paged_evict_move_kernel(PagedCache c, EvictShape e, FastDiv cpr, FastDiv budget, FastDiv heads, uint32_t total) {
    const uint32_t u = blockIdx.x * 256u + threadIdx.x;
    if (u >= total) return;
    const uint32_t row = cpr.div(u), ch = u - row * cpr.d;
    const int from = e.kept[row];
    if (from < 0) return;
    const uint32_t bh = budget.div(row), to = row - bh * budget.d;
    const uint32_t b = heads.div(bh), h = bh - b * heads.d;
    move_chunk(c, e, b, h, (uint32_t)from, to, ch);
}

}  // namespace

int paged_evict(const PagedCache& c, const EvictShape& e, hipStream_t s) {
    const int64_t rows = (int64_t)e.B * e.Hkv * e.budget, total = rows * (c.row_bytes / 16);
    if (total > 0x7fffff00) return fail(MYFA_E_UNSUPPORTED, "paged eviction: %lld chunks of 16 bytes in one call", (long long)total);
    const uint32_t chunks = c.row_bytes / 16;
    const FastDiv cpr(chunks > 0 ? chunks : 1);
    auto select = [&](auto kern) { launch_kernel(kern, dim3((unsigned)(e.B * e.Hkv)), dim3(kSelThreads), 0, s, e, c, cpr); };
    // One launch while a head's kept keys are few.  Measured (us, one launch / two), chunks a head: 8 heads 2048 8.4 / 9.9,
    // 4096 9.9 / 10.1, 8192 13.2 / 10.4; 32 heads 4096 10.9 / 10.5, 8192 14.7 / 11.4; 512 heads 4096 31.6 / 34.0.
    if (chunks > 0 && (int64_t)e.budget * chunks <= kMoveChunks && e.cap <= 8 * kSelThreads) {
        if (e.cap <= 2 * kSelThreads) select(paged_evict_select_kernel<2, true>);
        else select(paged_evict_select_kernel<8, true>);
        return check_launch("paged eviction");
    }
    if (e.cap <= 2 * kSelThreads) select(paged_evict_select_kernel<2, false>);
    else if (e.cap <= 8 * kSelThreads) select(paged_evict_select_kernel<8, false>);
    else if (e.cap <= 16 * kSelThreads) select(paged_evict_select_kernel<16, false>);
    else select(paged_evict_select_kernel<0, false>);
    if (total > 0)
        launch_kernel(paged_evict_move_kernel, dim3((unsigned)cdiv(total, 256)), dim3(256), 0, s, c, e, cpr,
                      FastDiv((uint32_t)e.budget), FastDiv((uint32_t)e.Hkv), (uint32_t)total);
    return check_launch("paged eviction");
}

}  // namespace myfa
