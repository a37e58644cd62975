// Pieces shared by the paged cache kernels.
//
// A cache is a pool of pages [pages, heads, page, d]: a page holds `page` consecutive keys of every head,
// so that one head's keys of a page are one contiguous piece for the workgroup that reads them.  A sequence
// is a row of a table of page numbers; key j of sequence b stands in page table[b, j / page], slot j % page.
// Page numbers are checked by every kernel before they become addresses: a key whose page number is outside
// the pool is never read or written.
#ifndef MYFA_PAGED_COMMON_H_
#define MYFA_PAGED_COMMON_H_
#include "attn_mfma_common.h"

namespace myfa {

// x / d for 0 <= x < 2^31 by one multiplication (d a run-time constant of the launch): with
// s = ceil(log2 d), m = ceil(2^(31+s) / d) < 2^32 and e = m d - 2^(31+s) < d <= 2^s, so
// x m / 2^(31+s) = x / d + x e / (d 2^(31+s)), whose excess is below 1 / d for x < 2^31.
struct FastDiv {
    uint32_t d, m, s;
    FastDiv() = default;
    explicit FastDiv(uint32_t dd) : d(dd) {
        s = 0;
        while ((1ull << s) < dd) ++s;
        m = (uint32_t)(((1ull << (31 + s)) + dd - 1) / dd);
    }
    __device__ __forceinline__ uint32_t div(uint32_t x) const { return (uint32_t)(((uint64_t)x * m) >> (31 + s)); }
};

struct PagedCache {
    const char *k, *v;
    int64_t kst[3], vst[3];            // strides of page, head, slot, in bytes
    const int* table;                  // [B, width]
    int num_pages, width, row_bytes;   // row_bytes = d * sizeof(T)
    FastDiv page;
};

struct DecodeShape {
    int B, H, Hkv, d;
    int window, sinks;
    float scale;
    const int* lens;                  // [B]
    int64_t qs[2];                    // strides of q: batch, head, in elements
};

struct AppendShape {
    int B, Hkv, n;
    int64_t ks[3], vs[3];             // strides of the new keys and values: batch, head, token, in bytes
    const int* lens;                  // [B]: where the new tokens begin
    const int* counts;                // [B] or null: how many of the n tokens
};

struct EvictShape {
    int B, Hkv, cap, new_cap, budget, sinks, recent;
    const int* lens;                  // [B]
    const float* sums;                // [B, Hkv, cap]
    float* new_sums;                  // [B, Hkv, new_cap]
    int* new_lens;                    // [B]
    int* kept;                        // [B, Hkv, budget]
    const int* new_table;             // [B, new_cap / page]
};

}  // namespace myfa
#endif  // MYFA_PAGED_COMMON_H_
