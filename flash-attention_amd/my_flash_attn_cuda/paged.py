"""A paged key/value cache: append, attention of one new token per sequence, eviction by attention weight.

The cache is two pools of pages, k_cache and v_cache (pages, Hkv, page, d): a page holds `page` consecutive keys of
every key/value head.  block_table, int32 (B, width), gives every sequence its pages: key j of sequence b stands in
page block_table[b, j // page], slot j % page; entries behind a sequence's last page are not read.  A sequence
holds at most width * page keys, its capacity.  Lengths and tables stay on the device: no call waits for the GPU,
and every call can be captured into a graph.  Page numbers outside the pool never become addresses.
What a call writes in place (the pools, weight_sum) has every element in memory of its own, and no history for autograd
to keep: expanded views, and in grad mode tensors that require grad, are refused there.
The reference has no cache (csrc/api.cpp:168-192 takes whole matrices).
"""
from ._lib import host as _host


def paged_kv_append(k, v, k_cache, v_cache, block_table, seq_lens, counts=None):
    """Writes n new keys and values per sequence into the cache, in place.

    k, v: (B, Hkv, n, d) of the cache's dtype, any strides with a dense last dimension and rows at multiples of
    16 bytes.  The tokens go to the places seq_lens[b] .. seq_lens[b] + n - 1 of their sequence; with counts, int32
    (B,), only the first counts[b] of them do (padded batches).  seq_lens is not changed: a caller adds n to it.
    A token whose place is outside [0, capacity) or on a page number outside the pool is dropped.  No two tokens
    of a call may have the same place."""
    _host.paged_kv_append(k, v, k_cache, v_cache, block_table, seq_lens, counts)


def paged_attn_decode(q, k_cache, v_cache, block_table, seq_lens, scale=1.0, window=0, sinks=0, weight_sum=None, return_lse=False):
    """Attention of one new token per sequence over its cached keys, its own (place seq_lens[b] - 1) among them.

    q: (B, H, d) of the cache's dtype, H a multiple of Hkv (query head h uses key/value head h // (H // Hkv)).
    window > 0: only the last `window` keys and the first `sinks` are seen; window = 0: all.
    weight_sum: float32 (B, Hkv, capacity), contiguous: the weights of every key that is seen, summed over the query heads
    that share it, are added to it in place (what paged_kv_evict goes by).
    Returns (B, H, d), with return_lse=True also the float32 (B, H) log-sum-exp of the seen scaled logits.  A
    sequence of length 0 gives 0 (-inf).  A length beyond the capacity, or a page number outside the pool where a
    key is seen, makes that sequence's results NaN."""
    return _host.paged_attn_decode(q, k_cache, v_cache, block_table, seq_lens, scale, window, sinks, weight_sum, return_lse)


def paged_kv_evict(k_cache, v_cache, weight_sum, block_table, seq_lens, new_block_table, budget, sinks=0, recent=0):
    """Cuts every sequence to at most `budget` keys per head, by what attention looked at.

    Every head of a longer sequence keeps its first `sinks` keys, its last `recent` keys and, of those between,
    the ones with the largest weight_sum (float32 (B, Hkv, capacity), see paged_attn_decode; equal sums: the lowest
    index; NaN above everything).  The kept keys and values are copied, in their order, to the pages of
    new_block_table, int32 (B, new_width) with new_width * page >= budget, in the same pools; sequences within the
    budget are copied whole.  Old pages are left as they were (pages that sequences share stay intact) and are the
    caller's to reuse; new ones must not be among those read, nor appear twice.
    Returns (new_weight_sum float32 (B, Hkv, new_width * page), 0 behind the kept; new_lens int32 (B,); kept int32
    (B, Hkv, budget): the kept keys' old places, ascending, -1 behind them)."""
    return _host.paged_kv_evict(k_cache, v_cache, weight_sum, block_table, seq_lens, new_block_table, budget, sinks, recent)
