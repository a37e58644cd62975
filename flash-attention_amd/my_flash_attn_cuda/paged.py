"""A paged key/value cache: append, attention of one new token per sequence, eviction by attention weight.

The cache is two pools of pages, k_cache and v_cache (pages, Hkv, page, d): a page holds `page` consecutive keys of
every key/value head.  block_table, int32 (B, width), gives every sequence its pages: key j of sequence b stands in
page block_table[b, j // page], slot j % page; entries behind a sequence's last page are not read.  A sequence
holds at most width * page keys, its capacity.  Lengths and tables stay on the device: no call waits for the GPU,
and every call can be captured into a graph.  Page numbers outside the pool never become addresses.
The reference has no cache (csrc/api.cpp:168-192 takes whole matrices).
"""
import ctypes

import torch

from . import _DTYPE_TAG, _check_ints, _check_input, _check_rows, _check_float, _lib, _on, _same_device, _stream


def _strides(s):
    return (ctypes.c_int64 * len(s))(*s)


def _check_cache(k_cache, v_cache, block_table, seq_lens):
    ks, vs = _check_rows(k_cache, "k_cache"), _check_rows(v_cache, "v_cache")
    _same_device(v_cache, k_cache, "v_cache")
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        raise RuntimeError("k_cache and v_cache must be (pages, heads, page, d) tensors of one shape")
    if k_cache.dtype != v_cache.dtype:
        raise RuntimeError("Scalar type mismatch!")
    if k_cache.dtype not in _DTYPE_TAG:
        raise RuntimeError(f"unsupported dtype {k_cache.dtype}")
    if k_cache.shape[1] < 1 or k_cache.shape[2] < 1:
        raise RuntimeError("a page holds at least one key of one head")
    if not isinstance(block_table, torch.Tensor) or block_table.dim() != 2:
        raise RuntimeError("block_table must be an int32 (B, width) tensor")
    _check_ints(block_table, block_table.shape, k_cache, "block_table")
    _check_ints(seq_lens, (block_table.shape[0],), k_cache, "seq_lens")
    return ks, vs


def paged_kv_append(k, v, k_cache, v_cache, block_table, seq_lens, counts=None):
    """Writes n new keys and values per sequence into the cache, in place.

    k, v: (B, Hkv, n, d) of the cache's dtype, any strides with a dense last dimension and rows at multiples of
    16 bytes.  The tokens go to the places seq_lens[b] .. seq_lens[b] + n - 1 of their sequence; with counts, int32
    (B,), only the first counts[b] of them do (padded batches).  seq_lens is not changed: a caller adds n to it.
    A token whose place is outside [0, capacity) or on a page number outside the pool is dropped.  No two tokens
    of a call may have the same place."""
    kcs, vcs = _check_cache(k_cache, v_cache, block_table, seq_lens)
    ks, vs = _check_rows(k, "k"), _check_rows(v, "v")
    _same_device(k, k_cache, "k"); _same_device(v, k_cache, "v")
    pages, heads, page, d = k_cache.shape
    if k.dim() != 4 or k.shape != v.shape or k.shape[0] != block_table.shape[0] or k.shape[1] != heads or k.shape[3] != d:
        raise RuntimeError("Wrong sizes!")
    if not (k.dtype == v.dtype == k_cache.dtype):
        raise RuntimeError("Scalar type mismatch!")
    if counts is not None:
        _check_ints(counts, (k.shape[0],), k_cache, "counts")
    with _on(k_cache):
        _lib.check(_lib.lib.myfa_paged_append(
            k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(),
            counts.data_ptr() if counts is not None else None, k.shape[0], heads, k.shape[2], d, pages, page, block_table.shape[1],
            _strides(ks), _strides(vs), _strides(kcs), _strides(vcs), _DTYPE_TAG[k_cache.dtype], _stream()))


def paged_attn_decode(q, k_cache, v_cache, block_table, seq_lens, scale=1.0, window=0, sinks=0, weight_sum=None, return_lse=False):
    """Attention of one new token per sequence over its cached keys, its own (place seq_lens[b] - 1) among them.

    q: (B, H, d) of the cache's dtype, H a multiple of Hkv (query head h uses key/value head h // (H // Hkv)).
    window > 0: only the last `window` keys and the first `sinks` are seen; window = 0: all.
    weight_sum: float32 (B, Hkv, capacity), contiguous: the weights of every key that is seen, summed over the query heads
    that share it, are added to it in place (what paged_kv_evict goes by).
    Returns (B, H, d), with return_lse=True also the float32 (B, H) log-sum-exp of the seen scaled logits.  A
    sequence of length 0 gives 0 (-inf).  A length beyond the capacity, or a page number outside the pool where a
    key is seen, makes that sequence's results NaN."""
    kcs, vcs = _check_cache(k_cache, v_cache, block_table, seq_lens)
    qs = _check_rows(q, "q")
    _same_device(q, k_cache, "q")
    pages, heads, page, d = k_cache.shape
    B, width = block_table.shape
    if q.dim() != 3 or q.shape[0] != B or q.shape[2] != d:
        raise RuntimeError("Wrong sizes!")
    if q.dtype != k_cache.dtype:
        raise RuntimeError("Scalar type mismatch!")
    H = q.shape[1]
    if H < 1 or H % heads:
        raise RuntimeError(f"{H} query heads are not a multiple of {heads} key/value heads")
    if int(window) != window or window < 0 or int(sinks) != sinks or sinks < 0:
        raise RuntimeError(f"window and sinks must be integers of at least 0, got {window} and {sinks}")
    if weight_sum is not None:
        _check_input(weight_sum, "weight_sum")
        _same_device(weight_sum, k_cache, "weight_sum")
        _check_float(weight_sum, "weight_sum")
        if tuple(weight_sum.shape) != (B, heads, width * page):
            raise RuntimeError(f"weight_sum must be {(B, heads, width * page)}, got {tuple(weight_sum.shape)}")
    out = torch.empty((B, H, d), dtype=q.dtype, device=q.device)
    lse = torch.empty((B, H), dtype=torch.float32, device=q.device) if return_lse else None
    nbytes = _lib.lib.myfa_paged_attn_decode_ws_bytes(B, H, heads, d, page, width, int(window), int(sinks), weight_sum is not None)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes > 0 else None
    with _on(k_cache):
        _lib.check(_lib.lib.myfa_paged_attn_decode(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), out.data_ptr(),
            lse.data_ptr() if return_lse else None, weight_sum.data_ptr() if weight_sum is not None else None,
            B, H, heads, d, pages, page, width, _strides(qs), _strides(kcs), _strides(vcs), int(window), int(sinks), float(scale),
            _DTYPE_TAG[q.dtype], ws.data_ptr() if ws is not None else None, nbytes, _stream()))
    return (out, lse) if return_lse else out


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
    kcs, vcs = _check_cache(k_cache, v_cache, block_table, seq_lens)
    pages, heads, page, d = k_cache.shape
    B, width = block_table.shape
    _check_input(weight_sum, "weight_sum")
    _same_device(weight_sum, k_cache, "weight_sum")
    _check_float(weight_sum, "weight_sum")
    if tuple(weight_sum.shape) != (B, heads, width * page):
        raise RuntimeError(f"weight_sum must be {(B, heads, width * page)}, got {tuple(weight_sum.shape)}")
    if not isinstance(new_block_table, torch.Tensor) or new_block_table.dim() != 2:
        raise RuntimeError("new_block_table must be an int32 (B, width) tensor")
    _check_ints(new_block_table, (B, new_block_table.shape[1]), k_cache, "new_block_table")
    if any(int(x) != x for x in (budget, sinks, recent)) or budget < 1 or sinks < 0 or recent < 0 or sinks + recent > budget:
        raise RuntimeError(f"budget ({budget}) must be at least 1 and hold sinks ({sinks}) and recent ({recent})")
    capacity = new_block_table.shape[1] * page
    if capacity < budget:
        raise RuntimeError(f"new_block_table holds {capacity} keys a sequence, the budget is {budget}")
    new_sums = torch.empty((B, heads, capacity), dtype=torch.float32, device=k_cache.device)
    new_lens = torch.empty((B,), dtype=torch.int32, device=k_cache.device)
    kept = torch.empty((B, heads, int(budget)), dtype=torch.int32, device=k_cache.device)
    with _on(k_cache):
        _lib.check(_lib.lib.myfa_paged_evict(
            k_cache.data_ptr(), v_cache.data_ptr(), weight_sum.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(),
            new_block_table.data_ptr(), new_sums.data_ptr(), new_lens.data_ptr(), kept.data_ptr(),
            B, heads, d, pages, page, width, new_block_table.shape[1], _strides(kcs), _strides(vcs),
            int(budget), int(sinks), int(recent), _DTYPE_TAG[k_cache.dtype], _stream()))
    return new_sums, new_lens, kept
