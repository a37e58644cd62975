"""Attention with a sliding window and a few first tokens that stay visible, forward and backward.

The reference's attention sees every key (csrc/api.cpp:168-192); this is the form that decoders with long
contexts use, beside flash_attn_fwd / flash_attn_bwd / flash_attn_func and in their manner.
"""
import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _DTYPE_TAG, _check_gpu, _check_ints, _check_input, _check_rows, _lib, _on, _same_device, _stream

WINDOW_MAX_HEAD_DIM = 256        # float16 / bfloat16
WINDOW_MAX_HEAD_DIM_F32 = 128


def _strides(s):
    return (ctypes.c_int64 * 3)(*s)


def _check_qkv(q, k, v, window, sinks, seq_lens, what):
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        _check_gpu(t, name)
    _same_device(k, q, "k"); _same_device(v, q, "v")
    if q.dim() != 4 or k.dim() != 4:
        raise RuntimeError(f"{what} expects (B, H, N, d) tensors, got {q.dim()}-D and {k.dim()}-D")
    B, H, nq, d = q.shape
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != d or nq > k.shape[2]:
        raise RuntimeError("Wrong sizes!")
    if not (q.dtype == k.dtype == v.dtype):
        raise RuntimeError("Scalar type mismatch!")
    if q.dtype not in _DTYPE_TAG:
        raise RuntimeError(f"unsupported dtype {q.dtype}")
    if H < 1 or k.shape[1] < 1 or H % k.shape[1]:
        raise RuntimeError(f"{H} query heads are not a multiple of {k.shape[1]} key/value heads")
    most = WINDOW_MAX_HEAD_DIM_F32 if q.dtype == torch.float32 else WINDOW_MAX_HEAD_DIM
    if d > most:
        raise RuntimeError(f"{what} supports head dims up to {most} for {q.dtype}, got {d}")
    if int(window) != window or window < 1 or int(sinks) != sinks or sinks < 0:
        raise RuntimeError(f"window must be an integer of at least 1 and sinks one of at least 0, got {window} and {sinks}")
    if seq_lens is not None:
        _check_ints(seq_lens, (B,), q, "seq_lens")
    if _padding(q):
        return (None,) * 3           # padded copies are taken
    return [_check_rows(t, name) for t, name in ((q, "q"), (k, "k"), (v, "v"))]


def _padding(t):
    """Zero columns up to the next head dim whose rows are whole 16-byte chunks change nothing."""
    return -t.shape[-1] % (16 // t.element_size())


def window_attn_fwd(q, k, v, window, sinks=0, scale=1.0, return_lse=False, seq_lens=None):
    """softmax(scale * q @ k^T) @ v per head, over the keys that a query sees.

    q: (B, H, Nq, d); k, v: (B, Hkv, Nk, d) with H a multiple of Hkv (query head h uses key/value head
    h // (H // Hkv)) and Nq <= Nk, GPU tensors of one dtype (float16, bfloat16 with d <= 256; float32 with
    d <= 128).  Any strides with a dense last dimension and rows at multiples of 16 bytes.
    Query i stands at position p = i + Nk - Nq and sees key j when j <= p and (p - j < window or j < sinks):
    the last `window` keys up to its own, and the first `sinks` keys.  window >= Nk is causal attention.
    seq_lens: int32 (B,), for sequences padded at their end: keys j >= seq_lens[b] are not seen, and rows with
    p >= seq_lens[b] see nothing.  What padding holds has no influence.  A row that sees nothing is 0
    (log-sum-exp -inf).
    Returns a dense (B, H, Nq, d) tensor, with return_lse=True also the float32 (B, H, Nq) log-sum-exp of the
    seen scaled logits."""
    qs, ks, vs = _check_qkv(q, k, v, window, sinks, seq_lens, "window_attn_fwd")
    B, H, nq, d = q.shape
    if _padding(q):
        pad = _padding(q)
        res = window_attn_fwd(*(torch.nn.functional.pad(t, (0, pad)) for t in (q, k, v)), window, sinks=sinks, scale=scale,
                              return_lse=return_lse, seq_lens=seq_lens)
        return (res[0][..., :d].contiguous(), res[1]) if return_lse else res[..., :d].contiguous()
    out = torch.empty((B, H, nq, d), dtype=q.dtype, device=q.device)
    lse = torch.empty((B, H, nq), dtype=torch.float32, device=q.device) if return_lse else None
    with _on(q):
        _lib.check(_lib.lib.myfa_window_attn_fwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else None,
            seq_lens.data_ptr() if seq_lens is not None else None, B, H, k.shape[1], nq, k.shape[2], d,
            _strides(qs), _strides(ks), _strides(vs), int(window), int(sinks), float(scale), _DTYPE_TAG[q.dtype], _stream()))
    return (out, lse) if return_lse else out


def window_attn_bwd(dout, q, k, v, out, lse, window, sinks=0, scale=1.0, seq_lens=None):
    """Gradients (dq, dk, dv) of window_attn_fwd: `out` and `lse` are its results (return_lse=True), `dout`, dense
    like `out`, the gradient of `out`.  dk and dv are summed over the query heads that share them.  Deterministic."""
    qs, ks, vs = _check_qkv(q, k, v, window, sinks, seq_lens, "window_attn_bwd")
    for t, name in ((dout, "dout"), (out, "out"), (lse, "lse")):
        _check_input(t, name)
        _same_device(t, q, name)
    if not (q.shape == out.shape == dout.shape):
        raise RuntimeError("Wrong sizes!")
    if not (q.dtype == out.dtype == dout.dtype):
        raise RuntimeError("Scalar type mismatch!")
    B, H, nq, d = q.shape
    hkv, nk = k.shape[1], k.shape[2]
    if lse.dtype != torch.float32 or tuple(lse.shape) != (B, H, nq):
        raise RuntimeError("lse must be the float32 (B, H, Nq) tensor returned by window_attn_fwd")
    if _padding(q):
        pad = _padding(q)
        padded = [torch.nn.functional.pad(t, (0, pad)) for t in (dout, q, k, v, out)]
        return tuple(g[..., :d].contiguous() for g in window_attn_bwd(*padded, lse, window, sinks=sinks, scale=scale, seq_lens=seq_lens))
    dq = torch.empty((B, H, nq, d), dtype=q.dtype, device=q.device)
    dk, dv = (torch.empty((B, hkv, nk, d), dtype=q.dtype, device=q.device) for _ in range(2))
    nbytes = _lib.lib.myfa_window_attn_bwd_ws_bytes(B, H, hkv, nq, nk, d, int(window), int(sinks))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    with _on(q):
        _lib.check(_lib.lib.myfa_window_attn_bwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), dout.data_ptr(),
            dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), seq_lens.data_ptr() if seq_lens is not None else None,
            B, H, hkv, nq, nk, d, _strides(qs), _strides(ks), _strides(vs), int(window), int(sinks), float(scale),
            _DTYPE_TAG[q.dtype], ws.data_ptr(), nbytes, _stream()))
    return dq, dk, dv


class _WindowAttnFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sinks, scale, seq_lens):
        out, lse = window_attn_fwd(q, k, v, window, sinks=sinks, scale=scale, return_lse=True, seq_lens=seq_lens)
        ctx.save_for_backward(q, k, v, out, lse, seq_lens)
        ctx.window, ctx.sinks, ctx.scale = window, sinks, scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, seq_lens = ctx.saved_tensors
        dq, dk, dv = window_attn_bwd(dout.contiguous(), q, k, v, out, lse, ctx.window, sinks=ctx.sinks, scale=ctx.scale, seq_lens=seq_lens)
        return dq, dk, dv, None, None, None, None


def window_attn_func(q, k, v, window, sinks=0, scale=1.0, seq_lens=None):
    """window_attn_fwd with autograd support, for everything it serves."""
    return _WindowAttnFunc.apply(q, k, v, window, sinks, scale, seq_lens)
