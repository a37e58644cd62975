"""Attention with a sliding window and a few first tokens that stay visible, forward and backward.

The reference's attention sees every key (csrc/api.cpp:168-192); this is the form that decoders with long
contexts use, beside flash_attn_fwd / flash_attn_bwd / flash_attn_func and in their manner.
"""
from ._lib import host as _host


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
    return _host.window_attn_fwd(q, k, v, window, sinks, scale, return_lse, seq_lens)


def window_attn_bwd(dout, q, k, v, out, lse, window, sinks=0, scale=1.0, seq_lens=None):
    """Gradients (dq, dk, dv) of window_attn_fwd: `out` and `lse` are its results (return_lse=True), `dout`, dense
    like `out`, the gradient of `out`.  dk and dv are summed over the query heads that share them.  Deterministic."""
    return _host.window_attn_bwd(dout, q, k, v, out, lse, window, sinks, scale, seq_lens)


def window_attn_func(q, k, v, window, sinks=0, scale=1.0, seq_lens=None):
    """window_attn_fwd with autograd support (once differentiable), for everything it serves.

    Capturing a training step into a graph: take the gradients with torch.autograd.grad, or let no autograd graph
    of the same leaves that was built outside live on (torch accumulates into a leaf on the stream it was first used on)."""
    return _host.window_attn_func(q, k, v, window, sinks, scale, seq_lens)
