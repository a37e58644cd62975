"""Window attention and attention over a cache in float64 on the CPU, from the definition, with bounds on how far the
kernels' results may be off.

The bounds follow the arithmetic.  u = finfo(T).eps / 2 is what one rounding to the element type costs, w = 2^-24
what one float32 operation does.  For a row with weights p:
  logits    float32 sums of d products: off by at most e = (d + 8) w scale sum|q||k| (its largest over the row's keys)
  weights   relative 2 e + (n + 16) w: numerator and denominator each have e, the denominator sums n terms
  out       sum p~ v with p~ rounded to the element type (relative u; in float16 also 2^-25, half its smallest
            step, per weight), and one rounding at the end:
            |err| <= sum p|v| (u + 2 e + 2 (n + 16) w) + u |out| + [f16] 2^-25 (sum|v| + 1)
  float32   P is not rounded: u is w there.
Gradients: dV like out, over rows; dP has d float32 products, delta also the error of the rounded out; dS is rounded
to the element type; the sums over keys or rows and one rounding at the end follow.
"""
import torch

W = 2.0 ** -24


def seen(nq, nk, window, sinks, length):
    """(nq, nk): which keys a row sees."""
    pos = torch.arange(nk - nq, nk)[:, None]
    key = torch.arange(nk)[None, :]
    return (key <= pos) & (pos < length) & (key < length) & ((pos - key < window) | (key < sinks))


def attention(q, k, v, visible, scale, dtype, dout=None):
    """q (B, H, nq, d), k, v (B, G, nk, d), visible (B, nq, nk) -> {name: (value, bound)} in float64.  Rows and keys that
    have no visible partner may hold anything."""
    B, H, nq, d = q.shape
    G, nk = k.shape[1], k.shape[2]
    rep = H // G
    u, tiny = torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == torch.float16 else 0.0
    vis = visible[:, None]                                            # (B, 1, nq, nk)
    row, key = vis.any(-1, keepdim=True), visible.any(1)[:, None, :, None]
    q = torch.where(row, q.double(), 0.0)
    k, v = (torch.where(key, t.double(), 0.0).repeat_interleave(rep, 1) for t in (k, v))
    s = (q @ k.transpose(-1, -2) * scale).masked_fill(~vis, float("-inf"))
    lse = torch.logsumexp(s, -1)
    p = torch.where(vis, torch.exp(s - torch.where(row.squeeze(-1), lse, 0.0)[..., None]), 0.0)
    n = nk + 16
    e = ((d + 8) * W * scale * torch.where(vis, q.abs() @ k.abs().transpose(-1, -2), 0.0)).amax(-1, keepdim=True)
    ew = 2 * e + 2 * n * W                                            # relative error of a weight
    out = p @ v
    b_out = (p @ v.abs()) * (u + ew) + u * out.abs() + tiny * (vis.double() @ v.abs() + 1)
    res = {"out": (out, b_out), "lse": (lse, (e + n * W).squeeze(-1) + 4 * W * lse.abs()), "p": (p, p * ew)}
    if dout is None:
        return res
    do = torch.where(row, dout.double(), 0.0)
    dp = do @ v.transpose(-1, -2)
    delta = (do * out).sum(-1, keepdim=True)
    b_dp = (d + 4) * W * (do.abs() @ v.abs().transpose(-1, -2))
    b_delta = (do.abs() * b_out).sum(-1, keepdim=True) + (d + 4) * W * (do * out).abs().sum(-1, keepdim=True)
    ds = p * (dp - delta)
    b_ds = torch.where(vis, p * (b_dp + b_delta + 4 * W * (dp.abs() + delta.abs())) * (1 + u) + ds.abs() * (ew + u) + tiny, 0.0)
    dq = ds @ k * scale
    b_dq = (b_ds @ k.abs() + n * W * (ds.abs() @ k.abs())) * scale + u * dq.abs() + tiny
    fold = lambda t: t.reshape(B, G, rep, nk, d).sum(2)  # noqa: E731
    m = rep * (nq + 16)
    dk = fold(ds.transpose(-1, -2) @ q * scale)
    b_dk = fold((b_ds.transpose(-1, -2) @ q.abs() + m * W * (ds.abs().transpose(-1, -2) @ q.abs())) * scale) + u * dk.abs() + tiny
    dv = fold(p.transpose(-1, -2) @ do)
    b_dv = fold((p * (u + ew + m * W) + torch.where(vis, tiny, 0.0)).transpose(-1, -2) @ do.abs()) + u * dv.abs() + tiny
    return {**res, "dq": (dq, b_dq), "dk": (dk, b_dk), "dv": (dv, b_dv)}


def check(name, got, want, slack=0.0):
    """Every element within its bound (and finite exactly where the reference is)."""
    value, bound = want
    got = got.detach().double().cpu()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    fine = torch.isfinite(value)
    assert torch.equal(torch.isfinite(got), fine), f"{name}: not finite where the definition is, or the reverse"
    assert torch.equal(got[~fine], value[~fine]), name
    err = (got - value).abs()[fine]
    over = err - bound.expand_as(value)[fine] * (1 + slack)
    assert err.numel() == 0 or float(over.max()) <= 0, f"{name}: {float(err.max()):.3g} off, {float(over.max()):.3g} over its bound"
