"""Window attention with sinks, forward and backward, on the GPU against its definition in float64 (window_reference.py
derives the bounds)."""
import pytest
import torch

import window_reference as ref

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def mfa():
    import my_flash_attn_cuda
    assert torch.cuda.is_available()
    return my_flash_attn_cuda


def _inputs(B, H, G, nq, nk, d, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=gen).to(dtype)  # noqa: E731
    return make(B, H, nq, d), make(B, G, nk, d), make(B, G, nk, d), make(B, H, nq, d)


def _visible(B, nq, nk, window, sinks, lens):
    return torch.stack([ref.seen(nq, nk, window, sinks, nk if lens is None else min(max(lens[b], 0), nk)) for b in range(B)])


def _run(mfa, q, k, v, dout, window, sinks, scale, lens):
    L = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, lse = mfa.window_attn_fwd(q, k, v, window, sinks=sinks, scale=scale, return_lse=True, seq_lens=L)
    dq, dk, dv = mfa.window_attn_bwd(dout, q, k, v, out, lse, window, sinks=sinks, scale=scale, seq_lens=L)
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def _compare(mfa, B, H, G, nq, nk, d, window, sinks, lens, dtype, seed=0):
    q, k, v, dout = _inputs(B, H, G, nq, nk, d, dtype, seed)
    scale = d ** -0.5
    want = ref.attention(q, k, v, _visible(B, nq, nk, window, sinks, lens), scale, dtype, dout)
    got = _run(mfa, *(t.cuda() for t in (q, k, v, dout)), window, sinks, scale, lens)
    for name in got:
        ref.check(name, got[name], want[name])


CASES = [
    # B, H, G, nq, nk, d, window, sinks, lens
    (1, 1, 1, 1, 1, 64, 1, 0, None),                   # one token
    (1, 2, 1, 1, 300, 64, 40, 3, None),                # one query at the end of a piece
    (2, 2, 2, 130, 130, 128, 1, 0, None),              # every query sees itself alone
    (1, 2, 2, 200, 200, 64, 1000, 0, None),            # window wider than the sequence: causal
    (1, 4, 2, 333, 333, 128, 64, 4, None),
    (1, 3, 1, 129, 515, 64, 100, 70, None),            # sinks over more than one tile
    (1, 2, 1, 300, 300, 64, 17, 300, None),            # everything is a sink
    (2, 6, 2, 77, 150, 80, 33, 1, [150, 90]),
    (3, 2, 2, 65, 65, 64, 20, 2, [65, 0, 1]),          # an empty sequence and one of one token
    (2, 2, 1, 40, 200, 64, 50, 4, [100, 170]),         # a piece that lies behind a sequence's length altogether
    (1, 8, 1, 257, 257, 128, 90, 5, None),             # eight heads share one
    (1, 2, 1, 640, 640, 64, 100, 130, None),           # two key blocks hold sinks
    (1, 1, 1, 150, 150, 16, 30, 2, None),
    (1, 2, 1, 100, 140, 20, 30, 2, [120]),             # head dims off the 16-byte grid are padded
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_against_definition(mfa, case, dtype):
    _compare(mfa, *case, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [136, 192, 256])
def test_wide_heads(mfa, d, dtype):
    _compare(mfa, 1, 2, 1, 150, 210, d, 60, 3, [200], dtype)


def test_long_sequence(mfa):
    _compare(mfa, 1, 2, 1, 2100, 2100, 128, 300, 4, None, BF16)


MANY = [
    # enough blocks for the kernels that take 128 rows a workgroup
    (8, 16, 16, 200, 200, 64, 1000, 0, None),
    (4, 48, 48, 130, 333, 128, 64, 4, [333, 200, 203, 0]),
    (2, 48, 24, 300, 300, 80, 33, 1, [300, 77]),
    (1, 60, 30, 513, 513, 128, 90, 5, None),
    (1, 48, 24, 640, 640, 64, 100, 130, None),
    (3, 36, 12, 257, 400, 128, 170, 3, [400, 399, 150]),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", MANY, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_many_rows(mfa, case, dtype):
    _compare(mfa, *case, dtype)


@pytest.mark.parametrize("case", [(4, 48, 48, 130, 333, 128, 64, 4, [333, 200, 203, 0]), (1, 96, 96, 700, 700, 32, 90, 5, None)],
                         ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_many_rows_float32(mfa, case):
    _compare(mfa, *case, F32)


def test_many_rows_wide_heads(mfa):
    _compare(mfa, 2, 72, 72, 140, 140, 192, 50, 3, [140, 90], BF16)


@pytest.mark.parametrize("fill", [float("nan"), float("inf")])
def test_padding_of_many_rows_may_hold_anything(mfa, fill):
    lens = [200, 137, 0, 64]
    q, k, v, dout = _inputs(4, 32, 32, 200, 200, 64, BF16, 1)
    want = ref.attention(q, k, v, _visible(4, 200, 200, 30, 2, lens), 0.125, BF16, dout)
    for b, n in enumerate(lens):
        for t in (q, k, v, dout):
            t[b, :, n:] = fill
    got = _run(mfa, *(t.cuda() for t in (q, k, v, dout)), 30, 2, 0.125, lens)
    for name in got:
        ref.check(name, got[name], want[name])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gradients_against_differences(mfa, dtype):
    """The gradients of the definition itself, against central differences of it: what the bounds are held to is the
    derivative of the forward."""
    q, k, v, dout = (t.double() for t in _inputs(1, 2, 1, 9, 14, 8, F32, 3))
    vis = _visible(1, 9, 14, 4, 2, [13])
    want = ref.attention(q, k, v, vis, 0.4, dtype, dout)
    for name, t in (("dq", q), ("dk", k), ("dv", v)):
        for at in [(0, 0, 2, 1), (0, 0, 7, 5), (0, 0, 5, 0)]:
            h = 1e-5
            vals = []
            for sign in (1, -1):
                x = {"dq": q, "dk": k, "dv": v}[name].clone()
                x[at] += sign * h
                args = [x if n == name else y for n, y in (("dq", q), ("dk", k), ("dv", v))]
                vals.append(float((ref.attention(*args, vis, 0.4, dtype)["out"][0] * dout).sum()))
            assert abs((vals[0] - vals[1]) / (2 * h) - float(want[name][0][at])) < 1e-7
    got = _run(mfa, *(t.to(dtype).cuda() for t in (q, k, v, dout)), 4, 2, 0.4, [13])
    rounded = ref.attention(*(t.to(dtype) for t in (q, k, v)), vis, 0.4, dtype, dout.to(dtype))
    for name in got:
        ref.check(name, got[name], rounded[name])


@pytest.mark.parametrize("fill", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_padding_may_hold_anything(mfa, fill, dtype):
    lens = [100, 37, 0]
    q, k, v, dout = _inputs(3, 4, 2, 100, 100, 64, dtype, 1)
    want = ref.attention(q, k, v, _visible(3, 100, 100, 30, 2, lens), 0.125, dtype, dout)
    for b, n in enumerate(lens):
        for t in (q, k, v, dout):
            t[b, :, n:] = fill
    got = _run(mfa, *(t.cuda() for t in (q, k, v, dout)), 30, 2, 0.125, lens)
    for name in got:
        ref.check(name, got[name], want[name])


def test_keys_before_every_window_may_hold_anything(mfa):
    q, k, v, dout = _inputs(1, 2, 1, 50, 400, 64, BF16, 2)
    vis = _visible(1, 50, 400, 30, 2, None)
    want = ref.attention(q, k, v, vis, 0.125, BF16, dout)
    hidden = ~vis.any(1)[0]
    k[:, :, hidden], v[:, :, hidden] = float("nan"), float("inf")
    got = _run(mfa, *(t.cuda() for t in (q, k, v, dout)), 30, 2, 0.125, None)
    for name in got:
        ref.check(name, got[name], want[name])


@pytest.mark.parametrize("what", ["v", "k", "q", "dout"])
@pytest.mark.parametrize("shape", [(1, 4, 2, 260, 260, 64, 20, 0, BF16), (1, 4, 2, 150, 260, 128, 20, 3, F16), (1, 2, 1, 200, 200, 64, 20, 2, F32),
                                   (1, 2, 1, 180, 180, 192, 20, 2, BF16),                                       # few rows
                                   (1, 128, 64, 260, 260, 64, 20, 3, BF16), (1, 100, 100, 260, 260, 128, 20, 0, BF16),  # many
                                   (1, 100, 100, 260, 260, 64, 20, 3, F32), (1, 100, 100, 200, 200, 160, 20, 2, F16)],
                         ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_what_a_row_does_not_see_may_hold_anything(mfa, shape, what):
    """A key, value, query or gradient row that is infinite or NaN reaches what sees it, and nothing else, though tiles hold
    both."""
    B, H, G, nq, nk, d, window, sinks, dtype = shape
    q, k, v, dout = _inputs(B, H, G, nq, nk, d, dtype, 4)
    vis = _visible(B, nq, nk, window, sinks, None)
    want = ref.attention(q, k, v, vis, 0.125, dtype, dout)
    at = 141                                             # a position
    row_bad, key_bad = torch.zeros(nq, dtype=torch.bool), torch.zeros(nk, dtype=torch.bool)
    if what in "kv":
        {"k": k, "v": v}[what][:, :, at] = float("nan") if what == "k" else float("inf")
        row_bad = vis[0][:, at].clone()
    else:
        {"q": q, "dout": dout}[what][:, :, at - (nk - nq)] = float("nan")
        row_bad[at - (nk - nq)] = True
    key_bad = vis[0][row_bad].any(0)
    out_bad = row_bad if what != "dout" else torch.zeros_like(row_bad)
    assert row_bad.any() and not row_bad.all() and not key_bad.all()
    got = _run(mfa, *(t.cuda() for t in (q, k, v, dout)), window, sinks, 0.125, None)
    for name, keep in (("out", ~out_bad), ("dq", ~row_bad), ("dk", ~key_bad), ("dv", ~key_bad)):
        ref.check(name, got[name][:, :, keep.cuda()], tuple(t[:, :, keep] for t in want[name]))
    if out_bad.any():
        assert not torch.isfinite(got["out"][:, :, out_bad.cuda()]).any()
    assert torch.isnan(got["dq"][:, :, row_bad.cuda()]).any(-1).all()


@pytest.mark.parametrize("shape", [(1, 4, 2, 260, 260, 64, 20, 3, BF16), (1, 2, 1, 200, 200, 128, 20, 2, F32), (1, 2, 1, 180, 180, 256, 20, 2, F16),     # few rows
                                   (1, 100, 100, 260, 260, 128, 20, 3, F16), (1, 100, 100, 200, 200, 160, 20, 2, BF16), (1, 100, 100, 200, 200, 96, 20, 2, F32)],
                         ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_a_column_that_is_not_finite(mfa, shape):
    """One column of a value, and of an output gradient, in a place that some rows of a tile see: the others keep theirs, and what does
    not depend on it keeps all."""
    B, H, G, nq, nk, d, window, sinks, dtype = shape
    q, k, v, dout = _inputs(B, H, G, nq, nk, d, dtype, 5)
    vis = _visible(B, nq, nk, window, sinks, None)
    want = ref.attention(q, k, v, vis, 0.125, dtype, dout)
    at, col = 141, 37
    others = torch.arange(d) != col

    def rows(t, keep):
        return t[:, :, keep.to(t.device)]
    v_bad = v.clone()
    v_bad[:, :, at, col] = float("inf")
    sees = vis[0][:, at]
    touched = vis[0][sees].any(0)                              # keys that share a row with it
    got = _run(mfa, *(t.cuda() for t in (q, k, v_bad, dout)), window, sinks, 0.125, None)
    ref.check("out", got["out"][..., others.cuda()], tuple(t.expand_as(want["out"][0])[..., others] for t in want["out"]))
    ref.check("out", rows(got["out"], ~sees), tuple(rows(t, ~sees) for t in want["out"]))
    ref.check("dq", rows(got["dq"], ~sees), tuple(rows(t, ~sees) for t in want["dq"]))
    ref.check("dk", rows(got["dk"], ~touched), tuple(rows(t, ~touched) for t in want["dk"]))
    ref.check("dv", got["dv"], want["dv"])
    assert not torch.isfinite(rows(got["out"], sees)[..., col]).any()
    d_bad = dout.clone()
    d_bad[:, :, at, col] = float("nan")
    touched = vis[0][at]
    got = _run(mfa, *(t.cuda() for t in (q, k, v, d_bad)), window, sinks, 0.125, None)
    keep = torch.arange(nq) != at
    ref.check("dq", rows(got["dq"], keep), tuple(rows(t, keep) for t in want["dq"]))
    ref.check("dk", rows(got["dk"], ~touched), tuple(rows(t, ~touched) for t in want["dk"]))
    ref.check("dv", got["dv"][..., others.cuda()], tuple(t.expand_as(want["dv"][0])[..., others] for t in want["dv"]))
    ref.check("dv", rows(got["dv"], ~touched), tuple(rows(t, ~touched) for t in want["dv"]))


def test_strided_views(mfa):
    """(B, N, H, d) layouts and slices of one fused projection give what dense copies give, bit for bit."""
    torch.manual_seed(0)
    fused = torch.randn(2, 190, 8, 64, device="cuda", dtype=BF16)
    q, k, v = fused[:, :, :4].transpose(1, 2), fused[:, :, 4:6].transpose(1, 2), fused[:, :, 6:].transpose(1, 2)
    dout = torch.randn(2, 4, 190, 64, device="cuda", dtype=BF16)
    lens = [190, 111]
    a = _run(mfa, q, k, v, dout, 50, 4, 0.125, lens)
    b = _run(mfa, q.contiguous(), k.contiguous(), v.contiguous(), dout, 50, 4, 0.125, lens)
    for name in a:
        assert torch.equal(a[name], b[name]), name
    one = k[:, :, :1].expand(2, 2, 190, 64)              # rows of stride 0
    a = _run(mfa, q, one, v, dout, 50, 4, 0.125, lens)
    b = _run(mfa, q, one.contiguous(), v, dout, 50, 4, 0.125, lens)
    for name in a:
        assert torch.equal(a[name], b[name]), name


def test_strides_beyond_32_bits(mfa):
    """Batches that lie more than 2^32 bytes apart."""
    dense = [t.cuda() for t in _inputs(2, 4, 2, 150, 150, 64, BF16, 3)]
    apart = (1 << 31) + 64
    pool = torch.empty(apart + 3 * 4 * 150 * 64, dtype=BF16, device="cuda")
    far, at = [], 0
    for t in dense[:3]:
        H = t.shape[1]
        x = pool.as_strided(t.shape, (apart, 150 * 64, 64, 1), at)
        x.copy_(t)
        far.append(x)
        at += H * 150 * 64
    want, got = _run(mfa, *dense, 30, 3, 0.125, None), _run(mfa, *far, dense[3], 30, 3, 0.125, None)
    for name in want:
        assert torch.equal(got[name], want[name]), name


def test_same_result_every_time(mfa):
    q, k, v, dout = (t.cuda() for t in _inputs(2, 8, 2, 700, 700, 128, BF16, 4))
    first = _run(mfa, q, k, v, dout, 128, 4, 0.1, [700, 600])
    for _ in range(3):
        again = _run(mfa, q, k, v, dout, 128, 4, 0.1, [700, 600])
        for name in first:
            assert torch.equal(first[name], again[name]), name


def test_large_logits(mfa):
    """Logits of some thousands: the running maximum moves far, and weights underflow."""
    q, k, v, dout = _inputs(1, 1, 1, 200, 200, 64, F32, 5)
    want = ref.attention(q * 30, k * 30, v, _visible(1, 200, 200, 90, 1, None), 1.0, F32)
    out, lse = mfa.window_attn_fwd((q * 30).cuda(), (k * 30).cuda(), v.cuda(), 90, sinks=1, scale=1.0, return_lse=True)
    ref.check("out", out, want["out"])
    ref.check("lse", lse, want["lse"])


def test_causal_case_agrees_with_flash_attn(mfa):
    q, k, v, _ = (t.cuda() for t in _inputs(2, 2, 2, 257, 257, 128, BF16, 6))
    want = ref.attention(*(t.cpu() for t in (q, k, v)), _visible(2, 257, 257, 257, 0, None), 0.09, BF16)
    ref.check("flash", mfa.flash_attn_fwd(q, k, v, scale=0.09, return_lse=True, causal=True)[0], want["out"])
    ref.check("window", mfa.window_attn_fwd(q, k, v, 257, scale=0.09), want["out"])


def test_autograd(mfa):
    q, k, v, dout = (t.cuda() for t in _inputs(2, 4, 2, 90, 90, 64, BF16, 7))
    lens = torch.tensor([90, 50], dtype=torch.int32, device="cuda")
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = mfa.window_attn_func(*leaves, 20, sinks=2, scale=0.125, seq_lens=lens)
    grads = torch.autograd.grad(out, leaves, dout.transpose(1, 2).contiguous().transpose(1, 2))     # a strided gradient
    want = _run(mfa, q, k, v, dout, 20, 2, 0.125, [90, 50])
    for name, g in zip(("dq", "dk", "dv"), grads):
        assert torch.equal(g, want[name]), name


def test_autograd_at_its_edges(mfa):
    q, k, v, dout = (t.cuda() for t in _inputs(1, 4, 2, 40, 64, 60, BF16, 7))               # (a head dim that is padded)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = mfa.window_attn_func(*leaves, 20, scale=0.125)
    want = torch.autograd.grad(out, leaves, dout, retain_graph=True)
    moved = torch.empty(dout.numel() + 1, dtype=dout.dtype, device="cuda")[1:].view(dout.shape)
    moved.copy_(dout)                                                                       # dense, off the 16-byte grid
    for a, b in zip(torch.autograd.grad(out, leaves, moved, retain_graph=True), want):
        assert torch.equal(a, b)
    ones = torch.autograd.grad(out, leaves, torch.ones_like(out), retain_graph=True)
    for a, b in zip(torch.autograd.grad(out.sum(), leaves, retain_graph=True), ones):      # an expanded gradient
        assert torch.equal(a, b)
    for a, b in zip(torch.autograd.grad(out, leaves[1:2], dout, retain_graph=True), want[1:2]):
        assert torch.equal(a, b)
    twice = torch.autograd.grad(out, leaves, dout, retain_graph=True, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(twice, want))
    with pytest.raises(RuntimeError, match="once"):
        twice[0].sum().backward()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(twice[0].sum(), leaves)
    assert not mfa.window_attn_func(q, k, v, 20).requires_grad
    with torch.no_grad():
        leaves[0].add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(out, leaves, dout)


def test_other_stream(mfa):
    q, k, v, dout = (t.cuda() for t in _inputs(1, 4, 2, 500, 500, 128, BF16, 8))
    want = _run(mfa, q, k, v, dout, 100, 4, 0.1, None)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _run(mfa, q, k, v, dout, 100, 4, 0.1, None)
    side.synchronize()
    for name in got:
        assert torch.equal(got[name], want[name]), name


def test_graph_replays(mfa):
    """Forward and backward captured, replayed over new inputs with eager work in between."""
    L = torch.tensor([300, 200], dtype=torch.int32, device="cuda")
    static = [t.cuda() for t in _inputs(2, 4, 2, 300, 300, 64, BF16, 9)]

    def step():
        out, lse = mfa.window_attn_fwd(*static[:3], 40, sinks=4, scale=0.125, return_lse=True, seq_lens=L)
        return (out, lse, *mfa.window_attn_bwd(static[3], *static[:3], out, lse, 40, sinks=4, scale=0.125, seq_lens=L))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(4):
        for t, x in zip(static, _inputs(2, 4, 2, 300, 300, 64, BF16, 20 + seed)):
            t.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


def test_captured_training_step(mfa):
    """Forward and gradients through autograd, captured; the workspace is the graph's own, whatever eager calls do in between."""
    leaves = [t.cuda().requires_grad_() for t in _inputs(2, 4, 2, 300, 300, 64, BF16, 9)[:3]]
    dout = _inputs(2, 4, 2, 300, 300, 64, BF16, 9)[3].cuda()

    def step(x):
        out = mfa.window_attn_func(*x, 40, sinks=4, scale=0.125)
        return (out.detach(), *torch.autograd.grad(out, x, dout))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(leaves)
    torch.cuda.current_stream().wait_stream(side)
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(leaves)
    with torch.cuda.graph(second):
        held2 = step(leaves)
    for seed in range(3):
        with torch.no_grad():
            for t, x in zip(leaves, _inputs(2, 4, 2, 300, 300, 64, BF16, 20 + seed)):
                t.copy_(x)
        graph.replay()
        second.replay()
        want = step([t.detach().clone().requires_grad_() for t in leaves])
        torch.cuda.synchronize()
        for a, b, c in zip(held, held2, want):
            assert torch.equal(a, c) and torch.equal(b, c)


def test_refusals(mfa):
    q, k, v, dout = (t.cuda() for t in _inputs(1, 4, 2, 32, 48, 64, BF16, 0))
    lens = torch.tensor([48], dtype=torch.int32, device="cuda")
    bad = [
        (dict(window=0), "window"), (dict(window=8, sinks=-1), "sinks"), (dict(window=8, scale=0.0), "scale"),
        (dict(window=8, scale=float("nan")), "scale"), (dict(window=8, seq_lens=lens.long()), "int32"),
        (dict(window=8, seq_lens=torch.tensor([48, 48], dtype=torch.int32, device="cuda")), "int32"),
        (dict(window=8, seq_lens=lens.cpu()), "CUDA tensor"),
    ]
    for kw, match in bad:
        with pytest.raises(RuntimeError, match=match):
            mfa.window_attn_fwd(q, k, v, **kw)
    with pytest.raises(RuntimeError, match="Wrong sizes"):
        mfa.window_attn_fwd(k, q[:, :2], q[:, :2], 8)                  # more queries than keys
    with pytest.raises(RuntimeError, match="Wrong sizes"):
        mfa.window_attn_fwd(q, k, v[:, :, 1:], 8)
    with pytest.raises(RuntimeError, match="multiple"):
        mfa.window_attn_fwd(q[:, :3], k, v, 8)
    with pytest.raises(RuntimeError, match="Scalar type"):
        mfa.window_attn_fwd(q, k.half(), v, 8)
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        mfa.window_attn_fwd(q.double(), k.double(), v.double(), 8)
    with pytest.raises(RuntimeError, match="head dims up to"):
        mfa.window_attn_fwd(*(torch.zeros(1, 2, 8, 264, device="cuda", dtype=BF16) for _ in range(3)), 8)
    with pytest.raises(RuntimeError, match="head dims up to"):
        mfa.window_attn_fwd(*(torch.zeros(1, 2, 8, 136, device="cuda") for _ in range(3)), 8)
    wide = torch.zeros(1, 4, 32, 65, device="cuda", dtype=BF16)
    with pytest.raises(RuntimeError, match="16 bytes"):
        mfa.window_attn_fwd(wide[..., :64], k, v, 8)
    with pytest.raises(RuntimeError, match="16 bytes"):
        mfa.window_attn_fwd(q.transpose(2, 3).contiguous().transpose(2, 3), k, v, 8)
    out, lse = mfa.window_attn_fwd(q, k, v, 8, return_lse=True)
    with pytest.raises(RuntimeError, match="contiguous"):
        mfa.window_attn_bwd(dout.transpose(1, 2).contiguous().transpose(1, 2), q, k, v, out, lse, 8)
    with pytest.raises(RuntimeError, match="lse must"):
        mfa.window_attn_bwd(dout, q, k, v, out, lse[:, :, :-1].contiguous(), 8)
    with pytest.raises(RuntimeError, match="Wrong sizes"):
        mfa.window_attn_bwd(dout[:, :2].contiguous(), q, k, v, out, lse, 8)


def test_empty_sizes(mfa):
    q, k, v = (torch.empty(*s, device="cuda", dtype=BF16) for s in ((0, 2, 5, 64), (0, 2, 5, 64), (0, 2, 5, 64)))
    assert mfa.window_attn_fwd(q, k, v, 4).shape == (0, 2, 5, 64)
    q, k = torch.empty(1, 2, 0, 64, device="cuda", dtype=BF16), torch.ones(1, 2, 7, 64, device="cuda", dtype=BF16)
    out, lse = mfa.window_attn_fwd(q, k, k, 4, return_lse=True)
    assert out.shape == (1, 2, 0, 64)
    dq, dk, dv = mfa.window_attn_bwd(out, q, k, k, out, lse, 4, sinks=1)
    assert dq.numel() == 0 and not dk.any() and not dv.any()


def _bwd_with_workspace(dout, q, k, v, out, lse, window, sinks, scale, lens, fill):
    """window_attn_bwd through the C entry, its workspace holding nothing but float32 `fill` before the call."""
    import ctypes

    from my_flash_attn_cuda import _lib
    B, H, nq, d = q.shape
    G, nk = k.shape[1:3]
    tag = {F32: _lib.MYFA_F32, F16: _lib.MYFA_F16, BF16: _lib.MYFA_BF16}[q.dtype]
    nbytes = _lib.lib.myfa_window_attn_bwd_ws_bytes(B, H, G, nq, nk, d, window, sinks, tag)
    ws = torch.full((nbytes // 4,), fill, device="cuda")
    grads = [torch.empty_like(t) for t in (q, k, v)]
    strides = [(ctypes.c_int64 * 3)(*t.stride()[:3]) for t in (q, k, v)]
    _lib.check(_lib.lib.myfa_window_attn_bwd(
        *(t.data_ptr() for t in (q, k, v, out, lse, dout, *grads)), None if lens is None else lens.data_ptr(),
        B, H, G, nq, nk, d, *strides, window, sinks, scale, tag, ws.data_ptr(), nbytes, torch.cuda.current_stream().cuda_stream))
    return dict(zip(("dq", "dk", "dv"), grads))


@pytest.mark.parametrize("case", [
    # few query blocks that meet many key blocks, the last rows of a head filling at most half of the 64 that dK, dV reads at a time
    (1, 8, 8, 1044, 1044, 128, 300, 0, None, BF16),
    (1, 8, 8, 1044, 1044, 128, 300, 4, None, F16),
    (1, 8, 8, 20, 1200, 128, 150, 3, None, BF16),
    (2, 8, 8, 70, 1100, 128, 2000, 0, [1100, 1050], BF16),
    (1, 8, 8, 65, 3300, 64, 400, 2, None, F16),
    (1, 64, 64, 20, 1100, 16, 200, 1, None, F32),
    (1, 4, 4, 33, 4200, 192, 500, 1, None, BF16),
    (1, 4, 2, 100, 100, 64, 30, 2, [90], BF16),              # few of both
    (2, 96, 48, 161, 300, 64, 64, 4, [300, 170], BF16),      # many of both
], ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_gradients_do_not_depend_on_the_workspace(mfa, case):
    B, H, G, nq, nk, d, window, sinks, lens, dtype = case
    q, k, v, dout = _inputs(B, H, G, nq, nk, d, dtype, 11)
    scale = d ** -0.5
    want = ref.attention(q, k, v, _visible(B, nq, nk, window, sinks, lens), scale, dtype, dout)
    q, k, v, dout = (t.cuda() for t in (q, k, v, dout))
    L = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, lse = mfa.window_attn_fwd(q, k, v, window, sinks=sinks, scale=scale, return_lse=True, seq_lens=L)
    zeros = _bwd_with_workspace(dout, q, k, v, out, lse, window, sinks, scale, L, 0.0)
    for name in zeros:
        ref.check(name, zeros[name], want[name])
    for fill in (float("nan"), float("inf"), -1e30):
        again = _bwd_with_workspace(dout, q, k, v, out, lse, window, sinks, scale, L, fill)
        for name in zeros:
            assert torch.equal(again[name], zeros[name]), (name, fill)


@pytest.mark.parametrize("case", [(4, 16, 16, 300, 300, 64, 20, 150, None), (2, 32, 16, 500, 500, 64, 20, 400, [500, 310]), (16, 32, 32, 200, 200, 16, 20, 190, None),
                                  (1, 2, 1, 900, 900, 128, 20, 300, None)], ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_many_sinks(mfa, case):
    """Several key blocks of sinks, split as far as the bound on the workspace lets them, or not at all."""
    _compare(mfa, *case, BF16)


@pytest.mark.parametrize("shape", [(1, 4, 2, 260, 260, 64, 20, 0, BF16), (1, 2, 1, 200, 200, 128, 20, 2, F32), (1, 2, 1, 180, 180, 192, 20, 2, F16),     # few rows
                                   (1, 100, 100, 260, 260, 128, 20, 3, F16), (1, 100, 100, 200, 200, 160, 20, 2, BF16)],
                         ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_a_hidden_value_does_not_change_a_bit_of_dq(mfa, shape):
    """Where a hidden key's column is infinite already, and is formed again, an infinite value beside it changes nothing: hidden
    weights are set to 0 behind the product that the value reaches.  (The forward forms such rows again, with other roundings: both
    calls go by one out and lse.)"""
    B, H, G, nq, nk, d, window, sinks, dtype = shape
    q, k, v, dout = (t.cuda() for t in _inputs(B, H, G, nq, nk, d, dtype, 12))
    at = 141
    k[:, :, at, 5] = float("inf")
    hidden = ~_visible(B, nq, nk, window, sinks, None)[0][:, at].cuda()
    out, lse = mfa.window_attn_fwd(q, k, v, window, sinks=sinks, scale=0.125, return_lse=True)
    first = mfa.window_attn_bwd(dout, q, k, v, out, lse, window, sinks=sinks, scale=0.125)[0][:, :, hidden]
    v[:, :, at] = float("inf")
    second = mfa.window_attn_bwd(dout, q, k, v, out, lse, window, sinks=sinks, scale=0.125)[0][:, :, hidden]
    assert torch.isfinite(first).all() and torch.equal(first, second)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
def test_rows_behind_the_length_do_not_change_the_others(mfa, d, dtype):
    """The same bits whether the rows behind a row exist or not: with logits this small the running maximum stays where the first tile
    leaves it (a lane's sum of 32 weights is below 2^8 everywhere), and rows that see nothing must not move it."""
    q, k, v, _ = (t.cuda() for t in _inputs(1, 32, 32, 1024, 1024, d, dtype, 13))
    out, lse = mfa.window_attn_fwd(q, k, v, 1024, scale=0.002, return_lse=True)
    for n in (1000, 900, 897):
        L = torch.tensor([n], dtype=torch.int32, device="cuda")
        cut, cut_lse = mfa.window_attn_fwd(q, k, v, 1024, scale=0.002, return_lse=True, seq_lens=L)
        assert torch.equal(cut[:, :, :n], out[:, :, :n]) and torch.equal(cut_lse[:, :, :n], lse[:, :, :n]), n
        assert not cut[:, :, n:].any()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_head_dim_of_zero(mfa, dtype):
    """All logits are 0: the log-sum-exp is the logarithm of how many keys a row sees."""
    q, k, v, dout = (t.cuda() for t in _inputs(2, 2, 1, 40, 50, 0, dtype))
    L = torch.tensor([50, 30], dtype=torch.int32, device="cuda")
    taken = torch.full((2, 2, 40), 7.0, device="cuda")       # (what an allocation of that size holds next)
    del taken
    out, lse = mfa.window_attn_fwd(q, k, v, 9, sinks=2, return_lse=True, seq_lens=L)
    assert out.shape == q.shape
    want = ref.attention(*(t.cpu() for t in (q, k, v)), _visible(2, 40, 50, 9, 2, [50, 30]), 1.0, dtype)
    ref.check("lse", lse, want["lse"])
    for g, t in zip(mfa.window_attn_bwd(dout, q, k, v, out, lse, 9, sinks=2, seq_lens=L), (q, k, v)):
        assert g.shape == t.shape


def test_results_do_not_depend_on_fresh_memory(mfa):
    """Outputs and workspaces filled with NaN before the call change nothing: torch does that to fresh memory in its deterministic mode."""
    cases = [(2, 6, 2, 77, 150, 80, 33, 1, [150, 90], BF16), (3, 2, 2, 65, 65, 64, 20, 2, [65, 0, 1], F32), (1, 2, 1, 640, 640, 64, 100, 130, None, F16),
             (4, 48, 48, 130, 333, 128, 64, 4, [333, 200, 203, 0], BF16), (1, 60, 30, 513, 513, 128, 90, 5, None, F16),
             (1, 96, 96, 700, 700, 32, 90, 5, None, F32), (2, 72, 72, 140, 140, 192, 50, 3, [140, 90], BF16), (1, 8, 8, 20, 1200, 128, 150, 3, None, BF16),
             (1, 2, 1, 100, 140, 20, 30, 2, [120], BF16)]

    def calls():
        for B, H, G, nq, nk, d, window, sinks, lens, dtype in cases:
            q, k, v, dout = (t.cuda() for t in _inputs(B, H, G, nq, nk, d, dtype, 17))
            yield _run(mfa, q, k, v, dout, window, sinks, d ** -0.5, lens)
    want = list(calls())
    before = torch.are_deterministic_algorithms_enabled(), torch.utils.deterministic.fill_uninitialized_memory
    try:
        torch.use_deterministic_algorithms(True, warn_only=True)
        torch.utils.deterministic.fill_uninitialized_memory = True
        assert torch.isnan(torch.empty(5, device="cuda")).all()
        for x, y in zip(calls(), want):
            for name in x:
                assert torch.equal(x[name], y[name]), name
    finally:
        torch.use_deterministic_algorithms(before[0])
        torch.utils.deterministic.fill_uninitialized_memory = before[1]
