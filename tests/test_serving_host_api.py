"""CPU tests of the window attention and paged cache entry points: refusals of the Python layer and of the C ABI that need
no GPU, and the index arithmetic the kernels share.  No kernel is launched here."""
import ctypes
import random

import pytest
import torch

import my_flash_attn_cuda as mfa
import window_reference as ref
from my_flash_attn_cuda import _lib

S3 = ctypes.c_int64 * 3


def test_cpu_tensors_are_rejected():
    x = torch.zeros(1, 2, 8, 64)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    sums = torch.zeros(1, 2, 16)
    for call in (lambda: mfa.window_attn_fwd(x, x, x, 4), lambda: mfa.window_attn_func(x, x, x, 4),
                 lambda: mfa.window_attn_bwd(x, x, x, x, x, x[..., 0], 4),
                 lambda: mfa.paged_kv_append(x, x, x, x, table, lens),
                 lambda: mfa.paged_attn_decode(x[:, :, 0], x, x, table, lens),
                 lambda: mfa.paged_kv_evict(x, x, sums, table, lens, table, 4)):
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            call()


def test_other_types_are_rejected():
    with pytest.raises(TypeError):
        mfa.window_attn_fwd(1, 2, 3, 4)
    with pytest.raises(TypeError):
        mfa.paged_attn_decode(None, None, None, None, None)


def _error(rc, code, text):
    assert rc == code, (rc, _lib.lib.myfa_last_error())
    assert text in _lib.lib.myfa_last_error().decode()


def test_c_abi_refusals_of_window_attention():
    lib, bf16, f32 = _lib.lib, _lib.MYFA_BF16, _lib.MYFA_F32
    st = S3(0, 0, 64)

    def fwd(B=1, H=2, G=1, nq=4, nk=8, d=64, window=4, sinks=0, scale=1.0, dtype=bf16, p=16, st=st):
        return lib.myfa_window_attn_fwd(p, p, p, p, None, None, B, H, G, nq, nk, d, st, st, st, window, sinks, scale, dtype, None)
    _error(fwd(B=-1), 1, "negative")
    _error(fwd(nq=9), 1, "more queries")
    _error(fwd(H=3, G=2), 1, "multiple")
    _error(fwd(G=0), 1, "multiple")
    _error(fwd(window=0), 1, "window")
    _error(fwd(sinks=-1), 1, "negative")
    _error(fwd(scale=0.0), 1, "scale")
    _error(fwd(scale=float("nan")), 1, "scale")
    _error(fwd(scale=float("inf")), 1, "scale")
    _error(fwd(d=60), 2, "head dim")
    _error(fwd(d=264), 2, "head dim")
    _error(fwd(d=132, dtype=f32), 2, "head dim")
    _error(fwd(dtype=7), 1, "dtype")
    _error(fwd(nk=1 << 29), 2, "2^28")
    _error(fwd(B=1 << 20, H=1 << 20), 2, "too many rows")
    _error(fwd(p=None), 1, "null")
    _error(fwd(p=8), 1, "aligned")
    _error(fwd(st=None), 1, "null strides")
    _error(fwd(st=S3(0, 0, 60)), 1, "16 bytes")
    _error(fwd(st=S3(0, 0, -64)), 2, "row stride")
    _error(fwd(st=S3(0, 0, 1 << 23)), 2, "row stride")
    assert fwd(B=0) == 0 and fwd(nq=0) == 0 and fwd(d=0) == 0        # nothing to do: no launch

    def bwd(ws, nbytes, p=16):
        return lib.myfa_window_attn_bwd(*([p] * 9), None, 1, 2, 1, 4, 8, 64, st, st, st, 4, 0, 1.0, bf16, ws, nbytes, None)
    need = lib.myfa_window_attn_bwd_ws_bytes(1, 2, 1, 4, 8, 64, 4, 0, bf16)
    assert need >= 2 * 2 * 4 * 4
    _error(bwd(16, need - 1), 1, "workspace")
    _error(bwd(None, need), 1, "workspace")
    _error(bwd(8, need), 1, "workspace")
    _error(bwd(16, need, p=None), 1, "null")


def test_c_abi_refusals_of_the_paged_cache():
    lib, bf16, f32 = _lib.lib, _lib.MYFA_BF16, _lib.MYFA_F32
    st = S3(2 * 16 * 64, 16 * 64, 64)

    def decode(B=1, H=4, G=2, d=64, pages=8, page=16, width=4, window=0, sinks=0, scale=1.0, dtype=bf16, p=16, ws=None, nbytes=0, st=st):
        return lib.myfa_paged_attn_decode(p, p, p, p, p, p, None, None, B, H, G, d, pages, page, width, st, st, st, window, sinks, scale, dtype, ws, nbytes, None)
    _error(decode(B=-1), 1, "negative")
    _error(decode(page=0), 1, "page")
    _error(decode(G=0), 1, "no heads")
    _error(decode(H=3), 1, "multiple")
    _error(decode(width=1 << 27, page=16), 2, "capacity")
    _error(decode(d=60), 2, "head dim")
    _error(decode(d=256, dtype=f32), 2, "head dim")
    _error(decode(scale=-1.0), 1, "scale")
    _error(decode(dtype=9), 1, "dtype")
    _error(decode(p=None), 1, "null")
    _error(decode(p=4), 1, "aligned")
    _error(decode(st=S3(4, 4, 4)), 1, "16 bytes")
    _error(decode(width=4096), 1, "workspace")                      # long enough to be split
    assert decode(B=0) == 0

    def append(n=1, B=1, p=16, st=st):
        return lib.myfa_paged_append(p, p, p, p, p, p, None, B, 2, n, 64, 8, 16, 4, st, st, st, st, bf16, None)
    _error(append(n=-1), 1, "negative")
    _error(append(n=1 << 28), 2, "chunks")
    _error(append(p=None), 1, "null")
    assert append(n=0) == 0 and append(B=0) == 0

    def evict(budget=8, sinks=0, recent=0, new_width=1, B=1, p=16):
        return lib.myfa_paged_evict(p, p, p, p, p, p, p, p, p, B, 2, 64, 8, 16, 4, new_width, st, st, budget, sinks, recent, bf16, None)
    _error(evict(budget=0), 1, "budget")
    _error(evict(sinks=5, recent=4), 1, "budget")
    _error(evict(sinks=-1), 1, "budget")
    _error(evict(recent=1 << 62, sinks=1), 1, "budget")
    _error(evict(budget=17), 1, "holds 16 keys")
    _error(evict(new_width=-1), 2, "new table")
    _error(evict(p=None), 1, "null")
    assert evict(B=0) == 0


def test_division_by_multiplication():
    """The kernels' x / d (paged_common.h, FastDiv): exact for every divisor and 0 <= x < 2^31."""
    rng = random.Random(0)
    for d in [1, 2, 3, 5, 7, 16, 24, 641, 65535, 65536, 65537, (1 << 28) - 1, 1 << 28] + [rng.randrange(1, 1 << 28) for _ in range(200)]:
        s = 0
        while (1 << s) < d:
            s += 1
        m = ((1 << (31 + s)) + d - 1) // d
        assert m < 1 << 32
        top = ((1 << 31) - 1) // d
        for x in {0, 1, d - 1, d, d + 1, top * d, top * d - 1, (1 << 31) - 1, rng.randrange(1 << 31), rng.randrange(top + 1) * d}:
            if 0 <= x < 1 << 31:
                assert x * m >> (31 + s) == x // d


def test_reference_masks():
    """The definition the GPU tests are held to, on a case small enough to see."""
    got = ref.seen(3, 5, 2, 1, 4).int().tolist()      # positions 2, 3, 4; length 4
    assert got == [[1, 1, 1, 0, 0], [1, 0, 1, 1, 0], [0, 0, 0, 0, 0]]


def test_capacities_that_32_bit_loops_cannot_walk_are_refused():
    """A loop over keys steps past the last one before it ends: close to 2^31 it would wrap and not end.  (Null pointers: what the sizes
    let through stops there, and nothing is launched.)"""
    lib, bf16 = _lib.lib, _lib.MYFA_BF16
    st = S3(2 * 16 * 64, 16 * 64, 64)
    limit = (1 << 31) - (1 << 16)

    def calls(page, width, new_width):
        yield lib.myfa_paged_append(*[None] * 7, 1, 2, 1, 64, 8, page, width, st, st, st, st, bf16, None)
        yield lib.myfa_paged_attn_decode(*[None] * 8, 1, 4, 2, 64, 8, page, width, st, st, st, 0, 0, 1.0, bf16, None, 0, None)
        yield lib.myfa_paged_evict(*[None] * 9, 1, 2, 64, 8, page, width, new_width, st, st, 1, 0, 0, bf16, None)
    for page, width in ((16, (1 << 27) - 1), (1 << 16, (1 << 15) - 1), (1, (1 << 28)), (1 << 28, 7), (16, limit // 16 + 1)):
        for rc in calls(page, width, 1):
            if page * width > limit:
                _error(rc, 2, "capacity")
            else:
                _error(rc, 1, "null")
        assert (lib.myfa_paged_attn_decode_ws_bytes(1, 4, 2, 64, page, width, 0, 0, 0) > 0) == (page * width <= limit)
    _error(list(calls(16, 4, limit // 16 + 1))[2], 2, "new table")
    _error(list(calls(16, 4, limit // 16))[2], 1, "null")


def test_workspace_of_the_window_backward_is_bounded():
    """However many keys are sinks: statistics of every query row, and parts as include/myfa.h bounds them."""
    rng = random.Random(1)
    shapes = [(4, 8, 8, 16384, 128, 256, 8192), (4, 8, 8, 16384, 128, 16, 16384), (1, 1, 1, 16384, 256, 100, 4000), (64, 8, 8, 16384, 128, 256, 4),
              (4, 32, 8, 4096, 128, 1024, 4), (1, 2, 1, 640, 64, 100, 130)]
    for _ in range(2000):
        nk, G = int(2 ** rng.uniform(0, 18)), rng.choice([1, 2, 3, 8, 32])
        shapes.append((int(2 ** rng.uniform(0, 7)), G * rng.choice([1, 2, 8]), G, nk, rng.choice([8, 64, 80, 128]), int(2 ** rng.uniform(0, 18)),
                       rng.choice([0, 1, 4, 100, nk // 2, nk, 1 << 40])))
    split = 0
    for B, H, G, nk, d, window, sinks in shapes:
        for dtype in (_lib.MYFA_BF16, _lib.MYFA_F32) if d <= 128 else (_lib.MYFA_BF16,):
            nq = rng.randrange(1, nk + 1)
            got = _lib.lib.myfa_window_attn_bwd_ws_bytes(B, H, G, nq, nk, d, window, sinks, dtype)
            stats = 8 * B * H * (-(-nq // 64) * 64)
            assert stats <= got <= stats + 2 * 4 * d * max(B * G * (nk + 127), 1024 * 128), (B, H, G, nq, nk, d, window, sinks)
            split += got > stats
    assert split > 200


@pytest.mark.parametrize("host", ["none", "other"])
def test_the_package_without_its_host_module(tmp_path, host):
    """Where the extension module is absent, or is of another torch, dense attention and softmax are there as before it existed, and the
    operators that need it say so."""
    import os
    import subprocess
    import sys
    src, pkg = os.path.dirname(_lib.__file__), tmp_path / "my_flash_attn_cuda"
    pkg.mkdir()
    for name in os.listdir(src):
        if name.endswith(".py") or name == "libmyfa_gfx950.so":
            os.symlink(os.path.join(src, name), pkg / name)
    if host == "other":
        (pkg / "_host.so").write_bytes(b"not for this Python")
    code = """
import torch, my_flash_attn_cuda as m
assert m._lib.__file__.startswith(%r)
x, i = torch.zeros(1, 2, 8, 64), torch.zeros(1, 2, dtype=torch.int32)
def message(call):
    try:
        call()
    except RuntimeError as e:
        return str(e)
for call in (lambda: m.flash_attn_fwd(x, x, x), lambda: m.softmax(x, -1), lambda: m.my_softmax(x[0, 0], 5)):
    assert "must be a CUDA tensor" in message(call), message(call)
for call in (lambda: m.window_attn_fwd(x, x, x, 4), lambda: m.window_attn_func(x, x, x, 4), lambda: m.window_attn_bwd(x, x, x, x, x, x, 4),
             lambda: m.paged_kv_append(x, x, x, x, i, i[0]), lambda: m.paged_attn_decode(x[0], x, x, i, i[0]), lambda: m.paged_kv_evict(x, x, x, i, i[0], i, 4)):
    assert "_host.so does not load" in message(call), message(call)
""" % str(tmp_path)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=tmp_path, env={**os.environ, "PYTHONPATH": str(tmp_path)})
    assert r.returncode == 0, r.stderr


def test_head_dim_of_zero():
    """An output of no elements is written by not launching anything; the other results of such a call are refused."""
    lib, bf16 = _lib.lib, _lib.MYFA_BF16
    st = S3(0, 0, 0)

    def fwd(lse):
        return lib.myfa_window_attn_fwd(16, 16, 16, 16, lse, None, 1, 2, 1, 4, 8, 0, st, st, st, 4, 0, 1.0, bf16, None)

    def decode(lse, sums):
        return lib.myfa_paged_attn_decode(16, 16, 16, 16, 16, 16, lse, sums, 1, 4, 2, 0, 8, 16, 4, st, st, st, 0, 0, 1.0, bf16, None, 0, None)
    assert fwd(None) == 0 and decode(None, None) == 0
    for rc in (fwd(16), decode(16, None), decode(None, 16)):
        _error(rc, 2, "head dim 0")
