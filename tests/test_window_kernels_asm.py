"""What the window and paged kernels need of their generated gfx950 code: the hand-written MFMA forms keep the result
latency, loops with MFMAs are free of scratch traffic, LDS and registers fit the workgroups a CU is meant to hold, and no
packed float32 arithmetic is generated.  CPU-only: hipcc cross-compiles."""
import functools
import importlib.util
import os
import re
import shutil

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
needs_hipcc = pytest.mark.skipif(not (shutil.which("hipcc") or os.path.exists("/opt/rocm/bin/hipcc")), reason="needs hipcc")


def _load(name, path):
    spec = importlib.util.spec_from_file_location(name, path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


chk = _load("check_mfma_hazards", os.path.join(ROOT, "tools", "check_mfma_hazards.py"))
build = _load("myfa_build", os.path.join(ROOT, "flash-attention_amd", "build.py"))
SOURCES = ["window_attn_fwd.hip", "window_attn_bwd.hip", "paged_attn.hip", "paged_evict.hip"]


@functools.lru_cache(None)
def _asm(src):
    at = build.FLAGS.index("-Xclang")
    return chk.compile_to_asm(os.path.join(build.CSRC, src), build.PER_SOURCE_FLAGS.get(src, []) + build.FLAGS[at:at + 4])


def _kernels(asm):
    """name -> (lines of its code, metadata)"""
    meta = {}
    for block in re.split(r"\n  - \.agpr_count:", asm)[1:]:
        name = re.search(r"\.name:\s+(\S+)", block).group(1)
        meta[name] = {k: int(v) for k, v in re.findall(r"\.(\w+):\s+(\d+)\s*$", block.split("\namdhsa")[0], re.M)}
    code = {}
    for body in re.split(r"\n\s*\.end_amdhsa_kernel", asm):
        m = re.search(r"^(_ZN4myfa\S+):", body, re.M)
        if m:
            code[m.group(1)] = body[m.end():].split("\n")
    return {n: (code[n], meta[n]) for n in meta if n in code}


def _innermost_mfma_loops(lines):
    labels = {ln.split(":")[0]: i for i, ln in enumerate(lines) if re.match(r"^\.LBB\d+_\d+:", ln)}
    loops = []
    for i, ln in enumerate(lines):
        b = re.match(r"^\s+s_c?branch\w*\s+(\.LBB\d+_\d+)", ln)
        if b and labels.get(b.group(1), i + 1) < i:
            loops.append((labels[b.group(1)], i))
    loops = [(a, z) for a, z in loops if sum("v_mfma" in ln for ln in lines[a:z]) >= 8]
    return [(a, z) for a, z in loops if not any((c, e) != (a, z) and a <= c and e <= z for c, e in loops)]


@needs_hipcc
def test_result_latency_of_hand_written_products():
    seen, bad = chk.check(_asm("window_attn_bwd.hip"))
    assert seen >= 2 * 2 * 32, "the kernels' hand-written MFMAs were not found in the assembly"
    assert bad == [], "\n".join(bad[:10])


@needs_hipcc
@pytest.mark.parametrize("src", SOURCES)
def test_no_packed_float32(src):
    assert re.findall(r"\bv_pk_(?:add|mul|fma)_f32\b", _asm(src)) == []


@needs_hipcc
@pytest.mark.parametrize("src", ["window_attn_fwd.hip", "window_attn_bwd.hip", "paged_attn.hip"])
def test_resources(src):
    kernels = _kernels(_asm(src))
    assert len(kernels) >= (9 if src == "paged_attn.hip" else 16)
    for name, (lines, r) in kernels.items():
        assert r["group_segment_fixed_size"] <= 160 * 1024, (name, r)
        if re.search(r"(fwd16|dq16)_kernel", name):                                    # two workgroups of four waves a CU
            assert r["vgpr_count"] <= 256 and 2 * r["group_segment_fixed_size"] <= 160 * 1024, (name, r)
        loops = _innermost_mfma_loops(lines)
        if "mfma" in "".join(lines):
            assert loops, name
        for a, z in loops:
            assert not [ln for ln in lines[a:z] if "scratch_" in ln], (name, a, z)
