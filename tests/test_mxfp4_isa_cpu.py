"""Static checks of the 4-bit GEMM kernels' and the text attention kernels' ISA (no GPU needed: hipcc cross-compiles): the hand-placed
256 x 256 loop is what its generator writes, its accumulators are read before the compiler reuses them, and no kernel of the four
sources uses scratch memory beyond what is stated."""
import os
import re
import subprocess
import sys

import pytest

sys.path.insert(0, os.path.dirname(__file__))
from test_w4a_isa_cpu import CSRC, HIPCC, ROOT, _analyse

SOURCES = ("ea_gemm.hip", "ea_gemm_mxfp4.hip", "ea_mxfp4.hip", "ea_attention_text.hip")


@pytest.fixture(scope="module")
def isa(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip(f"{HIPCC} not found: the ISA check needs the cross-compiler")
    d = tmp_path_factory.mktemp("isa")
    out = {}
    for src in SOURCES:
        o = str(d / (src + ".s"))
        r = subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Wno-unused-value", "-Wno-inline-asm", "-Xclang", "-target-feature",
                            "-Xclang", "-packed-fp32-ops", "-x", "hip", "-S", "--cuda-device-only", os.path.join(CSRC, src), "-o", o],
                           capture_output=True, text=True)
        assert r.returncode == 0, r.stderr[-2000:]
        out[src] = open(o).read().split("\n")
    return out


def _kernels(text, fragment):
    for i, l in enumerate(text):
        if re.match(rf"_ZN\w*{fragment}\w*:", l):
            yield l.split(":")[0], text[i:next(k for k in range(i, len(text)) if ".end_amdhsa_kernel" in text[k])]


def test_the_256_kernel(isa):
    found = list(_kernels(isa["ea_gemm.hip"], "gemm256_mxfp4_w4_kernel"))
    assert found
    for name, body in found:
        # (one address of the epilogue may wait out the loop in scratch memory)
        assert sum("scratch_" in l for l in body) <= 2 and not any(re.search(r"v_pk_(add|mul|fma)_f32", l) for l in body)
        errors, _, _, n_loop_mfma, _ = _analyse(name, body)
        assert n_loop_mfma == [256], (name, n_loop_mfma)                       # two K tiles of 2 x 64 products
        assert not errors, "\n".join(errors[:10])


def test_generated_loop_is_the_committed_one(tmp_path):
    out = str(tmp_path / "x.inc")
    env = {k: v for k, v in os.environ.items() if not k.startswith("EA_W4A_")}
    env["EA_GEN_OUT"] = out
    r = subprocess.run([sys.executable, os.path.join(ROOT, "tools", "gen_gemm_mxfp4_asm.py")], env=env, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-1500:]
    text = open(out).read()
    assert text == open(os.path.join(CSRC, "ea_gemm_mxfp4_w4_loop.inc")).read()
    loop = text[text.index('"1:'):text.index("s_cbranch_scc1 1b")]              # its one way out in the middle: an odd number of tiles
    assert loop.count("v_mfma") == 256 and re.findall(r"s_c?branch\w* \w+", loop) == ["s_cbranch_scc0 9f"]


@pytest.mark.parametrize("src,fragment,count", [("ea_gemm_mxfp4.hip", "gemm_mxfp4", None), ("ea_mxfp4.hip", "mxfp4", None), ("ea_attention_text.hip", "attention_text", 28)])
def test_scratch_and_no_packed_fp32(isa, src, fragment, count):
    found = list(_kernels(isa[src], fragment))
    assert found and (count is None or len(found) == count), [n for n, _ in found]
    for name, body in found:
        assert not [l for l in body if re.search(r"v_pk_(add|mul|fma)_f32", l)], name
        size = [int(l.split()[-1]) for l in body if ".amdhsa_private_segment_fixed_size" in l]
        # (three workgroups per CU at D = 64: a few registers of the bias forms spill, and that is faster than two)
        allowed = 128 if "attention_text_kernelILi64E" in name and "ELb1EEE" in name else 0
        assert len(size) == 1 and size[0] <= allowed, (name, size)
