"""The row arithmetic that the 256 x 256 kernel of gemm_mxfp4 takes from csrc/ea_mxfp4_rows.h, evaluated on the host: every 16-byte
request for scales, of every workgroup, wave, lane and K tile, stays inside the operand's scale buffer, and the rows that are stored get
their own scales.  The buffers are as large as the library says they are."""
import ctypes
import os
import random
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MAIN = r"""
#include "ea_mxfp4_rows.h"
// requests of the kernel for an operand of `rows` rows in kt K tiles, scale buffer of `bytes`: tiles of 256 rows from `first` on,
// `own` of them this element's.  0 = fine, 1 = a request leaves the buffer, 2 = a stored row without its scales
extern "C" int check(long long rows, long long first, long long own, long long kt, long long bytes) {
    for (long long row0 = 0; row0 < own; row0 += 256)
        for (int half = 0; half < 2; ++half)
            for (int lane = 0; lane < 64; ++lane) {
                const long long in = row0 + half * 128 + 2 * lane;
                const long long at = mxw4_scale_offset(first + in, rows);
                for (long long t = 0; t < kt; t += kt > 1 ? kt - 1 : 1) {
                    const long long from = t * rows * 8 + at;
                    if (from < 0 || from + 16 > bytes) return 1;
                }
                for (int e = 0; e < 2; ++e)
                    if (in + e < own && at + 8 * e != (first + in + e) * 8) return 2;
            }
    return 0;
}
extern "C" int pad() { return MXW4_SCALE_PAD; }
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not found")
    d = tmp_path_factory.mktemp("rows")
    src, so = str(d / "main.cpp"), str(d / "rows.so")
    open(src, "w").write(MAIN)
    subprocess.run([gxx, "-std=c++17", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, "easyanimate_amd", "csrc"), src, "-o", so], check=True)
    lib = ctypes.CDLL(so)
    lib.check.argtypes = [ctypes.c_longlong] * 5
    return lib


def _cases():
    rng = random.Random(5)
    yield from [(1, 256, 256, 1), (1, 257, 264, 1), (3, 3841, 1000, 7), (2, 3999, 8200, 14), (1, 4096, 18944, 14), (5, 129, 8, 2), (7, 1, 16, 3)]
    for _ in range(200):
        yield rng.randint(1, 6), rng.randint(1, 5000), 8 * rng.randint(1, 2400), rng.randint(1, 75)


def test_scale_requests_stay_inside(lib_built, host):
    from easyanimate_amd import _lib
    workspace = _lib.load().ea_gemm_mxfp4_workspace_bytes
    for batch, M, N, kt in _cases():
        assert host.check(N, 0, N, kt, N * kt * 8) == 0, ("weights", N, kt)              # N % 8 == 0: no pad needed
        a_rows = batch * M
        if a_rows < 2:
            continue
        # activations quantised into the workspace: codes, scales (and, in other plans, partial products behind them)
        scales = workspace(batch, M, N, 256 * kt, 1) - a_rows * kt * 128
        assert scales >= a_rows * kt * 8 + host.pad()
        for b in range(batch):
            assert host.check(a_rows, b * M, M, kt, a_rows * kt * 8 + host.pad()) == 0, (batch, M, kt, b)
        if batch == 1 and M % 2 == 0:                                                    # stored by the caller: nothing behind them
            assert host.check(M, 0, M, kt, M * kt * 8) == 0, (M, kt)


def test_the_check_sees_a_request_outside(host):
    """An odd number of rows without the pad does not fit: the last pair reaches 8 bytes behind the last K tile."""
    assert host.check(257, 0, 257, 3, 257 * 3 * 8) == 1
