"""gemm_mxfp4 does not work in place: a result that begins where an operand does is refused in front of any launch."""
import pytest


@pytest.mark.parametrize("which", ["A", "X", "W"])
def test_a_result_on_an_operand_is_refused(lib_built, which):
    from easyanimate_amd import _lib
    lib = _lib.load()
    at = {n: (i + 1) << 20 for i, n in enumerate(("A", "As", "W", "Ws"))}          # aligned addresses that nothing reads
    x = 9 << 20
    M, N, K = 4, 64, 64
    stored = which != "X"
    c = x if which == "X" else at[which]
    rc = lib.ea_gemm_mxfp4(at["A"] if stored else None, at["As"] if stored else None, None if stored else x, at["W"], at["Ws"], None, c, None, None,
                           1, M, N, K, K, 0, N, 0, 0, 0, 0, 0, None, 0, None)
    assert rc == -1 and b"must not overlap" in lib.ea_last_error_string()
