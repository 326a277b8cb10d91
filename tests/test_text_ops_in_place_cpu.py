"""gemm_mxfp4 and attention_text do not work in place: a result that begins where an operand does is refused in front of any launch."""
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


@pytest.mark.parametrize("which", [0, 1, 2])
def test_attention_does_not_work_in_place_either(lib_built, which):
    import ctypes
    from easyanimate_amd import _lib
    lib = _lib.load()
    qkv = [1 << 20, 2 << 20, 3 << 20]
    strides = (ctypes.c_int64 * 11)(*((512, 128, 64) * 3 + (1280, 256)))
    rc = lib.ea_attention_text_bf16(*qkv, qkv[which], ctypes.addressof(strides), 1, 4, 2, 5, 9, 64, 1.0, 0, 0.0, None, 0, None, None, 0, 0, None, None, None,
                                    None, 0, None)
    assert rc == -1 and b"must not overlap" in lib.ea_last_error_string()
