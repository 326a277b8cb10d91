"""What ops.attention_text refuses, without a GPU."""
import ctypes

import pytest
import torch


def _t(*s, dtype=torch.bfloat16):
    return torch.zeros(*s, dtype=dtype)


def test_refuses(lib_built):
    from easyanimate_amd import ops
    q, k = _t(2, 4, 5, 64), _t(2, 2, 9, 64)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.attention_text(q, k, k, 0.125)
    for a in ((q.float(), k, k), (q, k.half(), k), (q, k, k.float())):
        with pytest.raises(TypeError):
            ops.attention_text(*a, 0.125)
    for a in ((q[0], k, k), (q, k, _t(2, 2, 8, 64)), (q, _t(1, 2, 9, 64), _t(1, 2, 9, 64)), (q, _t(2, 3, 9, 64), _t(2, 3, 9, 64)),
              (q, _t(2, 2, 9, 128), _t(2, 2, 9, 128)), (_t(2, 4, 5, 80), _t(2, 2, 9, 80), _t(2, 2, 9, 80))):
        with pytest.raises(ValueError):
            ops.attention_text(*a, 0.125)
    for s in (0.0, -1.0, 2e30, float("inf"), float("nan")):
        with pytest.raises(ValueError):
            ops.attention_text(q, k, k, s)
    for kw in (dict(cap=-1.0), dict(cap=1e-31), dict(cap=1e31), dict(cap=float("nan")), dict(cap=float("inf")), dict(bias=_t(4, 8, dtype=torch.float32)), dict(bias=_t(3, 9, dtype=torch.float32)),
               dict(bias=_t(4, 18, dtype=torch.float32)[:, ::2]), dict(q_docs=i(2, 5)), dict(kv_docs=i(2, 9)), dict(q_docs=i(2, 9), kv_docs=i(2, 9)),
               dict(q_docs=i(2, 5), kv_docs=i(9, 2).t()), dict(prefix=i(2)), dict(prefix=i(3), causal=True), dict(valid=i(1)), dict(q_start=i(2, 1))):
        with pytest.raises(ValueError):
            ops.attention_text(q, k, k, 0.125, **kw)
    for kw in (dict(valid=torch.zeros(2)), dict(q_start=torch.zeros(2, dtype=torch.int64)), dict(bias=_t(4, 9)), dict(q_docs=_t(2, 5), kv_docs=_t(2, 9))):
        with pytest.raises(TypeError):
            ops.attention_text(q, k, k, 0.125, **kw)


def test_abi_refuses(lib_built):
    from easyanimate_amd import _lib
    lib = _lib.load()
    p = 1 << 20            # an aligned address that nothing reads: every call ends in front of the launch

    def call(q=p, k=p, v=p, out=p, strides=(512, 128, 64) * 3 + (512, 256), B=1, Hq=4, Hkv=2, Sq=5, Sk=9, D=64, scale=1.0, causal=0, cap=0.0, bias=None,
             reach=0, qd=None, kd=None, prefix=None, valid=None, start=None, ws=None, wsb=0):
        arr = (ctypes.c_int64 * 11)(*strides) if strides else None
        return lib.ea_attention_text_bf16(q, k, v, out, ctypes.addressof(arr) if arr else None, B, Hq, Hkv, Sq, Sk, D, scale, causal, cap, bias, reach, qd, kd, 0,
                                          0, prefix, valid, start, ws, wsb, None)

    st = lambda i, v: tuple(v if n == i else 256 for n in range(11))
    bad = [dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(strides=None), dict(q=p + 8), dict(out=p + 2), dict(B=0), dict(Hkv=3), dict(Hkv=0),
           dict(Sq=-1), dict(Sk=0), dict(Sk=-5), dict(D=80), dict(D=256), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
           dict(cap=-1.0), dict(cap=float("nan")), dict(bias=p, reach=-1), dict(qd=p), dict(kd=p), dict(prefix=p), dict(strides=st(1, 4)), dict(strides=st(9, -8)), dict(strides=st(5, 1 << 24)), dict(strides=st(8, 1 << 24)),
           dict(strides=st(10, 248)), dict(strides=st(9, 0), B=2), dict(scale=2e30), dict(cap=1e-31), dict(cap=1e31), dict(cap=1e-20, scale=1e12), dict(B=65535, Hq=512),
           
           dict(qd=p, kd=p, Sq=40), dict(Sq=64, Sk=4096), dict(Sq=64, Sk=4096, ws=p, wsb=16), dict(Sq=0x7fffffff), dict(B=70000)]
    for kw in bad:
        assert call(**kw) == -1, kw
        assert b"ea_attention_text_bf16" in lib.ea_last_error_string()
    assert call(Sq=0) == 0
    ws = lib.ea_attention_text_workspace_bytes
    assert ws(1, 4, 2, 1, 100, 64, 0) == 0 and ws(1, 4, 2, 1, 16384, 128, 0) > 0 and ws(1, 4, 2, 5, 0, 64, 0) == 0 and ws(1, 4, 3, 5, 9, 64, 0) == 0
    assert ws(2, 64, 64, 512, 512, 64, 1) == 2 * 8 * 8          # the documents' range per 64-key tile
