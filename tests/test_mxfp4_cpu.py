"""What the 4-bit operators refuse, without a GPU: argument checks happen in front of any launch."""
import pytest
import torch


def _q(rows, k):
    from easyanimate_amd import ops
    kt = (k + 255) // 256
    return ops.Mxfp4(torch.zeros(kt, rows, 128, dtype=torch.uint8), torch.zeros(kt, rows, 8, dtype=torch.uint8), rows, k)


def test_quantize_refuses(lib_built):
    from easyanimate_amd import ops
    with pytest.raises(TypeError):
        ops.mxfp4_quantize(torch.zeros(2, 64))
    for shape in ((64,), (2, 3, 64), (4, 0)):
        with pytest.raises(ValueError):
            ops.mxfp4_quantize(torch.zeros(shape, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="GPU"):
        ops.mxfp4_quantize(torch.zeros(2, 64, dtype=torch.bfloat16))


def test_storage_refuses(lib_built):
    from easyanimate_amd import ops
    q = _q(4, 300)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.mxfp4_dequantize(q)
    ok = dict(codes=q.codes, scales=q.scales, rows=4, k=300)
    ops.Mxfp4(**ok)
    for bad in (dict(k=600), dict(k=0), dict(rows=5), dict(scales=q.scales[:1]), dict(codes=torch.zeros(2, 128, 4, dtype=torch.uint8).transpose(1, 2)),
                dict(codes=torch.zeros(2 * 4 * 128 + 8, dtype=torch.uint8)[8:].view(2, 4, 128))):
        with pytest.raises(ValueError):
            ops.Mxfp4(**{**ok, **bad})
    with pytest.raises(TypeError):
        ops.Mxfp4(**{**ok, "codes": q.codes.int()})
    with pytest.raises(RuntimeError):
        ops.Mxfp4(**{**ok, "codes": q.codes.to("meta")})


def test_product_refuses(lib_built):
    from easyanimate_amd import ops
    W = _q(16, 64)
    x = torch.zeros(3, 64, dtype=torch.bfloat16)
    for args in ((x.float(), W), (x, torch.zeros(16, 64, dtype=torch.bfloat16))):
        with pytest.raises(TypeError):
            ops.gemm_mxfp4(*args, None)
    for bad in (torch.zeros(64, dtype=torch.bfloat16), torch.zeros(3, 96, dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            ops.gemm_mxfp4(bad, W, None)
    with pytest.raises(ValueError):
        ops.gemm_mxfp4(_q(3, 32), W, None)
    with pytest.raises(ValueError):
        ops.gemm_mxfp4(x, W, None, 9)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.gemm_mxfp4(x, W, None)


def test_abi_refuses(lib_built):
    """The C entries: no launch, EA_ERR_ARG and a message."""
    from easyanimate_amd import _lib
    lib = _lib.load()
    p = 1 << 20      # an aligned address that nothing reads: every call below ends in front of the launch

    def gemm(A=p, As=p, X=None, W=p, Ws=p, bias=None, C=p, res=None, gate=None, batch=1, M=4, N=16, K=64, lda=64, abs_=0, ldc=16, cbs=0, ldres=0,
             rbs=0, gbs=0, epi=0, ws=None, wsb=0):
        return lib.ea_gemm_mxfp4(A, As, X, W, Ws, bias, C, res, gate, batch, M, N, K, lda, abs_, ldc, cbs, ldres, rbs, gbs, epi, ws, wsb, None)

    bad = [dict(A=None), dict(As=None), dict(W=None), dict(Ws=None), dict(C=None), dict(X=p), dict(N=12), dict(N=0), dict(K=0), dict(M=-1),
           dict(batch=0), dict(batch=70000), dict(ldc=8), dict(X=p, A=None, As=None, batch=2, ws=p, wsb=1 << 20), dict(ldc=12), dict(cbs=4), dict(epi=4), dict(epi=-1), dict(epi=2), dict(epi=2, res=p), dict(C=p + 8),
           dict(A=p + 4), dict(As=p + 4), dict(bias=p + 4), dict(A=None, As=None, X=p, M=17), dict(A=None, As=None, X=p, K=60),
           dict(A=None, As=None, X=p, lda=60), dict(A=None, As=None, X=p, lda=-8), dict(A=None, As=None, X=p + 1), dict(M=100, K=16384),
           dict(M=100, K=16384, ws=p, wsb=64), dict(M=100, K=16384, ws=p + 8, wsb=1 << 30),
           dict(epi=2, res=p, gate=p, ldres=12), dict(epi=2, res=p, gate=p, gbs=2), dict(epi=2, res=p + 4, gate=p)]
    for kw in bad:
        assert gemm(**kw) == -1, kw
        assert b"ea_gemm_mxfp4" in lib.ea_last_error_string()
    assert gemm(M=0) == 0 and gemm(M=0, A=None, As=None, C=None) == 0
    ws = lib.ea_gemm_mxfp4_workspace_bytes
    assert ws(1, 16, 64, 1 << 20, 0) == 0 and ws(1, 100, 256, 16384, 0) > 0 and ws(0, 100, 256, 16384, 0) == 0
    assert ws(2, 3, 64, 500, 1) == 2 * 2 * 3 * 128 + 256         # two K tiles of six rows: codes, scale bytes up to a whole 256
    quant = lambda x=p, c=p, s=p, rows=4, K=64, ld=64: lib.ea_mxfp4_quantize_bf16(x, c, s, rows, K, ld, None)
    for kw in (dict(x=None), dict(c=None), dict(s=None), dict(rows=-1), dict(K=0), dict(ld=63), dict(c=p + 8), dict(s=p + 4), dict(rows=1 << 40)):
        assert quant(**kw) == -1, kw
    assert quant(rows=0, x=None) == 0
    deq = lambda c=p, s=p, y=p, rows=4, K=64: lib.ea_mxfp4_dequantize_bf16(c, s, y, rows, K, None)
    for kw in (dict(c=None), dict(s=None), dict(y=None), dict(rows=-1), dict(K=-3), dict(y=p + 2), dict(rows=1 << 40)):
        assert deq(**kw) == -1, kw
    assert deq(rows=0) == 0
