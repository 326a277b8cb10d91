"""The text operators' kernels behind the electric-fence allocator (see test_fence_gpu.py): every operand, workspace and result ends
(mode left: starts) at an unmapped page.  Graphs and side streams stay out: that allocator knows neither."""
import pytest

from test_fence_gpu import _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", ["right", "left"])
@pytest.mark.parametrize("file,select", [("test_mxfp4_gpu.py", "sizes or strides or read_back or (product_variants and not 16000) or (large_tiles and plain) or "
                                          "large_tiles_batched or product_batched or writes_where"),
                                         ("test_mxfp4_stored_gpu.py", "batches or (71 and plain)"),
                                         ("test_attention_text_gpu.py", "causal_sizes or no_mask or forms or long or strides or nothing or start")],
                         ids=["mxfp4", "stored", "attention"])
def test_text_operators_behind_the_fence(file, select, mode):
    r = _run(["-m", "pytest", f"tests/{file}", "-q", "-m", "gpu", "-p", "no:cacheprovider", "-x", "-k", select], env={"EA_GUARD_MODE": mode})
    tail = r.stdout[-1500:] + r.stderr[-1500:]
    print(f"[fence] {file} mode {mode}: rc {r.returncode}\n{tail}")
    assert r.returncode == 0 and "passed" in r.stdout and "slack_hits=0" in r.stderr, tail
    assert "Memory access fault" not in r.stderr and "OUT-OF-BOUNDS" not in r.stderr, tail
