"""The FP8 product at its limits: of waits, of sums of one sign, of shapes."""
import pytest

pytestmark = pytest.mark.gpu


def test_a_product_longer_than_the_wait_limit():
    # the limit is one wait's, not the call's: a product of several times the
    # least limit is no timeout
    import torch
    from shear_b200 import _capi as C, ops
    lib, ctx = C.load(), ops.Context(0)
    c = torch.full((65_536, 8192), 0x38, dtype=torch.uint8, device="cuda")  # ones
    s = torch.full((65_536, 64), 127, dtype=torch.uint8, device="cuda")
    out = torch.empty(65_536, 65_536, dtype=torch.bfloat16, device="cuda")
    times = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    ops.matmul_fp8(c[:256], s[:256], c[:256], s[:256], ctx=ctx)
    assert lib.tessa_set_wait_timeout_ns(ctx.handle, 10_000_000) == 0
    times[0].record()
    ops.matmul_fp8(c, s, c, s, out=out, ctx=ctx)
    times[1].record()
    ops.async_status(ctx)
    assert times[0].elapsed_time(times[1]) > 15.0  # 70 TFLOP, so that the test is one
    assert (out == 8192).all()
