"""Outputs that the caller gives: what autograd knows of them, and where they may lie."""
import pytest

pytestmark = pytest.mark.gpu


def _calls(torch, ops):
    """(a tensor to write to, the call that writes to it)"""
    table, ids = torch.randn(20, 32, device="cuda"), torch.randint(0, 20, (6,), device="cuda")
    c, s = ops.quantize_fp8(table)
    return {
        "lookup": (6, lambda out: ops.embedding_lookup(table, ids, out=out)),
        "lookup's gradient": (20, lambda out: ops.embedding_grad(table[:6], ids, 20, out=out)),
        "added gradient": (20, lambda out: ops.embedding_grad(table[:6], ids, 20, out=out, accumulate=True)),
        "product": (20, lambda out: ops.matmul_fp8(c, s, *ops.quantize_fp8(torch.randn(32, 32, device="cuda")), out=out)),
        "distillation": (6, lambda out: ops.distill_topk_grad(out, ids.view(6, 1), ids.float().view(6, 1), out=out)),
    }


@pytest.mark.parametrize("name", ["lookup", "lookup's gradient", "added gradient", "product", "distillation"])
def test_a_graph_that_saved_the_output_finds_it_written(name):
    import torch
    from shear_b200 import ops
    rows, call = _calls(torch, ops)[name]
    x = torch.randn(rows, 32, device="cuda").requires_grad_()
    y = x * 2.0
    saved = y.square().sum()
    call(y.detach())  # shares y's memory, as torch's own in-place calls on it do
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.backward()
    # outputs that the call makes, and refused calls, leave everything as it was
    with torch.inference_mode():
        z = torch.empty(rows, 32, device="cuda")
        call(z.normal_())
    call(z)  # (an inference tensor counts no versions)
    ops.async_status()


def _strided(torch, flat, rows, cols, step, at):
    return torch.as_strided(flat, (rows, cols), (step, 1), at)


@pytest.mark.parametrize("rows,logits,out", [  # (row stride, first element) of rows of 100
    (6, (100, 0), (100, 100)), (6, (100, 100), (100, 0)),    # one row on, one row back
    (6, (200, 0), (200, 50)), (6, (200, 150), (200, 0)),     # columns in common, or the neighbour's
    (1, (100, 0), (100, 99)), (2, (300, 0), (300, 399)),     # one element
    (4, (200, 0), (400, 350)), (4, (150, 500), (1000, 0)),   # strides that meet later
])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_gradient_that_overlaps_the_logits_is_refused(rows, logits, out, dtype):
    import torch
    from shear_b200 import ops
    from shear_b200._capi import TessaError
    flat = torch.randn(8000, device="cuda").to(getattr(torch, dtype))
    before = flat.clone()
    ids, t = torch.randint(0, 100, (rows, 3), device="cuda"), torch.randn(rows, 3, device="cuda")
    with pytest.raises(TessaError) as e:
        ops.distill_topk_grad(_strided(torch, flat, rows, 100, *logits), ids, t, out=_strided(torch, flat, rows, 100, *out))
    assert e.value.code == -1 and torch.equal(flat, before)


@pytest.mark.parametrize("rows,logits,out", [
    (6, (200, 0), (200, 100)), (6, (200, 100), (200, 0)),    # side by side
    (6, (201, 0), (201, 101)), (1, (100, 0), (100, 100)), (3, (100, 0), (100, 300)),
    (3, (400, 0), (200, 100)), (2, (1000, 300), (500, 0)),   # in each other's gaps
    (6, (200, 0), (200, 0)),                                 # in place
])
def test_a_gradient_beside_the_logits(rows, logits, out):
    import torch
    from shear_b200 import ops
    flat = torch.randn(8000, device="cuda")
    ids, t = torch.randint(0, 100, (rows, 3), device="cuda"), torch.randn(rows, 3, device="cuda")
    z = _strided(torch, flat, rows, 100, *logits)
    want = ops.distill_topk_grad(z, ids, t)
    got = ops.distill_topk_grad(z, ids, t, out=_strided(torch, flat, rows, 100, *out))
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_the_least_temperatures():
    # all weight on the largest logit, in list and row, or a refusal; never NaN
    import torch
    from shear_b200 import ops
    from shear_b200._capi import TessaError
    z, t = torch.tensor([[0.5, 1.0, -1.0, 1.0]], device="cuda"), torch.tensor([[0.25, 1.0]], device="cuda")
    ids = torch.tensor([[1, 0]], device="cuda")
    for tau in (1e-38, 4.3e-39):
        _, lse, grad = ops.distill_topk_grad(z, ids, t, tau, row_weights=torch.full((1,), 1e37, device="cuda"))
        scale = float(torch.tensor(tau).double()) * float(torch.tensor(1e37).double())
        want = torch.tensor([[-scale, scale / 2, 0.0, scale / 2]], device="cuda")
        assert torch.allclose(grad, want, rtol=1e-5, atol=0) and lse.isfinite().all()
    for tau in (4.2e-39, 1e-40, 1e-45):
        with pytest.raises(TessaError) as e:
            ops.distill_topk_grad(z, ids, t, tau)
        assert e.value.code == -1
