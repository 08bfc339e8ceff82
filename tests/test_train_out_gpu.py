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
