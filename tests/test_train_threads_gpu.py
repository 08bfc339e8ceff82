"""The enqueue-only calls from several threads: shared contexts, and backwards,
which torch runs on a thread of its own."""
import os
import subprocess
import sys
import threading

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_threads_share_a_context():
    # the first calls on a context, together; one of them has a bad id, which is
    # reported once, to whichever thread asks first
    import ctypes

    import torch
    from shear_b200 import _capi as C, ops
    lib = C.load()
    table = torch.randn(100, 32, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(8)]
    out = torch.empty(8, 50, 32, device="cuda")
    for turn in range(60):
        ctx, bad, codes = ops.Context(0), turn % 8, []
        ids = torch.randint(0, 100, (8, 50), device="cuda")
        ids[bad, 7] = 100
        args = [C.LookupArgs(table.data_ptr(), 100, 32, 32, 0, ids[i].data_ptr(), 64, 0, 50, 1.0, out[i].data_ptr(), 32)
                for i in range(8)]
        torch.cuda.synchronize()
        start = threading.Barrier(8)

        def work(i, call=lib.tessa_embedding_lookup, status=lib.tessa_async_status, h=ctx.handle):
            arg, stream = args[i], ctypes.c_void_p(streams[i].cuda_stream)
            start.wait(30)
            codes.append(call(h, arg, stream))
            codes.append(status(h, stream))

        threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
        for t in threads:
            t.start()
        for t in threads:
            t.join(60)
        torch.cuda.synchronize()
        codes.append(lib.tessa_async_status(ctx.handle, None))
        assert len(codes) == 17 and sorted(codes) == [-5] + [0] * 16, (turn, codes)
        ctx.close()


@pytest.mark.parametrize("name", ["lookup", "distill"])
def test_an_error_in_a_backward_reaches_the_caller(name):
    import torch
    from shear_b200 import ops, train
    from shear_b200._capi import TessaError
    t = torch.randn(20, 30, device="cuda").requires_grad_()
    ids = torch.randint(0, 20, (20, 3), device="cuda")
    y = train.lookup(t, ids) if name == "lookup" else train.distill(t, ids, torch.randn(20, 3, device="cuda"))
    ops.async_status()
    ids.data[4, 1] = 30  # between the two
    y.sum().backward()
    with pytest.raises(TessaError) as e:
        ops.async_status()
    assert e.value.code == -5
    ops.async_status()


CAPTURE = """
import torch
from shear_b200 import ops, train
g = torch.Generator().manual_seed(0)
rand = lambda *s: torch.randn(*s, generator=g).cuda().requires_grad_()
table, x, w, z = rand(50, 32), rand(40, 64), rand(30, 64), rand(8, 90)
ids, lists, teacher = (torch.randint(0, 50, (20,), generator=g).cuda(), torch.randint(0, 90, (8, 4), generator=g).cuda(),
                       torch.randn(8, 4, generator=g).cuda())
def forward():
    return train.lookup(table, ids).sum(), train.product_fp8(x, w).sum(), train.distill(z, lists, teacher).sum()
def backward(y):
    return torch.autograd.grad(y, (table, x, w, z))
side = torch.cuda.Stream()
with torch.cuda.stream(side):
    forward()  # no backward has run when the capture begins
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        grads = backward(sum(forward()))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(grads, backward(sum(forward()))):
        assert torch.equal(a, b) and a.abs().sum() > 0
ops.async_status()
print("same")
"""


def test_a_first_backward_inside_a_capture():
    run = subprocess.run([sys.executable, "-c", CAPTURE], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip() == "same", run.stderr[-2000:]
