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
