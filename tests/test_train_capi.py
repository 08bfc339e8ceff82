"""The training calls' C ABI: arguments that the host refuses before any launch."""
import ctypes

import pytest

from shear_b200 import _capi as C

INVALID, UNSUPPORTED = -1, -6


def test_null_arguments():
    lib = C.load()
    n = ctypes.c_uint64(7)
    calls = [
        lambda: lib.tessa_embedding_lookup(None, C.LookupArgs(), None),
        lambda: lib.tessa_embedding_grad(None, C.LookupGradArgs(), None, 0, None),
        lambda: lib.tessa_embedding_grad_workspace(1, 1, 1, None),
        lambda: lib.tessa_quantize_fp8(None, C.Fp8QuantizeArgs(), None),
        lambda: lib.tessa_matmul_fp8(None, C.Fp8MatmulArgs(), None, 0, None),
        lambda: lib.tessa_matmul_fp8_workspace(None, 1, 1, 16, n),
        lambda: lib.tessa_distill_topk(None, C.DistillArgs(), None, 0, None),
        lambda: lib.tessa_distill_topk_workspace(None, n),
        lambda: lib.tessa_distill_topk_workspace(C.DistillArgs(), None),
    ]
    for call in calls:
        assert call() == INVALID
        assert lib.tessa_last_error_message()


def test_workspace_sizes():
    # sizes need no device: they grow with the work, and nothing needs nothing
    lib = C.load()

    def grad(count, rows, dim):
        n = ctypes.c_uint64()
        C.check(lib.tessa_embedding_grad_workspace(count, rows, dim, n))
        return n.value

    assert grad(0, 10, 10) == 0
    assert grad(1, 10, 10) <= grad(1000, 10, 10) <= grad(10_000, 10, 10) < grad(10_000, 10, 1000) < grad(100_000, 10, 1000)
    assert grad(100_000, 1000, 64) % 256 == 0

    def distill(rows, vocab, k, grad_at):
        n = ctypes.c_uint64()
        C.check(lib.tessa_distill_topk_workspace(
            C.DistillArgs(None, rows, vocab, vocab, 1, k, None, None, 32, 1.0, None, None, None, grad_at, vocab), n))
        return n.value

    assert distill(100, 1000, 32, 256) == 0 and distill(100, 1_000_000, 32, None) == 0
    assert distill(100, 1_000_000, 32, 256) >= 100 * 32 * 12


@pytest.mark.gpu
def test_refusals_before_any_launch():
    import torch
    from shear_b200 import ops
    lib, h = C.load(), ops.context(0).handle
    f = torch.zeros(1 << 16, device="cuda")
    i = torch.zeros(4096, dtype=torch.int32, device="cuda")
    ws = torch.zeros(1 << 22, dtype=torch.uint8, device="cuda")
    p, q, w = f.data_ptr(), i.data_ptr(), ws.data_ptr()

    def refused(call, args, *rest, code=INVALID):
        got = call(h, args, *rest)
        assert got == code, (got, lib.tessa_last_error_message())

    # table, rows, stride, dim, type, ids, bits, out type, count, scale, out, stride
    good = [p, 64, 64, 64, 0, q, 32, 0, 16, 1.0, p + 65536, 64]
    assert lib.tessa_embedding_lookup(h, C.LookupArgs(*good), None) == 0
    for at, v in ((0, None), (0, p + 2), (2, 63), (4, 3), (5, None), (5, q + 2), (6, 16), (7, 9), (10, None), (11, 8)):
        refused(lib.tessa_embedding_lookup, C.LookupArgs(*good[:at], v, *good[at + 1:]), None)
    for at, v in ((1, 1 << 32), (2, 1 << 41), (8, 1 << 31)):
        refused(lib.tessa_embedding_lookup, C.LookupArgs(*good[:at], v, *good[at + 1:]), None, code=UNSUPPORTED)

    # dout, stride, dim, type, ids, bits, grad type, count, scale, accumulate, grad, stride, rows
    good = [p, 8, 8, 0, q, 32, 0, 4096 + 904, 1.0, 0, p + 196608, 8, 64]
    i5 = torch.zeros(5000, dtype=torch.int32, device="cuda")
    good[4] = i5.data_ptr()
    need = ctypes.c_uint64()
    C.check(lib.tessa_embedding_grad_workspace(5000, 64, 8, need))
    assert lib.tessa_embedding_grad(h, C.LookupGradArgs(*good), w, need.value, None) == 0
    for at, v in ((0, None), (1, 7), (3, 3), (5, 8), (9, 2), (10, None), (11, 7)):
        refused(lib.tessa_embedding_grad, C.LookupGradArgs(*good[:at], v, *good[at + 1:]), w, need.value, None)
    for space, size in ((None, need.value), (w, need.value - 1), (w + 16, need.value)):
        refused(lib.tessa_embedding_grad, C.LookupGradArgs(*good), space, size, None)

    # x, rows, cols, stride, type, reserved, codes, scales, codes of columns, scales
    good = [p, 32, 64, 64, 0, 0, w, w + 4096, w + 8192, w + 16384]
    assert lib.tessa_quantize_fp8(h, C.Fp8QuantizeArgs(*good), None) == 0
    for at, v in ((0, None), (3, 63), (4, 3), (6, None), (7, None), (6, w + 8), (8, w + 8200), (9, None)):
        refused(lib.tessa_quantize_fp8, C.Fp8QuantizeArgs(*good[:at], v, *good[at + 1:]), None)
    refused(lib.tessa_quantize_fp8, C.Fp8QuantizeArgs(*good[:6], None, None, None, None), None)

    # codes, scales, codes, scales, m, n, k, out, stride, type, reserved
    good = [w, w + 4096, w, w + 4096, 32, 32, 64, p, 32, 0, 0]
    C.check(lib.tessa_matmul_fp8_workspace(h, 32, 32, 64, need))
    assert need.value == 0 and lib.tessa_matmul_fp8(h, C.Fp8MatmulArgs(*good), None, 0, None) == 0
    for at, v in ((0, None), (1, None), (0, w + 8), (1, w + 4097), (6, 72), (7, None), (8, 31), (9, 3)):
        refused(lib.tessa_matmul_fp8, C.Fp8MatmulArgs(*good[:at], v, *good[at + 1:]), None, 0, None)

    # logits, rows, vocab, stride, type, k, ids, teacher, bits, temperature, weights, loss, lse, grad, stride
    good = [p, 16, 64, 64, 0, 4, q, p + 65536, 32, 1.0, None, p + 131072, None, p + 196608, 64]
    assert lib.tessa_distill_topk(h, C.DistillArgs(*good), None, 0, None) == 0
    for at, v in ((0, None), (3, 63), (4, 3), (5, 1025), (6, None), (7, None), (8, 64 + 1), (9, 0.0), (9, -1.0),
                  (9, float("nan")), (9, float("inf")), (14, 63)):
        got = lib.tessa_distill_topk(h, C.DistillArgs(*good[:at], v, *good[at + 1:]), None, 0, None)
        assert got in (INVALID, UNSUPPORTED), (at, v, got)
    ops.async_status()


def test_workspace_of_rows_too_long_to_count():
    # columns are counted in 32 bits: rows whose last step would wrap around are refused
    lib = C.load()
    n = ctypes.c_uint64()
    assert lib.tessa_embedding_grad_workspace(10_000, 2, 0xfffffc00, n) == 0
    assert n.value >= 10_000 // 32 * 2 * 0xfffffc00 * 4
    for dim in (0xfffffc01, 0xfffffffd, 0xffffffff):
        assert lib.tessa_embedding_grad_workspace(10_000, 2, dim, n) == UNSUPPORTED


@pytest.mark.gpu
def test_rows_too_long_to_count():
    # refused before any launch, so that no memory of that size has to be there
    import torch
    from shear_b200 import ops
    lib, h = C.load(), ops.context(0).handle
    t = torch.zeros(4096, device="cuda")
    p = t.data_ptr()
    for dim in (0xfffffc01, 0xffffffff):
        assert lib.tessa_embedding_lookup(h, C.LookupArgs(p, 1, dim, dim, 0, p, 32, 0, 1, 1.0, p, dim), None) == UNSUPPORTED
        assert lib.tessa_embedding_grad(h, C.LookupGradArgs(p, dim, dim, 0, p, 32, 0, 1, 1.0, 0, p, dim, 1), None, 0,
                                        None) == UNSUPPORTED
