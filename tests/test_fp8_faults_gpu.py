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


@pytest.mark.parametrize("n", [1, 9, 16])
def test_a_billion_rows(n):
    # few columns: read in registers, and by tiles either way round (rows of 18 bytes do not suit TMA)
    import torch
    from shear_b200 import ops
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 64 << 30:
        pytest.skip("needs 64 GiB of device memory")
    m, width = 1_090_000_000, 16
    a = torch.full((m, width), 0x38, dtype=torch.uint8, device="cuda")       # ones
    s = torch.full((m, 4), 127, dtype=torch.uint8, device="cuda")
    marks = [0, 1, 255, 256, m // 2, 2 ** 30 - 1, 2 ** 30, m - 257, m - 1]
    for i, r in enumerate(marks):
        a[r] = 0x40                                                          # twos
        s[r, 0] = 127 + i
    b = torch.full((n, width), 0x38, dtype=torch.uint8, device="cuda")
    t = torch.full((n, 4), 127, dtype=torch.uint8, device="cuda")
    t[:, 0] += torch.arange(n, device="cuda", dtype=torch.uint8) % 4         # column j times 2^(j % 4)
    out = ops.matmul_fp8(a, s, b, t, out_dtype=torch.bfloat16)
    ops.async_status()
    column = 2.0 ** (torch.arange(n, device="cuda") % 4)
    want = torch.tensor([32.0 * 2.0 ** i for i in range(len(marks))], device="cuda")[:, None] * column
    assert torch.equal(out[marks].float(), want)
    out[marks] = (16.0 * column).bfloat16()
    for first in range(0, m, 1 << 26):
        assert (out[first: first + (1 << 26)] == (16.0 * column).bfloat16()).all()


def test_products_of_too_many_tiles_are_refused():
    # before any launch: the operands are not there
    import torch
    from shear_b200 import _capi as C, ops
    lib, h = C.load(), ops.context(0).handle
    p = torch.zeros(256, device="cuda").data_ptr()
    most = 2 ** 31 - 1
    assert lib.tessa_matmul_fp8(h, C.Fp8MatmulArgs(p, p, p, p, most, most, 16, p, most, 1, 0), None, 0, None) == -6
    assert lib.tessa_matmul_fp8(h, C.Fp8MatmulArgs(p, p, p, p, 2 ** 31, 1, 16, p, 1, 1, 0), None, 0, None) == -6


@pytest.mark.parametrize("m,n", [(130, 300), (16, 40), (1, 300), (7, 5)])
@pytest.mark.parametrize("k", [4096, 8192, 40_000, 131_072])
def test_long_sums_of_one_sign(m, n, k):
    # An f32 accumulator that is cut towards zero loses up to 2^-23 of itself a
    # step of 32 terms, and with terms of one sign it grows evenly: half of that
    # a step, of the whole.  Parts of at most 8192 terms, 256 steps, keep that
    # from growing with k; within a step 33 terms are held to 24 bits of the
    # largest, and parts are added with rounding.  With few rows on one side
    # blocks of 128 are added with rounding, half of 2^-24 of the whole each.
    import torch
    from shear_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(k + m)
    codes = [torch.randint(0x30, 0x48, (r, k), generator=g, device="cuda").to(torch.uint8) for r in (m, n)]
    scales = [torch.full((r, -(-k // 512) * 4), 127, dtype=torch.uint8, device="cuda") for r in (m, n)]
    got = ops.matmul_fp8(codes[0], scales[0], codes[1], scales[1])
    ops.async_status()
    a, b = (c.view(torch.float8_e4m3fn).double() for c in codes)
    want = a @ b.t()
    few = min(m, n) <= 8
    steps = -(-k // 128) / 2 * 2.0 ** -24 + 5 * 2.0 ** -23 if few else 257 / 2 * 2.0 ** -23 + -(-k // 8192) * 2.0 ** -24
    assert ((got.double() - want).abs() <= (steps + 33 * 2.0 ** -24) * want).all(), float(((got - want) / want).abs().max())
