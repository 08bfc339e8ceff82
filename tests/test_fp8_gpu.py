"""FP8 block codes against their definition, and the product against 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _e4m3_table():
    """The value of every E4M3 byte: bias 7, three fraction bits, 0x7f / 0xff NaN, no infinities."""
    v = np.zeros(256)
    for b in range(256):
        e, f = (b >> 3) & 15, b & 7
        v[b] = (f / 8 * 2.0 ** -6 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7)) * (-1 if b & 128 else 1)
        if b & 127 == 127:
            v[b] = np.nan
    return v


TABLE = _e4m3_table()


def _encode(x):
    """Codes and scale bytes of x's rows (64-bit arithmetic on exact inputs)."""
    rows, cols = x.shape
    pad, nb = -(-cols // 16) * 16, -(-cols // 128)
    codes = np.zeros((rows, pad), np.uint8)
    scales = np.zeros((rows, -(-nb // 4) * 4), np.uint8)
    grid = np.sort(TABLE[:127])          # 0 .. 448
    for b in range(nb):
        blk = x[:, b * 128: (b + 1) * 128].astype(np.float64)
        ok = np.isfinite(blk)
        amax = np.abs(np.where(ok, blk, 0.0)).max(axis=1)
        _, e = np.frexp(amax / 448.0)    # amax / 448 = f 2^e, 0.5 <= f < 1
        e = np.where(np.ldexp(1.0, e - 1) * 448.0 >= amax, e - 1, e)
        byte = np.where(amax > 0, np.clip(e + 127, 0, 254), 0)
        scales[:, b] = byte
        y = np.where(ok, blk, 0.0) * np.ldexp(1.0, 127 - byte)[:, None]
        a = np.abs(y)
        hi = np.searchsorted(grid, a)    # grid[hi - 1] < a <= grid[hi]
        lo = np.maximum(hi - 1, 0)
        mid = (grid[lo] + grid[hi]) / 2
        c = np.where((a > mid) | ((a == mid) & (hi % 2 == 0)), hi, lo)
        c = np.where(a == grid[hi], hi, c)
        c = np.where(ok, c | (np.signbit(blk) * 128), 0x7f)
        codes[:, b * 128: b * 128 + blk.shape[1]] = c
    return codes, scales


def _decode(codes, scales):
    s = np.ldexp(1.0, scales.astype(np.int64) - 127).repeat(128, axis=1)[:, : codes.shape[1]]
    return TABLE[codes] * s


def _bytes(t):
    import torch
    return t.view(torch.uint8).cpu().numpy()


def _values(rng, rows, cols, dtype):
    import torch
    x = rng.standard_normal((rows, cols)) * np.exp(rng.uniform(-4, 4, (rows, 1)))
    return torch.from_numpy(x.astype(np.float32)).to(getattr(torch, dtype))


@pytest.mark.parametrize("rows,cols,dtype,pad", [
    (1, 1, "float32", 0), (1, 128, "float32", 0), (3, 129, "bfloat16", 0), (130, 100, "float16", 0),
    (257, 768, "bfloat16", 0), (64, 1000, "float16", 24), (50, 515, "float32", 1), (513, 36, "bfloat16", 4),
    (1000, 130, "float32", 0), (2, 5003, "bfloat16", 0),
])
def test_codes(rows, cols, dtype, pad):
    import torch
    from shear_b200 import ops
    rng = np.random.default_rng(rows * 7 + cols)
    x = _values(rng, rows, cols, dtype)
    x[0] = 0.0
    x[rows // 2, cols // 2] = 448.0 * 2.0 ** -3
    wide = torch.full((rows, cols + pad), 1e4, dtype=x.dtype, device="cuda")
    wide[:, :cols] = x.cuda()
    dev = wide[:, :cols]
    host = x.double().numpy()
    want, want_t = _encode(host), _encode(np.ascontiguousarray(host.T))
    for got in (ops.quantize_fp8(dev), ops.quantize_fp8_both(dev)[:2]):
        assert got[0].dtype == torch.float8_e4m3fn and got[1].dtype == torch.uint8
        assert np.array_equal(_bytes(got[0]) & 0x7f, want[0] & 0x7f) and np.array_equal(_bytes(got[1]), want[1])
        assert np.array_equal(TABLE[_bytes(got[0])], TABLE[want[0]])
    for got in (ops.quantize_fp8(dev, transpose=True), ops.quantize_fp8_both(dev)[2:]):
        assert np.array_equal(TABLE[_bytes(got[0])], TABLE[want_t[0]]) and np.array_equal(_bytes(got[1]), want_t[1])


def test_codes_at_the_edges():
    # every E4M3 value and every midpoint between two, the border of each
    # binade of the maximum, subnormal and huge blocks, NaN and infinities
    import torch
    from shear_b200 import ops
    grid = TABLE[:127]
    mids = (grid[1:] + grid[:-1]) / 2
    rows = []
    for f in (1.0, 2.0 ** -100, 2.0 ** 100, 2.0 ** -133):
        r = np.zeros(256)
        r[:127], r[128:254] = grid * f, mids * f
        r[127] = r[255] = 448.0 * f
        rows.append(r)
    for amax in (448.0, np.nextafter(np.float32(448.0), np.float32(500)), 1.0, 1.75, 1.7500001, 3.4028235e38, 1e-45, 1e-40):
        r = np.zeros(256)
        r[:] = np.float32(amax) * np.linspace(-1, 1, 256).astype(np.float32)
        rows.append(r)
    special = np.linspace(-3, 3, 256)
    special[[3, 200]] = np.nan
    special[[4, 130]] = np.inf, -np.inf
    rows.append(special)
    rows.append(np.full(256, np.nan))
    x = np.array(rows, np.float32)
    codes, scales = ops.quantize_fp8(torch.from_numpy(x).cuda())
    want = _encode(x.astype(np.float64))
    assert np.array_equal(_bytes(scales), want[1])
    got, exp = TABLE[_bytes(codes)], TABLE[want[0]]
    assert np.array_equal(np.isnan(got), np.isnan(exp)) and np.array_equal(np.nan_to_num(got), np.nan_to_num(exp))
    codes_t, scales_t = ops.quantize_fp8(torch.from_numpy(np.ascontiguousarray(x.T)).cuda(), transpose=True)
    assert np.array_equal(_bytes(codes_t) & 0x7f, _bytes(codes) & 0x7f) and np.array_equal(_bytes(scales_t), _bytes(scales))


def _product_case(m, n, k, out, seed=0, ld=0):
    import torch
    from shear_b200 import ops
    rng = np.random.default_rng(m * 31 + n * 7 + k + seed)
    pad = -(-k // 16) * 16
    # codes of every magnitude, scales over 40 binades, different in every block and row
    def operand(rows):
        c = rng.integers(0, 256, (rows, pad)).astype(np.uint8)
        c[(c & 127) == 127] = 0
        c[:, k:] = 0
        s = np.zeros((rows, -(-pad // 512) * 4), np.uint8)
        nb = -(-pad // 128)
        s[:, :nb] = rng.integers(107, 148, (rows, nb))
        return c, s
    (ac, as_), (bc, bs) = operand(m), operand(n)
    a, b = _decode(ac, as_), _decode(bc, bs)
    want, mag = a @ b.T, np.abs(a) @ np.abs(b).T
    dev = [torch.from_numpy(t).cuda() for t in (ac, as_, bc, bs)]
    dst = None
    if ld:
        wide = torch.full((m, n + ld), 5.0, dtype=getattr(torch, out), device="cuda")
        dst = wide[:, :n]
    got = ops.matmul_fp8(*dev, out_dtype=getattr(torch, out), out=dst)
    ops.async_status()
    # Each step of 32 products adds 33 terms, each held to at least 24 bits of
    # the largest; then one rounding to the output type.
    info = torch.finfo(getattr(torch, out))
    bound = -(-pad // 32) * 33 * 2.0 ** -24 * mag + info.eps / 2 * np.abs(want)
    g = got.double().cpu().numpy()
    near = np.abs(np.abs(want) - info.max) <= bound  # may round to infinity or to the largest value
    over = (np.abs(want) > info.max) & ~near         # past what the output type holds
    assert (g[over] == np.sign(want[over]) * np.inf).all()
    err = np.abs(np.where(over | near, want, g) - want)
    assert (err <= bound).all(), float((err / bound).max())
    if ld:
        assert (wide[:, n:] == 5.0).all()
    again = ops.matmul_fp8(*dev, out_dtype=getattr(torch, out))
    assert torch.equal(again, got)


@pytest.mark.parametrize("m,n,k,out", [
    (1, 1, 16, "float32"), (1, 128, 128, "float32"), (1, 1000, 768, "float32"), (16, 127, 130, "bfloat16"),
    (17, 129, 512, "float32"), (100, 200, 1000, "float32"), (128, 128, 2048, "float32"), (129, 300, 513, "bfloat16"),
    (240, 256, 640, "float32"), (241, 257, 656, "float32"), (500, 1000, 96, "bfloat16"),
    (1000, 1500, 768, "float32"), (777, 2049, 1000, "bfloat16"), (33, 70_001, 128, "float32"),
])
def test_product(m, n, k, out):
    _product_case(m, n, k, out)


@pytest.mark.parametrize("m,n,k,out", [
    (1, 5, 16, "float32"), (2, 300, 768, "bfloat16"), (3, 1000, 640, "float16"), (4, 129, 4112, "float32"),
    (1, 20_001, 1040, "float32"), (1, 40, 16_400, "float32"), (300, 1, 400, "float32"), (1000, 3, 208, "bfloat16"),
    (129, 4, 2048, "float32"), (4, 4, 1024, "float32"), (30_000, 2, 1296, "float16"),
])
def test_product_with_few_rows(m, n, k, out):
    # one query against a table, and a table against one query
    _product_case(m, n, k, out)
    _product_case(m, n, k, out, seed=1, ld=5)


@pytest.mark.parametrize("m,n", [(1, 40), (40, 2)])
def test_few_rows_at_the_ends_of_the_scales(m, n):
    # sixteen products of 1 * 1 under scales whose product is any power of two,
    # past what f32 holds too; the byte 255 stands for NaN
    import torch
    from shear_b200 import ops
    one = torch.full((max(m, n), 16), 0x38, dtype=torch.uint8, device="cuda")
    for sa, sb in ((0, 0), (0, 254), (254, 0), (254, 254), (127, 127), (127, 1), (1, 1), (60, 61), (3, 104), (200, 178),
                   (200, 183), (255, 0), (0, 255), (255, 255)):
        a = torch.full((m, 4), sa, dtype=torch.uint8, device="cuda")
        b = torch.full((n, 4), sb, dtype=torch.uint8, device="cuda")
        got = ops.matmul_fp8(one[:m], a, one[:n], b).cpu().numpy()
        with np.errstate(over="ignore", under="ignore"):
            want = np.nan if 255 in (sa, sb) else np.float32(np.ldexp(16.0, sa + sb - 254))
        assert np.array_equal(got, np.full((m, n), want, np.float32), equal_nan=True), (sa, sb, got.flat[0], want)


@pytest.mark.parametrize("m,n,k", [(5, 100, 20_000), (64, 64, 40_000), (200, 768, 9000), (300, 130, 16_385)])
def test_product_with_a_long_sum(m, n, k):
    # few tiles and a long K: parts of K by several units, added in order
    _product_case(m, n, k, "float32")
    _product_case(m, n, k, "bfloat16", seed=1, ld=9)


def test_product_strided_out_and_nothing():
    import torch
    from shear_b200 import ops
    _product_case(70, 90, 256, "float32", ld=3)
    _product_case(70, 90, 256, "bfloat16", ld=7)
    z = torch.zeros(3, 0, dtype=torch.float8_e4m3fn, device="cuda")
    s = torch.zeros(3, 0, dtype=torch.uint8, device="cuda")
    assert (ops.matmul_fp8(z, s, z, s) == 0).all()
    c, t = ops.quantize_fp8(torch.randn(4, 32, device="cuda"))
    assert ops.matmul_fp8(c[:0], t[:0], c, t).shape == (0, 4)
    assert ops.matmul_fp8(c, t, c[:0], t[:0]).shape == (4, 0)


def test_nan_codes_reach_their_row_alone():
    import torch
    from shear_b200 import ops
    x = torch.randn(5, 300, device="cuda")
    w = torch.randn(7, 300, device="cuda")
    x[2, 150] = float("inf")
    y = ops.matmul_fp8(*ops.quantize_fp8(x), *ops.quantize_fp8(w))
    assert y[2].isnan().all() and y[[0, 1, 3, 4]].isfinite().all()


def test_gradients_of_a_product():
    # dx = dy w and dw = dy^T x by the same product, on codes along the other
    # axis: against 64-bit products of the codes, and against differences of
    # sum(dy * (x w^T)), which is linear in each, so that the difference over
    # operands that E4M3 holds exactly is exact.
    import torch
    from shear_b200 import ops
    rng = np.random.default_rng(2)
    x = torch.from_numpy(rng.integers(-8, 9, (33, 50)).astype(np.float32)).cuda()
    w = torch.from_numpy(rng.integers(-8, 9, (140, 50)).astype(np.float32)).cuda()
    dy = torch.from_numpy(rng.integers(-8, 9, (33, 140)).astype(np.float32)).cuda()
    xq, wq, dq = ops.quantize_fp8_both(x), ops.quantize_fp8_both(w), ops.quantize_fp8_both(dy)
    y = ops.matmul_fp8(*xq[:2], *wq[:2])
    dx = ops.matmul_fp8(*dq[:2], *wq[2:])
    dw = ops.matmul_fp8(*dq[2:], *xq[2:])
    assert torch.equal(y.double(), x.double() @ w.double().t())
    assert torch.equal(dx.double(), dy.double() @ w.double())
    assert torch.equal(dw.double(), dy.double().t() @ x.double())
    for i, j in ((0, 0), (32, 49), (7, 31)):
        bump = x.clone()
        bump[i, j] = 9.0 if x[i, j] < 8 else -9.0
        y2 = ops.matmul_fp8(*ops.quantize_fp8(bump), *wq[:2])
        slope = ((y2 - y).double() * dy).sum() / (bump[i, j] - x[i, j]).double()
        assert abs(slope.item() - dx[i, j].item()) < 1e-9


def test_another_stream():
    import torch
    from shear_b200 import ops
    x, w = torch.randn(100, 700, device="cuda"), torch.randn(300, 700, device="cuda")
    want = ops.matmul_fp8(*ops.quantize_fp8(x), *ops.quantize_fp8(w))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.matmul_fp8(*ops.quantize_fp8(x), *ops.quantize_fp8(w))
    s.synchronize()
    assert torch.equal(got, want)


def test_refusals():
    import torch
    from shear_b200 import ops
    from shear_b200._capi import TessaError
    x = torch.randn(8, 64, device="cuda")
    for bad in (x.double(), x.cpu(), x[0], x.t()):
        with pytest.raises(ValueError):
            ops.quantize_fp8(bad)
    c, s = ops.quantize_fp8(x)
    d, t = ops.quantize_fp8(torch.randn(8, 80, device="cuda"))
    for bad in ((c.float(), s, c, s), (c, s.float(), c, s), (c, s[:4], c, s), (c, s, d, t), (c[:, :48], s, c, s),
                (c.cpu(), s.cpu(), c, s)):
        with pytest.raises(ValueError):
            ops.matmul_fp8(*bad)
    for out in (torch.empty(8, 7, device="cuda"), torch.empty(8, 8, device="cuda").double()):
        with pytest.raises(ValueError):
            ops.matmul_fp8(c, s, c, s, out=out)
    raw = torch.zeros(8 * 64 + 8, dtype=torch.uint8, device="cuda")
    off = raw[8:].view(8, 64)  # rows that do not start on 16 bytes
    with pytest.raises(TessaError) as e:
        ops.matmul_fp8(off, s, c, s)
    assert e.value.code == -1
