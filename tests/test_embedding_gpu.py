"""Embedding lookup and its gradient against plain 64-bit sums."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

LEAST = {"float32": 2.0 ** -149, "bfloat16": 2.0 ** -133, "float16": 2.0 ** -24}  # spacing near zero


def _bound(name, value, magnitude, n):
    """One rounding to the output type (half of eps, the spacing above 1) of a
    sum held in f32, plus the f32 sum's own error, n * 2^-24 of the magnitudes."""
    import torch
    return torch.finfo(getattr(torch, name)).eps / 2 * np.abs(value) + LEAST[name] + (n + 2) * 2.0 ** -24 * magnitude


def _rows(torch, shape, dtype, seed, pad=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn(shape[0], shape[1] + pad, generator=g, device="cuda").to(dtype)
    return x[:, :shape[1]]


@pytest.mark.parametrize("rows,dim,count,dtype,out,ids,pad", [
    (1, 1, 1, "float32", "float32", "int32", 0),
    (1000, 128, 64, "float32", "float32", "int32", 0),
    (1000, 768, 4097, "bfloat16", "bfloat16", "int64", 0),
    (77, 181, 300, "float16", "float16", "int32", 0),      # odd columns: element accesses
    (77, 100, 300, "float16", "float32", "int64", 0),      # rows that are 8-byte aligned
    (500, 96, 1001, "float32", "bfloat16", "int32", 5),    # strided rows, odd stride
    (500, 96, 1001, "bfloat16", "float32", "int32", 8),    # strided rows, vector stride
    (3, 2048, 70, "float16", "bfloat16", "int64", 0),
    (40, 33, 0, "float32", "float32", "int64", 0),         # no ids
])
def test_lookup(rows, dim, count, dtype, out, ids, pad):
    import torch
    from shear_b200 import ops
    table = _rows(torch, (rows, dim), getattr(torch, dtype), 1, pad)
    rng = np.random.default_rng(rows + dim)
    idx = rng.integers(0, rows, count)
    idx[::7] = -1
    t = torch.from_numpy(idx).to(getattr(torch, ids)).cuda()
    got = ops.embedding_lookup(table, t, 1.7, out_dtype=getattr(torch, out))
    assert got.shape == (count, dim) and got.dtype == getattr(torch, out)
    want = np.float64(np.float32(1.7)) * table.double().cpu().numpy()[idx]
    want[idx < 0] = 0.0
    assert (np.abs(got.double().cpu().numpy() - want) <= _bound(out, want, np.abs(want), 0)).all()
    ops.async_status()


def test_lookup_shapes_streams_and_out():
    import torch
    from shear_b200 import ops
    table = torch.randn(50, 24, device="cuda")
    ids = torch.randint(0, 50, (3, 5, 2), device="cuda")
    assert torch.equal(ops.embedding_lookup(table, ids), table[ids])
    # every second id of a longer list, and an output inside a wider buffer
    wide = torch.full((30, 40), 7.0, device="cuda")
    every = torch.randint(0, 50, (60,), device="cuda")
    ops.embedding_lookup(table, every[::2], out=wide[:, 8:32])
    assert torch.equal(wide[:, 8:32], table[every[::2]])
    assert (wide[:, :8] == 7).all() and (wide[:, 32:] == 7).all()
    # a stream of the caller's own
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.embedding_lookup(table, ids)
    s.synchronize()
    assert torch.equal(got, table[ids])


def _grad_case(rows, dim, idx, dtype, out, ids, scale, pad=0, accumulate=False):
    import torch
    from shear_b200 import ops
    n = len(idx)
    dout = _rows(torch, (n, dim), getattr(torch, dtype), 2, pad)
    t = torch.from_numpy(np.asarray(idx)).to(getattr(torch, ids)).cuda()
    base = _rows(torch, (rows, dim), getattr(torch, out), 3) if accumulate else None
    dst = base.clone() if accumulate else None
    got = ops.embedding_grad(dout, t, rows, scale, out_dtype=getattr(torch, out), out=dst, accumulate=accumulate)
    ops.async_status()
    d = dout.double().cpu().numpy() * np.float64(np.float32(scale))
    want, mag = np.zeros((rows, dim)), np.zeros((rows, dim))
    named = np.asarray(idx) >= 0
    np.add.at(want, np.asarray(idx)[named], d[named])
    np.add.at(mag, np.asarray(idx)[named], np.abs(d[named]))
    n_of = np.bincount(np.asarray(idx)[named], minlength=rows)[:, None] if n else np.zeros((rows, 1))
    if accumulate:
        b = base.double().cpu().numpy()
        want, mag = want + b, mag + np.abs(b)
    have = got.double().cpu().numpy()
    err = np.abs(have - want)
    assert (err <= _bound(out, want, mag, n_of + 3)).all(), float((err - _bound(out, want, mag, n_of + 3)).max())
    if accumulate:  # rows that no id names keep their bits
        idle = n_of[:, 0] == 0
        assert torch.equal(got[torch.from_numpy(idle).cuda()], base[torch.from_numpy(idle).cuda()])
    again = ops.embedding_grad(dout, t, rows, scale, out_dtype=getattr(torch, out),
                               out=base.clone() if accumulate else None, accumulate=accumulate)
    assert torch.equal(got, again)  # the order of the sums does not change
    return got


def _zipf(rng, n, rows):
    return np.minimum((10.0 * ((rows / 10.0 + 1.0) ** rng.random(n) - 1.0)).astype(np.int64), rows - 1)


@pytest.mark.parametrize("rows,dim,count,dtype,out,ids", [
    (1, 1, 1, "float32", "float32", "int32"),
    (5, 7, 31, "float32", "float32", "int64"),
    (5, 8, 32, "bfloat16", "float32", "int64"),
    (5, 9, 33, "float16", "float16", "int32"),
    (1000, 128, 2048, "float32", "float32", "int32"),
    (1000, 128, 2049, "float32", "float32", "int32"),
    (1023, 64, 5000, "bfloat16", "bfloat16", "int32"),     # one digit
    (1024, 64, 5000, "float32", "float32", "int64"),       # two digits
    (200_000, 128, 20_001, "float32", "float32", "int32"),
    (3_000_000, 32, 20_000, "bfloat16", "float32", "int64"),  # three digits
    (700, 768, 9000, "bfloat16", "bfloat16", "int64"),
    (700, 1030, 4100, "float16", "float32", "int32"),
    (300, 181, 4100, "bfloat16", "float16", "int32"),
])
@pytest.mark.parametrize("zipf", [False, True])
def test_grad(rows, dim, count, dtype, out, ids, zipf):
    rng = np.random.default_rng(count + dim)
    idx = _zipf(rng, count, rows) if zipf else rng.integers(0, rows, count)
    idx[::11] = -1
    _grad_case(rows, dim, idx, dtype, out, ids, 1.25)


@pytest.mark.parametrize("rows", [3, 900, 5000, 3_000_000])  # one to three digits
@pytest.mark.parametrize("count", [255, 256, 257, 1024, 1025, 16_384, 16_385, 131_073])
def test_grad_at_the_borders_of_the_sorts(rows, count):
    # one block, one cluster of one to sixteen blocks, several kernels
    rng = np.random.default_rng(rows + count)
    idx = _zipf(rng, count, rows)
    idx[5::97] = -1
    _grad_case(rows, 4, idx, "float32", "float32", "int32", 1.0)
    _grad_case(rows, 8, idx, "float32", "bfloat16", "int64", 1.0, accumulate=True)


@pytest.mark.parametrize("rows,count", [(1, 5000), (2, 64), (2, 96), (3, 40_000)])
def test_grad_runs_over_many_tiles(rows, count):
    # one id throughout; a border exactly on a tile's; a run of hundreds of tiles beside short ones
    _grad_case(rows, 36, np.zeros(count, np.int64), "float32", "float32", "int32", 1.0)
    idx = np.zeros(count, np.int64)
    idx[count // 2:] = rows - 1
    _grad_case(rows, 36, idx, "float32", "float32", "int32", 0.5)
    idx[: count // 3] = -1
    _grad_case(rows, 36, idx, "bfloat16", "float32", "int64", 0.5)


@pytest.mark.parametrize("out", ["float32", "bfloat16"])
def test_grad_accumulates(out):
    rng = np.random.default_rng(5)
    _grad_case(400, 72, _zipf(rng, 6000, 400), "float32", out, "int32", 0.3, accumulate=True)
    _grad_case(4000, 72, rng.integers(0, 4000, 900), "float32", out, "int32", 0.3, accumulate=True)


def test_grad_strides_empty_and_shape():
    import torch
    from shear_b200 import ops
    rng = np.random.default_rng(6)
    _grad_case(90, 50, rng.integers(0, 90, 3000), "float32", "float32", "int32", 2.0, pad=3)
    _grad_case(90, 64, rng.integers(0, 90, 3000), "bfloat16", "float32", "int32", 2.0, pad=8)
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    got = ops.embedding_grad(torch.zeros(0, 8, device="cuda"), none, 5)
    assert got.shape == (5, 8) and (got == 0).all()
    # gradients of a batch of lists, into a wider buffer whose margins stay
    ids = torch.randint(0, 20, (6, 7), device="cuda")
    d = torch.randn(6, 7, 12, device="cuda")
    wide = torch.full((20, 16), 3.0, device="cuda")
    ops.embedding_grad(d, ids, 20, out=wide[:, 2:14])
    want = torch.zeros(20, 12, dtype=torch.float64, device="cuda").index_add_(0, ids.reshape(-1), d.reshape(-1, 12).double())
    assert torch.allclose(wide[:, 2:14].double(), want, rtol=0, atol=1e-5)
    assert (wide[:, :2] == 3).all() and (wide[:, 14:] == 3).all()


def test_grad_against_differences():
    # d/dtable of sum(w * lookup(table)) is linear: a difference of the whole
    # step in f32 tables of small whole numbers is exact.
    import torch
    from shear_b200 import ops
    rng = np.random.default_rng(8)
    table = torch.from_numpy(rng.integers(-4, 5, (6, 5)).astype(np.float32)).cuda()
    ids = torch.from_numpy(rng.integers(-1, 6, 40)).cuda()
    w = torch.from_numpy(rng.integers(-4, 5, (40, 5)).astype(np.float32)).cuda()
    grad = ops.embedding_grad(w, ids, 6, 2.0)
    f0 = (ops.embedding_lookup(table, ids, 2.0) * w).double().sum()
    for v in range(6):
        for c in range(5):
            t = table.clone()
            t[v, c] += 1.0
            assert ((ops.embedding_lookup(t, ids, 2.0) * w).double().sum() - f0).item() == grad[v, c].item()


def test_bad_ids_are_reported_and_read_nothing():
    import torch
    from shear_b200 import ops
    from shear_b200._capi import TessaError
    table = torch.randn(10, 16, device="cuda")
    for bad in (10, -2, 2 ** 31 - 1):
        ids = torch.tensor([1, bad, 3], device="cuda")
        got = ops.embedding_lookup(table, ids)
        with pytest.raises(TessaError) as e:
            ops.async_status()
        assert e.value.code == -5
        assert torch.equal(got[0], table[1]) and (got[1] == 0).all() and torch.equal(got[2], table[3])
        ops.async_status()  # reported once
        g = ops.embedding_grad(torch.ones(3, 16, device="cuda"), ids, 10)
        torch.cuda.synchronize()
        with pytest.raises(TessaError):  # the next call reports it too
            ops.embedding_lookup(table, ids[:1])
        assert g.sum().item() == 32.0
    ops.async_status()


def test_refusals():
    import torch
    from shear_b200 import ops
    table = torch.randn(10, 16, device="cuda")
    ids = torch.zeros(3, dtype=torch.int64, device="cuda")
    for bad in (dict(table=table.double()), dict(table=table.cpu()), dict(table=table[0]), dict(ids=ids.to(torch.int16)),
                dict(ids=ids.cpu()), dict(table=table.t()), dict(out=torch.empty(2, 16, device="cuda")),
                dict(out=torch.empty(3, 16, device="cuda"), out_dtype=torch.float16)):
        a = {"table": table, "ids": ids, **bad}
        with pytest.raises(ValueError):
            ops.embedding_lookup(**a)
    dout = torch.randn(3, 16, device="cuda")
    for bad in (dict(dout=dout[:2]), dict(dout=dout.double()), dict(ids=ids.to(torch.uint8)), dict(accumulate=True),
                dict(out=torch.empty(9, 16, device="cuda"))):
        a = {"dout": dout, "ids": ids, "table_rows": 10, **bad}
        with pytest.raises(ValueError):
            ops.embedding_grad(**a)
