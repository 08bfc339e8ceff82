"""Offsets past 2^32 elements: the last rows of matrices of more than four
billion against the same rows alone (10 to 20 GB on the device)."""
import pytest

pytestmark = pytest.mark.gpu

ROWS, DIM = 4_400_000, 1024  # 4.5e9 elements


def _room(torch, gib):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip(f"needs {gib} GiB of device memory")


def test_lookup_and_its_gradient():
    import torch
    from shear_b200 import ops
    _room(torch, 24)
    table = torch.empty(ROWS, DIM, dtype=torch.bfloat16, device="cuda")
    table[-4:] = torch.randn(4, DIM, device="cuda").bfloat16()
    ids = torch.tensor([ROWS - 1, ROWS - 3, ROWS - 4, ROWS - 1], device="cuda")
    assert torch.equal(ops.embedding_lookup(table, ids), table[ids])
    d = torch.randn(4, DIM, device="cuda").bfloat16()
    want = torch.zeros(4, DIM, device="cuda")
    want.index_add_(0, ids - (ROWS - 4), d.float())  # two terms at most: one rounding
    ops.embedding_grad(d, ids, ROWS, out=table)
    assert torch.equal(table[-4:], want.bfloat16()) and (table[:4] == 0).all()
    # as many rows of gradients, of which the last count
    table.zero_()
    table[-2:] = d[:2]
    many = torch.randint(0, 50, (ROWS,), device="cuda")
    got = ops.embedding_grad(table, many, 60, out_dtype=torch.float32)
    want = torch.zeros(60, DIM, device="cuda").index_add_(0, many[-2:], d[:2].float())
    assert torch.equal(got, want)


def test_codes():
    import torch
    from shear_b200 import ops
    _room(torch, 24)
    x = torch.zeros(ROWS, DIM, dtype=torch.bfloat16, device="cuda")
    x[-300:] = torch.randn(300, DIM, device="cuda").bfloat16()
    c, s = ops.quantize_fp8(x)
    tail = ops.quantize_fp8(x[-300:])
    assert torch.equal(c[-300:].view(torch.uint8), tail[0].view(torch.uint8)) and torch.equal(s[-300:], tail[1])
    assert (s[:1000] == 0).all()
    del c, s
    first = (ROWS - 300) // 128 * 128  # columns: whole blocks of 128 rows
    c, s = ops.quantize_fp8(x, transpose=True)
    tail = ops.quantize_fp8(x[first:], transpose=True)
    assert torch.equal(c[:, first:].view(torch.uint8), tail[0].view(torch.uint8))
    n = -(-(ROWS - first) // 128)
    assert torch.equal(s[:, first // 128:first // 128 + n], tail[1][:, :n])


@pytest.mark.parametrize("m,n", [(4400, 1_000_003), (1_000_003, 4400), (3, 1_000_003)])
def test_product(m, n):
    # whole numbers up to 8 over 64 of K: codes, products and sums are exact, and below 2^13
    import torch
    from shear_b200 import ops
    _room(torch, 24)
    a = torch.randint(-8, 9, (m, 64), device="cuda").bfloat16()
    b = torch.randint(-8, 9, (n, 64), device="cuda").bfloat16()
    y = ops.matmul_fp8(*ops.quantize_fp8(a), *ops.quantize_fp8(b), out_dtype=torch.float32 if m == 3 else torch.bfloat16)
    for i, j in ((slice(m - 2, m), slice(n - 999, n)), (slice(0, 2), slice(0, 999)), (slice(m // 2, m // 2 + 2), slice(n - 50, n))):
        assert torch.equal(y[i, j], (a[i].double() @ b[j].double().t()).to(y.dtype))
    assert torch.equal(y[m - 1, ::9973], (a[m - 1].double() @ b[::9973].double().t()).to(y.dtype))


def test_distillation():
    import torch
    from shear_b200 import ops
    _room(torch, 24)
    rows, vocab, k = 4400, 1_000_003, 8
    z = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    z[-3:] = torch.randn(3, vocab, device="cuda").bfloat16()
    ids = torch.randint(0, vocab, (rows, k), device="cuda")
    tl = torch.randn(rows, k, device="cuda")
    alone = ops.distill_topk_grad(z[-3:].clone(), ids[-3:], tl[-3:], 2.0)
    got = ops.distill_topk_grad(z, ids, tl, 2.0, out=z)
    # the few rows are split otherwise: f32 sums of a million in another order, 64 u relative as bounded for one row
    for x, y in zip(got[:2], alone[:2]):
        assert torch.allclose(x[-3:], y, rtol=2.0 ** -17, atol=0)
    # one bf16 step where the two f32 values round apart
    g, w = got[2][-3:].float(), alone[2].float()
    assert ((g - w).abs() <= 2.0 ** -7 * w.abs()).all()
    # all logits equal: the gradient is 1 / vocab wherever the list is not
    row = got[2][1].float()
    row[ids[1]] = 2.0 / vocab
    assert torch.allclose(row, torch.full_like(row, 2.0 / vocab), rtol=2.0 ** -8, atol=0)
