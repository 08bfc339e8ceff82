"""Distillation from a teacher's list against its formulas in 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _reference(z, ids, tl, tau, w):
    """loss, lse, grad in 64 bits, row by row, as the formulas stand."""
    rows, vocab = z.shape
    loss, lse, grad = np.zeros(rows), np.full(rows, -np.inf), np.zeros((rows, vocab))
    for r in range(rows):
        x = z[r] / tau
        top = x.max() if vocab else -np.inf
        entries = [(i, t / tau) for i, t in zip(ids[r], tl[r]) if i >= 0 and t > -np.inf]
        if top == -np.inf:
            continue
        log_s = np.log(np.exp(x - top).sum())
        lse[r] = top + log_s
        if not entries:
            continue
        t = np.array([e[1] for e in entries])
        p = np.exp(t - t.max())
        log_p = t - t.max() - np.log(p.sum())
        p /= p.sum()
        grad[r] = np.exp(x - top - log_s)  # (top + log_s loses log_s where top is the type's lowest value)
        for (i, _), pj, lp in zip(entries, p, log_p):
            grad[r, i] -= pj
            if pj > 0:
                loss[r] += tau * tau * pj * (lp - (x[i] - top - log_s))
        grad[r] *= tau * w[r]
    return loss, lse, grad


def _check(z, ids, tl, tau, w, dtype, got):
    """Bounds.  An exponent e = (z - m) / tau * log2(e) is held in f32: three
    roundings, |e| * 3u * ln 2 in the exponential's relative error, beside
    2^-22 of the exponential itself; sums of n in f32, here by threads in short
    chains: another 64u.  q and P inherit that; the gradient is rounded once to
    its type.  The loss adds k terms of which each has the error of lse and of
    the list's own logarithm."""
    import torch
    loss, lse, grad = _reference(z, ids, tl, tau, w)
    fine = np.where(np.abs(z) < 1e4, z, 0.0)  # masked logits' exponentials are 0 whatever their exponent's error
    reach = np.abs(fine).max() / tau + np.abs(np.where(np.isfinite(tl), tl, 0.0)).max(initial=0.0) / tau
    rel = 2.0 ** -21 + (64 + 8 * reach) * U
    g_loss, g_lse, g_grad = [None if t is None else t.double().cpu().numpy() for t in got]
    ok = np.isfinite(lse)
    assert (np.isfinite(g_lse) == ok).all()
    assert (np.abs(g_lse - lse)[ok] <= rel * (1 + np.abs(lse[ok]))).all()
    inf = np.abs(loss) > np.finfo(np.float32).max  # listed logits of the type's lowest value: past what f32 holds
    assert (np.isinf(g_loss) == inf).all()
    assert (np.abs(g_loss - loss)[~inf] <= tau * tau * 2 * rel * (1 + reach + np.abs(loss[~inf]))).all()
    if g_grad is not None:
        eps = torch.finfo(getattr(torch, dtype)).eps / 2
        least = {"float32": 2.0 ** -126, "bfloat16": 2.0 ** -126, "float16": 2.0 ** -24}[dtype]
        scale = tau * np.abs(w)[:, None]
        # q - P cancels where the student has learnt the list: both terms' errors stay
        p_part = np.maximum(np.abs(grad), np.exp(np.minimum(z / tau - np.where(ok, lse, 0.0)[:, None], 0.0)) * scale)
        bound = eps * np.abs(grad) + least + 2 * rel * (np.abs(grad) + p_part)
        assert np.isfinite(g_grad).all()
        assert (np.abs(g_grad - grad) <= bound).all(), float((np.abs(g_grad - grad) / bound).max())
        quiet = ~(np.asarray(loss) != 0) & ~ok
        assert (g_grad[quiet] == 0).all()


def _make(rng, rows, vocab, k, dtype):
    import torch
    z = torch.from_numpy(rng.standard_normal((rows, vocab)).astype(np.float32) * 2).to(getattr(torch, dtype))
    ids = np.stack([rng.permutation(vocab)[:k] if vocab >= k else rng.integers(0, vocab, k) for _ in range(rows)]).reshape(rows, k)
    tl = (rng.standard_normal((rows, k)) * 3).astype(np.float32)
    return z, ids.astype(np.int64), tl


def _run(z, ids, tl, tau, w, id_dtype="int64", pad=0, in_place=False):
    import torch
    from shear_b200 import ops
    dev = z.cuda()
    if pad:
        wide = torch.full((z.shape[0], z.shape[1] + pad), 50.0, dtype=z.dtype, device="cuda")
        wide[:, : z.shape[1]] = dev
        dev = wide[:, : z.shape[1]]
    i = torch.from_numpy(ids).to(getattr(torch, id_dtype)).cuda()
    t = torch.from_numpy(tl).cuda()
    weights = None if w is None else torch.from_numpy(w.astype(np.float32)).cuda()
    alone = ops.distill_topk(dev, i, t, tau)
    loss, lse, grad = ops.distill_topk_grad(dev, i, t, tau, weights, out=dev if in_place else None)
    ops.async_status()
    if not in_place:
        again = ops.distill_topk_grad(dev, i, t, tau, weights)
        for x, y in zip((loss, lse, grad), again):
            assert torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0))  # equal inputs, equal bits
    # the loss alone may split its row otherwise: near, not equal
    assert torch.allclose(alone[1], lse, rtol=1e-5, atol=1e-5)
    return loss, lse, grad


@pytest.mark.parametrize("rows,vocab,k,tau,dtype,ids,pad", [
    (1, 1, 1, 1.0, "float32", "int32", 0),
    (2, 3, 2, 1.0, "bfloat16", "int64", 0),
    (5, 7, 9, 2.0, "float16", "int64", 0),          # fewer candidates than entries: ids repeat
    (3, 1000, 32, 1.0, "float32", "int32", 0),
    (4, 1001, 33, 0.5, "float16", "int32", 0),      # rows that start off a 16-byte border
    (7, 16384, 32, 2.0, "bfloat16", "int64", 0),
    (7, 16385, 32, 2.0, "bfloat16", "int64", 3),    # strided, odd
    (300, 4099, 64, 1.0, "bfloat16", "int32", 5),
    (320, 50_003, 100, 2.0, "float16", "int64", 0),
    (2, 200_000, 32, 1.0, "float32", "int32", 0),
    (1, 1_000_003, 64, 1.0, "bfloat16", "int32", 0),
    (1, 1_000_003, 64, 1.0, "float32", "int32", 0),  # a row that no cluster keeps
    (2, 5000, 1024, 1.0, "float32", "int64", 0),    # the longest list
    (2, 5000, 0, 1.0, "float32", "int64", 0),       # no list at all
])
def test_loss_and_gradient(rows, vocab, k, tau, dtype, ids, pad):
    rng = np.random.default_rng(vocab + k)
    z, i, t = _make(rng, rows, vocab, k, dtype)
    w = rng.uniform(0.25, 2.0, rows)
    got = _run(z, i, t, tau, w, ids, pad)
    _check(z.double().numpy(), i, t.astype(np.float64), tau, w.astype(np.float32).astype(np.float64), dtype, got)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("vocab,rows,tau", [(777, 12, 2.0), (777, 12, 0.5), (70_001, 12, 2.0), (1_200_000, 2, 0.5)])
def test_masks_and_short_lists(dtype, vocab, rows, tau):
    import torch
    rng = np.random.default_rng(vocab)
    k = 20
    z, i, t = _make(rng, rows, vocab, k, dtype)
    low = torch.finfo(getattr(torch, dtype)).min
    z[0, ::2] = float("-inf")                       # masked candidates, some of them listed
    z[0, torch.from_numpy(i[0, :4])] = float("-inf")
    z[1, 1:] = float("-inf")                        # one candidate left, not listed
    i[1] = np.arange(2, 2 + k) % vocab
    if rows > 2:
        z[2, :] = float("-inf")                     # nothing left
        if tau > 1.0:                               # (lse = lowest / tau has to be an f32)
            z[3, :] = low                           # masks of the type's lowest value: all equal
        z[4, 5:] = low
        i[5, :] = -1                                # an empty list
        t[6, :] = -np.inf                           # a list without weight
        t[7, 3:] = -np.inf                          # short lists, either way
        i[8, 2:] = -1
        i[9, :] = i[9, 0]                           # one id throughout
        i[10, 10:] = i[10, :10]                     # every id twice
        t[11, 0] = 500.0                            # a teacher that is certain
    w = np.ones(rows)
    got = _run(z, i, t, tau, None)
    _check(z.double().numpy(), i, t.astype(np.float64), tau, w, dtype, got)


@pytest.mark.parametrize("k", [31, 32, 33, 100, 1024])
@pytest.mark.parametrize("pool", [1, 7, 300, 5000])
@pytest.mark.parametrize("vocab", [5003, 120_001])
def test_repeated_ids(k, pool, vocab):
    # lists of a warp and longer ones, with few, some and nearly no ids twice;
    # rows of one CTA, and rows that a cluster shares
    rng = np.random.default_rng(k + pool)
    z, _, t = _make(rng, 6, vocab, 4, "float32")
    t = (rng.standard_normal((6, k)) * 3).astype(np.float32)
    i = rng.permutation(vocab)[:pool][rng.integers(0, pool, (6, k))]
    i[3, ::3] = -1
    got = _run(z, i, t, 1.5, None)
    _check(z.double().numpy(), i, t.astype(np.float64), 1.5, np.ones(6), "float32", got)


def test_nan_and_inf_stay_in_their_row():
    import torch
    from shear_b200 import ops
    z = torch.randn(4, 300, device="cuda")
    z[1, 17] = float("nan")
    z[2, 18] = float("inf")
    ids = torch.arange(5, device="cuda").repeat(4, 1)
    t = torch.randn(4, 5, device="cuda")
    loss, lse, grad = ops.distill_topk_grad(z, ids, t)
    assert loss[1].isnan() and grad[1].isnan().all() and not loss[2].isfinite()
    clean = ops.distill_topk_grad(z[::3].contiguous(), ids[::3], t[::3])
    for x, y in zip((loss[::3], lse[::3], grad[::3]), clean):
        assert torch.equal(x, y) and x.isfinite().all()


@pytest.mark.parametrize("vocab,dtype", [(1000, "float32"), (60_001, "bfloat16"), (1_100_000, "float32")])
def test_gradient_in_place_of_the_logits(vocab, dtype):
    rng = np.random.default_rng(3)
    z, i, t = _make(rng, 3, vocab, 16, dtype)
    apart = _run(z, i, t, 1.5, None)
    placed = _run(z, i, t, 1.5, None, in_place=True)
    import torch
    for x, y in zip(apart, placed):
        assert torch.equal(x, y)


def test_gradient_against_differences():
    # Central differences of the loss in f32 logits: f has third derivatives of
    # at most tau^2 / tau^3 = 1 / tau, so h^2 / 6 / tau, and the f32 loss is good
    # to 2^-20 of about 10: that / h.
    import torch
    from shear_b200 import ops
    rng = np.random.default_rng(4)
    z, i, t = _make(rng, 2, 40, 6, "float32")
    i[0, 5] = i[0, 0]
    i[1, 4:] = -1
    tau, h = 2.0, 2.0 ** -5
    z, i, t = z.cuda(), torch.from_numpy(i).cuda(), torch.from_numpy(t).cuda()
    _, _, grad = ops.distill_topk_grad(z, i, t, tau)
    plus = z.repeat(40, 1, 1) + h * torch.eye(40, device="cuda")[:, None, :]
    minus = z.repeat(40, 1, 1) - h * torch.eye(40, device="cuda")[:, None, :]
    f = [ops.distill_topk(x.reshape(80, 40), i.repeat(40, 1), t.repeat(40, 1), tau)[0].double().view(40, 2)
         for x in (plus, minus)]
    slope = ((f[0] - f[1]) / (2 * h)).t()
    assert (slope - grad.double()).abs().max().item() <= h * h / 6 / tau + 10 * 2.0 ** -20 / h


def test_bad_ids_and_refusals():
    import torch
    from shear_b200 import ops
    from shear_b200._capi import TessaError
    z = torch.randn(3, 50, device="cuda")
    ids = torch.randint(0, 50, (3, 4), device="cuda")
    t = torch.randn(3, 4, device="cuda")
    for bad in (50, -2, 2 ** 40):
        wrong = ids.clone()
        wrong[1, 2] = bad
        got = ops.distill_topk_grad(z, wrong, t)
        with pytest.raises(TessaError) as e:
            ops.async_status()
        assert e.value.code == -5
        wrong[1, 2] = -1  # it counted as no entry
        want = ops.distill_topk_grad(z, wrong, t)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    for bad in (dict(logits=z.double()), dict(logits=z.cpu()), dict(logits=z[:, ::2]), dict(teacher_ids=ids[:2]),
                dict(teacher_ids=ids.to(torch.int16)), dict(teacher_logits=t[:, :3]),
                dict(teacher_logits=ids), dict(row_weights=torch.ones(2, device="cuda")),
                dict(out=torch.empty(3, 49, device="cuda")), dict(out=torch.empty(3, 50, device="cuda").half())):
        with pytest.raises(ValueError):
            ops.distill_topk_grad(**{"logits": z, "teacher_ids": ids, "teacher_logits": t, **bad})
    for bad in (dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("nan")),
                dict(teacher_ids=torch.zeros(3, 1025, dtype=torch.int64, device="cuda"),
                     teacher_logits=torch.zeros(3, 1025, device="cuda"))):
        with pytest.raises(TessaError) as e:
            ops.distill_topk_grad(**{"logits": z, "teacher_ids": ids, "teacher_logits": t, **bad})
        assert e.value.code == -1
    empty = ops.distill_topk_grad(z[:0], ids[:0], t[:0])
    assert empty[0].shape == (0,) and empty[2].shape == (0, 50)
