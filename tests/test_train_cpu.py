"""The trainer and the differentiable functions with plain torch in place of
the kernels, so that they run without a GPU."""
import threading

import pytest

torch = pytest.importorskip("torch")


def _rows_of(ids, rows):
    return (ids >= 0) & (ids < rows)


def _lookup(table, ids, scale=1.0, **_):
    ok = _rows_of(ids, table.shape[0])
    if not table.shape[0]:
        return table.new_zeros(*ids.shape, table.shape[1])
    return torch.where(ok.unsqueeze(-1), scale * table[torch.where(ok, ids, 0).long()], 0.0)


def _lookup_grad(dout, ids, table_rows, scale=1.0, out=None, accumulate=False, **_):
    ok = _rows_of(ids, table_rows)
    if out is None:
        out = dout.new_zeros(table_rows, dout.shape[-1])
    return out.index_add_(0, ids[ok].long(), scale * dout[ok])


def _codes(x, transpose=False, **_):
    return (x.t(), None) if transpose else (x, None)


def _product(a, a_scales, b, b_scales, out_dtype=None, **_):
    return a.float() @ b.float().t()


def _distill(logits, teacher_ids, teacher_logits, temperature=1.0, row_weights=None, out=None, **_):
    rows, vocab = logits.shape
    w = torch.ones(rows) if row_weights is None else row_weights
    loss, lse, grad = torch.zeros(rows), torch.full((rows,), float("-inf")), torch.zeros(rows, vocab)
    for r in range(rows):
        there = _rows_of(teacher_ids[r], vocab) & (teacher_logits[r] > float("-inf"))
        if not there.any():
            continue
        ids, x = teacher_ids[r][there].long(), logits[r].float() / temperature
        log_p, log_q = torch.log_softmax(teacher_logits[r][there] / temperature, 0), torch.log_softmax(x, 0)
        loss[r] = temperature ** 2 * (log_p.exp() * (log_p - log_q[ids])).sum()
        lse[r] = torch.logsumexp(x, 0)
        grad[r] = w[r] * temperature * log_q.exp().index_add(0, ids, -log_p.exp())
    if out is not None:
        grad = out.copy_(grad)
    return loss, lse, grad


@pytest.fixture
def train(monkeypatch):
    from shear_b200 import train
    plain = {"embedding_lookup": _lookup, "embedding_grad": _lookup_grad, "quantize_fp8": _codes,
             "quantize_fp8_both": lambda x, **k: (*_codes(x), *_codes(x, True)), "matmul_fp8": _product,
             "distill_topk_grad": _distill, "distill_topk": lambda *a, **k: _distill(*a, **k)[:2]}
    for name, f in plain.items():
        monkeypatch.setattr(train.ops, name, torch.no_grad()(f))  # as kernels do, they leave no graph
    seen = []  # (operator, context)
    for name in plain:
        f = getattr(train.ops, name)
        monkeypatch.setattr(train.ops, name, lambda *a, _f=f, _n=name, **k: (seen.append((_n, k.get("ctx"))), _f(*a, **k))[1])
    monkeypatch.setattr(train.ops, "context", lambda device=0: f"context of {threading.current_thread().name}")
    train.seen = seen
    yield train
    del train.seen


def _trainer(train, rows=12, dim=5):
    g = torch.Generator().manual_seed(0)
    ids = torch.stack([torch.randperm(rows, generator=g)[:4] for _ in range(6)]).int()
    return (train.TableTrainer(torch.randn(rows, dim, generator=g), 0.1, 1.5, 0.5), ids,
            torch.randn(6, 4, generator=g))


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("bad", [12, 2 ** 31 - 1, -7])
def test_an_id_outside_the_table_takes_no_part(train, bad, dtype):
    batch = torch.tensor([3, bad, 0, 5, bad, 11], dtype=dtype)
    runs = []
    for b in (batch, torch.where(batch == bad, -1, batch)):
        trainer, ids, logits = _trainer(train)
        # no list names its own row, nor the first or last one
        ids = torch.where((ids == batch.unsqueeze(1)) | (ids == 0) | (ids == 11), -1, ids)
        runs.append((trainer.step(b, ids, logits), trainer.table, trainer.scores(b)[0]))
    for x, y in zip(runs[0][:2], runs[1][:2]):
        assert torch.equal(x, y) and x.isfinite().all()
    ok = (batch != bad).nonzero()[:, 0]
    z = runs[0][2]
    assert torch.equal(z[ok], runs[1][2][ok])
    assert torch.equal((z == float("-inf")).nonzero()[:, 1][ok], batch[ok].long())  # a row's own score alone


def test_a_table_without_rows(train):
    trainer = train.TableTrainer(torch.zeros(0, 5), 0.1)
    batch = torch.full((3,), -1, dtype=torch.int32)
    assert float(trainer.step(batch, batch.unsqueeze(1), torch.zeros(3, 1))) == 0.0


@pytest.mark.parametrize("filler", [0.0, float("nan"), float("inf")])
def test_padding_rows_take_no_part_whatever_their_lists(train, filler):
    # the lists of padding rows name every row, and hold anything
    trainer, ids, logits = _trainer(train)
    start, batch = trainer.table.clone(), torch.tensor([3, 8, 5], dtype=torch.int32)
    lists = torch.where(ids[:3] == batch.unsqueeze(1), -1, ids[:3])
    want = trainer.step(batch, lists, logits[:3]), trainer.table.clone()
    share = trainer.recall(batch, lists)
    trainer.table.copy_(start)
    padded = torch.tensor([-1, 3, -1, 8, 5, -1], dtype=torch.int32)
    all_lists, all_logits = torch.arange(12).int().view(3, 4).repeat(2, 1), torch.full((6, 4), filler)
    all_lists[padded >= 0], all_logits[padded >= 0] = lists, logits[:3]
    got = trainer.step(padded, all_lists, all_logits), trainer.table
    for x, y in zip(got, want):
        assert x.isfinite().all() and torch.allclose(x, y, rtol=1e-5, atol=1e-6)
    assert trainer.recall(padded, all_lists) == share


def _first_order_cases(train):
    """(name, function of the tensors, tensors): scalars by the three functions."""
    g = torch.Generator().manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=g)
    ids, lists = torch.tensor([2, 0, 2]), torch.tensor([[0, 3], [1, 2], [4, 1]])
    return [
        ("lookup", lambda t: train.lookup(t, ids).pow(3).sum(), (rand(4, 5),)),
        ("product_fp8", lambda x, w: train.product_fp8(x, w).sum(), (rand(3, 4), rand(5, 4))),
        ("product_fp8", lambda x, w: train.product_fp8(2 * x, -w).sum(), (rand(3, 4), rand(5, 4))),
        ("product_fp8", lambda x: train.product_fp8(x, torch.ones(2, 4)).square().sum(), (rand(3, 4),)),
        ("product_fp8", lambda w: train.product_fp8(torch.ones(2, 4), w).square().sum(), (rand(3, 4),)),
        ("distill", lambda z: train.distill(z, lists, torch.ones(3, 2), 1.5).sum(), (rand(3, 5),)),
    ]


@pytest.mark.parametrize("case", range(6))
def test_a_second_derivative_is_refused_not_lost(train, case):
    name, f, tensors = _first_order_cases(train)[case]
    tensors = [t.requires_grad_() for t in tensors]
    once = torch.autograd.grad(f(*tensors), tensors)
    grads = torch.autograd.grad(f(*tensors), tensors, create_graph=True)
    for x, y in zip(grads, once):
        assert torch.equal(x, y)
    for g, t in zip(grads, reversed(tensors)):  # with two: each gradient depends on the other tensor
        with pytest.raises(RuntimeError, match=f"{name} .*second"):
            torch.autograd.grad(g.square().sum() + tensors[0].sum() + tensors[-1].sum(), t, retain_graph=True)
        with pytest.raises(RuntimeError, match=f"{name} .*second"):
            (g.square().sum() + t.sum()).backward(retain_graph=True)


def test_a_second_derivative_past_these_functions(train):
    # what does not depend on their gradients, or is linear, goes through
    t = torch.randn(4, 3).requires_grad_()
    (g,) = torch.autograd.grad(train.lookup(t, torch.tensor([1, 1])).sum() + t.pow(3).sum(), t, create_graph=True)
    (h,) = torch.autograd.grad(g.sum(), t)
    assert torch.equal(h, 6 * t.detach())
    x, w, v = (torch.randn(2, 3).requires_grad_() for _ in range(3))
    y = train.product_fp8(x, w).sum() + v.pow(2).sum()
    (gv,) = torch.autograd.grad(y, v, create_graph=True)
    y.backward(create_graph=True)
    gv.sum().backward()
    assert torch.equal(v.grad.detach(), 2 * v.detach() + 2)


def test_backwards_use_the_context_of_their_forward(train):
    # as torch does on a GPU: the backward on another thread
    for _, f, tensors in _first_order_cases(train):
        y = f(*(t.requires_grad_() for t in tensors))
        del train.seen[:]
        backward = threading.Thread(target=y.backward, name="backward")
        backward.start()
        backward.join()
        here = f"context of {threading.current_thread().name}"
        assert train.seen and all(used == here for _, used in train.seen), train.seen


@pytest.mark.parametrize("shape", [(), (3,), (0,), (2, 3), (2, 0, 3)])
@pytest.mark.parametrize("dim", [0, 1, 4])
def test_lookups_of_any_shape(train, shape, dim):
    t = torch.randn(5, dim).requires_grad_()
    ids = torch.randint(0, 5, shape)
    train.lookup(t, ids).sum().backward()
    assert torch.equal(t.grad, torch.bincount(ids.reshape(-1), minlength=5)[:, None].expand(5, dim).float())


def test_a_product_holds_neither_operand(train):
    # what leads a second derivative back to them holds no memory of its own
    x, w = torch.randn(3, 4).requires_grad_(), torch.randn(5, 4).requires_grad_()
    y = train.product_fp8(2 * x, -w)
    for link in y.grad_fn.links:
        assert link.requires_grad and link.untyped_storage().nbytes() == 0


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_lists_of_either_type(train, dtype):
    trainer, ids, logits = _trainer(train)
    start, batch = trainer.table.clone(), torch.tensor([-1, 8, 5], dtype=torch.int32)
    lists = torch.where(ids[:3] == batch.unsqueeze(1), -1, ids[:3])
    want = trainer.step(batch, lists, logits[:3]), trainer.table.clone()
    trainer.table.copy_(start)
    got = trainer.step(batch.to(dtype), lists.to(dtype), logits[:3]), trainer.table
    for x, y in zip(got, want):
        assert torch.equal(x, y)
