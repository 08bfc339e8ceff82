"""Training a table: the operators together, as torch functions and as a step."""
import json
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("args", [["--rows", "1"], ["--rows", "65536"], ["--k", "0"], ["--rows", "16", "--k", "16"],
                                  ["--steps", "0"], ["--temperature", "0"]])
def test_the_command_refuses(args, capsys):
    from shear_b200 import train
    with pytest.raises(SystemExit):
        train.main(args)
    assert "error" in capsys.readouterr().err


def test_refusals():
    import torch
    from shear_b200 import train
    for table in (torch.zeros(4, 4, dtype=torch.float64), torch.zeros(4)):
        with pytest.raises(ValueError):
            train.TableTrainer(table, 1.0)
    with pytest.raises(ValueError):
        train.TableTrainer(torch.zeros(4, 4), 1.0, temperature=0.0)
    for rows in (1, train.MAX_ROWS + 1):
        with pytest.raises(ValueError):
            train.teacher_lists(torch.zeros(1, 4).expand(rows, 4), 4)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(7,), (3, 5), (0,)])
def test_lookup_gradient(shape):
    import torch
    from shear_b200 import train
    g = torch.Generator().manual_seed(1)
    table = torch.randn(11, 20, generator=g).cuda().requires_grad_()
    ids = torch.randint(0, 3, shape, generator=g).cuda()
    out = train.lookup(table, ids, 0.5)
    assert torch.equal(out, 0.5 * table.detach()[ids])  # an exact scale
    up = torch.randn(*shape, 20, generator=g).cuda()
    out.backward(up)
    want = torch.zeros(11, 20, dtype=torch.float64, device="cuda")
    want.index_add_(0, ids.reshape(-1), 0.5 * up.double().reshape(-1, 20))
    # sums of at most n terms of one id, each addition rounded once
    n = ids.numel()
    mag = torch.zeros_like(want).index_add_(0, ids.reshape(-1), 0.5 * up.double().abs().reshape(-1, 20))
    assert ((table.grad.double() - want).abs() <= (n + 1) * 2.0 ** -24 * mag).all()
    table.grad = None
    train.lookup(table, ids).sum().backward()  # one value broadcast over the gradient
    count = torch.bincount(ids.reshape(-1), minlength=11).float()
    assert torch.equal(table.grad, count[:, None].expand(11, 20))


@pytest.mark.gpu
@pytest.mark.parametrize("need", ["both", "x", "w"])
def test_product_gradient(need):
    # small whole numbers: the codes, the products and their sums are exact
    import torch
    from shear_b200 import train
    g = torch.Generator().manual_seed(2)
    x, w = (torch.randint(-8, 9, s, generator=g).float().cuda() for s in ((33, 50), (140, 50)))
    x.requires_grad_(need != "w")
    w.requires_grad_(need != "x")
    y = train.product_fp8(x, w)
    assert torch.equal(y.double(), x.detach().double() @ w.detach().double().t())
    up = torch.randint(-8, 9, (33, 140), generator=g).float().cuda()
    for dy in (up, up[:, :1].expand(33, 140), up[:1, :1].expand(33, 140), up.t().contiguous().t()):
        x.grad = w.grad = None
        y.backward(dy, retain_graph=True)
        if need != "w":
            assert torch.equal(x.grad.double(), dy.double() @ w.detach().double())
        if need != "x":
            assert torch.equal(w.grad.double(), dy.double().t() @ x.detach().double())


@pytest.mark.gpu
def test_distillation_gradient_is_the_operators():
    import torch
    from shear_b200 import ops, train
    g = torch.Generator().manual_seed(3)
    z = torch.randn(9, 301, generator=g).cuda().requires_grad_()
    ids = torch.stack([torch.randperm(301, generator=g)[:6] for _ in range(9)]).int().cuda()
    tl = torch.randn(9, 6, generator=g).cuda()
    loss = train.distill(z, ids, tl, 2.0)
    weights = torch.rand(9, generator=g).cuda()
    for up in (weights, torch.ones(1, device="cuda").expand(9)):
        z.grad = None
        loss.backward(up, retain_graph=True)
        want_loss, _, want = ops.distill_topk_grad(z.detach(), ids, tl, 2.0, row_weights=up.contiguous())
        assert torch.equal(z.grad, want)
        # loss alone may split a row otherwise: sums of 301 terms in another order
        assert torch.allclose(loss.detach(), want_loss, rtol=0, atol=301 * 2.0 ** -24 * 4 * 10)


def _trainer(rows=500, dim=40, k=8, seed=0):
    import torch
    from shear_b200 import train
    vectors = train.synthetic_vectors(rows, 64, seed)
    ids, logits = train.teacher_lists(vectors, k)
    table = torch.randn(rows, dim, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")
    return train.TableTrainer(table, 0.1, 1.5, 0.25), ids, logits


@pytest.mark.gpu
def test_teacher_lists():
    import torch
    from shear_b200 import train
    x = train.synthetic_vectors(300, 32, 1)
    ids, logits = train.teacher_lists(x, 5)
    assert ids.shape == logits.shape == (300, 5) and (ids >= 0).all() and (ids < 300).all()
    assert (ids != torch.arange(300, device="cuda")[:, None]).all()
    assert (logits <= 0).all() and float(logits.mean()) == pytest.approx(-1.0, rel=1e-5)
    short = train.teacher_lists(x[:3], 5)
    assert (short[0][:, 2:] == -1).all() and short[1].isfinite().all()


@pytest.mark.gpu
def test_step_follows_the_loss():
    # the step's direction against differences of its own loss: along the
    # gradient g = (before - after) / rate, loss(table - e g) - loss(table + e g)
    # = -2 e |g|^2 up to third order, the codes' rounding (a share 2^-4 of each
    # of table, x and dz) and the scores' (2^-9): a quarter at most
    import torch
    trainer, ids, logits = _trainer()
    batch = torch.arange(0, 500, 2, device="cuda").int()
    start = trainer.table.clone()

    def loss(table):
        x = 0.25 * table[batch.long()].double()
        z = x @ table.double().t()
        z[torch.arange(250), batch.long()] = float("-inf")
        lq = torch.log_softmax(z / 1.5, 1).gather(1, ids[batch.long()].long())
        lp = torch.log_softmax(logits[batch.long()].double() / 1.5, 1)
        return float((1.5 ** 2 * (lp.exp() * (lp - lq)).sum(1)).mean())

    got = float(trainer.step(batch, ids[batch.long()], logits[batch.long()]))
    assert got == pytest.approx(loss(start), rel=0.05)
    g = ((start - trainer.table) / 0.1).double()
    e = 1e-3 / float(g.norm())
    slope = (loss(start.double() + e * g) - loss(start.double() - e * g)) / (2 * e)
    assert slope == pytest.approx(float((g * g).sum()), rel=0.25)


@pytest.mark.gpu
def test_padding_rows_and_determinism():
    import torch
    trainer, ids, logits = _trainer()
    start = trainer.table.clone()
    none = torch.full((16,), -1, dtype=torch.int32, device="cuda")
    assert float(trainer.step(none, ids[:16], logits[:16])) == 0.0
    assert torch.equal(trainer.table, start)
    batch = torch.randint(0, 500, (64,), generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").int()
    runs = []
    for _ in range(2):
        trainer.table.copy_(start)
        loss = trainer.step(batch, ids[batch.long()], logits[batch.long()])
        runs.append((loss.clone(), trainer.table.clone()))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
    assert not torch.equal(runs[0][1], start) and runs[0][1].isfinite().all()


@pytest.mark.gpu
def test_step_in_a_graph_and_on_another_stream():
    import torch
    trainer, ids, logits = _trainer()
    start = trainer.table.clone()
    batch = torch.arange(100, device="cuda").int()
    loss = trainer.step(batch, ids[:100], logits[:100])
    want = loss.clone(), trainer.table.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        trainer.table.copy_(start)
        loss = trainer.step(batch, ids[:100], logits[:100])
        side.synchronize()
        assert torch.equal(loss, want[0]) and torch.equal(trainer.table, want[1])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            loss = trainer.step(batch, ids[:100], logits[:100])
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):
        trainer.table.copy_(start)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, want[0]) and torch.equal(trainer.table, want[1])


@pytest.mark.gpu
def test_the_command_learns():
    run = subprocess.run([sys.executable, "-m", "shear_b200.train", "--rows", "3000", "--steps", "80", "--batch", "512",
                          "--k", "8"], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]
    r = json.loads(run.stdout.strip().splitlines()[-1])
    assert r["loss_last"] < 0.7 * r["loss_first"] and r["recall_after"] > r["recall_before"] + 0.1


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [500, 2 ** 31 - 1, -2])
def test_an_id_outside_the_table_is_reported(bad):
    # the step, or the wait behind it, raises; the device goes on, and so does the table
    import torch
    from shear_b200 import ops
    from shear_b200._capi import TessaError
    trainer, ids, logits = _trainer()
    start = trainer.table.clone()
    batch = torch.arange(40, device="cuda").int()
    want = trainer.step(batch, ids[:40], logits[:40]), trainer.table.clone()
    trainer.table.copy_(start)
    wrong = batch.clone()
    wrong[7] = bad
    with pytest.raises(TessaError) as e:
        trainer.step(wrong, ids[:40], logits[:40])
        ops.async_status()
    assert e.value.code == -5
    torch.cuda.synchronize()
    assert trainer.table.isfinite().all()
    trainer.table.copy_(start)
    got = trainer.step(batch, ids[:40], logits[:40])
    ops.async_status()
    assert torch.equal(got, want[0]) and torch.equal(trainer.table, want[1])


@pytest.mark.gpu
def test_padding_rows_with_lists_of_anything():
    import torch
    trainer, ids, logits = _trainer()
    start = trainer.table.clone()
    batch = torch.arange(100, 140, device="cuda").int()
    want = trainer.step(batch, ids[100:140], logits[100:140]), trainer.table.clone()
    padded = torch.cat([batch, torch.full((24,), -1, device="cuda", dtype=torch.int32)])
    lists = torch.cat([ids[100:140], torch.arange(8, device="cuda").int().repeat(24, 1)])  # id 0 among them
    for filler in (0.0, float("nan"), float("inf")):
        trainer.table.copy_(start)
        loss = trainer.step(padded, lists, torch.cat([logits[100:140], torch.full((24, 8), filler, device="cuda")]))
        # the same sums, of which the products' may be split otherwise (bf16 scores, FP8 codes of a step's size)
        assert torch.allclose(loss, want[0], rtol=1e-4)
        assert torch.allclose(trainer.table, want[1], rtol=0, atol=float((want[1] - start).abs().max()) / 16)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["lookup", "product_fp8", "distill"])
def test_second_derivatives_are_refused(name):
    import torch
    from shear_b200 import train
    t, w = (torch.randn(9, 32, device="cuda").requires_grad_() for _ in range(2))
    ids = torch.tensor([[1, 2], [0, 3], [5, 4], [7, 8], [3, 3], [1, 0], [8, 0], [2, 6], [4, 5]], device="cuda")
    y = {"lookup": lambda: train.lookup(t, ids).square(), "product_fp8": lambda: train.product_fp8(t, w),
         "distill": lambda: train.distill(t, ids, torch.ones(9, 2, device="cuda"))}[name]().sum()
    (plain,) = torch.autograd.grad(y, t, retain_graph=True)
    (g,) = torch.autograd.grad(y, t, create_graph=True)
    assert torch.equal(g.detach(), plain)
    with pytest.raises(RuntimeError, match=f"{name} has no second derivative"):
        torch.autograd.grad(g.square().sum() + t.sum() + w.sum(), w if name == "product_fp8" else t)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(), (3,), (0,), (2, 3), (2, 0, 3)])
@pytest.mark.parametrize("dim", [0, 1, 4])
def test_lookups_of_any_shape(shape, dim):
    import torch
    from shear_b200 import ops, train
    t = torch.randn(5, dim, device="cuda").requires_grad_()
    ids = torch.randint(0, 5, shape, device="cuda")
    y = train.lookup(t, ids)
    assert y.shape == (*shape, dim)
    y.sum().backward()
    want = torch.bincount(ids.reshape(-1), minlength=5)[:, None].expand(5, dim).float()
    assert torch.equal(t.grad, want)
    assert torch.equal(ops.embedding_grad(torch.ones(*shape, dim, device="cuda"), ids, 5), want)
