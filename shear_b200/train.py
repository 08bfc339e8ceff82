"""Training a table of vectors on the neighbour lists that the leaf operator
makes: a smaller table learns to rank as the given vectors do.

One step, for a batch of rows of the table (:meth:`TableTrainer.step`):

    x    = scale * table[ids]                    embedding_lookup
    z    = x . table^T                           matmul_fp8 (own row masked)
    loss = tau^2 KL(softmax(teacher / tau) over the list || softmax(z / tau))
    dz                                           distill_topk_grad, over z itself
    dx   = dz . table,  dtable = dz^T . x        matmul_fp8 on codes along the other axis
    dtable += scale * sum of dx over equal ids   embedding_grad
    table -= rate * dtable

The teacher's list is what :func:`shear_b200.ops.leaf_topk_sq8` returns: ids
(-1 where a leaf is smaller than the list) and distances.  A step only
enqueues work, so it can be captured in a CUDA graph.

:func:`lookup`, :func:`product_fp8` and :func:`distill` are the same operators
as differentiable torch functions, for models of one's own.  They have first
derivatives only: a second one through them raises.

``python -m shear_b200.train`` runs the whole path on synthetic vectors and
prints the loss and the share of the teacher's neighbours that the table ranks
among its own first k, before and after.
"""
from __future__ import annotations

import argparse
import json

import torch

from . import ops

MAX_ROWS = 65535  # rows of one leaf: teacher_lists compares all of them


class _FirstOrder(torch.autograd.Function):
    """A gradient as it is, for which nothing but an error leads back to what it depends on."""

    @staticmethod
    def forward(ctx, name, grad, *depends):
        ctx.name = name
        return grad.detach()

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError(f"{ctx.name} has no second derivative")


def _first_order(name, grad, *depends):
    """`grad` from a kernel, which leaves no graph: where one is being made
    (create_graph), a second derivative through it has to fail, not to vanish."""
    if grad is None or not torch.is_grad_enabled() or not any(t is not None and t.requires_grad for t in depends):
        return grad
    return _FirstOrder.apply(name, grad, *(t for t in depends if t is not None))


def _link(t):
    """What depends on the matrix t without holding memory that the graph does not hold anyway."""
    return t if t.is_leaf else t.repeat(0, 1)


# torch runs backwards on threads of its own, and ops.context() is a thread's:
# each backward works on the context of its forward, so that what its kernels
# report reaches the caller of the forward (ops.async_status()), and no context
# is made inside a graph capture.


class _Lookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale):
        out = ops.embedding_lookup(table, ids, scale)
        ctx.save_for_backward(ids)
        ctx.rows, ctx.scale, ctx.context = table.shape[0], scale, ops.context(out.get_device())
        return out

    @staticmethod
    def backward(ctx, dout):
        (ids,) = ctx.saved_tensors
        grad = ops.embedding_grad(_rows(ops._as_rows(dout)), ids.reshape(-1), ctx.rows, ctx.scale, ctx=ctx.context)
        return _first_order("lookup", grad, dout), None, None


class _ProductFp8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, out_dtype, links):
        need_x, need_w = ctx.needs_input_grad[:2]
        # dx needs w's codes along columns, dw those of x
        xc, xs, *x_t = ops.quantize_fp8_both(x) if need_w else ops.quantize_fp8(x)
        wc, ws, *w_t = ops.quantize_fp8_both(w) if need_x else ops.quantize_fp8(w)
        ctx.save_for_backward(*x_t, *w_t)
        ctx.types, ctx.links, ctx.context = (x.dtype, w.dtype), links, ops.context(x.get_device())
        return ops.matmul_fp8(xc, xs, wc, ws, out_dtype=out_dtype)

    @staticmethod
    def backward(ctx, dy):
        need_x, need_w = ctx.needs_input_grad[:2]
        saved = list(ctx.saved_tensors)
        x_t = (saved.pop(0), saved.pop(0)) if need_w else None
        dx = dw = None
        given, dy = dy, _rows(dy)
        if need_x and need_w:
            c, s, ct, st = ops.quantize_fp8_both(dy, ctx=ctx.context)
        elif need_x:
            c, s = ops.quantize_fp8(dy, ctx=ctx.context)
        else:
            ct, st = ops.quantize_fp8(dy, transpose=True, ctx=ctx.context)
        if need_x:
            dx = ops.matmul_fp8(c, s, *saved, out_dtype=ctx.types[0], ctx=ctx.context)
        if need_w:
            dw = ops.matmul_fp8(ct, st, *x_t, out_dtype=ctx.types[1], ctx=ctx.context)
        x, w = ctx.links
        return _first_order("product_fp8", dx, given, w), _first_order("product_fp8", dw, given, x), None, None


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher_ids, teacher_logits, temperature):
        loss = ops.distill_topk(logits, teacher_ids, teacher_logits, temperature)[0]
        ctx.save_for_backward(logits, teacher_ids, teacher_logits)
        ctx.temperature, ctx.context = temperature, ops.context(loss.get_device())
        return loss

    @staticmethod
    def backward(ctx, dloss):
        logits, ids, teacher = ctx.saved_tensors
        grad = ops.distill_topk_grad(logits, ids, teacher, ctx.temperature, row_weights=dloss, ctx=ctx.context)[2]
        return _first_order("distill", grad, dloss, logits), None, None, None


def _rows(t):
    """t, or a copy where its rows are not contiguous (a broadcast gradient)."""
    return t if (t.stride(1) == 1 or t.shape[1] <= 1) and (t.stride(0) >= t.shape[1] or t.shape[0] <= 1) else t.contiguous()


def lookup(table, ids, scale: float = 1.0):
    """Differentiable :func:`shear_b200.ops.embedding_lookup`; the table's gradient is dense and has its type."""
    return _Lookup.apply(table, ids, scale)


def product_fp8(x, w, out_dtype=torch.float32):
    """Differentiable ``x . w^T`` of FP8 codes of x [m, k] and w [n, k]
    (:func:`shear_b200.ops.matmul_fp8`): the gradients are products of FP8
    codes too, of the incoming gradient with those of w and of x."""
    both = torch.is_grad_enabled() and x.requires_grad and w.requires_grad
    return _ProductFp8.apply(x, w, out_dtype, (_link(x), _link(w)) if both else (None, None))


def distill(logits, teacher_ids, teacher_logits, temperature: float = 1.0):
    """Differentiable :func:`shear_b200.ops.distill_topk`: the loss of each row."""
    return _Distill.apply(logits, teacher_ids, teacher_logits, temperature)


def teacher_lists(vectors, k: int):
    """Every row's k nearest other rows: (ids int32 [rows, k], logits f32
    [rows, k], minus the squared distance over the lists' mean one)."""
    rows, dim = vectors.shape
    if not 1 < rows <= MAX_ROWS:
        raise ValueError(f"{rows} rows: 2 to {MAX_ROWS} are compared in one leaf")
    codes, scales, norms = ops.quantize_sq8(vectors)[:3]
    members = torch.arange(rows, dtype=torch.int32, device=vectors.device)
    ids, dists = ops.leaf_topk_sq8(codes, scales, norms, members, members, [0], [rows], k)
    ids, dists = ids.view(rows, k), dists.view(rows, k)
    valid = ids >= 0
    dists = torch.where(valid, dists, 0.0)
    mean = dists.sum() / valid.sum().clamp(min=1)
    return ids, -dists / mean.clamp(min=torch.finfo(torch.float32).tiny)


class TableTrainer:
    """Gradient descent on a table [rows, dim] (f32, updated in place) from teachers' lists.

    scale: of the looked-up rows; with logits scale * x . table^T.  The
    products run on FP8 codes, everything else in f32 but for the scores,
    which are bf16.
    """

    def __init__(self, table, rate: float, temperature: float = 1.0, scale: float = 1.0):
        if table.dtype != torch.float32 or table.dim() != 2:
            raise ValueError("the table must be a 2-D float32 tensor")
        if not temperature > 0:
            raise ValueError("temperature must be positive")
        self.table, self.rate, self.temperature, self.scale = table, rate, temperature, scale
        self._no_entry = torch.full((), -1, dtype=torch.int32, device=table.device)

    def _named(self, ids):
        """(ids brought into the table, which of them name a row of it)."""
        rows = self.table.shape[0]
        inside = ids.clamp(0, max(rows - 1, 0))
        return inside, inside == ids if rows else torch.zeros_like(ids, dtype=torch.bool)

    def scores(self, ids):
        """scale * table[ids] . table^T in bf16, each row's own score -inf; and the codes that its gradient needs."""
        return self._scores(ids, self._named(ids)[0])

    def _scores(self, ids, inside):
        x = ops.embedding_lookup(self.table, ids, self.scale)
        xq, wq = ops.quantize_fp8_both(x), ops.quantize_fp8_both(self.table)
        z = ops.matmul_fp8(*xq[:2], *wq[:2], out_dtype=torch.bfloat16)
        if z.shape[1]:  # (the row of an id outside the table takes no part, whichever of its scores this hides)
            z.scatter_(1, inside.long().unsqueeze(1), float("-inf"))
        return z, xq[2:], wq[2:]

    def step(self, ids, teacher_ids, teacher_logits):
        """One step on the batch; returns its mean loss (a device scalar).  Rows of id -1 take
        no part, nor do those of an id outside the table, which the next call reports."""
        inside, named = self._named(ids)
        z, x_t, w_t = self._scores(ids, inside)
        # a padding row's list may hold anything, an entry of the hidden score among
        # it, of which the loss is infinite: only without entries it takes no part
        teacher_ids = torch.where(named.unsqueeze(1), teacher_ids, self._no_entry)
        weights = named.float()
        weights /= weights.sum().clamp(min=1.0)
        loss, _, dz = ops.distill_topk_grad(z, teacher_ids, teacher_logits, self.temperature, weights, out=z)
        c, s, ct, st = ops.quantize_fp8_both(dz)
        grad = ops.matmul_fp8(ct, st, *x_t)
        dx = ops.matmul_fp8(c, s, *w_t)
        ops.embedding_grad(dx, ids, self.table.shape[0], self.scale, out=grad, accumulate=True)
        self.table.add_(grad, alpha=-self.rate)
        return loss @ weights

    def recall(self, ids, teacher_ids) -> float:
        """Share of the teacher's neighbours of these rows among the table's own first k."""
        inside, named = self._named(ids)
        z = self._scores(ids, inside)[0]
        teacher_ids = torch.where(named.unsqueeze(1), teacher_ids, self._no_entry)
        got = z.topk(teacher_ids.shape[1], dim=1).indices.int()
        hit = (got.unsqueeze(2) == teacher_ids.unsqueeze(1)).any(1) & (teacher_ids >= 0)
        return float(hit.sum() / (teacher_ids >= 0).sum().clamp(min=1))


def synthetic_vectors(rows: int, dim: int, seed: int, device="cuda"):
    """Rows around rows / 50 centres, of unit length."""
    g = torch.Generator(device=device).manual_seed(seed)
    centres = torch.randn(max(1, rows // 50), dim, generator=g, device=device)
    which = torch.randint(centres.shape[0], (rows,), generator=g, device=device)
    x = centres[which] + 0.5 * torch.randn(rows, dim, generator=g, device=device)
    return torch.nn.functional.normalize(x)


def main(argv=None) -> dict:
    p = argparse.ArgumentParser(prog="python -m shear_b200.train", description="Train a smaller table on SQ8 neighbour lists.")
    p.add_argument("--rows", type=int, default=20000)
    p.add_argument("--dim", type=int, default=128, help="of the given vectors")
    p.add_argument("--table-dim", type=int, default=32, help="of the table that is trained")
    p.add_argument("--k", type=int, default=16, help="length of the teacher's lists")
    p.add_argument("--batch", type=int, default=2048)
    p.add_argument("--steps", type=int, default=200)
    p.add_argument("--rate", type=float, help="default rows / 400: a row is in a batch that much more seldom")
    p.add_argument("--temperature", type=float, default=1.0)
    p.add_argument("--scale", type=float, default=16.0, help="of the looked-up rows")
    p.add_argument("--seed", type=int, default=0)
    a = p.parse_args(argv)
    if not 1 < a.rows <= MAX_ROWS:
        p.error(f"--rows must be 2 to {MAX_ROWS}")
    if min(a.dim, a.table_dim, a.k, a.batch, a.steps) < 1 or a.k >= a.rows:
        p.error("--dim, --table-dim, --k, --batch and --steps must be positive, and --k below --rows")
    if not a.temperature > 0:
        p.error("--temperature must be positive")
    vectors = synthetic_vectors(a.rows, a.dim, a.seed)
    teacher_ids, teacher_logits = teacher_lists(vectors, a.k)
    g = torch.Generator(device="cuda").manual_seed(a.seed + 1)
    # start from a random projection of the vectors
    table = torch.nn.functional.normalize(vectors @ torch.randn(a.dim, a.table_dim, generator=g, device="cuda"))
    trainer = TableTrainer(table, a.rows / 400 if a.rate is None else a.rate, a.temperature, a.scale)
    sample = torch.randperm(a.rows, generator=g, device="cuda")[:min(a.rows, 1024)].int()
    before = trainer.recall(sample, teacher_ids[sample.long()])
    losses = []
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for i in range(a.steps):
        if i == min(3, a.steps - 1):
            start.record()
        ids = torch.randint(a.rows, (a.batch,), generator=g, device="cuda").int()
        losses.append(trainer.step(ids, teacher_ids[ids.long()], teacher_logits[ids.long()]))
    end.record()
    ops.async_status()
    losses = torch.stack(losses).tolist()
    result = {"rows": a.rows, "dim": a.dim, "table_dim": a.table_dim, "k": a.k, "batch": a.batch, "steps": a.steps,
              "loss_first": losses[0], "loss_last": losses[-1], "recall_before": before,
              "recall_after": trainer.recall(sample, teacher_ids[sample.long()]),
              "ms_per_step": start.elapsed_time(end) / (a.steps - min(3, a.steps - 1))}
    print(json.dumps(result))
    return result


if __name__ == "__main__":
    main()
