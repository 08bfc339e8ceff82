"""Cases of the embedding-training operators: the FP8 block-scaled product and
its gradients, the embedding lookup and its gradient, and the distillation loss
from a teacher's top-k list.

``run`` computes a case in plain torch (``own`` false) or through the package's
entry points (``own`` true); ``exact`` computes the definition in 64 bits.
Sizes are those of the framework's own configurations (200,000 x 128,
1M x 768, 768-d and 512-d vectors, lists of 32 and 64 entries) and ragged ones.
"""
import math

import torch

own = False

DEV = "cuda"
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
INT = {"i32": torch.int32, "i64": torch.int64}


def listed():
    return [
        # One query scored against the whole 200,000-vector collection: latency.
        dict(name="score_1x200000x128", op="product", m=1, n=200_000, k=128, x="f32", out="f32", grads=False),
        # A query batch scored against the collection at 768 dimensions: the largest product.
        dict(name="score_4096x200000x768", op="product", m=4096, n=200_000, k=768, x="bf16", out="bf16", grads=False),
        # One training step's scores, batch x candidates, with both gradients.
        dict(name="step_2048x16384x768", op="product", m=2048, n=16_384, k=768, x="bf16", out="bf16", grads=True),
        # Odd everything: rows, candidates and dimensions that end inside a tile and inside a scale block.
        dict(name="step_777x5003x1000", op="product", m=777, n=5_003, k=1_000, x="f16", out="f32", grads=True),
        # The rows of one small batch: latency.
        dict(name="lookup_64_of_200000x128", op="lookup", t=64, v=200_000, d=128, x="f32", ids="i32", zipf=False, grad=False),
        # 8,192 queries with 32 candidates each, out of a million vectors.
        dict(name="lookup_262144_of_1Mx768", op="lookup", t=262_144, v=1_000_000, d=768, x="bf16", ids="i64", zipf=False, grad=False),
        # The gradient of a batch whose popular rows come up thousands of times.
        dict(name="lookup_grad_131072_of_200000x128", op="lookup", t=131_072, v=200_000, d=128, x="f32", ids="i32", zipf=True, grad=True),
        # The gradient of the large batch over the million-row table.
        dict(name="lookup_grad_262144_of_1Mx768", op="lookup", t=262_144, v=1_000_000, d=768, x="bf16", ids="i64", zipf=True, grad=True),
        # Loss alone (validation) of a few queries over the whole collection.
        dict(name="distill_4x200000_k32", op="distill", t=4, v=200_000, k=32, x="f32", ids="i32", tau=1.0, ragged=False, grad=False),
        # The training step's loss and gradient over its candidates.
        dict(name="distill_grad_2048x16384_k32", op="distill", t=2048, v=16_384, k=32, x="bf16", ids="i32", tau=2.0, ragged=False, grad=True),
        # Loss and gradient over a million candidates.
        dict(name="distill_grad_1024x1M_k64", op="distill", t=1024, v=1_000_000, k=64, x="bf16", ids="i32", tau=1.0, ragged=False, grad=True),
        # Odd sizes, short and empty lists, repeated ids, masked candidates.
        dict(name="distill_grad_333x50003_k100", op="distill", t=333, v=50_003, k=100, x="f16", ids="i64", tau=2.0, ragged=True, grad=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["product", "lookup", "distill"])
    if op == "product":
        while True:
            c = dict(op=op, m=_log(rng, 1, 16_384), n=_log(rng, 64, 300_000), k=_log(rng, 64, 2_048),
                     x=rng.choice(["f32", "bf16", "f16"]), out=rng.choice(["f32", "bf16"]), grads=rng.random() < 0.4)
            if c["m"] * c["n"] * c["k"] * (3 if c["grads"] else 1) <= 4096 * 200_000 * 768 and c["m"] * c["n"] <= 4096 * 200_000:
                return c
    if op == "lookup":
        while True:
            c = dict(op=op, t=_log(rng, 1, 524_288), v=_log(rng, 1_000, 1_000_000), d=_log(rng, 32, 2_048),
                     x=rng.choice(["f32", "bf16", "f16"]), ids=rng.choice(["i32", "i64"]),
                     zipf=rng.random() < 0.5, grad=rng.random() < 0.5)
            if c["v"] * c["d"] <= 1_000_000 * 768 and c["t"] * c["d"] <= 262_144 * 768:
                return c
    while True:
        c = dict(op=op, t=_log(rng, 1, 8_192), v=_log(rng, 1_000, 1_000_000), k=_log(rng, 8, 128),
                 x=rng.choice(["f32", "bf16", "f16"]), ids=rng.choice(["i32", "i64"]),
                 tau=rng.choice([0.5, 1.0, 2.0]), ragged=rng.random() < 0.4, grad=rng.random() < 0.7)
        if c["t"] * c["v"] * SIZE[c["x"]] <= 1024 * 1_000_000 * 2 and c["k"] < c["v"] // 4:
            return c


def work(case):
    c = case
    e = SIZE[c["x"]]
    if c["op"] == "product":
        m, n, k, o = c["m"], c["n"], c["k"], SIZE[c["out"]]
        kb = 4 * math.ceil(math.ceil(k / 128) / 4)
        if not c["grads"]:  # x, the collection's codes and scales, the scores
            return {"bytes": m * k * e + n * (k + kb) + m * n * o, "flops": 2 * m * n * k}
        # x, w and dout once; scores and both gradients
        return {"bytes": (m * k + n * k + m * n) * e + m * n * o + (m + n) * k * o, "flops": 6 * m * n * k}
    if c["op"] == "lookup":
        ib = 4 if c["ids"] == "i32" else 8
        rows = c["v"] if c["grad"] else c["t"]
        return {"bytes": c["t"] * (ib + c["d"] * e) + rows * c["d"] * e, "flops": c["t"] * c["d"]}
    ib = 4 if c["ids"] == "i32" else 8
    return {"bytes": c["t"] * c["v"] * e * (2 if c["grad"] else 1) + c["t"] * (c["k"] * (4 + ib) + 12), "flops": 4 * c["t"] * c["v"]}


# ------------------------------------------------------------------ inputs

def _vectors(g, rows, dim, dtype):
    """L2-normalised rows around 64 centres of unlike spread, as embeddings are."""
    centres = torch.randn(64, dim, generator=g, device=DEV)
    spread = 0.05 + 0.45 * torch.rand(64, dim, generator=g, device=DEV)
    which = torch.randint(0, 64, (rows,), generator=g, device=DEV)
    x = torch.randn(rows, dim, generator=g, device=DEV).mul_(spread[which]).add_(centres[which])
    return x.div_(x.norm(dim=1, keepdim=True)).to(dtype)


def _ids(g, count, rows, zipf, dtype):
    if not zipf:
        return torch.randint(0, rows, (count,), generator=g, device=DEV).to(dtype)
    # Popularity ~ 1 / (rank + 10), the popular rows anywhere in the table.
    u = torch.rand(count, generator=g, device=DEV, dtype=torch.float64)
    rank = (10.0 * ((rows / 10.0 + 1.0) ** u - 1.0)).to(torch.int64).clamp_(0, rows - 1)
    return torch.randperm(rows, generator=g, device=DEV)[rank].to(dtype)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    dt = DT[c["x"]]
    s = {"case": c}
    if c["op"] == "product":
        s["x"] = _vectors(g, c["m"], c["k"], dt)
        w = _vectors(g, c["n"], c["k"], dt)
        if c["grads"]:
            s["w"] = w
            # rows of softmax-minus-target: small everywhere, a few large entries
            s["dout"] = (torch.randn(c["m"], c["n"], generator=g, device=DEV) * 1e-2).to(dt)
            top = torch.randint(0, c["n"], (c["m"], 1), generator=g, device=DEV)
            top = (top + c["n"] // 16 * torch.arange(16, device=DEV)) % c["n"]
            s["dout"].scatter_(1, top, -torch.rand(c["m"], 16, generator=g, device=DEV).to(dt))
        else:
            # the collection is held in codes (one byte a value) and scale bytes
            codes, e = _to_blocks(w.float())
            n, kb = e.shape
            s["w_codes"] = torch.zeros(n, -(-c["k"] // 16) * 16, dtype=torch.float8_e4m3fn, device=DEV)
            s["w_codes"][:, :c["k"]] = codes.reshape(n, -1)[:, :c["k"]]
            s["w_scales"] = torch.zeros(n, -(-kb // 4) * 4, dtype=torch.uint8, device=DEV)
            s["w_scales"][:, :kb] = (e + 127).to(torch.uint8)
        return s
    if c["op"] == "lookup":
        s["ids"] = _ids(g, c["t"], c["v"], c["zipf"], INT[c["ids"]])
        s["scale"] = math.sqrt(c["d"])
        if c["grad"]:
            s["dout"] = torch.randn(c["t"], c["d"], generator=g, device=DEV).mul_(1e-2).to(dt)
        else:
            s["table"] = _vectors(g, c["v"], c["d"], dt)
        return s
    t, v, k = c["t"], c["v"], c["k"]
    s["z"] = torch.randn(t, v, generator=g, device=DEV).mul_(2.0).to(dt)
    # distinct ids a row: a random start and odd steps through the candidates
    start = torch.randint(0, v, (t, 1), generator=g, device=DEV)
    step = torch.randint(1, v // k, (t, 1), generator=g, device=DEV)
    ids = (start + step * torch.arange(k, device=DEV)) % v
    s["tl"] = -torch.sort(torch.rand(t, k, generator=g, device=DEV) * 8.0, dim=1).values
    # the student has learnt something: the listed candidates score higher
    s["z"].scatter_add_(1, ids, (s["tl"] + 8.0).to(dt))
    if c["ragged"]:
        masked = torch.randint(0, v, (t, max(1, v // 16)), generator=g, device=DEV)
        keep = s["z"].gather(1, ids)
        s["z"].scatter_(1, masked, float("-inf"))
        low = masked[:, : max(1, v // 64)]
        s["z"].scatter_(1, low, torch.finfo(dt).min)
        s["z"].scatter_(1, ids, keep)
        ids[:, -1] = ids[:, 0]  # an id that is listed twice
        length = torch.randint(0, k + 1, (t, 1), generator=g, device=DEV)
        length[0] = 0
        ids = torch.where(torch.arange(k, device=DEV) < length, ids, torch.full_like(ids, -1))
    s["ids"] = ids.to(INT[c["ids"]])
    s["weights"] = 0.5 + torch.rand(t, generator=g, device=DEV)
    return s


# ------------------------------------------------------------ plain forms

def _two_to(e):
    """2^e in f32, exactly, for whole e in -127..127 (pow may be an ulp off)."""
    return torch.where(e < -126, torch.full_like(e, 1 << 22), (e + 127) << 23).view(torch.float32)


def _to_blocks(x):
    """Blocks of 128 along the rows: codes [rows, blocks, 128] and the power of two of each block's scale."""
    rows, k = x.shape
    nb = -(-k // 128)
    b = torch.zeros(rows, nb * 128, dtype=torch.float32, device=x.device)
    b[:, :k] = x
    b = b.view(rows, nb, 128)
    frac, e = torch.frexp(b.abs().amax(dim=2))
    # the least power of two that brings the block's largest value to 448 = 0.875 * 2^9 or below
    e = torch.where(frac == 0, torch.full_like(e, -127), (e - 9 + (frac > 0.875).to(e.dtype)).clamp(-127, 127))
    return (b * _two_to(-e)[:, :, None]).to(torch.float8_e4m3fn), e


def _from_blocks(codes, e, k):
    return (codes.float() * _two_to(e)[:, :, None]).reshape(codes.shape[0], -1)[:, :k]


def _rounded(x):
    codes, e = _to_blocks(x.float())
    return _from_blocks(codes, e, x.shape[1])


def _plain_product(s):
    c = s["case"]
    out = DT[c["out"]]
    if not c["grads"]:
        n, kp = s["w_codes"].shape
        kb = -(-c["k"] // 128)
        codes = torch.zeros(n, kb * 128, dtype=torch.float8_e4m3fn, device=DEV)
        codes[:, :kp] = s["w_codes"]
        w = _from_blocks(codes.view(n, kb, 128), s["w_scales"][:, :kb].to(torch.int32) - 127, c["k"])
        return (_rounded(s["x"]) @ w.t()).to(out)
    y = _rounded(s["x"]) @ _rounded(s["w"]).t()
    dx = _rounded(s["dout"]) @ _rounded(s["w"].t()).t()
    dw = _rounded(s["dout"].t()) @ _rounded(s["x"].t()).t()
    return {"y": y.to(out), "dx": dx.to(out), "dw": dw.to(out)}


def _plain_lookup(s):
    c = s["case"]
    ids = s["ids"].long()
    if not c["grad"]:
        return (s["table"][ids].float() * s["scale"]).to(s["table"].dtype)
    grad = torch.zeros(c["v"], c["d"], dtype=torch.float32, device=DEV)
    grad.index_add_(0, ids, s["dout"].float())
    return (grad * s["scale"]).to(s["dout"].dtype)


def _plain_distill(s):
    c = s["case"]
    tau = c["tau"]
    listed_ = s["ids"] >= 0
    at = s["ids"].long().clamp(min=0)
    z = s["z"].float()
    top = z.amax(dim=1, keepdim=True)
    u = torch.exp((z - top) / tau)
    total = u.sum(dim=1, keepdim=True)
    logq = (z.gather(1, at) - top) / tau - torch.log(total)
    lse = top / tau + torch.log(total)
    t = torch.where(listed_, s["tl"], torch.full_like(s["tl"], float("-inf")))
    tmax = t.amax(dim=1, keepdim=True)
    some = tmax > float("-inf")
    d = torch.where(listed_, (t - torch.where(some, tmax, torch.zeros_like(tmax))) / tau, torch.zeros_like(t))
    w = torch.where(listed_, torch.exp(d), torch.zeros_like(d))
    sum_w = torch.where(some, w.sum(dim=1, keepdim=True), torch.ones_like(tmax))
    p = w / sum_w
    terms = torch.where(listed_, p * (d - torch.log(sum_w) - logq), torch.zeros_like(p))
    loss = tau * tau * terms.sum(dim=1)
    lse = lse[:, 0]
    if not c["grad"]:
        return {"loss": loss, "lse": lse}
    grad = u.div_(total)
    grad.scatter_add_(1, at, -p)
    grad *= torch.where(some, tau * s["weights"][:, None], torch.zeros_like(tmax))
    return {"loss": loss, "lse": lse, "grad": grad.to(s["z"].dtype)}


def _own(s):
    from shear_b200 import ops

    c = s["case"]
    if c["op"] == "product":
        if not c["grads"]:
            return ops.matmul_fp8(*ops.quantize_fp8(s["x"]), s["w_codes"], s["w_scales"], out_dtype=DT[c["out"]])
        x, xs, xt, xts = ops.quantize_fp8_both(s["x"])
        w, ws, wt, wts = ops.quantize_fp8_both(s["w"])
        y = ops.matmul_fp8(x, xs, w, ws, out_dtype=DT[c["out"]])
        d, ds, dt, dts = ops.quantize_fp8_both(s["dout"])
        dx = ops.matmul_fp8(d, ds, wt, wts, out_dtype=DT[c["out"]])
        dw = ops.matmul_fp8(dt, dts, xt, xts, out_dtype=DT[c["out"]])
        return {"y": y, "dx": dx, "dw": dw}
    if c["op"] == "lookup":
        if not c["grad"]:
            return ops.embedding_lookup(s["table"], s["ids"], s["scale"])
        return ops.embedding_grad(s["dout"], s["ids"], c["v"], s["scale"], out_dtype=s["dout"].dtype)
    if not c["grad"]:
        loss, lse = ops.distill_topk(s["z"], s["ids"], s["tl"], c["tau"])
        return {"loss": loss, "lse": lse}
    loss, lse, grad = ops.distill_topk_grad(s["z"], s["ids"], s["tl"], c["tau"], s["weights"])
    return {"loss": loss, "lse": lse, "grad": grad}


def run(state):
    if own:
        return _own(state)
    return {"product": _plain_product, "lookup": _plain_lookup, "distill": _plain_distill}[state["case"]["op"]](state)


# ------------------------------------------------- the definitions, 64 bits

def _pow2_64(power):
    """2^power in 64 bits, written as its bits."""
    return ((power.to(torch.int64) + 1023) << 52).view(torch.float64)


def _e4m3_blocks64(x):
    """x in 64 bits with each block of 128 columns rounded as the codec defines it: values on the
    e4m3 grid (3 fraction bits, least exponent -6, ties to even) times the block's power of two."""
    rows, k = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -k % 128)).reshape(-1, 128)
    amax = b.abs().amax(dim=1, keepdim=True)
    power = torch.ceil(torch.log2((amax / 448.0).clamp(min=2.0 ** -127)))
    # log2 may be off by one at an exact power of two: settle it by comparison
    power = torch.where(amax <= 448.0 * _pow2_64(power - 1), power - 1, power)
    power = torch.where(amax > 448.0 * _pow2_64(power), power + 1, power).clamp(-127, 127)
    scale = _pow2_64(power)
    y = b / scale
    exponent = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -20)))
    exponent = torch.where(_pow2_64(exponent) > y.abs(), exponent - 1, exponent)
    exponent = torch.where(_pow2_64(exponent + 1) <= y.abs(), exponent + 1, exponent).clamp(min=-6.0)
    ulp = _pow2_64(exponent - 3)
    return (torch.round(y / ulp) * ulp * scale).reshape(rows, -1)[:, :k]


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "product":
        if not c["grads"]:
            # the collection's codes are an input: their values are what they stand for
            w = s["w_codes"][:, :c["k"]].double()
            w = w * _pow2_64(s["w_scales"].to(torch.int64) - 127).repeat_interleave(128, dim=1)[:, :c["k"]]
            return _e4m3_blocks64(s["x"]) @ w.t()
        x, w, d = s["x"], s["w"], s["dout"]
        y = _e4m3_blocks64(x) @ _e4m3_blocks64(w).t()
        dx = torch.einsum("mn,kn->mk", _e4m3_blocks64(d), _e4m3_blocks64(w.t()))
        dw = torch.einsum("nm,km->nk", _e4m3_blocks64(d.t()), _e4m3_blocks64(x.t()))
        return {"y": y, "dx": dx, "dw": dw}
    if c["op"] == "lookup":
        ids = s["ids"].long()
        if not c["grad"]:
            return s["table"].index_select(0, ids).double() * s["scale"]
        # equal ids side by side, then sums between their borders
        order = torch.argsort(ids, stable=True)
        uniq, counts = torch.unique_consecutive(ids[order], return_counts=True)
        grad = torch.zeros(c["v"], c["d"], dtype=torch.float64, device=DEV)
        grad[uniq] = torch.segment_reduce(s["dout"].double()[order], "sum", lengths=counts, axis=0) * s["scale"]
        return grad
    tau, t = c["tau"], c["t"]
    valid = s["ids"] >= 0
    at = torch.where(valid, s["ids"].long(), torch.zeros_like(s["ids"].long()))
    loss = torch.zeros(t, dtype=torch.float64, device=DEV)
    lses = torch.zeros(t, dtype=torch.float64, device=DEV)
    grad = torch.zeros(t, c["v"], dtype=torch.float64, device=DEV) if c["grad"] else None
    for r in range(0, t, 128):
        rows = slice(r, min(t, r + 128))
        z = s["z"][rows].double() / tau
        ok = valid[rows]
        lses[rows] = torch.logsumexp(z, dim=1)
        log_q = z - lses[rows][:, None]
        tl = torch.where(ok, s["tl"][rows].double() / tau, torch.full_like(s["tl"][rows].double(), -math.inf))
        any_ = ok.any(dim=1, keepdim=True)
        log_p = tl - torch.where(any_, torch.logsumexp(tl, dim=1, keepdim=True), torch.zeros_like(tl[:, :1]))
        p = torch.exp(log_p)
        diff = torch.where(ok, log_p - log_q.gather(1, at[rows]), torch.zeros_like(log_p))
        loss[rows] = tau * tau * (p * diff).sum(dim=1)
        if grad is not None:
            target = torch.zeros_like(z).scatter_add_(1, at[rows], p)
            grad[rows] = tau * s["weights"][rows].double()[:, None] * (torch.exp(log_q) - target) * any_
    if grad is None:
        return {"loss": loss, "lse": lses}
    return {"loss": loss, "lse": lses, "grad": grad}
