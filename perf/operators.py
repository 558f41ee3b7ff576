"""Measured cases of the token-policy operators: layer norm, the cross entropy of a large-vocabulary head and the
distillation of a teacher's top logits into such a head, each forward and with gradients.

`run` computes them in plain torch operations in 32 bits (`own` false) or through the framework's entry points
(`own` true); `exact` computes them in 64 bits from the definitions."""
import math

import torch

own = False

EPS = 1e-5
BF16, F32 = torch.bfloat16, torch.float32


def listed():
    return [
        # one step of a rollout: a few dozen environments, one token each; launch latency is all there is
        dict(name="norm_step", op="norm", rows=32, cols=1024, dtype="bf16", pad=0, affine=True),
        # a training batch's activations at the large MLP's hidden width
        dict(name="norm_batch", op="norm", rows=65536, cols=2048, dtype="bf16", pad=0, affine=True),
        # the same batch on the way back, with the reductions over its rows
        dict(name="norm_grad_batch", op="norm_grad", rows=65536, cols=2048, dtype="bf16", pad=0, affine=True),
        # a ragged batch of an odd width in f32, rows cut out of a wider buffer
        dict(name="norm_grad_odd", op="norm_grad", rows=5001, cols=1003, dtype="f32", pad=5, affine=True),
        # scoring a handful of tokens (a rollout step's log-probabilities): the head's weights are read once
        dict(name="ce_step", op="ce", n=16, v=32768, d=1024, bias=True, ignored=0.0, weighted=False, pad=0),
        # evaluation of a batch of demonstrations: losses alone
        dict(name="ce_eval", op="ce", n=4096, v=32768, d=2048, bias=False, ignored=0.0, weighted=False, pad=0),
        # fine-tuning on answers: odd sizes everywhere, prompts' rows left out, a weight (advantage) per row
        dict(name="ce_grad_odd", op="ce_grad", n=2047, v=50021, d=1000, bias=True, ignored=0.4, weighted=True, pad=0),
        # a full training batch over the widest vocabulary
        dict(name="ce_grad_batch", op="ce_grad", n=16384, v=131072, d=2048, bias=False, ignored=0.0, weighted=False,
             pad=0),
        # how far a student is from its teacher on a few hundred tokens
        dict(name="distill_eval", op="distill", n=300, v=65536, d=1024, k=20, temp=1.0, bias=False, weighted=False,
             pad=0),
        # a small action vocabulary, a small student: launches count
        dict(name="distill_grad_small", op="distill_grad", n=64, v=1000, d=512, k=8, temp=1.0, bias=True,
             weighted=False, pad=0),
        # an ordinary distillation batch with softened answers, ragged and empty answer lists
        dict(name="distill_grad_batch", op="distill_grad", n=4096, v=65537, d=1024, k=64, temp=2.0, bias=True,
             weighted=True, pad=0),
        # a wide student
        dict(name="distill_grad_wide", op="distill_grad", n=2048, v=131072, d=4096, k=32, temp=1.0, bias=False,
             weighted=False, pad=0),
    ]


def _spread(rng, low, high, grain=0):
    """A whole number spread over the logarithm of [low, high], a multiple of `grain` where that is not zero."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if grain:
        v = max(grain, v // grain * grain)
    return min(high, max(low, v))


def draw(rng):
    odd = rng.random() < 0.5
    kind = rng.choice(("norm", "norm_grad", "ce", "ce_grad", "distill", "distill_grad"))
    pad = rng.choice((0, 0, 8, 3))
    if kind.startswith("norm"):
        cols = _spread(rng, 8, 16384, 0 if odd else 8)
        rows = _spread(rng, 1, min(131072, (1 << 27) // (cols + pad)))
        return dict(op=kind, rows=rows, cols=cols, dtype=rng.choice(("bf16", "f32")), pad=pad,
                    affine=rng.random() < 0.8)
    v = _spread(rng, 64, 131072, 0 if odd else 64)
    d = _spread(rng, 32, 4096, 0 if odd else 32)
    n = _spread(rng, 1, max(1, min(16384, (16384 * 131072 * 2048) // (v * d))))
    case = dict(op=kind, n=n, v=v, d=d, bias=rng.random() < 0.5, weighted=rng.random() < 0.5, pad=pad)
    if kind.startswith("ce"):
        case["ignored"] = rng.choice((0.0, 0.0, 0.2, 0.6))
    else:
        case["k"] = min(v, _spread(rng, 1, 128))
        case["temp"] = rng.choice((1.0, 1.0, 0.7, 2.0))
    return case


# ---------------------------------------------------------------------------------------------- inputs
def _rows(n, c, pad, dtype, fill):
    """An n x c matrix of `fill`'s values in rows of c + pad."""
    buf = torch.zeros(n, c + pad, dtype=dtype, device="cuda")
    x = buf[:, :c]
    x.copy_(fill)
    return x


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=F32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case=case)
    if case["op"].startswith("norm"):
        n, c, dtype = case["rows"], case["cols"], (BF16 if case["dtype"] == "bf16" else F32)
        # activations of a residual stream: a common offset per column, rows of different scale
        x = _randn(gen, n, c).mul_(torch.exp(0.5 * _randn(gen, n, 1))).add_(0.3 * _randn(gen, 1, c))
        s["x"] = _rows(n, c, case["pad"], dtype, x)
        s["w"] = 1.0 + 0.1 * _randn(gen, c) if case["affine"] else None
        s["b"] = 0.1 * _randn(gen, c) if case["affine"] else None
        if case["op"] == "norm_grad":
            s["dy"] = _rows(n, c, case["pad"], dtype, _randn(gen, n, c).mul_(1e-2))
            xf = s["x"].float()
            s["mean"] = xf.mean(1)
            s["rstd"] = torch.rsqrt((xf - s["mean"][:, None]).square().mean(1) + EPS)
        return s
    n, v, d = case["n"], case["v"], case["d"]
    s["w"] = _rows(v, d, case["pad"], BF16, _randn(gen, v, d).mul_(1.5 / math.sqrt(d)))
    s["bias"] = (0.2 * _randn(gen, v)).to(BF16) if case["bias"] else None
    s["scale"] = _randn(gen, n).div_(n) if case["weighted"] else torch.full((n,), 1.0 / n, device="cuda")
    # hidden states that lean towards the rows of their answers, from not at all to surely
    x = _randn(gen, n, d)
    if case["op"].startswith("ce"):
        t = torch.randint(0, v, (n,), generator=gen, device="cuda")
        lean = torch.rand(n, 1, generator=gen, device="cuda") * 6.0
        x += lean * s["w"][t].float()
        left_out = torch.rand(n, generator=gen, device="cuda") < case["ignored"]
        s["target"] = torch.where(left_out, torch.full_like(t, -1), t).to(torch.int32)
    else:
        k = case["k"]
        first = torch.randint(0, v, (n, 1), generator=gen, device="cuda")
        ids = (first + torch.arange(k, device="cuda")[None] * max(1, v // k)) % v  # distinct within a row
        s["teacher"] = (2.5 * _randn(gen, n, k)).sort(1, descending=True).values.contiguous()
        x += (torch.rand(n, 1, generator=gen, device="cuda") * 4.0) * s["w"][ids[:, 0]].float()
        # answer lists end early; some rows (padding of a batch) have none
        count = torch.randint(max(1, k // 2), k + 1, (n, 1), generator=gen, device="cuda")
        count *= torch.rand(n, 1, generator=gen, device="cuda") >= 0.03
        s["ids"] = torch.where(torch.arange(k, device="cuda")[None] < count, ids, torch.full_like(ids, -1)).to(torch.int32)
    s["x"] = _rows(n, d, case["pad"], BF16, x)
    return s


# ---------------------------------------------------------------------------------------------- one pass
def run(s):
    return _framework(s) if own else _plain(s)


def _framework(s):
    from pufferlean_b200 import tokens

    case = s["case"]
    op = case["op"]
    if op == "norm":
        return tokens.layer_norm(s["x"], s["w"], s["b"], EPS)
    if op == "norm_grad":
        return tokens.layer_norm_grad(s["dy"], s["x"], s["w"], s["mean"], s["rstd"])
    if op == "ce":
        return tokens.vocab_ce(s["x"], s["w"], s["target"], s["bias"])
    if op == "ce_grad":
        return tokens.vocab_ce_grad(s["x"], s["w"], s["target"], s["bias"], s["scale"])
    if op == "distill":
        return tokens.vocab_distill(s["x"], s["w"], s["ids"], s["teacher"], s["bias"], case["temp"])
    return tokens.vocab_distill_grad(s["x"], s["w"], s["ids"], s["teacher"], s["bias"], case["temp"], s["scale"])


def _plain(s):
    op = s["case"]["op"]
    if op == "norm":
        x = s["x"].float()
        mean = x.mean(1)
        x = x - mean[:, None]
        rstd = 1.0 / torch.sqrt((x * x).mean(1) + EPS)
        y = x * rstd[:, None]
        if s["w"] is not None:
            y = y * s["w"] + s["b"]
        return y.to(s["x"].dtype), mean, rstd
    if op == "norm_grad":
        dy, rstd = s["dy"].float(), s["rstd"][:, None]
        xh = (s["x"].float() - s["mean"][:, None]) * rstd
        dw, db = (dy * xh).sum(0), dy.sum(0)
        if s["w"] is not None:
            dy = dy * s["w"]
        dx = rstd * (dy - dy.mean(1, keepdim=True) - xh * (dy * xh).mean(1, keepdim=True))
        return dx.to(s["x"].dtype), dw, db
    return _plain_head(s)


def _plain_head(s):
    case = s["case"]
    x, w = s["x"].float(), s["w"].float()
    temp = case.get("temp", 1.0)
    z = x @ w.t()
    if s["bias"] is not None:
        z += s["bias"].float()
    if temp != 1.0:
        z /= temp
    if "target" in s:
        ids = s["target"].long()[:, None]
        here = ids >= 0
        p = here.float()
        ids = ids.clamp(min=0)
        logp = torch.zeros_like(p)
    else:
        here = s["ids"] >= 0
        ids = s["ids"].long().clamp(min=0)
        t = torch.where(here, s["teacher"] / temp, -math.inf)
        top = t.max(1, keepdim=True).values
        t = t - torch.where(torch.isfinite(top), top, 0.0)
        p = torch.exp(t)
        total = p.sum(1, keepdim=True).clamp(min=1e-30)
        p = p / total
        logp = torch.where(here, t - torch.log(total), 0.0)
    some = here.any(1)
    zk = torch.gather(z, 1, ids)
    top = z.max(1, keepdim=True).values
    z -= top
    z.exp_()
    total = z.sum(1, keepdim=True)
    lse = (top + torch.log(total))[:, 0]
    loss = torch.where(some, lse + (p * (logp - zk)).sum(1), 0.0)
    lse = torch.where(some, lse, 0.0)
    if not case["op"].endswith("grad"):
        return loss, lse
    scale = torch.where(some, s["scale"] / temp, 0.0)[:, None]
    z *= scale / total
    z.scatter_add_(1, ids, -scale * p)
    dx = (z @ w).to(BF16)
    dw = (z.t() @ x).to(BF16)
    return loss, lse, dx, dw, (z.sum(0).to(BF16) if s["bias"] is not None else None)


# ---------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op.startswith("norm"):
        x = s["x"].double()
        w = s["w"].double() if s["w"] is not None else torch.ones(x.shape[1], dtype=torch.float64, device="cuda")
        if op == "norm":
            mean = x.sum(1) / x.shape[1]
            var = ((x - mean[:, None]) ** 2).sum(1) / x.shape[1]
            rstd = (var + EPS) ** -0.5
            y = torch.einsum("rc,r,c->rc", x - mean[:, None], rstd, w)
            return (y if s["b"] is None else y + s["b"].double()), mean, rstd
        dy, mean, rstd = s["dy"].double(), s["mean"].double(), s["rstd"].double()
        xh = torch.einsum("rc,r->rc", x - mean[:, None], rstd)
        g = dy * w
        c = x.shape[1]
        along = torch.einsum("rc,rc->r", g, xh) / c
        dx = (g - (g.sum(1) / c)[:, None] - xh * along[:, None]) * rstd[:, None]
        return dx, torch.einsum("rc,rc->c", dy, xh), dy.sum(0)
    return _exact_head(s)


def _exact_head(s):
    case = s["case"]
    n, v = case["n"], case["v"]
    temp = case.get("temp", 1.0)
    w = s["w"].double()
    loss = torch.zeros(n, dtype=torch.float64, device="cuda")
    lse = torch.zeros_like(loss)
    grad = case["op"].endswith("grad")
    dx, dw, db = (torch.zeros(n, case["d"], dtype=torch.float64, device="cuda"), torch.zeros_like(w),
                  torch.zeros(v, dtype=torch.float64, device="cuda")) if grad else (None, None, None)
    step = max(1, (1 << 28) // v)
    for r0 in range(0, n, step):
        r = slice(r0, min(n, r0 + step))
        x = s["x"][r].double()
        u = torch.einsum("nd,vd->nv", x, w)
        if s["bias"] is not None:
            u = u + s["bias"].double()
        u = u / temp
        want = torch.zeros_like(u)  # the answer's distribution over the whole vocabulary
        if "target" in s:
            t = s["target"][r].long()
            i = torch.nonzero(t >= 0)[:, 0]
            want[i, t[i]] = 1.0
            entropy = torch.zeros(len(t), dtype=torch.float64, device="cuda")
        else:
            ids = s["ids"][r].long()
            q = torch.where(ids >= 0, s["teacher"][r].double() / temp, -math.inf)
            q = torch.nan_to_num(torch.softmax(q, 1), nan=0.0)
            entropy = torch.special.entr(q).sum(1)
            i, k = torch.nonzero(ids >= 0, as_tuple=True)
            want.index_put_((i, ids[i, k]), q[i, k], accumulate=True)
        some = want.sum(1)  # one, or zero where the row has no answer
        all_lse = torch.logsumexp(u, 1)
        lse[r] = all_lse * (some > 0.5)
        loss[r] = (all_lse - (want * u).sum(1) - entropy) * (some > 0.5)
        if grad:
            dz = (torch.softmax(u, 1) * (some > 0.5)[:, None] - want) * (s["scale"][r].double() / temp)[:, None]
            dx[r] = dz @ w
            dw += dz.t() @ x
            db += dz.sum(0)
    if not grad:
        return loss, lse
    return loss, lse, dx, dw, (db if s["bias"] is not None else None)


# ---------------------------------------------------------------------------------------------- what a pass needs
def work(case):
    op = case["op"]
    if op.startswith("norm"):
        n, c, size = case["rows"], case["cols"], (2 if case["dtype"] == "bf16" else 4)
        params = 8 * c if case["affine"] else 0
        if op == "norm":
            return dict(bytes=2 * n * c * size + params + 8 * n, flops=8 * n * c)
        return dict(bytes=3 * n * c * size + 8 * n + params // 2 + 8 * c, flops=14 * n * c)
    n, v, d, k = case["n"], case["v"], case["d"], case.get("k", 1)
    rows = n * (1.0 - case.get("ignored", 0.0))  # rows that are left out need nothing
    grad = op.endswith("grad")
    each = 2 * (rows * d + v * d) + (2 * v if case["bias"] else 0)
    lists = 4 * n if "k" not in case else 8 * n * k
    return dict(bytes=each * (2 if grad else 1) + lists + 8 * n + (4 * n if grad else 0),
                flops=(6 if grad else 2) * rows * v * d)
