"""Measured cases of the recurrent token policy's operators: drawing tokens from logits (temperature, top-k, top-p,
min-p), the norms around a block with its gate and residual scale, and the gated delta rule, a matrix memory per head
(packed sequences in chunks, with gradients, and one token at a time).

`run` computes them in plain torch operations (`own` false) or through the framework's entry points (`own` true);
`exact` computes them in 64 bits from the definitions."""
import math

import torch

own = False

EPS = 1e-5
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
CHUNK = 64  # of the plain form


def listed():
    return [
        # a rollout's step: a few dozen environments draw their next token with the usual filters; launch latency counts
        dict(name="sample_step", op="sample", n=32, v=32768, dtype="bf16", pad=0, temp=0.8, k=50, p=0.95, min_p=0.0,
             per_row=False),
        # a large batch of rollouts over the widest vocabulary, nucleus alone: no small candidate set is known before
        dict(name="sample_nucleus", op="sample", n=1024, v=131072, dtype="bf16", pad=0, temp=1.0, k=0, p=0.9, min_p=0.0,
             per_row=False),
        # the policy's own distribution, as on-policy learning wants it, each environment at its own temperature; odd
        # vocabulary, f32 logits in a wider buffer
        dict(name="sample_odd", op="sample", n=2047, v=50021, dtype="f32", pad=3, temp=1.0, k=0, p=1.0, min_p=0.0,
             per_row=True),
        # one step of a rollout through a block
        dict(name="block_step", op="block", rows=32, cols=1024, dtype="bf16", pad=0, gate=True, post=True),
        # a training batch at the large MLP's hidden width
        dict(name="block_batch", op="block", rows=65536, cols=2048, dtype="bf16", pad=0, gate=True, post=True),
        # the same on the way back
        dict(name="block_grad_batch", op="block_grad", rows=65536, cols=2048, dtype="bf16", pad=0, gate=True, post=True),
        # a ragged batch of an odd width in f32, without a gate
        dict(name="block_grad_odd", op="block_grad", rows=5001, cols=1003, dtype="f32", pad=5, gate=False, post=True),
        # a rollout's step of the memory: every environment's state is read and written
        dict(name="delta_step", op="delta_step", n=256, hk=8, hv=16, dk=128, dv=128),
        # scoring a few long sequences
        dict(name="delta_long", op="delta", lengths="even", n_seq=4, length=8192, hk=16, hv=16, dk=128, dv=128,
             reset=0.0, state=True),
        # a training batch of rollout segments, with episodes that end inside them
        dict(name="delta_grad_batch", op="delta_grad", lengths="even", n_seq=64, length=512, hk=8, hv=8, dk=128, dv=128,
             reset=0.004, state=True),
        # episodes of different lengths packed one behind the other, odd widths, keys shared by three heads of values
        dict(name="delta_grad_odd", op="delta_grad", lengths="ragged", n_seq=37, length=150, hk=2, hv=6, dk=72, dv=100,
             reset=0.01, state=False),
    ]


def _spread(rng, low, high, grain=0):
    """A whole number spread over the logarithm of [low, high], a multiple of `grain` where that is not zero."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if grain:
        v = max(grain, v // grain * grain)
    return min(high, max(low, v))


def draw(rng):
    odd = rng.random() < 0.5
    kind = rng.choice(("sample", "sample", "block", "block_grad", "delta_step", "delta", "delta_grad", "delta_grad"))
    if kind == "sample":
        v = _spread(rng, 16, 131072, 0 if odd else 16)
        n = _spread(rng, 1, max(1, min(4096, (1 << 27) // v)))
        return dict(op=kind, n=n, v=v, dtype=rng.choice(("bf16", "f32")), pad=rng.choice((0, 0, 8, 3)),
                    temp=rng.choice((1.0, 1.0, 0.6, 1.3)), k=rng.choice((0, 0, _spread(rng, 1, 1000))),
                    p=rng.choice((1.0, 0.5, 0.9, 0.99)), min_p=rng.choice((0.0, 0.0, 0.02, 0.1)),
                    per_row=rng.random() < 0.3)
    if kind.startswith("block"):
        cols = _spread(rng, 8, 8192, 0 if odd else 8)
        pad = rng.choice((0, 0, 8, 3))
        return dict(op=kind, rows=_spread(rng, 1, min(131072, (1 << 27) // (cols + pad))), cols=cols, pad=pad,
                    dtype=rng.choice(("bf16", "f32")), gate=rng.random() < 0.7, post=rng.random() < 0.7)
    hk = _spread(rng, 1, 8)
    hv = hk * rng.choice((1, 1, 2, 3))
    dk = _spread(rng, 8, 128, 0 if odd else 8)
    dv = _spread(rng, 8, 128, 0 if odd else 8)
    if kind == "delta_step":
        return dict(op=kind, n=_spread(rng, 1, max(1, 4096 // hv)), hk=hk, hv=hv, dk=dk, dv=dv)
    length = _spread(rng, 1, 2048)
    n_seq = _spread(rng, 1, max(1, min(256, (1 << 18) // (length * hv))))
    return dict(op=kind, lengths=rng.choice(("even", "ragged")), n_seq=n_seq, length=length, hk=hk, hv=hv, dk=dk, dv=dv,
                reset=rng.choice((0.0, 0.01)), state=rng.random() < 0.5)


# ---------------------------------------------------------------------------------------------- inputs
def _rows(n, c, pad, dtype, fill):
    """An n x c matrix of `fill`'s values in rows of c + pad."""
    buf = torch.zeros(n, c + pad, dtype=dtype, device="cuda")
    x = buf[:, :c]
    x.copy_(fill)
    return x


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=F32)


def _rand(gen, *shape):
    return torch.rand(*shape, generator=gen, device="cuda", dtype=F32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case=case)
    op = case["op"]
    if op == "sample":
        n, v, dtype = case["n"], case["v"], (BF16 if case["dtype"] == "bf16" else F32)
        # from rows that hardly prefer any token to rows that are all but sure
        logits = _randn(gen, n, v).mul_(1.0 + 3.0 * _rand(gen, n, 1))
        s["logits"] = _rows(n, v, case["pad"], dtype, logits)
        s["u"] = _rand(gen, n)
        if case["per_row"]:
            s["temp"] = case["temp"] * (0.5 + _rand(gen, n))
            s["p"] = (case["p"] - 0.2 * _rand(gen, n)) if case["p"] < 1.0 else torch.ones(n, device="cuda")
            s["k"] = torch.randint(0, 2 * case["k"] + 1, (n,), generator=gen, device="cuda", dtype=torch.int32)
            s["min_p"] = case["min_p"] * _rand(gen, n)
        else:
            s["temp"], s["p"], s["k"], s["min_p"] = case["temp"], case["p"], case["k"], case["min_p"]
        return s
    if op.startswith("block"):
        n, c, pad, dtype = case["rows"], case["cols"], case["pad"], (BF16 if case["dtype"] == "bf16" else F32)
        # the residual stream and a block's output: rows of different scale, columns with an offset
        s["x"] = _rows(n, c, pad, dtype, _randn(gen, n, c).mul_(torch.exp(0.5 * _randn(gen, n, 1))))
        s["branch"] = _rows(n, c, pad, dtype, _randn(gen, n, c).add_(0.2 * _randn(gen, 1, c)))
        s["gate"] = _rows(n, c, pad, dtype, _randn(gen, n, c)) if case["gate"] else None
        s["post_weight"] = 1.0 + 0.1 * _randn(gen, c)
        s["weight"] = 1.0 + 0.1 * _randn(gen, c)
        s["scale"] = 0.5
        if op == "block_grad":
            s["dr"] = _rows(n, c, pad, dtype, _randn(gen, n, c).mul_(1e-2))
            s["dy"] = _rows(n, c, pad, dtype, _randn(gen, n, c).mul_(1e-2))
            r, _, s["rstd_branch"], s["rstd"] = _block_plain(s)
            s["r"] = _rows(n, c, pad, dtype, r)
        return s
    hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
    if op == "delta_step":
        n, n_seq = case["n"], case["n"]
    else:
        n_seq, most = case["n_seq"], case["length"]
        lengths = [most] * n_seq
        if case["lengths"] == "ragged":  # some of them empty; the case's own, whatever the seed
            draw = torch.rand(n_seq, generator=torch.Generator().manual_seed(n_seq + 1000 * most))
            lengths = [0 if f < 0.04 else max(1, int(round(2 * f * most))) for f in draw.tolist()]
            if sum(lengths) == 0:
                lengths[0] = 1
        n = sum(lengths)
        s["lengths"] = lengths
        ends = torch.tensor(lengths).cumsum(0)
        s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), ends]).to(torch.int32).cuda()
        # the same as a rectangle of whole chunks (plain form): which row of the packed ones stands where, the last
        # (a row of zeros behind them) where there is none; and where each packed row stands
        wide = max(1, -(-max(lengths) // CHUNK)) * CHUNK
        col, length = torch.arange(wide)[None], torch.tensor(lengths)[:, None]
        s["rect"] = torch.where(col < length, ends[:, None] - length + col, n).cuda()
        s["place"] = (torch.arange(n_seq * wide).view(n_seq, wide))[col < length].cuda()
    # one projection's output holds queries, keys and values side by side; queries and keys have length one
    wide = torch.empty(n, 2 * hk * dk + hv * dv, dtype=BF16, device="cuda")
    s["q"] = wide[:, :hk * dk].view(n, hk, dk)
    s["k"] = wide[:, hk * dk:2 * hk * dk].view(n, hk, dk)
    s["v"] = wide[:, 2 * hk * dk:].view(n, hv, dv)
    for name, lean in (("q", 0.0), ("k", 0.5)):
        x = _randn(gen, n, hk, dk) + lean * _randn(gen, 1, hk, dk)  # keys have something in common
        s[name].copy_(x / x.norm(dim=2, keepdim=True).clamp(min=1e-6))
    s["v"].copy_(_randn(gen, n, hv, dv))
    # decays from almost none to a memory of a few tokens; an episode's first token forgets everything
    s["g"] = -torch.exp(_randn(gen, n, hv) - 3.0)
    s["beta"] = torch.sigmoid(_randn(gen, n, hv))
    s["scale"] = dk ** -0.5
    if case.get("reset"):
        s["g"][_rand(gen, n) < case["reset"]] = -math.inf
    s["state"] = _randn(gen, n_seq, hv, dk, dv).mul_(0.1) if case.get("state", True) else None
    if op == "delta_grad":
        s["do"] = _randn(gen, n, hv, dv).to(BF16)
        s["dstate"] = _randn(gen, n_seq, hv, dk, dv).mul_(0.1)
    return s


# ---------------------------------------------------------------------------------------------- one pass
def run(s):
    if own:
        return _framework(s)
    op = s["case"]["op"]
    if op == "sample":
        return _sample_plain(s)
    if op == "block":
        return _block_plain(s)
    if op == "block_grad":
        return _block_grad_plain(s)
    if op == "delta_step":
        return _delta_step_plain(s)
    return _delta_plain(s, op == "delta_grad")


def _framework(s):
    from pufferlean_b200 import tokens

    op = s["case"]["op"]
    if op == "sample":
        return tokens.sample(s["logits"], s["u"], s["temp"], s["k"], s["p"], s["min_p"])
    if op == "block":
        return tokens.block_norm(s["x"], s["branch"], s["gate"], s["post_weight"], s["weight"], s["scale"], EPS,
                                 s["case"]["post"])
    if op == "block_grad":
        return tokens.block_norm_grad(s["dr"], s["dy"], s["branch"], s["gate"], s["r"], s["rstd_branch"], s["rstd"],
                                      s["post_weight"], s["weight"], s["scale"])
    if op == "delta_step":
        return tokens.delta_rule_step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], s["scale"])
    if op == "delta":
        o, final, _ = tokens.delta_rule(s["q"], s["k"], s["v"], s["g"], s["beta"], s["offsets"], s["state"], s["scale"])
        return o, final
    o, final, saved = tokens.delta_rule(s["q"], s["k"], s["v"], s["g"], s["beta"], s["offsets"], s["state"], s["scale"],
                                        save=True)
    dq, dk, dv, dg, dbeta, dstate = tokens.delta_rule_grad(s["do"], s["dstate"], s["q"], s["k"], s["v"], s["g"],
                                                           s["beta"], s["offsets"], saved, s["scale"])
    return (o, final, dq, dk, dv, dg, dbeta) + ((dstate,) if s["state"] is not None else ())


def _column(x, n):
    """An option of every row, given as one number or one per row, as a column of doubles."""
    if torch.is_tensor(x):
        return x.double()[:, None]
    return torch.full((n, 1), float(x), dtype=F64, device="cuda")


def _sample_plain(s):
    n, v = s["logits"].shape
    temp, p, min_p, k = (_column(s[o], n) for o in ("temp", "p", "min_p", "k"))
    z = s["logits"].double()
    top = z.max(1, keepdim=True).values
    e = torch.exp((z - top) / temp)
    if torch.is_tensor(s["k"]) or s["k"] or torch.is_tensor(s["p"]) or s["p"] < 1.0:
        order = torch.sort(s["logits"].float(), dim=1, descending=True, stable=True).indices  # ties: lowest index first
        se = torch.gather(e, 1, order)
        among = torch.arange(v, device="cuda")[None] < torch.where(k > 0, k, float(v))
        se = torch.where(among, se, 0.0)
        mass = torch.cumsum(se, 1)
        keep = among & ((mass - se < p * mass[:, -1:]) | (p >= 1.0))
        keep[:, 0] = True
        kept = torch.zeros_like(keep).scatter_(1, order, keep)
        e = torch.where(kept, e, 0.0)
        del order, se, among, mass, keep, kept
    e = torch.where(e >= min_p, e, 0.0)
    cdf = torch.cumsum(e, 1)
    total = cdf[:, -1:]
    token = (cdf <= s["u"].double()[:, None] * total).sum(1, keepdim=True).clamp(max=v - 1)
    logp = (torch.gather(z, 1, token) - top) / temp - torch.log(total)
    return token[:, 0].to(torch.int32), logp[:, 0].float()


def _block_plain(s):
    case = s["case"]
    n = s["branch"].float()
    rstd_branch = None
    if case["post"]:
        rstd_branch = torch.rsqrt(n.square().mean(1) + EPS)
        n = n * rstd_branch[:, None]
    n = n * s["post_weight"]
    if s["gate"] is not None:
        n = n * torch.sigmoid(s["gate"].float())
    r = (s["x"].float() + s["scale"] * n).to(s["x"].dtype)
    f = r.float()
    rstd = torch.rsqrt(f.square().mean(1) + EPS)
    return r, (f * rstd[:, None] * s["weight"]).to(r.dtype), rstd_branch, rstd


def _block_grad_plain(s):
    dtype = s["r"].dtype
    dy, r, b = s["dy"].float(), s["r"].float(), s["branch"].float()
    rh = r * s["rstd"][:, None]
    dweight = (dy * rh).sum(0)
    dy = dy * s["weight"]
    d = s["dr"].float() + s["rstd"][:, None] * (dy - rh * (dy * rh).mean(1, keepdim=True))
    bh = b if s["rstd_branch"] is None else b * s["rstd_branch"][:, None]
    dn = d * s["scale"]
    dgate = None
    if s["gate"] is not None:
        a = torch.sigmoid(s["gate"].float())
        dgate = (dn * bh * s["post_weight"] * a * (1.0 - a)).to(dtype)
        dn = dn * a
    dpost = (dn * bh).sum(0)
    db = dn * s["post_weight"]
    if s["rstd_branch"] is not None:
        db = s["rstd_branch"][:, None] * (db - bh * (db * bh).mean(1, keepdim=True))
    return d.to(dtype), db.to(dtype), dgate, dpost, dweight


def _delta_step_plain(s):
    group = s["case"]["hv"] // s["case"]["hk"]
    q, k = (s[n].float().repeat_interleave(group, 1) for n in ("q", "k"))
    state = s["state"] * torch.exp(s["g"])[:, :, None, None]
    u = s["beta"][:, :, None] * (s["v"].float() - torch.matmul(k[:, :, None], state)[:, :, 0])
    state = state + k[..., None] * u[:, :, None]
    return (s["scale"] * torch.matmul(q[:, :, None], state)[:, :, 0]).to(BF16), state


def _delta_plain(s, grad):
    """Chunks of 64 tokens: within one, u = (I + A)^-1 b with A lower triangular, so that a chunk is a few products."""
    case = s["case"]
    hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
    group, (n_seq, length) = hv // hk, s["rect"].shape
    nc = length // CHUNK
    leaves = [s[n].detach().float() for n in ("q", "k", "v", "g", "beta")]
    state = s["state"] if s["state"] is not None else torch.zeros(n_seq, hv, dk, dv, device="cuda")
    leaves.append(state.detach().clone())
    reset = torch.isinf(leaves[3])
    leaves[3] = torch.where(reset, 0.0, leaves[3])
    with torch.set_grad_enabled(grad):
        if grad:
            leaves = [x.requires_grad_() for x in leaves]
        q, k, v, g, beta, state = leaves

        def chunks(x):  # [chunks, sequences, heads, 64, ...]
            x = torch.cat([x, torch.zeros_like(x[:1])])[s["rect"]]
            x = x.view((n_seq, nc, CHUNK) + tuple(x.shape[2:]))
            return x.permute((1, 0, 3, 2) + tuple(range(4, x.dim())))

        q, k = (chunks(x).repeat_interleave(group, 2) for x in (q, k))
        v, beta = chunks(v), chunks(beta)[..., None]
        cum = torch.cumsum(chunks(g).double(), -1)
        era = torch.cumsum(chunks(reset.float()), -1)
        low = torch.ones(CHUNK, CHUNK, device="cuda").tril().bool()
        among = low & (era[..., :, None] == era[..., None, :])
        decay = torch.where(among, torch.exp(torch.where(among, cum[..., :, None] - cum[..., None, :], 0.0)), 0.0).float()
        since = torch.where(era == 0, torch.exp(torch.where(era == 0, cum, 0.0)), 0.0).float()[..., None]
        last = era == era[..., -1:]
        until = torch.where(last, torch.exp(torch.where(last, cum[..., -1:] - cum, 0.0)), 0.0).float()[..., None]
        a = (beta * (k @ k.transpose(-1, -2)) * decay).tril(-1)
        with torch.no_grad():
            inv = torch.eye(CHUNK, device="cuda").expand_as(a).clone()
            for i in range(1, CHUNK):
                inv[..., i, :i] = -(a[..., i:i + 1, :i] @ inv[..., :i, :i])[..., 0, :]
        if grad:  # the same value, with the derivative of an inverse
            inv = inv - inv @ (a - a.detach()) @ inv
        p = (q @ k.transpose(-1, -2)) * decay
        o = []
        for c in range(nc):
            u = inv[c] @ (beta[c] * (v[c] - since[c] * (k[c] @ state)))
            o.append(s["scale"] * (since[c] * (q[c] @ state) + p[c] @ u))
            state = since[c][..., -1:, :] * state + k[c].transpose(-1, -2) @ (until[c] * u)
        o = torch.stack(o, 1).permute(0, 1, 3, 2, 4).reshape(n_seq * length, hv, dv)[s["place"]]
        if not grad:
            return o.to(BF16), state
        grads = torch.autograd.grad((o, state), leaves, (s["do"].float(), s["dstate"]))
    dq, dk_, dv_, dg, dbeta, dstate = grads
    dg = torch.where(reset, 0.0, dg)
    out = (o.detach().to(BF16), state.detach(), dq.to(BF16), dk_.to(BF16), dv_.to(BF16), dg, dbeta)
    return out + ((dstate,) if s["state"] is not None else ())


# ---------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op == "sample":
            return _sample_exact(s)
        if op == "block":
            return _block_exact(s)
        if op == "block_grad":
            return _block_grad_exact(s)
        if op == "delta_step":
            return _delta_step_exact(s)
        return _delta_exact(s, op == "delta_grad")


def _sample_exact(s):
    """Row by row: the kept tokens as an explicit set, the draw by a search in their cumulative sums."""
    n, v = s["logits"].shape
    if n * v > 1 << 28:
        return None
    tokens, logps = [], []
    pick = lambda o, i: s[o][i].double() if torch.is_tensor(s[o]) else float(s[o])
    ks = s["k"].tolist() if torch.is_tensor(s["k"]) else [s["k"]] * n
    ps = s["p"].tolist() if torch.is_tensor(s["p"]) else [s["p"]] * n
    for i in range(n):
        row = s["logits"][i].double()
        w = torch.softmax(row / pick("temp", i), 0)
        ids = torch.arange(v, device="cuda")
        if ks[i] or ps[i] < 1.0:
            order = torch.argsort(row, descending=True, stable=True)
            if ks[i]:
                order = order[:ks[i]]
            if ps[i] < 1.0:
                share = torch.cumsum(w[order], 0)
                share = share / share[-1].clone()
                count = torch.searchsorted(share, torch.full((1,), ps[i], dtype=F64, device="cuda"))[0] + 1
                order = torch.where(torch.arange(len(order), device="cuda") < count, order, -1)
            ids = torch.sort(order).values
        wi = torch.where(ids >= 0, w[ids.clamp(min=0)], 0.0)
        wi = torch.where(wi >= pick("min_p", i) * w.max(), wi, 0.0)
        cdf = torch.cumsum(wi, 0)
        j = torch.searchsorted(cdf, (s["u"][i].double() * cdf[-1])[None], right=True).clamp(max=len(ids) - 1)
        tokens.append(ids[j])
        logps.append(torch.log(wi[j] / cdf[-1]))
    return torch.cat(tokens).to(torch.int32), torch.cat(logps)


def _block_exact(s):
    b, x = s["branch"].double(), s["x"].double()
    rb = None
    if s["case"]["post"]:
        rb = (torch.einsum("rc,rc->r", b, b) / b.shape[1] + EPS) ** -0.5
        b = torch.einsum("rc,r->rc", b, rb)
    a = s["scale"] * s["post_weight"].double() / (1.0 + torch.exp(-s["gate"].double())) if s["gate"] is not None else (
        s["scale"] * s["post_weight"].double())
    r = x + a * b
    # the second norm is of the residual stream as it is stored, in the inputs' type
    stored = r.to(s["x"].dtype).double()
    rr = (torch.einsum("rc,rc->r", stored, stored) / b.shape[1] + EPS) ** -0.5
    return r, torch.einsum("rc,r,c->rc", stored, rr, s["weight"].double()), rb, rr


def _block_grad_exact(s):
    c = s["r"].shape[1]
    rh = torch.einsum("rc,r->rc", s["r"].double(), s["rstd"].double())
    gy = s["dy"].double() * s["weight"].double()
    along = torch.einsum("rc,rc->r", gy, rh) / c
    d = s["dr"].double() + torch.einsum("rc,r->rc", gy - torch.einsum("rc,r->rc", rh, along), s["rstd"].double())
    bh = s["branch"].double()
    if s["rstd_branch"] is not None:
        bh = torch.einsum("rc,r->rc", bh, s["rstd_branch"].double())
    a, dgate = torch.ones_like(d), None
    if s["gate"] is not None:
        t = torch.exp(-s["gate"].double())
        a = 1.0 / (1.0 + t)
        dgate = s["scale"] * d * bh * s["post_weight"].double() * a * (t / (1.0 + t))
    db = s["scale"] * d * a * s["post_weight"].double()
    dpost = torch.einsum("rc,rc->c", s["scale"] * d * a, bh)
    if s["rstd_branch"] is not None:
        db = torch.einsum("rc,r->rc", db - bh * (torch.einsum("rc,rc->r", db, bh) / c)[:, None], s["rstd_branch"].double())
    return d, db, dgate, dpost, torch.einsum("rc,rc->c", s["dy"].double(), rh)


def _delta_step_exact(s):
    group = s["case"]["hv"] // s["case"]["hk"]
    k, q = (torch.repeat_interleave(s[n].double(), group, 1) for n in ("k", "q"))
    st = torch.einsum("nhij,nh->nhij", s["state"].double(), torch.exp(s["g"].double()))
    err = s["v"].double() - torch.einsum("nhij,nhi->nhj", st, k)
    st = st + torch.einsum("nhi,nhj,nh->nhij", k, err, s["beta"].double())
    return s["scale"] * torch.einsum("nhij,nhi->nhj", st, q), st


def _delta_exact(s, grad):
    """One token of every sequence after the other; the way back from states kept every 64 tokens."""
    case = s["case"]
    hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
    group, lengths = hv // hk, s["lengths"]
    n_seq, steps = len(lengths), max(lengths)
    if steps * (3 if grad else 1) * (1e-3 + n_seq * hv * dk * dv * 8e-11) > 20.0:
        return None
    n = s["q"].shape[0]
    start = s["offsets"][:-1].long()
    live = torch.tensor(lengths, device="cuda")
    q, k = (s[x].double().repeat_interleave(group, 1) for x in ("q", "k"))
    v, beta, a, do = s["v"].double(), s["beta"].double(), torch.exp(s["g"].double()), None
    state = torch.zeros(n_seq, hv, dk, dv, dtype=F64, device="cuda")
    if s["state"] is not None:
        state += s["state"]
    o = torch.zeros(n, hv, dv, dtype=F64, device="cuda")

    def forward(t, state):
        on = live > t
        at = (start + t).clamp(max=n - 1)
        m = on[:, None].double()
        sd = state * torch.where(on[:, None], a[at], 1.0)[..., None, None]
        err = v[at] - torch.einsum("nhij,nhi->nhj", sd, k[at])
        u = err * (beta[at] * m)[..., None]
        return on, at, sd, err, u, sd + torch.einsum("nhi,nhj->nhij", k[at], u)

    kept = []
    for t in range(steps):
        if grad and t % 64 == 0:
            kept.append(state)
        on, at, _, _, _, state = forward(t, state)
        out = s["scale"] * torch.einsum("nhij,nhi->nhj", state, q[at])
        o.index_add_(0, at, torch.where(on[:, None, None], out, 0.0))
    if not grad:
        return o, state
    final, do = state, s["do"].double()
    ds = s["dstate"].double()
    dq, dkk = torch.zeros(n, hv, dk, dtype=F64, device="cuda"), torch.zeros(n, hv, dk, dtype=F64, device="cuda")
    dvv, dg, dbeta = torch.zeros_like(o), torch.zeros(n, hv, dtype=F64, device="cuda"), torch.zeros(n, hv, dtype=F64,
                                                                                                   device="cuda")
    for c in range(len(kept) - 1, -1, -1):
        state, path = kept[c], []
        for t in range(64 * c, min(steps, 64 * c + 64)):
            path.append(forward(t, state))
            state = path[-1][-1]
        for on, at, sd, err, u, state in reversed(path):
            m = on[:, None].double()
            dot = do[at] * m[..., None] * s["scale"]
            dq.index_add_(0, at, torch.einsum("nhij,nhj->nhi", state, dot))
            ds = ds + torch.einsum("nhi,nhj->nhij", q[at], dot)
            du = torch.einsum("nhij,nhi->nhj", ds, k[at])
            dr = du * (beta[at] * m)[..., None]
            dkk.index_add_(0, at, (torch.einsum("nhij,nhj->nhi", ds, u) - torch.einsum("nhij,nhj->nhi", sd, dr)) * m[..., None])
            dbeta.index_add_(0, at, (du * err).sum(-1) * m)
            dvv.index_add_(0, at, dr)
            ds = ds - torch.einsum("nhi,nhj->nhij", k[at], dr)
            dg.index_add_(0, at, torch.einsum("nhij,nhij->nh", ds, sd) * m)
            ds = ds * torch.where(on[:, None], a[at], 1.0)[..., None, None]
    fold = lambda x: x.view(n, hk, group, dk).sum(2)
    return (o, final, fold(dq), fold(dkk), dvv, dg, dbeta) + ((ds,) if s["state"] is not None else ())


# ---------------------------------------------------------------------------------------------- what a pass needs
def work(case):
    op = case["op"]
    if op == "sample":
        n, v = case["n"], case["v"]
        return dict(bytes=n * v * (2 if case["dtype"] == "bf16" else 4) + 12 * n, flops=8 * n * v)
    if op.startswith("block"):
        n, c, size = case["rows"], case["cols"], (2 if case["dtype"] == "bf16" else 4)
        gate, post = int(case["gate"]), int(case["post"])
        if op == "block":
            return dict(bytes=n * c * size * (4 + gate) + 4 * n * (1 + post) + 8 * c, flops=n * c * (10 + 6 * gate))
        return dict(bytes=n * c * size * (6 + 2 * gate) + 4 * n * (1 + post) + 16 * c, flops=n * c * (22 + 12 * gate))
    hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
    if op == "delta_step":
        n = case["n"]
        return dict(bytes=n * (hv * dk * dv * 8 + 2 * (2 * hk * dk + 2 * hv * dv) + 8 * hv), flops=8 * n * hv * dk * dv)
    n, states = case["n_seq"] * case["length"], 4 * case["n_seq"] * hv * dk * dv
    each = 2 * (2 * hk * dk + 2 * hv * dv) + 8 * hv
    if op == "delta":
        return dict(bytes=n * each + states * (1 + int(case["state"])), flops=8 * n * hv * dk * dv)
    # forward, then the inputs again with do in and their gradients out
    return dict(bytes=n * (each + 2 * (4 * hk * dk + 3 * hv * dv) + 16 * hv) + states * (2 + 2 * int(case["state"])),
                flops=24 * n * hv * dk * dv)
