"""Token-policy operators (layer norm, large-vocabulary cross entropy, distillation from top logits) against plain
64-bit implementations, their gradients also against differences, and what they refuse.

Tolerances come from the formats. bf16 (8 significant bits) rounded to nearest is off by at most B = 2^-8 of the value, f16 (11) by H = 2^-11,
f32 by F = 2^-24; a sum of n f32 terms taken in any order is off by at most n F' of the sum of magnitudes, F' = 2^-23
covering tensor-core accumulation, which truncates (16 products per step)."""
import math

import pytest

torch = pytest.importorskip("torch")

import pufferlean_b200 as plb  # noqa: E402
from pufferlean_b200 import tokens  # noqa: E402

pytestmark = pytest.mark.gpu

B, H, F, F2 = 2.0 ** -8, 2.0 ** -11, 2.0 ** -24, 2.0 ** -23
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


@pytest.fixture(scope="module", autouse=True)
def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.backends.cuda.matmul.allow_tf32 = False


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=F32)


def _strided(t, pad, offset=0):
    """t's values in rows of cols + pad of a larger buffer, starting `offset` elements in."""
    if not pad and not offset:
        return t.contiguous()
    buf = torch.full((t.shape[0] * (t.shape[1] + pad) + offset + pad,), float("nan"), dtype=t.dtype, device=t.device)
    v = buf[offset:offset + t.shape[0] * (t.shape[1] + pad)].view(t.shape[0], t.shape[1] + pad)[:, :t.shape[1]]
    v.copy_(t)
    return v


def _close(got, ref, tol, what):
    assert got.shape == ref.shape, what
    bad = (got.double() - ref).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((got.double() - ref).abs().max())}"


# ------------------------------------------------------------------------------------------------ layer norm
def _norm_ref(x, w, b, eps):
    x = x.double()
    m = x.mean(1)
    r = 1.0 / torch.sqrt((x - m[:, None]).square().mean(1) + eps)
    y = (x - m[:, None]) * r[:, None]
    if w is not None:
        y = y * w.double()
    if b is not None:
        y = y + b.double()
    return y, m, r


def _norm_grad_ref(dy, x, w, m, r):
    dy, m, r = dy.double(), m.double()[:, None], r.double()[:, None]
    xh = (x.double() - m) * r
    g = dy * w.double() if w is not None else dy
    dx = r * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return dx, (dy * xh).sum(0), dy.sum(0), xh, g


NORM_SHAPES = [(1, 1), (1, 8), (3, 7), (5, 256), (33, 129), (17, 1000), (2, 1003), (9, 2048), (300, 64), (1200, 520),
               (7, 4096), (6, 5003), (3, 8192), (5, 12288), (2, 16384), (3, 16385), (2, 40001)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", NORM_SHAPES)
@pytest.mark.parametrize("layout", ["plain", "padded", "odd"])
def test_layer_norm(shape, dtype, layout):
    rows, cols = shape
    g = _gen(rows * 131 + cols)
    pad, off = {"plain": (0, 0), "padded": (16, 0), "odd": (3, 1)}[layout]
    x = _strided((_randn(g, rows, cols) * 2 + 3 * _randn(g, rows, 1)).to(dtype), pad, off)
    dy = _strided(_randn(g, rows, cols).to(dtype), pad, off)
    w, b = 1 + 0.2 * _randn(g, cols), _randn(g, cols)
    if layout == "padded":
        w, b = None, (b if cols % 2 else None)
    y, m, r = tokens.layer_norm(x, w, b, 1e-5)
    yr, mr, rr = _norm_ref(x, w, b, 1e-5)
    out = B if dtype == BF16 else F
    big = x.double().abs().amax(1)
    n = math.log2(cols + 1) + 32  # additions a value passes through on its way into a sum
    tol_m = n * F2 * big
    _close(m, mr, tol_m, "mean")
    # the variance is off by n F' of itself and by (mean's error)^2 and r's error times the values
    tol_r = rr * (n * F2 + tol_m * rr * 2 + 4 * F2)
    _close(r, rr, tol_r, "rstd")
    wd = w.double().abs() if w is not None else torch.ones(cols, dtype=F64, device="cuda")
    tol = (x.double() - mr[:, None]).abs() * tol_r[:, None] * wd + (tol_m * rr)[:, None] * wd + 8 * F * (yr.abs() + wd)
    if b is not None:
        tol = tol + 2 * F * b.double().abs()
    _close(y, yr, tol + (out + F) * yr.abs() + 1e-30, "y")

    dx, dw, db = tokens.layer_norm_grad(dy, x, w, m, r)
    dxr, dwr, dbr, xh, gg = _norm_grad_ref(dy, x, w, m, r)
    rd = r.double()[:, None]
    sums = gg.abs().mean(1, keepdim=True) + xh.abs() * (gg * xh).abs().mean(1, keepdim=True)
    off_xh = F2 * (x.double().abs() + m.double()[:, None].abs()) * rd  # cancellation in x - m
    tol = rd * (n * F2 * sums * 2 + 8 * F2 * (gg.abs() + sums)
                + off_xh * (gg * xh).abs().mean(1, keepdim=True)
                + xh.abs() * (gg.abs() * off_xh).mean(1, keepdim=True)) + out * dxr.abs() + 1e-30
    _close(dx, dxr, tol, "dx")
    nr = math.sqrt(rows) + 64  # additions in a column's sum: in parts, so far fewer than its rows
    dyd = dy.double().abs()
    _close(dw, dwr, nr * F2 * (dyd * (xh.abs() + off_xh / F2)).sum(0) + 1e-30, "dw")
    _close(db, dbr, nr * F2 * dyd.sum(0) + 1e-30, "db")
    only = tokens.layer_norm_grad(dy, x, w, m, r, params=False)
    assert only[1] is None and torch.equal(only[0], dx)


def test_layer_norm_many_rows():
    """More rows than one pass of the grid holds, twice: the same bits."""
    g = _gen(5)
    x, dy = _randn(g, 20011, 96).to(BF16), _randn(g, 20011, 96).to(BF16)
    w = 1 + 0.1 * _randn(g, 96)
    y, m, r = tokens.layer_norm(x, w)
    a = tokens.layer_norm_grad(dy, x, w, m, r)
    b = tokens.layer_norm_grad(dy, x, w, m, r)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    _, dwr, dbr, xh, _ = _norm_grad_ref(dy, x, w, m, r)
    _close(a[1], dwr, 256 * F2 * (dy.double().abs() * xh.abs()).sum(0), "dw")
    _close(a[2], dbr, 256 * F2 * dy.double().abs().sum(0), "db")


def test_layer_norm_difference():
    """<dx, d> and <dw, e> against central differences of <dy, y> along exact directions (f32)."""
    g = _gen(11)
    rows, cols, h = 6, 320, 2.0 ** -7
    x = (torch.randint(-64, 65, (rows, cols), generator=g, device="cuda") / 32).to(F32)
    d = torch.randint(-1, 2, (rows, cols), generator=g, device="cuda").to(F32)
    w, e = 1 + 0.2 * _randn(g, cols), torch.randint(-1, 2, (cols,), generator=g, device="cuda").to(F32)
    dy = _randn(g, rows, cols)

    def f(xx, ww):
        return float((tokens.layer_norm(xx, ww, None)[0].double() * dy.double()).sum())

    y, m, r = tokens.layer_norm(x, w, None)
    dx, dw, _ = tokens.layer_norm_grad(dy, x, w, m, r)
    scale = float((dy.double().abs() * (y.double().abs() + 1)).sum())
    # rounding of f over 2 h, and h^2 of the third derivative (of order |d|^3 |dy| r^3, r about 1)
    tol = 8 * F2 * scale / h + 40 * h * h * float(dy.abs().sum())
    assert abs((f(x + h * d, w) - f(x - h * d, w)) / (2 * h) - float((dx.double() * d).sum())) < tol
    assert abs((f(x, w + h * e) - f(x, w - h * e)) / (2 * h) - float((dw.double() * e).sum())) < tol


def test_layer_norm_no_rows():
    x = torch.empty(0, 24, device="cuda")
    y, m, r = tokens.layer_norm(x)
    assert y.shape == (0, 24) and m.shape == (0,)
    dx, dw, db = tokens.layer_norm_grad(x, x, None, m, r)
    assert dx.shape == (0, 24) and not dw.any() and not db.any()


def test_layer_norm_constant_rows():
    """A constant row has variance zero: y = bias, a finite gradient."""
    x = torch.full((3, 72), 7.0, device="cuda", dtype=BF16)
    b = torch.arange(72, device="cuda", dtype=F32)
    y, m, r = tokens.layer_norm(x, None, b, 1e-5)
    assert torch.equal(y, b.to(BF16).expand(3, 72))
    dx, dw, db = tokens.layer_norm_grad(torch.ones_like(x), x, None, m, r)
    assert torch.isfinite(dx.float()).all() and not dw.any()


# ------------------------------------------------------------------------------------------------ the head
def _head_case(g, N, V, D, K, bias, pad, off, spread=2.0, left_out=0.25):
    x = _randn(g, N, D)
    w = _randn(g, V, D) * (spread / math.sqrt(D))
    w = _strided(w.to(BF16), pad, off)
    b = (0.5 * _randn(g, V)).to(BF16) if bias else None
    scale = _randn(g, N)
    if K == 0:
        t = torch.randint(0, V, (N,), generator=g, device="cuda")
        x = x + 2 * torch.rand(N, 1, generator=g, device="cuda") * w[t].float()
        drop = torch.rand(N, generator=g, device="cuda") < left_out
        ids, teacher = torch.where(drop, -1 - t, t).to(torch.int32), None
    else:
        ids = torch.randint(0, V, (N, K), generator=g, device="cuda")  # repeated ids occur
        drop = torch.rand(N, K, generator=g, device="cuda") < left_out
        drop |= torch.rand(N, 1, generator=g, device="cuda") < left_out / 2
        ids = torch.where(drop, -1, ids).to(torch.int32)
        teacher = 2 * _randn(g, N, K)
        teacher[torch.rand(N, K, generator=g, device="cuda") < 0.05] = -math.inf
    return _strided(x.to(BF16), pad, off), w, b, ids, teacher, scale


def _answers(ids, teacher, V, T):
    """The dense [N, V] answer distribution, its negative entropy per row, and which rows have one (64 bits)."""
    if teacher is None:
        has = ids >= 0
        p = has.double()[:, None]
        at = ids.long().clamp(min=0)[:, None]
        ent = torch.zeros(len(ids), dtype=F64, device="cuda")
    else:
        here = (ids >= 0) & (teacher > -math.inf)
        has = here.any(1)
        t = torch.where(here, teacher.double() / T, -math.inf)
        p = torch.softmax(torch.where(has[:, None], t, 0.0), 1) * has[:, None]
        at = ids.long().clamp(min=0)
        ent = torch.xlogy(p, p).sum(1)
    want = torch.zeros(ids.shape[0], V, dtype=F64, device="cuda").scatter_add_(1, at, p)
    return want, ent, has


def _head_ref(x, w, b, ids, teacher, T, scale):
    xd, wd = x.double(), w.double()
    u = xd @ wd.t()
    if b is not None:
        u = u + b.double()
    u = u / T
    want, ent, has = _answers(ids, teacher, w.shape[0], T)
    lse = torch.logsumexp(u, 1)
    hit = torch.where(want > 0, want * u, 0.0).sum(1)
    loss = torch.where(has, ent - hit + lse, 0.0)
    q = torch.exp(u - lse[:, None])
    s = torch.where(has, scale.double() / T, 0.0)[:, None]
    dz = torch.where(has[:, None], s * (q - want), 0.0)
    return dict(u=u, lse=torch.where(has, lse, 0.0), loss=loss, dz=dz, q=q, s=s, has=has)


def _head_tol(ref, x, w, b, ids, T):
    """Largest error of a row's logits, and of its loss: D / 16 truncating steps and 32 more additions, the two
    roundings of the scaled sum, 2^-21 for the exponentials and the logarithm of the sum."""
    xa = torch.where(ref["has"][:, None], x.double().abs(), 0.0)
    mag = (xa @ w.double().abs().t()).amax(1) / T
    if b is not None:
        finite = torch.where(torch.isfinite(b.float()), b.double().abs(), 0.0).clamp(max=1e6)
        mag = mag + finite.max() / T
    z = (x.shape[1] / 16 + 32) * F2 * mag
    return z, 2 * z + 2.0 ** -20 * (1 + ref["lse"].abs() + ref["loss"].abs())


def _check_head(x, w, b, ids, teacher, T, scale, dw_f32=False, piece_bytes=0):
    N, D = x.shape
    ref = _head_ref(x, w, b, ids, teacher, T, scale)
    tol_z, tol_loss = _head_tol(ref, x, w, b, ids, T)
    if teacher is None:
        fwd = tokens.vocab_ce(x, w, ids, b)
        got = tokens.vocab_ce_grad(x, w, ids, b, scale, dw_f32, piece_bytes)
    else:
        fwd = tokens.vocab_distill(x, w, ids, teacher, b, T)
        got = tokens.vocab_distill_grad(x, w, ids, teacher, b, T, scale, dw_f32, piece_bytes)
    for loss, lse in (fwd, got[:2]):
        _close(loss, ref["loss"], tol_loss, "loss")
        _close(lse, ref["lse"], tol_loss, "lse")
        assert not loss[~ref["has"]].any() and not lse[~ref["has"]].any()
    _, _, dx, dw, db = got
    # dz: one rounding to bf16 (B), the f16 term (H), the logits' error on both sides of the softmax; terms below
    # 2^-40 of their segment's largest are flushed
    off = (B + H) * ref["dz"].abs() + (H + 4 * tol_z[:, None] + 2.0 ** -18) * (ref["s"].abs() * ref["q"]) \
        + 2.0 ** -18 * ref["dz"].abs()
    off = torch.where(ref["has"][:, None], off + 2.0 ** -40 * ref["s"].abs(), 0.0)
    wa, xa = w.double().abs(), torch.where(ref["has"][:, None], x.double(), 0.0).abs()
    steps = lambda n: (n / 16 + 200) * F2  # noqa: E731
    V = w.shape[0]
    dxr = ref["dz"] @ w.double()
    _close(dx, dxr, off @ wa + steps(V) * (ref["dz"].abs() @ wa) + B * 1.01 * dxr.abs() + 1e-30, "dx")
    xd = torch.where(ref["has"][:, None], x.double(), 0.0)
    dwr = ref["dz"].t() @ xd
    out = F if dw_f32 else B
    assert dw.dtype == (F32 if dw_f32 else BF16)
    _close(dw, dwr, off.t() @ xa + steps(N) * (ref["dz"].abs().t() @ xa) + out * 1.01 * dwr.abs() + 1e-30, "dw")
    if b is not None:
        dbr = ref["dz"].sum(0)
        _close(db, dbr, off.sum(0) + steps(16 * N) * ref["dz"].abs().sum(0) + out * 1.01 * dbr.abs() + 1e-30, "dbias")
    else:
        assert db is None
    return got


HEAD_SHAPES = [(1, 1, 1), (1, 130, 64), (2, 65, 33), (16, 1024, 256), (63, 257, 8), (64, 128, 72), (65, 300, 513),
               (127, 2000, 40), (128, 129, 128), (129, 700, 264), (200, 5003, 100), (300, 64, 1000), (1000, 777, 136),
               (4200, 130, 48), (31, 40000, 64), (150, 20001, 96)]


@pytest.mark.parametrize("shape", HEAD_SHAPES)
@pytest.mark.parametrize("bias,layout", [(True, "plain"), (False, "padded"), (True, "odd")])
def test_vocab_ce(shape, bias, layout):
    N, V, D = shape
    pad, off = {"plain": (0, 0), "padded": (8, 8), "odd": (5, 3)}[layout]
    x, w, b, ids, _, scale = _head_case(_gen(N + 7 * V + 31 * D), N, V, D, 0, bias, pad, off)
    _check_head(x, w, b, ids, None, 1.0, scale, dw_f32=layout == "padded")


@pytest.mark.parametrize("shape", HEAD_SHAPES)
@pytest.mark.parametrize("K,T,bias", [(1, 1.0, False), (5, 2.0, True), (70, 0.7, False)])
def test_vocab_distill(shape, K, T, bias):
    N, V, D = shape
    x, w, b, ids, teacher, scale = _head_case(_gen(N + 3 * V + 11 * D + K), N, V, D, K, bias, 0, 0)
    _check_head(x, w, b, ids, teacher, T, scale, dw_f32=K == 5)


@pytest.mark.parametrize("dw_f32", [False, True])
@pytest.mark.parametrize("N,V,D", [(700, 3001, 200), (515, 400, 72), (1025, 25000, 264)])
def test_vocab_pieces(N, V, D, dw_f32):
    """Several pieces of rows (the smallest: 128 each): the losses' bits and dx's do not change; rows without an
    answer leave some pieces short or empty."""
    x, w, b, ids, _, scale = _head_case(_gen(N), N, V, D, 0, True, 0, 0, left_out=0.45)
    many = _check_head(x, w, b, ids, None, 1.0, scale, dw_f32, piece_bytes=1)
    one = _check_head(x, w, b, ids, None, 1.0, scale, dw_f32)
    assert torch.equal(many[0], one[0]) and torch.equal(many[1], one[1])


@pytest.mark.parametrize("N", [5, 128, 129, 400])
def test_vocab_no_row_counts(N):
    x, w, b, ids, _, scale = _head_case(_gen(N), N, 300, 64, 0, True, 0, 0)
    ids = torch.full_like(ids, -1)
    loss, lse, dx, dw, db = tokens.vocab_ce_grad(x, w, ids, b, scale)
    assert not any(t.any() for t in (loss, lse, dx, dw, db))
    teacher = torch.full((N, 3), -math.inf, device="cuda")
    out = tokens.vocab_distill_grad(x, w, torch.zeros(N, 3, dtype=torch.int32, device="cuda"), teacher, b)
    assert not any(t.any() for t in out)


def test_vocab_no_rows():
    w = torch.ones(40, 16, dtype=BF16, device="cuda")
    x, t = torch.empty(0, 16, dtype=BF16, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda")
    loss, lse, dx, dw, db = tokens.vocab_ce_grad(x, w, t, torch.zeros(40, dtype=BF16, device="cuda"))
    assert loss.shape == (0,) and dx.shape == (0, 16) and not dw.any() and not db.any()


@pytest.mark.parametrize("N", [9, 260])
def test_vocab_left_out_rows_hold_anything(N):
    """NaN and infinities in the hidden states of rows that do not count reach nothing."""
    x, w, b, ids, _, scale = _head_case(_gen(N), N, 500, 96, 0, True, 0, 0, left_out=0.4)
    clean = tokens.vocab_ce_grad(x, w, ids, b, scale)
    x = x.clone()
    x[(ids < 0).nonzero()[:, 0], ::3] = float("nan")
    x[(ids < 0).nonzero()[:, 0], 1::3] = float("inf")
    scale = torch.where(ids < 0, float("nan"), scale)
    dirty = tokens.vocab_ce_grad(x, w, ids, b, scale)
    for c, d in zip(clean, dirty):
        assert torch.equal(c, d)


@pytest.mark.parametrize("value", [-math.inf, torch.finfo(BF16).min])
@pytest.mark.parametrize("N", [20, 300])
def test_vocab_masked_vocabulary(N, value):
    """A bias of -inf, or of the type's lowest value, takes tokens (whole tiles of them) out of the softmax."""
    x, w, b, ids, _, scale = _head_case(_gen(N), N, 1500, 64, 0, True, 0, 0)
    b[200:1100] = value
    b[1499] = value
    ids = torch.where((ids >= 200) & (ids < 1100) | (ids == 1499), 7, ids)
    loss, lse, dx, dw, db = _check_head(x, w, b, ids, None, 1.0, scale)
    assert not dw[200:1100].any() and not db[200:1100].any()


def test_vocab_wide_logits():
    """Logits spread over hundreds (a confident, badly scaled head): sure answers and hopeless ones."""
    x, w, b, ids, _, scale = _head_case(_gen(3), 200, 900, 128, 0, False, 0, 0, spread=60.0)
    _check_head(x, w, b, ids, None, 1.0, scale)


def test_vocab_sure_answer():
    """A target at probability 1 - 1e-5: its gradient is small and still right to bf16."""
    g = _gen(4)
    w = _randn(g, 400, 64).to(BF16)
    t = torch.randint(0, 400, (50,), generator=g, device="cuda").to(torch.int32)
    x = (0.33 * w[t.long()].float()).to(BF16)
    _check_head(x, w, None, t, None, 1.0, torch.ones(50, device="cuda"))


def test_vocab_repeated_ids_add_up():
    g = _gen(6)
    x, w = _randn(g, 4, 64).to(BF16), _randn(g, 100, 64).to(BF16)
    ids = torch.tensor([[5, 5, 9], [9, 5, 9], [5, -1, 5], [9, 9, 9]], dtype=torch.int32, device="cuda")
    _check_head(x, w, None, ids, _randn(g, 4, 3), 1.0, torch.ones(4, device="cuda"))


@pytest.mark.parametrize("N", [6, 200])
def test_vocab_index_past_the_vocabulary(N):
    """Seen in the row's loss (NaN); no other row's loss is touched, nothing is read out of range."""
    x, w, b, ids, _, scale = _head_case(_gen(N), N, 70, 64, 0, False, 0, 0, left_out=0.0)
    good = tokens.vocab_ce(x, w, ids)[0]
    bad = ids.clone()
    bad[3] = 70
    loss = tokens.vocab_ce(x, w, bad)[0]
    assert torch.isnan(loss[3])
    keep = torch.arange(N, device="cuda") != 3
    assert torch.equal(loss[keep], good[keep])
    assert torch.isnan(tokens.vocab_ce_grad(x, w, bad)[2][3].float()).all()
    k = torch.stack([ids, bad], 1).contiguous()
    assert torch.isnan(tokens.vocab_distill(x, w, k, torch.zeros(N, 2, device="cuda"))[0][3])


def test_vocab_nan_is_seen():
    """NaN in a row that counts: that row's loss, not the others'."""
    x, w, b, ids, _, scale = _head_case(_gen(8), 140, 300, 64, 0, False, 0, 0, left_out=0.0)
    good = tokens.vocab_ce(x, w, ids)[0]
    x = x.clone()
    x[77, 5] = float("nan")
    loss = tokens.vocab_ce(x, w, ids)[0]
    assert torch.isnan(loss[77]) and int(torch.isnan(loss).sum()) == 1
    keep = torch.arange(140, device="cuda") != 77
    assert torch.equal(loss[keep], good[keep])


@pytest.mark.parametrize("distill", [False, True])
def test_vocab_difference(distill):
    """<dx, d>, <dW, e>, <dbias, f> against central differences of the summed loss, along directions that bf16
    holds exactly."""
    g = _gen(21)
    N, V, D, h = 160, 333, 48, 2.0 ** -5
    grid = lambda *s: (torch.randint(-24, 25, s, generator=g, device="cuda") / 16).to(BF16)  # noqa: E731
    sign = lambda *s: torch.randint(-1, 2, s, generator=g, device="cuda").float()  # noqa: E731
    x, w, b = grid(N, D), (grid(V, D).float() / 8).to(BF16), grid(V)
    scale = torch.rand(N, generator=g, device="cuda") + 0.5
    T = 2.0 if distill else 1.0
    ids = torch.randint(0, V, (N, 4) if distill else (N,), generator=g, device="cuda").to(torch.int32)
    teacher = _randn(g, N, 4) if distill else None

    def f(dx=0, dw=0, db=0):
        xx, ww, bb = (x.float() + dx).to(BF16), (w.float() + dw).to(BF16), (b.float() + db).to(BF16)
        assert torch.equal(xx.float(), x.float() + dx) and torch.equal(ww.float(), w.float() + dw)
        assert torch.equal(bb.float(), b.float() + db)
        loss = tokens.vocab_distill(xx, ww, ids, teacher, bb, T)[0] if distill else tokens.vocab_ce(xx, ww, ids, bb)[0]
        return float((loss.double() * scale.double()).sum())

    if distill:
        _, _, dx, dw, db = tokens.vocab_distill_grad(x, w, ids, teacher, b, T, scale)
    else:
        _, _, dx, dw, db = tokens.vocab_ce_grad(x, w, ids, b, scale)
    ref = _head_ref(x, w, b, ids, teacher, T, scale)
    size = float(scale.sum()) * 10
    for name, grad, step, reach in (("dx", dx, sign(N, D), w.double().abs().sum(1).max()),
                                    ("dw", dw, sign(V, D) / 8, x.double().abs().sum(1).max() / 8),
                                    ("db", db, sign(V), torch.tensor(1.0))):
        move = h * step
        num = (f(**{name: move}) - f(**{name: -move})) / (2 * h)
        got = float((grad.double() * step.double()).sum())
        # the third derivative of log-sum-exp along a step that moves the logits by c h is at most c^3; the
        # logits here move by far less than `reach` (signs cancel), c = 4 sqrt(D) typical steps covers them
        c = 4 * math.sqrt(D) * (1.0 if name == "db" else 0.25)
        c = 2.0 if name == "db" else c
        tol = size / 10 * c ** 3 * h * h / 6 + 2.0 ** -18 * size / h + 2 * B * float(ref["dz"].abs().sum()) * c
        assert abs(num - got) < tol, (name, num, got, tol)


def test_vocab_other_stream():
    """Calls on two streams at once, each with its own workspace, give the bits of one stream's."""
    a = _head_case(_gen(1), 300, 4000, 128, 0, True, 0, 0)
    c = _head_case(_gen(2), 500, 3000, 64, 0, True, 0, 0)
    want = [tokens.vocab_ce_grad(q[0], q[1], q[3], q[2], q[5]) for q in (a, c)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(5):
        for i, q in enumerate((a, c)):
            with torch.cuda.stream(streams[i]):
                got[i] = tokens.vocab_ce_grad(q[0], q[1], q[3], q[2], q[5])
    torch.cuda.synchronize()
    for p, q in zip(want, got):
        assert all(torch.equal(s, t) for s, t in zip(p, q))


def test_vocab_repeats_bit_for_bit():
    x, w, b, ids, teacher, scale = _head_case(_gen(9), 900, 6000, 200, 6, True, 0, 0)
    one = tokens.vocab_distill_grad(x, w, ids, teacher, b, 1.5, scale)
    for _ in range(3):
        two = tokens.vocab_distill_grad(x, w, ids, teacher, b, 1.5, scale)
        assert all(torch.equal(s, t) for s, t in zip(one, two))


def test_launches_are_the_librarys():
    n0 = plb.kernel_launch_count()
    x, w, b, ids, _, scale = _head_case(_gen(9), 40, 600, 64, 0, False, 0, 0)
    tokens.vocab_ce(x, w, ids)
    assert plb.kernel_launch_count() > n0


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    x = torch.zeros(4, 16, dtype=BF16, device="cuda")
    w = torch.zeros(9, 16, dtype=BF16, device="cuda")
    t = torch.zeros(4, dtype=torch.int32, device="cuda")
    k = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    f = torch.zeros(4, 2, device="cuda")
    for call in (
        lambda: tokens.vocab_ce(x.float(), w, t),
        lambda: tokens.vocab_ce(x, w.float(), t),
        lambda: tokens.vocab_ce(x, w[:, :8], t),
        lambda: tokens.vocab_ce(x, w, t.long()),
        lambda: tokens.vocab_ce(x, w, t[:3]),
        lambda: tokens.vocab_ce(x.cpu(), w, t),
        lambda: tokens.vocab_ce(x, w.cpu(), t),
        lambda: tokens.vocab_ce(x.t(), w, t),
        lambda: tokens.vocab_ce(x[0], w, t),
        lambda: tokens.vocab_ce(x, w, t, torch.zeros(9, device="cuda")),
        lambda: tokens.vocab_ce(x, w, None),
        lambda: tokens.vocab_ce_grad(x, w, t, None, torch.zeros(3, device="cuda")),
        lambda: tokens.vocab_ce(x, w[:0], t),
        lambda: tokens.vocab_distill(x, w, k, None),
        lambda: tokens.vocab_distill(x, w, k, f.half()),
        lambda: tokens.vocab_distill(x, w, k, f[:, :1]),
        lambda: tokens.vocab_distill(x, w, k[:, :0], f[:, :0]),
        lambda: tokens.vocab_distill(x, w, t, f),
        lambda: tokens.vocab_distill(x, w, k, f, None, 0.0),
        lambda: tokens.vocab_distill(x, w, k, f, None, float("nan")),
        lambda: tokens.layer_norm(x.half()),
        lambda: tokens.layer_norm(x, torch.zeros(16, dtype=BF16, device="cuda")),
        lambda: tokens.layer_norm(x, None, torch.zeros(15, device="cuda")),
        lambda: tokens.layer_norm(x, None, None, -1.0),
        lambda: tokens.layer_norm(x[:, :0]),
        lambda: tokens.layer_norm_grad(x.float(), x, None, f[:, 0].contiguous(), f[:, 1].contiguous()),
        lambda: tokens.layer_norm_grad(x, x, None, None, None),
        lambda: tokens.layer_norm_grad(x, x, None, f[:, 0], f[:, 1]),
    ):
        with pytest.raises(plb.PufferError):
            call()


def test_c_entries_refuse():
    """The C entries check sizes, strides and workspaces on the host and launch nothing."""
    L = plb.lib()
    x = torch.zeros(4, 16, dtype=BF16, device="cuda")
    w = torch.zeros(9, 16, dtype=BF16, device="cuda")
    t = torch.zeros(4, dtype=torch.int32, device="cuda")
    o = torch.zeros(8, device="cuda")
    ws = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    n0 = plb.kernel_launch_count()
    a = (x.data_ptr(), 16, w.data_ptr(), 16, None, t.data_ptr())
    tail = (o.data_ptr(), o.data_ptr() + 16)
    big = (ws.data_ptr(), 1 << 20, None)
    assert L.pl_vocab_ce_dev(*a, 4, 9, 16, *tail, ws.data_ptr(), 8, None) == -1  # workspace too small
    assert b"workspace" in L.pl_last_error()
    assert L.pl_vocab_ce_dev(*a, 4, 9, 16, *tail, ws.data_ptr() + 4, (1 << 20) - 4, None) == -1  # its alignment
    assert L.pl_vocab_ce_dev(*a, 4, 9, 17, *tail, *big) == -1  # stride below the width
    assert L.pl_vocab_ce_dev(*a, 4, 0, 16, *tail, *big) == -1
    assert L.pl_vocab_ce_dev(*a[:5], None, 4, 9, 16, *tail, *big) == -1
    assert L.pl_vocab_distill_dev(*a, None, 2, 1.0, 4, 9, 16, *tail, *big) == -1
    assert L.pl_vocab_ce_dev(*a, 1 << 31, 9, 16, *tail, *big) == -1
    assert L.pl_layernorm_dev(x.data_ptr(), 8, None, None, 4, 16, 1e-5, 1, x.data_ptr(), 16, *tail, None) == -1
    assert L.pl_layernorm_grad_dev(x.data_ptr(), 16, x.data_ptr(), 16, None, *tail, 4, 16, 1, x.data_ptr(), 16,
                                   o.data_ptr(), None, ws.data_ptr(), 4, None) == -1
    assert plb.kernel_launch_count() == n0


def test_calls_can_be_captured():
    """The calls enqueue and return: a training step's operators replay from a CUDA graph with the same bits."""
    x, w, b, ids, _, scale = _head_case(_gen(12), 300, 2000, 128, 0, True, 0, 0)
    gain = 1 + 0.1 * _randn(_gen(13), 128)

    def step():
        y, m, r = tokens.layer_norm(x, gain)
        loss, lse, dy, dw, db = tokens.vocab_ce_grad(y, w, ids, b, scale)
        return (y, loss, lse, dw, db) + tokens.layer_norm_grad(dy, x, gain, m, r)

    want = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for t in got:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for p, q in zip(want, got):
        assert torch.equal(p, q)


def test_example_learns():
    """examples/token_policy.py at a small size: the cross entropy falls by a nat at least towards the demonstrations'
    entropy, the divergence from the teacher by a tenth of itself."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "token_policy.py")
    spec = importlib.util.spec_from_file_location("token_policy", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    first, last, dfirst, dlast = mod.train(vocab=1024, width=128, batch=2048, steps=40, say=lambda *_: None)
    assert last < first - 1.0 and dlast < 0.9 * dfirst, (first, last, dfirst, dlast)


@pytest.mark.parametrize("D", [1024, 4096])
def test_vocab_lse_is_unbiased(D):
    """Logits that lean towards their weight row lose on average nothing to the accumulator's truncation: the slope of
    the error over 8,192 rows stays below 2^-21 (D 2^-30 without the correction: 2^-20 and 2^-18)."""
    g = _gen(D)
    w = (_randn(g, 1, D) * (1.5 / math.sqrt(D)))
    x = (_randn(g, 8192, D) + 4 * torch.rand(8192, 1, generator=g, device="cuda") * w).to(BF16)
    w = w.to(BF16)
    lse = tokens.vocab_ce(x, w, torch.zeros(8192, dtype=torch.int32, device="cuda"))[1].double()
    z = (x.double() @ w.double().t())[:, 0]
    assert abs(float(((lse - z) * z).sum() / (z * z).sum())) < 2.0 ** -21


@pytest.mark.parametrize("N", [1, 5, 33, 64])
@pytest.mark.parametrize("K", [0, 4])
def test_vocab_few_rows_round_once(N, K):
    """Up to 64 rows the gradients carry dz in two parts: what is left is their own rounding to bf16 and the f16 terms'
    (H of each probability's share)."""
    x, w, b, ids, teacher, scale = _head_case(_gen(40 + N), N, 900, 128, K, True, 0, 0, left_out=0.0)
    T = 1.5 if K else 1.0
    ref = _head_ref(x, w, b, ids, teacher, T, scale)
    tol_z, _ = _head_tol(ref, x, w, b, ids, T)
    if K:
        _, _, dx, dw, _ = tokens.vocab_distill_grad(x, w, ids, teacher, b, T, scale)
    else:
        _, _, dx, dw, _ = tokens.vocab_ce_grad(x, w, ids, b, scale)
    off = 2 * B * B * ref["dz"].abs() + (H + 4 * tol_z[:, None] + 2.0 ** -18) * (ref["s"].abs() * ref["q"]) \
        + 2.0 ** -18 * ref["dz"].abs() + 2.0 ** -40
    off = torch.where(ref["has"][:, None], off, 0.0)
    dxr = ref["dz"] @ w.double()
    _close(dx, dxr, off @ w.double().abs() + 1e-4 * B * (ref["dz"].abs() @ w.double().abs()) + B * 1.01 * dxr.abs(), "dx")
    dwr = ref["dz"].t() @ x.double()
    _close(dw, dwr, off.t() @ x.double().abs() + 1e-4 * B * (ref["dz"].abs().t() @ x.double().abs())
           + B * 1.01 * dwr.abs(), "dw")


@pytest.mark.parametrize("N,V,D,K", [(40, 70, 32, 512), (300, 600, 64, 300), (9, 3000, 200, 128)])
def test_vocab_distill_long_lists(N, V, D, K):
    """As many entries as a row may have, and lists that name most of the vocabulary, some of it many times."""
    x, w, b, ids, teacher, scale = _head_case(_gen(K), N, V, D, K, True, 0, 0)
    _check_head(x, w, b, ids, teacher, 1.0, scale)


def test_vocab_wide_rows():
    x, w, b, ids, _, scale = _head_case(_gen(77), 140, 500, 9001, 0, True, 3, 1)
    _check_head(x, w, b, ids, None, 1.0, scale)


def test_vocab_past_32_bits():
    """Terms beyond 2^31 elements, in two pieces: rows at both ends against 64 bits, and the weight gradient of a few
    tokens summed over all rows."""
    g = _gen(99)
    N, V, D = 16500, 131100, 64
    x, w = _randn(g, N, D).to(BF16), (_randn(g, V, D) * 0.2).to(BF16)
    t = torch.randint(0, V, (N,), generator=g, device="cuda").to(torch.int32)
    t[-3] = V - 1
    t[5] = 0
    loss, lse, dx, dw, _ = tokens.vocab_ce_grad(x, w, t)
    rows = torch.tensor([0, 5, 8191, 8192, 12345, N - 3, N - 1], device="cuda")
    ones = torch.ones(len(rows), device="cuda")
    xs, ts = x[rows], t[rows]
    ref = _head_ref(xs, w, None, ts, None, 1.0, ones)
    tol_z, tol_loss = _head_tol(ref, xs, w, None, ts, 1.0)
    _close(loss[rows], ref["loss"], tol_loss, "loss")
    _close(lse[rows], ref["lse"], tol_loss, "lse")
    off = (B + H) * ref["dz"].abs() + (H + 4 * tol_z[:, None] + 2.0 ** -18) * ref["q"] + 2.0 ** -18 * ref["dz"].abs()
    wa = w.double().abs()
    dxr = ref["dz"] @ w.double()
    _close(dx[rows], dxr, off @ wa + (V / 16 + 200) * F2 * (ref["dz"].abs() @ wa) + B * 1.01 * dxr.abs(), "dx")
    cols = torch.tensor([0, 1, 77777, V - 1], device="cuda")
    q = torch.exp(x.double() @ w[cols].double().t() - lse.double()[:, None])
    dz = q - (t[:, None] == cols[None]).double()
    dwr = dz.t() @ x.double()
    xa = x.double().abs()
    off = (B + H) * dz.abs() + (H + 2.0 ** -16) * q
    _close(dw[cols], dwr, off.t() @ xa + (N / 16 + 200) * F2 * (dz.abs().t() @ xa) + B * 1.01 * dwr.abs(), "dw")


def test_layer_norm_past_32_bits():
    rows, cols = 140000, 16384
    x = torch.empty(rows, cols, dtype=BF16, device="cuda")
    x.normal_(generator=_gen(3))
    y, m, r = tokens.layer_norm(x)
    at = torch.tensor([0, 1, 131071, 131072, rows - 1], device="cuda")
    yr, mr, rr = _norm_ref(x[at], None, None, 1e-5)
    _close(m[at], mr, torch.full_like(mr, 64 * F2 * 6), "mean")
    _close(y[at], yr, (B + 2.0 ** -16) * yr.abs() + 2.0 ** -16, "y")
    dx, dw, db = tokens.layer_norm_grad(y, x, None, m, r)
    dxr, _, _, xh, gg = _norm_grad_ref(y[at], x[at], None, m[at], r[at])
    _close(dx[at], dxr, B * dxr.abs() + 2.0 ** -16 * (1 + xh.abs()) * (1 + gg.abs()), "dx")
    assert torch.isfinite(dw).all() and torch.isfinite(db).all()
