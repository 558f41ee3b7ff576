"""The norms around a block with its gate and residual scale, forward and backward, against plain 64-bit implementations.

Tolerances: a bf16 result rounded to nearest is off by at most B = 2^-8 of its value, f32 by F = 2^-24. A sum of n f32 terms
is off by at most its depth times F2 = 2^-23 of the sum of magnitudes; the gate's exponential by 2^-21 + |gate| 2^-23 of its
value (its argument is rounded once)."""
import math

import pytest

torch = pytest.importorskip("torch")

import pufferlean_b200 as plb  # noqa: E402
from pufferlean_b200 import tokens  # noqa: E402

pytestmark = pytest.mark.gpu
B, F, F2 = 2.0 ** -8, 2.0 ** -24, 2.0 ** -23
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


@pytest.fixture(scope="module", autouse=True)
def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _strided(t, pad, offset):
    buf = torch.full((t.shape[0] * (t.shape[1] + pad) + offset + pad + 8,), float("nan"), dtype=t.dtype, device="cuda")
    v = buf[offset:offset + t.shape[0] * (t.shape[1] + pad)].view(t.shape[0], t.shape[1] + pad)[:, :t.shape[1]]
    v.copy_(t)
    return v


def _close(got, ref, tol, what):
    assert got.shape == ref.shape, what
    off = (got.double() - ref).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(off.max())}"


def _inputs(rows, cols, dtype, gate, pad, offset, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    m = lambda t: _strided(t.to(dtype), pad, offset)
    x, branch = m(r(rows, cols) * 2), m(r(rows, cols) + 0.3)
    ga = m(3 * r(rows, cols)) if gate else None
    return x, branch, ga, 1 + 0.2 * r(cols), 1 + 0.2 * r(cols), m(r(rows, cols)), m(r(rows, cols))


def _forward(x, branch, gate, w1, w2, scale, eps, post, r_stored=None):
    b = branch.double()
    rb = 1 / torch.sqrt(b.square().mean(1) + eps) if post else None
    n = b * (rb[:, None] if post else 1.0)
    if w1 is not None:
        n = n * w1.double()
    a = torch.sigmoid(gate.double()) if gate is not None else torch.ones_like(n)
    add = scale * a * n
    r = x.double() + add
    s = r if r_stored is None else r_stored.double()
    rr = 1 / torch.sqrt(s.square().mean(1) + eps)
    y = s * rr[:, None]
    return r, (y * w2.double() if w2 is not None else y), rb, rr, add


def _backward(dr, dy, branch, gate, r, rb, rr, w1, w2, scale):
    w1 = w1.double() if w1 is not None else torch.ones(r.shape[1], dtype=F64, device="cuda")
    w2 = w2.double() if w2 is not None else torch.ones_like(w1)
    dy, r, b, rr = dy.double(), r.double(), branch.double(), rr.double()[:, None]
    rh = r * rr
    g = dy * w2
    d = rr * (g - rh * (g * rh).mean(1, keepdim=True))
    if dr is not None:
        d = d + dr.double()
    bh = b if rb is None else b * rb.double()[:, None]
    a = torch.sigmoid(gate.double()) if gate is not None else torch.ones_like(d)
    na = torch.sigmoid(-gate.double()) if gate is not None else None
    t = scale * d * a * w1
    db = t if rb is None else rb.double()[:, None] * (t - bh * (t * bh).mean(1, keepdim=True))
    return d, db, (None if gate is None else t * na * bh), (scale * d * a * bh), dy * rh, t, bh, g, rh


SHAPES = [(1, 1), (1, 8), (3, 7), (5, 256), (33, 129), (17, 1000), (2, 1003), (9, 2048), (300, 64), (1200, 520), (7, 4096),
          (6, 5003), (3, 8192), (5, 12288), (2, 16384), (3, 16385), (2, 40001)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("layout", ["plain", "padded", "odd"])
def test_block(shape, dtype, layout):
    rows, cols = shape
    pad, offset = {"plain": (0, 0), "padded": (16, 8), "odd": (3, 1)}[layout]
    eps, scale, out = 1e-5, (0.5 if cols % 2 else -1.25), (B if dtype == BF16 else F)
    for gate, post in ((True, True), (False, True), (True, False), (False, False)):
        x, branch, ga, w1, w2, dr, dy = _inputs(rows, cols, dtype, gate, pad, offset, rows * 131 + cols)
        if layout == "padded":
            w1, w2 = (None, w2) if post else (w1, None)
        r, y, rb, rr = tokens.block_norm(x, branch, ga, w1, w2, scale, eps, post)
        rref, yref, rbref, rrref, add = _forward(x, branch, ga, w1, w2, scale, eps, post, r)
        assert r.dtype == y.dtype == dtype and (rb is None) == (not post)
        n = math.log2(cols + 1) + 64  # additions a value passes through on its way into a sum
        if post:
            _close(rb, rbref, (n * F2 + 4 * F2) * rbref, "rstd_branch")
        ex = 0.0 if ga is None else 2.0 ** -21 + ga.double().abs() * F2
        tol_add = add.abs() * (n * F2 + 12 * F2 + ex)
        _close(r, rref, tol_add + (out + 2 * F) * (rref.abs() + tol_add) + 1e-30, "r")
        _close(rr, rrref, (n * F2 + 4 * F2) * rrref, "rstd")
        _close(y, yref, yref.abs() * (n * F2 + 8 * F2 + out), "y")

        some_dr = dr if cols % 3 else None
        got = tokens.block_norm_grad(some_dr, dy, branch, ga, r, rb, rr, w1, w2, scale)
        d, db, dg, dw1, dw2, t, bh, g, rh = _backward(some_dr, dy, branch, ga, r, rb, rr, w1, w2, scale)
        rd = rr.double()[:, None]
        along = (g * rh).abs().mean(1, keepdim=True)
        tol_d = (n + 8) * F2 * (rd * (g.abs() + rh.abs() * along) + (0 if some_dr is None else dr.double().abs()))
        _close(got[0], d, tol_d + out * (d.abs() + tol_d) + 1e-30, "dx")
        f = t.abs() / d.abs().clamp(min=1e-300)  # what t multiplies d with
        tol_t = f * tol_d + t.abs() * (8 * F2 + ex)
        if gate:
            h = torch.sigmoid(-ga.double()) * bh.abs()
            _close(got[2], dg, h * tol_t + dg.abs() * (8 * F2 + ex + out) + out * h * tol_t + 1e-30, "dgate")
        else:
            assert got[2] is None
        tol = tol_t
        if post:
            tol = rb.double()[:, None] * (tol_t + bh.abs() * (tol_t * bh.abs()).mean(1, keepdim=True)
                                          + (n + 8) * F2 * (t.abs() + bh.abs() * (t * bh).abs().mean(1, keepdim=True)))
        _close(got[1], db, tol + out * (db.abs() + tol) + 4 * F2 * db.abs() + 1e-30, "dbranch")
        nr = math.sqrt(rows) + 64  # additions in a column's sum: in parts, so far fewer than its rows
        w = w1.double().abs().clamp(min=1e-30) if w1 is not None else 1.0
        _close(got[3], dw1.sum(0), (nr * F2 * dw1.abs() + tol_t * bh.abs() / w + 8 * F2 * dw1.abs()).sum(0) + 1e-30, "dw1")
        _close(got[4], dw2.sum(0), (nr + 8) * F2 * dw2.abs().sum(0) + 1e-30, "dw2")
        only = tokens.block_norm_grad(some_dr, dy, branch, ga, r, rb, rr, w1, w2, scale, params=False)
        assert only[3] is None and only[4] is None and torch.equal(only[0], got[0]) and torch.equal(only[1], got[1])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(1100, 2056), (700, 2049), (700, 4096), (500, 4104), (500, 5003), (300, 8200), (200, 16384)])
def test_many_wide_rows(shape, dtype):
    """Rows that several blocks share, enough of them that each group of blocks has many one after the other."""
    test_block(shape, dtype, "plain")


@pytest.mark.parametrize("cols", [8, 1003, 4096, 20000])
def test_f32_gates_at_any_size(cols):
    """In f32 the gate's error does not grow with its size: an exponential and a division of at most two units each (2^-23), a sum
    and a product of half a unit: 6 at most. sigmoid times 1 - sigmoid is t / (1 + t)^2: the exponential once, sum and division
    twice, and up to four products and a difference: 10."""
    g = torch.linspace(-80.0, 80.0, 3 * cols, device="cuda").view(3, cols)
    one, zero = torch.ones_like(g), torch.zeros_like(g)
    r, _, _, rstd = tokens.block_norm(zero, one, g, post=False)
    a, na = torch.sigmoid(g.double()), torch.sigmoid(-g.double())
    _close(r, a, 6 * F2 * a, "r")
    dx, db, dg, _, _ = tokens.block_norm_grad(one, zero, one, g, r, None, rstd)
    _close(dx, one.double(), 0 * a, "dx")
    _close(db, a, 6 * F2 * a, "dbranch")
    _close(dg, a * na, 10 * F2 * a * na, "dgate")


@pytest.mark.parametrize("cols", [4096, 8192, 16384])
def test_wide_rows_in_graphs_and_on_two_streams(cols):
    x, branch, ga, w1, w2, dr, dy = _inputs(400, cols, BF16, True, 0, 0, cols)
    r, y, rb, rr = tokens.block_norm(x, branch, ga, w1, w2, 1.0, 1e-5, True)
    call = lambda: tokens.block_norm_grad(dr, dy, branch, ga, r, rb, rr, w1, w2, 1.0)
    want = call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = call()
    for _ in range(3):
        for t in kept:
            t.zero_()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(kept, want))
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(call())
    torch.cuda.synchronize()
    for other in got:
        assert all(torch.equal(a, b) for a, b in zip(other, want))
    tokens.check()


@pytest.mark.parametrize("post", [True, False])
def test_gradients_are_differences(post):
    """Central differences of sum(r cr + y cy) in f32 rows: the step h = 1e-2 is off by h^2 of a third derivative of order one
    and by 2^-23 of the sum (about 10) over h."""
    rows, cols, h = 3, 40, 1e-2
    x, branch, gate, w1, w2, cr, cy = _inputs(rows, cols, F32, True, 0, 0, 5)

    def loss(x, branch, gate, w1, w2):
        r, y, _, _ = tokens.block_norm(x, branch, gate, w1, w2, 0.7, 1e-5, post)
        return float((r.double() * cr.double()).sum() + (y.double() * cy.double()).sum())

    r, _, rb, rr = tokens.block_norm(x, branch, gate, w1, w2, 0.7, 1e-5, post)
    grads = tokens.block_norm_grad(cr, cy, branch, gate, r, rb, rr, w1, w2, 0.7)
    args = [x, branch, gate, w1, w2]
    for i, grad in enumerate(grads):
        for at in (0, 17, 39):
            ends = []
            for side in (h, -h):
                moved = [a.clone() for a in args]
                moved[i].view(-1)[at] += side
                ends.append(loss(*moved))
            assert abs((ends[0] - ends[1]) / (2 * h) - float(grad.reshape(-1)[at])) < 5e-3, (i, at)


def test_weights_at_any_float():
    """Weights that begin at 4 bytes take the single-value path: the same results to the rounding of its sums' order."""
    x, branch, gate, w1, w2, dr, dy = _inputs(9, 256, F32, True, 0, 0, 4)
    off = lambda w: torch.cat([w[:1], w])[1:]
    assert off(w1).data_ptr() % 16
    a = tokens.block_norm(x, branch, gate, w1, w2)
    b = tokens.block_norm(x, branch, gate, off(w1), off(w2))
    ga = tokens.block_norm_grad(dr, dy, branch, gate, a[0], a[2], a[3], w1, w2)
    gb = tokens.block_norm_grad(dr, dy, branch, gate, a[0], a[2], a[3], off(w1), off(w2))
    for p, q in zip(a + ga, b + gb):
        assert ((p - q).abs() <= 64 * F2 * (1 + p.abs() + 16)).all()


def test_extremes():
    """Gates at both ends, rows of zeros, infinities in one row that leave the others alone."""
    x = torch.randn(4, 64, device="cuda")
    branch = torch.randn(4, 64, device="cuda")
    gate = torch.randn(4, 64, device="cuda")
    gate[0, 0], gate[0, 1], gate[0, 2], gate[0, 3] = 200.0, -200.0, math.inf, -math.inf
    x[1] = 0
    branch[1] = 0
    branch[2, 5] = math.inf
    r, y, rb, rr = tokens.block_norm(x, branch, gate)
    ok = [0, 1, 3]
    rref, yref, _, _, _ = _forward(x, branch, gate, None, None, 1.0, 1e-5, True)
    _close(r[ok], rref[ok], 1e-5 * (1 + rref[ok].abs()), "r")
    _close(y[ok], yref[ok], 1e-5 * (1 + yref[ok].abs()), "y")
    grads = tokens.block_norm_grad(x, y, branch, gate, r, rb, rr, params=False)
    assert all(torch.isfinite(t[ok]).all() for t in grads[:3])
    assert (grads[2][0, :4] == 0).all()


def test_streams_capture_and_bits():
    x, branch, gate, w1, w2, dr, dy = _inputs(1000, 1024, BF16, True, 0, 0, 1)
    fwd = tokens.block_norm(x, branch, gate, w1, w2)
    want = tokens.block_norm_grad(dr, dy, branch, gate, fwd[0], fwd[2], fwd[3], w1, w2)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            f = tokens.block_norm(x, branch, gate, w1, w2)
            got.append(tokens.block_norm_grad(dr, dy, branch, gate, f[0], f[2], f[3], w1, w2))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        f = tokens.block_norm(x, branch, gate, w1, w2)
        g = tokens.block_norm_grad(dr, dy, branch, gate, f[0], f[2], f[3], w1, w2)
    for t in g:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_more_than_2_31_values():
    """The last rows of a matrix whose offsets pass 32 bits are those of a small one; sums over all rows see each row once."""
    rows, cols, last = 1_050_000, 2048, 5
    small = _inputs(last, cols, BF16, True, 0, 0, 2)
    big = [torch.zeros(rows, cols, device="cuda", dtype=BF16) if t.dim() == 2 else t for t in small]
    for b, t in zip(big, small):
        if b.dim() == 2:
            b[rows - last:] = t
    x, branch, gate, w1, w2, dr, dy = big
    r, y, rb, rr = tokens.block_norm(x, branch, gate, w1, w2)
    sr, sy, srb, srr = tokens.block_norm(small[0], small[1], small[2], w1, w2)
    for a, b in ((r, sr), (y, sy), (rb, srb), (rr, srr)):
        assert torch.equal(a[rows - last:], b)
    del x, y
    g = tokens.block_norm_grad(dr, dy, branch, gate, r, rb, rr, w1, w2)
    sg = tokens.block_norm_grad(small[5], small[6], small[1], small[2], sr, srb, srr, w1, w2)
    for a, b in zip(g[:3], sg[:3]):
        assert torch.equal(a[rows - last:], b)
    for a, b in zip(g[3:], sg[3:]):  # every other row adds exact zeros; the five rows' order differs
        assert ((a - b).abs() <= 8 * F2 * 5 * (1 + b.abs())).all()


def test_no_rows_and_refusals():
    x = torch.zeros(4, 16, device="cuda")
    w = torch.ones(16, device="cuda")
    r, y, rb, rr = tokens.block_norm(x[:0], x[:0], None, w, w)
    assert r.shape == y.shape == (0, 16) and rb.shape == rr.shape == (0,)
    g = tokens.block_norm_grad(None, y, x[:0], None, r, rb, rr, w, w)
    assert g[0].shape == (0, 16) and (g[3] == 0).all() and (g[4] == 0).all()
    f = torch.ones(4, device="cuda")
    for call in (lambda: tokens.block_norm(x, x.bfloat16()), lambda: tokens.block_norm(x, x[:3]),
                 lambda: tokens.block_norm(x, x, x[:, :8]), lambda: tokens.block_norm(x, x, None, w[:8]),
                 lambda: tokens.block_norm(x, x, None, w, w.double()), lambda: tokens.block_norm(x.half(), x.half()),
                 lambda: tokens.block_norm(x, x, eps=-1.0), lambda: tokens.block_norm(x.cpu(), x.cpu()),
                 lambda: tokens.block_norm(x, x.cpu()), lambda: tokens.block_norm(x[:, :0], x[:, :0]),
                 lambda: tokens.block_norm_grad(x, x, x, None, x, f, f[:2], w, w),
                 lambda: tokens.block_norm_grad(x, x, x, None, x, f, None, w, w),
                 lambda: tokens.block_norm_grad(x.t(), x, x, None, x, f, f, w, w),
                 lambda: tokens.block_norm_grad(x, None, x, None, x, f, f, w, w)):
        with pytest.raises(plb.PufferError):
            call()
