"""The gated delta rule (chunks, gradient, single tokens) against a plain 64-bit recurrence, token by token.

Tolerances: bf16 results are off by at most B = 2^-8 of their value. Products carry f32 operands as two bf16 parts: each
loses at most 2^-17 of an operand, and the product of the two second parts, 3 * 2^-17 in all of the product's bound by
norms. The rule contracts (keys of length one, beta below 1, decays below 1), so an old error does not grow, and a
result passes through at most 5 products of each chunk (states, outputs), 12 (gradients), whose terms may be four times
their sum."""
import math

import pytest

torch = pytest.importorskip("torch")

import pufferlean_b200 as plb  # noqa: E402
from pufferlean_b200 import tokens  # noqa: E402

pytestmark = pytest.mark.gpu
B, PART = 2.0 ** -8, 3 * 2.0 ** -17
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


@pytest.fixture(scope="module", autouse=True)
def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _inputs(lengths, hk, hv, dk, dv, seed, reset=0.0, pad=0, front=0, behind=0, wide=0):
    """front, behind: rows of no sequence; wide: extra columns beside every token's heads."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n = sum(lengths) + front + behind
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")

    def rows(t):
        n, h, d = t.shape
        buf = torch.full((n, h * (d + pad) + wide), float("nan"), device="cuda", dtype=BF16)
        v = buf[:, wide:].view(n, h, d + pad)[:, :, :d] if not wide else buf[:, wide:].unflatten(1, (h, d + pad))[:, :, :d]
        v.copy_(t)
        return v

    unit = lambda t: t / t.norm(dim=2, keepdim=True)
    q, k, v = rows(unit(r(n, hk, dk))), rows(unit(r(n, hk, dk) + r(1, hk, dk))), rows(r(n, hv, dv))
    g = -torch.exp(r(n, hv) - 2.0)
    g[torch.rand(n, generator=gen, device="cuda") < reset] = -math.inf
    beta = torch.sigmoid(r(n, hv))
    off = [front]
    for x in lengths:
        off.append(off[-1] + x)
    offsets = torch.tensor(off, dtype=torch.int32, device="cuda")
    state = r(len(lengths), hv, dk, dv) * 0.3
    return q, k, v, g, beta, offsets, state, rows(r(n, hv, dv)), r(len(lengths), hv, dk, dv) * 0.3


def _ref(q, k, v, g, beta, offsets, state, scale, do=None, dstate=None):
    """Outputs, final states and, with do, gradients; also the largest state norm of each head."""
    n, hk, dk = q.shape
    hv, dv = v.shape[1:]
    rep = hv // hk
    qd, kd = (t.double().repeat_interleave(rep, 1) for t in (q, k))
    vd, a, b = v.double(), torch.exp(g.double()), beta.double()
    o = torch.zeros(n, hv, dv, dtype=F64, device="cuda")
    final = state.double().clone()
    zeros = lambda *s: torch.zeros(*s, dtype=F64, device="cuda")
    grads = [zeros(n, hv, dk), zeros(n, hv, dk), zeros(n, hv, dv), zeros(n, hv), zeros(n, hv), zeros(*state.shape)]
    big = 0.0
    off = offsets.tolist()
    for s in range(len(off) - 1):
        S, path = state[s].double(), []
        for t in range(off[s], off[s + 1]):
            sd = S * a[t][:, None, None]
            err = vd[t] - torch.einsum("hij,hi->hj", sd, kd[t])
            S = sd + torch.einsum("hi,hj->hij", kd[t], err * b[t][:, None])
            o[t] = scale * torch.einsum("hij,hi->hj", S, qd[t])
            path.append((sd, err, S))
            big = max(big, float(S.flatten(1).norm(dim=1).max()), float(vd[t].norm(dim=1).max()))
        final[s] = S
        if do is None:
            continue
        dS = dstate[s].double() if dstate is not None else torch.zeros_like(S)
        for t in range(off[s + 1] - 1, off[s] - 1, -1):
            sd, err, S = path[t - off[s]]
            dot = scale * do[t].double()
            grads[0][t] = torch.einsum("hij,hj->hi", S, dot)
            dS = dS + torch.einsum("hi,hj->hij", qd[t], dot)
            du = torch.einsum("hij,hi->hj", dS, kd[t])
            dr = du * b[t][:, None]
            grads[1][t] = torch.einsum("hij,hj->hi", dS, err * b[t][:, None]) - torch.einsum("hij,hj->hi", sd, dr)
            grads[2][t] = dr
            grads[4][t] = (du * err).sum(-1)
            dS = dS - torch.einsum("hi,hj->hij", kd[t], dr)
            grads[3][t] = (dS * sd).sum((-1, -2))
            dS = dS * a[t][:, None, None]
        grads[5][s] = dS
    for i in (0, 1):
        grads[i] = grads[i].view(n, hk, rep, dk).sum(2)
    return o, final, grads, big


def _near(got, ref, rel, what, floor=0.0):
    """By norm."""
    off = (got.double() - ref)
    norm = float(ref.norm())
    assert torch.isfinite(off).all(), what
    assert float(off.norm()) <= rel * norm + floor, (what, float(off.norm()), norm)


def _check(lengths, hk, hv, dk, dv, seed=0, with_state=True, scale=None, grad=True, **more):
    q, k, v, g, beta, offsets, state, do, dstate = _inputs(lengths, hk, hv, dk, dv, seed, **more)
    sc = dk ** -0.5 if scale is None else scale
    given = state if with_state else None
    first = state if with_state else torch.zeros_like(state)
    o, final, saved = tokens.delta_rule(q, k, v, g, beta, offsets, given, scale, save=grad)
    ro, rfinal, rgrads, big = _ref(q, k, v, g, beta, offsets, first, sc, do if grad else None, dstate)
    chunks = max([1] + [-(-x // 64) for x in lengths])
    state_off = chunks * 5 * PART * big
    assert o.shape == v.shape and o.dtype == BF16 and final.shape == state.shape
    off = (o.double() - ro).abs()
    assert (off <= B * ro.abs() + abs(sc) * 2 * state_off).all(), float(off.max())
    assert ((final.double() - rfinal).flatten(2).norm(dim=2) <= state_off).all()
    if not grad:
        assert saved is None
        return
    grads = tokens.delta_rule_grad(do, dstate, q, k, v, g, beta, offsets, saved, scale)
    for name, x, r in zip(("dq", "dk", "dv", "dg", "dbeta", "dstate"), grads, rgrads):
        assert x.dtype == (BF16 if name in ("dq", "dk", "dv") else F32) and x.shape == r.shape, name
        # dg can vanish while its terms do not (a first token without a state): it is a sum of rows less a sum of columns of
        # at most 64 terms each in f32, off by 64 * 2^-23 of what those sums hold, and they are bounded by the sums over tokens of
        # |q| |dq| and |k| |dk|
        floor = 0.0 if name != "dg" else 64 * 2.0 ** -23 * float(
            (q.double().norm(dim=2) * rgrads[0].norm(dim=2)).sum() + (k.double().norm(dim=2) * rgrads[1].norm(dim=2)).sum())
        _near(x, r, 12 * 4 * PART + (B if x.dtype == BF16 else 0.0), name, floor)
    return q, k, v, g, beta, offsets, state, do, dstate, grads


@pytest.mark.parametrize("lengths", [[1], [2], [63], [64], [65], [128], [200], [1, 0, 64, 3, 130, 0, 65], [0, 0], [0, 5]])
def test_lengths(lengths):
    _check(lengths, 2, 2, 64, 64)
    _check(lengths, 1, 1, 128, 128, seed=1, with_state=False)


@pytest.mark.parametrize("dk,dv", [(1, 1), (8, 8), (16, 200), (24, 40), (63, 65), (64, 64), (65, 63), (72, 100), (100, 72),
                                   (128, 128), (128, 129), (127, 320), (40, 512)])
def test_widths(dk, dv):
    _check([70, 3, 129], 1, 2, dk, dv, seed=dk)


@pytest.mark.parametrize("hk,hv", [(1, 1), (1, 5), (2, 6), (3, 3), (4, 16)])
def test_shared_heads(hk, hv):
    _check([90, 20], hk, hv, 32, 24, seed=hv)


@pytest.mark.parametrize("reset", [0.01, 0.2, 1.0])
def test_resets(reset):
    *_, g, beta, offsets, state, do, dstate, grads = _check([300, 64, 17], 2, 4, 64, 48, reset=reset, seed=7)
    assert (grads[3][g < -104] == 0).all()


@pytest.mark.parametrize("layout", [dict(pad=8), dict(pad=4), dict(pad=2), dict(pad=3), dict(wide=8), dict(wide=4),
                                    dict(wide=2), dict(wide=5, pad=1)])
def test_strides(layout):
    _check([100, 31], 2, 4, 64, 72, seed=11, **layout)
    _check([100, 31], 2, 2, 100, 40, seed=12, **layout)


def test_one_projection():
    """Queries, keys and values side by side in one tensor, as a projection leaves them: the same bits as packed ones."""
    q, k, v, g, beta, offsets, state, do, dstate = _inputs([150, 70], 2, 4, 64, 32, 3)
    n = q.shape[0]
    wide = torch.cat([q.reshape(n, -1), k.reshape(n, -1), v.reshape(n, -1)], 1)
    views = wide[:, :128].view(n, 2, 64), wide[:, 128:256].view(n, 2, 64), wide[:, 256:].view(n, 4, 32)
    a = tokens.delta_rule(q, k, v, g, beta, offsets, state)
    b = tokens.delta_rule(*views, g, beta, offsets, state)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_rows_of_no_sequence():
    q, k, v, g, beta, offsets, state, do, dstate, grads = _check([70, 9], 2, 4, 40, 32, seed=2, front=5, behind=13)
    o = tokens.delta_rule(q, k, v, g, beta, offsets, state)[0]
    for t in (o, grads[0], grads[1], grads[2], grads[3], grads[4]):
        assert (t[:5] == 0).all() and (t[84:] == 0).all()


def test_even_sequences_need_no_offsets():
    q, k, v, g, beta, offsets, state, do, dstate = _inputs([100] * 3, 2, 2, 64, 64, 5)
    a = tokens.delta_rule(q, k, v, g, beta, offsets, state, save=True)
    b = tokens.delta_rule(q, k, v, g, beta, None, state, save=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    ga = tokens.delta_rule_grad(do, dstate, q, k, v, g, beta, offsets, a[2])
    gb = tokens.delta_rule_grad(do, dstate, q, k, v, g, beta, None, b[2])
    assert all(torch.equal(x, y) for x, y in zip(ga, gb))
    one = tokens.delta_rule(q, k, v, g, beta)  # one sequence, no state
    assert one[1].shape == (1, 2, 64, 64) and one[2] is None


def test_long_sequence_and_offsets():
    """A long sequence, and rows whose offsets in the tensors pass 32 bits."""
    _check([2500], 1, 2, 128, 64, seed=9)
    n, h, d = 300000, 16, 512  # v: 2.4e9 values
    v = torch.empty(n, h, d, device="cuda", dtype=BF16)
    q, k, vs, g, beta, offsets, state, do, dstate = _inputs([100], 1, h, 16, d, 4)
    v[n - 100:] = vs
    put = lambda t, fill: torch.cat([torch.full((n - 100,) + tuple(t.shape[1:]), fill, device="cuda", dtype=t.dtype), t])
    at = torch.tensor([n - 100, n], dtype=torch.int32, device="cuda")
    o, final, _ = tokens.delta_rule(put(q, 0.0), put(k, 0.0), v, put(g, 0.0), put(beta, 0.0), at, state)
    want = tokens.delta_rule(q, k, vs, g, beta, offsets, state)
    assert torch.equal(o[n - 100:], want[0]) and torch.equal(final, want[1])
    assert not o[:n - 100:997].any()


@pytest.mark.parametrize("lengths", [[64], [300], [2500], [130, 64, 1, 700]])
@pytest.mark.parametrize("dk,dv,reset", [(128, 64, 0.0), (64, 72, 0.01), (40, 130, 0.0)])
@pytest.mark.parametrize("decay", [1.0, 0.0])
def test_f32_results(lengths, dk, dv, reset, decay):
    """f32 results by norm, with decays and without any. Products of three bf16 parts hold all of an f32 operand; their sums are cut off
    towards zero at each of their 4 to 8 steps of 16, by 2^-23 at most and half of it on average: 4 * 2^-23, and 2^-22 for the
    decays' exponentials. A result passes through five to twelve products, whose errors add up by squares: sqrt(12) * 6 * 2^-23. Two
    parts of an operand would be 2^-18 off."""
    q, k, v, g, beta, offsets, state, do, dstate = _inputs(lengths, 1, 2, dk, dv, dk + len(lengths), reset=reset)
    g = torch.where(torch.isinf(g), g, g * decay)
    o, final, saved = tokens.delta_rule(q, k, v, g, beta, offsets, state, save=True)
    grads = tokens.delta_rule_grad(do, dstate, q, k, v, g, beta, offsets, saved)
    _, rfinal, rgrads, _ = _ref(q, k, v, g, beta, offsets, state, dk ** -0.5, do, dstate)
    tol = math.sqrt(12) * 6 * 2.0 ** -23
    floor = 2.0 ** -23 * float((q.double().norm(dim=2) * rgrads[0].norm(dim=2)).norm()
                               + (k.double().norm(dim=2) * rgrads[1].norm(dim=2)).norm()) * 8
    _near(final, rfinal, tol, "final")
    _near(grads[3], rgrads[3], tol, "dg", floor)
    _near(grads[4], rgrads[4], tol, "dbeta")
    _near(grads[5], rgrads[5], tol, "dstate")


@pytest.mark.parametrize("state", [None, 0.0])
def test_first_tokens_of_an_empty_memory(state):
    """Nothing depends on what a first token keeps of no state: its dg is zero, not nearly; and right where there is a state."""
    q, k, v, g, beta, offsets, st, do, dstate = _inputs([1, 1, 70, 1, 130], 2, 4, 72, 100, 37)
    first = offsets[:-1].long()
    given = None if state is None else torch.zeros_like(st)
    _, _, saved = tokens.delta_rule(q, k, v, g, beta, offsets, given, save=True)
    dg = tokens.delta_rule_grad(do, dstate, q, k, v, g, beta, offsets, saved)[3]
    assert (dg[first] == 0).all() and (dg[first[2] + 1] != 0).all()
    _, _, saved = tokens.delta_rule(q, k, v, g, beta, offsets, st, save=True)
    dg = tokens.delta_rule_grad(do, dstate, q, k, v, g, beta, offsets, saved)[3]
    _, _, rgrads, _ = _ref(q, k, v, g, beta, offsets, st, 72 ** -0.5, do, dstate)
    _near(dg[first], rgrads[3][first], math.sqrt(12) * 6 * 2.0 ** -23, "dg")


@pytest.mark.parametrize("g0", [-0.5, -1.0, -1.9])
def test_states_that_fade(g0):
    """What reaches a state through 40 tokens that keep little of it is right relative to itself, though it is 2^-29 to 2^-110."""
    q, k, v, g, beta, offsets, state, do, dstate = _inputs([40, 7], 2, 2, 64, 64, 29)
    g = g0 + 0.1 * g
    _, _, saved = tokens.delta_rule(q, k, v, g, beta, offsets, state, save=True)
    grads = tokens.delta_rule_grad(torch.zeros_like(do), dstate, q, k, v, g, beta, offsets, saved)
    _, _, rgrads, _ = _ref(q, k, v, g, beta, offsets, state, 0.125, torch.zeros_like(do), dstate)
    for s in (0, 1):
        _near(grads[5][s], rgrads[5][s], math.sqrt(12) * 6 * 2.0 ** -23, "dstate")


def test_tokens_that_write_nothing():
    """beta zero, or next to it: the token leaves the state as it is, has no dv, and still a dbeta."""
    q, k, v, g, beta, offsets, state, do, dstate = _inputs([150, 70, 64], 2, 4, 64, 72, 23, reset=0.02)
    beta[::3] = 0.0
    beta[1::7] = 1e-20
    beta[64:128] = 0.0  # a chunk's worth
    o, final, saved = tokens.delta_rule(q, k, v, g, beta, offsets, state, save=True)
    grads = tokens.delta_rule_grad(do, dstate, q, k, v, g, beta, offsets, saved)
    ro, rfinal, rgrads, _ = _ref(q, k, v, g, beta, offsets, state, 0.125, do, dstate)
    assert (grads[2][beta == 0] == 0).all()
    _near(o, ro, B, "o")
    tol = math.sqrt(12) * 6 * 2.0 ** -23
    floor = 2.0 ** -20 * float((q.double().norm(dim=2) * rgrads[0].norm(dim=2)).norm()
                               + (k.double().norm(dim=2) * rgrads[1].norm(dim=2)).norm())
    for name, x, r in zip(("final", "dq", "dk", "dv", "dg", "dbeta", "dstate"), (final,) + grads, [rfinal] + rgrads):
        _near(x, r, B if x.dtype == BF16 else tol, name, floor if name == "dg" else 0.0)
    zero = beta == 0
    _near(grads[4][zero], rgrads[4][zero], tol, "dbeta where beta is zero")


def _same(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dk,dv", [(64, 64), (100, 72)])
def test_what_is_not_finite_stays_where_it_belongs(dk, dv):
    """A NaN reaches what its sequence has in its chunk and behind it, and nothing else: not the sequences beside it, not the
    other heads, not rows of no sequence, which are not read either; and a first token that forgets forgets any state."""
    q, k, v, g, beta, offsets, state, do, dstate = _inputs([100, 150, 70], 2, 4, dk, dv, 17, front=3, behind=9)
    g[offsets[:-1].long()] = -math.inf

    def both(*a, st=state):
        q, k, v, g, beta, do = a
        o, final, saved = tokens.delta_rule(q, k, v, g, beta, offsets, st, save=True)
        return (o, final) + tokens.delta_rule_grad(do, dstate, q, k, v, g, beta, offsets, saved)

    clean = [t.clone() for t in (q, k, v, g, beta, do)]
    want = both(*clean)
    assert _same(both(*clean, st=torch.full_like(state, math.nan)), want)
    assert _same(both(*clean, st=torch.full_like(state, math.inf)), want)
    for t in clean:  # rows of no sequence
        t[:3] = math.nan
        t[-9:] = -math.inf
    assert _same(both(*clean), want)
    for i, t in enumerate(clean):  # the middle sequence, its last chunk; q and k of the second key head, value heads 2 and 3
        dirty = [x.clone() for x in clean]
        dirty[i][103 + 140, 1 if i < 2 else 2] = math.nan
        got = both(*dirty)
        rows = torch.ones(len(q), dtype=torch.bool, device="cuda")
        rows[103:253] = False
        for x, y in zip(got, want):
            if x.shape[0] == 3:
                assert torch.equal(x[::2], y[::2]) and torch.equal(x[1, :2], y[1, :2]), i
            else:
                heads = 1 if x.shape[1] == 2 else 2
                assert torch.equal(x[rows], y[rows]) and torch.equal(x[:, :heads], y[:, :heads]), i
        assert torch.equal(got[0][103:103 + 128], want[0][103:103 + 128]), i  # the chunks before it


def test_gradients_take_what_was_saved():
    q, k, v, g, beta, offsets, state, do, dstate = _inputs([130, 7], 2, 4, 32, 32, 6)
    _, _, saved = tokens.delta_rule(q, k, v, g, beta, offsets, state, save=True)
    want = tokens.delta_rule_grad(do, dstate, q, k, v, g, beta, offsets, saved)
    for t in (q, k, g, beta):  # (all but v)
        t.fill_(math.nan)
    assert _same(tokens.delta_rule_grad(do, dstate, q, k, v, g, beta, offsets, saved), want)


def test_optional_gradients():
    q, k, v, g, beta, offsets, state, do, dstate = _inputs([130, 7], 2, 4, 32, 32, 6)
    _, _, saved = tokens.delta_rule(q, k, v, g, beta, offsets, state, save=True)
    a = tokens.delta_rule_grad(do, None, q, k, v, g, beta, offsets, saved)
    b = tokens.delta_rule_grad(do, torch.zeros_like(dstate), q, k, v, g, beta, offsets, saved)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_gradients_are_differences():
    """Central differences of sum(o co) + sum(final cf) in g, beta and the state (f32 arguments; o is bf16, so co is zero on
    it and the loss goes through the final state, which is f32): steps of h = 1e-2, off by h^2 and by 1e-5 of the sum over h."""
    q, k, v, g, beta, offsets, state, do, dstate = _inputs([90], 1, 1, 16, 8, 8)
    g = g.clamp(min=-0.3)

    def loss(g, beta, state):
        return float((tokens.delta_rule(q, k, v, g, beta, offsets, state)[1].double() * dstate.double()).sum())

    _, _, saved = tokens.delta_rule(q, k, v, g, beta, offsets, state, save=True)
    grads = tokens.delta_rule_grad(torch.zeros_like(do), dstate, q, k, v, g, beta, offsets, saved)
    args, h = [g, beta, state], 1e-2
    for i, grad in enumerate(grads[3:]):
        for at in (0, 60, 70, 89):
            ends = []
            for side in (h, -h):
                moved = [a.clone() for a in args]
                moved[i].view(-1)[at] += side
                ends.append(loss(*moved))
            assert abs((ends[0] - ends[1]) / (2 * h) - float(grad.reshape(-1)[at])) < 1e-2, (i, at)


@pytest.mark.parametrize("n,hk,hv,dk,dv", [(1, 1, 1, 1, 1), (3, 2, 4, 16, 24), (5, 1, 3, 63, 65), (2, 2, 2, 64, 64),
                                           (4, 3, 3, 72, 100), (7, 2, 4, 128, 128), (2, 1, 2, 100, 33), (3, 1, 1, 128, 514)])
def test_step(n, hk, hv, dk, dv):
    """One token at a time is the recurrence itself: f32 sums of dk terms."""
    q, k, v, g, beta, _, _, _, _ = _inputs([n], hk, hv, dk, dv, dk + dv)
    g[0] = -math.inf
    state = torch.randn(n, hv, dk, dv, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    o, new = tokens.delta_rule_step(q, k, v, g, beta, state, 0.3)
    rep = hv // hk
    qd, kd = (t.double().repeat_interleave(rep, 1) for t in (q, k))
    sd = state.double() * torch.exp(g.double())[..., None, None]
    err = v.double() - torch.einsum("nhij,nhi->nhj", sd, kd)
    ref = sd + torch.einsum("nhi,nhj,nh->nhij", kd, err, beta.double())
    ro = 0.3 * torch.einsum("nhij,nhi->nhj", ref, qd)
    tol = 2.0 ** -23 * (32 + math.log2(dk + 1))
    bound = torch.einsum("nhij,nhi->nhj", sd.abs(), kd.abs()) + v.double().abs()
    tol_s = tol * (sd.abs() + torch.einsum("nhi,nhj,nh->nhij", kd.abs(), bound, beta.double()))
    assert ((new.double() - ref).abs() <= tol_s).all()
    reach = torch.einsum("nhij,nhi->nhj", sd.abs(), qd.abs()) + (kd * qd).abs().sum(-1, keepdim=True) * bound
    assert ((o.double() - ro).abs() <= B * ro.abs() + 0.3 * 2 * tol * reach).all()
    bad = state.clone()
    bad[0] = math.nan  # a reset forgets whatever was there
    o2, new2 = tokens.delta_rule_step(q, k, v, g, beta, bad, 0.3, out=bad)
    assert new2.data_ptr() == bad.data_ptr() and torch.equal(o2, o) and torch.equal(new2, new)


def test_states_at_any_float():
    """States that begin at 4 or 8 bytes give the same bits as aligned ones."""
    q, k, v, g, beta, offsets, state, _, _ = _inputs([3], 1, 2, 32, 128, 4)
    state = torch.randn(3, 2, 32, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    want = tokens.delta_rule_step(q, k, v, g, beta, state)
    one = tokens.delta_rule(q, k, v, g, beta, offsets, state[:1].contiguous())
    for shift in (1, 2, 3):
        buf = torch.zeros(state.numel() + 4, device="cuda")
        moved = buf[shift:shift + state.numel()].view_as(state)
        moved.copy_(state)
        o, new = tokens.delta_rule_step(q, k, v, g, beta, moved, out=moved)
        assert torch.equal(new, want[1]) and (o.float() - want[0].float()).abs().max() <= B * want[0].float().abs().max()
        moved.copy_(state)
        again = tokens.delta_rule(q, k, v, g, beta, offsets, moved[:1])
        assert torch.equal(again[0], one[0]) and torch.equal(again[1], one[1])


def test_steps_are_the_sequence():
    q, k, v, g, beta, offsets, state, _, _ = _inputs([70], 2, 4, 64, 64, 21, reset=0.03)
    o, final, _ = tokens.delta_rule(q, k, v, g, beta, offsets, state)
    s, steps = state.clone(), []
    for t in range(70):
        out, s = tokens.delta_rule_step(q[t:t + 1], k[t:t + 1], v[t:t + 1], g[t:t + 1], beta[t:t + 1], s, out=s)
        steps.append(out)
    off = (torch.cat(steps).double() - o.double()).abs()
    big = float(final.norm(dim=(2, 3)).max()) + 12.0
    assert (off <= 2 * B * o.double().abs() + 2 * 5 * PART * big).all()
    assert ((s - final).double().flatten(2).norm(dim=2) <= 2 * 5 * PART * big).all()


def test_bits_streams_and_capture():
    q, k, v, g, beta, offsets, state, do, dstate = _inputs([200, 65, 1], 2, 4, 64, 72, 31, reset=0.02)

    def both():
        o, final, saved = tokens.delta_rule(q, k, v, g, beta, offsets, state, save=True)
        return (o, final) + tokens.delta_rule_grad(do, dstate, q, k, v, g, beta, offsets, saved)

    want = both()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(both())
    torch.cuda.synchronize()
    for x in got:
        assert all(torch.equal(a, b) for a, b in zip(x, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for t in out:
        t.zero_()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals():
    q, k, v, g, beta, offsets, state, do, dstate = _inputs([20, 12], 2, 4, 16, 24, 1)
    ok = tokens.delta_rule(q, k, v, g, beta, offsets, state, save=True)
    saved = ok[2]
    run = tokens.delta_rule
    for call in (lambda: run(q.float(), k, v, g, beta), lambda: run(q, k[:5], v, g, beta), lambda: run(q, k, v[:, :3], g, beta),
                 lambda: run(q, k, v, g[:, :2], beta), lambda: run(q, k, v, g.double(), beta), lambda: run(q, k, v, g, beta.t()),
                 lambda: run(q, k, v, g, beta, offsets.long()), lambda: run(q, k, v, g, beta, offsets[:2], state),
                 lambda: run(q, k, v, g, beta, offsets, state[:, :, :8]), lambda: run(q, k, v, g, beta, offsets, state.double()),
                 lambda: run(q, k, v, g, beta, None, torch.zeros(3, 4, 16, 24, device="cuda")),
                 lambda: run(q, k, v, g, beta, offsets, state, math.nan),
                 lambda: run(q.transpose(1, 2), k, v, g, beta), lambda: run(q.cpu(), k, v, g, beta),
                 lambda: run(q, k, v, g.cpu(), beta),
                 lambda: run(torch.zeros(4, 1, 129, device="cuda", dtype=BF16), torch.zeros(4, 1, 129, device="cuda", dtype=BF16),
                             torch.zeros(4, 1, 8, device="cuda", dtype=BF16), g[:4, :1].contiguous(), beta[:4, :1].contiguous()),
                 lambda: tokens.delta_rule_grad(do, dstate, q, k, v, g, beta, offsets, None),
                 lambda: tokens.delta_rule_grad(do, dstate, q, k, v, g, beta, offsets, (saved[0][:64], 2)),
                 lambda: tokens.delta_rule_grad(do[:, :2], dstate, q, k, v, g, beta, offsets, saved),
                 lambda: tokens.delta_rule_grad(do, dstate[:1], q, k, v, g, beta, offsets, saved),
                 lambda: tokens.delta_rule_step(q, k, v, g, beta, state),
                 lambda: tokens.delta_rule_step(q[:2], k[:2], v[:2], g[:2], beta[:2], None),
                 lambda: tokens.delta_rule_step(q[:1], k[:1], v[:1], g[:1], beta[:1], state[:1], out=state[:1].double())):
        with pytest.raises(plb.PufferError):
            call()
    both = torch.zeros(3, 4, 16, 24, device="cuda")
    with pytest.raises(plb.PufferError):
        tokens.delta_rule_step(q[:2], k[:2], v[:2], g[:2], beta[:2], both[:2], out=both[1:])


def test_nothing():
    q, k, v, g, beta, _, _, _, _ = _inputs([4], 1, 2, 16, 8, 1)
    none = [t[:0] for t in (q, k, v, g, beta)]
    state = torch.randn(2, 2, 16, 8, device="cuda")
    o, final, saved = tokens.delta_rule(*none, torch.zeros(3, dtype=torch.int32, device="cuda"), state, save=True)
    assert o.shape == (0, 2, 8) and torch.equal(final, state)
    grads = tokens.delta_rule_grad(o, state, *none, torch.zeros(3, dtype=torch.int32, device="cuda"), saved)
    assert torch.equal(grads[5], state)
    o, final, _ = tokens.delta_rule(*none, torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert o.shape == (0, 2, 8) and final.shape == (0, 2, 16, 8)
    o, new = tokens.delta_rule_step(*none, state[:0])
    assert o.shape == (0, 2, 8) and new.shape == (0, 2, 16, 8)
