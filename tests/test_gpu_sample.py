"""Drawing tokens (temperature, top-k, top-p, min-p, given random numbers) against a plain 64-bit implementation.

Sums and exponentials are f64 on both sides, so a token differs only where u comes within about 1e-12 of a border, which
these fixed inputs do not; logp is rounded once, to f32 (2^-24 of it; the logarithm's own error is far below)."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import pufferlean_b200 as plb  # noqa: E402
from pufferlean_b200 import tokens  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _row(z, u, temp, k, p, min_p):
    """(token, logp) of one row of doubles."""
    if np.isnan(z).any() or z.max() in (np.inf, -np.inf) or any(math.isnan(x) for x in (u, temp, p, min_p)):
        return -1, math.nan
    order = np.argsort(-z, kind="stable")
    if temp == 0 or p <= 0:
        return int(order[0]), 0.0
    e = np.exp((z - z.max()) / temp)
    if 0 < k < len(z):
        order = order[:k]
    mass = np.cumsum(e[order])
    keep = (mass - e[order] < p * mass[-1]) | (p >= 1)
    keep &= e[order] >= min(min_p, 1.0)
    keep[0] = True
    kept = np.zeros(len(z))
    kept[order[keep]] = e[order[keep]]
    cdf = np.cumsum(kept)
    t = int(np.searchsorted(cdf, min(max(u, 0.0), 1.0) * cdf[-1], side="right"))
    if t >= len(z) or kept[t] == 0:
        t = int(np.nonzero(kept)[0][-1])
    return t, (z[t] - z.max()) / temp - math.log(cdf[-1])


def _check(logits, u, temp=1.0, k=0, p=1.0, min_p=0.0):
    token, logp = tokens.sample(logits, u, temp, k, p, min_p)
    assert token.dtype == torch.int32 and logp.dtype == F32 and token.shape == logp.shape == u.shape
    z, us = logits.double().cpu().numpy(), u.double().cpu().numpy()
    at = lambda o, i: (o[i].item() if torch.is_tensor(o) else o)
    for i in range(len(us)):
        t, lp = _row(z[i], us[i], *(at(o, i) for o in (temp, k, p, min_p)))
        got, glp = int(token[i]), float(logp[i])
        assert got == t, (i, got, t, float(us[i]))
        assert (math.isnan(lp) and math.isnan(glp)) or abs(glp - lp) <= 2.0 ** -24 * abs(lp) + 1e-12, (i, glp, lp)
    return token


def _logits(n, v, dtype, seed, pad=0, offset=0, sigma=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    buf = torch.full((n * (v + pad) + offset + 8,), float("nan"), device="cuda", dtype=dtype)
    x = buf[offset:offset + n * (v + pad)].view(n, v + pad)[:, :v]
    x.copy_(torch.randn(n, v, generator=g, device="cuda") * sigma)
    return x, torch.rand(n, generator=g, device="cuda")


OPTIONS = [dict(), dict(temp=0.7), dict(k=5), dict(p=0.9), dict(min_p=0.05), dict(temp=1.3, k=40, p=0.8, min_p=0.01),
           dict(k=1), dict(temp=0.0), dict(k=1500, p=0.95), dict(p=0.0), dict(min_p=1.0), dict(k=100000)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,v", [(1, 1), (3, 2), (7, 17), (4, 1000), (3, 2049), (2, 16385), (3, 50021)])
@pytest.mark.parametrize("pad,offset", [(0, 0), (3, 1), (16, 8)])
def test_sizes_and_layouts(n, v, dtype, pad, offset):
    x, u = _logits(n, v, dtype, v + pad, pad, offset)
    for o in OPTIONS:
        _check(x, u, **o)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("v", [131072, 262144])
def test_widest(v, dtype):
    for sigma in (0.01, 1.0, 4.0):
        x, u = _logits(2, v, dtype, v, sigma=sigma)
        for o in (dict(), dict(k=50, p=0.95), dict(p=0.9), dict(p=0.9999), dict(p=0.9999999), dict(p=1e-4), dict(k=30000, p=0.5), dict(min_p=0.3)):
            _check(x, u, **o)


def test_many_rows():
    x, u = _logits(3000, 97, BF16, 5)
    _check(x, u, temp=0.8, k=20, p=0.9)
    _check(x, u)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,v", [(4, 16383), (4, 16384), (66, 16400), (67, 16400), (33, 131072), (34, 98311), (3, 200003)])
def test_both_sides_of_a_split(n, v, dtype):
    """Rows are split over several blocks from a length and up to a number of rows on: the same tokens on either side."""
    x, u = _logits(n, v, dtype, n + v, pad=3)
    for o in (dict(), dict(temp=0.8, k=50, p=0.95), dict(p=0.9)):
        a = tokens.sample(x, u, *(o.get(key, d) for key, d in (("temp", 1.0), ("k", 0), ("p", 1.0))))
        _check(x[:4], u[:4], **o)
        many = 70 if n < 70 else n
        times = -(-many // n)
        b = tokens.sample(x.repeat(times, 1)[:many], u.repeat(times)[:many],
                          *(o.get(key, d) for key, d in (("temp", 1.0), ("k", 0), ("p", 1.0))))
        assert torch.equal(a[0], b[0][:n]) and (a[1] - b[1][:n]).abs().max() <= 2.0 ** -22 * a[1].abs().max()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("v", [64, 5000, 131072])
def test_equal_logits(dtype, v):
    """Borders inside groups of equal logits, down to rows of one value: the lowest indices stay."""
    g = torch.Generator(device="cuda").manual_seed(v)
    u = torch.tensor([0.0, 0.25, 0.5, 0.999], device="cuda")
    flat = torch.full((4, v), -3.25, device="cuda", dtype=dtype)
    few = torch.randint(0, 3, (4, v), generator=g, device="cuda").to(dtype)
    for x in (flat, few):
        for o in (dict(), dict(k=7), dict(k=v // 2 + 1), dict(p=0.5), dict(k=v // 2, p=0.3), dict(p=0.9, min_p=0.2)):
            _check(x, u, **o)
    zeros = torch.zeros(4, v, device="cuda", dtype=dtype)
    zeros[:, ::2] = -0.0  # one value
    _check(zeros, u, k=3)
    assert int(tokens.sample(zeros, u, top_k=1)[0].max()) == 0


def test_nearly_equal_logits():
    """Distances that f32 cannot resolve against the largest logit, more of them than a list holds."""
    v = 6000
    x = torch.arange(v, device="cuda", dtype=F32).mul_(1e-12)[None].repeat(3, 1)
    x[:, 17] = 8.0
    u = torch.tensor([0.3, 0.9999, 0.99999], device="cuda")
    for o in (dict(k=10), dict(k=4000), dict(p=0.7), dict(p=0.9), dict(p=0.5, k=5000)):
        _check(x, u, **o)


def test_masks():
    g = torch.Generator(device="cuda").manual_seed(3)
    n, v = 6, 4099
    u = torch.rand(n, generator=g, device="cuda")
    u[0], u[1] = 0.0, 1.0 - 2.0 ** -24
    for dtype in (F32, BF16):
        for masked in (-math.inf, torch.finfo(dtype).min, -1e9):
            x = torch.randn(n, v, generator=g, device="cuda").to(dtype)
            hide = torch.rand(n, v, generator=g, device="cuda") < 0.9
            hide[2] = True
            hide[2, 4098] = False  # one token left
            x[hide] = masked
            for o in (dict(), dict(k=3), dict(k=2000), dict(p=0.9), dict(k=50, p=0.5, min_p=0.1), dict(temp=0.0)):
                token = _check(x, u, **o)
                assert int(token[2]) == 4098
                assert not hide[torch.arange(n), token.long()].any()
            low = torch.full((n, v), masked, device="cuda", dtype=dtype)  # nothing left, or all alike
            token = _check(low, u)
            assert (token == -1).all() if masked == -math.inf else (token >= 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,v", [(3, 9001), (2, 50021), (150, 9001), (150, 20011)])
def test_few_tokens_left(n, v, dtype):
    """All but a few tokens share one value, a mask's or another, and the rest are wherever a sample of the row may miss them."""
    g = torch.Generator(device="cuda").manual_seed(v + n)
    u = torch.rand(n, generator=g, device="cuda")
    for masked in (torch.finfo(dtype).min, -1e9, -700.0, -5.0):
        for left in (1, 3):
            x = torch.full((n, v), masked, device="cuda", dtype=dtype)
            at = torch.randint(0, v, (n, left), generator=g, device="cuda")
            x.scatter_(1, at, torch.randn(n, left, generator=g, device="cuda").to(dtype))
            for o in (dict(), dict(k=2), dict(k=50), dict(k=3000), dict(p=0.9), dict(k=50, p=0.5, min_p=0.1), dict(min_p=0.1)):
                _check(x, u, **o)


def test_bad_rows():
    x, u = _logits(9, 300, F32, 1)
    x[0, 7] = math.nan
    x[1, 299] = math.inf
    x[2] = -math.inf
    temp, p, min_p = (torch.full((9,), f, device="cuda") for f in (1.0, 0.9, 0.1))
    temp[3], temp[4], p[5], min_p[6], u[7] = math.nan, -1.0, math.nan, math.nan, math.nan
    token, logp = tokens.sample(x, u, temp, 0, p, min_p)
    assert (token[:8] == -1).all() and torch.isnan(logp[:8]).all()
    assert int(token[8]) >= 0 and bool(torch.isfinite(logp[8]))
    temp[3] = math.inf
    assert int(tokens.sample(x, u, temp)[0][3]) == -1


def test_options_by_row():
    n, v = 40, 3001
    x, u = _logits(n, v, F32, 9)
    g = torch.Generator(device="cuda").manual_seed(2)
    temp = torch.rand(n, generator=g, device="cuda") + 0.3
    temp[::7] = 0.0
    k = torch.randint(0, 60, (n,), generator=g, device="cuda", dtype=torch.int32)
    p = torch.rand(n, generator=g, device="cuda") * 1.2
    min_p = torch.rand(n, generator=g, device="cuda") * 0.2
    _check(x, u, temp, k, p, min_p)
    _check(x, u, temp, 0, p, 0.0)
    _check(x, u, 0.9, k, 1.0, min_p)


@pytest.mark.parametrize("temp", [1e-30, 1e-3, 50.0, 1e20])
def test_temperatures(temp):
    x, u = _logits(8, 5003, F32, 4)
    for o in (dict(), dict(k=9), dict(p=0.9), dict(k=3000, p=0.9)):
        _check(x, u, temp=temp, **o)


FILTERS = [dict(), dict(k=3), dict(k=1100), dict(p=0.85), dict(k=40, p=0.85, min_p=0.3), dict(min_p=0.45)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,v", [(3, 37), (2, 20011), (301, 1300)])  # a long row: a cluster, otherwise a block
@pytest.mark.parametrize("top", [0.0, -0.0, 1e-40, -1e-40, 3.0])
def test_tiniest_temperatures(top, n, v, dtype):
    """The largest logit is zero, or next to it: equal logits (both zeros are one) share the mass at any temperature. (Below 1e-38
    they count as that: it makes no difference to logits that are further apart than 1e-35.)"""
    x, u = _logits(n, v, dtype, v)
    x.sub_(x.max() + 1.0).add_(top)
    for i, at in enumerate((0, 11, 12, 29, 36)):
        x[:, at] = -top if top == 0.0 and i % 2 else top
    for temp in (1e-22, 1e-30, 1e-36, 1e-38, 1e-40, 1.4e-45, 1e-61, 1e-100, 1e-310):
        for o in FILTERS:
            token = _check(x, u, temp=temp, **o)
            assert (token >= 0).all()
        if temp >= 1e-45:
            _check(x, u, temp=torch.full((n,), temp, device="cuda"), p=torch.full((n,), 0.85, device="cuda"))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,v", [(2, 20011), (160, 1300)])
@pytest.mark.parametrize("temp", [2e-22, 1e-22, 1e-30, 1e-36, 2.0 ** -126])
def test_logits_as_small_as_the_temperature(temp, n, v, dtype):
    """Logits of a few temperatures around zero, down to numbers below the smallest normal one."""
    x, u = _logits(n, v, F32, v)
    x = (x.double() * temp).to(dtype)
    x[:, 5], x[:, 6] = 0.0, -0.0
    for o in FILTERS:
        _check(x, u, temp=temp, **o)


def test_temperatures_below_the_least():
    x, u = _logits(4, 700, F32, 3)
    x = x * 1e-37 * 0.1  # differences of a few 1e-38
    want = tokens.sample(x, u, 1e-38)
    for temp in (9e-39, 1e-40, 1e-300, torch.full((4,), 1e-42, device="cuda")):
        got = tokens.sample(x, u, temp)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    _check(x, u, temp=1e-38)


def test_temperatures_above_the_most():
    x, u = _logits(4, 700, F32, 3)
    want = tokens.sample(x, u, 1e30, 0, 0.7)
    for temp in (1e31, 1e300, torch.full((4,), 1e38, device="cuda")):
        got = tokens.sample(x, u, temp, 0, 0.7)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("k,p,min_p", [(0, 1.0, 0.0), (6, 1.0, 0.0), (0, 0.8, 0.0), (0, 1.0, 0.1)])
def test_shares(k, p, min_p):
    """Evenly spaced numbers give every token its share, to one draw."""
    n, v = 4096, 12
    x = torch.randn(v, generator=torch.Generator().manual_seed(k), dtype=F32).cuda()[None].repeat(n, 1)
    u = (torch.arange(n, device="cuda", dtype=torch.float64) + 0.5).div_(n).float()
    token, logp = tokens.sample(x, u, 1.0, k, p, min_p)
    count = torch.bincount(token.long(), minlength=v).double()
    seen = torch.zeros(v, dtype=torch.float64, device="cuda").scatter_(0, token.long(), torch.exp(logp.double()))
    assert (count - n * seen).abs().max() <= 1 + n * 2.0 ** -23
    assert abs(float(seen.sum()) - 1) < 1e-5


def test_same_bits_streams_and_capture():
    x, u = _logits(33, 50021, BF16, 8)
    want = [tokens.sample(x, u, 0.9, *o) for o in ((0, 0.9, 0.0), (50, 0.95, 0.0))]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(3):
        with torch.cuda.stream(s1):
            a = tokens.sample(x, u, 0.9, 0, 0.9, 0.0)
        with torch.cuda.stream(s2):
            b = tokens.sample(x, u, 0.9, 50, 0.95, 0.0)
        got.append((a, b))
    torch.cuda.synchronize()
    for pair in got:
        for g, w in zip(pair, want):
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tokens.sample(x, u, 0.9, 50, 0.95, 0.0)
    x.copy_(torch.roll(x, 1, 0))
    u.copy_(torch.roll(u, 1, 0))
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0], torch.roll(want[1][0], 1)) and torch.equal(out[1], torch.roll(want[1][1], 1))


def test_more_than_2_31_logits():
    n, v = 16500, 131072
    x = torch.empty(n, v, device="cuda", dtype=BF16)
    tail, u = _logits(3, v, BF16, 12)
    x[:-3] = 0
    x[:, 5] = 30.0
    x[-3:] = tail
    us = torch.full((n,), 0.5, device="cuda")
    us[-3:] = u
    token, logp = tokens.sample(x, us, 1.0, 0, 0.9)
    want = tokens.sample(tail, u, 1.0, 0, 0.9)
    assert torch.equal(token[-3:], want[0]) and torch.equal(logp[-3:], want[1])
    assert (token[:-3] == 5).all()


def test_refusals():
    x, u = _logits(4, 64, F32, 1)
    k = torch.ones(4, dtype=torch.int64, device="cuda")
    for call in (lambda: tokens.sample(x.half(), u), lambda: tokens.sample(x, u[:3]), lambda: tokens.sample(x, u.double()),
                 lambda: tokens.sample(x, u, -1.0), lambda: tokens.sample(x, u, math.nan), lambda: tokens.sample(x, u, math.inf),
                 lambda: tokens.sample(x, u, 1.0, -1), lambda: tokens.sample(x, u, 1.0, 1.5), lambda: tokens.sample(x, u, 1.0, k),
                 lambda: tokens.sample(x, u, 1.0, 0, math.nan), lambda: tokens.sample(x, u, 1.0, 0, 1.0, math.nan),
                 lambda: tokens.sample(x, u, "warm"), lambda: tokens.sample(x.t(), u), lambda: tokens.sample(x[0], u),
                 lambda: tokens.sample(x.cpu(), u), lambda: tokens.sample(x, u.cpu()), lambda: tokens.sample(x[:, :0], u),
                 lambda: tokens.sample(torch.empty(1, 262145, device="cuda"), u[:1])):
        with pytest.raises(plb.PufferError):
            call()
    token, logp = tokens.sample(x[:0], u[:0])
    assert token.numel() == logp.numel() == 0
