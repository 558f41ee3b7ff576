"""Edges of the token-policy operators: logits that a mask or a constant makes equal over the whole vocabulary, a process
that uses them on two devices, calls from two threads, a process whose first call is captured, device
waits that ran out, inputs that require gradients, and matrices of more than 2^31 elements.
Tolerances as in test_gpu_tokens.py."""
import ctypes as C
import math
import os
import subprocess
import sys
import threading

import pytest

torch = pytest.importorskip("torch")

import pufferlean_b200 as plb  # noqa: E402
from pufferlean_b200 import tokens  # noqa: E402
from .test_gpu_tokens import (B, BF16, F2, F64, H, _answers, _close, _gen, _head_case, _head_ref, _head_tol,  # noqa: E402
                              _norm_grad_ref, _randn)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


# ------------------------------------------------------------------------------------------------ equal logits
def _check_flat(x, w, b, ids, teacher, T, scale, logit):
    """Every logit of row n is logit[n], exactly, so q = 1 / V however large it is. What is left of _check_head's bounds
    is without the logits' own error. (logsumexp would lose log V beside a large logit in 64 bits too.)"""
    N, V = len(x), w.shape[0]
    if teacher is None:
        loss, lse, dx, dw, db = tokens.vocab_ce_grad(x, w, ids, b, scale)
    else:
        loss, lse, dx, dw, db = tokens.vocab_distill_grad(x, w, ids, teacher, b, T, scale)
    want, ent, has = _answers(ids, teacher, V, T)
    log_v = math.log(V)
    _close(loss, torch.where(has, ent + log_v, 0.0), 2.0 ** -20 * (1 + log_v + ent.abs()), "loss")
    u = logit / T
    if float(u.abs().max()) < 6e37:  # above, a bias counts as 1e38 in units of log 2
        _close(lse, torch.where(has, u + log_v, 0.0), 2.0 ** -21 * (1 + log_v + u.abs()), "lse")
    s = torch.where(has, scale.double() / T, 0.0)[:, None]
    dz = s * (1.0 / V - want)
    off = (B + H) * dz.abs() + (H + 2.0 ** -18) * s.abs() / V + 2.0 ** -18 * dz.abs()
    xd = torch.where(has[:, None], x.double(), 0.0)
    wa, xa = w.double().abs(), xd.abs()
    dxr, dwr = dz @ w.double(), dz.t() @ xd
    _close(dx, dxr, off @ wa + (V / 16 + 200) * F2 * (dz.abs() @ wa) + B * 1.01 * dxr.abs() + 1e-30, "dx")
    _close(dw, dwr, off.t() @ xa + (N / 16 + 200) * F2 * (dz.abs().t() @ xa) + B * 1.01 * dwr.abs() + 1e-30, "dw")
    if b is not None:
        dbr = dz.sum(0)
        _close(db, dbr, off.sum(0) + (N + 200) * F2 * dz.abs().sum(0) + B * 1.01 * dbr.abs() + 1e-30, "dbias")


@pytest.mark.parametrize("value", [torch.finfo(BF16).min, -1e30, -2.0 ** 29, -1.5 * 2.0 ** 26, -1.25 * 2.0 ** 23, 2.0 ** 25,
                                   -1e4, 0.0])
@pytest.mark.parametrize("K,T", [(0, 1.0), (3, 2.0)])
@pytest.mark.parametrize("N,V", [(20, 1500), (300, 1500), (140, 19100)])
def test_whole_vocabulary_masked(N, V, K, T, value):
    """One finite bias on every token (a mask that leaves a row nothing): the softmax is uniform, as in plain f32. The
    hidden states and the weights share no column, so that the bias is all there is to a logit."""
    x, w, b, ids, teacher, scale = _head_case(_gen(N + V + K), N, V, 64, K, True, 0, 0)
    x[:, 32:] = 0
    w[:, :32] = 0
    b[:] = value
    _check_flat(x, w, b, ids, teacher, T, scale, torch.full((N,), float(b[0]), dtype=F64, device="cuda"))


@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** 24, 1.5 * 2.0 ** 27, 2.0 ** 60])
@pytest.mark.parametrize("N,V", [(20, 1500), (300, 19100)])
def test_equal_large_logits(N, V, size):
    """The same from the product: every token has one large logit."""
    g = _gen(N + V)
    x, w, _, ids, _, scale = _head_case(g, N, V, 64, 0, False, 0, 0)
    x[:, 32:] = 0
    w[:, :32] = 0
    x[:, 0] = torch.where(torch.rand(N, generator=g, device="cuda") < 0.5, -1.0, 1.0).to(BF16)
    w[:, 0] = size
    _check_flat(x, w, None, ids, None, 1.0, scale, x[:, 0].double() * size)


# ------------------------------------------------------------------------------------------------ devices
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")
def test_two_devices():
    """One process, one device after the other: the same bits on both."""
    x, w, b, ids, _, scale = _head_case(_gen(3), 300, 3000, 128, 0, True, 0, 0)
    one = tokens.vocab_ce_grad(x, w, ids, b, scale)
    two = tokens.vocab_ce_grad(*(t.to("cuda:1") for t in (x, w, ids, b, scale)))
    for p, q in zip(one, two):
        assert torch.equal(p, q.to("cuda:0"))


@pytest.mark.parametrize("device", range(max(1, min(2, torch.cuda.device_count()))))
def test_the_librarys_device_stays(device):
    """The device that the caller gave the library is still the library's after a call on cuda:0 tensors, and torch's is
    still torch's."""
    L, now = plb.lib(), C.c_int()
    x = torch.ones(4, 64, device="cuda:0")
    before = torch.cuda.current_device()
    assert L.pl_set_device(device) == 0
    try:
        tokens.layer_norm(x)
        assert L.pl_get_device(C.byref(now)) == 0 and now.value == device
    finally:
        assert L.pl_set_device(before) == 0
    assert torch.cuda.current_device() == before


# ------------------------------------------------------------------------------------------------ threads
class _DistillCall:
    """A distillation with gradients through the C entry, with buffers and a stream of its own. With these sizes the
    kernel from terms to gradients takes 53,248 bytes of shared memory at K = 64 and 51,200 at K = 20."""
    N, V, D = 4096, 5000, 8

    def __init__(self, K):
        self.K = K
        self.x, self.w, self.b, self.ids, self.teacher, _ = _head_case(_gen(K), self.N, self.V, self.D, K, True, 0, 0)
        self.size = plb.lib().pl_vocab_ws(self.N, self.V, self.D, K, 1, 1, 0, 0)
        self.ws = torch.empty(self.size, dtype=torch.uint8, device="cuda")
        self.out = [torch.empty(s, dtype=t, device="cuda") for s, t in
                    ((self.N, torch.float32), (self.N, torch.float32), ((self.N, self.D), BF16), ((self.V, self.D), BF16),
                     (self.V, BF16))]
        self.stream = torch.cuda.Stream()

    def __call__(self):
        loss, lse, dx, dw, db = (t.data_ptr() for t in self.out)
        return plb.lib().pl_vocab_distill_grad_dev(
            self.x.data_ptr(), self.D, self.w.data_ptr(), self.D, self.b.data_ptr(), self.ids.data_ptr(),
            self.teacher.data_ptr(), self.K, 1.0, None, self.N, self.V, self.D, loss, lse, dx, self.D, dw, self.D, db, 0, 0,
            self.ws.data_ptr(), self.size, self.stream.cuda_stream)


def test_two_threads():
    """Calls of one kernel with different needs from two threads: every launch is accepted, the bits are one thread's."""
    calls = [_DistillCall(64), _DistillCall(20)]
    torch.cuda.synchronize()
    limit = C.c_int()
    want = []
    for c in calls:
        assert c() == 0, plb.lib().pl_last_error()
        torch.cuda.synchronize()
        want.append([t.clone() for t in c.out])
        # what was allowed for the first call still is after the second, smaller one
        assert plb.lib().pl_test_vocab_dz_smem(C.byref(limit)) == 0 and limit.value >= 53248
    failed = []

    def go(c):
        for _ in range(200):
            if c():
                failed.append(plb.lib().pl_last_error())

    threads = [threading.Thread(target=go, args=(c,)) for c in calls]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    assert not failed
    for c, w in zip(calls, want):
        assert all(torch.equal(p, q) for p, q in zip(c.out, w))


# ------------------------------------------------------------------------------------------------ capture
FIRST_CALL = """
import sys
import torch
from pufferlean_b200 import tokens

g = torch.Generator(device="cuda").manual_seed(1)
x = torch.randn(300, 64, generator=g, device="cuda").to(torch.bfloat16)
w = torch.randn(2000, 64, generator=g, device="cuda").to(torch.bfloat16)
b = torch.randn(2000, generator=g, device="cuda").to(torch.bfloat16)
ids = torch.randint(0, 2000, (300, 5), generator=g, device="cuda").to(torch.int32)
teacher = torch.randn(300, 5, generator=g, device="cuda")
gain = torch.ones(64, device="cuda")


def step():
    y, m, r = tokens.layer_norm(x, gain)
    if sys.argv[1] == "ce":
        out = tokens.vocab_ce_grad(y, w, ids[:, 0].contiguous(), b)
    else:
        out = tokens.vocab_distill_grad(y, w, ids, teacher, b, 2.0)
    return out + tokens.layer_norm_grad(out[2], x, gain, m, r)


torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
for t in got:
    t.zero_()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(p, q) for p, q in zip(got, step()))
print("same bits")
"""


@pytest.mark.parametrize("which", ["ce", "distill"])
def test_first_call_can_be_captured(which):
    """A process whose first calls of all are made under capture: nothing has to be run before."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    p = subprocess.run([sys.executable, "-c", FIRST_CALL, which], capture_output=True, text=True, timeout=300, cwd=root,
                       env=dict(os.environ, PYTHONPATH=root))
    assert p.returncode == 0 and "same bits" in p.stdout, p.stderr[-2000:]


# ------------------------------------------------------------------------------------------------ waits that ran out
@pytest.mark.parametrize("K", [0, 3])
@pytest.mark.parametrize("N", [40, 300])
def test_wait_that_ran_out_is_seen(N, K):
    """A recorded timeout (written from the host) makes the losses and gradients NaN until check() has reported it; then
    the calls are what they were."""
    x, w, b, ids, teacher, scale = _head_case(_gen(N + K), N, 700, 64, K, True, 0, 0)
    has = (ids >= 0) if K == 0 else ((ids >= 0) & (teacher > -math.inf)).any(1)

    def call():
        if K == 0:
            return (tokens.vocab_ce(x, w, ids, b)[0],) + tokens.vocab_ce_grad(x, w, ids, b, scale)
        return (tokens.vocab_distill(x, w, ids, teacher, b)[0],) + tokens.vocab_distill_grad(x, w, ids, teacher, b, 1.0, scale)

    tokens.check()
    want = call()
    assert plb.lib().pl_test_set_device_error(0x103) == 0
    try:
        bad, loss, _, dx, dw, db = call()
        for t in (bad, loss):
            assert torch.isnan(t[has]).all() and not t[~has].any()
        assert torch.isnan(dx[has].float()).all() and not dx[~has].any()
        assert torch.isnan(dw.float()).all() and torch.isnan(db.float()).all()
    finally:
        with pytest.raises(plb.PufferError, match="ran out"):
            tokens.check()
    tokens.check()
    for device in (0, "cuda", torch.device("cuda", 0)):
        tokens.check(device)
    assert all(torch.equal(p, q) for p, q in zip(want, call()))


def test_check_waits_for_every_stream():
    """A record that a stream of its own has yet to write is seen. (The write comes after work of some milliseconds.)"""
    a = torch.ones(8192, 8192, device="cuda")
    tokens.check()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(10):
            a @ a
        done = torch.cuda.Event()
        done.record()
    tokens.check()
    assert done.query()


def test_check_refuses():
    for device in ("cpu", torch.cuda.device_count(), -1):
        with pytest.raises((plb.PufferError, RuntimeError)):
            tokens.check(device)


# ------------------------------------------------------------------------------------------------ autograd
def test_results_carry_no_graph():
    """Parameters that require a gradient are taken as they are; nothing that comes back does, and the bits are the same."""
    x, w, b, ids, teacher, scale = _head_case(_gen(17), 70, 300, 64, 3, True, 0, 0)
    gain = torch.ones(64, device="cuda")

    def calls():
        y, m, r = tokens.layer_norm(x, gain)
        return ((y, m, r) + tokens.layer_norm_grad(x, x, gain, m, r) + tokens.vocab_ce(x, w, ids[:, 0].contiguous(), b)
                + tokens.vocab_ce_grad(x, w, ids[:, 0].contiguous(), b, scale) + tokens.vocab_distill(x, w, ids, teacher, b)
                + tokens.vocab_distill_grad(x, w, ids, teacher, b, 1.0, scale))

    want = calls()
    x, w, b, gain = (t.detach().requires_grad_() for t in (x, w, b, gain))
    got = calls()
    assert not any(t.requires_grad for t in got)
    assert all(torch.equal(p, q) for p, q in zip(want, got))


# ------------------------------------------------------------------------------------------------ past 32 bits
@pytest.mark.parametrize("piece_bytes,rows", [(6 << 30, (0, 5, 8191, 16375, 16376, 16377, 16400, 16497, 16499)),
                                              (0, (0, 5, 8191, 8318, 8319, 8320, 8321, 16497, 16499))])
def test_vocab_terms_past_32_bits(piece_bytes, rows):
    """16,500 rows of terms, 131,136 apart: 2^31 elements end inside row 16,376 when one piece holds them all; by the
    default bound there are two pieces, of 8,320 rows and the rest. Rows on both sides of either border, and the
    gradients of a few tokens, which sum over all rows."""
    g = _gen(98)
    N, V, D = 16500, 131100, 64
    x, w = _randn(g, N, D).to(BF16), (_randn(g, V, D) * 0.2).to(BF16)
    b = (0.3 * _randn(g, V)).to(BF16)
    t = torch.randint(0, V, (N,), generator=g, device="cuda").to(torch.int32)
    cols = torch.tensor([0, 1, 77777, V - 1], device="cuda")
    rows = torch.tensor(rows, device="cuda")
    t[rows] = cols.repeat(3)[:len(rows)].to(torch.int32)  # their answers lie in the columns that are looked at
    scale = torch.ones(N, device="cuda")
    scale[rows] = 64.0  # one of these rows in the wrong place stands out of a sum over all
    loss, lse, dx, dw, db = tokens.vocab_ce_grad(x, w, t, b, scale, False, piece_bytes)
    xs, ts = x[rows], t[rows]
    ref = _head_ref(xs, w, b, ts, None, 1.0, scale[rows])
    tol_z, tol_loss = _head_tol(ref, xs, w, b, ts, 1.0)
    _close(loss[rows], ref["loss"], tol_loss, "loss")
    _close(lse[rows], ref["lse"], tol_loss, "lse")
    off = (B + H) * ref["dz"].abs() + (H + 4 * tol_z[:, None] + 2.0 ** -18) * ref["s"].abs() * ref["q"] \
        + 2.0 ** -18 * ref["dz"].abs()
    wa = w.double().abs()
    dxr = ref["dz"] @ w.double()
    _close(dx[rows], dxr, off @ wa + (V / 16 + 200) * F2 * (ref["dz"].abs() @ wa) + B * 1.01 * dxr.abs(), "dx")
    sd = scale.double()[:, None]
    lse64 = torch.empty(N, dtype=F64, device="cuda")
    for r in range(0, N, 500):
        lse64[r:r + 500] = torch.logsumexp(x[r:r + 500].double() @ w.double().t() + b.double(), 1)
    _close(lse, lse64, 2.0 ** -16 * (1 + lse64.abs()), "lse of every row")
    q = torch.exp(x.double() @ w[cols].double().t() + b[cols].double() - lse64[:, None])
    dz = sd * (q - (t[:, None] == cols[None]).double())
    xa = x.double().abs()
    off = (B + H) * dz.abs() + (H + 2.0 ** -15) * sd * q
    dwr, dbr = dz.t() @ x.double(), dz.sum(0)
    _close(dw[cols], dwr, off.t() @ xa + (N / 16 + 200) * F2 * (dz.abs().t() @ xa) + B * 1.01 * dwr.abs(), "dw")
    _close(db[cols], dbr, off.sum(0) + (N + 200) * F2 * dz.abs().sum(0) + B * 1.01 * dbr.abs(), "dbias")


def test_layer_norm_sums_past_32_bits():
    """The parameters' gradients sum over rows on both sides of element 2^31 (row 131,072); the rows there weigh a
    thousandfold, so that one left out or taken twice stands out."""
    rows, cols = 140000, 16384
    x = torch.empty(rows, cols, dtype=BF16, device="cuda")
    x.normal_(generator=_gen(3))
    y, m, r = tokens.layer_norm(x)
    y[131070:131075] *= 1000
    y[-1] *= 1000
    dx, dw, db = tokens.layer_norm_grad(y, x, None, m, r)
    at = torch.tensor([0, 1, 8191, 8192, cols - 1], device="cuda")
    xh = (x[:, at].double() - m.double()[:, None]) * r.double()[:, None]
    dy = y[:, at].double()
    n = rows / 148 + 64  # a block's rows one after the other, then the blocks' sums
    off_xh = F2 * (x[:, at].double().abs() + m.double()[:, None].abs()) * r.double()[:, None]
    _close(dw[at], (dy * xh).sum(0), n * F2 * (dy.abs() * xh.abs()).sum(0) + (dy.abs() * off_xh).sum(0), "dw")
    _close(db[at], dy.sum(0), n * F2 * dy.abs().sum(0), "db")
    some = torch.tensor([131071, 131072, 131074, rows - 1], device="cuda")
    dxr, _, _, xh, gg = _norm_grad_ref(y[some], x[some], None, m[some], r[some])
    size = gg.abs() + gg.abs().mean(1, keepdim=True) + xh.abs() * (gg * xh).abs().mean(1, keepdim=True)
    _close(dx[some], dxr, B * dxr.abs() + 2.0 ** -16 * r[some].double()[:, None] * size, "dx")
