"""The host side of drawing tokens, of the norms around a block and of the gated delta rule: entries are bound, check their
arguments before they look for a device, plan workspaces that hold what they say, and the calls refuse CPU tensors."""
import ctypes

import pytest

import pufferlean_b200 as plb

torch = pytest.importorskip("torch")
from pufferlean_b200 import tokens  # noqa: E402

INVALID, NO_DEVICE = -1, -6
P = 1 << 12  # never read: every call below fails before a launch


@pytest.fixture(scope="module")
def L():
    return plb.lib()


def _shape(**more):
    d = dict(tokens=100, sequences=2, heads_k=2, heads_v=4, dk=64, dv=64, q_token=128, q_head=64, k_token=128, k_head=64,
             v_token=256, v_head=64, scale=0.125)
    d.update(more)
    return plb.DeltaShape(**d)


def test_entries_are_bound(L):
    for name in ("pl_sample_dev", "pl_block_norm_dev", "pl_block_norm_grad_ws", "pl_block_norm_grad_dev", "pl_delta_ws",
                 "pl_delta_saved", "pl_delta_dev", "pl_delta_grad_dev", "pl_delta_step_dev"):
        assert getattr(L, name).argtypes is not None


def test_sample_arguments(L):
    def call(logits=P, ld=64, rows=4, v=64, temp=1.0, k=0, p=1.0, min_p=0.0, u=P, token=P, logp=P):
        return L.pl_sample_dev(logits, ld, rows, v, 1, u, None, temp, None, k, None, p, None, min_p, token, logp, None)

    nan = float("nan")
    for bad in (dict(v=0), dict(v=65), dict(ld=300000, v=262145), dict(temp=-1.0), dict(temp=nan), dict(temp=float("inf")),
                dict(p=nan), dict(min_p=nan), dict(logits=None), dict(u=None), dict(token=None), dict(logp=None),
                dict(logits=P + 1), dict(rows=1 << 28)):
        assert call(**bad) == INVALID, bad
        assert L.pl_last_error()
    assert call(rows=0) == 0
    assert call(rows=0, temp=1e31) == 0 and call(rows=0, temp=1e-310) == 0  # count as the largest and the least
    if plb.device_count() == 0:
        assert call() == NO_DEVICE


def test_block_arguments(L):
    def fwd(x=P, ldx=16, branch=P, gate=None, ldg=0, eps=1e-5, post=1, rows=4, cols=16, r=P, ldr=16, rb=P, rstd=P):
        return L.pl_block_norm_dev(x, ldx, branch, 16, gate, ldg, None, None, 1.0, eps, post, rows, cols, 1, r, ldr, P, 16, rb,
                                   rstd, None)

    def bwd(dr=P, lddr=16, dy=P, gate=None, ldg=0, dg=None, lddg=0, rows=4, cols=16, dx=P, dw=P, ws=P, size=1 << 20):
        return L.pl_block_norm_grad_dev(dr, lddr, dy, 16, P, 16, gate, ldg, P, 16, P, P, None, None, 1.0, rows, cols, 1, dx, 16,
                                        P, 16, dg, lddg, dw, dw, ws, size, None)

    for bad in (dict(ldx=8), dict(cols=0), dict(x=None), dict(branch=None), dict(gate=P, ldg=8), dict(eps=float("nan")),
                dict(rb=None), dict(rstd=None), dict(r=None), dict(ldr=15), dict(rows=1 << 31)):
        assert fwd(**bad) == INVALID, bad
    assert fwd(rows=0) == 0
    if plb.device_count() == 0:
        assert fwd(rb=None, post=0) == NO_DEVICE
        assert bwd() == NO_DEVICE  # the device is looked for before a workspace's size
    for bad in (dict(lddr=8), dict(cols=0), dict(gate=P, ldg=16, dg=P, lddg=8), dict(rows=1 << 31)):
        assert bwd(**bad) == INVALID, bad
    assert L.pl_block_norm_grad_ws(1, 64) == 2 * 64 * 4
    assert L.pl_block_norm_grad_ws(1 << 20, 64) == L.pl_block_norm_grad_ws(1 << 19, 64)
    assert L.pl_block_norm_grad_ws(1000, 20000) == (64 * 2 * 20000 + 1000) * 4  # wide rows keep a number each


def test_delta_arguments(L):
    big = 1 << 40

    def fwd(s, q=P, o=P, final=P, saved=None, saved_bytes=0, ws=P, size=big, offsets=P):
        return L.pl_delta_dev(ctypes.byref(s), q, P, P, P, P, offsets, None, o, final, saved, saved_bytes, ws, size, None)

    def bwd(s, saved=P, saved_bytes=big, ws=P, size=big, dq=P):
        return L.pl_delta_grad_dev(ctypes.byref(s), P, 256, 64, None, P, P, P, P, P, P, saved, saved_bytes, dq, P, P, P, P, P,
                                   ws, size, None)

    for bad in (dict(dk=0), dict(dk=129), dict(dv=0), dict(dv=1025), dict(heads_k=0), dict(heads_v=5), dict(heads_v=1),
                dict(tokens=1 << 30), dict(sequences=65536), dict(sequences=0), dict(scale=float("nan"))):
        assert fwd(_shape(**bad)) == INVALID, bad
        assert bwd(_shape(**bad)) == INVALID, bad
    s = _shape()
    need, saved = L.pl_delta_ws(ctypes.byref(s), 0), L.pl_delta_saved(ctypes.byref(s))
    for bad in (dict(q=None), dict(o=None), dict(final=None), dict(ws=None), dict(ws=P + 16), dict(size=need - 1),
                dict(saved=P, saved_bytes=saved - 1), dict(saved=P + 8, saved_bytes=big)):
        assert fwd(s, **bad) == INVALID, bad
    assert fwd(_shape(tokens=101), offsets=None) == INVALID  # not two sequences of one length
    for bad in (dict(saved=None), dict(saved_bytes=saved - 1), dict(size=L.pl_delta_ws(ctypes.byref(s), 1) - 1), dict(dq=None)):
        assert bwd(s, **bad) == INVALID, bad
    assert L.pl_delta_dev(None, P, P, P, P, P, P, None, P, P, None, 0, P, big, None) == INVALID
    if plb.device_count() == 0:
        assert fwd(s) == bwd(s) == NO_DEVICE
        assert L.pl_delta_step_dev(ctypes.byref(s), P, P, P, P, P, P, P, P, None) == NO_DEVICE
    assert L.pl_delta_step_dev(ctypes.byref(s), P, P, P, P, P, None, P, P, None) == INVALID
    assert fwd(_shape(tokens=0, sequences=0)) == 0


def test_delta_workspaces(L):
    """Chunks never share a slot and all slots fit, whatever the lengths."""
    g = torch.Generator().manual_seed(0)
    for _ in range(200):
        n = int(torch.randint(1, 12, (1,), generator=g))
        lengths = [int(x) for x in torch.randint(0, 200, (n,), generator=g)]
        front = int(torch.randint(0, 70, (1,), generator=g))
        total = front + sum(lengths) + int(torch.randint(0, 70, (1,), generator=g))
        seen, at = set(), front
        for s, length in enumerate(lengths):
            for c in range(-(-length // 64)):
                slot = at // 64 + s + c
                assert slot not in seen and slot < total // 64 + n
                seen.add(slot)
            at += length
        s = _shape(tokens=total, sequences=n)
        slots = total // 64 + n
        assert L.pl_delta_saved(ctypes.byref(s)) >= slots * 4 * (64 * 64 + 64 * 64) * 4
        assert L.pl_delta_ws(ctypes.byref(s), 1) > L.pl_delta_ws(ctypes.byref(s), 0)


def test_cpu_tensors_are_refused():
    x, u = torch.zeros(4, 16), torch.zeros(4)
    q, g, st = torch.zeros(4, 2, 16, dtype=torch.bfloat16), torch.zeros(4, 2), torch.zeros(4, 2, 16, 16)
    for call in (lambda: tokens.sample(x, u), lambda: tokens.block_norm(x, x), lambda: tokens.sample([1.0], u),
                 lambda: tokens.block_norm_grad(x, x, x, None, x, u, u), lambda: tokens.delta_rule(q, q, q, g, g),
                 lambda: tokens.delta_rule_grad(q, None, q, q, q, g, g, None, None),
                 lambda: tokens.delta_rule_grad(q, None, q, q, q, g, g, None, (u, 1)),
                 lambda: tokens.delta_rule_step(q, q, q, g, g, st)):
        with pytest.raises(plb.PufferError):
            call()
