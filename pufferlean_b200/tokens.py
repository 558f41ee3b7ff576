"""Operators of a token policy on CUDA tensors: layer norm, the large-vocabulary head's cross entropy, and
distillation of a teacher's top logits into the head, each forward and with its gradients.

A policy whose actions are tokens ends in a layer norm and a head of V outputs, V in the tens of thousands (the
update paths of this package stop at 128). These calls take torch tensors as they lie (rows may be strided, the last
dimension contiguous), enqueue on torch's current stream and return new tensors; workspaces come from torch's
allocator, so calls on several streams do not share any. The C entry points behind them are declared in
include/pufferlean_b200.h (pl_layernorm_dev, pl_vocab_ce_dev, ...). There is no CPU fallback.

    y, mean, rstd = layer_norm(x, weight, bias)
    loss, lse, dy, dw, db = vocab_ce_grad(y2d, head, target, head_bias, row_scale)
    dx, dweight, dbias = layer_norm_grad(dy, x, weight, mean, rstd)

Gradients are of sum_n row_scale_n * loss_n (descent).
"""
from __future__ import annotations

import torch

from . import PufferError, _check, lib

_BF16, _F32, _I32 = torch.bfloat16, torch.float32, torch.int32


def _need(ok, what, msg, *args):
    if not ok:
        raise PufferError(f"{what}: " + msg % args if args else f"{what}: {msg}")


def _matrix(t, what, name, dtypes, device=None):
    """Checks a 2-D tensor of contiguous rows on the GPU; returns its row stride in elements."""
    _need(isinstance(t, torch.Tensor) and t.is_cuda, what, "%s must be a CUDA tensor", name)
    _need(t.dim() == 2, what, "%s must have two dimensions, has %d", name, t.dim())
    _need(t.dtype in dtypes, what, "%s has type %s", name, t.dtype)
    _need(device is None or t.device == device, what, "%s is on %s, not on %s", name, t.device, device)
    rows, cols = t.shape
    st, sc = t.stride()
    _need(cols <= 1 or sc == 1, what, "%s: the values of a row must be contiguous (stride %d)", name, sc)
    if rows <= 1:
        return max(cols, st) if st >= cols else cols
    _need(st >= cols, what, "%s: row stride %d below %d columns", name, st, cols)
    return st


def _vector(t, what, name, dtype, shape, device):
    """Checks a contiguous tensor of this type and shape (or None); returns its address."""
    if t is None:
        return None
    _need(isinstance(t, torch.Tensor) and t.device == device, what, "%s must be a tensor on %s", name, device)
    _need(t.dtype == dtype, what, "%s has type %s, not %s", name, t.dtype, dtype)
    _need(tuple(t.shape) == tuple(shape), what, "%s has shape %s, not %s", name, tuple(t.shape), tuple(shape))
    _need(t.is_contiguous(), what, "%s must be contiguous", name)
    return t.data_ptr()


class _On:
    """Makes a tensor's device current for torch and for the library, and names its current stream."""

    __slots__ = ("guard", "index")

    def __init__(self, device):
        self.index = device.index
        self.guard = None if self.index == torch.cuda.current_device() else torch.cuda.device(device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        _check(lib().pl_set_device(self.index), "pl_set_device")
        return torch.cuda.current_stream(self.index).cuda_stream

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)
            lib().pl_set_device(torch.cuda.current_device())
        return False


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(y, mean, rstd) of the rows of x [rows, cols] (f32 or bf16); weight and bias [cols] f32 or None, mean and rstd
    [rows] f32 (what layer_norm_grad takes)."""
    what = "layer_norm"
    ldx = _matrix(x, what, "x", (_F32, _BF16))
    rows, cols = x.shape
    wp = _vector(weight, what, "weight", _F32, (cols,), x.device)
    bp = _vector(bias, what, "bias", _F32, (cols,), x.device)
    with _On(x.device) as st:
        y = torch.empty((rows, cols), dtype=x.dtype, device=x.device)
        stats = torch.empty((2, rows), dtype=_F32, device=x.device)
        at = stats.data_ptr()
        _check(lib().pl_layernorm_dev(x.data_ptr(), ldx, wp, bp, rows, cols, eps, x.dtype == _BF16, y.data_ptr(), cols,
                                      at, at + 4 * rows, st), "pl_layernorm_dev")
    return y, stats[0], stats[1]


def layer_norm_grad(dy, x, weight, mean, rstd, params=True):
    """(dx, dweight, dbias) of layer_norm: dx in x's type, dweight and dbias [cols] f32 (None with params=False)."""
    what = "layer_norm_grad"
    ldx = _matrix(x, what, "x", (_F32, _BF16))
    rows, cols = x.shape
    lddy = _matrix(dy, what, "dy", (x.dtype,), x.device)
    _need(dy.shape == x.shape, what, "dy has shape %s, not %s", tuple(dy.shape), tuple(x.shape))
    wp = _vector(weight, what, "weight", _F32, (cols,), x.device)
    mp = _vector(mean, what, "mean", _F32, (rows,), x.device)
    rp = _vector(rstd, what, "rstd", _F32, (rows,), x.device)
    _need(mp is not None and rp is not None, what, "mean and rstd are needed")
    with _On(x.device) as st:
        L = lib()
        dx = torch.empty((rows, cols), dtype=x.dtype, device=x.device)
        dp = ws = None
        size = 0
        if params:
            dp = torch.empty((2, cols), dtype=_F32, device=x.device)
            size = L.pl_layernorm_grad_ws(rows, cols)
            ws = torch.empty(size, dtype=torch.uint8, device=x.device)
        _check(L.pl_layernorm_grad_dev(dy.data_ptr(), lddy, x.data_ptr(), ldx, wp, mp, rp, rows, cols, x.dtype == _BF16,
                                       dx.data_ptr(), cols, dp[0].data_ptr() if params else None,
                                       dp[1].data_ptr() if params else None, ws.data_ptr() if params else None, size,
                                       st), "pl_layernorm_grad_dev")
    return (dx, dp[0], dp[1]) if params else (dx, None, None)


def _head(what, x, w, bias, ids, teacher, temperature, row_scale, grad, dw_f32=False, piece_bytes=0):
    ldx = _matrix(x, what, "x", (_BF16,))
    dev = x.device
    ldw = _matrix(w, what, "w", (_BF16,), dev)
    n, d = x.shape
    v = w.shape[0]
    _need(w.shape[1] == d, what, "w has %d columns, x has %d", w.shape[1], d)
    _need(v > 0 and d > 0, what, "w has shape %s", tuple(w.shape))
    bp = _vector(bias, what, "bias", _BF16, (v,), dev)
    distill = teacher is not None
    if distill:
        _need(isinstance(ids, torch.Tensor) and ids.dim() == 2 and ids.shape[1] > 0, what,
              "ids must have shape (%d, K) with K > 0", n)
        k = ids.shape[1]
        ip = _vector(ids, what, "ids", _I32, (n, k), dev)
        tp = _vector(teacher, what, "teacher", _F32, (n, k), dev)
        _need(temperature > 0.0, what, "temperature %g", temperature)
    else:
        k = 0
        _need(ids is not None, what, "target is needed")
        ip = _vector(ids, what, "target", _I32, (n,), dev)
    sp = _vector(row_scale, what, "row_scale", _F32, (n,), dev)
    with _On(dev) as st:
        L = lib()
        aligned = ldx % 8 == 0 and ldw % 8 == 0 and x.data_ptr() % 16 == 0 and w.data_ptr() % 16 == 0
        size = L.pl_vocab_ws(n, v, d, k, bias is not None, grad, aligned, piece_bytes)
        out = torch.empty((2, n), dtype=_F32, device=dev)
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        lp, wsp = out.data_ptr(), ws.data_ptr()
        if not grad:
            if distill:
                rc = L.pl_vocab_distill_dev(x.data_ptr(), ldx, w.data_ptr(), ldw, bp, ip, tp, k, temperature, n, v, d, lp,
                                            lp + 4 * n, wsp, size, st)
            else:
                rc = L.pl_vocab_ce_dev(x.data_ptr(), ldx, w.data_ptr(), ldw, bp, ip, n, v, d, lp, lp + 4 * n, wsp, size, st)
            _check(rc, what)
            return out[0], out[1]
        dx = torch.empty((n, d), dtype=_BF16, device=dev)
        dw = torch.empty((v, d), dtype=_F32 if dw_f32 else _BF16, device=dev)
        db = torch.empty(v, dtype=dw.dtype, device=dev) if bias is not None else None
        tail = (sp, n, v, d, lp, lp + 4 * n, dx.data_ptr(), d, dw.data_ptr(), d, None if db is None else db.data_ptr(),
                dw_f32, piece_bytes, wsp, size, st)
        if distill:
            rc = L.pl_vocab_distill_grad_dev(x.data_ptr(), ldx, w.data_ptr(), ldw, bp, ip, tp, k, temperature, *tail)
        else:
            rc = L.pl_vocab_ce_grad_dev(x.data_ptr(), ldx, w.data_ptr(), ldw, bp, ip, *tail)
        _check(rc, what)
    return out[0], out[1], dx, dw, db


def vocab_ce(x, w, target, bias=None):
    """(loss, lse) [N] f32 of the head z = x w^T + bias against target [N] int32: loss = lse - z[target], the negative
    log-probability. x [N, D], w [V, D], bias [V] bf16. A negative target leaves its row out (loss = lse = 0); one past
    the vocabulary makes the row's loss NaN."""
    return _head("vocab_ce", x, w, bias, target, None, 1.0, None, False)


def vocab_ce_grad(x, w, target, bias=None, row_scale=None, dw_f32=False, piece_bytes=0):
    """(loss, lse, dx, dw, dbias) of sum_n row_scale_n loss_n: dx bf16, dw and dbias bf16 or (dw_f32) f32, dbias None
    without a bias. piece_bytes bounds the softmax terms held at a time (0: 4 GiB)."""
    return _head("vocab_ce_grad", x, w, bias, target, None, 1.0, row_scale, True, dw_f32, piece_bytes)


def vocab_distill(x, w, ids, teacher, bias=None, temperature=1.0):
    """(loss, lse) [N] f32 of the head's distribution q = softmax((x w^T + bias) / temperature) against the teacher's
    p = softmax(teacher / temperature) over its K top entries (ids, teacher [N, K]; a negative id or a logit of -inf is
    absent): loss = KL(p | q). A row without entries is left out (loss = lse = 0)."""
    _need(teacher is not None, "vocab_distill", "teacher is needed")
    return _head("vocab_distill", x, w, bias, ids, teacher, temperature, None, False)


def vocab_distill_grad(x, w, ids, teacher, bias=None, temperature=1.0, row_scale=None, dw_f32=False, piece_bytes=0):
    """(loss, lse, dx, dw, dbias) of sum_n row_scale_n loss_n, as vocab_ce_grad."""
    _need(teacher is not None, "vocab_distill_grad", "teacher is needed")
    return _head("vocab_distill_grad", x, w, bias, ids, teacher, temperature, row_scale, True, dw_f32, piece_bytes)
