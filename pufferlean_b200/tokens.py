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

import functools

import torch

from . import PufferError, _check, lib

_BF16, _F32, _I32 = torch.bfloat16, torch.float32, torch.int32
_NORM_TYPES = (_F32, _BF16)


def _need(ok, what, msg, *args):
    if not ok:
        raise PufferError(f"{what}: " + msg % args if args else f"{what}: {msg}")


def _matrix(t, what, name, dtypes, device=None):
    """Checks a 2-D tensor of contiguous rows on the GPU; returns its row stride in elements."""
    if isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in dtypes and t.dim() == 2 and (
            device is None or t.device == device):
        rows, cols = t.shape
        st, sc = t.stride()
        if sc == 1 and st >= cols:
            return st
        if cols <= 1 and rows <= 1:
            return 1
        if cols == 1 and st >= 1:  # a stride over one value says nothing
            return st
        if rows <= 1 and sc == 1:
            return cols
        raise PufferError(f"{what}: {name} must have contiguous rows that do not overlap (shape {(rows, cols)}, "
                          f"strides {(st, sc)})")
    _need(isinstance(t, torch.Tensor) and t.is_cuda, what, "%s must be a CUDA tensor", name)
    _need(t.dim() == 2, what, "%s must have two dimensions, has %d", name, t.dim())
    _need(t.dtype in dtypes, what, "%s has type %s", name, t.dtype)
    raise PufferError(f"{what}: {name} is on {t.device}, not on {device}")


def _vector(t, what, name, dtype, shape, device):
    """Checks a contiguous tensor of this type and shape; returns its address."""
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.device == device and t.is_contiguous():
        return t.data_ptr()
    _need(isinstance(t, torch.Tensor) and t.device == device, what, "%s must be a tensor on %s", name, device)
    _need(t.dtype == dtype, what, "%s has type %s, not %s", name, t.dtype, dtype)
    _need(tuple(t.shape) == tuple(shape), what, "%s has shape %s, not %s", name, tuple(t.shape), tuple(shape))
    raise PufferError(f"{what}: {name} must be contiguous")


@functools.lru_cache(maxsize=1024)
def _vocab_ws(n, v, d, k, bias, grad, aligned, piece_bytes):
    return lib().pl_vocab_ws(n, v, d, k, bias, grad, aligned, piece_bytes)


def _like(t):
    """A new contiguous tensor of t's shape and type."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _enter(device):
    """Makes a tensor's device the library's for this call; returns (torch's device to go back to or None, the stream
    torch is on there). The checks above and this run on every call: a small call costs little more than they do."""
    index = device.index
    was = torch.cuda.current_device()
    lib().pl_set_device(index)
    return (None if was == index else was), torch._C._cuda_getCurrentRawStream(index)


def _leave(was):
    if was is not None:
        lib().pl_set_device(was)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(y, mean, rstd) of the rows of x [rows, cols] (f32 or bf16); weight and bias [cols] f32 or None, mean and rstd
    [rows] f32 (what layer_norm_grad takes)."""
    what = "layer_norm"
    ldx = _matrix(x, what, "x", _NORM_TYPES)
    rows, cols = x.shape
    dev, dtype = x.device, x.dtype
    wp = None if weight is None else _vector(weight, what, "weight", _F32, (cols,), dev)
    bp = None if bias is None else _vector(bias, what, "bias", _F32, (cols,), dev)
    y = _like(x)
    mean = torch.empty(rows, dtype=_F32, device=dev)
    rstd = torch.empty_like(mean)
    was, st = _enter(dev)
    rc = lib().pl_layernorm_dev(x.data_ptr(), ldx, wp, bp, rows, cols, eps, dtype is _BF16, y.data_ptr(), cols,
                                mean.data_ptr(), rstd.data_ptr(), st)
    _leave(was)
    if rc:
        _check(rc, what)
    return y, mean, rstd


def layer_norm_grad(dy, x, weight, mean, rstd, params=True):
    """(dx, dweight, dbias) of layer_norm: dx in x's type, dweight and dbias [cols] f32 (None with params=False)."""
    what = "layer_norm_grad"
    ldx = _matrix(x, what, "x", _NORM_TYPES)
    rows, cols = x.shape
    dev, dtype = x.device, x.dtype
    lddy = _matrix(dy, what, "dy", (dtype,), dev)
    _need(dy.shape == x.shape, what, "dy has shape %s, not %s", tuple(dy.shape), tuple(x.shape))
    wp = None if weight is None else _vector(weight, what, "weight", _F32, (cols,), dev)
    _need(mean is not None and rstd is not None, what, "mean and rstd are needed")
    mp = _vector(mean, what, "mean", _F32, (rows,), dev)
    rp = _vector(rstd, what, "rstd", _F32, (rows,), dev)
    dx = _like(x)
    dw = db = dwp = dbp = wsp = None
    size = 0
    if params:
        dw = torch.empty(cols, dtype=_F32, device=dev)
        db = torch.empty_like(dw)
        size = lib().pl_layernorm_grad_ws(rows, cols)
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        dwp, dbp, wsp = dw.data_ptr(), db.data_ptr(), ws.data_ptr()
    was, st = _enter(dev)
    rc = lib().pl_layernorm_grad_dev(dy.data_ptr(), lddy, x.data_ptr(), ldx, wp, mp, rp, rows, cols, dtype is _BF16,
                                     dx.data_ptr(), cols, dwp, dbp, wsp, size, st)
    _leave(was)
    if rc:
        _check(rc, what)
    return dx, dw, db


def _head(what, x, w, bias, ids, teacher, temperature, row_scale, grad, dw_f32=False, piece_bytes=0):
    ldx = _matrix(x, what, "x", (_BF16,))
    dev = x.device
    ldw = _matrix(w, what, "w", (_BF16,), dev)
    n, d = x.shape
    v = w.shape[0]
    _need(w.shape[1] == d, what, "w has %d columns, x has %d", w.shape[1], d)
    _need(v > 0 and d > 0, what, "w has shape %s", tuple(w.shape))
    bp = None if bias is None else _vector(bias, what, "bias", _BF16, (v,), dev)
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
    sp = None if row_scale is None else _vector(row_scale, what, "row_scale", _F32, (n,), dev)
    L = lib()
    aligned = d % 8 == 0 and ldx % 8 == 0 and ldw % 64 == 0 and x.data_ptr() % 16 == 0 and w.data_ptr() % 128 == 0
    loss = torch.empty(n, dtype=_F32, device=dev)
    lse = torch.empty_like(loss)
    dx = dw = db = None
    if grad:
        dx = _like(x)
        dw = torch.empty((v, d), dtype=_F32, device=dev) if dw_f32 else _like(w)
        db = torch.empty_like(bias, dtype=dw.dtype) if bias is not None else None
    size = _vocab_ws(n, v, d, k, bias is not None, grad, aligned, piece_bytes)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    head = (x.data_ptr(), ldx, w.data_ptr(), ldw, bp, ip)
    tail = (n, v, d, loss.data_ptr(), lse.data_ptr())
    room = (ws.data_ptr(), size)
    was, st = _enter(dev)
    if grad:
        tail = (sp, *tail, dx.data_ptr(), d, dw.data_ptr(), d, None if db is None else db.data_ptr(), dw_f32,
                piece_bytes)
        if distill:
            rc = L.pl_vocab_distill_grad_dev(*head, tp, k, temperature, *tail, *room, st)
        else:
            rc = L.pl_vocab_ce_grad_dev(*head, *tail, *room, st)
    elif distill:
        rc = L.pl_vocab_distill_dev(*head, tp, k, temperature, *tail, *room, st)
    else:
        rc = L.pl_vocab_ce_dev(*head, *tail, *room, st)
    _leave(was)
    if rc:
        _check(rc, what)
    return (loss, lse, dx, dw, db) if grad else (loss, lse)


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
