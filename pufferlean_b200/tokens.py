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

Gradients are of sum_n row_scale_n * loss_n (descent). The results carry no autograd graph, whatever their inputs require:
gradients come from the *_grad calls, and a loss of these calls adds nothing to a backward().
"""
from __future__ import annotations

import importlib.util
import os

import torch

from . import HERE, PufferError, lib


def _load():
    """The module of csrc/pl_torch.cpp (raises if it was not built)."""
    lib()
    path = os.path.join(HERE, "_build", "pl_torch.so")
    if not os.path.exists(path):
        raise PufferError(f"{path} is missing; build it with `python -m pufferlean_b200.build`")
    spec = importlib.util.spec_from_file_location("pl_torch", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.set_error(PufferError)
    return mod


_ext = _load()


def check(device=None):
    """Waits for a device (torch's current one) and raises PufferError if a wait inside one of this package's kernels ran
    out since the last check. Such waits are bounded: a fault ends in unwritten outputs, not in a hang, and the calls
    below, which return before their work is done, cannot report it. Until this has been called their losses and
    gradients are NaN then. For a training loop: where it synchronizes anyway. Not during a stream capture."""
    if device is None:
        index = torch.cuda.current_device() if torch.cuda.is_available() else -1
    else:
        device = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        if device.type != "cuda":
            raise PufferError(f"check: {device} is not a CUDA device")
        index = torch.cuda.current_device() if device.index is None else device.index
    _ext.check(index)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(y, mean, rstd) of the rows of x [rows, cols] (f32 or bf16); weight and bias [cols] f32 or None, mean and rstd
    [rows] f32 (what layer_norm_grad takes)."""
    return _ext.layer_norm(x, weight, bias, eps)


def layer_norm_grad(dy, x, weight, mean, rstd, params=True):
    """(dx, dweight, dbias) of layer_norm: dx in x's type, dweight and dbias [cols] f32 (None with params=False)."""
    return _ext.layer_norm_grad(dy, x, weight, mean, rstd, params)


def vocab_ce(x, w, target, bias=None):
    """(loss, lse) [N] f32 of the head z = x w^T + bias against target [N] int32: loss = lse - z[target], the negative
    log-probability. x [N, D], w [V, D], bias [V] bf16. A negative target leaves its row out (loss = lse = 0); one past
    the vocabulary makes the row's loss NaN."""
    return _ext.vocab("vocab_ce", x, w, target, None, bias, 1.0, None, False, False, 0)


def vocab_ce_grad(x, w, target, bias=None, row_scale=None, dw_f32=False, piece_bytes=0):
    """(loss, lse, dx, dw, dbias) of sum_n row_scale_n loss_n: dx bf16, dw and dbias bf16 or (dw_f32) f32, dbias None
    without a bias. dw_f32 saves the last rounding only: the logits' gradient goes into the products as bf16 (up to 64
    rows: as two bf16 parts). piece_bytes bounds the softmax terms held at a time (0: 4 GiB); loss and lse do not depend
    on it, the order of the gradients' sums does."""
    return _ext.vocab("vocab_ce_grad", x, w, target, None, bias, 1.0, row_scale, True, dw_f32, piece_bytes)


def vocab_distill(x, w, ids, teacher, bias=None, temperature=1.0):
    """(loss, lse) [N] f32 of the head's distribution q = softmax((x w^T + bias) / temperature) against the teacher's
    p = softmax(teacher / temperature) over its K top entries (ids, teacher [N, K]; a negative id or a logit of -inf is
    absent): loss = sum_k p_k (log p_k - log q_id(k)), KL(p | q) where the row's ids differ (entries of one id add up, their
    log p_k stay the single ones). A row without entries is left out (loss = lse = 0)."""
    if teacher is None:
        raise PufferError("vocab_distill: teacher is needed")
    return _ext.vocab("vocab_distill", x, w, ids, teacher, bias, temperature, None, False, False, 0)


def vocab_distill_grad(x, w, ids, teacher, bias=None, temperature=1.0, row_scale=None, dw_f32=False, piece_bytes=0):
    """(loss, lse, dx, dw, dbias) of sum_n row_scale_n loss_n, as vocab_ce_grad."""
    if teacher is None:
        raise PufferError("vocab_distill_grad: teacher is needed")
    return _ext.vocab("vocab_distill_grad", x, w, ids, teacher, bias, temperature, row_scale, True, dw_f32, piece_bytes)
