"""Operators of a token policy on CUDA tensors: layer norm, the large-vocabulary head's cross entropy, and
distillation of a teacher's top logits into the head, each forward and with its gradients; drawing tokens from logits; the
norms around a block with its gate and residual scale; and a matrix memory per head, the gated delta rule.

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


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token int32, logp f32) [N]: one token per row of logits [N, V] (f32 or bf16, V up to 262,144), drawn with the given
    numbers u [N] f32 in [0, 1), so that a draw can be repeated. The options are numbers, or tensors [N] with one for each
    row (f32; top_k int32). As a number a negative top_k or temperature is refused; in a tensor the one means all, the other
    spoils its row. By falling logit, equal ones by index: the first top_k stay (0: all); of these those before
    which less than top_p of their mass comes; of these those with at least min_p of the largest probability; the first
    always. logp is the token's log-probability among those that stay, at this temperature (what an importance ratio
    divides by). temperature 0 takes the first, one between 0 and 1e-38 counts as 1e-38, one above 1e30 as 1e30, a min_p above 1
    as 1. A logit of -inf is never drawn; a row with a NaN or +inf, with nothing but -inf, with an option that is NaN or
    with a negative or infinite temperature gets token -1 and logp NaN."""
    return _ext.sample(logits, u, temperature, top_k, top_p, min_p)


def block_norm(x, branch, gate=None, branch_weight=None, weight=None, scale=1.0, eps=1e-5, post=True):
    """(r, y, rstd_branch, rstd): a block's output on its way back into the residual stream x, and the next block's input.
    r = x + scale * sigmoid(gate) * branch_weight * rms(branch), y = weight * rms(r) with rms(z) = z / sqrt(mean z^2 + eps).
    x, branch, gate [rows, cols] f32 or bf16 (gate None: no gate), the weights [cols] f32 or None. post=False leaves the
    first norm out (rstd_branch None). The statistics [rows] f32 are what block_norm_grad takes."""
    return _ext.block_norm(x, branch, gate, branch_weight, weight, scale, eps, post)


def block_norm_grad(dr, dy, branch, gate, r, rstd_branch, rstd, branch_weight=None, weight=None, scale=1.0, params=True):
    """(dx, dbranch, dgate, dbranch_weight, dweight) of block_norm from the gradients dr of r (None: zero) and dy of y. dgate
    is None without a gate, the weights' gradients [cols] f32 with params=False."""
    return _ext.block_norm_grad(dr, dy, branch, gate, r, rstd_branch, rstd, branch_weight, weight, scale, params)


def _scale(q, scale):
    return q.shape[-1] ** -0.5 if scale is None else scale


def delta_rule(q, k, v, g, beta, offsets=None, state=None, scale=None, save=False):
    """(o, final_state, saved): the gated delta rule over packed sequences. Every head of values keeps a matrix S, and with
    a = exp(g): u_t = beta_t (v_t - a_t S^T k_t), S <- a_t S + k_t u_t^T, o_t = scale S^T q_t (scale None: dk ** -0.5).

    q, k [N, Hk, dk], v [N, Hv, dv] bf16 (views of one wider projection will do), g, beta [N, Hv] f32, state and final_state
    [S, Hv, dk, dv] f32; dk up to 128, dv up to 1,024, Hv a multiple of Hk. offsets [S + 1] int32: sequence s has rows
    offsets[s] to offsets[s + 1]; None: as many sequences of one length as `state` has (one without a state). Rows outside all
    sequences get zeros. g = -inf forgets the (finite) state: an episode's first token. With keys of length one and beta below 2
    the rule is stable. `saved` (None without save) is what delta_rule_grad takes: for 64 tokens of a head of 128 x 128 with a
    key head of its own 198 KB, four times what q, k and v hold.

    All inputs but g have to be finite: 64 tokens are worked on at once, so a NaN or an infinity (one that an unstable rule has
    come to, too) reaches any token of its sequence in its 64 and behind them, past a g of -inf as well; other sequences and
    heads stay clean, and a sequence's first token with g = -inf forgets any state."""
    if offsets is not None:
        sequences = offsets.shape[0] - 1
    else:
        sequences = 1 if state is None else state.shape[0]
    o, final, saved = _ext.delta_rule(q, k, v, g, beta, offsets, sequences, state, _scale(q, scale), save)
    return o, final, ((saved, sequences) if save else None)


def delta_rule_grad(do, dstate, q, k, v, g, beta, offsets, saved, scale=None):
    """(dq, dk, dv, dg, dbeta, dstate) of delta_rule from the gradients do [N, Hv, dv] bf16 of o and dstate of the final
    state (None: zero); the last of the results is that of the first state. The other arguments are the forward call's, `saved`
    what it returned, with the values of q, k, g and beta that count; v is read again. dq, dk, dv bf16, dg, dbeta, dstate f32."""
    if saved is None:
        raise PufferError("delta_rule_grad: saved is needed (delta_rule with save=True)")
    return _ext.delta_rule_grad(q, k, v, g, beta, offsets, saved[1], do, dstate, _scale(q, scale), saved[0])


def delta_rule_step(q, k, v, g, beta, state, scale=None, out=None):
    """(o, state): delta_rule for one token of every row, state [N, Hv, dk, dv] f32. The new states go into `out`, which may
    be `state` itself, or a new tensor. A g of -inf forgets any state, one that is not finite too."""
    return _ext.delta_rule_step(q, k, v, g, beta, state, _scale(q, scale), out)
