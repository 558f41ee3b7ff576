"""A token policy trained with the framework's operators: demonstrations first, then a teacher's top answers.

The policy reads a token and answers with one of V tokens: an embedding row, a layer norm, and a head of V outputs.
Its teacher is a fixed head over fixed features. Each step is what a training loop does:

    y, mean, rstd          = layer_norm(embedding[tokens], gain, shift)
    loss, _, dy, dhead, db = vocab_ce_grad(y, head, targets, bias, scale)      (or vocab_distill_grad)
    dx, dgain, dshift      = layer_norm_grad(dy, ...)

and an update in which the head's momentum is orthogonalised by pl_ns_batched_bf16_dev, as Muon does for the
framework's other policies; gain, shift, bias and the embedding take plain gradient steps.

    python examples/token_policy.py [--vocab 2048] [--width 256] [--batch 4096] [--steps 60]
"""
import argparse
import ctypes
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import pufferlean_b200 as plb  # noqa: E402
from pufferlean_b200 import tokens  # noqa: E402

NS = [3.4445, -4.7750, 2.0315] * 5  # the quintic Newton-Schulz table, five steps


class TokenPolicy:
    """Parameters of the policy and one optimiser step; the masters are f32, the head's working copy is bf16."""

    def __init__(self, vocab, width, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.embedding = torch.randn(vocab, width, generator=g, device="cuda")
        self.gain = torch.ones(width, device="cuda")
        self.shift = torch.zeros(width, device="cuda")
        self.head = torch.randn(vocab, width, generator=g, device="cuda") * (0.02 / width ** 0.5)
        self.bias = torch.zeros(vocab, device="cuda")
        self.momentum = torch.zeros_like(self.head)
        self.coeffs = (ctypes.c_double * len(NS))(*NS)

    def step(self, seen, answer, lr):
        """One step on tokens `seen`; answer(y, head, bias) returns (loss, lse, dy, dhead, dbias)."""
        x = self.embedding[seen].to(torch.bfloat16)
        y, mean, rstd = tokens.layer_norm(x, self.gain, self.shift)
        loss, _, dy, dhead, dbias = answer(y, self.head.to(torch.bfloat16), self.bias.to(torch.bfloat16))
        dx, dgain, dshift = tokens.layer_norm_grad(dy, x, self.gain, mean, rstd)
        # Muon on the head: Nesterov momentum, orthogonalised on the tensor cores
        self.momentum.mul_(0.95).add_(dhead)
        update = (dhead + 0.95 * self.momentum)
        update = (update / (update.norm() + 1e-12)).to(torch.bfloat16)
        rows, cols = update.shape
        rc = plb.lib().pl_ns_batched_bf16_dev(update.data_ptr(), 1, rows, cols, 1e-7, self.coeffs, 5,
                                              torch.cuda.current_stream().cuda_stream)
        if rc:
            raise plb.PufferError(plb.lib().pl_last_error().decode())
        self.head.add_(update.float(), alpha=-lr * max(1.0, rows / cols) ** 0.5)
        self.bias.add_(dbias, alpha=-20 * lr)
        self.gain.add_(dgain, alpha=-lr)
        self.shift.add_(dshift, alpha=-lr)
        self.embedding.index_add_(0, seen, dx.float(), alpha=-20 * lr)
        return loss


def train(vocab=2048, width=256, batch=4096, steps=60, k=16, temperature=2.0, seed=0, say=print):
    """Returns the mean losses of the first and last step of both phases."""
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    teacher = torch.randn(vocab, width, generator=g, device="cuda") @ (
        torch.randn(width, vocab, generator=g, device="cuda") * (3.0 / width ** 0.5))
    policy = TokenPolicy(vocab, width, seed)
    scale = torch.full((batch,), 1.0 / batch, device="cuda")
    seen_all = torch.randint(0, vocab, (2 * steps, batch), generator=g, device="cuda")
    out = []

    def phase(name, offset, answer_for):
        first = last = None
        for i in range(steps):
            seen = seen_all[offset + i]
            loss = policy.step(seen, answer_for(seen), 0.02 * (1 - i / steps) + 0.001)
            if i in (0, steps - 1):
                counted = loss != 0
                mean = float(loss.sum() / counted.sum())
                first, last = (mean if first is None else first), mean
            if i % 20 == 0 or i == steps - 1:
                say(f"{name} step {i}: {float(loss.mean()):.4f}")
        out.extend((first, last))

    def demonstrations(seen):  # one in eight is missing
        target = torch.distributions.Categorical(logits=teacher[seen]).sample().to(torch.int32)
        target[::8] = -1
        return lambda y, w, b: tokens.vocab_ce_grad(y, w, target, b, scale, dw_f32=True)

    def answers(seen):
        logits, ids = teacher[seen].topk(k, dim=1)
        ids = ids.to(torch.int32).contiguous()
        return lambda y, w, b: tokens.vocab_distill_grad(y, w, ids, logits.contiguous(), b, temperature, scale,
                                                         dw_f32=True)

    phase("demonstrations", 0, demonstrations)
    phase("distillation", steps, answers)
    return out


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--vocab", type=int, default=2048)
    ap.add_argument("--width", type=int, default=256)
    ap.add_argument("--batch", type=int, default=4096)
    ap.add_argument("--steps", type=int, default=60)
    a = ap.parse_args()
    first, last, dfirst, dlast = train(a.vocab, a.width, a.batch, a.steps)
    print(f"cross entropy {first:.3f} -> {last:.3f}, distillation {dfirst:.3f} -> {dlast:.3f}")


if __name__ == "__main__":
    main()
