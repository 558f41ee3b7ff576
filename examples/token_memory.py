"""A recurrent token policy: it sees a token, remembers, and answers with a token that it draws.

The environment shows random tokens and pays for the one that it showed `back` steps ago, so a policy without a memory
earns nothing. The policy is an embedding, one block with a matrix memory, and a head of V outputs:

    u, mean, rstd      = layer_norm(x)                              x: the embedding's rows
    q, k, v, g, beta   = projections of u
    o, state, saved    = delta_rule(q, k, v, g, beta, offsets, state)
    r, y, rb, rr       = block_norm(x, o W_out, u W_gate)
    loss, _, dy, ...   = vocab_ce_grad(y, head, answers, bias, advantages)

A rollout takes the same block one token at a time (delta_rule_step) and draws its answers (sample); what it drew goes through
the block once more, all episodes packed one behind the other, for the gradient. Each is one call per operator;
the projections are torch's products.

    python examples/token_memory.py [--vocab 64] [--width 128] [--envs 256] [--steps 40] [--updates 30]
"""
import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from pufferlean_b200 import tokens  # noqa: E402

BF16 = torch.bfloat16


class MemoryPolicy:
    """Parameters (f32 masters, bf16 copies in the products) and the block in both its forms."""

    def __init__(self, vocab, width, heads=2, dk=32, dv=32, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *s, scale=1.0: torch.randn(*s, generator=g, device="cuda") * scale
        self.heads, self.dk, self.dv, self.width, self.vocab = heads, dk, dv, width, vocab
        inner = heads * dv
        self.p = dict(embedding=rand(vocab, width), gain=torch.ones(width, device="cuda"),
                      qkv=rand(width, 2 * heads * dk + inner, scale=width ** -0.5),
                      decay=rand(width, heads, scale=0.1 * width ** -0.5), write=rand(width, heads, scale=width ** -0.5),
                      gate=rand(width, width, scale=width ** -0.5), out=rand(inner, width, scale=inner ** -0.5),
                      post=torch.ones(width, device="cuda"), final=torch.ones(width, device="cuda"),
                      head=rand(vocab, width, scale=0.1 * width ** -0.5), bias=torch.zeros(vocab, device="cuda"))

    def _inputs(self, seen, first):
        """What the memory takes, from tokens seen [n] and whether each begins an episode."""
        p = self.p
        x = p["embedding"][seen].to(BF16)
        u, mean, rstd = tokens.layer_norm(x, p["gain"])
        wide = u @ p["qkv"].to(BF16)
        h, dk = self.heads, self.dk
        raw = wide[:, :2 * h * dk].view(-1, 2 * h, dk).float()
        length = raw.norm(dim=2, keepdim=True) + 1e-6
        unit = (raw / length).to(BF16)
        f = u.float()
        decay, write = f @ p["decay"], f @ p["write"]
        g = -torch.nn.functional.softplus(decay - 3.0)
        g = torch.where(first[:, None], -math.inf, g)  # a new episode forgets the one before it
        parts = dict(x=x, u=u, mean=mean, rstd=rstd, raw=raw, length=length, decay=decay, write=write)
        return parts, (unit[:, :h], unit[:, h:], wide[:, 2 * h * dk:].view(-1, h, self.dv), g.contiguous(),
                       torch.sigmoid(write))

    def _block(self, parts, o):
        p = self.p
        parts["branch"] = o.reshape(len(o), -1) @ p["out"].to(BF16)
        parts["gated"] = parts["u"] @ p["gate"].to(BF16)
        return tokens.block_norm(parts["x"], parts["branch"], parts["gated"], p["post"], p["final"])

    def act(self, seen, first, state, u, temperature=1.0, top_k=0, top_p=1.0):
        """One step of every environment: (answers, their log-probabilities, states); state is updated in place."""
        parts, memory = self._inputs(seen, first)
        o, state = tokens.delta_rule_step(*memory, state, out=state)
        _, y, _, _ = self._block(parts, o)
        logits = y @ self.p["head"].to(BF16).t() + self.p["bias"].to(BF16)
        answers, logp = tokens.sample(logits, u, temperature, top_k, top_p)
        return answers, logp, state

    def gradients(self, seen, first, answers, scale, offsets, state):
        """(loss [n], gradients by parameter) of sum_n scale_n * (minus the log-probability of answer n)."""
        p, n, h, dk = self.p, len(seen), self.heads, self.dk
        parts, memory = self._inputs(seen, first)
        o, _, saved = tokens.delta_rule(*memory, offsets, state, save=True)
        r, y, rb, rr = self._block(parts, o)
        loss, _, dy, dhead, dbias = tokens.vocab_ce_grad(y, p["head"].to(BF16), answers, p["bias"].to(BF16), scale,
                                                         dw_f32=True)
        dx, dbranch, dgated, dpost, dfinal = tokens.block_norm_grad(None, dy, parts["branch"], parts["gated"], r, rb, rr,
                                                                    p["post"], p["final"])
        flat = o.reshape(n, -1)
        d = dict(head=dhead, bias=dbias, post=dpost, final=dfinal, out=(flat.t() @ dbranch).float(),
                 gate=(parts["u"].t() @ dgated).float())
        do = (dbranch @ p["out"].to(BF16).t()).view(n, h, self.dv)
        dq, dk_, dv, dg, dbeta, _ = tokens.delta_rule_grad(do, None, *memory, offsets, saved)
        # back through q / |q|, k / |k| and the gates' activations
        dunit, unit = torch.cat([dq, dk_], 1).float(), parts["raw"] / parts["length"]
        draw = (dunit - unit * (dunit * unit).sum(2, keepdim=True)) / parts["length"]
        dwide = torch.cat([draw.reshape(n, -1), dv.reshape(n, -1).float()], 1).to(BF16)
        ddecay = -dg * torch.sigmoid(parts["decay"] - 3.0)
        beta = memory[4]
        dwrite = dbeta * beta * (1 - beta)
        f = parts["u"].float()
        d.update(qkv=(parts["u"].t() @ dwide).float(), decay=f.t() @ ddecay, write=f.t() @ dwrite)
        du = ((dwide @ p["qkv"].to(BF16).t()).float() + (dgated @ p["gate"].to(BF16).t()).float()
              + ddecay @ p["decay"].t() + dwrite @ p["write"].t()).to(BF16)
        more, d["gain"], _ = tokens.layer_norm_grad(du, parts["x"], p["gain"], parts["mean"], parts["rstd"])
        d["embedding"] = torch.zeros_like(p["embedding"]).index_add_(0, seen, dx.float() + more.float())
        return loss, d


def rollout(policy, envs, steps, back, gen, state=None):
    """Tokens shown, answers, log-probabilities and rewards [envs, steps] of one episode per environment."""
    shown = torch.randint(0, policy.vocab, (steps, envs), generator=gen, device="cuda")
    state = torch.zeros(envs, policy.heads, policy.dk, policy.dv, device="cuda")
    answers, logps = [], []
    for t in range(steps):
        first = torch.full((envs,), t == 0, device="cuda")
        a, logp, state = policy.act(shown[t], first, state, torch.rand(envs, generator=gen, device="cuda"))
        answers.append(a)
        logps.append(logp)
    answers, logps = torch.stack(answers), torch.stack(logps)
    reward = torch.zeros(steps, envs, device="cuda")
    reward[back:] = (answers[back:] == shown[:steps - back]).float()
    return tuple(x.t().contiguous() for x in (shown, answers, logps, reward))


def train(vocab=64, width=128, envs=256, steps=40, updates=30, back=2, lr=2e-3, seed=0, say=print):
    """Returns the mean reward per step of the first and the last update."""
    policy = MemoryPolicy(vocab, width, seed=seed)
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    moments = {k: (torch.zeros_like(v), torch.zeros_like(v)) for k, v in policy.p.items()}
    offsets = torch.arange(envs + 1, dtype=torch.int32, device="cuda") * steps
    state = torch.zeros(envs, policy.heads, policy.dk, policy.dv, device="cuda")
    out = []
    for i in range(updates):
        shown, answers, _, reward = rollout(policy, envs, steps, back, gen)
        advantage = (reward - reward.mean()) / (reward.std() + 1e-6)
        first = torch.zeros(envs, steps, dtype=torch.bool, device="cuda")
        first[:, 0] = True
        _, d = policy.gradients(shown.reshape(-1), first.reshape(-1), answers.reshape(-1),
                                advantage.reshape(-1) / advantage.numel(), offsets, state)
        for k, w in policy.p.items():  # Adam
            m, v = moments[k]
            m.mul_(0.9).add_(d[k], alpha=0.1)
            v.mul_(0.99).addcmul_(d[k], d[k], value=0.01)
            w.addcdiv_(m / (1 - 0.9 ** (i + 1)), (v / (1 - 0.99 ** (i + 1))).sqrt().add_(1e-8), value=-lr)
        out.append(float(reward.mean()))
        if i % 10 == 0 or i == updates - 1:
            say(f"update {i}: {out[-1]:.4f} of a step's answers right")
    tokens.check()
    return out[0], out[-1]


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("vocab", 64), ("width", 128), ("envs", 256), ("steps", 40), ("updates", 30)):
        ap.add_argument(f"--{name}", type=int, default=value)
    a = ap.parse_args()
    train(a.vocab, a.width, a.envs, a.steps, a.updates)


if __name__ == "__main__":
    main()
