"""The recurrent token policy's operators together, as examples/token_memory.py uses them: its gradients against autograd in 64
bits, a rollout's log-probabilities against the training pass's, and the example's run."""
import os
import sys

import pytest

torch = pytest.importorskip("torch")

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu
F64 = torch.float64


@pytest.fixture(scope="module", autouse=True)
def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _loss64(p, policy, seen, first, answers, scale, lengths):
    """The policy's loss in 64 bits, a token at a time, for autograd. Parameters and inputs are what the policy rounds to
    bf16; nothing else is rounded."""
    h, dk, dv = policy.heads, policy.dk, policy.dv
    x = p["embedding"][seen]
    u = (x - x.mean(1, keepdim=True)) / torch.sqrt(x.var(1, unbiased=False, keepdim=True) + 1e-5) * p["gain"]
    wide = u @ p["qkv"]
    raw = wide[:, :2 * h * dk].view(-1, 2 * h, dk)
    unit = raw / (raw.norm(dim=2, keepdim=True) + 1e-6)
    q, k, v = unit[:, :h], unit[:, h:], wide[:, 2 * h * dk:].view(-1, h, dv)
    a = torch.exp(-torch.nn.functional.softplus(u @ p["decay"] - 3.0))
    a = torch.where(first[:, None], torch.zeros_like(a), a)
    beta = torch.sigmoid(u @ p["write"])
    outs, at = [], 0
    for n in lengths:
        s = torch.zeros(h, dk, dv, dtype=F64, device="cuda")
        for t in range(at, at + n):
            s = s * a[t][:, None, None]
            e = v[t] - torch.einsum("hij,hi->hj", s, k[t])
            s = s + torch.einsum("hi,hj->hij", k[t], e * beta[t][:, None])
            outs.append(dk ** -0.5 * torch.einsum("hij,hi->hj", s, q[t]).reshape(-1))
        at += n
    branch = torch.stack(outs) @ p["out"]
    rms = lambda z: z / torch.sqrt(z.square().mean(1, keepdim=True) + 1e-5)
    r = x + torch.sigmoid(u @ p["gate"]) * rms(branch) * p["post"]
    z = (rms(r) * p["final"]) @ p["head"].t() + p["bias"]
    logp = torch.log_softmax(z, 1).gather(1, answers[:, None].long())[:, 0]
    return -logp, (-logp * scale.double()).sum()


def _policy():
    import token_memory

    policy = token_memory.MemoryPolicy(40, 64, heads=2, dk=16, dv=24, seed=3)
    gen = torch.Generator(device="cuda").manual_seed(5)
    policy.p["head"] = torch.randn(40, 64, generator=gen, device="cuda") * 0.3
    policy.p["decay"] = torch.randn(64, 2, generator=gen, device="cuda") * 0.1
    policy.p = {k: (v.to(torch.bfloat16).float() if v.dim() == 2 else v) for k, v in policy.p.items()}
    return policy, gen


def test_gradients():
    """bf16 rounds to 2^-8; a parameter's gradient passes through at most fourteen roundings of activations and their
    gradients, which add up to 14 * 2^-8 = 5.5e-2 of its norm if none cancels."""
    policy, gen = _policy()
    lengths = [70, 1, 0, 33]
    n = sum(lengths)
    seen = torch.randint(0, 40, (n,), generator=gen, device="cuda")
    answers = torch.randint(0, 40, (n,), generator=gen, device="cuda").to(torch.int32)
    first = torch.zeros(n, dtype=torch.bool, device="cuda")
    first[[0, 20, 70, 71]] = True  # an episode ends inside the first sequence
    scale = torch.randn(n, generator=gen, device="cuda") / n
    offsets = torch.tensor([0, 70, 71, 71, 104], dtype=torch.int32, device="cuda")
    state = torch.randn(4, 2, 16, 24, generator=gen, device="cuda")  # forgotten by every first token
    loss, grads = policy.gradients(seen, first, answers, scale, offsets, state)
    p = {k: v.double().requires_grad_() for k, v in policy.p.items()}
    want, total = _loss64(p, policy, seen, first, answers, scale, lengths)
    assert ((loss.double() - want).abs() <= 14 * 2.0 ** -8 * (1 + want.abs())).all()
    for (k, w), g in zip(p.items(), torch.autograd.grad(total, list(p.values()))):
        assert grads[k].shape == g.shape
        off = float((grads[k].double() - g).norm() / g.norm())
        assert off <= 14 * 2.0 ** -8, (k, off)


def test_rollout_and_training_agree():
    """The same tokens one at a time and packed: log-probabilities differ by the roundings of activations and of the logits
    (bf16), of which there are seven in either pass."""
    import token_memory

    policy, gen = _policy()
    envs, steps = 5, 37
    shown, answers, logps, _ = token_memory.rollout(policy, envs, steps, 2, gen)
    assert (answers >= 0).all() and (answers < 40).all()
    first = torch.zeros(envs, steps, dtype=torch.bool, device="cuda")
    first[:, 0] = True
    offsets = torch.arange(envs + 1, dtype=torch.int32, device="cuda") * steps
    state = torch.zeros(envs, 2, 16, 24, device="cuda")
    loss, _ = policy.gradients(shown.reshape(-1), first.reshape(-1), answers.reshape(-1),
                               torch.ones(envs * steps, device="cuda"), offsets, state)
    big = float(loss.max()) + 1
    assert ((loss + logps.reshape(-1)).abs() <= 2 * 7 * 2.0 ** -8 * big).all()


def test_example_runs():
    import token_memory

    said = []
    first, last = token_memory.train(vocab=32, width=64, envs=32, steps=12, updates=3, say=said.append)
    assert 0 <= first <= 1 and 0 <= last <= 1 and said
