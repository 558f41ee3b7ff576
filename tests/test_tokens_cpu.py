"""The token-policy operators' host side: their C entries are exported and bound, check their arguments before they look
for a device, plan workspaces that grow with what they hold, and the Python calls refuse CPU tensors."""
import pytest

import pufferlean_b200 as plb

torch = pytest.importorskip("torch")
from pufferlean_b200 import tokens  # noqa: E402

INVALID, NO_DEVICE = -1, -6


@pytest.fixture(scope="module")
def L():
    return plb.lib()


def test_entries_are_bound(L):
    for name in ("pl_layernorm_dev", "pl_layernorm_grad_ws", "pl_layernorm_grad_dev", "pl_vocab_ws", "pl_vocab_ce_dev",
                 "pl_vocab_ce_grad_dev", "pl_vocab_distill_dev", "pl_vocab_distill_grad_dev"):
        assert getattr(L, name).argtypes is not None


def test_arguments_are_checked_first(L):
    p = 1 << 12  # never read: every call fails before a launch
    bad = [
        L.pl_layernorm_dev(p, 8, None, None, 4, 16, 1e-5, 1, p, 16, p, p, None),  # stride below the width
        L.pl_layernorm_dev(p, 16, None, None, 4, 0, 1e-5, 1, p, 16, p, p, None),  # no columns
        L.pl_layernorm_dev(None, 16, None, None, 4, 16, 1e-5, 1, p, 16, p, p, None),
        L.pl_layernorm_dev(p, 16, None, None, 4, 16, float("nan"), 1, p, 16, p, p, None),
        L.pl_layernorm_grad_dev(p, 16, p, 16, None, p, p, 4, 0, 1, p, 16, None, None, None, 0, None),
        L.pl_vocab_ce_dev(p, 16, p, 16, None, p, 4, 9, 17, p, p, p, 1 << 20, None),
        L.pl_vocab_ce_dev(p, 16, p, 16, None, p, 4, 0, 16, p, p, p, 1 << 20, None),
        L.pl_vocab_ce_dev(p, 16, None, 16, None, p, 4, 9, 16, p, p, p, 1 << 20, None),
        L.pl_vocab_ce_dev(p, 16, p, 16, None, None, 4, 9, 16, p, p, p, 1 << 20, None),
        L.pl_vocab_ce_dev(p, 16, p, 16, None, p, 1 << 31, 9, 16, p, p, p, 1 << 20, None),
        L.pl_vocab_ce_grad_dev(p, 16, p, 16, None, p, None, 4, 9, 16, p, p, p, 16, None, 16, None, 0, 0, p, 1 << 20, None),
        L.pl_vocab_ce_grad_dev(p, 16, p, 16, p, p, None, 4, 9, 16, p, p, p, 16, p, 16, None, 0, 0, p, 1 << 20, None),
        L.pl_vocab_ce_grad_dev(p, 16, p, 16, None, p, None, 4, 9, 16, p, p, p, 16, p, 8, None, 0, 0, p, 1 << 20, None),
        L.pl_vocab_distill_dev(p, 16, p, 16, None, p, None, 2, 1.0, 4, 9, 16, p, p, p, 1 << 20, None),
        L.pl_vocab_distill_dev(p, 16, p, 16, None, p, p, 0, 1.0, 4, 9, 16, p, p, p, 1 << 20, None),
        L.pl_vocab_distill_dev(p, 16, p, 16, None, p, p, 513, 1.0, 4, 9, 16, p, p, p, 1 << 20, None),
        L.pl_vocab_distill_dev(p, 16, p, 16, None, p, p, 2, 0.0, 4, 9, 16, p, p, p, 1 << 20, None),
        L.pl_vocab_distill_dev(p, 16, p, 16, None, p, p, 2, float("nan"), 4, 9, 16, p, p, p, 1 << 20, None),
    ]
    assert all(rc == INVALID for rc in bad), bad
    assert L.pl_last_error()
    if plb.device_count() == 0:
        assert L.pl_vocab_ce_dev(p, 16, p, 16, None, p, 4, 9, 16, p, p, p, 1 << 30, None) == NO_DEVICE


def test_workspaces(L):
    assert L.pl_vocab_ws(0, 1000, 64, 0, 1, 1, 1, 0) == 0
    base = L.pl_vocab_ws(4096, 50000, 1024, 0, 0, 1, 1, 0)
    terms = 4096 * 50048 * 2
    assert terms < base < terms * 1.6  # the terms and little else: no logits, no f32 copy of the weights
    assert L.pl_vocab_ws(4096, 50000, 1024, 0, 0, 0, 1, 0) < terms / 8  # the loss alone keeps statistics only
    assert L.pl_vocab_ws(4096, 50000, 1024, 0, 1, 1, 1, 0) > base  # a bias adds its column sums
    assert L.pl_vocab_ws(4096, 50000, 1024, 64, 0, 1, 1, 0) > base  # answers
    assert L.pl_vocab_ws(4096, 50000, 1024, 0, 0, 1, 0, 0) > base  # copies of unaligned matrices
    small = L.pl_vocab_ws(4096, 50000, 1024, 0, 0, 1, 1, 64 << 20)  # pieces of 64 MB, dw summed in f32
    assert small < (64 << 20) + 50000 * 1024 * 4 + (128 << 20) < base
    for n in (1, 127, 128, 129, 5000, 100000):
        for v in (1, 129, 18944, 18945, 131072):
            assert L.pl_vocab_ws(n, v, 77, 3, 1, 1, 1, 0) <= L.pl_vocab_ws(n, v, 77, 3, 1, 1, 0, 0)
    assert L.pl_layernorm_grad_ws(1, 64) == 2 * 64 * 4
    assert L.pl_layernorm_grad_ws(1 << 20, 64) == L.pl_layernorm_grad_ws(1 << 19, 64)


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(9, 16, dtype=torch.bfloat16)
    t, k = torch.zeros(4, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.int32)
    f = torch.zeros(4, 2)
    for call in (lambda: tokens.layer_norm(x), lambda: tokens.layer_norm_grad(x, x, None, f[:, 0], f[:, 1]),
                 lambda: tokens.vocab_ce(x, w, t), lambda: tokens.vocab_ce_grad(x, w, t),
                 lambda: tokens.vocab_distill(x, w, k, f), lambda: tokens.vocab_distill_grad(x, w, k, f),
                 lambda: tokens.vocab_distill(x, w, k, None), lambda: tokens.layer_norm([1.0])):
        with pytest.raises(plb.PufferError):
            call()
