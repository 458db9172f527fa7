"""The cross entropy in pieces of the vocabulary at the limits of its numbers and sizes: infinite
weights, logits of the lowest value, long sums."""

import math

import pytest
import torch

from offload_adam_b200.ops.linear_ce import linear_cross_entropy

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]
BF16 = torch.bfloat16


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n", [5, 64, 65, 100, 300])
def test_a_word_of_minus_infinity(n, device):
    """A word whose logits are all -inf has no part in any row: its row of the head's gradient is
    zero and the other words' gradients are as without it."""
    gen = torch.Generator().manual_seed(n)
    h = (torch.rand(n, 64, generator=gen) + 0.5).to(BF16).to(device)
    w = (0.1 * torch.randn(600, 64, generator=gen)).to(BF16).to(device)
    labels = torch.randint(10, 600, (n,), generator=gen)
    labels[::4] = -100
    labels = labels.to(device)
    w[7, 0] = -math.inf
    w.requires_grad_(True)
    loss = linear_cross_entropy(h, w, labels, reduction="sum")
    gw, = torch.autograd.grad(loss, w)
    rows = labels != -100
    z = h[rows].double() @ w.detach().double().T
    logp = torch.log_softmax(z, 1)
    at = torch.arange(len(z), device=device)
    exact = -logp[at, labels[rows]].sum()
    d = logp.exp()
    assert (d[:, 7] == 0).all()
    d[at, labels[rows]] -= 1
    want = d.T @ h[rows].double()
    assert (gw[7] == 0).all()
    # logits of 64 terms below 3 and their sums are off by ((64 / 16 + 4) * 4 + 128) 2^-23 < 2^-15; losses
    # are above 4
    assert abs(loss.double() - exact) <= exact * 2.0 ** -16
    # d, the rows of h times 1 - p and the result round to bf16 (2^-8 each)
    off = (3 * 2.0 ** -8 + 2.0 ** -13) * (d.abs().T @ h[rows].double().abs())
    assert ((gw.double() - want).abs() <= off).all()
