"""The cross entropy in pieces of the vocabulary against the same loss in 64 bits: kernels on the
GPU, the operations of PyTorch on the CPU."""

import math

import pytest
import torch

from offload_adam_b200 import _ext
from offload_adam_b200.ops.linear_ce import linear_cross_entropy

gpu = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _leave_no_cached_blocks():
    """Tests that measure peak memory count whole cached blocks, whoever left them."""
    yield
    if torch.cuda.is_available():
        torch.cuda.empty_cache()


DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]


def _inputs(n, hidden, vocab, device, ignored=0.2, dtype=torch.bfloat16, seed=0):
    gen = torch.Generator().manual_seed(seed)
    h = torch.randn(n, hidden, generator=gen)
    w = torch.randn(vocab, hidden, generator=gen) / math.sqrt(hidden)
    labels = torch.randint(0, vocab, (n,), generator=gen)
    h[::3] += 4 * w[labels[::3]]  # rows that are sure of their label
    labels[torch.rand(n, generator=gen) < ignored] = -100
    g = torch.rand(n, generator=gen) - 0.3
    return h.to(device, dtype), w.to(device, dtype), labels.to(device), g.to(device)


def _run(h, w, labels, g, reduction, **kw):
    h, w = h.detach().clone().requires_grad_(True), w.detach().clone().requires_grad_(True)
    loss = linear_cross_entropy(h, w, labels, reduction=reduction, **kw)
    loss.backward(g if reduction == "none" else g[0])
    return loss.detach(), h.grad, w.grad


def _exact(h, w, labels, g, reduction, ignore=-100):
    """(losses of the rows, result, gradients) and how far the kernels' gradients may be off."""
    h, w = h.detach().double(), w.detach().double()
    rows = (labels != ignore).nonzero(as_tuple=True)[0]
    x, lab = h[rows], labels[rows]
    z = x @ w.T
    logp = torch.log_softmax(z, 1)
    at = torch.arange(len(rows), device=h.device)
    losses = torch.zeros(len(labels), dtype=torch.float64, device=h.device)
    losses[rows] = -logp[at, lab]
    scale = {"none": g[rows].double(), "sum": g[0].double(), "mean": g[0].double() / max(1, len(rows))}[reduction]
    d = logp.exp()
    d[at, lab] -= 1
    d = d * scale.expand(len(rows))[:, None]
    gh = torch.zeros_like(h)
    gh[rows] = d @ w
    gw = d.T @ x
    result = {"none": losses, "sum": losses.sum(), "mean": losses.sum() / max(1, len(rows))}[reduction]
    # each entry of d and the result round to bf16, by up to 2^-8 of their value; an error of e in
    # a logit is one of e in d relative to p = d + [label], and of 4 e with the sum's
    e = _logit_error(h.shape[1], z)
    p = (d.abs() + torch.zeros_like(d).index_put_((at, lab), scale.abs().expand(len(rows)))) * 4 * e
    off = 2.0 ** -8 * d.abs() + p
    tol_h = torch.zeros_like(h)
    tol_h[rows] = off @ w.abs()
    return result, gh, gw, tol_h + 2.0 ** -8 * gh.abs() + 1e-30, off.T @ x.abs() + 2.0 ** -8 * gw.abs() + 1e-30


def _logit_error(hidden, z):
    """The sum of a logit takes hidden / 16 additions in fp32, each off by one unit (2^-23) of
    the running sum; exponentials and their sum add as much as 128 more."""
    top = z.abs().max().item() if z.numel() else 0.0
    return ((hidden / 16 + 4) * (top + 1) + 128) * 2.0 ** -23


def _check(h, w, labels, g, reduction, **kw):
    got = _run(h, w, labels, g, reduction, **kw)
    ignore = kw.get("ignore_index", -100)
    want = _exact(h, w, labels, g, reduction, ignore)
    rows = labels != ignore
    tol = 2 * _logit_error(h.shape[1], h[rows].double() @ w.double().T) * (len(labels) if reduction == "sum" else 1)
    tol += 2.0 ** -23 * want[0].abs().max().item() if want[0].numel() else 0.0
    assert got[0].dtype == torch.float32 and got[0].shape == want[0].shape
    assert (got[0].double() - want[0]).abs().max() <= tol
    assert got[1].dtype == h.dtype and got[2].dtype == w.dtype
    assert ((got[1].double() - want[1]).abs() <= want[3]).all()
    assert ((got[2].double() - want[2]).abs() <= want[4]).all()
    assert (got[1][labels == ignore] == 0).all()
    return got


# rows and words around a tile of one CTA (128) and of a pair (256), rows around the few that run
# the narrow products (16 and 64), inner sizes around a stage (64), pieces that end with one word
SIZES = [(1, 8, 1), (1, 64, 257), (2, 72, 7), (16, 264, 300), (17, 72, 129), (63, 64, 128), (64, 128, 127), (64, 1032, 5000), (65, 256, 129), (127, 264, 255),
         (128, 8, 256), (129, 840, 513), (255, 64, 1000), (256, 256, 1024), (257, 520, 2049), (700, 136, 4099)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("n,hidden,vocab", SIZES)
def test_matches_64_bits(n, hidden, vocab, reduction, device):
    _check(*_inputs(n, hidden, vocab, device), reduction)


@gpu
@pytest.mark.parametrize("piece", [1, 256, 300, 768, 4096, 1 << 20])
@pytest.mark.parametrize("n,hidden,vocab", [(3, 64, 2561), (40, 136, 2100), (300, 200, 2560), (513, 96, 1025)])
def test_pieces(n, hidden, vocab, piece):
    _check(*_inputs(n, hidden, vocab, "cuda"), "mean", piece=piece)
