"""The cross entropy in pieces of the vocabulary at the limits of its numbers and sizes: infinite
weights, logits of the lowest value, long sums, waits that give up, any label."""

import math

import pytest
import torch

from offload_adam_b200 import _ext
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


def _far(n, vocab, device, shift):
    """Logits that differ by at most 8, all of them `shift` away from 0, both exact in bf16 products:
    the hidden state's first value is 1 and carries the shift."""
    gen = torch.Generator().manual_seed(n + vocab)
    h = torch.zeros(n, 64)
    h[:, 0] = 1.0
    h[:, 1:9] = torch.randint(0, 2, (n, 8), generator=gen).float()
    w = torch.zeros(vocab, 64)
    w[:, 0] = shift
    if abs(shift) < 1e30:  # beside the lowest value there is no room for any difference
        w[:, 1:9] = torch.randint(0, 2, (vocab, 8), generator=gen).float()
    labels = torch.randint(0, vocab, (n,), generator=gen)
    labels[2::5] = -100
    return h.to(BF16).to(device), w.to(BF16).to(device), labels.to(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shift", [0.0, -2.0 ** 20, 2.0 ** 20, torch.finfo(BF16).min, torch.finfo(BF16).max])
@pytest.mark.parametrize("n,vocab", [(5, 600), (20, 601), (100, 600), (300, 1025)])
def test_logits_far_from_zero(n, vocab, shift, device):
    """Only the differences of a row's logits matter, also where their logarithm's sum is lost beside
    the logits, as for a row whose words are all masked with the type's lowest value."""
    h, w, labels = _far(n, vocab, device, shift)
    h.requires_grad_(True)
    w.requires_grad_(True)
    loss = linear_cross_entropy(h, w, labels, reduction="none")
    gh, gw = torch.autograd.grad(loss.sum(), (h, w))
    rows = (labels != -100).nonzero(as_tuple=True)[0]
    x, y = h.detach().double()[rows], w.detach().double()
    z = x[:, 1:] @ y[:, 1:].T  # without the shift, the same in every logit
    logp = torch.log_softmax(z, 1)
    at = torch.arange(len(rows), device=device)
    exact = -logp[at, labels[rows]]
    # every logit is exact; the losses are those of sums of exponentials, (|x| + 4) 2^-24 off each and
    # 2^-24 with each of fewer than 1025 additions at most
    assert ((loss[rows].double() - exact).abs() <= 2.0 ** -13 * (1 + exact)).all()
    assert (loss[labels == -100] == 0).all() and (gh[labels == -100] == 0).all()
    d = logp.exp()
    d[at, labels[rows]] -= 1
    want_h, want_w = d @ y, d.T @ x
    # d, the rows of h times 1 - p and the results round to bf16, 2^-8 each; sums of up to 1025
    # products in fp32 add 2^-13
    assert ((gw.double() - want_w).abs() <= (3 * 2.0 ** -8 + 2.0 ** -12) * (d.abs().T @ x.abs()) + 1e-30).all()
    off = (2 * 2.0 ** -8 + 2.0 ** -12) * (d.abs() @ y.abs())
    assert ((gh[rows].double() - want_h).abs() <= off + 1e-30).all()


def _even(n, vocab, device, seed=0):
    """Words that are all as likely but word 0, the label of every row, which is next to impossible: the
    gradient of the logits is 1 / (vocab - 1), rounded to bf16, and -1 at the label."""
    gen = torch.Generator(device=device).manual_seed(seed)
    h = torch.randint(64, 193, (n, 64), generator=gen, device=device).float() / 128
    h[:, 0] = 1.0
    w = torch.zeros(vocab, 64, device=device)
    w[0, 0] = -128.0
    return h.to(BF16), w.to(BF16), torch.zeros(n, dtype=torch.int64, device=device)


@gpu
@pytest.mark.parametrize("reduction", ["sum", "none"])
@pytest.mark.parametrize("n", [65535, 65536, 65537, 131073, 200000, (1 << 20) + 37])
def test_head_gradient_over_many_rows(n, reduction):
    h, w, labels = _even(n, 97, "cuda", seed=n)
    labels[5::7] = -100
    w.requires_grad_(True)
    g = torch.randint(0, 2, (n,), device="cuda").float() + 1 if reduction == "none" else torch.full((), 0.5, device="cuda")
    gw, = torch.autograd.grad(linear_cross_entropy(h, w, labels, reduction=reduction), w, g)
    rows = labels != -100
    total = (h[rows].double() * (g[rows][:, None].double() if reduction == "none" else g.double())).sum(0)
    share = torch.tensor(1 / 96).to(BF16).item()  # not a power of two: products of 16 bits
    want = torch.cat([-total[None], total.expand(96, 64) * share])
    # the rows that count are exact in bf16; each of 4096 additions is off by 2^-23 of the sum at
    # most, and sums of 65536 rows add up in fp32; the result rounds to bf16
    assert ((gw.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -11) * want.abs()).all()


@gpu
def test_gradients_of_more_rows_than_an_accumulator_sums():
    """Random rows in two groups, in pieces, with the gradient of the hidden states: against 64 bits, and
    the same bits again."""
    n, hidden, vocab = 70000, 72, 700
    gen = torch.Generator(device="cuda").manual_seed(1)
    h = torch.randn(n, hidden, device="cuda", generator=gen).to(BF16).requires_grad_(True)
    w = (torch.randn(vocab, hidden, device="cuda", generator=gen) / math.sqrt(hidden)).to(BF16).requires_grad_(True)
    for count in (n, 65536, 66000, 300, 0):  # rows that count: the second group has many, few or none
        labels = torch.randint(0, vocab, (n,), device="cuda", generator=gen)
        labels[torch.randperm(n, device="cuda", generator=gen)[count:]] = -100
        rows = labels != -100
        x, y = h.detach().double()[rows], w.detach().double()
        z = x @ y.T
        d = z.softmax(1)
        d[torch.arange(len(x), device="cuda"), labels[rows]] -= 1
        want_h, want_w = d @ y / max(1, count), d.T @ x / max(1, count)
        tol_w = d.abs().T @ x.abs() / max(1, count) * (3 * 2.0 ** -8 + 2.0 ** -11)
        tol_h = d.abs() @ y.abs() / max(1, count) * (2 * 2.0 ** -8 + 2.0 ** -11)
        first = None
        for piece in (None, 256):
            gh, gw = torch.autograd.grad(linear_cross_entropy(h, w, labels, piece=piece), (h, w))
            assert ((gw.double() - want_w).abs() <= tol_w).all()
            assert ((gh[rows].double() - want_h).abs() <= tol_h).all()
            assert (gh[~rows] == 0).all()
            again = torch.autograd.grad(linear_cross_entropy(h, w, labels, piece=piece), (h, w))
            assert torch.equal(gh, again[0]) and torch.equal(gw, again[1])
            first = gw if first is None else first
            assert torch.equal(gw, first)  # pieces change nothing of the head's gradient


@gpu
@pytest.mark.parametrize("n,hidden,vocab,piece", [
    (4, 64, (1 << 20) + 1, None), (60, 4736, (1 << 18) + 1, None),  # few rows
    (2432, 1024, (1 << 20) + 1, 1 << 20), (2432, 1024, (1 << 18) + 1, 1 << 62),  # more tiles than pairs of SMs
    (300, 64, (1 << 21) + 1, 1 << 62)])  # more than one piece holds
def test_gradient_of_hidden_states_over_many_words(n, hidden, vocab, piece):
    """Every word but the label is as likely, so that a row's gradient is the mean of the words."""
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    w = torch.randint(64, 193, (vocab, hidden), generator=gen, device="cuda", dtype=torch.int16).to(BF16).div_(128)
    w[:, 0] = 0.0
    w[0] = 0.0
    w[0, 0] = -128.0
    h = torch.zeros(n, hidden, device="cuda", dtype=BF16)
    h[:, 0] = 1.0
    h.requires_grad_(True)
    labels = torch.zeros(n, dtype=torch.int64, device="cuda")
    gh, = torch.autograd.grad(linear_cross_entropy(h, w, labels, reduction="sum", piece=piece), h)
    total = torch.zeros(hidden, dtype=torch.float64, device="cuda")
    for s in range(1, vocab, 1 << 16):
        total += w[s:s + (1 << 16)].sum(0, dtype=torch.float64)
    want = total / (vocab - 1)
    want[0] = 128.0
    # 1 / (vocab - 1) is exact in bf16; 4096 additions are off by 2^-23 of the sum each at most, and up to 32
    # such sums add up in fp32; the result rounds to bf16
    assert ((gh.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -11) * want).all()


@gpu
@pytest.mark.parametrize("n,hidden", [(20, 8192), (20, 8200), (300, 8192), (300, 8200), (300, 16384), (130, 16456), (20, 1 << 17), (130, 1 << 17),
                                      (50, 1 << 18), (300, 1 << 18)])
def test_logits_of_many_terms(n, hidden):
    """Logits of 32 that are sums of terms of one sign, the same for every word but the label."""
    gen = torch.Generator(device="cuda").manual_seed(hidden)
    vocab = 257
    h = torch.randint(64, 193, (n, hidden), generator=gen, device="cuda").float() / 128
    h = (h / h.mean(1, keepdim=True)).to(BF16)
    word = ((torch.rand(hidden, device="cuda", generator=gen) + 0.5) * 32 / hidden).to(BF16)
    w = word.expand(vocab, hidden).clone()
    w[0] = 0.0
    labels = torch.zeros(n, dtype=torch.int64, device="cuda")
    labels[1::3] = -100
    h.requires_grad_(True)
    w.requires_grad_(True)
    loss = linear_cross_entropy(h, w, labels, reduction="none")
    gh, gw = torch.autograd.grad(loss.sum(), (h, w))
    rows = labels == 0
    z = h.detach().double()[rows] @ word.double()
    assert 30 < z.min() and z.max() < 34
    # chains of 512 terms are off by 2^-23 of their sum with each of 32 additions at most, hidden / 256 of
    # them by 2^-24 of the sum each
    assert ((loss[rows].double() - (z + math.log(vocab - 1))).abs() <= 34 * (2.0 ** -18 + hidden / 256 * 2.0 ** -24) + 2.0 ** -16).all()
    total = h.detach().double()[rows].sum(0)
    # 1 - p is 1 to 2^-37.  A chain of 8192 terms is 512 additions, each off by 2^-23 of its sum at most: all
    # chains together 34 2^-14 < 2^-8.9 in a logit, as much in d; the chains add up in fp32; d and the result
    # round to bf16
    for got, want in ((gw[0], -total), (gw[1:], total / (vocab - 1))):
        assert ((got.double() - want).abs() <= (2 * 2.0 ** -8 + 2.0 ** -8.9 + 2.0 ** -12) * want.abs()).all()
    want = word.double().expand(int(rows.sum()), hidden)
    assert ((gh[rows].double() - want).abs() <= (2 * 2.0 ** -8 + 2.0 ** -8.9 + 2.0 ** -12) * want.abs()).all()
    assert (gh[~rows] == 0).all()


@gpu
@pytest.mark.parametrize("n,hidden,vocab", [(20, 8264, 700), (300, 8264, 1025), (700, 12288, 4099)])
def test_random_logits_of_many_terms(n, hidden, vocab):
    gen = torch.Generator(device="cuda").manual_seed(n)
    h = torch.randn(n, hidden, device="cuda", generator=gen).to(BF16).requires_grad_(True)
    w = (torch.randn(vocab, hidden, device="cuda", generator=gen) / math.sqrt(hidden)).to(BF16).requires_grad_(True)
    labels = torch.randint(0, vocab, (n,), device="cuda", generator=gen)
    labels[::5] = -100
    rows = labels != -100
    x, y = h.detach().double()[rows], w.detach().double()
    d = (x @ y.T).softmax(1)
    p = d.clone()
    d[torch.arange(len(x), device="cuda"), labels[rows]] -= 1
    for piece in (None, 256):
        gh, gw = torch.autograd.grad(linear_cross_entropy(h, w, labels, reduction="sum", piece=piece), (h, w))
        # logits below 6, 512 additions in a chain: 2^-23 * 512 * 6 < 2^-11 in each
        off = (d.abs() * 2.0 ** -8 + p * 2.0 ** -10)
        assert ((gh[rows].double() - d @ y).abs() <= off @ y.abs() + (2.0 ** -8 + 2.0 ** -12) * (d.abs() @ y.abs())).all()
        assert ((gw.double() - d.T @ x).abs() <= off.T @ x.abs() + (2 * 2.0 ** -8 + 2.0 ** -12) * (d.abs().T @ x.abs())).all()


# every kind of launch: few rows whose last block joins, or a launch behind it; sums in one chain or
# several; rows that go straight out, splits, pieces, groups of rows
@gpu
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("n,hidden,vocab,piece", [
    (5, 64, 300, None), (40, 72, 3000, None), (8, 136, 9001, 1024), (100, 64, 300, None), (100, 1032, 700, None), (300, 520, 5000, None),
    (300, 264, 5000, 1024), (100, 8264, 300, None), (66000, 64, 300, None)])
def test_a_wait_that_gives_up(n, hidden, vocab, piece, reduction):
    """A pipeline that waits in vain ends its launch: the results of that call are NaN, the next call that
    looks raises, and everything after it is as before."""
    C = _ext.load(required=True)
    gen = torch.Generator(device="cuda").manual_seed(n)
    h = torch.randn(n, hidden, device="cuda", generator=gen).to(BF16).requires_grad_(True)
    w = (torch.randn(vocab, hidden, device="cuda", generator=gen) / math.sqrt(hidden)).to(BF16).requires_grad_(True)
    labels = torch.randint(0, vocab, (n,), device="cuda", generator=gen)
    labels[::4] = -100
    rows = labels != -100
    g = torch.ones(n if reduction == "none" else (), device="cuda")

    def forward():
        return linear_cross_entropy(h, w, labels, reduction=reduction, piece=piece)

    def grads(loss):
        return torch.autograd.grad(loss, (h, w), g, retain_graph=True)

    def in_vain(f, *args):
        before = C.linear_ce_wait_limit(0)
        try:
            out = f(*args)
        finally:
            C.linear_ce_wait_limit(before)
        torch.cuda.synchronize()
        return out

    def all_nan(loss):
        return loss.isnan().all() if reduction == "mean" else loss[rows].isnan().all() and (loss[~rows] == 0).all()

    def gradients_nan(gh, gw):
        return gw.isnan().all() and gh[rows].isnan().all() and (gh[~rows] == 0).all()

    good = forward()
    want = grads(good)
    with torch.no_grad():
        assert all_nan(in_vain(forward))
        with pytest.raises(RuntimeError, match="gave up waiting"):
            forward()
        assert torch.equal(forward(), good)
    lost = in_vain(forward)
    assert all_nan(lost)
    with pytest.raises(RuntimeError, match="gave up waiting"):
        grads(lost)
    assert gradients_nan(*grads(lost))
    again = forward()
    assert torch.equal(again, good)
    assert gradients_nan(*in_vain(grads, again))
    with pytest.raises(RuntimeError, match="gave up waiting"):
        forward()
    again = forward()
    assert torch.equal(again, good)
    for a, b in zip(grads(again), want):
        assert torch.equal(a, b)
    for one in (0, 1):  # one gradient alone
        again = forward()
        alone, = in_vain(torch.autograd.grad, again, (h, w)[one], g)
        assert alone[rows].isnan().all() if one == 0 else alone.isnan().all()
        with pytest.raises(RuntimeError, match="gave up waiting"):
            forward()


@gpu
@pytest.mark.parametrize("n", [20, 300, 5000])
def test_two_labels_outside_the_vocabulary_raise_once(n):
    gen = torch.Generator(device="cuda").manual_seed(n)
    h = torch.randn(n, 64, device="cuda", generator=gen).to(BF16)
    w = torch.randn(300, 64, device="cuda", generator=gen).to(BF16)
    labels = torch.randint(0, 300, (n,), device="cuda", generator=gen)
    want = linear_cross_entropy(h, w, labels)
    bad = labels.clone()
    bad[1], bad[n - 1] = 300, -7
    assert linear_cross_entropy(h, w, bad).isnan()  # waits for it
    with pytest.raises(IndexError, match="label 300 .* outside its vocabulary"):
        linear_cross_entropy(h, w, labels)
    assert torch.equal(linear_cross_entropy(h, w, labels), want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("ignored", [400, -1, -(1 << 62), 1 << 62, 7])
@pytest.mark.parametrize("n", [5, 70])
def test_any_label_may_be_the_ignored_one(n, ignored, reduction, device):
    """Losses and gradients are those with -100 in its place, whatever stands in the ignored rows."""
    gen = torch.Generator().manual_seed(n)
    h = torch.randn(n, 64, generator=gen).to(BF16).to(device)
    w = (torch.randn(300, 64, generator=gen) / 8).to(BF16).to(device).requires_grad_(True)
    labels = torch.randint(8, 300, (n,), generator=gen).to(device)
    out = torch.arange(n, device=device) % 3 == 1
    h[out] = math.nan
    h.requires_grad_(True)
    results = []
    for index in (-100, ignored):
        loss = linear_cross_entropy(h, w, torch.where(out, index, labels), reduction=reduction, ignore_index=index)
        gh, gw = torch.autograd.grad(loss.sum(), (h, w))
        assert loss.isfinite().all() and gw.isfinite().all() and gh.isfinite().all()
        assert (gh[out] == 0).all() and (reduction != "none" or (loss[out] == 0).all())
        results.append((loss, gh, gw))
    for a, b in zip(*results):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("n", [5, 100])
def test_losses_of_a_masked_row_to_the_last_bits(n):
    """Every word at the lowest value: each logit is one exact product, the label's is the largest, so
    that log 600 is rounded to fp32 alone."""
    h = torch.zeros(n, 64, device="cuda", dtype=BF16)
    h[:, 0] = 1.0
    w = torch.zeros(600, 64, device="cuda", dtype=BF16)
    w[:, 0] = torch.finfo(BF16).min
    loss = linear_cross_entropy(h, w, torch.arange(n, device="cuda"), reduction="none")
    assert ((loss.double() - math.log(600)).abs() <= 2.0 ** -23 * math.log(600)).all()


@gpu
@pytest.mark.parametrize("n,hidden,vocab,piece", [(66000, 72, 700, 256), (100, 8264, 300, None), (40, 8264, 1300, 512), (300, 520, 5000, 1024)])
def test_long_sums_captured_and_replayed(n, hidden, vocab, piece):
    """Loss and gradients in a graph, replayed on other inputs and another number of rows that count; what
    ignored rows hold reaches nothing."""
    gen = torch.Generator(device="cuda").manual_seed(n)

    def inputs():
        h = torch.randn(n, hidden, device="cuda", generator=gen).to(BF16)
        w = (torch.randn(vocab, hidden, device="cuda", generator=gen) / math.sqrt(hidden)).to(BF16)
        labels = torch.randint(0, vocab, (n,), device="cuda", generator=gen)
        out = torch.rand(n, device="cuda", generator=gen) < 0.5 * torch.rand((), device="cuda", generator=gen)
        labels[out], h[out] = -100, math.nan
        return h, w, labels

    def step(x, y, labels):
        loss = linear_cross_entropy(x, y, labels, piece=piece)
        return (loss.detach(),) + torch.autograd.grad(loss, (x, y))

    h, w, labels = inputs()
    x, y = h.requires_grad_(True), w.requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step(x, y, labels)
        with torch.cuda.graph(graph, stream=side):
            outs = step(x, y, labels)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        a, b, c = inputs()
        want = step(a.requires_grad_(True), b.requires_grad_(True), c)
        assert want[0].isfinite() and want[1].isfinite().all() and want[2].isfinite().all()
        with torch.no_grad():
            x.copy_(a)
            y.copy_(b)
            labels.copy_(c)
        graph.replay()
        torch.cuda.synchronize()
        for got, ref in zip(outs, want):
            assert torch.equal(got, ref)


@gpu
@pytest.mark.parametrize("n", [3, 100])
def test_in_inference_mode(n):
    gen = torch.Generator(device="cuda").manual_seed(n)
    h = torch.randn(n, 64, device="cuda", generator=gen).to(BF16)
    w = torch.randn(300, 64, device="cuda", generator=gen).to(BF16)
    labels = torch.randint(0, 300, (n,), device="cuda", generator=gen)
    for reduction in ("mean", "none"):
        want = linear_cross_entropy(h, w, labels, reduction=reduction)
        with torch.inference_mode():
            assert torch.equal(linear_cross_entropy(h, w, labels, reduction=reduction), want)
