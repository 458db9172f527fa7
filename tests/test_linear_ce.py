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
    # each entry of d and the result round to bf16, by up to 2^-8 of their value, and so do the rows
    # of h, times 1 - p and g, that go into gw; an error of e in a logit is one of e in d relative
    # to p = d + [label], and of 4 e with the sum's
    e = _logit_error(h.shape[1], z)
    p = (d.abs() + torch.zeros_like(d).index_put_((at, lab), scale.abs().expand(len(rows)))) * 4 * e
    off = 2.0 ** -8 * d.abs() + p
    tol_h = torch.zeros_like(h)
    tol_h[rows] = off @ w.abs()
    return result, gh, gw, tol_h + 2.0 ** -8 * gh.abs() + 1e-30, \
        (off + 2.0 ** -8 * (1 + 2.0 ** -8) * d.abs()).T @ x.abs() + 2.0 ** -8 * gw.abs() + 1e-30


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
# the narrow products (16 and 64), are packed a block or a warp each (512) or in two launches (4096),
# inner sizes around a stage (64) and a chain of sums (512)
SIZES = [(1, 8, 1), (1, 64, 257), (2, 72, 7), (16, 264, 300), (17, 72, 129), (63, 64, 128), (64, 128, 127), (64, 1032, 5000), (65, 256, 129), (127, 264, 255),
         (128, 8, 256), (129, 840, 513), (255, 64, 1000), (256, 256, 1024), (257, 520, 2049), (700, 136, 4099),
         (512, 64, 300), (513, 72, 300), (4096, 8, 65), (4097, 16, 130), (9000, 8, 40), (130, 1032, 700), (300, 128, 5000)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("n,hidden,vocab", SIZES)
def test_matches_64_bits(n, hidden, vocab, reduction, device):
    _check(*_inputs(n, hidden, vocab, device), reduction)


# pieces that end with one word, and that leave some splits of the sum over the words nothing
@gpu
@pytest.mark.parametrize("piece", [1, 256, 300, 768, 2048, 4096, 1 << 62])
@pytest.mark.parametrize("n,hidden,vocab", [(3, 64, 2561), (40, 136, 2100), (20, 64, 4097), (70, 64, 4097), (300, 200, 2560), (513, 96, 1025)])
def test_pieces(n, hidden, vocab, piece):
    _check(*_inputs(n, hidden, vocab, "cuda"), "mean", piece=piece)


# the head's gradient of few rows has tiles of 128 words and 256 columns, which a block takes along
# the rows: shares that begin and end within a row of tiles, of one tile, of none; ends that are odd
@gpu
@pytest.mark.parametrize("ignored", [0.0, 0.6, 1.0])
@pytest.mark.parametrize("n,hidden,vocab,piece", [(33, 1288, 9001, None), (64, 264, 20001, None), (1, 2056, 5121, None), (17, 776, 19000, 8192),
                                                  (5, 4104, 1153, None), (64, 8, 30001, 16384), (48, 136, 18945, None)])
def test_few_rows_and_many_words(n, hidden, vocab, piece, ignored):
    _check(*_inputs(n, hidden, vocab, "cuda", ignored=ignored), "mean", piece=piece)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n", [5, 70])
def test_ignored_rows_take_no_part(n, device):
    """Whatever stands in them: a padded batch's NaN and infinities reach no sum."""
    h, w, labels, g = _inputs(n, 64, 300, device, ignored=0.0)
    labels[n // 2:] = -100
    clean = _run(h, w, labels, g, "sum")
    h[n // 2:] = math.nan
    h[-1] = math.inf
    got = _run(h, w, labels, g, "sum")
    for a, b in zip(clean, got):
        assert torch.equal(a, b)
    assert (got[1][n // 2:] == 0).all()
    each = _run(h, w, labels, g, "none")
    assert (each[0][n // 2:] == 0).all() and (each[0][:n // 2] > 0).all()
    # another label that is ignored
    again = _run(h, w, torch.where(labels == -100, 7, labels), g, "sum", ignore_index=7) if not (labels == 7).any() else got
    assert torch.equal(got[0], again[0])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n", [3, 100])
def test_no_row_counts(n, device):
    h, w, labels, g = _inputs(n, 64, 300, device)
    labels.fill_(-100)
    for reduction in ("mean", "sum", "none"):
        loss, gh, gw = _run(h, w, labels, g, reduction)
        assert (loss == 0).all() and (gh == 0).all() and (gw == 0).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.float16])
def test_other_dtypes(dtype, device):
    h, w, labels, g = _inputs(40, 36, 300, device, dtype=dtype)
    got, want = _run(h, w, labels, g, "mean", piece=77), _exact(h, w, labels, g, "mean")
    eps = max(torch.finfo(dtype).eps, 2.0 ** -20 if dtype != torch.float64 else 0)
    for a, b in zip(got, want):
        assert a.dtype == (dtype if a.dim() else torch.promote_types(dtype, torch.float32))
        assert ((a.double() - b).abs() <= 16 * eps * (b.abs() + b.abs().max())).all()


def test_gradients_against_differences():
    """The plain route in fp64: (f(x + e) - f(x - e)) / 2 e, off by e^2 and 1e-16 / e."""
    h, w, labels, g = _inputs(6, 5, 11, "cpu", dtype=torch.float64)
    g = g.double()
    for reduction in ("none", "mean"):
        def f(a, b):
            loss = linear_cross_entropy(a, b, labels, reduction=reduction, piece=4)
            return (loss * g).sum() if reduction == "none" else loss
        assert torch.autograd.gradcheck(f, (h.requires_grad_(True), w.requires_grad_(True)), eps=1e-5, atol=1e-8)


@gpu
def test_gradient_against_differences_on_the_gpu():
    """Along one direction: what the loss changes by against the gradient's product with it."""
    h, w, labels, g = _inputs(128, 256, 1000, "cuda", ignored=0.0)
    _, gh, gw = _run(h, w, labels, torch.ones_like(g), "sum")
    # steps that bf16 holds exactly: one bit of every value of h (or w) up and down
    for x, grad, at in ((h, gh, 0), (w, gw, 1)):
        step = 2.0 ** -6 * x.abs().double()
        bits = x.view(torch.int16)
        up, down = (bits + 2).view(torch.bfloat16), (bits - 2).view(torch.bfloat16)  # away from 0, towards 0
        ok = (x.abs() > 1e-3) & (up.isfinite()) & ((up.double() - x.double()).abs() <= step)
        sign = grad.double().sign() * x.double().sign()  # so that all contributions add up
        plus, minus = torch.where(sign > 0, up, down), torch.where(sign > 0, down, up)
        plus, minus = torch.where(ok, plus, x), torch.where(ok, minus, x)
        pair = [(plus, w) if at == 0 else (h, plus), (minus, w) if at == 0 else (h, minus)]
        with torch.no_grad():
            a, b = (linear_cross_entropy(p, q, labels, reduction="sum").double() for p, q in pair)
        change = ((plus.double() - minus.double()) * grad.double()).sum()
        # third-order terms: steps of up to 2^-6 of each value move logits by a few hundredths
        assert abs((a - b) - change) <= 0.02 * abs(change)


@gpu
@pytest.mark.parametrize("n", [9, 130])
def test_layouts_in_place_and_copied(n):
    """Rows with a pitch, at any element, transposed, expanded, batched."""
    h, w, labels, g = _inputs(n, 72, 300, "cuda")
    plain = _run(h, w, labels, g, "mean")

    def variant(x, how):
        if how == "pitch":
            y = torch.full((x.shape[0], x.shape[1] + 24), math.nan, device="cuda", dtype=x.dtype)[:, 8:8 + x.shape[1]]
        elif how == "odd pitch":
            y = torch.full((x.shape[0], x.shape[1] + 3), math.nan, device="cuda", dtype=x.dtype)[:, :x.shape[1]]
        elif how == "odd start":
            y = torch.full((x.numel() + 1,), math.nan, device="cuda", dtype=x.dtype)[1:].view(x.shape)
        else:
            y = torch.empty((x.shape[1], x.shape[0]), device="cuda", dtype=x.dtype).T
        return y.copy_(x)

    for a in ("pitch", "odd pitch", "odd start", "turned"):
        for b in ("pitch", "odd pitch", "odd start", "turned"):
            x, y = variant(h, a).requires_grad_(True), variant(w, b).requires_grad_(True)
            loss = linear_cross_entropy(x, y, labels)
            gx, gy = torch.autograd.grad(loss, (x, y), g[0])
            assert torch.equal(loss, plain[0]) and torch.equal(gx, plain[1]) and torch.equal(gy, plain[2])
    one = h[:1].expand(n, 72).detach().requires_grad_(True)
    loss = linear_cross_entropy(one, w, labels)
    dense = linear_cross_entropy(one.detach().contiguous(), w, labels)
    assert torch.equal(loss, dense)
    batch = torch.cat([h, h[:1]]).view(1, n + 1, 72)[:, :-1].expand(2, n, 72)
    each = linear_cross_entropy(batch, w, labels.expand(2, n), reduction="none")
    assert each.shape == (2, n) and torch.equal(each[0], each[1])
    assert torch.equal(each[0], linear_cross_entropy(h, w, labels, reduction="none"))


# one launch joins the sums of up to 8 rows (4 beyond 65536 words), another one those of more
@gpu
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("n,vocab", [(1, 131072), (1, 131073), (4, 65537), (5, 65537), (8, 65536), (9, 65536), (8, 65537), (3, 100)])
def test_rows_have_the_same_loss_in_any_company(n, vocab, reduction):
    h, w, labels, _ = _inputs(n + 30, 16, vocab, "cuda", ignored=0.0)
    all_rows = linear_cross_entropy(h, w, labels, reduction="none")
    some = labels.clone()
    some[n:] = -100
    some[0] = -100
    for x, y, want in ((h[:n], labels[:n], all_rows[:n]), (h[:n], some[:n], torch.where(some[:n] < 0, 0.0, all_rows[:n]))):
        got = linear_cross_entropy(x, w, y, reduction=reduction)
        rows = int((y >= 0).sum())
        if reduction == "none":
            assert torch.equal(got, want)
        else:  # summed in fp64 and rounded once; the mean takes 1 / rows in fp32
            exact = want.double().sum() / (max(1, rows) if reduction == "mean" else 1)
            assert abs(got.double() - exact) <= exact * (2.0 ** -23 + 2.0 ** -24)


@gpu
@pytest.mark.parametrize("n", [5, 100])
def test_logits_of_any_size(n):
    """Infinite ones, the lowest finite ones, a row that one word fills."""
    h, w, labels, _ = _inputs(n, 64, 600, "cuda", ignored=0.0)
    h[:, 0], w[:, 0], w[:, 1] = 1.0, 0.0, 0.0
    h[:, 1] = 0.0
    w[::2, 0] = torch.finfo(torch.bfloat16).min  # every other word as good as masked
    labels = labels | 1
    w[7, 1], h[1, 1] = 40.0, 10.0                # row 1: word 7 is sure
    got = _run(h, w, labels, torch.ones(n, device="cuda"), "none")
    z = h.double() @ w.double().T
    want = torch.logsumexp(z, 1) - z[torch.arange(n, device="cuda"), labels]
    assert ((got[0].double() - want).abs() <= _logit_error(64, z[:, 1::2]) + 2.0 ** -22 * want.abs()).all()
    assert got[1].isfinite().all() and got[2].isfinite().all()
    assert (got[2][::2] == 0).all()
    lowest = torch.zeros(n, 64, device="cuda", dtype=torch.bfloat16)
    lowest[:, 0] = 1.0
    head = torch.zeros(600, 64, device="cuda", dtype=torch.bfloat16)
    head[:, 0] = torch.finfo(torch.bfloat16).min  # all of a row: each word is as likely
    loss = linear_cross_entropy(lowest, head, labels, reduction="none")
    # the sum's logarithm is lost beside 3.4e38
    assert loss.isfinite().all() and ((loss - math.log(600)).abs() <= math.log(600) + 1).all()
    h[0, 0] = math.inf
    plain, ours = torch.nn.functional.cross_entropy(h.float() @ w.float().T, labels, reduction="none"), \
        linear_cross_entropy(h, w, labels, reduction="none")
    assert torch.equal(plain.isfinite(), ours.isfinite())


@gpu
@pytest.mark.parametrize("n", [20, 300])
def test_label_outside_the_vocabulary_is_refused(n):
    h, w, labels, g = _inputs(n, 64, 1000, "cuda")
    for bad_label in (1000, -1, 1 << 40):
        bad = labels.clone()
        bad[n // 2] = bad_label
        with torch.no_grad():
            assert linear_cross_entropy(h, w, bad).isnan()  # waits for it
            with pytest.raises(IndexError, match=f"label {bad_label} .* outside its vocabulary"):
                linear_cross_entropy(h, w, labels)
    good = _run(h, w, labels, g, "mean")
    assert good[0].isfinite()


@gpu
def test_same_bits_again_on_another_stream_and_in_another_thread():
    import threading

    args = _inputs(333, 264, 3000, "cuda")
    first = _run(*args, "mean", piece=1024)
    results = []

    def work():
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(s):
            results.append(_run(*args, "mean", piece=1024))
        s.synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    work()
    assert len(results) == 4
    for r in results:
        for a, b in zip(first, r):
            assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("n", [20, 200])
def test_captured_and_replayed(n):
    """Two graphs of one loss each, replayed in turn on inputs that change."""
    jobs = [_inputs(n, 64, 1000, "cuda", seed=s) for s in (0, 1)]
    want = [_run(*j, "mean") for j in jobs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs, leaves = [], [], []
    with torch.cuda.stream(side):
        for h, w, labels, g in jobs:
            x, y = h.clone().requires_grad_(True), w.clone().requires_grad_(True)

            def step():
                loss = linear_cross_entropy(x, y, labels)
                return (loss.detach(),) + torch.autograd.grad(loss, (x, y), g[0])

            step()  # the first call allocates what it keeps
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(step())
            graphs.append(graph)
            leaves.append((x, y))
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for out, ref in zip(outs, want):
        for a, b in zip(out, ref):
            assert torch.equal(a, b)
    with torch.no_grad():
        leaves[0][0].copy_(jobs[1][0])
        leaves[0][1].copy_(jobs[1][1])
        jobs[0][2].copy_(jobs[1][2])
        jobs[0][3].copy_(jobs[1][3])
    graphs[0].replay()
    torch.cuda.synchronize()
    for a, b in zip(outs[0], want[1]):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("n", [3, 8])
def test_scores_of_few_rows_replayed_and_side_by_side(n, reduction):
    """Without a graph, in one launch for the product and its sums: captured twice, replayed with other
    labels, the two replays at the same time on two streams."""
    jobs = [_inputs(n, 72, 5000, "cuda", ignored=0.3, seed=s) for s in range(2)]

    def score(job):
        with torch.no_grad():
            return linear_cross_entropy(*job[:3], reduction=reduction)

    streams, graphs, outs = [torch.cuda.Stream() for _ in jobs], [], []
    for job, stream in zip(jobs, streams):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            score(job)
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=stream):
                outs.append(score(job))
    for k in range(4):
        torch.cuda.synchronize()
        for job in jobs:
            job[2].copy_(job[2].roll(1))
        want = [score(job) for job in jobs]
        torch.cuda.synchronize()
        for _ in range(20):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for out, ref in zip(outs, want):
            assert torch.equal(out, ref)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n", [20, 70])
def test_one_gradient_no_gradient_and_a_graph_used_twice(n, device):
    h, w, labels, g = _inputs(n, 64, 5000, device)
    both = _run(h, w, labels, g, "mean")
    for want_h, want_w in ((True, False), (False, True)):
        x, y = h.clone().requires_grad_(want_h), w.clone().requires_grad_(want_w)
        linear_cross_entropy(x, y, labels).backward(g[0])
        assert (x.grad is not None) == want_h and (y.grad is not None) == want_w
        assert torch.equal(x.grad if want_h else y.grad, both[1] if want_h else both[2])
    with torch.no_grad():
        assert not linear_cross_entropy(h, w, labels).requires_grad
    x = h.clone().requires_grad_(True)
    loss = linear_cross_entropy(x, w, labels)
    a, = torch.autograd.grad(loss, x, retain_graph=True)
    b, = torch.autograd.grad(loss, x, retain_graph=True)
    assert torch.equal(a, b)
    scale = torch.ones((), device=device, requires_grad=True)
    c, = torch.autograd.grad(loss * scale, x, create_graph=True)
    assert torch.equal(a, c)
    with pytest.raises(RuntimeError, match="second derivative|differentiate twice"):
        c.float().sum().backward()


@gpu
def test_saved_tensors_may_move():
    args = _inputs(100, 64, 1001, "cuda")
    plain = _run(*args, "none")
    with torch.autograd.graph.save_on_cpu():
        moved = _run(*args, "none")
    for a, b in zip(plain, moved):
        assert torch.equal(a, b)


@gpu
def test_no_logits_are_kept():
    """Forward: a hundredth of the logits, beside the packed rows.  Backward: one piece."""
    n, hidden, vocab = 2048, 256, 32000
    h, w, labels, _ = _inputs(n, hidden, vocab, "cuda")
    h.requires_grad_(True)
    w.requires_grad_(True)
    linear_cross_entropy(h, w, labels, piece=1024).backward()  # whatever the first call takes
    h.grad = w.grad = None
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    loss = linear_cross_entropy(h, w, labels, piece=1024)
    rows = 2 * n * hidden
    assert torch.cuda.max_memory_allocated() - before <= rows + 16 * n * vocab / 128 + (1 << 20)
    assert torch.cuda.memory_allocated() - before <= rows + (1 << 20)
    loss.backward()
    grads = 2 * hidden * (n + vocab)
    # packed rows, one piece in bf16, the sums of the hidden states' gradient, the gradients
    assert torch.cuda.max_memory_allocated() - before <= rows + 2 * n * 1024 + 4 * n * hidden + grads + (4 << 20)


def test_refusals():
    h, w, labels, _ = _inputs(6, 8, 20, "cpu", dtype=torch.float32)
    for kw, error, match in (
            (dict(reduction="max"), ValueError, "reduction"), (dict(piece=-1), ValueError, "piece"),
            (dict(piece=2.5), ValueError, "piece"), (dict(piece=True), ValueError, "piece")):
        with pytest.raises(error, match=match):
            linear_cross_entropy(h, w, labels, **kw)
    for args, match in (((h[:, :4], w, labels), "do not fit"), ((h, w[:0], labels), "do not fit"), ((h, w[0], labels), "do not fit"),
                        ((h, w, labels[:3]), "labels"), ((h, w, labels.int()), "labels"),
                        ((h, w.double(), labels), "float64"), ((h.long(), w.long(), labels), "int64")):
        with pytest.raises(ValueError, match=match):
            linear_cross_entropy(*args)
    for bad in (20, -1):
        with pytest.raises(IndexError, match="outside the vocabulary"):
            linear_cross_entropy(h, w, torch.full_like(labels, bad))
    from offload_adam_b200.qweight import Int8QWeight
    with pytest.raises(TypeError, match="packed"):
        linear_cross_entropy(h, torch.nn.Parameter(Int8QWeight.from_float(w)), labels)
    assert linear_cross_entropy(h[:0], w, labels[:0]) == 0
    assert linear_cross_entropy(h[:0], w, labels[:0], reduction="none").shape == (0,)


@gpu
def test_refusals_on_the_gpu():
    h, w, labels, _ = _inputs(6, 8, 20, "cuda")
    with pytest.raises(ValueError, match="one device"):
        linear_cross_entropy(h, w.cpu(), labels)
    with pytest.raises(ValueError, match="one device"):
        linear_cross_entropy(h, w, labels.cpu())
    C = _ext.load(required=True)
    for args in ((h.float(), w.float(), labels, 1, -100, 0), (h[:, :4], w[:, :4], labels, 1, -100, 0),
                 (h, w, labels.int(), 1, -100, 0), (h, w, labels, 3, -100, 0), (h, w, labels, 1, -100, -1)):
        with pytest.raises(RuntimeError, match="linear_cross_entropy"):
            C.linear_ce(*args)
    assert linear_cross_entropy(h[:0], w, labels[:0]) == 0
    # hidden sizes that the kernels do not take run PyTorch's operations
    h, w, labels, g = _inputs(30, 12, 50, "cuda")
    _check(h, w, labels, g, "mean")


@gpu
def test_kernels_run_under_autocast():
    h, w, labels, g = _inputs(100, 64, 3000, "cuda")
    want = _run(h, w, labels, g, "mean")
    x, y = h.float().requires_grad_(True), w.float().requires_grad_(True)
    C = _ext.load(required=True)
    before = C.launch_count()
    with torch.autocast("cuda", torch.bfloat16):
        loss = linear_cross_entropy(x, y, labels)
    assert C.launch_count() > before
    loss.backward(g[0])
    assert torch.equal(loss.detach(), want[0]) and torch.equal(x.grad, want[1].float()) and torch.equal(y.grad, want[2].float())
    with torch.autocast("cuda", torch.bfloat16), pytest.raises(ValueError, match="one device"):
        linear_cross_entropy(x, y, labels.cpu())


@pytest.mark.parametrize("device", DEVICES)
def test_under_autocast(device):
    h, w, labels, g = _inputs(40, 64, 300, device)
    plain = _run(h, w, labels, g, "mean")
    x, y = h.float().requires_grad_(True), w.float().requires_grad_(True)
    with torch.autocast(device, dtype=torch.bfloat16):
        loss = linear_cross_entropy(x, y, labels)
    loss.backward(g[0])
    assert x.grad.dtype == y.grad.dtype == torch.float32
    assert abs(loss - plain[0]) <= 1e-5 * plain[0]
    for a, b in ((x.grad, plain[1]), (y.grad, plain[2])):
        assert (a - b.float()).norm() <= 3 * 2.0 ** -8 * b.float().norm()


# ------------------------------------------------------------------ as it is used
def _tiny(device, **kw):
    from offload_adam_b200.models.llama import build_llama, tiny_llama
    return build_llama(tiny_llama(**kw), device=device, seed=0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("tied", [True, False])
@pytest.mark.parametrize("piece", [0, 300])
def test_model_with_pieces(device, tied, piece):
    """The model's loss in pieces against its loss in chunks of rows: both round the gradients to
    bf16, the chunks the logits as well."""
    chunks, pieces = _tiny(device, tie_embeddings=tied), _tiny(device, tie_embeddings=tied, ce_piece=piece)
    ids = torch.randint(0, 1024, (2, 70), generator=torch.Generator().manual_seed(3)).to(device)
    labels = ids.clone()
    labels[:, :9] = -100
    a, b = chunks(ids, labels=labels), pieces(ids, labels=labels)
    assert abs(a.item() - b.item()) <= 2.0 ** -8 * abs(a.item())
    a.backward()
    b.backward()
    for (name, p), q in zip(chunks.named_parameters(), pieces.parameters()):
        off = (p.grad.double() - q.grad.double()).norm() / p.grad.double().norm()
        assert off <= 4 * 2.0 ** -8, name  # the logits' rounding, and each route's own


@pytest.mark.parametrize("device", DEVICES)
def test_huggingface_loss_with_pieces(device):
    transformers = pytest.importorskip("transformers")
    from offload_adam_b200.models.hf import causal_lm_loss
    cfg = transformers.LlamaConfig(vocab_size=512, hidden_size=128, intermediate_size=256, num_hidden_layers=1,
                                   num_attention_heads=4, num_key_value_heads=2, tie_word_embeddings=False, use_cache=False)
    torch.manual_seed(0)
    model = transformers.LlamaForCausalLM(cfg).to(torch.bfloat16).to(device).train()
    ids = torch.randint(0, 512, (2, 32), generator=torch.Generator().manual_seed(5)).to(device)
    want = model(input_ids=ids, labels=ids).loss
    got = causal_lm_loss(model, ids, piece=256)
    assert abs(got.item() - want.item()) <= 2.0 ** -8 * want.item()
    got.backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in model.parameters())


@pytest.mark.parametrize("device", DEVICES)
def test_loss_norm_clipping_and_step_together(device):
    """One training step in the new operators against the same in fp32 PyTorch on the same
    gradients: loss, norm, clipped gradients and the step's parameters."""
    from offload_adam_b200 import Adam, clip_grad_norm_, grad_norm
    bound = 0.05
    one, two = _tiny(device, ce_piece=256), _tiny(device, ce_piece=256)
    # decoupled, as in the trainers: a decay that is added to the gradient can cancel it, and then the
    # last bit of the gradient decides the step's sign
    kw = dict(lr=1e-2, mode="fp32_master", decoupled_weight_decay=True)
    inside, after = Adam(one.parameters(), max_grad_norm=bound, **kw), Adam(two.parameters(), **kw)
    gen = torch.Generator().manual_seed(4)
    for it in range(2):
        ids = torch.randint(0, 1024, (2, 64), generator=gen).to(device)
        for model in (one, two):
            model.zero_grad()
            model(ids, labels=ids).backward()
        norm = grad_norm(two.parameters())
        want = torch.sqrt(sum(p.grad.double().square().sum() for p in two.parameters()))
        assert abs(norm.item() - want.item()) <= 2.0 ** -23 * want.item()
        assert norm.item() > bound
        assert torch.equal(clip_grad_norm_(two.parameters(), bound), norm)
        assert grad_norm(two.parameters()).item() <= bound * (1 + 2.0 ** -8)
        inside.step()
        after.step()
        assert all(p.isfinite().all() for p in one.parameters())
        if it > 0:
            continue  # the weights, and with them the gradients, are apart by roundings from here on
        assert inside.grad_norm == norm
        for p, q in zip(one.parameters(), two.parameters()):
            # the first step is lr g / (|g| + eps): off by less than lr where g is off by its rounding to
            # bf16, 2^-8; and the weights round to bf16
            assert ((p.double() - q.double()).abs() <= 1e-2 * 2.0 ** -7 + 2.0 ** -7 * q.double().abs()).all()
