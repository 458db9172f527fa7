"""The last part of a training step, measured operator by operator: the loss over a large
vocabulary and its gradients, the global norm of the gradients, and their clipping.

Four kinds of case:

``score``  the loss of every token, forward only (evaluation, log-probabilities of answers).
``loss``   the loss and the gradients of the hidden states and of the head's weight.
``norm``   the global norm of all gradients of a model (what a trainer logs).
``clip``   the norm, and all gradients scaled in place to at most ``max_norm``.
"""

import math

import torch

own = False  # True: the package's operators; False: their plain form in elementary PyTorch

IGNORE = -100
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _loss(kind, tokens, hidden, vocab, reduction, ignored):
    return dict(kind=kind, tokens=tokens, hidden=hidden, vocab=vocab, reduction=reduction, ignored=ignored)


def _grads(kind, hidden, inter, kv, layers, vocab, dtype, norm="2", tied=False, flat=False):
    """``dtype`` "mixed": matrices in bf16, vectors and the embedding in fp32.  ``flat``: all
    gradients are views of one buffer, one behind the other."""
    return dict(kind=kind, hidden=hidden, inter=inter, kv=kv, layers=layers, vocab=vocab, dtype=dtype, norm=norm,
                tied=tied, flat=flat)


def listed():
    return [
        # log-probability of one token under the 8B head: the weight is read once, 1.05 GB
        _loss("score", 1, 4096, 128256, "none", 0.0) | dict(name="score_token"),
        # a prompt's log-probabilities under the head of the 8B model with the larger vocabulary
        _loss("score", 2048, 4096, 151936, "none", 0.0) | dict(name="score_prompt"),
        # the smallest training step: tiny_llama, 2 x 128 tokens
        _loss("loss", 256, 256, 1024, "mean", 0.0) | dict(name="loss_tiny"),
        # a ragged batch, odd sizes, padding ignored
        _loss("loss", 777, 840, 32003, "mean", 0.2) | dict(name="loss_ragged"),
        # a short answer under the 70B head: few rows, 2.1 GB of weight
        _loss("loss", 32, 8192, 128256, "mean", 0.0) | dict(name="loss_few_rows"),
        # fine-tuning: prompts ignored (half of the tokens), a weight for each token
        _loss("loss", 4096, 4096, 151936, "none", 0.5) | dict(name="loss_finetune"),
        # pre-training: 4096 tokens under the 8B head
        _loss("loss", 4096, 4096, 128256, "mean", 0.0) | dict(name="loss_wide"),
        # tiny_llama: 20 small tensors, bound by launches and by the host
        _grads("clip", 256, 688, 256, 2, 1024, "bf16", tied=True) | dict(name="clip_tiny"),
        # 291 tensors of odd sizes in one bucket: starts at any element
        _grads("clip", 250, 667, 125, 32, 5001, "bf16", flat=True) | dict(name="clip_bucket"),
        # odd dimensions, fp32 gradients of vectors and embedding beside bf16 matrices
        _grads("clip", 840, 2241, 420, 1, 32003, "mixed") | dict(name="clip_mixed"),
        # one layer of the 8B shape with embedding and head: 1.3 G gradients
        _grads("clip", 4096, 14336, 1024, 1, 128256, "bf16") | dict(name="clip_wide"),
        # the same, norm only
        _grads("norm", 4096, 14336, 1024, 1, 128256, "bf16") | dict(name="norm_wide"),
    ]


# ---------------------------------------------------------------------------- draw
MOST_PRODUCTS = 4096 * 4096 * 128256  # tokens x hidden x vocab of the largest listed case
MOST_ELEMENTS = 1.2e9


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def draw(rng):
    """One more case of the ranges above."""
    if rng.random() < 0.6:
        kind = rng.choice(["score", "loss", "loss"])
        while True:
            hidden = max(8, int(_log(rng, 64, 8200)) // 8 * 8)
            vocab = int(_log(rng, 500, 152000))
            tokens = int(_log(rng, 1, 8200))
            if rng.random() < 0.5:
                vocab, tokens = max(64, vocab // 64 * 64), max(1, tokens // 16 * 16)
            if tokens * hidden * vocab <= MOST_PRODUCTS and tokens * vocab <= 4096 * 152000:
                break
        return _loss(kind, tokens, hidden, vocab, rng.choice(["mean", "sum", "none"]), rng.choice([0.0, 0.1, 0.3, 0.7]))
    kind = rng.choice(["clip", "clip", "norm"])
    dtype = rng.choice(["bf16", "bf16", "fp32", "fp16", "mixed"])
    while True:
        hidden = int(_log(rng, 64, 4200))
        if rng.random() < 0.5:
            hidden = max(64, hidden // 64 * 64)
        layers = int(_log(rng, 1, 40))
        inter = int(hidden * rng.uniform(2.0, 4.0))
        vocab = int(_log(rng, 500, 130000))
        flat = layers > 5 or (dtype != "mixed" and rng.random() < 0.3)
        if flat and dtype == "mixed":
            dtype = "bf16"
        c = _grads(kind, hidden, inter, max(1, hidden // rng.choice([1, 2, 4, 8])), layers, vocab, dtype,
                   rng.choice(["2", "2", "2", "1", "inf"]), rng.random() < 0.4, flat)
        if sum(math.prod(s) for s in _shapes(c)) * (2 if dtype in ("fp32", "mixed") else 1) <= MOST_ELEMENTS:
            return c


# ------------------------------------------------------------------------- prepare
def _shapes(c):
    """Shapes of a Llama-shaped model's parameters."""
    h, i, kv = c["hidden"], c["inter"], c["kv"]
    layer = [(h,), (h, h), (kv, h), (kv, h), (h, h), (h,), (i, h), (i, h), (h, i)]
    return [(c["vocab"], h)] + layer * c["layers"] + [(h,)] + ([] if c["tied"] else [(c["vocab"], h)])


def _dtype_of(c, index, shape):
    if c["dtype"] == "mixed":
        return torch.float32 if index == 0 or len(shape) == 1 else torch.bfloat16
    return DTYPES[c["dtype"]]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] in ("score", "loss"):
        n, hidden, vocab = case["tokens"], case["hidden"], case["vocab"]
        w = torch.empty(vocab, hidden, device="cuda", dtype=torch.bfloat16).normal_(std=0.02, generator=gen)
        labels = torch.randint(0, vocab, (n,), device="cuda", generator=gen)
        h = torch.randn(n, hidden, device="cuda", generator=gen)  # what the last norm leaves
        # a trained model is sure of many tokens: their state points at the label's row
        sure = (torch.rand(n, 1, device="cuda", generator=gen) < 0.5).float()
        h += sure * 12.0 / (0.02 ** 2 * hidden) * w[labels].float()
        labels[torch.rand(n, device="cuda", generator=gen) < case["ignored"]] = IGNORE
        state = dict(kind=case["kind"], h=h.to(torch.bfloat16), w=w, labels=labels, reduction=case["reduction"])
        if case["kind"] == "loss":
            state["h"].requires_grad_(True)
            state["w"].requires_grad_(True)
            # the share of a micro-batch, or a weight for each token
            state["g"] = (torch.rand(n, device="cuda", generator=gen) / n if case["reduction"] == "none" else
                          torch.full((), 0.25 if case["reduction"] == "mean" else 0.25 / n, device="cuda"))
        return state
    shapes = _shapes(case)
    if case["flat"]:
        flat = torch.empty(sum(math.prod(s) for s in shapes), device="cuda", dtype=DTYPES[case["dtype"]])
        pieces = [t.view(s) for t, s in zip(flat.split([math.prod(s) for s in shapes]), shapes)]
    else:
        flat = None
        pieces = [torch.empty(s, device="cuda", dtype=_dtype_of(case, i, s)) for i, s in enumerate(shapes)]
    params = []
    for piece in pieces:
        # gradients of different tensors differ in size
        piece.normal_(std=1e-3 * math.exp(torch.randn((), generator=gen, device="cuda").item()), generator=gen)
        p = torch.nn.Parameter(torch.empty_like(piece))
        p.grad = piece
        params.append(p)
    norm = float(case["norm"])
    size = torch.stack([torch.linalg.vector_norm(p.grad, norm, dtype=torch.float32) for p in params])
    return dict(kind=case["kind"], params=params, flat=flat, norm=norm,
                max_norm=0.3 * torch.linalg.vector_norm(size, norm).item())


# ----------------------------------------------------------------------------- run
def _plain_loss(state):
    h, w, labels = state["h"].detach().float(), state["w"].detach().float(), state["labels"]
    valid = labels != IGNORE
    at = labels.clamp(min=0)[:, None]
    z = h @ w.T
    top = z.amax(1, keepdim=True)
    z = z - top
    picked = z.gather(1, at)[:, 0]
    z = z.exp_()
    total = z.sum(1, dtype=torch.float64)
    losses = (total.log() - picked) * valid
    count = valid.sum().clamp(min=1)
    out = {"none": losses, "sum": losses.sum(), "mean": losses.sum() / count}[state["reduction"]].float()
    if state["kind"] == "score":
        return out
    scale = state["g"].double() / count if state["reduction"] == "mean" else state["g"].double()
    scale = scale * valid
    d = z.mul_((1.0 / total).float()[:, None])
    d.scatter_add_(1, at, torch.full_like(d[:, :1], -1.0))
    d.mul_(scale.float()[:, None])
    return [out, (d @ w).to(torch.bfloat16), (d.T @ h).to(torch.bfloat16)]


def _plain_norm(params, norm):
    each = [p.grad.double() if p.grad.numel() <= 1 << 16 else p.grad.float() for p in params]
    if norm == math.inf:
        return torch.stack([x.abs().amax().float() for x in each]).amax()
    if norm == 1.0:
        return torch.stack([x.abs().sum(dtype=torch.float64) for x in each]).sum().float()
    return torch.stack([x.square().sum(dtype=torch.float64) for x in each]).sum().sqrt().float()


def run(state):
    kind = state["kind"]
    if kind in ("score", "loss"):
        if not own:
            return _plain_loss(state)
        from offload_adam_b200.ops.linear_ce import linear_cross_entropy
        h, w = state["h"], state["w"]
        if kind == "score":
            with torch.no_grad():
                return linear_cross_entropy(h, w, state["labels"], reduction=state["reduction"], ignore_index=IGNORE)
        h.grad = w.grad = None
        loss = linear_cross_entropy(h, w, state["labels"], reduction=state["reduction"], ignore_index=IGNORE)
        loss.backward(state["g"])
        return [loss.detach(), h.grad, w.grad]
    params, norm = state["params"], state["norm"]
    if kind == "norm":
        if not own:
            return _plain_norm(params, norm)
        from offload_adam_b200 import grad_norm
        return grad_norm(params, norm_type=norm)
    # the gradients of a step are there once only: a bound that falls a little from pass to pass
    # leaves every pass something to clip
    max_norm = state["max_norm"]
    state["max_norm"] = max_norm * 0.9999
    if own:
        from offload_adam_b200 import clip_grad_norm_
        total = clip_grad_norm_(params, max_norm, norm_type=norm)
    else:
        total = _plain_norm(params, norm)
        coef = (max_norm / (total + 1e-6)).clamp(max=1.0)
        for p in params:
            p.grad.copy_(p.grad.float() * coef)
    return [total, state["flat"] if state["flat"] is not None else [p.grad for p in params]]


# --------------------------------------------------------------------------- exact
def exact(case, seed):
    """The same from the definitions, in 64 bits."""
    state = prepare(case, seed)
    if case["kind"] in ("norm", "clip"):
        grads, norm = [p.grad for p in state["params"]], state["norm"]
        each = torch.stack([torch.linalg.vector_norm(g, norm, dtype=torch.float64) for g in grads])
        total = torch.linalg.vector_norm(each, norm)
        if case["kind"] == "norm":
            return total
        factor = min(1.0, state["max_norm"] / (total.item() + 1e-6))
        if state["flat"] is not None:
            return [total, state["flat"].double() * factor]
        return [total, [g.double() * factor for g in grads]]
    h, w, labels = state["h"].detach().double(), state["w"].detach().double(), state["labels"]
    n = labels.numel()
    count = max(1, int((labels != IGNORE).sum()))
    losses = torch.zeros(n, device="cuda", dtype=torch.float64)
    gh = torch.zeros_like(h)
    gw = torch.zeros_like(w) if case["kind"] == "loss" else None
    for s in range(0, n, 1024):
        rows = torch.arange(s, min(n, s + 1024), device="cuda")
        rows = rows[labels[rows] != IGNORE]
        if not rows.numel():
            continue
        logp = torch.log_softmax(h[rows] @ w.T, dim=1)
        here = torch.arange(rows.numel(), device="cuda")
        losses[rows] = -logp[here, labels[rows]]
        if gw is not None:
            d = logp.exp_()
            d[here, labels[rows]] -= 1.0
            g = state["g"].double()
            d *= g[rows][:, None] if case["reduction"] == "none" else g / (count if case["reduction"] == "mean" else 1)
            gh[rows] = d @ w
            gw.addmm_(d.T, h[rows])
    out = losses if case["reduction"] == "none" else losses.sum() / (count if case["reduction"] == "mean" else 1)
    return out if gw is None else [out, gh, gw]


# ---------------------------------------------------------------------------- work
def work(case):
    if case["kind"] in ("score", "loss"):
        n, hidden, vocab = case["tokens"], case["hidden"], case["vocab"]
        valid = n * (1.0 - case["ignored"])
        moved = 2 * hidden * (valid + vocab) + 8 * n + (4 * n if case["reduction"] == "none" else 4)
        if case["kind"] == "score":
            return {"bytes": moved, "flops": 2 * valid * hidden * vocab}
        # two more products; the gradients go out once
        return {"bytes": moved + 2 * hidden * (n + vocab), "flops": 6 * valid * hidden * vocab}
    read = sum(math.prod(s) * _dtype_of(case, i, s).itemsize for i, s in enumerate(_shapes(case)))
    return {"bytes": read * (1 if case["kind"] == "norm" else 2), "flops": 0}
