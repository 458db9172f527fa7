"""The global gradient norm and clipping against 64 bits, and ``Adam`` with a bound on the norm."""

import math

import pytest
import torch

from offload_adam_b200 import Adam, _ext, clip_grad_norm_, grad_norm
from offload_adam_b200.adam import STATE_DTYPES

gpu = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _leave_no_cached_blocks():
    """Tests that measure peak memory count whole cached blocks, whoever left them."""
    yield
    if torch.cuda.is_available():
        torch.cuda.empty_cache()


DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]
NORMS = [2.0, 1.0, math.inf]
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF_STEP = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}
# around a vector (8 or 16 values) and a chunk (256 vectors), one value and none
SIZES = [1, 7, 8, 15, 16, 17, 0, 2047, 2048, 2049, 4095, 4096, 4097, 100003]


def _params(sizes, dtypes, device, shift=0, std=1e-2, seed=0):
    gen = torch.Generator().manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        dtype = dtypes[i % len(dtypes)]
        p = torch.nn.Parameter(torch.zeros(n, dtype=dtype, device=device))
        g = torch.randn(n + shift, generator=gen) * std
        p.grad = g.to(dtype).to(device)[shift:]
        out.append(p)
    return out


def _exact_norm(params, norm):
    each = torch.stack([torch.linalg.vector_norm(p.grad.double(), norm) for p in params if p.grad is not None and p.grad.numel()])
    return torch.linalg.vector_norm(each, norm).item()


def _check_clip(params, max_norm, norm, **kw):
    want = _exact_norm(params, norm)
    before = [p.grad.double() for p in params]
    got = clip_grad_norm_(params, max_norm, norm_type=norm, **kw)
    assert got.dtype == F32 and got.shape == ()
    assert abs(got.item() - want) <= 2.0 ** -23 * want  # rounded to fp32 once
    coef = min(1.0, max_norm / (want + 1e-6))
    for p, b in zip(params, before):
        # the coefficient takes four roundings to fp32, the product one, the result one to its type
        tol = b.abs() * coef * (HALF_STEP[p.grad.dtype] + 5 * 2.0 ** -24) + (2.0 ** -25 if p.grad.dtype == F16 else 0)
        assert ((p.grad.double() - b * coef).abs() <= tol * 1.0001).all()
        if coef == 1.0:
            assert torch.equal(p.grad.double(), b)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("norm", NORMS)
@pytest.mark.parametrize("dtypes", [(BF16,), (F16,), (F32,), (BF16, F32, F16)])
@pytest.mark.parametrize("shift", [0, 1, 9])
def test_norm_and_clip(device, norm, dtypes, shift):
    params = _params(SIZES, dtypes, device, shift)
    want = _exact_norm(params, norm)
    assert abs(grad_norm(params, norm).item() - want) <= 2.0 ** -23 * want
    _check_clip(params, 0.3 * want, norm)
    _check_clip(params, 10 * want, norm)


@gpu
@pytest.mark.parametrize("sizes", [[33] * 161, [5] * 160, [17] * 1300, [9] * 1301 + [70000], [1] * 2700, [40_000_003, 5]])
def test_tables_of_every_size(sizes):
    """A launch takes 160 or 1300 tensors; more take several."""
    params = _params(sizes, (BF16, F32), "cuda", shift=3)
    C = _ext.load(required=True)
    n0 = C.launch_count()
    a, b = grad_norm(params), grad_norm(params)
    assert torch.equal(a, b)
    assert C.launch_count() - n0 == 2 * (-(-len(sizes) // 1300) + 1)
    _check_clip(params, 0.5 * _exact_norm(params, 2.0), 2.0)


@gpu
@pytest.mark.parametrize("count", [160, 448, 449, 1300])
def test_tables_that_are_just_full(count):
    params = _params([5, 33, 20000] * (count // 3) + [9] * (count % 3), (BF16, F32, F16), "cuda", shift=1)
    _check_clip(params, 0.5 * _exact_norm(params, 1.0), 1.0)


@gpu
def test_parameters_of_any_container_and_order():
    a = _params(SIZES, (BF16, F32), "cuda")
    none, meta = torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(3, device="meta"))
    want = grad_norm(a)
    for each in (tuple(a), iter(a), [none] + a, [meta] + a + [none], a[::-1], dict(enumerate(a)).values()):
        assert torch.equal(grad_norm(each), want)
    assert torch.equal(grad_norm(a[1]), grad_norm([a[1]]))


@pytest.mark.parametrize("device", DEVICES)
def test_views_of_one_bucket_leave_their_neighbours(device):
    flat = torch.randn(5000, generator=torch.Generator().manual_seed(1)).to(BF16).to(device)
    keep = flat.clone()
    params = []
    for a, b in ((1, 18), (18, 19), (40, 2089), (3001, 4999)):
        p = torch.nn.Parameter(torch.zeros(b - a, dtype=BF16, device=device))
        p.grad = flat[a:b]
        params.append(p)
    _check_clip(params, 1.0, 2.0)
    for a, b in ((0, 1), (19, 40), (2089, 3001), (4999, 5000)):
        assert torch.equal(flat[a:b], keep[a:b])
    assert not torch.equal(flat[1:18], keep[1:18])


@pytest.mark.parametrize("device", DEVICES)
def test_layouts_and_lists(device):
    def param(g):
        p = torch.nn.Parameter(torch.zeros_like(g))
        p.grad = g
        return p

    base = torch.randn(64, 96, generator=torch.Generator().manual_seed(2)).to(BF16).to(device)
    turned, every_second = param(base[:32].T), param(base[32:, ::2])
    gap = base[32:, 1::2].clone()
    none = torch.nn.Parameter(torch.zeros(3, device=device))
    want = _exact_norm([turned, every_second], 2.0)
    listed = [turned, none, every_second, turned, every_second]  # twice: counts once
    before = [turned.grad.double(), every_second.grad.double()]
    got = clip_grad_norm_(iter(listed), 0.5 * want)
    assert abs(got.item() - want) <= 2.0 ** -23 * want
    for p, b in zip((turned, every_second), before):
        assert ((p.grad.double() - 0.5 * b).abs() <= 0.5 * b.abs() * (2.0 ** -8 + 1e-6)).all()
    assert torch.equal(base[32:, 1::2], gap)
    assert torch.equal(grad_norm(turned), grad_norm([turned]))
    assert grad_norm([none]) == 0 and clip_grad_norm_([], 1.0) == 0


@pytest.mark.parametrize("device", DEVICES)
def test_largest_and_smallest_values(device):
    """A square in fp32 would overflow, or vanish."""
    for value in (3e38, 1e-30):
        p = torch.nn.Parameter(torch.zeros(300, dtype=BF16, device=device))
        p.grad = torch.full((300,), value, device=device).to(BF16)
        p.grad[64:] = 0
        want = _exact_norm([p], 2.0)
        got = grad_norm([p]).item()
        assert got == want or abs(got - want) <= 2.0 ** -23 * want or (want > 3.4e38 and got == math.inf)
    p.grad = torch.zeros(300, dtype=BF16, device=device)
    assert grad_norm([p]) == 0
    clip_grad_norm_([p], 1.0)
    assert (p.grad == 0).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("norm", NORMS)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_values_that_are_not_finite(device, norm, bad):
    def make():
        params = _params([5, 3000, 40], (BF16, F32), device)
        params[1].grad[2999] = bad
        return params

    ours, theirs = make(), make()
    got = clip_grad_norm_(ours, 1.0, norm)
    want = torch.nn.utils.clip_grad_norm_(theirs, 1.0, norm, foreach=False)
    assert got.isnan() == want.isnan() and got.isinf() == want.isinf()
    for a, b in zip(ours, theirs):  # NaN everywhere, or 0 beside the NaN of inf * 0
        assert torch.equal(a.grad.isnan(), b.grad.isnan())
    ours = make()
    keep = [p.grad.clone() for p in ours]
    with pytest.raises(RuntimeError, match="not finite"):
        clip_grad_norm_(ours, 1.0, norm, error_if_nonfinite=True)
    for p, k in zip(ours, keep):
        assert torch.equal(p.grad[p.grad.isfinite()], k[k.isfinite()])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("norm", NORMS)
def test_error_if_nonfinite_clips_what_is_finite(device, norm):
    params = _params(SIZES, (BF16, F32), device)
    _check_clip(params, 0.1, norm, error_if_nonfinite=True)


def test_refusals():
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.ones(4)
    for bad in (-1.0, math.nan, torch.ones(())):
        with pytest.raises(ValueError, match="largest norm"):
            clip_grad_norm_([p], bad)
        with pytest.raises(ValueError, match="largest norm"):
            Adam([torch.nn.Parameter(torch.zeros(4, dtype=BF16))], max_grad_norm=bad)
    for bad in (3.0, 0.0, -math.inf):
        with pytest.raises(ValueError, match="norm_type"):
            grad_norm([p], bad)
        with pytest.raises(ValueError, match="norm_type"):
            clip_grad_norm_([], 1.0, bad)
    e = torch.nn.Embedding(4, 2, sparse=True)
    e(torch.tensor([1])).sum().backward()
    with pytest.raises(TypeError, match="sparse"):
        grad_norm(e.parameters())
    assert torch.equal(p.grad, torch.ones(4))


@gpu
def test_refusals_of_the_kernels():
    flat = torch.ones(64, device="cuda", dtype=BF16)
    p, q = torch.nn.Parameter(torch.zeros(40, device="cuda", dtype=BF16)), torch.nn.Parameter(torch.zeros(40, device="cuda", dtype=BF16))
    p.grad, q.grad = flat[:40], flat[24:]
    with pytest.raises(ValueError, match="share a part"):
        clip_grad_norm_([p, q], 1.0)
    q.grad = torch.ones(1, device="cuda", dtype=BF16).expand(40)
    with pytest.raises(ValueError, match="share memory"):
        clip_grad_norm_([q], 1.0)
    assert abs(grad_norm([q]).item() - math.sqrt(40)) <= 2.0 ** -23 * math.sqrt(40)
    cpu = torch.nn.Parameter(torch.zeros(4))
    cpu.grad = torch.ones(4)
    with pytest.raises(ValueError, match="several devices"):
        grad_norm([p, cpu])
    assert (flat == 1).all()


@gpu
def test_another_stream_and_graphs_that_share_nothing():
    a, b = _params(SIZES, (BF16,), "cuda"), _params([3000, 5], (F32,), "cuda", seed=1)
    want = [_exact_norm(a, 2.0), _exact_norm(b, 2.0)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, norms = [], []
    with torch.cuda.stream(side):
        assert abs(grad_norm(a).item() - want[0]) <= 2.0 ** -23 * want[0]
        for params in (a, b):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                norms.append(clip_grad_norm_(params, 0.05))
            graphs.append(g)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for n, w in zip(norms, want):
        assert abs(n.item() - w) <= 2.0 ** -23 * w
    for g, params in zip(graphs, (a, b)):
        g.replay()
        torch.cuda.synchronize()
        assert _exact_norm(params, 2.0) <= 0.05 * (1 + 2.0 ** -8)


def test_a_gradient_changed_in_place_is_noticed():
    x = torch.ones(3, requires_grad=True)
    x.grad = torch.full((3,), 2.0)
    y = torch.ones(3, requires_grad=True) * x.grad
    clip_grad_norm_([x], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


@gpu
def test_a_gradient_changed_by_the_kernel_is_noticed():
    x = torch.ones(3, requires_grad=True, device="cuda")
    x.grad = torch.full((3,), 2.0, device="cuda")
    y = torch.ones(3, requires_grad=True, device="cuda") * x.grad
    clip_grad_norm_([x], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("mode", list(STATE_DTYPES))
@pytest.mark.parametrize("bound", [0.02, 1e6])
def test_adam_with_a_bound_on_the_norm(device, mode, bound):
    """The same bits as gradients scaled in fp32 inside the step of each parameter."""
    from offload_adam_b200.ops.adam_step import STEP_FNS

    sizes = [1, 17, 4096, 5000]

    def make():
        params = _params(sizes, (BF16,), device)
        for i, p in enumerate(params):
            p.data = torch.randn(sizes[i], generator=torch.Generator().manual_seed(i)).to(BF16).to(device)
        return params

    ours, each = make(), make()
    opt = Adam(ours, lr=1e-2, mode=mode, seed=7, max_grad_norm=bound, decoupled_weight_decay=True)
    free = Adam(each, lr=1e-2, mode=mode, seed=7, decoupled_weight_decay=True)
    for it in range(2):
        want = _exact_norm(ours, 2.0)
        opt.step()
        assert abs(opt.grad_norm.item() - want) <= 2.0 ** -23 * want
        norm = grad_norm(each)
        # divided as two tensors: a number over a tensor is its reciprocal, rounded, times the number
        coef = (torch.full_like(norm, bound) / (norm + 1e-6)).clamp(max=1.0).reshape(1)
        for p in each:
            free._init_state_if_empty(p, free.state[p])
            st = free.state[p]
            st["step"] += 1
            seed = {"seed": free._rng.getrandbits(63)} if mode == "stochastic_rounding" else {}
            STEP_FNS[mode](p.data, {**{k: st[k] for k in STATE_DTYPES[mode]}, "grad": p.grad}, 1e-2, 0.01, 0.9, 0.999, 1e-8,
                           st["step"], decoupled_weight_decay=True, clip_coef=coef, **seed)
    for p, q in zip(ours, each):
        assert torch.equal(p, q)
        assert torch.equal(p.grad, q.grad)  # the gradients themselves stay
        for k in STATE_DTYPES[mode]:
            assert torch.equal(opt.state[p][k], free.state[q][k])
