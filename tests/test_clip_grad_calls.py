"""Calls of the gradient norm and clipping: autocast, gradients that share memory."""

import math

import pytest
import torch

from offload_adam_b200 import Adam, _ext, clip_grad_norm_, grad_norm

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]
BF16, F32 = torch.bfloat16, torch.float32


def _param(g):
    p = torch.nn.Parameter(torch.zeros_like(g, memory_format=torch.contiguous_format))
    p.grad = g
    return p


def _random(*shape, device, dtype=BF16, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(device, dtype)


@gpu
@pytest.mark.parametrize("dtype", [BF16, torch.float16])
def test_kernels_run_under_autocast(dtype):
    """Autocast has no bearing on an operator that casts nothing: the same launches and bits."""
    C = _ext.load(required=True)

    def params():
        return [_param(_random(300, 7, device="cuda")), _param(_random(50, device="cuda", dtype=F32, seed=1))]

    def calls():
        out, launches = [], []
        for f in (grad_norm, lambda p: clip_grad_norm_(p, 0.5), lambda p: clip_grad_norm_(p, 0.5, error_if_nonfinite=True)):
            p = params()
            before = C.launch_count()
            out.append(f(p))
            launches.append(C.launch_count() - before)
            out += [x.grad for x in p]
        p = [torch.nn.Parameter(torch.ones(300, 7, device="cuda", dtype=BF16))]
        p[0].grad = _random(300, 7, device="cuda")
        opt = Adam(p, lr=1e-2, mode="fp32_master", max_grad_norm=0.5)
        before = C.launch_count()
        opt.step()
        launches.append(C.launch_count() - before)
        return out + [opt.grad_norm, p[0].detach()], launches

    want, launches = calls()
    with torch.autocast("cuda", dtype):
        got, under = calls()
    assert under == launches and all(launches)
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and torch.equal(a, b)


def _close(got, want):
    assert abs(got.item() - want) <= 2.0 ** -23 * want


def _check_scaled(tensors, before, coef):
    for t, b in zip(tensors, before):
        # the coefficient takes four roundings to fp32, the product one, the result one to bf16
        assert ((t.double() - coef * b).abs() <= coef * b.abs() * (2.0 ** -8 + 6 * 2.0 ** -24)).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("norm", [2.0, 1.0, math.inf])
def test_one_gradient_by_several_views(device, norm):
    """Counts once and is scaled once, with and without gaps, listed one behind the other or not."""
    base = _random(32, 64, device=device)
    flat = _random(40 * 30, device=device, seed=1)
    other = _param(_random(77, device=device, seed=2))
    views = [base[:, ::2], flat.view(40, 30), base[:, ::2], flat.view(40, 30).T, flat, base[:, ::2]]
    params = [_param(v) for v in views] + [other]
    each = [base[:, ::2], flat, other.grad]
    want = torch.linalg.vector_norm(torch.cat([x.double().reshape(-1) for x in each]), norm).item()
    before, gaps = [x.double() for x in each], base[:, 1::2].clone()
    _close(grad_norm(params, norm), want)
    _close(clip_grad_norm_(params, 0.5 * want, norm), want)
    _check_scaled(each, before, 0.5)
    assert torch.equal(base[:, 1::2], gaps)


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_that_share_a_part(device):
    """A norm reads each of them; scaled in place they are refused, as they stand, unless they have gaps:
    then what they share is scaled once."""
    flat = _random(64, device=device)
    keep = flat.clone()
    for views in ((flat[:40], flat[24:]), (flat[:40], flat[:41]), (flat[:9], flat[:5], flat[:9])):
        params = [_param(v) for v in views]
        once = list({v.numel(): v for v in views}.values()) if len(views) == 3 else views
        want = math.sqrt(sum(v.double().square().sum().item() for v in once))
        _close(grad_norm(params), want)
        for kw in ({}, dict(error_if_nonfinite=True)):
            with pytest.raises(ValueError, match="share a part"):
                clip_grad_norm_(params, 0.1, **kw)
    assert torch.equal(flat, keep)
    base = _random(32, 64, device=device, seed=3)
    before = base.double()
    views = [base[:, :40], base[:, 8:50], base[::2, 5:9], base[:, 50:]]
    want = math.sqrt(sum(v.double().square().sum().item() for v in views))
    _close(clip_grad_norm_([_param(v) for v in views], 0.25 * want), want)
    _check_scaled([base], [before], 0.25)
    rows = _random(63, device=device, seed=4)
    before = rows.double()
    want = rows.double().as_strided((32, 32), (1, 1)).norm().item()
    _close(clip_grad_norm_([_param(rows.as_strided((32, 32), (1, 1)))], 0.5 * want), want)
    _check_scaled([rows], [before], 0.5)
    one = torch.ones(1, device=device, dtype=BF16)
    with pytest.raises(ValueError, match="share memory"):
        clip_grad_norm_([_param(one.expand(40))], 0.1)
    _close(grad_norm([_param(one.expand(40))]), math.sqrt(40))
    assert one == 1
