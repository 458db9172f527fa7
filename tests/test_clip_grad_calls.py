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
