"""The global norm of all gradients of a model, and clipping.

The reference clips inside its offloaded optimizers only (reference:
src/offload_adam/offload_adam.py:555-561: stack, vector_norm, clamp) and multiplies every
gradient in a pass of its own.  Here any 1300 gradients take one launch for the norm
and one to scale them (``csrc/clip_ops.cu``), and ``Adam`` folds the coefficient into its step.
"""

from __future__ import annotations

import math

import torch

from .. import _ext
from .dispatch import _PLAIN, eager

_NORMS = {2.0: 0, 1.0: 1, math.inf: 2}
_KERNEL_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def check_max_norm(max_norm):
    if isinstance(max_norm, torch.Tensor) or not float(max_norm) >= 0:
        raise ValueError(f"the largest norm must be a number of at least 0, not {max_norm!r}")
    return float(max_norm)


def _gradients(parameters):
    grads = [p.grad for p in parameters if p.grad is not None]
    for g in grads:
        if g.is_sparse or type(g) not in _PLAIN:
            raise TypeError(f"the norm of a sparse or {type(g).__name__} gradient is not supported")
        if not g.is_floating_point():
            raise TypeError(f"the norm of a gradient of {g.dtype} is not supported")
        if g.device != grads[0].device:
            raise ValueError(f"gradients on several devices: {grads[0].device} and {g.device}")
    return grads


def _kernels(grads):
    return grads[0].is_cuda and all(g.dtype in _KERNEL_DTYPES for g in grads) and eager(casts=False)


def _dense(g):
    return torch.ops.aten.is_non_overlapping_and_dense(g)


def _once(grads):
    """Every gradient once, however often it is listed and whatever tensor it is a view by."""
    return list({(g.data_ptr(), g.dtype) + ((g.numel(),) if _dense(g) else (g.shape, g.stride())): g
                 for g in grads if g.numel()}.values())


def _check_sharing(grads):
    """What cannot be scaled in place."""
    end = 0
    for g in sorted(filter(_dense, grads), key=lambda g: g.data_ptr()):
        if g.data_ptr() < end:
            raise ValueError("two gradients share a part of their memory")
        end = g.data_ptr() + g.numel() * g.element_size()
    for g in grads:
        if any(z == 0 and n > 1 for z, n in zip(g.stride(), g.shape)):
            raise ValueError("a gradient whose elements share memory cannot be clipped in place")


def _plain(grads, norm_type, max_norm, scale):
    """``{coefficient, norm}`` in the operations of PyTorch, summed in fp64."""
    grads = _once(grads)
    if scale:
        _check_sharing(grads)
    each = [torch.linalg.vector_norm(g, norm_type, dtype=torch.float64) for g in grads]
    total = torch.linalg.vector_norm(torch.stack(each), norm_type).float() if each else torch.zeros(())
    # a division of two tensors rounds once; a number over a tensor is its reciprocal times the number
    out = torch.stack([(torch.full_like(total, max_norm) / (total + 1e-6)).clamp(max=1.0), total])
    if scale:
        def scaled(g):
            wide = torch.promote_types(g.dtype, torch.float32)
            return g.to(wide) * out[0].to(wide)

        # those with gaps may share memory with others: all of them before anything is written
        gaps = [(g, scaled(g)) for g in grads if not _dense(g)]
        for g in filter(_dense, grads):
            g.copy_(scaled(g))
        for g, x in gaps:
            g.copy_(x)
    return out


def _norm_code(norm_type):
    code = _NORMS.get(float(norm_type))
    if code is None:
        raise ValueError(f"norm_type must be 1, 2 or inf, not {norm_type!r}")
    return code


def _run(parameters, norm_type, max_norm, scale, both=False):
    """The norm, or with ``both`` ``{coefficient, norm}``; None without a gradient."""
    code = _norm_code(norm_type)
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    elif type(parameters) is not list:
        parameters = list(parameters)
    # hundreds of small tensors are bound by what the host does for each of them: the usual case
    # is looked over in C++ (291 tensors: 163 us a call without, 28 with it)
    if parameters and getattr(parameters[0], "is_cuda", False) and eager(casts=False):
        out = _ext.load(required=True).param_grad_norm(parameters, code, max_norm, scale, both)
        if out is not None:
            return out
    grads = _gradients(parameters)
    if not grads:
        return None
    with torch.no_grad():
        if _kernels(grads):
            out = _ext.load(required=True).grad_norm(grads, code, max_norm, scale)
        else:
            out = _plain(grads, float(norm_type), max_norm, scale)
        return out if both else out[1]


def grad_norm(parameters, norm_type=2.0):
    """Norm of all gradients of ``parameters`` (a tensor or an iterable) as if they were one
    vector: an fp32 scalar on their device, without a synchronisation.

    ``norm_type`` is 1, 2 or infinity; the gradients are plain dense tensors on one device.  Parameters
    without a gradient are passed over, a gradient that is listed twice, by whatever view, counts once;
    with no gradient at all the norm is 0.  The sum is kept in fp64 and has the same bits in every run.
    """
    out = _run(parameters, norm_type, 0.0, False)
    return torch.zeros(()) if out is None else out


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False, foreach=None):
    """Scales all gradients of ``parameters`` in place so that their norm (see
    :func:`grad_norm`) is at most ``max_norm``; returns the norm before.

    Called as ``torch.nn.utils.clip_grad_norm_``: every gradient is multiplied by
    ``min(1, max_norm / (norm + 1e-6))``, in fp32, and rounded once; a coefficient of 1 touches
    nothing.  Unlike there, the norm is of order 1, 2 or infinity, all gradients are on one device, tensor
    subclasses (``DTensor``) are refused, a gradient that is listed twice counts and is scaled once, and
    gradients that share a part of their memory are refused unless they have gaps (what those share is scaled
    once).  ``error_if_nonfinite=True`` waits for the norm and raises, with the gradients as they
    were, when it is infinite or NaN.  ``foreach`` is accepted and has no effect.
    """
    max_norm = check_max_norm(max_norm)
    if not error_if_nonfinite:
        out = _run(parameters, norm_type, max_norm, True)
        return torch.zeros(()) if out is None else out
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    out = _run(parameters, norm_type, max_norm, False, True)
    if out is None:
        return torch.zeros(())
    if not math.isfinite(out[1].item()):
        raise RuntimeError(f"the norm of order {norm_type} of the gradients is not finite; they are not clipped")
    grads = _gradients(parameters)
    with torch.no_grad():
        if _kernels(grads):
            _ext.load(required=True).grad_scale(grads, out)
        else:
            _plain(grads, float(norm_type), max_norm, True)
        return out[1]


@torch.no_grad()
def clip_coefficient(parameters, max_norm):
    """``(min(1, max_norm / (norm + 1e-6)), norm)`` of the L2 norm, as device scalars; for a
    step that applies the coefficient itself.  ``(None, None)`` without a gradient."""
    out = _run(parameters, 2.0, float(max_norm), False, True)
    return (None, None) if out is None else (out[:1], out[1])
