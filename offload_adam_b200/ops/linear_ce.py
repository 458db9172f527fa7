"""Softmax cross entropy of ``h @ weight.T`` in pieces of the vocabulary, without the logits.

The reference's trainers use Liger's fused linear cross-entropy for the same purpose
(reference: examples/e2e_train/train.py:76-115).  ``models.llama.chunked_linear_cross_entropy``
cuts the rows instead and holds the bf16 logits of a few thousand of them.  Here nothing of
the logits outlives a tile: forward keeps a copy of the rows that count and 20 bytes for each, backward
forms the gradient of one piece of the vocabulary at a time.  That costs one more product (four where the
other route has three) and saves its memory; rows whose label is ignored cost nothing, and logits are
not rounded to bf16.

Which one: with gradients, ``mean`` and every row counting, 4096 to 65536 rows of 4096 under 128256 words
take 1.3 times as long here (13.0 for 10.0 ms, 228 for 167) and 0.2 to 0.6 times the memory beside
the gradients; 32 rows of 8192 take 1.4 times as long (W is read three times).  With half of the rows
ignored (4096 x 4096 x 151936) it is 8.4 ms for 11.4, and small heads, bound by launches there, take a half to
a fifth here.  Losses of rows, and weights for them, there are only here.
"""

from __future__ import annotations

import torch

from .. import _ext
from .dispatch import _PLAIN, eager

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}
_PIECE = 16384  # words at a time in the operations of PyTorch


class _PlainLinearCE(torch.autograd.Function):
    """The operations of PyTorch, piece by piece: CPU tensors, other dtypes, and whatever else
    the kernels do not take.  fp32 inside, fp64 for fp64."""

    @staticmethod
    def forward(ctx, h, weight, labels, reduction, ignore_index, piece):
        wide = torch.float64 if h.dtype == torch.float64 else torch.float32
        valid = labels != ignore_index
        rows = valid.nonzero(as_tuple=True)[0]
        lab = labels[rows]
        if ((lab < 0) | (lab >= weight.shape[0])).any():
            raise IndexError("linear_cross_entropy: a label is outside the vocabulary")
        x = h[rows].to(wide)
        top = torch.full((len(rows),), -torch.inf, dtype=wide, device=h.device)
        total, picked = torch.zeros_like(top), torch.zeros_like(top)
        for s in range(0, weight.shape[0], piece):
            w = weight[s:s + piece].to(wide)
            z = x @ w.T
            new = torch.maximum(top, z.amax(1))
            shift = torch.where(new == -torch.inf, 0.0, new)
            total = total * (top - shift).exp() + (z - shift[:, None]).exp().sum(1)
            top = new
            here = (lab >= s) & (lab < s + w.shape[0])
            at = (lab - s).clamp(0, w.shape[0] - 1)
            picked = torch.where(here, z.gather(1, at[:, None])[:, 0], picked)
        # two numbers: their sum would lose the logarithm beside large logits
        rest = total.log()
        ctx.save_for_backward(h, weight, labels, top, rest)
        ctx.args = reduction, ignore_index, piece
        losses = torch.zeros(labels.shape, dtype=wide, device=h.device)
        losses[rows] = (top - picked) + rest
        if reduction == "none":
            return losses
        return losses.sum() / (max(1, len(rows)) if reduction == "mean" else 1)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        with torch.autocast(g.device.type, enabled=False):
            return _PlainLinearCE._backward(ctx, g)

    @staticmethod
    def _backward(ctx, g):
        h, weight, labels, top, rest = ctx.saved_tensors
        reduction, ignore_index, piece = ctx.args
        rows = (labels != ignore_index).nonzero(as_tuple=True)[0]
        lab, x = labels[rows], h[rows].to(top.dtype)
        scale = g[rows] if reduction == "none" else g / (max(1, len(rows)) if reduction == "mean" else 1)
        scale = scale.to(top.dtype).expand(len(rows))[:, None]
        gx = torch.zeros_like(x) if ctx.needs_input_grad[0] else None
        gw = torch.empty_like(weight) if ctx.needs_input_grad[1] else None
        for s in range(0, weight.shape[0], piece):
            w = weight[s:s + piece].to(top.dtype)
            d = (x @ w.T - top[:, None] - rest[:, None]).exp()
            here = ((lab >= s) & (lab < s + w.shape[0])).nonzero(as_tuple=True)[0]
            d[here, lab[here] - s] -= 1
            d *= scale
            if gx is not None:
                gx += d @ w
            if gw is not None:
                gw[s:s + piece] = (d.T @ x).to(gw.dtype)
        gh = None
        if gx is not None:
            gh = torch.zeros_like(h)
            gh[rows] = gx.to(h.dtype)
        return gh, gw, None, None, None, None


def linear_cross_entropy(h, weight, labels, reduction="mean", ignore_index=-100, piece=None):
    """Cross entropy of the logits ``h @ weight.T`` against ``labels``.

    Args:
        h: hidden states, ``(..., hidden)``.
        weight: the head, ``(vocab, hidden)``, a dense tensor of the dtype of ``h`` (under autocast
            both are cast to its dtype).
        labels: int64, of the shape of ``h`` without its last dimension.
        reduction: ``"mean"`` over the rows that count (0 when there are none), ``"sum"``, or
            ``"none"``: one loss a row, of the shape of ``labels``, 0 for ignored rows.
        ignore_index: rows with this label take no part: whatever ``h`` holds there, they
            contribute nothing and their gradient is zero.
        piece: words of the vocabulary whose gradient backward holds at a time; rounded up
            to a multiple of 256 where the kernels run, 2^20 at most there.  ``None`` or 0: as many as take
            256 MB.

    The result is fp32 (fp64 for fp64 inputs) and differentiable once with respect to ``h`` and
    ``weight``.  Plain bf16 CUDA tensors whose ``hidden`` is a multiple of 8 (2^18 at most; 2^24 rows,
    2^26 words) run the kernels (``csrc/linear_ce.cu``); everything else runs operations of PyTorch
    piece by piece, and wait for the GPU.  Beside the gradients the kernels take a copy of the rows that
    count, until backward, ``rows * vocab / 16`` bytes in forward, and in backward one piece, a second copy
    of the rows and the fp32 sums of the hidden states' gradient, one for each 65536 words of a piece or
    more where few tiles would leave SMs idle (beyond 65536 rows also of one piece of the head's).

    A label outside the vocabulary is an ``IndexError``.  The kernels see it when they run: the
    loss of that call is NaN, and the next call that looks (its backward, or the next loss)
    raises.  So it is with a kernel that waits two seconds for its own pipeline in vain: the results of
    that call are NaN, and the next one is a ``RuntimeError``.
    """
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {tuple(_REDUCTIONS)}, not {reduction!r}")
    if piece is not None and (not isinstance(piece, int) or isinstance(piece, bool) or piece < 0):
        raise ValueError(f"piece must be None or a whole number of words, not {piece!r}")
    # the usual call is looked over in C++: short ones are bound by the host
    if type(h) in _PLAIN and type(weight) in _PLAIN and type(labels) is torch.Tensor and h.is_cuda and eager():
        out = _ext.load(required=True).linear_ce(h, weight, labels, _REDUCTIONS[reduction], ignore_index, piece or 0,
                                                 False)
        if out is not None:
            return out
    if hasattr(weight, "_payload"):
        raise TypeError("linear_cross_entropy: the head's weight is packed; leave lm_head out of the quantization")
    if weight.dim() != 2 or h.dim() < 1 or h.shape[-1] != weight.shape[1] or weight.numel() == 0:
        raise ValueError(f"linear_cross_entropy: hidden states {tuple(h.shape)} do not fit a head of {tuple(weight.shape)}")
    if labels.shape != h.shape[:-1] or labels.dtype != torch.int64:
        raise ValueError(f"linear_cross_entropy: int64 labels of shape {tuple(h.shape[:-1])} are needed, not "
                         f"{labels.dtype} of {tuple(labels.shape)}")
    if torch.is_autocast_enabled(h.device.type):
        dtype = torch.get_autocast_dtype(h.device.type)
        with torch.autocast(h.device.type, enabled=False):  # nothing inside is to be cast again
            return linear_cross_entropy(h.to(dtype), weight.to(dtype), labels, reduction, ignore_index, piece)
    if not h.is_floating_point() or h.dtype != weight.dtype:
        raise ValueError(f"linear_cross_entropy: hidden states of {h.dtype} and a head of {weight.dtype}")
    if not (h.device == weight.device == labels.device):
        raise ValueError("linear_cross_entropy: hidden states, head and labels must be on one device")
    shape = labels.shape
    if len(shape) != 1:
        h, labels = h.reshape(-1, h.shape[-1]), labels.reshape(-1)
    out = _PlainLinearCE.apply(h, weight, labels, reduction, ignore_index, piece or _PIECE)
    return out.view(shape) if reduction == "none" and len(shape) != 1 else out
