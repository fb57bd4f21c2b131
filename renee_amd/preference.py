"""A preference loss over pairs of labels of a query, for fine-tuning on what was clicked against what was shown beside it.  No
counterpart in the reference, whose only loss is BCE (dl_base.py:576-594).

Pair p of row b says that label chosen[p] is better than rejected[p] for embed[b]:

    margin = embed[b] . (W[chosen] - W[rejected]) - reference
    loss   = sum weight * (-(1 - label_smoothing) log sigmoid(beta margin) - label_smoothing log sigmoid(-beta margin))

the log ratio of a softmax over the labels, whose normaliser cancels, less that of a frozen reference (pair_margins of the embeddings and
labels before the tuning).  Two ways in:

    loss = preference_loss(embed, labels, rowptr, chosen, rejected, reference=ref)   # labels are not trained: an MX4Labels, say
    loss.backward()                                                                  # embed.grad

    layer.fwd_grad(embed, pos_x, pos_y)                                # a training step of the classifier:
    layer.preference_grad(embed, rowptr, chosen, rejected, reference=ref)   # the pairs' gradient is added to its G
    grad_input = layer.backward_pass(embed)                            # dX, dW and the update carry it
"""
from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from ._lib import check, lib
from .mx4 import MX4Labels, TYPES, _On, _rows
from .xfc import XFCLayer, _require


def _list(t: torch.Tensor | None, dtype: torch.dtype, n: int, device: torch.device, what: str) -> torch.Tensor | None:
    if t is None:
        return None
    if not (isinstance(t, torch.Tensor) and t.dim() == 1):
        raise RuntimeError(f"{what} must be a 1-D tensor")
    if t.dtype != dtype:
        raise TypeError(f"{what} must be {dtype}")
    if n >= 0 and t.shape[0] != n:
        raise RuntimeError(f"{what} must have {n} entries")
    if t.device != device:
        t = t.to(device)
    return t if t.is_contiguous() else t.contiguous()


def _labels(labels):
    """(weights or codes, leading dimension, scales, labels, dims) of what pairs can be scored with."""
    if isinstance(labels, XFCLayer):
        return labels.xfc_weight, labels.dims, None, labels.numy, labels.dims
    if isinstance(labels, MX4Labels):
        return labels.codes, 0, labels.scales, labels.numy, labels.dims
    _require(isinstance(labels, torch.Tensor) and labels.dim() == 2, "labels must be an XFCLayer, an MX4Labels or a (labels, dims) tensor")
    _require(labels.dtype == torch.float16, "a label matrix must be float16", TypeError)
    _require(labels.is_cuda, "expected a GPU tensor")
    numy, dims = labels.shape
    _require((labels.stride(1) == 1 or dims <= 1) and labels.stride(0) % 8 == 0 and labels.stride(0) >= dims and labels.data_ptr() % 16 == 0,
             "a label matrix must have rows of whole 16-byte pieces")  # never copied: it may be most of the memory
    return labels, labels.stride(0), None, numy, dims


def preference(embed: torch.Tensor, labels, rowptr: torch.Tensor, chosen: torch.Tensor, rejected: torch.Tensor,
               reference: torch.Tensor | None = None, pair_weight: torch.Tensor | None = None, beta: float = 0.1,
               label_smoothing: float = 0.0, scale: float = 1.0, g: torch.Tensor | None = None, grad_dtype: torch.dtype = torch.float32,
               need_grad: bool = True, need_margin: bool = True):
    """(loss, margin, grad_input) of the pairs, outside autograd: the summed loss (one float32), the pairs' margins (float32) and scale
    times the gradient of `embed`, or None with `g`, a G buffer of a training step to whose entries the pairs' gradient is added
    instead.  need_grad and need_margin leave out what is not wanted.

    rowptr int32[batch + 1], chosen and rejected int32[pairs] (coo_to_csr makes such lists); reference and pair_weight float32[pairs].
    A pair with a label that is none (-1, say) or weight 0 is not there, whatever else it holds."""
    W, ldw, scales, numy, dims = _labels(labels)
    device = W.device
    x = _rows(embed, device, dims, "embed")
    bsz = x.shape[0]
    _require(numy > 0 and dims % 8 == 0 and dims <= 4096, "dims must be a multiple of 8 up to 4096, with one label at least")
    chosen = _list(chosen, torch.int32, -1, device, "chosen")
    P = chosen.numel()
    rejected = _list(rejected, torch.int32, P, device, "rejected")
    rowptr = _list(rowptr, torch.int32, bsz + 1, device, "rowptr")
    reference = _list(reference, torch.float32, P, device, "reference")
    pair_weight = _list(pair_weight, torch.float32, P, device, "pair_weight")
    _require(0.0 <= label_smoothing <= 1.0, "label_smoothing must be in 0..1", ValueError)
    _require(math.isfinite(beta), "beta must be finite", ValueError)
    _require(grad_dtype in TYPES, "grad_dtype must be float16, bfloat16 or float32", TypeError)
    if g is not None:
        _require(g.dtype == torch.float16 and g.dim() == 2 and g.device == device and g.shape[0] == bsz and g.shape[1] >= numy and
                 (g.stride(1) == 1 or g.shape[1] <= 1) and (g.stride(0) >= numy or bsz <= 1), "g must be float16 (batch, numy) on the labels' device")
    loss = torch.empty((), dtype=torch.float32, device=device)
    margin = torch.empty(P, dtype=torch.float32, device=device) if need_margin else None
    grad = torch.empty(bsz, dims, dtype=grad_dtype, device=device) if g is None and need_grad else None
    L = lib()
    need = L.xfc_preference_workspace_bytes(bsz, P, dims)
    ws = torch.empty(need, dtype=torch.uint8, device=device)

    def at(t):
        return None if t is None else t.data_ptr()

    with _On(device) as stream:
        rc = L.xfc_preference(x.data_ptr(), TYPES[x.dtype], x.stride(0) if bsz > 1 else dims, W.data_ptr(), ldw, at(scales), numy, dims,
                              rowptr.data_ptr(), chosen.data_ptr(), rejected.data_ptr(), at(reference), at(pair_weight), bsz, P, beta,
                              label_smoothing, scale, loss.data_ptr(), at(margin), at(grad), TYPES[grad_dtype], dims, at(g),
                              0 if g is None else g.stride(0) if bsz > 1 else max(g.stride(0), numy), ws.data_ptr(), need, stream)
    check(rc, "xfc_preference")
    return loss, margin, grad


def pair_margins(embed: torch.Tensor, labels, rowptr: torch.Tensor, chosen: torch.Tensor, rejected: torch.Tensor) -> torch.Tensor:
    """embed[b] . (W[chosen] - W[rejected]) of every pair: what a frozen model gives as `reference`."""
    return preference(embed, labels, rowptr, chosen, rejected, need_grad=False)[1]


class _Preference(torch.autograd.Function):
    @staticmethod
    def forward(ctx, embed, labels, rowptr, chosen, rejected, reference, pair_weight, beta, label_smoothing, scale):
        loss, _, grad = preference(embed, labels, rowptr, chosen, rejected, reference, pair_weight, beta, label_smoothing, scale,
                                   need_grad=ctx.needs_input_grad[0], need_margin=False)
        ctx.embed_dtype, ctx.embed_device = embed.dtype, embed.device
        ctx.save_for_backward(grad)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        # Kept in fp32 and rounded once, behind the factor: a loss scale is there to keep what a narrower type would lose before it.
        (grad,) = ctx.saved_tensors
        out = torch.mul(grad, grad_out, out=torch.empty_like(grad, dtype=ctx.embed_dtype))
        return out.to(ctx.embed_device), None, None, None, None, None, None, None, None, None


def preference_loss(embed: torch.Tensor, labels, rowptr: torch.Tensor, chosen: torch.Tensor, rejected: torch.Tensor,
                    reference: torch.Tensor | None = None, pair_weight: torch.Tensor | None = None, beta: float = 0.1,
                    label_smoothing: float = 0.0, scale: float = 1.0) -> torch.Tensor:
    """The loss as a differentiable scalar: backward() sends scale times its gradient into embed's graph, kept in float32 and rounded
    to embed's type once, behind the factor that comes down the graph (a gradient scaler's, say).  `labels` (an XFCLayer, an
    MX4Labels or a float16 matrix) are not trained by it, whether or not a matrix requires grad; XFCLayer.preference_grad does that.
    reference and pair_weight are numbers of the pairs: either is refused if it requires grad."""
    if torch.is_grad_enabled():
        for t, what in ((reference, "reference"), (pair_weight, "pair_weight")):
            _require(not (isinstance(t, torch.Tensor) and t.requires_grad), f"{what} gets no gradient: pass {what}.detach()")
    if isinstance(labels, torch.Tensor):
        labels = labels.detach()
    return _Preference.apply(embed, labels, rowptr, chosen, rejected, reference, pair_weight, float(beta), float(label_smoothing),
                             float(scale))
