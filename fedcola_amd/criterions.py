"""Criteria of the client step, looked up by name like the reference does in ``torch.nn.__dict__``
(/root/reference/src/criterions/__init__.py:3-8, src/server/fedavgserver.py:76-80, src/client/fedavgclient.py:23).

``ContrastiveLoss`` restates torchmultimodal's ``ContrastiveLossWithTemperature`` (un-vendored third party; single
process: no gather): logit_scale = log(1/0.07) clamped to [0, log 100]; a fresh module is built every step at
fedavgclient.py:95, so the temperature never trains.  Both modules run the fused HIP kernels and support autograd
through a thin Function (the fully fused path is ``fc_client_step``)."""
from __future__ import annotations

import math

import torch
import torch.nn as nn

from . import _lib
from ._lib import check, ptr
from .operands import address, as_rows, check_sizes, in_place, on_device, operand_type


def contrastive_tau() -> float:
    ls = torch.tensor(math.log(1 / 0.07), dtype=torch.float32).clamp(math.log(1.0), math.log(100.0))
    return float(torch.exp(ls))


class _ContrastiveFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a, b, tau):
        a = a.contiguous().float()
        b = b.contiguous().float()
        B, D = a.shape
        L = _lib.lib()
        scratch = torch.empty(int(L.fc_contrastive_scratch_floats(B)), device=a.device)
        lossbuf = torch.zeros(2, device=a.device)
        da, db = torch.empty_like(a), torch.empty_like(b)
        check(L.fc_contrastive_loss_fwd_bwd(ptr(a), ptr(b), B, D, tau, ptr(scratch), scratch.numel(), ptr(lossbuf), ptr(da), ptr(db),
                                            _lib.stream_ptr()))
        ctx.save_for_backward(da, db)
        return lossbuf[1].clone()

    @staticmethod
    def backward(ctx, g):
        da, db = ctx.saved_tensors
        return g * da, g * db, None


class ContrastiveLoss(nn.Module):
    def __init__(self):
        super().__init__()
        self.logit_scale = nn.Parameter(torch.tensor(math.log(1 / 0.07)))

    def forward(self, embeddings_a, embeddings_b):
        self.logit_scale.data.clamp_(math.log(1.0), math.log(100.0))
        return _ContrastiveFn.apply(embeddings_a, embeddings_b, float(torch.exp(self.logit_scale)))


class _CEFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, y):
        logits = logits.contiguous().float()
        B, Cn = logits.shape
        lossbuf = torch.zeros(2, device=logits.device)
        dl = torch.empty_like(logits)
        check(_lib.lib().fc_ce_loss_fwd_bwd(ptr(logits), ptr(y.contiguous().long()), B, Cn, ptr(lossbuf), ptr(dl), _lib.stream_ptr()))
        ctx.save_for_backward(dl)
        return lossbuf[1].clone()

    @staticmethod
    def backward(ctx, g):
        (dl,) = ctx.saved_tensors
        return g * dl, None


class CrossEntropyLoss(nn.Module):
    def forward(self, logits, targets):
        return _CEFn.apply(logits, targets)


# ------------------------------------------------------------------------------------------------ a linear layer's loss over a vocabulary
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def linear_cross_entropy_forward(hidden, weight, targets, ignore_index=-100, reduction="mean"):
    """Cross entropy of the logits ``hidden @ weight.T`` against ``targets`` without keeping the logits: ``(loss, saved)``, ``saved`` for
    ``linear_cross_entropy_backward``.  hidden [..., D] and weight [V, D] in one type, bf16 or fp32; targets int64 of hidden's leading shape.
    loss: fp32, a scalar ("mean" over the targets that are not ignore_index, "sum") or of the targets' shape ("none")."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction {reduction!r}: none, mean or sum")
    code, dev = operand_type("linear_cross_entropy", hidden, weight)
    if weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1] or weight.numel() == 0:
        raise ValueError(f"linear_cross_entropy: hidden {tuple(hidden.shape)} and weight {tuple(weight.shape)} do not match")
    if targets.shape != hidden.shape[:-1] or targets.dtype != torch.int64 or targets.device != dev:
        raise ValueError(f"linear_cross_entropy: targets are int64 of shape {tuple(hidden.shape[:-1])} on {dev}, not {targets.dtype} {tuple(targets.shape)} on {targets.device}")
    check_sizes("linear_cross_entropy", targets.numel(), weight.shape[1], 1 << 20, weight.shape[0], 1 << 30)
    x, ldx = as_rows(hidden)
    w, ldw = as_rows(weight)
    y = targets.contiguous()
    T, (V, D), L, red = x.shape[0], w.shape, _lib.lib(), _REDUCTIONS[reduction]
    loss = torch.empty(targets.shape if red == 0 else (), device=dev)
    with on_device(dev) as stream:
        saved = torch.empty(L.fc_linear_ce_saved_bytes(code, T, V, D), dtype=torch.uint8, device=dev)
        ws = torch.empty(L.fc_linear_ce_workspace_bytes(code, T, V, D, not in_place(w, ldw, T), 0), dtype=torch.uint8, device=dev)
        check(L.fc_linear_ce_fwd(code, x.data_ptr(), ldx, w.data_ptr(), ldw, y.data_ptr(), T, V, D, ignore_index, red, loss.data_ptr(), saved.data_ptr(),
                                 saved.numel(), ws.data_ptr(), ws.numel(), stream))
    return loss, (saved, hidden.shape, red, (V, code))


def linear_cross_entropy_backward(gloss, saved, weight, need_hidden=True, need_weight=True):
    """Gradients ``(dhidden, dweight)`` for the gradient ``gloss`` of the loss (fp32, of its shape); None where not needed.  weight: the forward's."""
    saved, shape, red, (V, saved_code) = saved
    code, dev = operand_type("linear_cross_entropy", weight)
    T, D, L = math.prod(shape[:-1]), shape[-1], _lib.lib()
    if weight.shape != (V, D) or code != saved_code or saved.device != dev:
        raise ValueError(f"linear_cross_entropy: weight {tuple(weight.shape)} of {weight.dtype} on {weight.device} is not of the size, type and device of the forward's")
    w, ldw = as_rows(weight)
    if gloss.shape != (shape[:-1] if red == 0 else ()) or gloss.device != dev:
        raise ValueError(f"linear_cross_entropy: a gradient of shape {tuple(gloss.shape)} on {gloss.device} is not that of the loss")
    g = gloss.float().contiguous()
    dx = torch.empty(shape, dtype=weight.dtype, device=dev) if need_hidden else None
    dw = torch.empty(V, D, dtype=weight.dtype, device=dev) if need_weight else None
    with on_device(dev) as stream:
        ws = torch.empty(L.fc_linear_ce_workspace_bytes(code, T, V, D, not in_place(w, ldw, T), 1), dtype=torch.uint8, device=dev)
        check(L.fc_linear_ce_bwd(code, w.data_ptr(), ldw, T, V, D, red, g.data_ptr(), saved.data_ptr(), saved.numel(), address(dx), D, address(dw), D,
                                 ws.data_ptr(), ws.numel(), stream))
    return dx, dw


class _LinearCEFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, ignore_index, reduction):
        loss, (saved, *how) = linear_cross_entropy_forward(hidden, weight, targets, ignore_index, reduction)
        ctx.save_for_backward(saved, weight)
        ctx.how = how
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        saved, weight = ctx.saved_tensors
        dx, dw = linear_cross_entropy_backward(g, (saved, *ctx.how), weight, ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        return dx, dw, None, None, None


class LinearCrossEntropyLoss(nn.Module):
    """``CrossEntropyLoss`` of a linear layer over a large vocabulary: ``loss(hidden, weight, targets)`` = cross entropy of
    ``hidden @ weight.T``, whose logits [rows, V] are not kept, but for a few rows (``linear_cross_entropy_forward``)."""

    def __init__(self, ignore_index=-100, reduction="mean"):
        super().__init__()
        if reduction not in _REDUCTIONS:
            raise ValueError(f"reduction {reduction!r}: none, mean or sum")
        self.ignore_index, self.reduction = ignore_index, reduction

    def forward(self, hidden, weight, targets):
        return _LinearCEFn.apply(hidden, weight, targets, self.ignore_index, self.reduction)


CRITERIA = {"ContrastiveLoss": ContrastiveLoss, "CrossEntropyLoss": CrossEntropyLoss}
