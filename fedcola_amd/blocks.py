"""Operators of a transformer block beside those of ``ModalityAgnosticTransformer``'s own blocks (LayerNorm, GELU MLP):

* ``gated_mlp``: the gated feed-forward block, y = (act(x Wg^T) * (x Wu^T)) Wo^T,
* ``norm_gate_residual``: what stands between two branches in one pass -- the norm after a branch, its gate and drop-path multiplier, the
  scaled residual, and the norm in front of the next branch.

Each has a forward and a backward function for programs that run their own backward pass, an autograd form and a module.  They run in
libfedcola_hip (``fc_gated_mlp_*``, ``fc_norm_gate_*``) on the current stream of their tensors' device; there is no CPU form."""
from __future__ import annotations

import math

import torch
import torch.nn as nn

from . import _lib
from ._lib import check
from .operands import address, as_rows, check_sizes, in_place, on_device, operand_type

_ACTS = {"silu": 0, "gelu": 1}
_NORMS = {"layer": 0, "rms": 1}


# ------------------------------------------------------------------------------------------------ gated feed-forward
def _mlp_operands(x, w_in, w_out, act):
    if act not in _ACTS:
        raise ValueError(f"gated_mlp: activation {act!r}: silu or gelu")
    code, dev = operand_type("gated_mlp", x, w_in, w_out)
    if w_in.dim() != 2 or w_out.dim() != 2 or x.dim() < 1 or x.shape[-1] != w_in.shape[1] or w_out.shape != (w_in.shape[1], w_in.shape[0] // 2) or \
            w_in.shape[0] % 2 or w_in.numel() == 0:
        raise ValueError(f"gated_mlp: x [..., D], w_in [2F, D], w_out [D, F] are expected, not {tuple(x.shape)}, {tuple(w_in.shape)}, {tuple(w_out.shape)}")
    check_sizes("gated_mlp", x.numel() // x.shape[-1], w_out.shape[0], 1 << 18, w_out.shape[1], 1 << 20)
    return code, dev, as_rows(x), as_rows(w_in), as_rows(w_out)


def _packed(T, F, w_in, w_out, *rows):
    if w_in[0].element_size() == 4:             # x and dy are laid out in planes anyway; the up rows are reached from the gate rows
        return not (in_place(*w_in, T) and in_place(*w_out, T) and (F + 512) * w_in[1] < 1 << 29)
    return not all(in_place(t, ld, T) for t, ld in (w_in, w_out, *rows))


def gated_mlp_forward(x, w_in, w_out, act="silu"):
    """y = (act(x wg^T) * (x wu^T)) w_out^T.  x [..., D]; w_in [2F, D]: wg over wu; w_out [D, F]; one type, bf16 or fp32.  act: "silu", "gelu" (erf).
    bf16: the hidden values are rounded to bf16 once between the products, for up to 32 rows to 16 bits of mantissa.  Up to 2^28 rows, D 2^18, F 2^20,
    and (F + 512) (D + 64) below 2^30."""
    code, dev, (x2, ldx), (wi, ldi), (wo, ldo) = _mlp_operands(x, w_in, w_out, act)
    T, D, F, L = x2.shape[0], wi.shape[1], wo.shape[1], _lib.lib()
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    packed = _packed(T, F, (wi, ldi), (wo, ldo), (x2, ldx))
    with on_device(dev) as stream:
        ws = torch.empty(L.fc_gated_mlp_workspace_bytes(code, T, D, F, packed, 0), dtype=torch.uint8, device=dev)
        check(L.fc_gated_mlp_fwd(code, _ACTS[act], x2.data_ptr(), ldx, wi.data_ptr(), ldi, wo.data_ptr(), ldo, T, D, F, y.data_ptr(), D, ws.data_ptr(),
                                 ws.numel(), stream))
    return y


def gated_mlp_backward(dy, x, w_in, w_out, act="silu", need=(True, True, True)):
    """Gradients ``(dx, dw_in, dw_out)`` for the gradient dy of y (None where not needed), from the inputs alone."""
    code, dev, (x2, ldx), (wi, ldi), (wo, ldo) = _mlp_operands(x, w_in, w_out, act)
    operand_type("gated_mlp", x, dy)
    if dy.shape != x.shape:
        raise ValueError(f"gated_mlp: dy {tuple(dy.shape)} is not of y's shape {tuple(x.shape)}")
    dy2, ldy = as_rows(dy)
    T, D, F, L = x2.shape[0], wi.shape[1], wo.shape[1], _lib.lib()
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need[0] else None
    dwi = torch.empty(2 * F, D, dtype=x.dtype, device=dev) if need[1] else None
    dwo = torch.empty(D, F, dtype=x.dtype, device=dev) if need[2] else None
    packed = _packed(T, F, (wi, ldi), (wo, ldo), (x2, ldx), (dy2, ldy))
    with on_device(dev) as stream:
        ws = torch.empty(L.fc_gated_mlp_workspace_bytes(code, T, D, F, packed, 1), dtype=torch.uint8, device=dev)
        check(L.fc_gated_mlp_bwd(code, _ACTS[act], dy2.data_ptr(), ldy, x2.data_ptr(), ldx, wi.data_ptr(), ldi, wo.data_ptr(), ldo, T, D, F, address(dx), D,
                                 address(dwi), D, address(dwo), F, ws.data_ptr(), ws.numel(), stream))
    return dx, dwi, dwo


class _GatedMlpFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_in, w_out, act):
        ctx.save_for_backward(x, w_in, w_out)
        ctx.act = act
        return gated_mlp_forward(x, w_in, w_out, act)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w_in, w_out = ctx.saved_tensors
        return (*gated_mlp_backward(dy, x, w_in, w_out, ctx.act, ctx.needs_input_grad[:3]), None)


def gated_mlp(x, w_in, w_out, act="silu"):
    """``gated_mlp_forward`` with autograd."""
    return _GatedMlpFn.apply(x, w_in, w_out, act)


class GatedMlp(nn.Module):
    """Gated feed-forward block of width ``dim``, ``hidden`` units (default: 2/3 of the 4 dim of a plain MLP, in whole 64s: the same parameters)."""

    def __init__(self, dim, hidden=None, act="silu", device=None, dtype=None):
        super().__init__()
        hidden = hidden or max(64, round(8 * dim / 3 / 64) * 64)
        if act not in _ACTS:
            raise ValueError(f"gated_mlp: activation {act!r}: silu or gelu")
        self.act = act
        self.w_in = nn.Parameter(torch.empty(2 * hidden, dim, device=device, dtype=dtype))
        self.w_out = nn.Parameter(torch.empty(dim, hidden, device=device, dtype=dtype))
        for w in (self.w_in, self.w_out):
            nn.init.kaiming_uniform_(w, a=math.sqrt(5))       # nn.Linear's

    def forward(self, x):
        return gated_mlp(x, self.w_in, self.w_out, self.act)


# ------------------------------------------------------------------------------------------------ norm, gate, residual, norm
_VECTORS = ("post_weight", "post_bias", "gate", "row_scale", "pre_weight", "pre_bias")


def _norm_operands(branch, residual, norm, eps, vectors):
    """type code, device, T, D, rows of a gate vector, rows of a multiplier, and the vectors, contiguous, in _VECTORS' order"""
    if norm not in _NORMS:
        raise ValueError(f"norm_gate_residual: norm {norm!r}: layer or rms")
    code, dev = operand_type("norm_gate_residual", branch, residual)
    shape = branch.shape
    if shape != residual.shape or not shape or not 1 <= shape[-1] <= 8192:
        raise ValueError(f"norm_gate_residual: branch {tuple(branch.shape)} and residual {tuple(residual.shape)} of one shape [..., D], D <= 8192, are expected")
    if not eps > 0:
        raise ValueError(f"norm_gate_residual: eps {eps}")
    D = shape[-1]
    T = shape[:-1].numel()
    pw, pb, gate, scale, nw, nb = vectors
    gate_rows = scale_rows = 0
    for i, v in enumerate(vectors):
        if v is None:
            continue
        if v.dtype is not torch.float32 or v.device != dev:
            raise ValueError(f"norm_gate_residual: {_VECTORS[i]} is float32 on {dev}, not {v.dtype} on {v.device}")
        s = v.shape
        if i == 3 or (i == 2 and len(s) == 2):       # one for each sample
            if len(s) != (1 if i == 3 else 2) or s[0] < 1 or T % s[0] or (i == 2 and s[1] != D):
                raise ValueError(f"norm_gate_residual: {_VECTORS[i]} {tuple(s)} does not match {T} rows of {D}")
            if i == 3:
                scale_rows = T // s[0]
            else:
                gate_rows = T // s[0]
        elif len(s) != 1 or s[0] != D:
            raise ValueError(f"norm_gate_residual: {_VECTORS[i]} {tuple(s)} does not match {T} rows of {D}")
    if (pb is not None and (pw is None or norm == "rms")) or (nb is not None and (nw is None or norm == "rms")):
        raise ValueError("norm_gate_residual: a bias goes with its weight and norm='layer'")
    return code, dev, T, D, gate_rows, scale_rows, [None if v is None else v.contiguous() for v in vectors]


def norm_gate_residual_forward(branch, residual, *, post_weight=None, post_bias=None, gate=None, row_scale=None, residual_scale=1.0, pre_weight=None,
                               pre_bias=None, norm="layer", eps=1e-5):
    """``r = residual_scale * residual + row_scale * gate * norm(branch)`` and ``h = norm(r)``: (r, h), h None without pre_weight.

    branch, residual [..., D] in one type, bf16 or fp32; the vectors fp32.  post_weight / post_bias [D]: the norm after the branch (None: no
    norm).  gate [D] for all rows or [S, D], one for each of S (fewer than 2^23) samples of equally many consecutive rows.  row_scale [S]: a sample's drop-path
    multiplier; 0 drops the branch, whatever it and its gate hold.  pre_weight / pre_bias [D]: the norm in front of the next branch.  norm: "layer" or
    "rms" (which has no bias)."""
    code, dev, T, D, gate_rows, scale_rows, v = _norm_operands(branch, residual, norm, eps, (post_weight, post_bias, gate, row_scale, pre_weight, pre_bias))
    y, ldy = as_rows(branch)
    x, ldx = as_rows(residual)
    r = torch.empty(residual.shape, dtype=residual.dtype, device=dev)
    h = torch.empty(residual.shape, dtype=residual.dtype, device=dev) if pre_weight is not None else None
    pw, pb, g, s, nw, nb = map(address, v)
    with on_device(dev) as stream:
        check(_lib.lib().fc_norm_gate_fwd(code, _NORMS[norm], y.data_ptr(), ldy, x.data_ptr(), ldx, T, D, pw, pb, g, gate_rows, s, scale_rows, residual_scale,
                                          nw, nb, eps, r.data_ptr(), address(h), stream))
    return r, h


def norm_gate_residual_backward(d_residual, d_normed, branch, residual, *, post_weight=None, post_bias=None, gate=None, row_scale=None, residual_scale=1.0,
                                pre_weight=None, pre_bias=None, norm="layer", eps=1e-5, weight_grads=True):
    """Gradients for those of r (d_residual) and h (d_normed), either None: a dict of ``branch``, ``residual`` and, for each vector that was
    given and with weight_grads, ``post_weight``, ``post_bias``, ``gate``, ``pre_weight``, ``pre_bias`` (fp32)."""
    code, dev, T, D, gate_rows, scale_rows, v = _norm_operands(branch, residual, norm, eps, (post_weight, post_bias, gate, row_scale, pre_weight, pre_bias))
    for t in (d_residual, d_normed):
        if t is not None:
            operand_type("norm_gate_residual", branch, t)
            if t.shape != branch.shape:
                raise ValueError(f"norm_gate_residual: a gradient of shape {tuple(t.shape)} for rows of shape {tuple(branch.shape)}")
    if d_normed is not None and pre_weight is None:
        raise ValueError("norm_gate_residual: d_normed without pre_weight")
    y, ldy = as_rows(branch)
    x, ldx = as_rows(residual)
    dr, lddr = as_rows(d_residual) if d_residual is not None else (None, 0)
    dh, lddh = as_rows(d_normed) if d_normed is not None else (None, 0)
    dy = torch.empty(branch.shape, dtype=branch.dtype, device=dev)
    dx = torch.empty(branch.shape, dtype=branch.dtype, device=dev)
    grads = [torch.empty(t.shape, device=dev) if t is not None and weight_grads and i != 3 else None for i, t in enumerate(v)]
    pw, pb, g, s, nw, _ = map(address, v)
    if not T and grads[2] is not None:
        grads[2].zero_()                                  # no rows: the library does not see how many gates there are
    gpw, gpb, gg, _, gnw, gnb = map(address, grads)
    L, ws, n = _lib.lib(), None, 0
    with on_device(dev) as stream:
        if weight_grads:
            n = L.fc_norm_gate_workspace_bytes(T, D, gate_rows)
            ws = torch.empty(n, dtype=torch.uint8, device=dev)
        check(L.fc_norm_gate_bwd(code, _NORMS[norm], address(dr), lddr, address(dh), lddh, y.data_ptr(), ldy, x.data_ptr(), ldx, T, D, pw, pb, g, gate_rows, s,
                                 scale_rows, residual_scale, nw, eps, dy.data_ptr(), dx.data_ptr(), gpw, gpb, gnw, gnb, gg, address(ws), n, stream))
    out = dict(branch=dy, residual=dx)
    out.update((k, t) for k, t in zip(_VECTORS, grads) if t is not None)
    return out


class _NormGateFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, branch, residual, residual_scale, norm, eps, *vectors):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(branch, residual, *vectors)
        ctx.how = dict(residual_scale=residual_scale, norm=norm, eps=eps)
        return norm_gate_residual_forward(branch, residual, **ctx.how, **dict(zip(_VECTORS, vectors)))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dr, dh):
        branch, residual, *vectors = ctx.saved_tensors
        if dr is None and dh is None:
            return (None,) * (5 + len(_VECTORS))
        d = norm_gate_residual_backward(dr, dh, branch, residual, weight_grads=any(ctx.needs_input_grad[5:]), **ctx.how, **dict(zip(_VECTORS, vectors)))
        return (d["branch"], d["residual"], None, None, None, *(d.get(k) for k in _VECTORS))


def norm_gate_residual(branch, residual, *, post_weight=None, post_bias=None, gate=None, row_scale=None, residual_scale=1.0, pre_weight=None, pre_bias=None,
                       norm="layer", eps=1e-5):
    """``norm_gate_residual_forward`` with autograd (row_scale, drawn by the caller, gets no gradient)."""
    if row_scale is not None and row_scale.requires_grad:
        raise ValueError("norm_gate_residual: row_scale has no gradient")
    return _NormGateFn.apply(branch, residual, residual_scale, norm, eps, post_weight, post_bias, gate, row_scale, pre_weight, pre_bias)


class NormGateResidual(nn.Module):
    """``norm_gate_residual`` with its own weights: the norm after a branch, a gate for each channel (initially ``gate_init``; None: none), the
    residual, and the norm in front of the next branch.  forward(branch, residual, row_scale=None, gate=None): (residual, normed); a ``gate``
    argument ([S, D], of a conditioning network, say) replaces the module's own."""

    def __init__(self, dim, norm="layer", eps=1e-5, gate_init=None, residual_scale=1.0, post=True, pre=True, device=None):
        super().__init__()
        if norm not in _NORMS:
            raise ValueError(f"norm_gate_residual: norm {norm!r}: layer or rms")
        self.norm, self.eps, self.residual_scale = norm, eps, residual_scale

        def vec(on, value):
            return nn.Parameter(torch.full((dim,), float(value), device=device)) if on else None
        self.post_weight, self.post_bias = vec(post, 1), vec(post and norm == "layer", 0)
        self.pre_weight, self.pre_bias = vec(pre, 1), vec(pre and norm == "layer", 0)
        self.gate = vec(gate_init is not None, gate_init or 0)

    def forward(self, branch, residual, row_scale=None, gate=None):
        return norm_gate_residual(branch, residual, post_weight=self.post_weight, post_bias=self.post_bias, gate=self.gate if gate is None else gate,
                                  row_scale=row_scale, residual_scale=self.residual_scale, pre_weight=self.pre_weight, pre_bias=self.pre_bias,
                                  norm=self.norm, eps=self.eps)
