"""The row-wise block operators in float64, with the elementwise rounding bounds of a kernel that follows their formulas: test infrastructure.

Every function returns (values, bounds): dicts of float64 tensors.  Bounds follow the kernels' roundings: ``u`` (half a step of the storage
type) for each stored or re-rounded value, ``acc(k)`` for a sum of k products in 32 bits -- at most k + 64 roundings of 2^-24 each, relative
to the sum of the magnitudes -- and 2^-20 for an exponential or erf built from the hardware's (their arguments stay under 2^6)."""
from __future__ import annotations

import math

import torch

F24 = 2.0 ** -24
FUN = 2.0 ** -20


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def acc(k):
    return (k + 64) * F24


def linear_ce(x, w, y, g, ignore_index, reduction, dtype):
    """g: gradient of the loss ([T] with "none", else a number)"""
    u = half_step(dtype)
    x, w = x.double(), w.double()
    keep = y != ignore_index
    x = torch.where(keep[:, None], x, 0.0)
    at = torch.where(keep, y, 0)
    logits = x @ w.t()
    off = acc(x.shape[1]) * (x.abs() @ w.abs().t())                  # a logit's error
    lse = torch.logsumexp(logits, 1)
    rows = torch.where(keep, lse - logits.gather(1, at[:, None])[:, 0], 0.0)
    worst = off.amax(1) if off.numel() else off.new_zeros(x.shape[0])
    brow = torch.where(keep, 2 * worst + FUN + 4 * F24 * (lse.abs() + rows.abs()), 0.0)
    n = int(keep.sum())
    if reduction == "none":
        loss, bloss, scale = rows, brow, g.double()
    else:
        div = n if reduction == "mean" else 1
        loss, bloss = rows.sum() / div if div else rows.new_tensor(math.nan), brow.sum() / max(div, 1) + 4 * F24 * rows.sum().abs() / max(div, 1)
        scale = torch.full_like(rows, float(g) / div if div else 0.0)
    scale = torch.where(keep, scale, 0.0)
    p = torch.exp(logits - lse[:, None])
    hot = torch.zeros_like(p)
    hot.scatter_(1, at[:, None], 1.0)
    dl = (p - hot) * scale[:, None]
    # p is off by a factor of its logit's and lse's error, and the exponential's; then dL is rounded to the storage type
    bdl = scale.abs()[:, None] * p * (off + worst[:, None] + 2 * FUN) * 1.1 + dl.abs() * (u + 4 * F24)
    dx = dl @ w
    dw = dl.t() @ x
    bdx = bdl @ w.abs() * 1.02 + acc(w.shape[0]) * (dl.abs() @ w.abs()) + u * dx.abs() * 1.01
    bdw = bdl.t() @ x.abs() * 1.02 + acc(x.shape[0]) * (dl.abs().t() @ x.abs()) + u * dw.abs() * 1.01
    return dict(loss=loss, dx=dx, dw=dw), dict(loss=bloss, dx=bdx, dw=bdw)


def _act(g, act):
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    cdf = 0.5 * (1 + torch.erf(g / math.sqrt(2)))
    return g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)


def gated_mlp(x, w_in, w_out, dy, act, dtype):
    u = half_step(dtype)
    uh = u * u if dtype == torch.bfloat16 and len(x) <= 32 else u       # h, dg and du of few rows are sums of two roundings
    x, w_in, w_out = x.double(), w_in.double(), w_out.double()
    f = w_out.shape[1]
    gu, bgu = x @ w_in.t(), acc(x.shape[1]) * (x.abs() @ w_in.abs().t())
    g, up, bg, bu = gu[:, :f], gu[:, f:], bgu[:, :f], bgu[:, f:]
    a, da = _act(g, act)
    ba, bda = 1.2 * bg + FUN * (g.abs() + 1) , 1.0 * bg + FUN * (g.abs() + 2)        # |act'| <= 1.13, |act''| <= 0.8
    h = a * up
    bh = (ba * up.abs() + bu * (a.abs() + ba)) + h.abs() * (uh + 4 * F24)
    y = h @ w_out.t()
    vals = dict(y=y)
    b = dict(y=bh @ w_out.abs().t() * 1.02 + acc(f) * (h.abs() @ w_out.abs().t()) + u * y.abs() * 1.01)
    if dy is not None:
        dy = dy.double()
        dh, bdh = dy @ w_out, acc(dy.shape[1]) * (dy.abs() @ w_out.abs())
        dg, du = dh * up * da, dh * a
        bdg = (bdh * up.abs() * da.abs() + dh.abs() * (bu * da.abs() + bda * (up.abs() + bu))) * 1.02 + dg.abs() * (uh + 6 * F24)
        bdu = (bdh * a.abs() + dh.abs() * ba) * 1.02 + du.abs() * (uh + 6 * F24)
        d, bd = torch.cat([dg, du], 1), torch.cat([bdg, bdu], 1)
        vals.update(dx=d @ w_in, dw_in=d.t() @ x, dw_out=dy.t() @ h)
        b.update(dx=bd @ w_in.abs() * 1.02 + acc(2 * f) * (d.abs() @ w_in.abs()), dw_in=bd.t() @ x.abs() * 1.02 + acc(len(x)) * (d.abs().t() @ x.abs()),
                 dw_out=dy.abs().t() @ bh * 1.02 + acc(len(x)) * (dy.abs().t() @ h.abs()))
        for k in ("dx", "dw_in", "dw_out"):
            b[k] = b[k] + u * vals[k].abs() * 1.01
    return vals, b


def _norm(v, bv, kind, eps):
    """normalised rows, their bound, 1 / deviation, its relative bound"""
    c = (v.shape[-1] / 64 + 16) * F24                                 # a row's sum: D / 64 adds in a lane and six over the lanes, with room
    top = v.abs().amax(-1, keepdim=True)
    d, bd = (v - v.mean(-1, keepdim=True), bv + bv.mean(-1, keepdim=True) + 2 * c * top) if kind == "layer" else (v, bv)
    ms = (d * d).mean(-1, keepdim=True)
    r = 1 / torch.sqrt(ms + eps)
    br = (2 * (d.abs() * bd).mean(-1, keepdim=True) + (bd * bd).mean(-1, keepdim=True) + c * ms) / (ms + eps) / 2 * 1.1 + 4 * F24   # relative
    hat = d * r
    return hat, bd * r * (1 + br) + hat.abs() * (br + 2 * F24), r, br


def _norm_bwd(d, bd, hat, bhat, r, br, kind):
    c = (hat.shape[-1] / 64 + 16) * F24
    m1, m2 = d.mean(-1, keepdim=True), (d * hat).mean(-1, keepdim=True)
    b1 = bd.mean(-1, keepdim=True) + c * d.abs().mean(-1, keepdim=True)
    b2 = (bd * hat.abs() + (d.abs() + bd) * bhat).mean(-1, keepdim=True) + c * (d * hat).abs().mean(-1, keepdim=True)
    if kind == "rms":
        m1, b1 = 0 * m1, 0 * b1
    v = r * (d - m1 - hat * m2)
    size = r * (d.abs() + m1.abs() + (hat * m2).abs())
    return v, r * (bd + b1 + hat.abs() * b2 + bhat * (m2.abs() + b2)) * (1 + br) + size * (br + 4 * F24)


def norm_gate(branch, residual, dtype, *, post_weight=None, post_bias=None, gate=None, row_scale=None, residual_scale=1.0, pre_weight=None, pre_bias=None,
              norm="layer", eps=1e-5, d_residual=None, d_normed=None):
    """branch, residual [S, N, D] (S samples)"""
    u = half_step(dtype)
    S, N, D = branch.shape
    dbl = lambda t, d=0.0: torch.full((), d, dtype=torch.float64, device=branch.device) if t is None else t.double()  # noqa: E731
    x = residual.double()
    s = dbl(row_scale, 1.0)
    s = s[:, None, None] if s.dim() else s
    y = torch.where(s == 0, 0.0, branch.double()) if row_scale is not None else branch.double()
    gt = dbl(gate, 1.0)
    gt = gt.reshape(-1, 1, D) if gate is not None and gate.dim() == 2 else gt
    if gate is not None and gate.dim() == 2 and gt.shape[0] != S:
        gt = gt.repeat_interleave(S // gt.shape[0], 0)
    zero = torch.zeros_like(y)
    if post_weight is not None:
        hat1, bh1, r1, br1 = _norm(y, zero, norm, eps)
        post, bpost = hat1 * dbl(post_weight) + dbl(post_bias), None
        bpost = bh1 * dbl(post_weight).abs() + 2 * F24 * ((hat1 * dbl(post_weight)).abs() + post.abs())
    else:
        hat1, post, bpost = y, y, zero
    r = residual_scale * x + s * gt * post
    br = (s * gt).abs() * bpost + 4 * F24 * ((residual_scale * x).abs() + (s * gt * post).abs())
    vals, b = dict(r=r), dict(r=br * 1.02 + u * r.abs() * 1.01)
    if pre_weight is not None:
        hat2, bh2, r2, br2 = _norm(r, br, norm, eps)
        h = hat2 * dbl(pre_weight) + dbl(pre_bias)
        vals["h"] = h
        b["h"] = (bh2 * dbl(pre_weight).abs() + 2 * F24 * ((hat2 * dbl(pre_weight)).abs() + h.abs())) * 1.02 + u * h.abs() * 1.01
    if d_residual is None and d_normed is None:
        return vals, b
    dr = zero if d_residual is None else d_residual.double()
    bdr = 2 * F24 * dr.abs()
    sums = (S * N / 4 + 64) * F24                                     # a weight gradient: at most a quarter of the rows in one lane's fp32 sum
    if d_normed is not None:
        dn = d_normed.double()
        vals.update(pre_weight=(dn * hat2).sum((0, 1)), pre_bias=dn.sum((0, 1)))
        b.update(pre_weight=(dn.abs() * bh2).sum((0, 1)) + sums * (dn * hat2).abs().sum((0, 1)), pre_bias=sums * dn.abs().sum((0, 1)))
        back, bback = _norm_bwd(dn * dbl(pre_weight), F24 * (dn * dbl(pre_weight)).abs(), hat2, bh2, r2, br2, norm)
        dr, bdr = dr + back, bdr + bback + 2 * F24 * (dr.abs() + back.abs())
    vals["residual"], b["residual"] = residual_scale * dr, (abs(residual_scale) * bdr + 2 * F24 * (residual_scale * dr).abs()) * 1.02 + u * (residual_scale * dr).abs() * 1.01
    dp, bdp = dr * s, (bdr + F24 * dr.abs()) * s.abs()
    if gate is not None:
        t, bt = dp * post, bdp * post.abs() + (dp.abs() + bdp) * bpost
        dims = 1 if gate.dim() == 2 else (0, 1)
        vals["gate"], b["gate"] = t.sum(dims), bt.sum(dims) + sums * t.abs().sum(dims)
        if gate.dim() == 2 and gate.shape[0] != S:
            vals["gate"], b["gate"] = (v.reshape(gate.shape[0], -1, D).sum(1) for v in (vals["gate"], b["gate"]))
    dh, bdh = dp * gt, bdp * gt.abs() + F24 * (dp * gt).abs()
    if post_weight is not None:
        vals.update(post_weight=(dh * hat1).sum((0, 1)), post_bias=dh.sum((0, 1)))
        b.update(post_weight=(bdh * hat1.abs() + (dh.abs() + bdh) * bh1).sum((0, 1)) + sums * (dh * hat1).abs().sum((0, 1)), post_bias=bdh.sum((0, 1)) + sums * dh.abs().sum((0, 1)))
        w = dbl(post_weight)
        dh, bdh = _norm_bwd(dh * w, bdh * w.abs() + F24 * (dh * w).abs(), hat1, bh1, r1, br1, norm)
    vals["branch"], b["branch"] = dh, bdh * 1.02 + u * dh.abs() * 1.01
    return vals, b
