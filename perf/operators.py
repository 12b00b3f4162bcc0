"""The measured cases of three operators of the client step:

  ce    linear + softmax cross entropy over a vocabulary, the logits never kept (loss; gradients of hidden states and weight)
  ffn   gated feed-forward block  y = (act(x Wg^T) * (x Wu^T)) Wo^T  with its backward pass
  norm  norm of a branch, gate, drop-path multiplier, scaled residual, norm in front of the next branch, with its backward pass

``run`` computes them with elementary torch operations in 32 bits (``own`` false) or through fedcola_amd (``own`` true)."""
import math

import torch

own = False

IGNORE = -100
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp32": 4}


def listed():
    return [
        # scoring one text position: the whole vocabulary matrix is read for one row, latency and bandwidth
        {"name": "ce_one_row", "op": "ce", "dtype": "bf16", "t": 1, "d": 384, "v": 30522, "ignored": 0.0, "train": False, "wide": 0},
        # masked-token training of a batch of 64 captions of 40 tokens: 15 % of the positions count
        {"name": "ce_masked_tokens", "op": "ce", "dtype": "bf16", "t": 2560, "d": 384, "v": 30522, "ignored": 0.85, "train": True, "wide": 0},
        # next-token training of the same batch at the base width: every position counts
        {"name": "ce_every_token", "op": "ce", "dtype": "bf16", "t": 2560, "d": 768, "v": 30522, "ignored": 0.0, "train": True, "wide": 0},
        # the parity mode's storage type, a ragged batch
        {"name": "ce_fp32", "op": "ce", "dtype": "fp32", "t": 601, "d": 384, "v": 30522, "ignored": 0.2, "train": True, "wide": 0},
        # a long packed batch at a large width, an odd vocabulary; the hidden states are a slice of a wider buffer
        {"name": "ce_large", "op": "ce", "dtype": "bf16", "t": 8192, "d": 2048, "v": 128001, "ignored": 0.1, "train": True, "wide": 64},
        # one token through the block
        {"name": "ffn_one_row", "op": "ffn", "dtype": "bf16", "t": 1, "d": 384, "f": 1024, "act": "silu", "train": False, "wide": 0},
        # the image tower's batch: 64 images of 197 tokens
        {"name": "ffn_images", "op": "ffn", "dtype": "bf16", "t": 12608, "d": 384, "f": 1024, "act": "gelu", "train": True, "wide": 0},
        # the parity mode's storage type, odd sizes
        {"name": "ffn_fp32", "op": "ffn", "dtype": "fp32", "t": 1379, "d": 192, "f": 515, "act": "silu", "train": True, "wide": 0},
        # a large block, hidden width no multiple of a tile
        {"name": "ffn_large", "op": "ffn", "dtype": "bf16", "t": 8192, "d": 4096, "f": 11000, "act": "silu", "train": True, "wide": 0},
        # one token between two branches
        {"name": "norm_one_row", "op": "norm", "dtype": "bf16", "b": 1, "n": 1, "d": 384, "kind": "layer", "gate": "sample", "drop": False, "train": False},
        # the image tower's batch with a gate for each image and drop path
        {"name": "norm_images", "op": "norm", "dtype": "bf16", "b": 64, "n": 197, "d": 384, "kind": "layer", "gate": "sample", "drop": True, "train": True},
        # long rows, many of them, one gate for all
        {"name": "norm_large", "op": "norm", "dtype": "bf16", "b": 8, "n": 8192, "d": 4096, "kind": "rms", "gate": "channel", "drop": False, "train": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("ce", "ffn", "norm"))
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    train = rng.random() < 0.7
    if op == "norm":
        d = _log(rng, 8, 8192)
        d = max(8, d // 8 * 8) if rng.random() < 0.7 else d
        b = _log(rng, 1, 64)
        n = _log(rng, 1, max(1, min(8192, (1 << 27) // (d * b))))
        return {"op": op, "dtype": dtype, "b": b, "n": n, "d": d, "kind": rng.choice(("layer", "rms")), "gate": rng.choice(("none", "channel", "sample")),
                "drop": rng.random() < 0.4, "train": train}
    d = _log(rng, 16, 4096)
    d = max(64, d // 64 * 64) if rng.random() < 0.6 else d
    wide = rng.choice((0, 0, 8, 13))
    most = 2e11 if dtype == "fp32" else 2e12
    if op == "ce":
        v = _log(rng, 50, 131072)
        t = _log(rng, 1, max(1, min(16384, int(most / (6 * d * v)))))
        return {"op": op, "dtype": dtype, "t": t, "d": d, "v": v, "ignored": rng.choice((0.0, 0.0, 0.3, 0.85)), "train": train, "wide": wide}
    f = _log(rng, 16, 12288)
    f = max(64, f // 64 * 64) if rng.random() < 0.6 else f
    t = _log(rng, 1, max(1, min(32768, int(most / (18 * d * f)))))
    return {"op": op, "dtype": dtype, "t": t, "d": d, "f": f, "act": rng.choice(("silu", "gelu")), "train": train, "wide": wide}


def _counted(case):
    """rows of a ce case whose target is not IGNORE"""
    return max(1, int(round(case["t"] * (1.0 - case["ignored"]))))


def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "ce":
        t, d, v, n = case["t"], case["d"], case["v"], _counted(case)
        if not case["train"]:
            return {"bytes": e * (n * d + v * d) + 8 * t + 4 * t, "flops": 2 * n * d * v}
        return {"bytes": e * (n * d + v * d) + 8 * t + e * (t * d + v * d), "flops": 6 * n * d * v}
    if case["op"] == "ffn":
        t, d, f = case["t"], case["d"], case["f"]
        if not case["train"]:
            return {"bytes": e * (2 * t * d + 3 * d * f), "flops": 6 * t * d * f}
        return {"bytes": e * (4 * t * d + 6 * d * f), "flops": 18 * t * d * f}
    t, d = case["b"] * case["n"], case["d"]
    return {"bytes": e * t * d * (8 if case["train"] else 4), "flops": t * d * (45 if case["train"] else 18)}


# ------------------------------------------------------------------------------------------------ inputs
def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DT[case["dtype"]]

    def rnd(*shape, scale=1.0, shift=0.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)

    s = {"op": case["op"], "train": case["train"]}
    if case["op"] == "ce":
        t, d, v = case["t"], case["d"], case["v"]
        s["x"] = rnd(t, d + case["wide"])[:, :d]                     # normalised hidden states
        s["w"] = rnd(v, d, scale=2.0 / math.sqrt(d))                 # logits of standard deviation 2
        y = torch.randint(0, v, (t,), generator=g, device="cuda")
        order = torch.randperm(t, generator=g, device="cuda")
        y[order[_counted(case):]] = IGNORE
        s["y"] = y
        s["g"] = torch.ones((), device="cuda")
    elif case["op"] == "ffn":
        t, d, f = case["t"], case["d"], case["f"]
        s["x"] = rnd(t, d + case["wide"])[:, :d]
        s["w_in"] = rnd(2 * f, d, scale=1.0 / math.sqrt(d))
        s["w_out"] = rnd(d, f, scale=1.0 / math.sqrt(f))
        s["act"] = case["act"]
        if case["train"]:
            s["dy"] = rnd(t, d)
    else:
        b, n, d = case["b"], case["n"], case["d"]
        f32 = torch.float32
        s.update(kind=case["kind"], eps=1e-5, alpha=0.9)
        s["branch"] = rnd(b, n, d, scale=0.7, shift=0.1)
        s["res"] = rnd(b, n, d, scale=1.5)
        s["post_w"], s["pre_w"] = rnd(d, scale=0.2, shift=1.0, dtype=f32), rnd(d, scale=0.2, shift=1.0, dtype=f32)
        s["post_b"], s["pre_b"] = (rnd(d, scale=0.1, dtype=f32), rnd(d, scale=0.1, dtype=f32)) if case["kind"] == "layer" else (None, None)
        s["gate"] = {"none": None, "channel": rnd(d, scale=0.3, shift=0.5, dtype=f32), "sample": rnd(b, d, scale=0.3, shift=0.5, dtype=f32)}[case["gate"]]
        s["scale"] = (torch.rand(b, generator=g, device="cuda") < 0.9).float() / 0.9 if case["drop"] else None
        if case["train"]:
            s["d_res"], s["d_normed"] = rnd(b, n, d), rnd(b, n, d)
    return s


def prepare(case, seed):
    return _inputs(case, seed)


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_ce(s):
    x, w, y = s["x"].float(), s["w"].float(), s["y"]
    keep = y != IGNORE
    at = torch.where(keep, y, 0)[:, None]
    logits = x @ w.t()
    top = logits.amax(1, keepdim=True)
    e = torch.exp(logits - top)
    total = e.sum(1, keepdim=True)
    rows = (top + torch.log(total) - logits.gather(1, at))[:, 0]
    rows = torch.where(keep, rows, 0.0)
    if not s["train"]:
        return {"loss": rows}
    count = keep.sum()
    p = e / total
    p.scatter_add_(1, at, torch.full_like(at, -1.0, dtype=torch.float32))
    p = p * (keep.float() * (s["g"] / count))[:, None]
    return {"loss": rows.sum() / count, "dx": (p @ w).to(s["x"].dtype), "dw": (p.t() @ x).to(s["w"].dtype)}


def _act(g, act):
    """activation and its derivative"""
    if act == "silu":
        sg = 1.0 / (1.0 + torch.exp(-g))
        return g * sg, sg * (1.0 + g * (1.0 - sg))
    cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_ffn(s):
    x, w_in, w_out = s["x"].float(), s["w_in"].float(), s["w_out"].float()
    f = w_out.shape[1]
    gu = x @ w_in.t()
    g, u = gu[:, :f], gu[:, f:]
    a, da = _act(g, s["act"])
    h = a * u
    out = {"y": (h @ w_out.t()).to(s["x"].dtype)}
    if s["train"]:
        dy = s["dy"].float()
        dh = dy @ w_out
        dgu = torch.cat([dh * u * da, dh * a], 1)
        out.update(dx=(dgu @ w_in).to(s["x"].dtype), dw_in=(dgu.t() @ x).to(s["w_in"].dtype), dw_out=(dy.t() @ h).to(s["w_out"].dtype))
    return out


def _plain_norm_fwd(v, kind, eps):
    """normalised rows and 1 / (their deviation)"""
    c = v - v.mean(-1, keepdim=True) if kind == "layer" else v
    r = 1.0 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    return c * r, r


def _plain_norm_bwd(d, hat, r, kind):
    back = d - hat * (d * hat).mean(-1, keepdim=True)
    return r * (back - d.mean(-1, keepdim=True) if kind == "layer" else back)


def _plain_norm(s):
    b, n, d = s["res"].shape
    kind, eps, dt = s["kind"], s["eps"], s["res"].dtype
    one = torch.ones((), device="cuda")
    gate = one if s["gate"] is None else s["gate"][:, None, :] if s["gate"].dim() == 2 else s["gate"]
    scale = one if s["scale"] is None else s["scale"][:, None, None]
    hat1, r1 = _plain_norm_fwd(s["branch"].float(), kind, eps)
    post = hat1 * s["post_w"] + (0.0 if s["post_b"] is None else s["post_b"])
    res = s["alpha"] * s["res"].float() + scale * (gate * post)
    hat2, r2 = _plain_norm_fwd(res, kind, eps)
    out = {"res": res.to(dt), "normed": (hat2 * s["pre_w"] + (0.0 if s["pre_b"] is None else s["pre_b"])).to(dt)}
    if not s["train"]:
        return out
    dn = s["d_normed"].float()
    dr = s["d_res"].float() + _plain_norm_bwd(dn * s["pre_w"], hat2, r2, kind)
    dpost = dr * scale
    dhat = dpost * gate
    out.update(d_branch=_plain_norm_bwd(dhat * s["post_w"], hat1, r1, kind).to(dt), d_res=(s["alpha"] * dr).to(dt),
               d_pre_w=(dn * hat2).double().sum((0, 1)).float(), d_post_w=(dhat * hat1).double().sum((0, 1)).float())
    if kind == "layer":
        out.update(d_pre_b=dn.double().sum((0, 1)).float(), d_post_b=dhat.double().sum((0, 1)).float())
    if s["gate"] is not None:
        out["d_gate"] = (dpost * post).double().sum(1 if s["gate"].dim() == 2 else (0, 1)).float()
    return out


# ------------------------------------------------------------------------------------------------ the framework's operators
def _own_ce(s):
    from fedcola_amd.criterions import linear_cross_entropy_backward, linear_cross_entropy_forward
    if not s["train"]:
        return {"loss": linear_cross_entropy_forward(s["x"], s["w"], s["y"], reduction="none")[0]}
    loss, saved = linear_cross_entropy_forward(s["x"], s["w"], s["y"], reduction="mean")
    dx, dw = linear_cross_entropy_backward(s["g"], saved, s["w"])
    return {"loss": loss, "dx": dx, "dw": dw}


def _own_ffn(s):
    from fedcola_amd.blocks import gated_mlp_backward, gated_mlp_forward
    out = {"y": gated_mlp_forward(s["x"], s["w_in"], s["w_out"], act=s["act"])}
    if s["train"]:
        out["dx"], out["dw_in"], out["dw_out"] = gated_mlp_backward(s["dy"], s["x"], s["w_in"], s["w_out"], act=s["act"])
    return out


def _own_norm(s):
    from fedcola_amd.blocks import norm_gate_residual_backward, norm_gate_residual_forward
    how = dict(post_weight=s["post_w"], post_bias=s["post_b"], gate=s["gate"], row_scale=s["scale"], residual_scale=s["alpha"], pre_weight=s["pre_w"],
               pre_bias=s["pre_b"], norm=s["kind"], eps=s["eps"])
    res, normed = norm_gate_residual_forward(s["branch"], s["res"], **how)
    out = {"res": res, "normed": normed}
    if not s["train"]:
        return out
    d = norm_gate_residual_backward(s["d_res"], s["d_normed"], s["branch"], s["res"], **how)
    out.update(d_branch=d["branch"], d_res=d["residual"], d_pre_w=d["pre_weight"], d_post_w=d["post_weight"])
    if s["kind"] == "layer":
        out.update(d_pre_b=d["pre_bias"], d_post_b=d["post_bias"])
    if s["gate"] is not None:
        out["d_gate"] = d["gate"]
    return out


def run(state):
    if own:
        return {"ce": _own_ce, "ffn": _own_ffn, "norm": _own_norm}[state["op"]](state)
    return {"ce": _plain_ce, "ffn": _plain_ffn, "norm": _plain_norm}[state["op"]](state)


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def _wide(s, *names):
    return [None if s[k] is None else s[k].double().requires_grad_(s["train"]) for k in names]


def exact(case, seed):
    """The definitions through torch's own functions in float64; gradients by differentiation."""
    F = torch.nn.functional
    s = _inputs(case, seed)
    train = s["train"]
    if case["op"] == "ce":
        x, w = _wide(s, "x", "w")
        loss = F.cross_entropy(F.linear(x, w), s["y"], ignore_index=IGNORE, reduction="mean" if train else "none")
        if not train:
            return {"loss": loss}
        dx, dw = torch.autograd.grad(loss, (x, w), s["g"].double())
        return {"loss": loss.detach(), "dx": dx, "dw": dw}
    if case["op"] == "ffn":
        x, w_in, w_out = _wide(s, "x", "w_in", "w_out")
        gate, up = F.linear(x, w_in).chunk(2, -1)
        y = F.linear((F.silu(gate) if s["act"] == "silu" else F.gelu(gate)) * up, w_out)
        if not train:
            return {"y": y}
        dx, dw_in, dw_out = torch.autograd.grad(y, (x, w_in, w_out), s["dy"].double())
        return {"y": y.detach(), "dx": dx, "dw_in": dw_in, "dw_out": dw_out}
    d = case["d"]
    branch, res, post_w, post_b, pre_w, pre_b, gate = _wide(s, "branch", "res", "post_w", "post_b", "pre_w", "pre_b", "gate")

    def norm(v, w, b):
        return F.layer_norm(v, (d,), w, b, s["eps"]) if s["kind"] == "layer" else v / (v.square().mean(-1, keepdim=True) + s["eps"]).sqrt() * w

    inner = norm(branch, post_w, post_b)
    if gate is not None:
        inner = inner * (gate.unsqueeze(1) if gate.dim() == 2 else gate)
    if s["scale"] is not None:
        inner = torch.einsum("b,bnd->bnd", s["scale"].double(), inner)
    r = res * s["alpha"] + inner
    h = norm(r, pre_w, pre_b)
    if not train:
        return {"res": r, "normed": h}
    wanted = {"d_branch": branch, "d_res": res, "d_pre_w": pre_w, "d_post_w": post_w, "d_pre_b": pre_b, "d_post_b": post_b, "d_gate": gate}
    wanted = {k: v for k, v in wanted.items() if v is not None}
    grads = torch.autograd.grad((r, h), list(wanted.values()), (s["d_res"].double(), s["d_normed"].double()))
    return {"res": r.detach(), "normed": h.detach(), **dict(zip(wanted, grads))}
