"""The block operators and the vocabulary loss without a GPU: their refusals, and the oracle that the GPU tests hold them to against torch."""
import ctypes as C
import math

import pytest
import torch

from oracle import blocks_oracle as O


def lib():
    from fedcola_amd import _lib
    return _lib.lib()


def refused(rc, word):
    assert rc < 0 and word in lib().fc_last_error().decode(), (rc, lib().fc_last_error())


A = C.c_void_p(1 << 20)          # an address that no refused call touches


def test_c_entries_refuse_bad_arguments():
    L = lib()

    def ce(dt=1, x=A, ldx=16, w=A, ldw=16, y=A, T=4, V=10, D=16, red=1, loss=A, saved=A, sb=1 << 20, ws=A, wb=1 << 24):
        return L.fc_linear_ce_fwd(dt, x, ldx, w, ldw, y, T, V, D, -100, red, loss, saved, sb, ws, wb, None)
    for kw, word in ((dict(dt=2), "dt"), (dict(T=-1), "sizes"), (dict(V=0), "sizes"), (dict(D=0), "sizes"), (dict(w=None), "weight"), (dict(ldw=8), "weight"), (dict(ldw=1 << 21), "weight")):
        refused(ce(**kw), word)

    def mlp(dt=1, act=0, x=A, ldx=16, wi=A, ldi=16, wo=A, ldo=32, T=4, D=16, F=32, ws=A):
        return L.fc_gated_mlp_fwd(dt, act, x, ldx, wi, ldi, wo, ldo, T, D, F, A, D, ws, 1 << 24, None)
    for kw, word in ((dict(dt=7), "dt"), (dict(act=2), "activation"), (dict(F=0), "sizes"), (dict(x=None), "null"), (dict(ldx=8), "stride"), (dict(ldo=16), "stride"),
                     (dict(F=1 << 20, D=1 << 12, ldi=1 << 12, ldo=1 << 20, ldx=1 << 12), "reach"), (dict(ws=C.c_void_p(8)), "aligned")):
        refused(mlp(**kw), word)

    def norm(dt=1, kind=0, y=A, ldy=16, x=A, T=8, D=16, wp=None, bp=None, gate=None, gr=0, rs=None, sr=0, eps=1e-5):
        return L.fc_norm_gate_fwd(dt, kind, y, ldy, x, 16, T, D, wp, bp, gate, gr, rs, sr, 1.0, None, None, eps, A, None, None)
    for kw, word in ((dict(dt=3), "dt"), (dict(kind=2), "norm"), (dict(D=8193, ldy=8193), "sizes"), (dict(y=None), "null"), (dict(ldy=8), "apart"), (dict(eps=0.0), "eps"),
                     (dict(gate=A, gr=3), "samples"), (dict(rs=A, sr=5), "samples"), (dict(bp=A), "bias"), (dict(kind=1, wp=A, bp=A), "bias")):
        refused(norm(**kw), word)


def test_sizes_of_workspaces():
    L = lib()
    assert L.fc_linear_ce_saved_bytes(1, 0, 9, 16) > 0 and L.fc_linear_ce_saved_bytes(1, -1, 9, 16) == L.fc_linear_ce_saved_bytes(1, 4, 0, 16) == 0
    # the logits of up to 32 rows are kept, of 128 beside a wide enough weight, and not of more than 128 MB
    assert L.fc_linear_ce_saved_bytes(1, 128, 1000, 2048) > 128 * 4000 + 128 * 4096 > L.fc_linear_ce_saved_bytes(1, 128, 1000, 2047)
    assert L.fc_linear_ce_saved_bytes(1, 32, 1 << 20, 64) > 32 << 22 > L.fc_linear_ce_saved_bytes(1, 33, 1 << 20, 64)
    assert L.fc_linear_ce_saved_bytes(0, 32, (1 << 20) + 1, 64) < 32 << 20
    for backward in (0, 1):
        small, packed = (L.fc_linear_ce_workspace_bytes(1, 100, 1000, 64, p, backward) for p in (0, 1))
        assert 0 < small and packed >= small + 1000 * 64 * 2
        assert L.fc_gated_mlp_workspace_bytes(1, 100, 64, 128, 1, backward) > L.fc_gated_mlp_workspace_bytes(1, 100, 64, 128, 0, backward) > 0
        # fp32: for few rows the weights stay where they are, for many they become planes
        few = [L.fc_gated_mlp_workspace_bytes(0, 512, 64, 128, p, backward) for p in (0, 1)]
        assert few[1] >= few[0] + 2 * 64 * 128 * 6
        assert L.fc_gated_mlp_workspace_bytes(0, 513, 64, 128, 0, backward) == L.fc_gated_mlp_workspace_bytes(0, 513, 64, 128, 1, backward) > few[1]
        # a workspace for packed operands is enough for ones in place
        for T, D, F in ((20, 4096, 64), (512, 2048, 64), (300, 64, 4096)):
            assert L.fc_gated_mlp_workspace_bytes(0, T, D, F, 1, backward) >= L.fc_gated_mlp_workspace_bytes(0, T, D, F, 0, backward)
            assert L.fc_linear_ce_workspace_bytes(0, T, 2 * F, D, 1, backward) >= L.fc_linear_ce_workspace_bytes(0, T, 2 * F, D, 0, backward)
        few = [L.fc_linear_ce_workspace_bytes(0, 512, 1000, 64, p, backward) for p in (0, 1)]
        assert few[1] >= few[0] + 1000 * 64 * 6 - 512


def test_forms_of_the_tested_sizes():
    """the GPU tests' sizes reach the forms that they are there for, whatever becomes of the model of the time"""
    from fedcola_amd import _lib
    from test_gpu_operators import LARGE, WALKS
    L = lib()
    for dt, T, V, D, _, wl, pieces in WALKS:
        packed = dt == "bf16" and wl in ("odd", "holes")
        for backward in (0, 1):
            form = L.fc_linear_ce_form(dt == "bf16", T, V, D, packed, backward)
            assert form & 0xffff == (256 if dt == "bf16" else 128) and form & _lib.FORM_WALK and bool(form & _lib.FORM_PIECES) == bool(pieces and backward)
    for T, D, F, wl, group in LARGE:
        assert L.fc_gated_mlp_form(1, T, D, F, wl in ("odd", "holes"), 0) == 256
        assert L.fc_gated_mlp_form(1, T, D, F, wl in ("odd", "holes"), 1) == 256 | (group and _lib.FORM_GROUP)
    assert L.fc_linear_ce_form(1, 0, 4, 4, 0, 0) == L.fc_gated_mlp_form(1, 4, 4, 0, 0, 0) == 0


def test_kept_logits_are_never_of_the_large_tiles():
    """the large tiles do not write them: wherever the backward reads kept logits, the forward takes another form"""
    import random
    from fedcola_amd import _lib
    L, r, kept = lib(), random.Random(0), 0
    for _ in range(20000):
        c = (r.randint(0, 1), r.randint(1, 130), int(2 ** r.uniform(1, 22)), int(2 ** r.uniform(0, 15)), r.randint(0, 1))
        if L.fc_linear_ce_form(*c, 1) & _lib.FORM_KEPT:
            kept += 1
            assert L.fc_linear_ce_form(*c, 0) & 0xffff < 256, c
    assert kept > 5000


def test_python_refuses_host_tensors_and_bad_choices():
    from fedcola_amd import blocks, criterions
    from fedcola_amd._lib import FedcolaHipError
    x, w, y = torch.zeros(4, 8), torch.zeros(10, 8), torch.zeros(4, dtype=torch.long)
    with pytest.raises(FedcolaHipError):
        criterions.LinearCrossEntropyLoss()(x, w, y)
    with pytest.raises(FedcolaHipError):
        blocks.GatedMlp(8)(x)
    with pytest.raises(FedcolaHipError):
        blocks.NormGateResidual(8)(x, x)
    for bad in (lambda: criterions.LinearCrossEntropyLoss(reduction="max"), lambda: blocks.GatedMlp(8, act="relu"), lambda: blocks.NormGateResidual(8, norm="batch"),
                lambda: blocks.gated_mlp(x, w, w, "tanh"), lambda: blocks.norm_gate_residual(x, x, norm="group")):
        with pytest.raises(ValueError):
            bad()


def test_rows_of_a_tensor():
    from fedcola_amd.operands import as_rows
    base = torch.arange(240.0).view(10, 24)
    for t, copied in ((base, False), (base[:, :7], False), (base.view(2, 5, 24), False), (base[::2, :5], False), (base.t(), True), (base[:1].expand(6, 24), True),
                      (base[:, ::2], True), (base[3:4, :9], False), (torch.zeros(0, 5), False), (torch.zeros(3, 0, 5), False), (base[0], False)):
        v, ld = as_rows(t)
        assert v.dim() == 2 and ld >= v.shape[1] and torch.equal(v.reshape(t.shape), t)
        assert v.shape[0] <= 1 or (v.stride(0) == ld and v.stride(1) == 1)
        if t.numel():
            assert (v.data_ptr() != t.data_ptr()) == copied


def test_sizes_that_32_bits_do_not_hold():
    from fedcola_amd.operands import check_sizes
    check_sizes("op", 1 << 28, 8, 8, 1 << 30, 1 << 30)
    for rows, v, d in (((1 << 28) + 1, 4, 4), ((1 << 32) + 5, 4, 4), (4, (1 << 30) + 1, 4), (4, 4, 9)):
        with pytest.raises(ValueError, match="at most"):
            check_sizes("op", rows, d, 8, v, 1 << 30)


# ---- the oracle itself: its values against torch's functions and autograd in float64
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_oracle_linear_ce(reduction):
    g = torch.Generator().manual_seed(0)
    x, w = torch.randn(9, 6, generator=g).double().requires_grad_(True), torch.randn(11, 6, generator=g).double().requires_grad_(True)
    y = torch.randint(0, 11, (9,), generator=g)
    y[[1, 4]] = -100
    loss = torch.nn.functional.cross_entropy(x @ w.t(), y, reduction=reduction)
    up = torch.randn(9, generator=g) if reduction == "none" else torch.tensor(0.3)
    dx, dw = torch.autograd.grad(loss, (x, w), up.double())
    v, b = O.linear_ce(x.detach(), w.detach(), y, up, -100, reduction, torch.bfloat16)
    for k, t in (("loss", loss), ("dx", dx), ("dw", dw)):
        assert torch.allclose(v[k], t, rtol=1e-6 if k != "loss" else 1e-12, atol=1e-7) and b[k].shape == t.shape and (b[k] >= 0).all()


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_oracle_gated_mlp(act):
    g = torch.Generator().manual_seed(1)
    x, wi, wo, dy = (torch.randn(*s, generator=g).double().requires_grad_(True) for s in ((5, 6), (14, 6), (6, 7), (5, 6)))
    a, u = (x @ wi.t()).chunk(2, -1)
    y = (getattr(torch.nn.functional, act)(a) * u) @ wo.t()
    grads = torch.autograd.grad(y, (x, wi, wo), dy)
    v, b = O.gated_mlp(x.detach(), wi.detach(), wo.detach(), dy.detach(), act, torch.bfloat16)
    for k, t in zip(("y", "dx", "dw_in", "dw_out"), (y, *grads)):
        assert torch.allclose(v[k], t, rtol=1e-10, atol=1e-12) and (b[k] > 0).all()


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("gate", ["all", "sample", "pairs"])
def test_oracle_norm_gate(kind, gate):
    g = torch.Generator().manual_seed(2)
    S, N, D = 4, 3, 6
    b, r, dr, dh = (torch.randn(S, N, D, generator=g).double().requires_grad_(True) for _ in range(4))
    v = {k: torch.randn(D, generator=g).double().requires_grad_(True) for k in ("post_weight", "post_bias", "pre_weight", "pre_bias")}
    if kind == "rms":
        v["post_bias"] = v["pre_bias"] = None
    v["gate"] = torch.randn(*{"all": (D,), "sample": (S, D), "pairs": (2, D)}[gate], generator=g).double().requires_grad_(True)
    s = torch.tensor([1.0, 0.0, 2.0, 0.5]).double()

    def norm(t, w, bias):
        return torch.nn.functional.layer_norm(t, (D,), w, bias, 1e-5) if kind == "layer" else t / (t.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w
    gt = v["gate"] if gate == "all" else v["gate"].repeat_interleave(S // v["gate"].shape[0], 0)[:, None]
    res = 0.7 * r + s[:, None, None] * gt * norm(b, v["post_weight"], v["post_bias"])
    h = norm(res, v["pre_weight"], v["pre_bias"])
    names = [k for k, t in v.items() if t is not None]
    grads = torch.autograd.grad((res, h), (b, r, *(v[k] for k in names)), (dr, dh))
    plain = {k: None if t is None else t.detach() for k, t in v.items()}
    val, bnd = O.norm_gate(b.detach(), r.detach(), torch.bfloat16, **plain, row_scale=s, residual_scale=0.7, norm=kind, d_residual=dr.detach(), d_normed=dh.detach())
    for k, t in zip(("r", "h", "branch", "residual", *names), (res, h, *grads)):
        assert torch.allclose(val[k], t, rtol=1e-9, atol=1e-10) and (bnd[k] >= 0).all(), k


def test_oracle_bounds_are_small_beside_the_values():
    """a bound that lets everything through tests nothing.  bf16: a few stored roundings of 2^-8 against sums over 32 to 64 terms whose magnitudes add
    up to about five times the sum: under 6 %.  fp32: sums of k <= 100 terms at (k + 64) 2^-24 <= 1e-5 each, three in a row, times that five and
    the function's 2^-20: under 1e-3, a quarter of bf16's single rounding, so that a value rounded to bf16 on the way is outside"""
    g = torch.Generator().manual_seed(3)
    x, w, y = torch.randn(64, 32, generator=g), torch.randn(50, 32, generator=g) / 4, torch.randint(0, 50, (64,), generator=g)
    wi, wo, dy = torch.randn(96, 32, generator=g) / math.sqrt(32), torch.randn(32, 48, generator=g) / math.sqrt(48), torch.randn(64, 32, generator=g)
    r3 = x.view(4, 16, 32)
    for dt, most in ((torch.bfloat16, 0.06), (torch.float32, 1e-3)):
        sets = (O.linear_ce(x, w, y, 1.0, -100, "mean", dt), O.gated_mlp(x, wi, wo, dy, "silu", dt),
                O.norm_gate(r3, dy.view(4, 16, 32), dt, post_weight=torch.ones(32), gate=torch.ones(32), pre_weight=torch.ones(32), d_residual=r3, d_normed=dy.view(4, 16, 32)))
        for v, b in sets:
            for k in v:
                assert b[k].norm() <= most * v[k].norm(), (dt, k, float(b[k].norm() / v[k].norm()))
