"""The block operators and the vocabulary loss on the GPU against float64, elementwise within the rounding bounds of oracle/blocks_oracle.py."""
import math

import pytest
import torch

from oracle import blocks_oracle as O

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
TINY = 1e-30
LOWEST = torch.finfo(torch.float32).min


def rnd(gen, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def within(got, want, bound, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got.double() - want).abs()
    bad = ~(off <= bound + TINY)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside; worst {float((off / (bound + TINY)).nan_to_num(1e9).max()):.3g} bounds, off {float(off.nan_to_num(1e9).max()):.3g}"


def layout(t, how):
    """the same values in another memory layout"""
    if how == "wide":                                     # rows of a wider buffer
        b = torch.full((t.shape[0], t.shape[1] + 8), 7.0, dtype=t.dtype, device=t.device)
        b[:, :t.shape[1]] = t
        return b[:, :t.shape[1]]
    if how == "odd":                                      # an odd row stride and an odd first element
        b = torch.full((t.shape[0] * (t.shape[1] + 3) + 1,), 7.0, dtype=t.dtype, device=t.device)
        v = b[1:].view(t.shape[0], t.shape[1] + 3)[:, :t.shape[1]]
        v.copy_(t)
        return v
    if how == "holes":                                    # the same with NaN all around
        b = torch.full((t.shape[0] * (t.shape[1] + 5) + 3,), math.nan, dtype=t.dtype, device=t.device)
        v = b[3:].view(t.shape[0], t.shape[1] + 5)[:, :t.shape[1]]
        v.copy_(t)
        return v
    if how == "turned":
        return t.t().contiguous().t()
    return t


# ------------------------------------------------------------------------------------------------ cross entropy over a vocabulary
def ce_case(T, V, D, dt, ignored, seed):
    g = gen(seed)
    x, w = rnd(g, T, D, dtype=DT[dt]), rnd(g, V, D, scale=2 / math.sqrt(D), dtype=DT[dt])
    y = torch.randint(0, V, (T,), generator=g, device="cuda")
    y[torch.rand(T, generator=g, device="cuda") < ignored] = -100
    return x, w, y


CE = [(1, 2, 1, 0.0, "", ""), (1, 1003, 384, 0.0, "", ""), (7, 50, 16, 0.0, "wide", ""), (33, 257, 64, 0.5, "", "odd"), (64, 1000, 100, 0.0, "odd", ""),
      (65, 513, 7, 0.3, "turned", "turned"), (300, 999, 72, 0.0, "", "wide"), (200, 4100, 136, 0.85, "", ""), (129, 130, 520, 0.0, "", ""), (1030, 6000, 64, 0.2, "", ""),
      (31, 700, 332, 0.0, "", "wide"), (17, 9000, 516, 0.2, "", "odd"), (64, 20, 4, 0.0, "", "turned"), (20, 333, 50, 0.1, "holes", "holes"), (200, 700, 131, 0.1, "", "holes"),
      (513, 300, 33, 0.0, "holes", "holes"), (1, 7, 4000, 0.0, "", ""), (90, 130, 2100, 0.5, "", ""), (300, 45, 1500, 0.9, "odd", "wide"), (40, 1030, 1290, 0.0, "", ""), (100, 9000, 1608, 0.2, "", "")]


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("T,V,D,ignored,xl,wl", CE)
def test_linear_cross_entropy(T, V, D, ignored, xl, wl, dt):
    from fedcola_amd.criterions import linear_cross_entropy_backward, linear_cross_entropy_forward
    x, w, y = ce_case(T, V, D, dt, ignored, T + V + D)
    if ignored == 0.0 and T > 3:
        y[2] = V - 1
        y[3] = 0
    for reduction in ("mean", "sum", "none"):
        g = rnd(gen(5), T) if reduction == "none" else torch.tensor(0.7, device="cuda")
        want, bound = O.linear_ce(x, w, y, g, -100, reduction, DT[dt])
        loss, saved = linear_cross_entropy_forward(layout(x, xl), layout(w, wl), y, reduction=reduction)
        dx, dw = linear_cross_entropy_backward(g, saved, layout(w, wl))
        assert loss.dtype == torch.float32 and dx.dtype == dw.dtype == DT[dt]
        if bool((y != -100).any()) or reduction != "mean":
            within(loss, want["loss"], bound["loss"], f"loss {reduction}")
        within(dx, want["dx"], bound["dx"], f"dx {reduction}")
        within(dw, want["dw"], bound["dw"], f"dw {reduction}")


@pytest.mark.parametrize("dt,T", [("bf16", 131072), ("fp32", 44000)])
def test_linear_cross_entropy_in_pieces(dt, T):
    """so many rows that the backward takes the vocabulary in several pieces (768 and 512 columns), the last one ragged"""
    from fedcola_amd.criterions import linear_cross_entropy_backward, linear_cross_entropy_forward
    x, w, y = ce_case(T, 1700, 24, dt, 0.4, 11)
    g = rnd(gen(6), T)
    want, bound = O.linear_ce(x, w, y, g, -100, "none", DT[dt])
    loss, saved = linear_cross_entropy_forward(x, w, y, reduction="none")
    dx, dw = linear_cross_entropy_backward(g, saved, w)
    within(loss, want["loss"], bound["loss"], "loss")
    within(dx, want["dx"], bound["dx"], "dx")
    within(dw, want["dw"], bound["dw"], "dw")


@pytest.mark.parametrize("layout_", ["", "holes"])
def test_linear_cross_entropy_in_pieces_of_a_weight_in_place(layout_):
    """fp32 rows few enough that the weight stays where it is, and many enough that the vocabulary comes in two pieces (65536 columns); backward twice"""
    from fedcola_amd.criterions import linear_cross_entropy_backward, linear_cross_entropy_forward
    x, w, y = ce_case(512, 70003, 13, "fp32", 0.3, 12)
    y[:2] = torch.tensor([70002, 65536], device="cuda")
    g = torch.tensor(1.3, device="cuda")
    want, bound = O.linear_ce(x, w, y, g, -100, "mean", DT["fp32"])
    loss, saved = linear_cross_entropy_forward(x, layout(w, layout_), y)
    first = linear_cross_entropy_backward(g, saved, layout(w, layout_))
    dx, dw = linear_cross_entropy_backward(g, saved, layout(w, layout_))
    within(loss, want["loss"], bound["loss"], "loss")
    within(dx, want["dx"], bound["dx"], "dx")
    within(dw, want["dw"], bound["dw"], "dw")
    assert torch.equal(dx, first[0]) and torch.equal(dw, first[1])


@pytest.mark.parametrize("T", [1, 32, 33])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_linear_cross_entropy_no_row_counts(dt, T):
    """every row ignored, with logits kept and not: no loss, zero gradients, nothing read of what the rows hold"""
    from fedcola_amd.criterions import linear_cross_entropy_backward, linear_cross_entropy_forward
    x, w, y = ce_case(T, 700, 72, dt, 0.0, 5)
    x.fill_(math.nan)
    y.fill_(-100)
    loss, saved = linear_cross_entropy_forward(x, w, y, reduction="sum")
    dx, dw = linear_cross_entropy_backward(torch.tensor(2.0, device="cuda"), saved, w)
    assert loss.item() == 0 and not dx.any() and not dw.any()


# sizes whose workgroups walk several tiles, the next one's loads under this one's epilogue: two to nine k-steps, ragged last tiles of rows, columns and k,
# rows that do not count (so that some workgroups find no second tile, or none at all), one piece of the vocabulary and two; type, T, V, D, ignored,
# weight's layout, pieces backward
WALKS = [("bf16", 1030, 20011, 128, 0.0, "", 0), ("bf16", 2560, 30522, 136, 0.85, "", 0), ("bf16", 1100, 30522, 520, 0.3, "wide", 0), ("bf16", 700, 30001, 130, 0.1, "odd", 0),
         ("bf16", 4000, 30522, 136, 0.2, "", 1), ("fp32", 600, 30000, 130, 0.0, "", 0), ("fp32", 1100, 30522, 72, 0.3, "", 1), ("fp32", 700, 20011, 200, 0.6, "holes", 0),
         ("fp32", 200, 30000, 130, 0.0, "", 0), ("fp32", 500, 20011, 66, 0.4, "holes", 0), ("fp32", 512, 70003, 130, 0.1, "", 1)]


@pytest.mark.parametrize("dt,T,V,D,ignored,wl,pieces", WALKS)
def test_linear_cross_entropy_workgroups_of_several_tiles(dt, T, V, D, ignored, wl, pieces):
    from fedcola_amd import _lib
    from fedcola_amd.criterions import linear_cross_entropy_backward, linear_cross_entropy_forward
    for backward in (0, 1):
        form = _lib.lib().fc_linear_ce_form(dt == "bf16", T, V, D, dt == "bf16" and wl in ("odd", "holes"), backward)
        assert form & 0xffff == (256 if dt == "bf16" else 128) and form & _lib.FORM_WALK and bool(form & _lib.FORM_PIECES) == bool(pieces and backward)
    x, w, y = ce_case(T, V, D, dt, ignored, T + V + D)
    y[:3] = torch.tensor([V - 1, 0, V - 1 - V % 256], device="cuda")
    g = torch.tensor(1.3, device="cuda")
    want, bound = O.linear_ce(x, w, y, g, -100, "mean", DT[dt])
    loss, saved = linear_cross_entropy_forward(x, layout(w, wl), y)
    dx, dw = linear_cross_entropy_backward(g, saved, layout(w, wl))
    u, n = O.half_step(DT[dt]), int((y != -100).sum())
    for got, k, terms in ((loss, "loss", 1), (dx, "dx", V), (dw, "dw", n)):
        within(got, want[k], bound[k], k)
        # The elementwise bound of a long sum is wide beside its value.  In norm: bf16's two stored roundings of u each; 6 / 32 additions a product, each
        # off by 2^-24 of a running sum of independent terms, whose largest is at most twice the last in the mean square; logit and exponential 2^-18.
        tol = (2 * u if dt == "bf16" else u) + 2 * 6 / 32 * terms * O.F24 + 2.0 ** -18
        assert (got.double() - want[k]).norm() <= tol * want[k].norm(), (k, float((got.double() - want[k]).norm() / want[k].norm()), tol)
    again = linear_cross_entropy_backward(g, saved, layout(w, wl))
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])


@pytest.mark.parametrize("D", [8, 64, 72, 96, 120, 136])
def test_linear_cross_entropy_gathers_a_rows_own_values(D):
    """aligned rows that are no whole 64 values wide, with NaN behind them: of what is gathered for the products, the padding is zeros"""
    from fedcola_amd.criterions import linear_cross_entropy_backward, linear_cross_entropy_forward
    T, V = 70, 130
    x, w, y = ce_case(T, V, D, "bf16", 0.3, D)
    wide = torch.full((T, D + 128), math.nan, dtype=torch.bfloat16, device="cuda")
    wide[:, :D] = x
    loss, saved = linear_cross_entropy_forward(wide[:, :D], w, y, reduction="sum")
    n, ld, t4 = int((y != -100).sum()), (D + 63) // 64 * 64, (T * 4 + 255) // 256 * 256
    at = 256 + 4 * t4                                                   # behind the count and the four tables
    rows = saved[0][at:at + T * ld * 2].view(torch.bfloat16).view(T, ld)[:n]
    assert torch.equal(rows[:, :D], x[y != -100]) and not rows[:, D:].any()
    want, bound = O.linear_ce(x, w, y, torch.tensor(1.0, device="cuda"), -100, "sum", DT["bf16"])
    dx, dw = linear_cross_entropy_backward(torch.tensor(1.0, device="cuda"), saved, w)
    within(loss, want["loss"], bound["loss"], "loss")
    within(dx, want["dx"], bound["dx"], "dx")
    within(dw, want["dw"], bound["dw"], "dw")


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_linear_cross_entropy_masked_rows_hold_anything(dt):
    from fedcola_amd.criterions import linear_cross_entropy_backward, linear_cross_entropy_forward
    x, w, y = ce_case(90, 300, 64, dt, 0.4, 3)
    one = torch.tensor(1.0, device="cuda")
    clean = torch.where((y == -100)[:, None], 0.0, x)
    dirty = x.clone()
    dirty[y == -100] = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(x.dtype).min], device="cuda", dtype=x.dtype).repeat(16)
    got = []
    for v in (clean, dirty):
        loss, saved = linear_cross_entropy_forward(v, w, y)
        got.append((loss, *linear_cross_entropy_backward(one, saved, w)))
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert not got[1][1][y == -100].any()
    # nothing counts: torch's mean, and gradients of zero; no rows at all
    for rows in (90, 0):
        none = torch.full((rows,), -100, device="cuda")
        loss, saved = linear_cross_entropy_forward(dirty[:rows], w, none)
        dx, dw = linear_cross_entropy_backward(one, saved, w)
        assert torch.isnan(loss) and dx.shape == (rows, 64) and not dx.any() and not dw.any()
        loss, saved = linear_cross_entropy_forward(dirty[:rows], w, none, reduction="sum")
        assert float(loss) == 0.0


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_linear_cross_entropy_of_no_rows_each(dt):
    """no rows and a loss for each: an empty loss, an empty gradient of the rows, zeros for the weight"""
    from fedcola_amd.criterions import linear_cross_entropy_backward, linear_cross_entropy_forward
    x, w, y = ce_case(4, 30, 24, dt, 0.0, 0)
    for shape in ((0,), (3, 0)):
        loss, saved = linear_cross_entropy_forward(x.new_empty(*shape, 24), w, y.new_empty(shape), reduction="none")
        assert loss.shape == shape and loss.dtype == torch.float32
        dx, dw = linear_cross_entropy_backward(torch.empty(shape, device="cuda"), saved, w)
        assert dx.shape == (*shape, 24) and dw.shape == w.shape and not dw.any()


def test_linear_cross_entropy_backward_takes_the_forwards_weight():
    """what a forward saved belongs to a weight of its type and size: another one is refused"""
    from fedcola_amd.criterions import linear_cross_entropy_backward, linear_cross_entropy_forward
    g = torch.tensor(1.0, device="cuda")
    for dt, other in (("fp32", torch.bfloat16), ("bf16", torch.float32)):
        x, w, y = ce_case(40, 300, 24, dt, 0.0, 2)
        _, saved = linear_cross_entropy_forward(x, w, y)
        for bad in (w.to(other), w[:299], torch.cat([w, w]), w[:, :16], w[0]):
            with pytest.raises(ValueError):
                linear_cross_entropy_backward(g, saved, bad)
        linear_cross_entropy_backward(g, saved, w.clone())


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("T,V,ignore", [(45, 300, 0), (300, 40, 39), (45, 300, -(1 << 40)), (20, 7, 1 << 33)])
def test_linear_cross_entropy_any_index_may_be_the_ignored_one(T, V, ignore, dt):
    """a class of the vocabulary (a padding token), and numbers that 32 bits do not hold"""
    from fedcola_amd.criterions import linear_cross_entropy_backward, linear_cross_entropy_forward
    x, w, y = ce_case(T, V, 48, dt, 0.0, T + V)
    y[torch.arange(T, device="cuda") % 3 == 1] = ignore
    g = torch.tensor(0.9, device="cuda")
    want, bound = O.linear_ce(x, w, y, g, ignore, "mean", DT[dt])
    loss, saved = linear_cross_entropy_forward(x, w, y, ignore_index=ignore)
    dx, dw = linear_cross_entropy_backward(g, saved, w)
    within(loss, want["loss"], bound["loss"], "loss")
    within(dx, want["dx"], bound["dx"], "dx")
    within(dw, want["dw"], bound["dw"], "dw")


def test_linear_cross_entropy_extreme_values():
    from fedcola_amd.criterions import linear_cross_entropy_backward, linear_cross_entropy_forward
    w = torch.zeros(300, 64, device="cuda")
    w[:, 0] = torch.linspace(-1, 1, 300, device="cuda")
    x = torch.zeros(4, 64, device="cuda")
    x[0, 0], x[1, 0], x[2, 0], x[3, 0] = 1e4, -1e4, 1e-30, 0.0          # logits of +-1e4: one class alone; all alike
    y = torch.tensor([299, 0, 5, 299], device="cuda")
    for dt in (torch.bfloat16, torch.float32):
        loss, saved = linear_cross_entropy_forward(x.to(dt), w.to(dt), y, reduction="none")
        want = torch.nn.functional.cross_entropy(x.to(dt).double() @ w.to(dt).double().t(), y, reduction="none")
        within(loss, want, 1e-5 + 2e-3 * 0 * want, "loss")
    # a target outside of the vocabulary, and a row of NaN: loud, and in their own rows
    for bad in (300, -1):
        y2 = y.clone()
        y2[1] = bad
        loss, saved = linear_cross_entropy_forward(x, w, y2, reduction="none")
        assert torch.isnan(loss).tolist() == [False, True, False, False]
        dx, dw = linear_cross_entropy_backward(torch.ones(4, device="cuda"), saved, w)
        assert torch.isnan(dx[1]).any() and not torch.isnan(dx[[0, 2, 3]]).any() and torch.isnan(dw).any()
    x[2] = math.nan
    loss, _ = linear_cross_entropy_forward(x, w, y, reduction="none")
    assert torch.isnan(loss).tolist() == [False, False, True, False]


def test_linear_cross_entropy_module():
    """autograd, leading dimensions, upstream factor, one gradient alone; against differences of the loss in a direction"""
    from fedcola_amd.criterions import LinearCrossEntropyLoss
    x, w, y = ce_case(6 * 9, 77, 40, "fp32", 0.2, 21)
    x = x.view(6, 9, 40).requires_grad_(True)
    w = w.requires_grad_(True)
    loss = LinearCrossEntropyLoss()(x, w, y.view(6, 9))
    (3 * loss).backward()
    assert x.grad.shape == x.shape
    d = rnd(gen(1), 6, 9, 40)
    e = rnd(gen(2), 77, 40)
    f = lambda t: float(torch.nn.functional.cross_entropy((x.detach().double() + t * d.double()).view(-1, 40) @ (w.detach().double() + t * e.double()).t(), y))  # noqa: E731
    slope = 3 * (f(1e-4) - f(-1e-4)) / 2e-4
    got = float((x.grad.double() * d.double()).sum() + (w.grad.double() * e.double()).sum())
    assert abs(got - slope) <= 1e-5 * max(1.0, abs(slope)), (got, slope)
    (gx,) = torch.autograd.grad(LinearCrossEntropyLoss()(x, w.detach(), y.view(6, 9)), x)
    assert torch.equal(gx * 3, x.grad) or (gx * 3 - x.grad).abs().max() <= 1e-6
    (gw,) = torch.autograd.grad(LinearCrossEntropyLoss(reduction="sum")(x.detach(), w, y.view(6, 9)), w)
    n = int((y != -100).sum())
    assert (gw * 3 / n - w.grad).abs().max() <= 1e-5 * gw.abs().max()


# ------------------------------------------------------------------------------------------------ gated feed-forward
MLP = [(1, 16, 8, "", ""), (1, 384, 1024, "", ""), (5, 7, 3, "", ""), (33, 64, 48, "wide", ""), (64, 1, 5, "", ""), (130, 100, 37, "odd", ""), (257, 192, 515, "", ""),
       (300, 136, 264, "", "turned"), (1000, 64, 24, "turned", "odd"), (700, 320, 640, "", ""), (40, 172, 300, "", "wide"), (64, 1100, 700, "odd", ""), (9, 260, 1028, "", "odd"), (32, 4, 2052, "", "turned"), (20, 37, 70, "holes", "holes"), (130, 101, 35, "", "holes"),
       (512, 130, 67, "", "holes"), (513, 67, 130, "holes", "holes"), (16, 200, 312, "", ""), (17, 200, 312, "", ""),
       (32, 520, 1032, "", ""), (2, 2056, 24, "", ""), (45, 3200, 130, "", ""), (150, 2051, 77, "", "holes"), (600, 1500, 45, "odd", "")]


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("T,D,F,xl,wl", MLP)
def test_gated_mlp(T, D, F, xl, wl, dt):
    from fedcola_amd.blocks import gated_mlp_backward, gated_mlp_forward
    g = gen(T + D + F)
    x, wi, wo, dy = rnd(g, T, D, dtype=DT[dt]), rnd(g, 2 * F, D, scale=1 / math.sqrt(D), dtype=DT[dt]), rnd(g, D, F, scale=1 / math.sqrt(F), dtype=DT[dt]), rnd(g, T, D, dtype=DT[dt])
    for act in ("silu", "gelu"):
        want, bound = O.gated_mlp(x, wi, wo, dy, act, DT[dt])
        a = layout(x, xl), layout(wi, wl), layout(wo, wl)
        got = dict(y=gated_mlp_forward(*a, act=act))
        got["dx"], got["dw_in"], got["dw_out"] = gated_mlp_backward(layout(dy, xl), *a, act=act)
        for k in want:
            assert got[k].dtype == DT[dt]
            within(got[k], want[k], bound[k], f"{act} {k}")


# sizes of the 256 x 256 tile: T, D, F, weights' layout, whether the gradients' products share a launch
LARGE = [(2100, 1032, 4104, "", 1), (4096, 1536, 4096, "", 0), (3001, 1100, 4100, "odd", 1), (4500, 2056, 3001, "holes", 0)]


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("T,D,F,wl,group", LARGE)
def test_gated_mlp_large_tiles(T, D, F, wl, group, act):
    """the large tile, forward and backward, whole and ragged in rows, units and k; the gradients' products in one launch and in three"""
    from fedcola_amd import _lib
    from fedcola_amd.blocks import gated_mlp_backward, gated_mlp_forward
    for backward in (0, 1):
        form = _lib.lib().fc_gated_mlp_form(1, T, D, F, wl in ("odd", "holes"), backward)
        assert form & 0xffff == 256 and not form & _lib.FORM_SLICED and bool(form & _lib.FORM_GROUP) == bool(group and backward)
    g = gen(T + D + F)
    dt = torch.bfloat16
    x, wi, wo, dy = rnd(g, T, D, dtype=dt), rnd(g, 2 * F, D, scale=1 / math.sqrt(D), dtype=dt), rnd(g, D, F, scale=1 / math.sqrt(F), dtype=dt), rnd(g, T, D, dtype=dt)
    want, bound = O.gated_mlp(x, wi, wo, dy, act, dt)
    a = layout(x, wl), layout(wi, wl), layout(wo, wl)
    got = dict(y=gated_mlp_forward(*a, act=act))
    got["dx"], got["dw_in"], got["dw_out"] = gated_mlp_backward(layout(dy, wl), *a, act=act)
    for k in want:
        within(got[k], want[k], bound[k], k)
        # in norm, where the roundings of one result's terms are independent: u for the stored hidden values, u for the result, u for everything in 32 bits
        assert (got[k].double() - want[k]).norm() <= 3 * O.half_step(dt) * want[k].norm(), (k, float((got[k].double() - want[k]).norm() / want[k].norm()))


def test_gated_mlp_extreme_values():
    """gates far out: the activation is 0 or the gate itself, its derivative 0 or 1, nothing overflows; no rows; no gradient wanted"""
    from fedcola_amd.blocks import gated_mlp_backward, gated_mlp_forward
    for dt in DT.values():
        x = torch.zeros(3, 8, device="cuda", dtype=dt)
        x[0, 0], x[1, 0], x[2, 0] = 200.0, -200.0, 0.0
        wi, wo = torch.zeros(8, 8, device="cuda", dtype=dt), torch.zeros(8, 4, device="cuda", dtype=dt)
        wi[:4, 0], wi[4:, 0], wo[0] = 1.0, 0.5, 1.0
        dy = torch.ones(3, 8, device="cuda", dtype=dt)
        for act in ("silu", "gelu"):
            y = gated_mlp_forward(x, wi, wo, act=act)
            assert y[:, 0].tolist() == [float(torch.tensor(4 * 200 * 100.0).to(dt)), 0.0, 0.0] and \
                 not y[:, 1:].any()
            dx, dwi, dwo = gated_mlp_backward(dy, x, wi, wo, act=act)
            assert dx[0, 0] == 4 * (100 + 0.5 * 200) and dx[1, 0] == 0.0 and all(torch.isfinite(t).all() for t in (dx, dwi, dwo))
        empty = gated_mlp_forward(x[:0], wi, wo)
        dx, dwi, dwo = gated_mlp_backward(dy[:0], x[:0], wi, wo)
        assert empty.shape == (0, 8) and dx.shape == (0, 8) and not dwi.any() and not dwo.any()
        assert gated_mlp_backward(dy, x, wi, wo, need=(False, False, True))[:2] == (None, None)


def test_gated_mlp_module():
    from fedcola_amd.blocks import GatedMlp
    m = GatedMlp(96, act="gelu", device="cuda")
    assert m.w_in.shape == (512, 96) and m.w_out.shape == (96, 256)
    x = rnd(gen(0), 4, 11, 96).requires_grad_(True)
    y = m(x)
    dy = rnd(gen(1), 4, 11, 96)
    y.backward(dy)
    xr, wi, wo = x.detach().double().requires_grad_(True), m.w_in.detach().double().requires_grad_(True), m.w_out.detach().double().requires_grad_(True)
    g, u = (xr @ wi.t()).chunk(2, -1)
    ref = (torch.nn.functional.gelu(g) * u) @ wo.t()
    ref.backward(dy.double())
    for a, b in ((y, ref), (x.grad, xr.grad), (m.w_in.grad, wi.grad), (m.w_out.grad, wo.grad)):
        assert (a.double() - b).norm() <= 2e-6 * b.norm()


# ------------------------------------------------------------------------------------------------ norm, gate, residual, norm
def norm_case(S, N, D, dt, kind, post, pre, gate, scale, seed):
    g = gen(seed)
    v = dict(post_weight=1 + 0.2 * rnd(g, D) if post else None, post_bias=0.1 * rnd(g, D) if post and kind == "layer" else None,
             pre_weight=1 + 0.2 * rnd(g, D) if pre else None, pre_bias=0.1 * rnd(g, D) if pre and kind == "layer" else None,
             gate={"": None, "all": rnd(g, D), "sample": rnd(g, S, D)}[gate], residual_scale=0.9, norm=kind, eps=1e-5,
             row_scale=((torch.rand(S, generator=g, device="cuda") < 0.6).float() / 0.6) if scale else None)
    b, r = rnd(g, S, N, D, scale=0.7, dtype=DT[dt]), rnd(g, S, N, D, scale=1.5, dtype=DT[dt])
    return b, r, rnd(g, S, N, D, dtype=DT[dt]), rnd(g, S, N, D, dtype=DT[dt]), v


NORM = [(1, 1, 384, "layer", 1, 1, "sample", 0), (3, 5, 1, "layer", 1, 1, "all", 1), (3, 5, 1, "rms", 1, 1, "sample", 0), (2, 7, 3, "rms", 1, 1, "", 1),
        (4, 197, 384, "layer", 1, 1, "sample", 1), (5, 40, 511, "layer", 1, 1, "all", 0), (2, 33, 512, "rms", 0, 1, "sample", 1), (3, 9, 513, "layer", 1, 0, "sample", 1),
        (2, 50, 1000, "layer", 0, 1, "", 0), (7, 3, 2048, "rms", 1, 1, "all", 1), (2, 6, 2051, "layer", 1, 1, "sample", 0), (1, 300, 4096, "rms", 1, 1, "all", 0),
        (2, 5, 4100, "layer", 1, 1, "all", 1), (3, 4, 5001, "rms", 1, 1, "sample", 0), (2, 3, 8192, "layer", 1, 1, "sample", 1), (2, 3, 64, "layer", 0, 0, "sample", 1),
        (1500, 2, 64, "layer", 1, 1, "sample", 1), (3, 70, 8, "layer", 1, 1, "sample", 1), (2, 333, 61, "layer", 1, 1, "sample", 1), (5, 33, 65, "rms", 1, 1, "all", 1),
        (2, 130, 128, "layer", 1, 1, "", 1), (37, 3, 129, "layer", 1, 1, "sample", 1), (3, 100, 256, "layer", 0, 1, "sample", 0), (2, 41, 257, "rms", 1, 1, "sample", 1),
        (1, 5000, 24, "layer", 1, 0, "all", 0)]


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("S,N,D,kind,post,pre,gate,scale", NORM)
def test_norm_gate_residual(S, N, D, kind, post, pre, gate, scale, dt):
    from fedcola_amd.blocks import norm_gate_residual_backward, norm_gate_residual_forward
    b, r, dr, dh, v = norm_case(S, N, D, dt, kind, post, pre, gate, scale, S + N + D)
    for mode in ("both", "r", "h"):
        a = dict(d_residual=dr if mode != "h" else None, d_normed=dh if mode != "r" and pre else None)
        if a["d_residual"] is None and a["d_normed"] is None:
            continue
        want, bound = O.norm_gate(b, r, DT[dt], **v, **a)
        gr, gh = norm_gate_residual_forward(b, r, **v)
        got = norm_gate_residual_backward(a["d_residual"], a["d_normed"], b, r, **v)
        within(gr, want["r"], bound["r"], "r")
        if pre:
            within(gh, want["h"], bound["h"], "h")
        else:
            assert gh is None
        for k, t in got.items():
            if k.startswith("pre") and a["d_normed"] is None:
                assert not t.any()
                continue
            within(t, want[k], bound[k], f"{mode} {k}")


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("T,D", [(64_999, 8), (65_001, 8), (140_003, 3)])
def test_norm_gate_residual_a_gate_for_each_row(T, D, dt):
    """as many gate vectors as rows, more of them than a launch has workgroups in its second dimension"""
    from fedcola_amd.blocks import norm_gate_residual_backward, norm_gate_residual_forward
    b, r, dr, dh, v = norm_case(T, 1, D, dt, "layer", 1, 1, "sample", 1, 3)
    want, bound = O.norm_gate(b, r, DT[dt], **v, d_residual=dr, d_normed=dh)
    gr, gh = norm_gate_residual_forward(b, r, **v)
    within(gr, want["r"], bound["r"], "r")
    within(gh, want["h"], bound["h"], "h")
    got = norm_gate_residual_backward(dr, dh, b, r, **v)
    for k, t in got.items():
        within(t, want[k], bound[k], k)
    some = norm_gate_residual_backward(dr, dh, b, r, weight_grads=False, **v)
    assert set(some) == {"branch", "residual"} and all(torch.equal(t, got[k]) for k, t in some.items())


def test_norm_gate_residual_layouts():
    """rows of wider buffers, odd strides, unaligned vectors: the same bits as contiguous operands where the values a lane holds are the same"""
    from fedcola_amd.blocks import norm_gate_residual_backward, norm_gate_residual_forward
    for dt in DT.values():
        b, r, dr, dh, v = norm_case(2, 30, 96, "bf16" if dt == torch.bfloat16 else "fp32", "layer", 1, 1, "sample", 1, 4)
        two = lambda t, how: layout(t.reshape(60, 96), how)  # noqa: E731
        ref = norm_gate_residual_forward(b.view(60, 96), r.view(60, 96), **v), norm_gate_residual_backward(dr.view(60, 96), dh.view(60, 96), b.view(60, 96), r.view(60, 96), **v)
        for how in ("wide", "odd", "turned"):
            a = two(b, how), two(r, how)
            o = norm_gate_residual_forward(*a, **v)
            g = norm_gate_residual_backward(two(dr, how), two(dh, how), *a, **v)
            tol = 2 * O.half_step(dt) + 64 * O.F24
            for x, y in [*zip(o, ref[0]), *((g[k], ref[1][k]) for k in g)]:
                assert (x.double() - y.double()).abs().max() <= tol * 4 * y.double().abs().max()


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_norm_gate_residual_dropped_branch_holds_anything(dt):
    from fedcola_amd.blocks import norm_gate_residual_backward, norm_gate_residual_forward
    b, r, dr, dh, v = norm_case(4, 6, 200, dt, "layer", 1, 1, "sample", 1, 8)
    v["row_scale"] = torch.tensor([1.5, 0.0, 0.0, 1.0], device="cuda")
    dirty = b.clone()
    dirty[1], dirty[2] = math.nan, math.inf
    out = [(*norm_gate_residual_forward(t, r, **v), *norm_gate_residual_backward(dr, dh, t, r, **v).values()) for t in (b, dirty)]
    for x, y in zip(*out):
        assert torch.isfinite(y).all() and torch.equal(x, y)
    g = norm_gate_residual_backward(dr, dh, dirty, r, **v)
    assert not g["branch"][1:3].any() and g["branch"][0].any() and not g["gate"][1:3].any()


@pytest.mark.parametrize("post", [0, 1])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("D", [40, 200, 1001, 3000])
def test_norm_gate_residual_dropped_samples_gate_holds_anything(D, dt, kind, post):
    """a row_scale of 0 drops the branch and its gate with it: no infinity or NaN of either reaches a result"""
    from fedcola_amd.blocks import norm_gate_residual_backward, norm_gate_residual_forward
    b, r, dr, dh, v = norm_case(4, 6, D, dt, kind, post, 1, "sample", 1, 8)
    v["row_scale"] = torch.tensor([1.5, 0.0, 0.0, 1.0], device="cuda")
    dirty, gate = b.clone(), v["gate"].clone()
    dirty[1], gate[1], gate[2] = math.nan, math.inf, math.nan
    out = []
    for t, g in ((b, v["gate"]), (dirty, gate)):
        d = norm_gate_residual_backward(dr, dh, t, r, **{**v, "gate": g})
        out.append((*norm_gate_residual_forward(t, r, **{**v, "gate": g}), *d.values()))
    for x, y in zip(*out):
        assert torch.isfinite(y).all() and torch.equal(x, y)
    assert not d["branch"][1:3].any() and not d["gate"][1:3].any()


@pytest.mark.parametrize("gate", ["all", "sample"])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_norm_gate_residual_of_no_rows(dt, gate):
    """no rows: empty results, and zeros for every gradient of a vector, the gate's among them"""
    from fedcola_amd.blocks import norm_gate_residual_backward, norm_gate_residual_forward
    S, D = 3, 200
    _, _, _, _, v = norm_case(S, 1, D, dt, "layer", 1, 1, gate, 1, 4)
    empty = torch.empty(S, 0, D, dtype=DT[dt], device="cuda")
    r, h = norm_gate_residual_forward(empty, empty, **v)
    assert r.shape == h.shape == empty.shape
    used = [torch.full(s, math.nan, device="cuda") for s in ((S, D), (D,)) for _ in range(32)]      # what new buffers are likely to hold
    del used
    got = norm_gate_residual_backward(empty, empty, empty, empty, **v)
    assert got["branch"].shape == got["residual"].shape == empty.shape
    for k in ("post_weight", "post_bias", "gate", "pre_weight", "pre_bias"):
        assert got[k].shape == v[k].shape and not got[k].any(), k


def test_norm_gate_residual_the_most_gates():
    """one gate fewer than the limit, a row each: the first, the last and some in between, and the weights' gradients in norm"""
    from fedcola_amd.blocks import norm_gate_residual_backward, norm_gate_residual_forward
    T, D = (1 << 23) - 1, 8
    b, r, dr, dh, v = norm_case(T, 1, D, "bf16", "rms", 1, 1, "sample", 0, 1)
    gr, gh = norm_gate_residual_forward(b, r, **v)
    got = norm_gate_residual_backward(dr, dh, b, r, **v)
    some = torch.tensor([0, 1, 59_999, 60_000, 65_535, 65_536, 4_194_304, T - 2, T - 1], device="cuda")
    want, bound = O.norm_gate(b[some], r[some], DT["bf16"], **{**v, "gate": v["gate"][some]}, d_residual=dr[some], d_normed=dh[some])
    for k, t in (("r", gr), ("h", gh), ("branch", got["branch"]), ("residual", got["residual"]), ("gate", got["gate"])):
        within(t[some], want[k], bound[k], k)
    hat = lambda t: t / (t.square().mean(-1, keepdim=True) + 1e-5).sqrt()  # noqa: E731
    dn = dh.double()[:, 0]
    res = 0.9 * r.double()[:, 0] + v["gate"].double() * (hat(b.double()[:, 0]) * v["post_weight"].double())
    want = (dn * hat(res)).sum(0)
    # a row's term is off by at most 40 roundings of 2^-24 (two norms, the residual, the product); the sum over the rows is in 64 bits
    assert ((got["pre_weight"].double() - want).abs() <= 40 * O.F24 * (dn * hat(res)).abs().sum(0)).all()


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("S,gates,N,D", [(6, 3, 5, 72), (12, 1, 9, 384), (8, 4, 33, 1100)])
def test_norm_gate_residual_gates_of_several_samples(S, gates, N, D, dt):
    """a gate for several samples' rows, each sample with a multiplier of its own; the branch without a norm, r and h of one gradient"""
    from fedcola_amd.blocks import norm_gate_residual_backward, norm_gate_residual_forward
    for post in (0, 1):
        b, r, dr, _, v = norm_case(S, N, D, dt, "rms", post, 1, "sample", 1, S + D)
        v["gate"] = v["gate"][:gates]
        want, bound = O.norm_gate(b, r, DT[dt], **v, d_residual=dr, d_normed=dr)
        gr, gh = norm_gate_residual_forward(b, r, **v)
        within(gr, want["r"], bound["r"], "r")
        within(gh, want["h"], bound["h"], "h")
        for k, t in norm_gate_residual_backward(dr, dr, b, r, **v).items():
            within(t, want[k], bound[k], k)


def test_norm_gate_residual_module():
    from fedcola_amd.blocks import NormGateResidual
    for kind in ("layer", "rms"):
        m = NormGateResidual(48, norm=kind, gate_init=0.5, residual_scale=0.8, device="cuda")
        b, r = rnd(gen(0), 3, 7, 48).requires_grad_(True), rnd(gen(1), 3, 7, 48).requires_grad_(True)
        s = torch.tensor([1.0, 0.0, 2.0], device="cuda")
        x, h = m(b, r, row_scale=s)
        dh = rnd(gen(2), 3, 7, 48)
        h.backward(dh)                                               # r's own gradient absent
        want, _ = O.norm_gate(b.detach(), r.detach(), torch.float32, post_weight=m.post_weight.detach(), post_bias=None if m.post_bias is None else m.post_bias.detach(),
                              gate=m.gate.detach(), row_scale=s, residual_scale=0.8, pre_weight=m.pre_weight.detach(),
                              pre_bias=None if m.pre_bias is None else m.pre_bias.detach(), norm=kind, d_normed=dh)
        for got, k in ((x, "r"), (h, "h"), (b.grad, "branch"), (r.grad, "residual"), (m.gate.grad, "gate"), (m.post_weight.grad, "post_weight"), (m.pre_weight.grad, "pre_weight")):
            assert (got.double() - want[k]).norm() <= 2e-6 * want[k].norm(), k


# ------------------------------------------------------------------------------------------------ together, as a program uses them
def tower(x, y, P, act="silu", s=None):
    """a residual stream through two gated feed-forward branches to the vocabulary loss; returns the loss"""
    from fedcola_amd.blocks import gated_mlp, norm_gate_residual
    from fedcola_amd.criterions import LinearCrossEntropyLoss
    r = x
    zero = torch.zeros_like(x)
    r, h = norm_gate_residual(zero, r, pre_weight=P["n0"], norm="rms")
    for i in range(2):
        b = gated_mlp(h, P[f"wi{i}"], P[f"wo{i}"], act)
        r, h = norm_gate_residual(b, r, post_weight=P[f"p{i}"], gate=P[f"g{i}"], row_scale=s, pre_weight=P[f"n{i + 1}"], norm="rms")
    return LinearCrossEntropyLoss()(h, P["w"], y)


def tower64(x, y, P, s):
    norm = lambda v, w: v / (v.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w  # noqa: E731
    r, h = x, norm(x, P["n0"])
    for i in range(2):
        g, u = (h @ P[f"wi{i}"].t()).chunk(2, -1)
        b = (torch.nn.functional.silu(g) * u) @ P[f"wo{i}"].t()
        r = r + s.double()[:, None, None] * norm(b, P[f"p{i}"]) * P[f"g{i}"]
        h = norm(r, P[f"n{i + 1}"])
    return torch.nn.functional.cross_entropy((h @ P["w"].t()).flatten(0, 1), y.flatten())


def tower_case(dt, B=3, N=41, D=64, F=136, V=500, seed=0):
    g = gen(seed)
    P = dict(w=rnd(g, V, D, scale=0.2, dtype=dt))
    for i in range(2):
        P.update({f"wi{i}": rnd(g, 2 * F, D, scale=1 / math.sqrt(D), dtype=dt), f"wo{i}": rnd(g, D, F, scale=1 / math.sqrt(F), dtype=dt),
                  f"p{i}": 1 + 0.1 * rnd(g, D), f"g{i}": 0.5 + 0.1 * rnd(g, D)})
    P.update({f"n{i}": 1 + 0.1 * rnd(g, D) for i in range(3)})
    y = torch.randint(0, V, (B, N), generator=g, device="cuda")
    y[:, -9:] = -100
    return rnd(g, B, N, D, dtype=dt), y, P, torch.tensor([1.0, 0.0, 2.0], device="cuda")[:B]


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_operators_together(dt):
    x, y, P, s = tower_case(DT[dt])
    leaves = {"x": x.requires_grad_(True), **{k: v.requires_grad_(True) for k, v in P.items()}}
    loss = tower(x, y, P, s=s)
    got = torch.autograd.grad(loss, list(leaves.values()))
    wide = {k: v.detach().double().requires_grad_(True) for k, v in leaves.items()}
    ref = tower64(wide["x"], y, wide, s)
    want = torch.autograd.grad(ref, list(wide.values()))
    # a gradient passes at most 16 stored roundings of u each, which are independent: their sum in norm stays under 16 u, and in fp32 under that
    # of 16 sums of about 500 terms
    tol = 16 * O.half_step(DT[dt]) if dt == "bf16" else 16 * O.acc(500)
    assert abs(loss.item() - ref.item()) <= tol * abs(ref.item())
    for k, a, b in zip(leaves, got, want):
        assert a.dtype == leaves[k].dtype
        assert (a.double() - b).norm() <= tol * b.norm(), (k, float((a.double() - b).norm() / b.norm()))


@pytest.mark.parametrize("dt,sizes", [("bf16", {}), ("fp32", {}), ("bf16", dict(B=1, N=12, D=1200)), ("fp32", dict(B=1, N=12, D=1200, V=301)), ("fp32", dict(B=1, N=200, D=1201))])
def test_operators_captured_into_a_graph(dt, sizes):
    """forward and backward of the tower captured once and replayed on new inputs, eager work in between: the eager results, to the bit"""
    x, y, P, s = tower_case(DT[dt], **sizes)
    st = torch.cuda.Stream()
    names = ["x", *P]
    sx, sy = x.clone(), y.clone()

    def step(x_, y_):
        leaves = {"x": x_.detach().requires_grad_(True), **{k: v.detach().requires_grad_(True) for k, v in P.items()}}
        loss = tower(leaves["x"], y_, leaves, s=s)
        return [loss.detach(), *torch.autograd.grad(loss, [leaves[k] for k in names])]
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        for _ in range(2):
            step(sx, sy)
    torch.cuda.current_stream().wait_stream(st)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(sx, sy)
    for k in range(4):
        x2, y2, _, _ = tower_case(DT[dt], seed=20 + k, **sizes)
        eager = step(x2, y2)
        sx.copy_(x2)
        sy.copy_(y2)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, eager):
            assert torch.equal(a, b)


def test_operators_on_two_streams_at_once_and_twice():
    """two calls at once on streams of their own, and again: the same bits as one after the other"""
    cases = [tower_case(torch.bfloat16, N=41 + 7 * i, seed=i) for i in range(2)]

    def step(c):
        x, y, P, s = c
        leaves = [t.detach().requires_grad_(True) for t in (x, *P.values())]
        loss = tower(leaves[0], y, dict(zip(P, leaves[1:])), s=s)
        return [loss.detach(), *torch.autograd.grad(loss, leaves)]
    alone = [step(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(3):
        got = []
        for c, st in zip(cases, streams):
            with torch.cuda.stream(st):
                got.append(step(c))
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_operator_refusals_on_the_device():
    from fedcola_amd import blocks, criterions
    x, w, y = ce_case(8, 20, 16, "bf16", 0.0, 0)
    ce = criterions.linear_cross_entropy_forward
    for bad in (lambda: ce(x, w.float(), y), lambda: ce(x, w[:, :8], y), lambda: ce(x, w, y.int()), lambda: ce(x, w, y[:4]), lambda: ce(x, w, y, reduction="max"),
                lambda: ce(x.half(), w.half(), y), lambda: ce(x, w, y.cpu()), lambda: ce(x, w[:0], y), lambda: blocks.gated_mlp_forward(x, w, w),
                lambda: blocks.gated_mlp_forward(x, w, w[:16, :10].contiguous(), act="relu"), lambda: blocks.norm_gate_residual_forward(x, x[:4]),
                lambda: blocks.norm_gate_residual_forward(x, x, gate=torch.ones(3, 16, device="cuda")), lambda: blocks.norm_gate_residual_forward(x, x, pre_bias=torch.ones(16, device="cuda")),
                lambda: blocks.norm_gate_residual_forward(x, x, gate=x[0]), lambda: blocks.norm_gate_residual_forward(x, x, eps=0.0),
                lambda: blocks.norm_gate_residual_forward(torch.ones(2, 8193, device="cuda"), torch.ones(2, 8193, device="cuda"))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("n", [(1 << 28) + 1, (1 << 32) + 5, 1 << 33])
def test_sizes_past_the_librarys_are_refused(n):
    """row counts, vocabularies and widths that 32 bits do not hold, or that a kernel's offsets do not: refused before anything is laid out (the
    operands are one element, expanded)"""
    from fedcola_amd import blocks, criterions
    one = torch.zeros((), dtype=torch.bfloat16, device="cuda")
    y = torch.zeros((), dtype=torch.int64, device="cuda")
    many = max(n, (1 << 30) + 1)
    for bad in (lambda: criterions.linear_cross_entropy_forward(one.expand(n, 1), one.expand(7, 1), y.expand(n)),
                lambda: criterions.linear_cross_entropy_forward(one.expand(2, 1), one.expand(many, 1), y.expand(2)),
                lambda: criterions.linear_cross_entropy_forward(one.expand(2, n), one.expand(3, n), y.expand(2)),
                lambda: blocks.gated_mlp_forward(one.expand(n, 1), one.expand(4, 1), one.expand(1, 2)),
                lambda: blocks.gated_mlp_forward(one.expand(2, n), one.expand(4, n), one.expand(n, 2)),
                lambda: blocks.gated_mlp_forward(one.expand(2, 1), one.expand(2 * n, 1), one.expand(1, n)),
                lambda: blocks.gated_mlp_backward(one.expand(n, 1), one.expand(n, 1), one.expand(4, 1), one.expand(1, 2))):
        with pytest.raises(ValueError, match="at most"):
            bad()


@pytest.mark.parametrize("T", [5, 40, 520])
def test_fp32_values_next_to_the_largest(T):
    """fp32 values above bf16's largest are finite: where they meet zeros they are not there, where they meet small values they count"""
    from fedcola_amd.blocks import gated_mlp_backward, gated_mlp_forward
    from fedcola_amd.criterions import linear_cross_entropy_backward, linear_cross_entropy_forward
    one = torch.tensor(1.0, device="cuda")
    x, w, y = ce_case(T, 300, 40, "fp32", 0.1, 7)
    x[:, 3], w[:, 3], w[5, 3] = 0.0, LOWEST, -LOWEST
    x[:, 4], w[:, 4] = -LOWEST, 0.0
    want, bound = O.linear_ce(x, w, y, one, -100, "sum", torch.float32)
    loss, saved = linear_cross_entropy_forward(x, w, y, reduction="sum")
    dx, dw = linear_cross_entropy_backward(one, saved, w)
    within(loss, want["loss"], bound["loss"], "loss")
    keep = [i for i in range(40) if i not in (3, 4)]                       # (the two columns' own gradients are sums of such values, past fp32's range)
    within(dx[:, keep], want["dx"][:, keep], bound["dx"][:, keep], "dx")
    within(dw[:, keep], want["dw"][:, keep], bound["dw"][:, keep], "dw")
    g = gen(T)
    D, F = 24, 36
    x, wi, wo, dy = rnd(g, T, D), rnd(g, 2 * F, D, scale=1 / math.sqrt(D)), rnd(g, D, F, scale=1 / math.sqrt(F)), rnd(g, T, D, scale=1e-6)
    x[:, 2], wi[:, 2] = LOWEST, 0.0
    x[0, 5], wi[:F, 5], wi[F:, 5] = LOWEST, 0.0, 2.0 ** -125          # an up projection of about -8 from one such value
    want, bound = O.gated_mlp(x, wi, wo, dy, "silu", torch.float32)
    within(gated_mlp_forward(x, wi, wo), want["y"], bound["y"], "y")
    for k, t in zip(("dx", "dw_in", "dw_out"), gated_mlp_backward(dy, x, wi, wo)):
        assert torch.isfinite(t).all()
        within(t, want[k], bound[k], k)


# ------------------------------------------------------------------------------------------------ offsets past 32 bits
def test_offsets_past_32_bits_in_the_vocabulary():
    """a weight of 4.9 GB, zeros but for three rows: everything has a closed form"""
    from fedcola_amd.criterions import linear_cross_entropy_backward, linear_cross_entropy_forward
    V, D, T = 1_200_000, 2048, 5
    w = torch.zeros(V, D, dtype=torch.bfloat16, device="cuda")
    hot = torch.tensor([0, V // 2 + 1, V - 1], device="cuda")
    w[hot] = rnd(gen(0), 3, D, scale=0.2).bfloat16()
    x = rnd(gen(1), T, D).bfloat16()
    y = torch.tensor([V - 1, 0, V // 2 + 1, 77, V - 2], device="cuda")
    loss, saved = linear_cross_entropy_forward(x, w, y, reduction="sum")
    dx, dw = linear_cross_entropy_backward(torch.tensor(1.0, device="cuda"), saved, w)
    wide = torch.cat([w[hot].double(), torch.zeros(1, D, device="cuda", dtype=torch.float64)])
    logits = x.double() @ wide.t()
    lse = torch.log(torch.exp(logits[:, :3]).sum(1) + (V - 3))
    at = torch.tensor([2, 0, 1, 3, 3], device="cuda")
    rows = lse - logits.gather(1, at[:, None])[:, 0]
    assert abs(loss.double() - rows.sum()) <= 1e-6 * rows.sum()
    p = torch.exp(logits - lse[:, None])
    # two roundings of u; a logit of 2048 products of about 0.13 each is off by at most (64 + 32) 2^-24 x 270 = 1.6e-3 (64 accumulations of 32
    # products), and so are lse and, twice, p
    tol = 1.1 * (2 * O.half_step(torch.bfloat16) + 4e-3)
    for k, v in enumerate(hot.tolist()):
        d = p[:, k] - (y == v).double()
        want = d @ x.double()
        within(dw[v], want, tol * (d.abs() @ x.double().abs()), f"dw row {v}")
    for v in (1, V // 2, V - 3):                                              # rows that nothing points at: 1 / V each
        d = p[:, 3]
        within(dw[v], d @ x.double(), tol * (d.abs() @ x.double().abs()), f"dw row {v}")
    d = p[:, :3] - (y[:, None] == hot).double()
    within(dx, d @ wide[:3], tol * (d.abs() @ wide[:3].abs()), "dx")


def test_offsets_past_32_bits_in_the_rows():
    """more than 4 GB of rows: the first, the last and some in between against the same rows alone"""
    from fedcola_amd.blocks import gated_mlp_backward, gated_mlp_forward, norm_gate_residual_backward, norm_gate_residual_forward
    T, D = 1_100_000, 2048
    x = torch.empty(T, D, dtype=torch.bfloat16, device="cuda").normal_(generator=gen(0))
    some = torch.tensor([0, 1, 524_288, 1_048_575, 1_048_577, T - 2, T - 1], device="cuda")
    wi, wo = rnd(gen(1), 32, D, scale=0.02).bfloat16(), rnd(gen(2), D, 16, scale=0.2).bfloat16()
    y = gated_mlp_forward(x, wi, wo)
    dx, _, _ = gated_mlp_backward(x, x, wi, wo, need=(True, False, False))
    want, bound = O.gated_mlp(x[some], wi, wo, x[some], "silu", torch.bfloat16)
    within(y[some], want["y"], bound["y"], "y")
    within(dx[some], want["dx"], bound["dx"], "dx")
    del y, dx
    v = dict(post_weight=torch.ones(D, device="cuda"), gate=rnd(gen(3), D), pre_weight=torch.ones(D, device="cuda"), norm="rms")
    r, h = norm_gate_residual_forward(x, x, **v)
    d = norm_gate_residual_backward(x, x, x, x, weight_grads=False, **v)
    one = x[some][None]
    want, bound = O.norm_gate(one, one, torch.bfloat16, **v, d_residual=one, d_normed=one)
    for got, k in ((r, "r"), (h, "h"), (d["branch"], "branch"), (d["residual"], "residual")):
        within(got[some][None], want[k], bound[k], k)
