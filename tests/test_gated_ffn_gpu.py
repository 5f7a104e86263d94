"""The gated feed-forward block and its backward pass against the formulas in 64 bits.

Tolerances, from the arithmetic. One product of split operands: a factor is off by at most 2^-23
of itself each, the dropped lo lo term is below 2^-22, and each of the 24 accumulations of a chunk
may truncate up to 2^-23 of the running sum, in all below (2 + 2 + 24) 2^-23 of |A||B| (3.4e-6);
the chunks then add in fp32, 2^-24 each. So an entry is off by TOL |A||B| with
TOL = 3.5e-6 + chunks * 6e-8, plus 2^-39 of a block's largest entry per operand entry (1e-11
relative to it, included in the constant for the distributions here). The activation adds a few
fp32 roundings (8 ulp, 1e-6). Bounds of later products are propagated through their factors."""
import numpy as np
import pytest
import torch

import mensurflow_b200 as mf

pytestmark = pytest.mark.gpu


def tol(depth):
    return 3.5e-6 + (depth + 127) // 128 * 6e-8


def few_rows(depth):
    """Up to 16 rows without saving: fp32 FMAs, a chain of depth / 8 at most (one warp's share) and
    then at most three halvings, eight ranks and, where lanes share the depth, five more."""
    return (depth / 8 + 16) * 2.0 ** -24


def act64(v, kind):
    if kind == "relu":
        return v.clamp(min=0), (v > 0).double()
    if kind == "silu":
        s = torch.sigmoid(v)
        return v * s, s * (1 + v * (1 - s))
    if kind == "gelu":
        cdf = torch.special.ndtr(v)
        return v * cdf, cdf + v * torch.exp(-v * v / 2) / np.sqrt(2 * np.pi)
    if kind == "gelu_tanh":
        s = torch.sigmoid(2 * np.sqrt(2 / np.pi) * (v + 0.044715 * v ** 3))
        return v * s, s + 2 * v * s * (1 - s) * np.sqrt(2 / np.pi) * (1 + 0.134145 * v * v)
    return v, torch.ones_like(v)


def want(x, wg, wu, wd, dy, kind, tol=tol):
    """Outputs of the forward and backward pass with their error bounds, all in 64 bits."""
    x, wg, wu, wd, dy = (t.double() for t in (x, wg, wu, wd, dy))
    g, u = x @ wg, x @ wu
    td, tf, tm = tol(x.shape[1]), tol(wd.shape[0]), tol(x.shape[0])
    eg, eu = td * (x.abs() @ wg.abs()), td * (x.abs() @ wu.abs())
    a, s = act64(g, kind)
    # |act'| <= 1.13; a relu slope may flip where |g| is within its error
    ea = 1.13 * eg + 1e-6 * a.abs()
    es = 1.2 * eg + 1e-6 + ((g.abs() <= eg).double() if kind == "relu" else 0)
    h = a * u
    eh = ea * u.abs() + a.abs() * eu + ea * eu + 1e-6 * h.abs()
    y = h @ wd
    out = {"y": (y, eh @ wd.abs() + tf * ((h.abs() + eh) @ wd.abs()))}
    dh = dy @ wd.t()
    edh = td * (dy.abs() @ wd.abs().t())
    dg, du = dh * u * s, dh * a
    edg = (edh * u.abs() + dh.abs() * eu) * (s.abs() + es) + (dh * u).abs() * es + \
        1e-6 * dg.abs()
    edu = edh * (a.abs() + ea) + dh.abs() * ea + 1e-6 * du.abs()
    ag, au, ah = dg.abs() + edg, du.abs() + edu, h.abs() + eh
    out["dx"] = (dg @ wg.t() + du @ wu.t(),
                 edg @ wg.abs().t() + edu @ wu.abs().t() +
                 2 * tf * (ag @ wg.abs().t() + au @ wu.abs().t()))
    out["dwg"] = (x.t() @ dg, x.abs().t() @ edg + tm * (x.abs().t() @ ag))
    out["dwu"] = (x.t() @ du, x.abs().t() @ edu + tm * (x.abs().t() @ au))
    out["dwd"] = (h.t() @ dy, eh.t() @ dy.abs() + tm * (ah.t() @ dy.abs()))
    return out


def close(got, pair, what):
    ref, bound = pair
    err = (got.double() - ref).abs()
    bad = ~(err <= bound + 1e-30)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} entries out of bounds, "
                           f"worst {float((err / (bound + 1e-30)).max()):.3g} times its bound")


def inputs(cuda, rows, d, f, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 7 + d * 3 + f)
    n = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    k = (2.0 / (d + f)) ** 0.5
    return n(rows, d), n(d, f) * k, n(d, f) * k, n(f, d) * k, n(rows, d)


SIZES = [(1, 1, 1), (2, 3, 5), (1, 1024, 640), (3, 257, 1030), (7, 96, 2050), (8, 640, 4096),
         (13, 500, 333), (16, 1028, 260), (17, 64, 96), (20, 700, 2304), (33, 65, 127), (90, 1500, 260),
         (128, 516, 3000), (64, 128, 256), (127, 129, 255),
         (128, 256, 128), (200, 100, 300), (257, 384, 513), (300, 1003, 771), (1031, 520, 900)]


@pytest.mark.parametrize("shape", SIZES)
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu", None])
def test_forward_and_backward(cuda, shape, act):
    x, wg, wu, wd, dy = inputs(cuda, *shape)
    ref = want(x, wg, wu, wd, dy, act)
    y, saved = mf.gated_ffn(x, wg, wu, wd, act, save=True)
    close(y, ref["y"], f"{shape} y")
    close(mf.gated_ffn(x, wg, wu, wd, act),
          want(x, wg, wu, wd, dy, act, few_rows)["y"] if shape[0] <= 16 else ref["y"],
          f"{shape} y without saving")
    grads = mf.gated_ffn_backward(dy, x, wg, wu, wd, act, saved=saved)
    for got, name in zip(grads, ("dx", "dwg", "dwu", "dwd")):
        close(got, ref[name], f"{shape} {name}")
    again = mf.gated_ffn_backward(dy, x, wg, wu, wd, act)      # projections computed again
    for got, name in zip(again, ("dx", "dwg", "dwu", "dwd")):
        close(got, ref[name], f"{shape} {name} without saved")
    assert mf.device_status() == 0


@pytest.mark.parametrize("rows", [1, 2, 4, 5, 16, 40, 128, 129])
@pytest.mark.parametrize("d,f", [(64, 200), (129, 333), (1024, 516), (2, 1)])
def test_weights_stored_outputs_first(cuda, rows, d, f):
    """transpose_w: the same block from [outputs, inputs] weights, gradients in their layout."""
    x, wg, wu, wd, dy = inputs(cuda, rows, d, f)
    ref = want(x, wg, wu, wd, dy, "silu")
    few = want(x, wg, wu, wd, dy, "silu", few_rows) if rows <= 16 else ref
    stored = [t.t().contiguous() for t in (wg, wu, wd)]
    close(mf.gated_ffn(x, *stored, transpose_w=True), few["y"], "y")
    y, saved = mf.gated_ffn(x, *stored, transpose_w=True, save=True)
    close(y, ref["y"], "y")
    dx, *dw = mf.gated_ffn_backward(dy, x, *stored, saved=saved, transpose_w=True)
    close(dx, ref["dx"], "dx")
    for got, name, w in zip(dw, ("dwg", "dwu", "dwd"), stored):
        assert got.shape == w.shape and got.is_contiguous()
        close(got.t(), ref[name], name)
    assert mf.device_status() == 0
