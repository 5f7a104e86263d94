"""The gated feed-forward block and its backward pass against the formulas in 64 bits.

Tolerances, from the arithmetic. One product of split operands: a factor is off by at most 2^-23
of itself each, the dropped lo lo term is below 2^-22, and each of the 24 accumulations of a chunk
may truncate up to 2^-23 of the running sum, in all below (2 + 2 + 24) 2^-23 of |A||B| (3.4e-6);
the chunks then add in fp32, 2^-24 each. So an entry is off by TOL |A||B| with
TOL = 3.5e-6 + chunks * 6e-8, plus 2^-39 of a block's largest entry per operand entry (1e-11
relative to it, included in the constant for the distributions here). The activation adds a few
fp32 roundings (8 ulp, 1e-6). Bounds of later products are propagated through their factors."""
import ctypes

import numpy as np
import pytest
import torch

import mensurflow_b200 as mf
from mensurflow_b200 import _lib

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


@pytest.mark.parametrize("shape", [(600, 700, 900), (2100, 260, 1300), (640, 2048, 300)])
def test_larger_tiles(cuda, shape):
    """Sizes that fill 256 x 256 tiles, share contractions in clusters and leave ragged ends."""
    x, wg, wu, wd, dy = inputs(cuda, *shape)
    ref = want(x, wg, wu, wd, dy, "gelu")
    y, saved = mf.gated_ffn(x, wg, wu, wd, "gelu", save=True)
    close(y, ref["y"], "y")
    grads = mf.gated_ffn_backward(dy, x, wg, wu, wd, "gelu", saved=saved)
    for got, name in zip(grads, ("dx", "dwg", "dwu", "dwd")):
        close(got, ref[name], name)
    assert mf.device_status() == 0


@pytest.mark.parametrize("rows", [1, 6, 16, 50, 300])
def test_views(cuda, rows):
    """Sliced, transposed and stepped tensors give what their packed copies give, bit for bit where
    the same kernel runs, and gradients of leading dimensions fold."""
    d, f = 132, 260
    x, wg, wu, wd, dy = inputs(cuda, rows, d, f)
    wide = torch.randn(rows, d + 9, device=cuda)
    wide[:, 4:4 + d] = x
    big = torch.randn(d, f + 13, device=cuda)
    big[:, 5:5 + f] = wg
    views = {
        "sliced rows": (wide[:, 4:4 + d], wg, wu, wd),
        "sliced weights": (x, big[:, 5:5 + f], wu, wd),
        "column-major weights": (x, wg.t().contiguous().t(), wu.t().contiguous().t(),
                                 wd.t().contiguous().t()),
        "one of each": (x, wg.t().contiguous().t(), wu, wd),
        "column-major rows": (x.t().contiguous().t(), wg, wu, wd),
        "stepped": (torch.repeat_interleave(x, 2, 1)[:, ::2], wg, wu, wd),
    }
    ref = want(x, wg, wu, wd, dy, "silu")
    few = want(x, wg, wu, wd, dy, "silu", few_rows) if rows <= 16 else ref
    for name, (a, b, c, e) in views.items():
        assert torch.equal(a, x) and torch.equal(b, wg)
        close(mf.gated_ffn(a, b, c, e), few["y"], name)
        y, saved = mf.gated_ffn(a, b, c, e, save=True)
        close(y, ref["y"], name)
        grads = mf.gated_ffn_backward(dy.t().contiguous().t(), a, b, c, e, saved=saved)
        for got, key in zip(grads, ("dx", "dwg", "dwu", "dwd")):
            assert got.is_contiguous()
            close(got, ref[key], f"{name} {key}")
    if rows % 2 == 0:
        three = x.view(2, rows // 2, d)
        y = mf.gated_ffn(three, wg, wu, wd)
        assert y.shape == three.shape
        close(y.reshape(rows, d), few["y"], "three dimensions")
        dx = mf.gated_ffn_backward(dy.view_as(three), three, wg, wu, wd, need_w=False)[0]
        assert dx.shape == three.shape
        close(dx.reshape(rows, d), ref["dx"], "three dimensions dx")
    vector = mf.gated_ffn(x[0], wg, wu, wd)
    assert vector.shape == (d,)
    assert mf.device_status() == 0


def test_needed_gradients_only(cuda):
    x, wg, wu, wd, dy = inputs(cuda, 140, 130, 200)
    full = mf.gated_ffn_backward(dy, x, wg, wu, wd)
    dx, *none = mf.gated_ffn_backward(dy, x, wg, wu, wd, need_w=False)
    assert none == [None] * 3 and torch.equal(dx, full[0])
    no_x, *dw = mf.gated_ffn_backward(dy, x, wg, wu, wd, need_x=False)
    assert no_x is None and all(torch.equal(a, b) for a, b in zip(dw, full[1:]))
    assert mf.gated_ffn_backward(dy, x, wg, wu, wd, need_x=False, need_w=False) == (None,) * 4


def test_empty(cuda):
    e = lambda *s: torch.empty(*s, device=cuda)  # noqa: E731
    x, wg, wu, wd, _ = inputs(cuda, 3, 20, 30)
    assert mf.gated_ffn(e(0, 20), wg, wu, wd).shape == (0, 20)
    assert mf.gated_ffn(e(2, 0, 20), wg, wu, wd).shape == (2, 0, 20)
    y, saved = mf.gated_ffn(e(0, 20), wg, wu, wd, save=True)
    dx, *dw = mf.gated_ffn_backward(e(0, 20), e(0, 20), wg, wu, wd, saved=saved)
    assert dx.shape == (0, 20) and all((t == 0).all() for t in dw)
    assert all(t.shape == w.shape for t, w in zip(dw, (wg, wu, wd)))
    zero = mf.gated_ffn(x, e(20, 0), e(20, 0), e(0, 20))          # no features: zeros
    assert zero.shape == (3, 20) and (zero == 0).all()
    dx, *dw = mf.gated_ffn_backward(x, x, e(20, 0), e(20, 0), e(0, 20))
    assert (dx == 0).all() and [tuple(t.shape) for t in dw] == [(20, 0), (20, 0), (0, 20)]
    assert mf.gated_ffn(e(4, 0), e(0, 30), e(0, 30), e(30, 0)).shape == (4, 0)
    assert mf.device_status() == 0


@pytest.mark.parametrize("rows", [9, 77, 700])
def test_rows_do_not_depend_on_one_another(cuda, rows):
    """A batch's rows keep their bits whatever the others hold: huge values, infinities, NaN."""
    x, wg, wu, wd, dy = inputs(cuda, rows, 101, 203)
    y = mf.gated_ffn(x, wg, wu, wd)
    half = rows // 2
    for filler in (1e6, 1e30, float("inf"), float("nan")):
        other = x.clone()
        other[half:] = filler
        got = mf.gated_ffn(other, wg, wu, wd)
        assert torch.equal(got[:half], y[:half]), filler
        if filler > 1e30 or filler != filler:
            assert not torch.isfinite(got[half:]).any()
    one = x.clone()
    one[3, 7] = float("inf")
    got = mf.gated_ffn(one, wg, wu, wd)
    assert not torch.isfinite(got[3]).any()
    keep = [i for i in range(rows) if i != 3]
    assert torch.equal(got[keep], y[keep])


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu", None])
def test_rows_without_a_gradient_take_no_part(cuda, act):
    """A padded batch: rows whose gradient is zero add nothing, whatever lies in them."""
    x, wg, wu, wd, dy = inputs(cuda, 210, 130, 190)
    dy[150:] = 0
    ref = want(x[:150], wg, wu, wd, dy[:150], act)
    for filler in (0.0, 3.0, 1e6, 1e30):
        x[150:] = filler
        for keep in (True, False):
            saved = mf.gated_ffn(x, wg, wu, wd, act, save=True)[1] if keep else None
            dx, *dw = mf.gated_ffn_backward(dy, x, wg, wu, wd, act, saved=saved)
            assert (dx[150:] == 0).all()
            close(dx[:150], ref["dx"], f"dx {filler}")
            for got, name in zip(dw, ("dwg", "dwu", "dwd")):
                close(got, ref[name], f"{name} {filler}")
    assert mf.device_status() == 0


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e12, 1e25])
def test_scales(cuda, scale):
    """Magnitudes far from 1: the scales carry them. The gate is x w_gate in both, the up projection
    scales with x in the first call."""
    x, wg, wu, wd, dy = inputs(cuda, 200, 96, 160)
    y = mf.gated_ffn(x * scale, wg / scale, wu, wd, "relu")
    ref = want(x, wg, wu, wd, dy, "relu")["y"]
    close(y.double() / scale, (ref[0], ref[1] * 1.01), f"x {scale}")
    y = mf.gated_ffn(x, wg, wu / scale, wd * scale, "relu")
    close(y, (ref[0], ref[1] * 1.01), f"w_down {scale}")


def test_gradients_against_differences(cuda):
    """Central differences of the loss in 64 bits of the inputs' own values, along random
    directions: the step's error is of order h^2, about 1e-5 of the derivative here."""
    x, wg, wu, wd, dy = inputs(cuda, 150, 40, 70)
    grads = mf.gated_ffn_backward(dy, x, wg, wu, wd, "gelu_tanh")

    def loss(tensors):
        a, b, c, e = tensors
        act, _ = act64(a @ b, "gelu_tanh")
        return float((((act * (a @ c)) @ e) * dy.double()).sum())

    base = [t.double() for t in (x, wg, wu, wd)]
    gen = torch.Generator(device="cuda").manual_seed(5)
    for i, g in enumerate(grads):
        step = torch.randn(base[i].shape, generator=gen, device=cuda, dtype=torch.float64)
        h = 1e-4
        plus = [t + h * step if j == i else t for j, t in enumerate(base)]
        minus = [t - h * step if j == i else t for j, t in enumerate(base)]
        slope = (loss(plus) - loss(minus)) / (2 * h)
        size = float((g.double().abs() * step.abs()).sum())
        assert abs(float((g.double() * step).sum()) - slope) <= 1e-5 * size


def test_streams_and_graphs(cuda):
    """On another stream, two streams at once, and captured into two graphs that replay in turn
    with new inputs: the results of plain calls, bit for bit."""
    x, wg, wu, wd, dy = inputs(cuda, 200, 130, 300)
    few = x[:4].contiguous()

    def everything(a, b, g):
        y, saved = mf.gated_ffn(a, wg, wu, wd, save=True)
        return (y, mf.gated_ffn(b, wg, wu, wd)) + mf.gated_ffn_backward(g, a, wg, wu, wd,
                                                                      saved=saved)

    plain = everything(x, few, dy)
    side = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for s in side:
            with torch.cuda.stream(s):
                results.append(everything(x, few, dy))
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(r, plain))
    ax, ag = x.clone(), dy.clone()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(everything(ax, ax[:4], ag))
        graphs.append(g)
    for seed in range(3):
        nx, _, _, _, ng = inputs(cuda, 200, 130, 300, seed + 1)
        ax.copy_(nx)
        ag.copy_(ng)
        expect = everything(ax, ax[:4], ag)
        for g, out in zip(graphs, outs):
            g.replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, expect))
    assert mf.device_status() == 0


def test_repeated_calls_give_the_same_bits(cuda):
    x, wg, wu, wd, dy = inputs(cuda, 700, 900, 500)
    first = mf.gated_ffn_backward(dy, x, wg, wu, wd)
    for _ in range(3):
        assert all(torch.equal(a, b)
                   for a, b in zip(first, mf.gated_ffn_backward(dy, x, wg, wu, wd)))


def test_saved_of_another_call_is_refused(cuda):
    x, wg, wu, wd, dy = inputs(cuda, 20, 30, 40)
    saved = mf.gated_ffn(x, wg, wu, wd, save=True)[1]
    with pytest.raises(TypeError):
        mf.gated_ffn_backward(dy, x, wg, wu, wd, saved=saved.buffer)
    with pytest.raises(ValueError, match="another call"):
        mf.gated_ffn_backward(dy[:5], x[:5], wg, wu, wd, saved=saved)
    with pytest.raises(ValueError, match="another call"):
        mf.gated_ffn_backward(dy, x, wg, wu, wd, "gelu", saved=saved)
    with pytest.raises(ValueError, match="another call"):
        mf.gated_ffn_backward(dy, x, wg, wu, wd,
                              saved=mf.GatedSaved(saved.buffer[:8], 20, 40, "silu"))
    with pytest.raises(ValueError, match="differs from x"):
        mf.gated_ffn_backward(dy[:, :5], x, wg, wu, wd)
    with pytest.raises(ValueError, match="different devices"):
        mf.gated_ffn(x, wg.cpu(), wu, wd)
    with pytest.raises(ValueError, match="different devices"):
        mf.gated_ffn_backward(dy.cpu(), x, wg, wu, wd)
    with pytest.raises(ValueError, match="different devices"):
        mf.embedding(x, torch.zeros(3, dtype=torch.int64))
    assert mf.device_status() == 0


@pytest.mark.parametrize("shape", [(300, 140, 600), (17, 520, 130), (1300, 260, 900)])
@pytest.mark.parametrize("down_transposed", [False, True])
@pytest.mark.parametrize("transposed", [False, True])
def test_layouts_of_the_weight_gradients(cuda, shape, transposed, down_transposed):
    """Each weight gradient row-major or column-major, with a row stride of its own, in guarded
    memory: what lies between the rows stays."""
    rows, d, f = shape
    x, wg, wu, wd, dy = inputs(cuda, rows, d, f)
    ref = mf.gated_ffn_backward(dy, x, wg, wu, wd, need_x=False)[1:]
    pad = 5

    def guarded(r, c, t):
        base = torch.full((c, r + pad) if t else (r, c + pad), -7.0, device=cuda)
        return base, (base[:, :r].t() if t else base[:, :c])

    outs = [guarded(d, f, transposed), guarded(d, f, transposed), guarded(f, d, down_transposed)]
    desc = _lib.GatedFfnDesc(x.data_ptr(), d, 1, wg.data_ptr(), f, 1, wu.data_ptr(), f, 1,
                             wd.data_ptr(), d, 1, rows, d, f, _lib.ACT_SILU, 0)
    o = _lib.GatedFfnGrads()
    o.grad, o.grad_rs, o.grad_cs = dy.data_ptr(), d, 1
    o.dw_gate, o.dw_up, o.dw_down = (b.data_ptr() for b, _ in outs)
    o.dw_rs, o.dw_cs = outs[0][1].stride()
    o.dw_down_rs, o.dw_down_cs = outs[2][1].stride()
    assert _lib.lib().mfk_gated_ffn_backward_f32(
        ctypes.byref(desc), ctypes.byref(o), None,
        ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    for (base, view), expect in zip(outs, ref):
        # another operand order adds the same terms in another order
        scale = expect.abs().max()
        assert float((view - expect).abs().max()) <= 2 * tol(rows) * 8 * float(scale)
        assert bool((base[:, -pad:] == -7.0).all())
    assert mf.device_status() == 0


def test_offsets_past_32_bits(cuda):
    """x, y and the gradients of more than 2^31 entries: the last rows against 64 bits. (The same
    rows alone share their contractions among clusters: other sums, other last bits.)"""
    d, f, rows = 8192, 130, 2 ** 18 + 77
    if torch.cuda.mem_get_info()[0] < 90e9:
        pytest.skip("needs 90 GB")
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.empty(rows, d, device=cuda)
    x.normal_(generator=g)
    wg, wu, wd = (torch.randn(*s, generator=g, device=cuda) * 0.02 for s in ((d, f), (d, f), (f, d)))
    last = 205                                   # 256 * 1024 + 77 ends 77 rows into a block
    y, saved = mf.gated_ffn(x, wg, wu, wd, save=True)
    close(y[-last:], want(x[-last:], wg, wu, wd, x[-last:], "silu")["y"], "y")
    del y
    grad = torch.zeros(rows, d, device=cuda)
    grad[-77:].normal_(generator=g)              # the rest adds nothing to the weights' gradients
    dx, *dw = mf.gated_ffn_backward(grad, x, wg, wu, wd, saved=saved)
    pairs = want(x[-77:], wg, wu, wd, grad[-77:], "silu")
    close(dx[-77:], pairs["dx"], "dx")
    for got, name in zip(dw, ("dwg", "dwu", "dwd")):
        close(got, pairs[name], name)
    assert not dx[:-77].any()
    assert mf.device_status() == 0


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu", None])
@pytest.mark.parametrize("filler", [float("nan"), float("inf"), -float("inf"), 3e38])
def test_rows_without_a_gradient_may_hold_anything(cuda, act, filler):
    """Rows whose gradient is zero add nothing and get a zero dx where x is not finite, or finite
    and the projections overflow: in whole rows and in single entries."""
    x, wg, wu, wd, dy = inputs(cuda, 210, 130, 190)
    dy[150:] = 0
    ref = want(x[:150], wg, wu, wd, dy[:150], act)
    x[150:200] = filler
    x[201:, 5] = filler
    for keep in (True, False):
        saved = mf.gated_ffn(x, wg, wu, wd, act, save=True)[1] if keep else None
        dx, *dw = mf.gated_ffn_backward(dy, x, wg, wu, wd, act, saved=saved)
        assert (dx[150:] == 0).all()
        close(dx[:150], ref["dx"], "dx")
        for got, name in zip(dw, ("dwg", "dwu", "dwd")):
            close(got, ref[name], name)
    assert mf.device_status() == 0


def exact_projections(cuda, rows, d, f, center, seed):
    """Inputs whose gate, up and dh are exact in fp32: gate = x[:, 0] w_gate[0] with w_gate[0]
    within 1/4 of `center`, up = x[:, 1] w_up[1], grad and w_down in few bits. The other columns of
    x are random and meet zeros in the weights."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    whole = lambda low, high, *s: torch.randint(low, high, s, generator=g, device=cuda).float()  # noqa: E731
    x = torch.randn(rows, d, generator=g, device=cuda)
    x[:, 0], x[:, 1] = 1.0, whole(1, 9, rows) / 8
    wg, wu = torch.zeros(d, f, device=cuda), torch.zeros(d, f, device=cuda)
    wg[0] = center + whole(-16, 17, f) / 64
    wu[1] = whole(-16, 17, f) / 8
    return x, wg, wu, whole(-8, 9, f, d) / 32, whole(-8, 9, rows, d) / 8


def rounded_act(g, kind):
    """Relative errors of act(g) and act'(g) in the kernels, from their expressions. The
    exponential's argument z carries 2.5 roundings (6.5 for tanh-GELU's cube), |z| 2^-24 each; ex2
    and rcp are off by 2^-22 and 2^-23, the few products by 2^-24; the derivative's factor beside the
    exponential, one sum without cancellation for gates this far out, adds as much again."""
    if kind == "silu":
        z = g.abs()
    elif kind == "gelu":
        z = g * g / 2
    elif kind == "gelu_tanh":
        z = 2.6 * 2 * np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3).abs()
    else:
        return torch.zeros_like(g), torch.zeros_like(g)
    a = z * 2.5 * 2.0 ** -24 + 2.0 ** -20
    return a, 1.2 * a + 2.0 ** -21


def check_backward_scales(got, x, wg, wu, wd, dy, kind, edh=0.0, what=""):
    """The gradients against 64 bits where gate and up are exact and dh is off by `edh`: the
    activation's roundings, 2^-36 of the largest entry of dgate, dup and h for the scale that a
    block of them shares (at most three powers of two above its largest entry), and the products'
    own error."""
    x, wg, wu, wd, dy = (t.double() for t in (x, wg, wu, wd, dy))
    g, u, dh = x[:, :1] @ wg[:1], x[:, 1:2] @ wu[1:2], dy @ wd.t()
    a, s = act64(g, kind)
    ea, es = rounded_act(g, kind)
    h, dg, du = a * u, dh * u * s, dh * a
    tf, tm = tol(wd.shape[0]), tol(x.shape[0])
    floor = lambda t: 2.0 ** -36 * t.abs().max()  # noqa: E731
    eh = h.abs() * (ea + 2.0 ** -22) + floor(h)
    edg = dg.abs() * (es + 2.0 ** -22) + edh * (u * s).abs() + floor(dg)
    edu = du.abs() * (ea + 2.0 ** -22) + edh * a.abs() + floor(du)
    ref = {
        "dx": (dg @ wg.t() + du @ wu.t(), edg @ wg.abs().t() + edu @ wu.abs().t() +
               2 * tf * ((dg.abs() + edg) @ wg.abs().t() + (du.abs() + edu) @ wu.abs().t())),
        "dwg": (x.t() @ dg, x.abs().t() @ (edg + tm * (dg.abs() + edg))),
        "dwu": (x.t() @ du, x.abs().t() @ (edu + tm * (du.abs() + edu))),
        "dwd": (h.t() @ dy, (eh + tm * (h.abs() + eh)).t() @ dy.abs()),
    }
    for t, name in zip(got, ("dx", "dwg", "dwu", "dwd")):
        close(t, ref[name], f"{what} {name}")


@pytest.mark.parametrize("act,center", [("silu", -20.0), ("silu", -40.0), ("gelu", -6.0),
                                        ("gelu_tanh", -5.0), ("gelu", 6.0), ("relu", -1.0)])
@pytest.mark.parametrize("shape", [(200, 96, 160), (3, 40, 130), (2100, 70, 2600),
                                   (520, 2000, 300), (1900, 4096, 2000), (1000, 8192, 1000)])
def test_saturated_gates(cuda, act, center, shape):
    """Blocks whose gates are all far out, where act and act' are tiny beside gate and up: the
    gradients keep their bits. Tiles of one CTA and of pairs, with the contraction shared by a
    cluster and not."""
    x, wg, wu, wd, dy = exact_projections(cuda, *shape, center, 7)
    for keep in (True, False):
        saved = mf.gated_ffn(x, wg, wu, wd, act, save=True)[1] if keep else None
        got = mf.gated_ffn_backward(dy, x, wg, wu, wd, act, saved=saved)
        check_backward_scales(got, x, wg, wu, wd, dy, act, what=str(keep))
    assert mf.device_status() == 0


@pytest.mark.parametrize("act", ["silu", "relu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("shape", [(200, 96, 160), (2100, 70, 2600)])
def test_closed_gates_beside_ordinary_rows(cuda, act, shape):
    """Rows with a gate of -2^16 and an up projection of up to 2^16: their h, dgate and dup are
    zero, and the other rows of the block keep their bits."""
    x, wg, wu, wd, dy = exact_projections(cuda, *shape, 1.0, 8)
    for row in (5, 140, shape[0] - 1):
        x[row, 0], x[row, 1] = -2.0 ** 16, 2.0 ** 16
    y, saved = mf.gated_ffn(x, wg, wu, wd, act, save=True)
    for s in (saved, None):
        got = mf.gated_ffn_backward(dy, x, wg, wu, wd, act, saved=s)
        check_backward_scales(got, x, wg, wu, wd, dy, act)
    assert mf.device_status() == 0


@pytest.mark.parametrize("act,center", [("silu", -20.0), ("gelu", -6.0)])
def test_overflow_beside_saturated_gates(cuda, act, center):
    """A row whose up projection overflows says nothing about its block's scale: the other rows' dx
    keep their bits."""
    x, wg, wu, wd, dy = exact_projections(cuda, 200, 96, 160, center, 10)
    wu[1] = wu[1].abs() + 1.5                    # times 3e38: every entry of the row overflows
    other = x.clone()
    other[140, 1] = 3e38
    for keep in (True, False):
        saved = mf.gated_ffn(other, wg, wu, wd, act, save=True)[1] if keep else None
        dx = mf.gated_ffn_backward(dy, other, wg, wu, wd, act, saved=saved)[0]
        assert not torch.isfinite(dx[140]).all()
        dx[140] = 0
        zero = dy.clone()
        zero[140] = 0
        check_backward_scales((dx,), x, wg, wu, wd, zero, act)
    assert mf.device_status() == 0


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gradients_of_very_different_size(cuda, act):
    """Rows whose gradients lie 2^-12 to 2^-36 below their neighbours': a block of grad shares one
    scale, so an entry is off by 2^-39 of the block's largest at most, and dx's rows by what follows
    from that."""
    x, wg, wu, wd, dy = exact_projections(cuda, 300, 96, 260, 0.5, 9)
    dy *= torch.pow(2.0, -12.0 * (torch.arange(300, device=cuda) % 4))[:, None]
    edh = 2.0 ** -39 * float(dy.abs().max()) * wd.double().abs().sum(1)[None, :]
    got = mf.gated_ffn_backward(dy, x, wg, wu, wd, act)
    check_backward_scales(got, x, wg, wu, wd, dy, act, edh=edh)
    assert mf.device_status() == 0


@pytest.mark.parametrize("rows", [1, 40, 300])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu"])
def test_a_gate_that_is_not_a_number(cuda, act, rows):
    """One NaN in w_gate: what depends on that feature's gate is NaN, its gradient through the
    activation's derivative too, and nothing else."""
    x, wg, wu, wd, dy = inputs(cuda, rows, 130, 190)
    wg[3, 77] = float("nan")
    assert torch.isnan(mf.gated_ffn(x, wg, wu, wd, act)).all()
    for keep in (True, False):
        saved = mf.gated_ffn(x, wg, wu, wd, act, save=True)[1] if keep else None
        dx, dwg, dwu, dwd = mf.gated_ffn_backward(dy, x, wg, wu, wd, act, saved=saved)
        assert torch.isnan(dx).all()
        rest = [i for i in range(190) if i != 77]
        for t in (dwg, dwu, dwd.t()):
            assert torch.isnan(t[:, 77]).all() and torch.isfinite(t[:, rest]).all()
    assert mf.device_status() == 0
