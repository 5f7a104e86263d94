"""Argument checks of the language-model operators, without a GPU: the Python calls refuse what
they cannot take before any device work, and the C entry points return status codes."""
import ctypes

import pytest
import torch

import mensurflow_b200 as mf
from mensurflow_b200 import _lib

F = torch.float32


def weights(d=4, f=6):
    return torch.ones(d, f), torch.ones(d, f), torch.ones(f, d)


def test_gated_ffn_refusals():
    wg, wu, wd = weights()
    x = torch.ones(3, 4)
    with pytest.raises(NotImplementedError):      # no CPU path
        mf.gated_ffn(x, wg, wu, wd)
    with pytest.raises(NotImplementedError):      # fp32 only
        mf.gated_ffn(x.half(), wg.half(), wu.half(), wd.half())
    with pytest.raises(ValueError, match="dtypes differ"):
        mf.gated_ffn(x, wg.double(), wu, wd)
    with pytest.raises(ValueError, match="undefined"):
        mf.gated_ffn(None, wg, wu, wd)
    with pytest.raises(ValueError, match="w_down"):
        mf.gated_ffn(x, wg, wu, None)
    with pytest.raises(ValueError, match="w_up"):
        mf.gated_ffn(x, wg, wu[:, :5], wd)
    with pytest.raises(ValueError, match="w_down"):
        mf.gated_ffn(x, wg, wu, wd.t())
    with pytest.raises(ValueError, match="does not fit"):
        mf.gated_ffn(torch.ones(3, 5), wg, wu, wd)
    with pytest.raises(ValueError, match="at least 1-D"):
        mf.gated_ffn(torch.ones(()), wg, wu, wd)
    with pytest.raises(ValueError, match="2-D"):
        mf.gated_ffn(x, wg[None], wu, wd)
    with pytest.raises(ValueError, match="activation"):
        mf.gated_ffn(x, wg, wu, wd, "swish")
    with pytest.raises(ValueError):               # stored the other way round
        mf.gated_ffn(x, wg, wu, wd, transpose_w=True)


def test_gated_ffn_backward_refusals():
    wg, wu, wd = weights()
    x = torch.ones(3, 4)
    with pytest.raises(NotImplementedError):
        mf.gated_ffn_backward(x, x, wg, wu, wd)
    with pytest.raises(ValueError, match="activation"):
        mf.gated_ffn_backward(x, x, wg, wu, wd, "tanh")


def test_orthogonalize_refusals():
    u = torch.ones(3, 4)
    with pytest.raises(NotImplementedError):
        mf.orthogonalize(u)
    with pytest.raises(NotImplementedError):
        mf.orthogonalize(u.bfloat16())
    with pytest.raises(ValueError, match="at least 2-D"):
        mf.orthogonalize(torch.ones(3))
    for steps in (0, -1, 1.5, True):
        with pytest.raises(ValueError, match="steps"):
            mf.orthogonalize(u, steps)
    with pytest.raises(ValueError, match="coefficients"):
        mf.orthogonalize(u, 5, (1.0, 2.0))
    for eps in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            mf.orthogonalize(u, eps=eps)


def test_embedding_refusals():
    table, ids, grad = torch.ones(5, 4), torch.zeros(3, dtype=torch.int64), torch.ones(3, 4)
    with pytest.raises(NotImplementedError):
        mf.embedding(table, ids)
    with pytest.raises(NotImplementedError):
        mf.embedding_grad(grad, ids, 5)
    with pytest.raises(ValueError, match="int64 or int32"):
        mf.embedding(table, ids.float())
    with pytest.raises(ValueError, match="2-D"):
        mf.embedding(table[0], ids)
    with pytest.raises(ValueError, match="undefined"):
        mf.embedding(table, [0, 1])
    with pytest.raises(ValueError, match="does not fit"):
        mf.embedding_grad(grad, ids[:2], 5)
    for rows in (-1, 2.0, True):
        with pytest.raises(ValueError, match="rows"):
            mf.embedding_grad(grad, ids, rows)
    for padding in (-1, 5):
        with pytest.raises(ValueError, match="padding"):
            mf.embedding_grad(grad, ids, 5, padding=padding)


def test_c_entry_points_refuse_before_any_launch():
    so, bad, unsupported = _lib.lib(), _lib.MFK_ERR_INVALID_ARGUMENT, _lib.MFK_ERR_UNSUPPORTED
    d = _lib.GatedFfnDesc()
    p = ctypes.c_void_p(4096)
    call = lambda y=p, ldy=4, saved=None: so.mfk_gated_ffn_f32(ctypes.byref(d), y, ldy, saved, None)  # noqa: E731
    assert so.mfk_gated_ffn_f32(None, p, 4, None, None) == bad
    d.rows, d.d, d.f = -1, 4, 6
    assert call() == bad
    d.rows = 3
    assert call() == bad                                  # no inputs
    d.x = d.w_gate = d.w_up = d.w_down = 4096
    assert call(None) == bad                              # no output
    assert call(p, 3) == bad                              # ldy < d
    d.activation = 9
    assert call() == bad
    d.activation = 0
    assert call(p, 4, ctypes.c_void_p(4100)) == bad       # saved not on 16 bytes
    d.rows = 0
    assert call() == _lib.MFK_OK                          # nothing to do
    d.rows = 2 ** 31
    assert call() == unsupported
    assert so.mfk_gated_ffn_saved_floats(-1, 4) == -1
    assert so.mfk_gated_ffn_saved_floats(129, 1) == 2 * (2 * 128 * 128 + 4 * 128)
    o = _lib.GatedFfnGrads()
    back = lambda: so.mfk_gated_ffn_backward_f32(ctypes.byref(d), ctypes.byref(o), None, None)  # noqa: E731
    d.rows = 3
    assert so.mfk_gated_ffn_backward_f32(ctypes.byref(d), None, None, None) == bad
    assert back() == bad                                  # no grad
    o.grad = 4096
    assert back() == _lib.MFK_OK                          # nothing wanted
    o.dw_gate = 4096
    assert back() == bad                                  # one weight gradient of three
    o.dw_up = o.dw_down = 4096
    o.dw_rs, o.dw_cs, o.dw_down_rs, o.dw_down_cs = 12, 2, 4, 1
    assert back() == unsupported                          # no unit stride
    o.dw_gate = o.dw_up = o.dw_down = None
    o.dx, o.ld_dx = 4096, 3
    assert back() == bad
    orth = lambda b, m, n, ld=9, steps=5, eps=0.0, u=p: so.mfk_orthogonalize_f32(  # noqa: E731
        u, b, m, n, n, m * n, p, ld, m * n, steps, 1.0, 1.0, 1.0, eps, None)
    assert orth(-1, 3, 4) == bad
    assert orth(1, 3, 4, steps=0) == bad
    assert orth(1, 3, 4, eps=-1.0) == bad
    assert orth(1, 3, 4, eps=float("nan")) == bad
    assert orth(1, 3, 4, ld=3) == bad
    assert orth(1, 3, 4, u=None) == bad
    assert orth(0, 3, 4) == _lib.MFK_OK
    assert orth(1, 2 ** 31, 4) == unsupported
    emb = lambda rows, dd, n, size=8, ld=4, t=p: so.mfk_embedding_f32(  # noqa: E731
        t, rows, dd, ld, p, size, n, 1.0, p, 4, None)
    assert emb(-1, 4, 3) == bad
    assert emb(5, 4, 3, size=2) == bad
    assert emb(0, 4, 3) == bad
    assert emb(5, 4, 3, ld=-1) == bad
    assert emb(5, 4, 3, t=None) == bad
    assert emb(5, 4, 0) == _lib.MFK_OK
    assert emb(2 ** 31, 4, 3) == unsupported
    grad = lambda n, dd, rows, size=8, ldg=4, out=p, ld=4: so.mfk_embedding_grad_f32(  # noqa: E731
        p, n, dd, ldg, p, size, rows, 1.0, -1, out, ld, None)
    assert grad(3, 4, -1) == bad
    assert grad(3, 4, 5, size=3) == bad
    assert grad(3, 4, 5, ldg=-1) == bad
    assert grad(3, 4, 5, out=None) == bad
    assert grad(3, 4, 5, ld=3) == bad
    assert grad(3, 4, 0) == _lib.MFK_OK
    assert grad(2 ** 31, 4, 5) == unsupported


def test_descriptor_layouts():
    assert ctypes.sizeof(_lib.GatedFfnDesc) == 4 * 24 + 24 + 8
    assert _lib.GatedFfnDesc.rows.offset == 96
    assert ctypes.sizeof(_lib.GatedFfnGrads) == 24 + 16 + 16 + 16 + 24


@pytest.mark.parametrize("rows", [1, 5, 16, 17, 300])
def test_rows_of_x_that_are_not_contiguous_are_refused(rows):
    """However many rows: the few-rows form has no strided reads either."""
    so, p = _lib.lib(), ctypes.c_void_p(4096)
    for rs, cs in ((8, 2), (1, rows), (0, 0)):
        if cs == 1:
            continue
        d = _lib.GatedFfnDesc(4096, rs, cs, 4096, 6, 1, 4096, 6, 1, 4096, 4, 1, rows, 4, 6, 0, 0)
        assert so.mfk_gated_ffn_f32(ctypes.byref(d), p, 4, None, None) == _lib.MFK_ERR_UNSUPPORTED
        assert so.mfk_gated_ffn_f32(ctypes.byref(d), p, 4, p, None) == _lib.MFK_ERR_UNSUPPORTED


@pytest.mark.parametrize("steps", [2 ** 31, 2 ** 32, 2 ** 32 + 5])
def test_steps_beyond_32_bits_are_refused(steps):
    """The entry point's count has 32 bits: 2^32 + 5 would be 5."""
    with pytest.raises(ValueError, match="steps"):
        mf.orthogonalize(torch.ones(3, 4), steps)


@pytest.mark.parametrize("padding", [1.5, 2.0, "1", True, [1]])
def test_padding_that_is_no_whole_number_is_refused(padding):
    with pytest.raises(ValueError, match="padding"):
        mf.embedding_grad(torch.ones(3, 4), torch.zeros(3, dtype=torch.int64), 5, padding=padding)
