"""The embedding lookup (one rounding: bit for bit) and its table's gradient (fp32 sums against
64 bits: adding c values one after another, in windows or not, is off by at most c 2^-24 of the
sum of their magnitudes; the scale adds one rounding)."""
import pytest
import torch

import mensurflow_b200 as mf
from mensurflow_b200 import _lib

pytestmark = pytest.mark.gpu


def close(got, grad, ids, rows, scale, padding=None):
    d = grad.shape[-1]
    flat, g = ids.reshape(-1).long(), grad.reshape(-1, d).double()
    keep = (flat >= 0) & (flat < rows)
    if padding is not None:
        keep &= flat != padding
    flat, g = flat[keep], g[keep]
    z = torch.zeros(rows, d, dtype=torch.float64, device=grad.device)
    ref = z.index_add(0, flat, g) * scale
    size = z.index_add(0, flat, g.abs()) * abs(scale)
    count = torch.bincount(flat, minlength=rows).double()[:, None]
    bound = (count + 2) * 2.0 ** -24 * size
    assert got.shape == (rows, d)
    assert bool(((got.double() - ref).abs() <= bound).all())
    assert bool((got[count[:, 0] == 0] == 0).all())


SIZES = [(1, 1, 1), (3, 5, 7), (64, 32, 129), (100, 1000, 64), (513, 300, 1003), (2049, 70000, 33),
         (5000, 17, 260), (4096, 40, 1024), (9000, 1, 516), (20000, 257, 96),
         (16384, 300, 8), (30000, 70000, 36), (65536, 1000, 5), (65537, 1000, 5), (100000, 17000000, 1)]


@pytest.mark.parametrize("n,rows,d", SIZES)
@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_lookup_and_gradient(cuda, n, rows, d, dtype):
    g = torch.Generator(device="cuda").manual_seed(n + rows + d)
    ids = (torch.rand(n, generator=g, device=cuda) ** 3 * rows).long().clamp_(max=rows - 1)
    ids = ids.to(dtype)
    table = torch.randn(rows, d, generator=g, device=cuda)
    grad = torch.randn(n, d, generator=g, device=cuda)
    assert torch.equal(mf.embedding(table, ids, 1.7), table[ids.long()] * 1.7)
    got = mf.embedding_grad(grad, ids, rows, 1.7)
    close(got, grad, ids, rows, 1.7)
    assert torch.equal(got, mf.embedding_grad(grad, ids, rows, 1.7))   # the same bits again
    assert mf.device_status() == 0
