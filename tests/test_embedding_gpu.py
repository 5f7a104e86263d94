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


def test_shapes_views_and_padding(cuda):
    g = torch.Generator(device="cuda").manual_seed(2)
    table = torch.randn(50, 40, generator=g, device=cuda)
    ids = torch.randint(0, 50, (3, 7, 5), generator=g, device=cuda)
    grad = torch.randn(3, 7, 5, 40, generator=g, device=cuda)
    for t in (table, torch.randn(50, 60, device=cuda)[:, 3:43].copy_(table),
              table.t().contiguous().t()):
        assert torch.equal(mf.embedding(t, ids), table[ids])
    one = table[:1].expand(50, 40)
    assert torch.equal(mf.embedding(one, ids), one[ids])
    assert mf.embedding(table, ids.transpose(0, 2)).equal(table[ids.transpose(0, 2)])
    assert mf.embedding(table, torch.tensor(7, device=cuda)).shape == (40,)
    for view in (grad, torch.cat([grad, grad], -1)[..., :40],
                 grad.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)):
        close(mf.embedding_grad(view, ids, 50, -0.5), grad, ids, 50, -0.5)
    padded = mf.embedding_grad(grad, ids, 50, padding=3)
    close(padded, grad, ids, 50, 1.0, padding=3)
    assert (padded[3] == 0).all()
    close(mf.embedding_grad(grad[0, 0, :1].expand(9, 40), ids.reshape(-1)[:9], 50),
          grad[0, 0, :1].expand(9, 40), ids.reshape(-1)[:9], 50, 1.0)
    assert mf.device_status() == 0


def test_empty(cuda):
    table = torch.randn(5, 4, device=cuda)
    none = torch.empty(0, dtype=torch.int64, device=cuda)
    assert mf.embedding(table, none).shape == (0, 4)
    assert (mf.embedding_grad(torch.empty(0, 4, device=cuda), none, 5) == 0).all()
    assert mf.embedding_grad(torch.empty(0, 4, device=cuda), none, 0).shape == (0, 4)
    assert mf.embedding(torch.empty(5, 0, device=cuda), none.new_zeros(3)).shape == (3, 0)


def test_ids_outside_the_table(cuda):
    """Zeros for the lookup, no part in the gradient, a bit in the device's error word, and no
    effect on kernels that wait (the bit is kept apart from theirs)."""
    table = torch.randn(10, 36, device=cuda)
    ids = torch.tensor([0, 10, -1, 9, 2 ** 40, 3], device=cuda)
    good = torch.tensor([True, False, False, True, False, True], device=cuda)
    grad = torch.randn(6, 36, device=cuda)
    y = mf.embedding(table, ids)
    assert torch.equal(y[good], table[ids[good]]) and (y[~good] == 0).all()
    a = torch.randn(300, 64, device=cuda)
    assert torch.isfinite(mf.gemm(a, a, transpose_b=True)).all()
    assert mf.device_status() == 0x20
    close(mf.embedding_grad(grad, ids, 10), grad, ids, 10, 1.0)
    assert mf.device_status() == 0x20
    assert mf.device_status() == 0
    close(mf.embedding_grad(grad[:1], ids[:1], 10), grad[:1], ids[:1], 10, 1.0)
    assert mf.device_status() == 0


@pytest.mark.parametrize("n", [300, 70000])
def test_one_id_and_every_id(cuda, n):
    """All tokens of one id (the longest run there is), and each id once (runs of one)."""
    grad = torch.randn(n, 12, device=cuda)
    same = torch.full((n,), 4, device=cuda)
    close(mf.embedding_grad(grad, same, 9), grad, same, 9, 1.0)
    each = torch.randperm(n, device=cuda)
    assert torch.equal(mf.embedding_grad(grad, each, n)[each], grad)


def test_streams_and_graphs(cuda):
    g = torch.Generator(device="cuda").manual_seed(6)
    table = torch.randn(3000, 64, generator=g, device=cuda)
    ids = torch.randint(0, 3000, (5000,), generator=g, device=cuda)
    grad = torch.randn(5000, 64, generator=g, device=cuda)
    both = lambda: (mf.embedding(table, ids, 2.0), mf.embedding_grad(grad, ids, 3000, 2.0))  # noqa: E731
    plain = both()
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got += [both() for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in got for a, b in zip(r, plain))
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(both())
        graphs.append(graph)
    for _ in range(3):
        ids.random_(0, 3000, generator=g)
        grad.normal_(generator=g)
        expect = both()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for o in outs for a, b in zip(o, expect))
    assert mf.device_status() == 0


@pytest.mark.parametrize("tokens", [4, 70000])
def test_minus_one_is_outside_the_table(cuda, tokens):
    """Without a padding id -1 is an id like any other outside the table."""
    ids = torch.arange(tokens, device=cuda) % 10
    ids[1] = -1
    grad = torch.randn(tokens, 8, device=cuda)
    close(mf.embedding_grad(grad, ids, 10), grad, ids, 10, 1.0)
    assert mf.device_status() == 0x20
    close(mf.embedding_grad(grad, ids.int(), 10, padding=3), grad, ids, 10, 1.0, padding=3)
    assert mf.device_status() == 0x20
    assert mf.device_status() == 0


def test_a_table_without_rows(cuda):
    ids = torch.zeros(3, dtype=torch.int64, device=cuda)
    with pytest.raises(ValueError, match="no rows"):
        mf.embedding(torch.empty(0, 4, device=cuda), ids)
    with pytest.raises(ValueError, match="no rows"):
        mf.embedding_grad(torch.zeros(3, 4, device=cuda), ids, 0)


def test_offsets_past_32_bits(cuda):
    """A table of more than 2^31 entries, and its gradient."""
    if torch.cuda.mem_get_info()[0] < 40e9:
        pytest.skip("needs 40 GB")
    rows, d = 2 ** 16 + 9, 2 ** 15 + 4
    table = torch.empty(rows, d, device=cuda)
    table.normal_()
    ids = torch.tensor([rows - 1, 0, rows - 1, 2 ** 16], device=cuda)
    assert torch.equal(mf.embedding(table, ids), table[ids])
    grad = torch.randn(4, d, device=cuda)
    out = mf.embedding_grad(grad, ids, rows)
    assert torch.equal(out[2 ** 16], grad[3]) and torch.equal(out[0], grad[1])
    assert torch.equal(out[rows - 1], grad[0] + grad[2])
    out[ids] = 0.0
    assert not out.any()
    assert mf.device_status() == 0


@pytest.mark.parametrize("d", [1, 3, 4, 16, 17, 31, 33, 64, 100, 128, 129, 132, 256, 260, 511, 512, 515])
@pytest.mark.parametrize("n,rows", [(1, 4), (130, 40), (6000, 3), (40000, 30000)])
def test_narrow_rows(cuda, n, rows, d):
    """Rows that fill part of a warp or block: several tokens or windows beside each other, and one
    run longer than a window's block."""
    g = torch.Generator(device="cuda").manual_seed(n + rows + d)
    ids = (torch.rand(n, generator=g, device=cuda) ** 4 * rows).long().clamp_(max=rows - 1)
    ids[n // 3: n // 2] = rows // 2
    table = torch.randn(rows, d, generator=g, device=cuda)
    grad = torch.randn(n, d, generator=g, device=cuda)
    assert torch.equal(mf.embedding(table, ids, 0.3), table[ids] * 0.3)
    got = mf.embedding_grad(grad, ids, rows, 0.3)
    close(got, grad, ids, rows, 0.3)
    assert torch.equal(got, mf.embedding_grad(grad, ids, rows, 0.3))
    base = torch.full((rows, d + 3), -7.0, device=cuda)      # unaligned rows
    base[:, 1:d + 1] = table
    assert torch.equal(mf.embedding(base[:, 1:d + 1], ids, 0.3), table[ids] * 0.3)
    wide = torch.cat([grad, grad], -1)
    close(mf.embedding_grad(wide[:, d:], ids, rows, 0.3), grad, ids, rows, 0.3)
    ids[0] = rows
    y = mf.embedding(table, ids)
    assert not y[0].any() and torch.equal(y[1:], table[ids[1:]])
    assert mf.device_status() == 0x20
    assert mf.device_status() == 0
