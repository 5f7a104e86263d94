"""The orthogonalised update against the Newton-Schulz iteration in 64 bits."""
import numpy as np
import pytest
import torch

import mensurflow_b200 as mf

pytestmark = pytest.mark.gpu

NS = (3.4445, -4.7750, 2.0315)


def want(u, steps=5, coefficients=NS, eps=1e-7):
    x = u.double()
    x = x / (torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True) + eps)
    a, b, c = coefficients
    tall = x.shape[-2] > x.shape[-1]
    for _ in range(steps):
        g = x.mT @ x if tall else x @ x.mT
        q = b * g + c * (g @ g)
        x = a * x + (x @ q if tall else q @ x)
    return x


def close(got, ref, steps=5):
    """Relative to each matrix's norm. One product is off by at most 4e-6 of |A||B|, for these
    matrices about 1e-6 of its norm; three products a step, and a step multiplies an error by at
    most 3.45 relative to a vanishing singular value (which grows alike) and by at most 2.3
    relative to one near 1: five steps stay below 3e-6 (1 + 2.3 + .. + 2.3^4), about 1e-4 in the
    worst case. An error in a formula shows at 1e-2 or more."""
    err = torch.linalg.vector_norm(got.double() - ref, dim=(-2, -1))
    size = torch.linalg.vector_norm(ref, dim=(-2, -1))
    assert bool((err <= 1e-4 * size + 1e-30).all()), float((err / size).max())


SIZES = [(1, 1), (1, 7), (9, 1), (2, 3), (64, 64), (64, 128), (127, 129), (128, 128), (130, 64),
         (128, 1024), (1024, 100), (1000, 128), (65, 640), (128, 1025), (1030, 90),
         (256, 200), (257, 513), (700, 300), (384, 1500), (1003, 771)]


@pytest.mark.parametrize("shape", SIZES)
def test_sizes(cuda, shape):
    g = torch.Generator(device="cuda").manual_seed(shape[0] * 31 + shape[1])
    u = torch.randn(*shape, generator=g, device=cuda) * 1e-3
    got = mf.orthogonalize(u)
    assert got.shape == u.shape
    close(got, want(u))
    assert mf.device_status() == 0


@pytest.mark.parametrize("shape", [(3, 64, 128), (300, 16, 40), (2, 3, 128, 257), (5, 200, 130),
                                   (40, 600, 100)])
def test_batches(cuda, shape):
    g = torch.Generator(device="cuda").manual_seed(sum(shape))
    u = torch.randn(*shape, generator=g, device=cuda)
    u = u * torch.logspace(-6, 6, shape[0], device=cuda).reshape(-1, *[1] * (len(shape) - 1))
    got = mf.orthogonalize(u)
    assert got.shape == u.shape
    close(got, want(u))
    alone = torch.stack([mf.orthogonalize(m) for m in u])     # a batch is its matrices
    close(alone, want(u))
    assert mf.device_status() == 0


def test_views_steps_and_coefficients(cuda):
    g = torch.Generator(device="cuda").manual_seed(3)
    u = torch.randn(3, 150, 70, generator=g, device=cuda)
    big = torch.randn(3, 160, 90, generator=g, device=cuda)
    big[:, 7:157, 5:75] = u
    for view in (big[:, 7:157, 5:75], u.mT.contiguous().mT, u.transpose(0, 1).contiguous().transpose(0, 1),
                 torch.repeat_interleave(u, 2, 2)[..., ::2]):
        assert torch.equal(view, u)
        close(mf.orthogonalize(view), want(u))
    for steps in (1, 2, 7):
        close(mf.orthogonalize(u, steps), want(u, steps))
    c = (1.5, -0.5, 0.0)                                   # the cubic iteration
    close(mf.orthogonalize(u, 12, c), want(u, 12, c))
    close(mf.orthogonalize(u[0].expand(4, 150, 70)), want(u[0].expand(4, 150, 70)))
    one = mf.orthogonalize(u[0].t())
    close(one, want(u[0].t()))
    large = torch.randn(520, 300, generator=g, device=cuda)
    for view in (large.t(), large.t().contiguous().t()):
        close(mf.orthogonalize(view), want(view))


def test_scales_zero_and_nonfinite(cuda):
    g = torch.Generator(device="cuda").manual_seed(4)
    for shape in ((60, 100), (200, 400)):
        u = torch.randn(*shape, generator=g, device=cuda)
        ref = want(u)
        for scale in (1e-3, 1e3, 1e25, 1e30):              # eps is negligible beside the norm
            close(mf.orthogonalize(u * scale), ref)
        close(mf.orthogonalize(u * 1e-25, eps=0.0), ref)
        assert (mf.orthogonalize(torch.zeros_like(u)) == 0).all()
        bad = torch.stack([u, u, u])
        bad[1, 3, 5] = float("nan")
        got = mf.orthogonalize(bad)
        assert torch.isnan(got[1]).all()
        close(got[::2], torch.stack([ref, ref]))
    assert mf.device_status() == 0


def test_empty(cuda):
    assert mf.orthogonalize(torch.empty(0, 5, device=cuda)).shape == (0, 5)
    assert mf.orthogonalize(torch.empty(0, 3, 5, device=cuda)).shape == (0, 3, 5)


def test_singular_values_gather_around_one(cuda):
    g = torch.Generator(device="cuda").manual_seed(9)
    u = torch.randn(256, 1000, generator=g, device=cuda)
    s = torch.linalg.svdvals(mf.orthogonalize(u).double())
    assert 0.6 < float(s.min()) and float(s.max()) < 1.3


@pytest.mark.parametrize("shape", [(2, 90, 120), (300, 700)])
def test_streams_and_graphs(cuda, shape):
    g = torch.Generator(device="cuda").manual_seed(1)
    u = torch.randn(*shape, generator=g, device=cuda)
    plain = mf.orthogonalize(u)
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got += [mf.orthogonalize(u) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(r, plain) for r in got)
    held = u.clone()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(mf.orthogonalize(held))
        graphs.append(graph)
    for _ in range(3):
        held.normal_(generator=g)
        expect = mf.orthogonalize(held)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, expect) for o in outs)
    assert mf.device_status() == 0


@pytest.mark.parametrize("shape", [(200, 5), (1000, 40), (600, 100), (5, 200), (90, 60)])
def test_what_ran_before_does_not_matter(cuda, shape):
    """The same bits whatever the kernels before left in shared memory."""
    u = torch.randn(32, *shape, device=cuda)
    other = torch.randn(148, 128, 1024, device=cuda)
    w = [torch.randn(*s, device=cuda) for s in ((512, 1024), (512, 1024), (1024, 512))]
    first = mf.orthogonalize(u)
    close(first, want(u))
    for x in (w[2] * 1e-30, torch.full_like(w[2], 1e15), torch.full_like(w[2], float("inf"))):
        mf.gated_ffn(x, *w)
        assert torch.equal(mf.orthogonalize(u), first)
    for x in (other * 1e30, other.mT):
        mf.orthogonalize(x)
        assert torch.equal(mf.orthogonalize(u), first)
    assert mf.device_status() == 0


@pytest.mark.parametrize("shape", [(60, 100), (200, 400), (400, 200), (3, 100, 300), (2, 300, 140)])
def test_norms_whose_reciprocal_leaves_fp32(cuda, shape):
    """With eps = 0 a power of two in front of the matrix changes nothing, bit for bit, from
    subnormal entries (norms below 2^-128) to the largest (norms above 2^128). Entries of ten bits
    keep all of them as subnormals. At 2^-149 the block scale ends at 2^126 and leaves up to 511
    2^-23 < 2^-14: exact, but subnormal in fp16, and a tensor product need not drop the same bits
    of its sums for operands without a leading one; there the iteration's tolerance holds."""
    g = torch.Generator(device="cuda").manual_seed(sum(shape))
    u = torch.randint(-511, 512, shape, generator=g, device=cuda).float()
    plain = mf.orthogonalize(u, eps=0.0)
    close(plain, want(u, eps=0.0))
    for power in (-149, -140, -120, 100, 118):
        scaled = torch.ldexp(u.double(), torch.tensor(power, device=cuda)).float()
        assert bool(torch.isfinite(scaled).all())
        got = mf.orthogonalize(scaled, eps=0.0)
        close(got, want(u, eps=0.0))
        assert power == -149 or torch.equal(got, plain), power
    assert mf.device_status() == 0


@pytest.mark.parametrize("shape", [(60, 100), (200, 400), (700, 300), (2, 1100, 1030)])
@pytest.mark.parametrize("c", [(1.5, 0.0, -0.5), (0.0, 1.5, -0.5), (1.5, -0.5, 0.0),
                               (1.25, 0.0, 0.0), (0.0, 0.0, 1.0), (0.0, 0.5, 0.0)])
def test_coefficients_of_zero(cuda, shape, c):
    g = torch.Generator(device="cuda").manual_seed(sum(shape))
    u = torch.randn(*shape, generator=g, device=cuda)
    for steps in (1, 3):
        close(mf.orthogonalize(u, steps, c), want(u, steps, c))
    assert mf.device_status() == 0


@pytest.mark.parametrize("shape", [(64, 128), (6, 100, 90), (128, 1000), (128, 1100), (200, 20000),
                                   (30000, 150), (256, 256), (1003, 771), (2, 500, 2000), (1024, 4096)])
def test_error_of_the_iteration(cuda, shape):
    """1e-5 of the norm, whatever the depth. An operand's two halves are off by 5e-8 of it rms. Of a
    chunk's 24 accumulations the eight of the high halves drop 3.4e-8 of the sum so far on average,
    1.4e-7 of the result; chunks are added in fp32. So a product is off by 2.1e-7 of its norm. In a
    step b g x has two such errors and c g g x four: (2 x 4.8 + 4 x 2.1) 2.1e-7 = 3.8e-6 where
    singular values are near 1, less before, and a step multiplies the errors of the steps before by
    at most 1.7 there: three steps' worth in the worst signs is 3.8e-6 (1 + 1.7 + ...), and a third
    of that as they come."""
    g = torch.Generator(device="cuda").manual_seed(sum(shape))
    u = torch.randn(*shape, generator=g, device=cuda)
    ref = want(u)
    err = torch.linalg.vector_norm(mf.orthogonalize(u).double() - ref, dim=(-2, -1))
    assert bool((err <= 1e-5 * torch.linalg.vector_norm(ref, dim=(-2, -1))).all())
    assert mf.device_status() == 0
