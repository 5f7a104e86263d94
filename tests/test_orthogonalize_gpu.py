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
