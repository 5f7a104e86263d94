"""The language-model operators together, as a training step uses them: embedding, two gated
blocks with residual connections, the loss's gradient back through both to the table, and the
weights moved along their orthogonalised gradients. Checked against the same step in 64 bits."""
import pytest
import torch

import mensurflow_b200 as mf

pytestmark = pytest.mark.gpu


def orthogonal64(u):
    x = u / (torch.linalg.matrix_norm(u) + 1e-7)
    tall = x.shape[0] > x.shape[1]
    for _ in range(5):
        g = x.mT @ x if tall else x @ x.mT
        q = -4.7750 * g + 2.0315 * (g @ g)
        x = 3.4445 * x + (x @ q if tall else q @ x)
    return x


def step64(table, blocks, ids, target, scale):
    t = table.double().requires_grad_()
    ws = [[w.double().requires_grad_() for w in b] for b in blocks]
    h = t[ids] * scale
    for wg, wu, wd in ws:
        h = h + (torch.nn.functional.silu(h @ wg) * (h @ wu)) @ wd
    loss = 0.5 * ((h - target.double()) ** 2).mean()
    loss.backward()
    return loss.detach(), t.grad, [[w.grad for w in b] for b in ws], h.detach()


def test_training_step(cuda):
    g = torch.Generator(device="cuda").manual_seed(11)
    n = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    rows, d, f, vocab = 190, 136, 300, 500
    table, scale = n(vocab, d) * 0.1, d ** 0.5
    blocks = [[n(d, f) / d ** 0.5, n(d, f) / d ** 0.5, n(f, d) / f ** 0.5] for _ in range(2)]
    ids = torch.randint(0, vocab, (2, rows // 2), generator=g, device=cuda)
    target = n(2, rows // 2, d)

    h = mf.embedding(table, ids, scale)
    inputs, saves = [], []
    for b in blocks:
        y, saved = mf.gated_ffn(h, *b, save=True)
        inputs.append(h)
        saves.append(saved)
        h = mf.add(h, y)
    grad = mf.scal(1.0 / h.numel(), mf.sub(h, target).reshape(-1)).view_as(h)
    grads = []
    for b, x, saved in zip(reversed(blocks), reversed(inputs), reversed(saves)):
        dx, *dw = mf.gated_ffn_backward(grad, x, *b, saved=saved)
        grads.append(dw)
        grad = mf.add(grad, dx)
    grads.reverse()
    d_table = mf.embedding_grad(grad, ids, vocab, scale)

    loss, want_table, want_blocks, want_h = step64(table, blocks, ids, target, scale)
    # two blocks and their backward pass: a product's 4e-6 of |A||B| (about 1e-6 of the result's
    # norm) through six products in a row with factors of order one
    rel = lambda a, b: float((a.double() - b).norm() / b.norm())  # noqa: E731
    assert rel(h, want_h) < 2e-5
    assert rel(d_table, want_table) < 5e-5
    for dw, want in zip(grads, want_blocks):
        for a, b in zip(dw, want):
            assert rel(a, b) < 5e-5
            # the update itself: the iteration's own error beside that of its input, which it
            # amplifies at most 3.4445^5 times in directions of vanishing size
            assert rel(mf.orthogonalize(a), orthogonal64(a.double())) < 1e-4
    stacked = mf.orthogonalize(torch.stack([grads[0][0], grads[1][0]]))
    for got, dw in zip(stacked, (grads[0][0], grads[1][0])):
        assert rel(got, orthogonal64(dw.double())) < 1e-4
    assert mf.device_status() == 0
