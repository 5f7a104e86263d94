"""Cases and plain forms of the language-model operators: the gated feed-forward block with its
backward pass, the orthogonalised update (Newton-Schulz) and the embedding with its gradient.

`run` computes one pass over what `prepare` made: in the plain form from elementary torch
operations in fp32, or, with `own` set, through this package's public calls. `exact` gives the
same outputs from the definitions in 64 bits.
"""
import math

import torch

own = False

# The quintic Newton-Schulz coefficients that the update's orthogonalisation commonly uses: they
# raise small singular values by 3.4445 a step and keep the large ones within about [0.7, 1.2].
NS = (3.4445, -4.7750, 2.0315)
NS_EPS = 1e-7


def listed():
    return [
        # one token through a block of the two-layer MLP's sizes: a decoding step, latency counts
        {"name": "ffn_token", "op": "ffn", "rows": 1, "d": 1024, "f": 4096, "act": "silu"},
        # eight sequences decoding together through a large block: a stream of the weights
        {"name": "ffn_tokens8", "op": "ffn", "rows": 8, "d": 4096, "f": 11008, "act": "silu"},
        # a prompt of 2048 tokens, exact GELU
        {"name": "ffn_prefill", "op": "ffn", "rows": 2048, "d": 2048, "f": 5632, "act": "gelu"},
        # one training step of the block at the two-layer MLP's sizes (batch 4096)
        {"name": "ffn_train", "op": "ffn_train", "rows": 4096, "d": 1024, "f": 4096,
         "act": "silu"},
        # the same on ragged sizes: a packed batch, a width that no tile divides, odd strides
        {"name": "ffn_train_ragged", "op": "ffn_train", "rows": 1531, "d": 1003, "f": 2731,
         "act": "gelu_tanh"},
        # a large training step
        {"name": "ffn_train_large", "op": "ffn_train", "rows": 8192, "d": 4096, "f": 11008,
         "act": "silu"},
        # the updates of many small matrices at once (per-head projections)
        {"name": "orth_heads", "op": "orth", "batch": 48, "m": 64, "n": 128},
        # the update of the MLP's first weight matrix
        {"name": "orth_mlp", "op": "orth", "batch": 1, "m": 1024, "n": 4096},
        # a tall matrix of odd sizes
        {"name": "orth_tall", "op": "orth", "batch": 1, "m": 2731, "n": 1003},
        # the update of a large block's projection
        {"name": "orth_large", "op": "orth", "batch": 1, "m": 4096, "n": 11008},
        # a decoding step's lookup: few tokens, a scaled table of an odd width
        {"name": "embed_few", "op": "embed", "tokens": 64, "vocab": 32000, "d": 1003},
        # a training step's lookup and the table's gradient, words as frequent as in text
        {"name": "embed_train", "op": "embed_train", "tokens": 16384, "vocab": 32000, "d": 2048},
    ]


def _between(rng, low, high):
    """A whole number in [low, high], spread over its logarithm, most often an odd one."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(["ffn", "ffn", "ffn_train", "orth", "orth", "embed", "embed_train"])
    act = rng.choice(["silu", "gelu", "gelu_tanh", "relu"])
    if op == "ffn":
        rows = _between(rng, 1, 16) if rng.random() < 0.5 else _between(rng, 17, 8192)
        return {"op": op, "rows": rows, "d": _between(rng, 64, 4096), "f": _between(rng, 96, 11008),
                "act": act}
    if op == "ffn_train":
        return {"op": op, "rows": _between(rng, 1, 8192), "d": _between(rng, 64, 4096),
                "f": _between(rng, 96, 11008), "act": act}
    if op == "orth":
        if rng.random() < 0.4:
            return {"op": op, "batch": _between(rng, 2, 64), "m": _between(rng, 8, 512),
                    "n": _between(rng, 8, 512)}
        return {"op": op, "batch": 1, "m": _between(rng, 32, 4096), "n": _between(rng, 32, 8192)}
    if op == "embed":
        return {"op": op, "tokens": _between(rng, 1, 16384), "vocab": _between(rng, 100, 65536),
                "d": _between(rng, 16, 2048)}
    return {"op": op, "tokens": _between(rng, 1, 65536), "vocab": _between(rng, 100, 65536),
            "d": _between(rng, 16, 1024)}


def _normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * std


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op = case["op"]
    if op in ("ffn", "ffn_train"):
        m, d, f = case["rows"], case["d"], case["f"]
        # normalised activations, Xavier-scaled weights, a mean loss's small gradient
        s = {"op": op, "act": case["act"], "x": _normal(g, m, d),
             "w_gate": _normal(g, d, f, std=math.sqrt(2.0 / (d + f))),
             "w_up": _normal(g, d, f, std=math.sqrt(2.0 / (d + f))),
             "w_down": _normal(g, f, d, std=math.sqrt(2.0 / (d + f)))}
        if op == "ffn_train":
            s["grad"] = _normal(g, m, d, std=1.0 / math.sqrt(m * d))
        return s
    if op == "orth":
        b, m, n = case["batch"], case["m"], case["n"]
        # a momentum buffer: a few strong directions over a noise floor
        r = min(8, m, n)
        u = _normal(g, b, m, n, std=1e-3)
        u += _normal(g, b, m, r, std=2e-3) @ _normal(g, b, r, n)
        return {"op": op, "update": u if b > 1 else u[0]}
    n, v, d = case["tokens"], case["vocab"], case["d"]
    # word frequencies fall as 1 / rank; the ranks are dealt to ids that lie all over the table
    rank = torch.exp(torch.rand(n, generator=g, device="cuda", dtype=torch.float64) *
                     math.log(v + 1)).long().clamp_(1, v) - 1
    ids = torch.randperm(v, generator=g, device="cuda")[rank]
    s = {"op": op, "ids": ids, "table": _normal(g, v, d, std=0.02), "scale": math.sqrt(d)}
    if op == "embed_train":
        s["grad"] = _normal(g, n, d, std=1.0 / math.sqrt(n * d))
    return s


def _act(v, kind):
    """act(v) and its derivative."""
    if kind == "relu":
        on = (v > 0).to(v.dtype)
        return v * on, on
    if kind == "silu":
        s = 1 / (1 + torch.exp(-v))
        return v * s, s * (1 + v * (1 - s))
    if kind == "gelu":
        phi = 0.5 * torch.special.erfc(v * -math.sqrt(0.5))
        return v * phi, phi + v * torch.exp(-0.5 * v * v) * (1 / math.sqrt(2 * math.pi))
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (v + 0.044715 * v * v * v))
    return (0.5 * v * (1 + t),
            0.5 * (1 + t) + 0.5 * v * (1 - t * t) * c * (1 + 3 * 0.044715 * v * v))


def _own(s):
    import mensurflow_b200 as mf

    if s["op"] == "ffn":
        return mf.gated_ffn(s["x"], s["w_gate"], s["w_up"], s["w_down"], s["act"])
    if s["op"] == "ffn_train":
        y, saved = mf.gated_ffn(s["x"], s["w_gate"], s["w_up"], s["w_down"], s["act"], save=True)
        return (y,) + mf.gated_ffn_backward(s["grad"], s["x"], s["w_gate"], s["w_up"],
                                            s["w_down"], s["act"], saved=saved)
    if s["op"] == "orth":
        return mf.orthogonalize(s["update"], 5, NS, NS_EPS)
    y = mf.embedding(s["table"], s["ids"], s["scale"])
    if s["op"] == "embed":
        return y
    return y, mf.embedding_grad(s["grad"], s["ids"], s["table"].shape[0], s["scale"])


def run(s):
    if own:
        return _own(s)
    if s["op"] in ("ffn", "ffn_train"):
        x = s["x"]
        gate, up = x @ s["w_gate"], x @ s["w_up"]
        a, slope = _act(gate, s["act"])
        h = a * up
        y = h @ s["w_down"]
        if s["op"] == "ffn":
            return y
        dy = s["grad"]
        dh = dy @ s["w_down"].t()
        dg, du = dh * up * slope, dh * a
        return (y, dg @ s["w_gate"].t() + du @ s["w_up"].t(), x.t() @ dg, x.t() @ du, h.t() @ dy)
    if s["op"] == "orth":
        u = s["update"]
        x = u.transpose(-2, -1) if u.shape[-2] > u.shape[-1] else u
        x = x / (torch.sqrt(torch.sum(x * x, (-2, -1), keepdim=True)) + NS_EPS)
        a, b, c = NS
        for _ in range(5):
            p = x @ x.transpose(-2, -1)
            x = a * x + (b * p + c * (p @ p)) @ x
        return x.transpose(-2, -1) if u.shape[-2] > u.shape[-1] else x
    y = s["table"][s["ids"]] * s["scale"]
    if s["op"] == "embed":
        return y
    return y, torch.zeros_like(s["table"]).index_add_(0, s["ids"], s["grad"] * s["scale"])


def work(case):
    op = case["op"]
    if op in ("ffn", "ffn_train"):
        m, d, f = case["rows"], case["d"], case["f"]
        if op == "ffn":
            return {"bytes": 4 * (2 * m * d + 3 * d * f), "flops": 6 * m * d * f}
        return {"bytes": 4 * (4 * m * d + 6 * d * f), "flops": 18 * m * d * f}
    if op == "orth":
        b, m, n = case["batch"], min(case["m"], case["n"]), max(case["m"], case["n"])
        # X X^T and its square are symmetric: half of each is enough
        return {"bytes": 8 * b * m * n, "flops": 5 * b * (3 * m * m * n + m * m * m)}
    n, v, d = case["tokens"], case["vocab"], case["d"]
    if op == "embed":
        return {"bytes": 8 * n + 8 * n * d, "flops": n * d}
    return {"bytes": 16 * n + 12 * n * d + 4 * v * d, "flops": 3 * n * d}


def _exact_act(v, kind):
    if kind == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v)), torch.where(v > 0, 1.0, 0.0).to(v.dtype)
    if kind == "silu":
        s = torch.sigmoid(v)
        return v * s, s + v * s * torch.sigmoid(-v)
    if kind == "gelu":
        cdf = torch.special.ndtr(v)
        return v * cdf, cdf + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    # 0.5 (1 + tanh z) = sigmoid(2 z)
    z = math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)
    s = torch.sigmoid(2 * z)
    return v * s, s + 2 * v * s * (1 - s) * math.sqrt(2 / math.pi) * (1 + 0.134145 * v ** 2)


def exact(case, seed):
    s = prepare(case, seed)
    wide = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v
            for k, v in s.items()}
    op = case["op"]
    if op in ("ffn", "ffn_train"):
        x, wg, wu, wd = wide["x"], wide["w_gate"], wide["w_up"], wide["w_down"]
        gate = torch.einsum("md,df->mf", x, wg)
        up = torch.einsum("md,df->mf", x, wu)
        a, slope = _exact_act(gate, case["act"])
        y = torch.einsum("mf,fd->md", a * up, wd)
        if op == "ffn":
            return y
        dh = torch.einsum("md,fd->mf", wide["grad"], wd)
        d_wd = torch.einsum("mf,md->fd", a * up, wide["grad"])
        d_gate, d_up = dh * slope * up, dh * a
        dx = torch.einsum("mf,df->md", d_gate, wg) + torch.einsum("mf,df->md", d_up, wu)
        return (y, dx, torch.einsum("md,mf->df", x, d_gate), torch.einsum("md,mf->df", x, d_up),
                d_wd)
    if op == "orth":
        x = wide["update"]
        x = x / (torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True) + NS_EPS)
        tall = x.shape[-2] > x.shape[-1]
        a, b, c = NS
        for _ in range(5):
            # x (a + b x^T x + c (x^T x)^2), on whichever side the Gram matrix is the smaller
            p = torch.matmul(x.mT, x) if tall else torch.matmul(x, x.mT)
            q = b * p + c * torch.matmul(p, p)
            x = a * x + (torch.matmul(x, q) if tall else torch.matmul(q, x))
        return x
    y = wide["table"].index_select(0, s["ids"]) * s["scale"]
    if op == "embed":
        return y
    d_table = torch.zeros_like(wide["table"])
    d_table.index_put_((s["ids"],), wide["grad"] * s["scale"], accumulate=True)
    return y, d_table
