"""What a decoder's training step does outside of attention, as operators that keep less between forward and
backward: embedded tokens with a scale and a gradient summed in the order of the tokens, the gated feed-forward
block, and the output head with its cross entropy, of which no logits are kept.  Each forward and backward.

``listed()`` gives calls that trainers make, ``draw(rng)`` others of the same ranges.  ``prepare`` makes what a
program holds before the call, ``run`` is one training pass (outputs and gradients): with ``own`` through
``pfeife_b200.ops``, else by elementary torch operations in 32 bits.  ``work`` counts the bytes and operations that
no implementation can do without, ``exact`` gives the same values from the definitions in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # token embedding of the smallest configured decoder: launches and host time count, not bytes
        {"name": "embed_tiny", "op": "embedding", "tokens": 64, "words": 256, "dim": 64, "padding": 0.0,
         "scale": 8.0, "table": "bf16", "dtype": "bf16"},
        # four sequences of 2048 tokens over the 32000 words of a decoder, fp32 weights and 16-bit activations
        {"name": "embed_master", "op": "embedding", "tokens": 8192, "words": 32000, "dim": 4096, "padding": 0.0,
         "scale": 64.0, "table": "fp32", "dtype": "bf16"},
        # a large vocabulary in 16 bits and long batches of which a third is one padding word
        {"name": "embed_padded", "op": "embedding", "tokens": 65536, "words": 128000, "dim": 2048, "padding": 0.33,
         "scale": 1.0, "table": "fp16", "dtype": "fp16"},
        # odd sizes in full precision
        {"name": "embed_odd", "op": "embedding", "tokens": 1027, "words": 30011, "dim": 777, "padding": 0.1,
         "scale": 27.87, "table": "fp32", "dtype": "fp32"},
        # feed-forward block of the smallest configured decoder, two sequences of 32 tokens
        {"name": "mlp_tiny", "op": "gated_mlp", "rows": 64, "dim": 64, "hidden": 128, "activation": "silu",
         "biases": False, "residual": True, "dtype": "bf16"},
        # one decoder layer of 4096 channels over 2048 tokens
        {"name": "mlp_layer", "op": "gated_mlp", "rows": 2048, "dim": 4096, "hidden": 11008, "activation": "silu",
         "biases": False, "residual": False, "dtype": "bf16"},
        # one transformer layer over the 64 x 64 latents of four images: GELU and biases
        {"name": "mlp_latents", "op": "gated_mlp", "rows": 16384, "dim": 640, "hidden": 2560, "activation": "gelu",
         "biases": True, "residual": False, "dtype": "fp16"},
        # a few tokens through the large layer: its weights are most of what moves
        {"name": "mlp_few", "op": "gated_mlp", "rows": 13, "dim": 4096, "hidden": 11008, "activation": "silu",
         "biases": False, "residual": True, "dtype": "bf16"},
        # head and loss of the smallest configured decoder
        {"name": "head_tiny", "op": "head", "sequences": 2, "seq": 32, "dim": 64, "words": 256, "counted": 1.0,
         "scale": 1.0, "dtype": "bf16"},
        # next-token loss over one sequence of 2048 tokens and 32000 words
        {"name": "head_layer", "op": "head", "sequences": 1, "seq": 2048, "dim": 4096, "words": 32000,
         "counted": 1.0, "scale": 1.0, "dtype": "bf16"},
        # answers of eight conversations under a loss scale: the prompts, half of the tokens, do not count
        {"name": "head_answers", "op": "head", "sequences": 8, "seq": 1024, "dim": 4096, "words": 32000,
         "counted": 0.5, "scale": 1024.0, "dtype": "fp16"},
        # rows of an odd number over a large vocabulary of an odd number of words: the largest case
        {"name": "head_wide", "op": "head", "sequences": 3, "seq": 1365, "dim": 2048, "words": 128011,
         "counted": 1.0, "scale": 1.0, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embedding", "gated_mlp", "gated_mlp", "head", "head"])
    kind = rng.choice(["bf16", "bf16", "fp16"])
    if op == "embedding":
        table = rng.choice(["fp32", kind])
        c = {"op": op, "tokens": _log(rng, 7, 65536), "words": _log(rng, 200, 200000),
             "dim": rng.choice([64, 768, 2048, 4096, _log(rng, 16, 4096)]), "padding": rng.choice([0.0, 0.0, 0.33]),
             "scale": rng.choice([1.0, 8.0, 27.87, 64.0]), "table": table,
             "dtype": rng.choice([kind, "fp32"]) if table == "fp32" else kind}
    elif op == "gated_mlp":
        dim = rng.choice([64, 640, 1280, 4096, 8 * _log(rng, 8, 640)])
        hidden = rng.choice([2 * dim, 4 * dim, 8 * _log(rng, 8, 1400), 8 * max(1, dim // 3)])
        c = {"op": op, "rows": _log(rng, 1, 16384), "dim": dim, "hidden": hidden,
             "activation": rng.choice(["silu", "silu", "gelu", "gelu_tanh"]), "biases": rng.random() < 0.4,
             "residual": rng.random() < 0.5, "dtype": kind}
        most, low = 1.6e12, "rows"
    else:
        sequences = rng.randint(1, 8)
        c = {"op": op, "sequences": sequences, "seq": max(8, _log(rng, 8, 16384) // sequences),
             "dim": rng.choice([64, 768, 2048, 4096, 8 * _log(rng, 8, 512)]),
             "words": rng.choice([256, 32000, _log(rng, 250, 128000)]), "counted": rng.choice([1.0, 1.0, 0.5, 0.2]),
             "scale": 1024.0 if kind == "fp16" else 1.0, "dtype": kind}
        most, low = 6.0e12, "seq"
    # no drawn case costs more than the largest listed one
    while work(c)["bytes"] > 1.05e9:
        wide = max((k for k in ("words", "tokens", "hidden") if k in c), key=lambda k: c[k])
        c[wide] = c[wide] // 32 * 24
    while op != "embedding" and work(c)["flops"] > most and c[low] > 12:
        c[low] = c[low] * 3 // 4
    return c


# ------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)


def _words(g, count, words):
    """Words by how often they are said: word i with a probability of log((i + 2) / (i + 1)) / log(words + 1)"""
    u = torch.rand(count, device="cuda", generator=g, dtype=torch.float64)
    return (u * math.log(words + 1)).exp().long().sub_(1).clamp_(0, words - 1)


def _distinct(tokens, words):
    """How many of the words a batch has, on average"""
    i = torch.arange(words, dtype=torch.float64)
    p = torch.log((i + 2) / (i + 1)) / math.log(words + 1)
    return int((1 - (1 - p) ** tokens).sum())


def prepare(case, seed):
    c, g, dtype = case, _gen(seed), DTYPES[case["dtype"]]
    s = {"case": c}
    if c["op"] == "embedding":
        N, V, D = c["tokens"], c["words"], c["dim"]
        ids = _words(g, N, V)
        if c["padding"]:
            ids[N - int(c["padding"] * N):] = 0
        s["ids"] = ids
        s["table"] = _randn(g, V, D, dtype=DTYPES[c["table"]], std=0.02).requires_grad_()
        s["dy"] = _randn(g, N, D, dtype=dtype)
    elif c["op"] == "gated_mlp":
        N, D, H = c["rows"], c["dim"], c["hidden"]
        s["x"] = _randn(g, N, D, dtype=dtype).requires_grad_()
        s["w1"] = _randn(g, 2 * H, D, dtype=dtype, std=1.5 * D ** -0.5).requires_grad_()
        s["w2"] = _randn(g, D, H, dtype=dtype, std=H ** -0.5).requires_grad_()
        s["b1"] = _randn(g, 2 * H, dtype=dtype, std=0.2).requires_grad_() if c["biases"] else None
        s["b2"] = _randn(g, D, dtype=dtype, std=0.2).requires_grad_() if c["biases"] else None
        s["residual"] = _randn(g, N, D, dtype=dtype) if c["residual"] else None
        s["dy"] = _randn(g, N, D, dtype=dtype)
    else:
        B, T, D, V = c["sequences"], c["seq"], c["dim"], c["words"]
        s["x"] = _randn(g, B, T, D, dtype=dtype).requires_grad_()
        s["weight"] = _randn(g, V, D, dtype=dtype, std=2.0 * D ** -0.5).requires_grad_()
        target = _words(g, B * T, V).view(B, T)
        target[:, :_prompt(c)] = -100
        target[:, -1] = -100                 # nothing follows the last token
        s["target"] = target
        s["grad"] = torch.tensor(c["scale"], device="cuda")
    return s


def _prompt(c):
    return int((1 - c["counted"]) * c["seq"])


# ------------------------------------------------------------------------------ one pass
def _act(z, kind):
    if kind == "silu":
        return z / (1 + torch.exp(-z))
    if kind == "gelu":
        return z * (1 + torch.erf(z * math.sqrt(0.5))) / 2
    return z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))) / 2


def _plain_mlp(s, kind):
    x, dtype = s["x"].float(), s["x"].dtype
    gu = x @ s["w1"].float().t()
    if s["b1"] is not None:
        gu = gu + s["b1"].float()
    H = gu.shape[-1] // 2
    y = (_act(gu[:, :H], kind) * gu[:, H:]) @ s["w2"].float().t()
    if s["b2"] is not None:
        y = y + s["b2"].float()
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(dtype)


def _plain_head(x, weight, target):
    x, target = x.flatten(0, 1).float(), target.flatten()
    counted = target >= 0
    z = x @ weight.float().t()
    z = z - z.detach().amax(-1, keepdim=True)
    picked = z.gather(-1, target.clamp(min=0).unsqueeze(-1)).squeeze(-1)
    loss = torch.where(counted, z.exp().sum(-1).log() - picked, 0.0)
    return (loss.double().sum() / counted.sum().clamp(min=1)).float()


def run(state):
    s, c = state, state["case"]
    if c["op"] == "embedding":
        if own:
            from pfeife_b200 import ops
            y = ops.scaled_embedding(s["ids"], s["table"], c["scale"], out_dtype=s["dy"].dtype)
        else:
            y = (s["table"].float()[s["ids"]] * c["scale"]).to(s["dy"].dtype)
        return [y.detach(), *torch.autograd.grad(y, s["table"], s["dy"])]
    if c["op"] == "gated_mlp":
        if own:
            from pfeife_b200 import ops
            y = ops.gated_mlp(s["x"], s["w1"], s["b1"], s["w2"], s["b2"], activation=c["activation"],
                              residual=s["residual"])
        else:
            y = _plain_mlp(s, c["activation"])
        leaves = [s[k] for k in ("x", "w1", "w2", "b1", "b2") if s[k] is not None]
        return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"])]
    if own:
        from pfeife_b200 import ops
        loss = ops.linear_cross_entropy(s["x"], s["weight"], s["target"])
    else:
        loss = _plain_head(s["x"], s["weight"], s["target"])
    return [loss.detach(), *torch.autograd.grad(loss, [s["x"], s["weight"]], s["grad"])]


def work(case):
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "embedding":
        wide = 4 if c["table"] == "fp32" else 2
        N, V, D = c["tokens"], c["words"], c["dim"]
        # read: the rows of the table that the tokens name and the gradient that arrives; written: the embedded
        # tokens and the whole gradient of the table
        rows = _distinct(N - int(c["padding"] * N), V)
        return {"bytes": 16 * N + rows * D * wide + 2 * N * D * size + V * D * wide, "flops": 2 * N * D}
    if c["op"] == "gated_mlp":
        N, D, H = c["rows"], c["dim"], c["hidden"]
        # read: x, the gradient that arrives, a residual and the weights; written: y, dx and the weights' gradients
        n = (4 + c["residual"]) * N * D + 6 * D * H + (2 * (2 * H + D) if c["biases"] else 0)
        return {"bytes": n * size, "flops": 18 * N * D * H}
    N, D, V = c["sequences"] * c["seq"], c["dim"], c["words"]
    counted = c["sequences"] * max(0, c["seq"] - 1 - _prompt(c))
    # read: the rows that count, the weights and the labels; written: the gradients of all rows and of the weights
    return {"bytes": ((counted + N) * D + 2 * V * D) * size + 8 * N, "flops": 6 * counted * D * V}


# ------------------------------------------------------------------------------ the same in 64 bits
def _slope64(z, kind):
    """(activation, its derivative)"""
    if kind == "silu":
        p = torch.sigmoid(z)
        return z * p, p + z * p * (1 - p)
    if kind == "gelu":
        phi = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    a = math.sqrt(2 / math.pi)
    p = torch.sigmoid(2 * a * (z + 0.044715 * z ** 3))
    return z * p, p + z * p * (1 - p) * 2 * a * (1 + 3 * 0.044715 * z * z)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    with torch.no_grad():
        if c["op"] == "embedding":
            table, ids, dy = s["table"], s["ids"], s["dy"]
            grad = torch.zeros(table.shape, dtype=torch.float64, device="cuda")
            grad.index_add_(0, ids, dy.double())
            return [table.double().index_select(0, ids).mul_(c["scale"]), grad.mul_(c["scale"])]
        if c["op"] == "gated_mlp":
            x, w1, w2, dy = (s[k].double() for k in ("x", "w1", "w2", "dy"))
            H = w2.shape[1]
            gate, up = x @ w1[:H].t(), x @ w1[H:].t()
            if s["b1"] is not None:
                gate, up = gate + s["b1"][:H].double(), up + s["b1"][H:].double()
            a, slope = _slope64(gate, c["activation"])
            h = a * up
            y = h @ w2.t()
            if s["b2"] is not None:
                y = y + s["b2"].double()
            if s["residual"] is not None:
                y = y + s["residual"].double()
            dh = dy @ w2
            dz = torch.cat([dh * up * slope, dh * a], 1)
            out = [y, dz @ w1, dz.t() @ x, dy.t() @ h]
            if s["b1"] is not None:
                out += [dz.sum(0), dy.sum(0)]
            return out
        x, w, target = s["x"].flatten(0, 1), s["weight"].double(), s["target"].flatten()
        rows = (target >= 0).nonzero().squeeze(1)
        dx = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
        dw = torch.zeros_like(w)
        loss, n = 0.0, max(1, len(rows))
        for part in rows.split(512):
            xr, t = x[part].double(), target[part]
            p = torch.log_softmax(xr @ w.t(), -1)
            at = torch.arange(len(part), device="cuda")
            loss = loss - p[at, t].sum()
            p = p.exp_()
            p[at, t] -= 1
            p *= c["scale"] / n
            dx[part] = p @ w
            dw += p.t() @ xr
        return [torch.as_tensor(loss / n, device="cuda"), dx.view(s["x"].shape), dw]
