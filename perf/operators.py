"""The operators of a decoder that is tuned on preferences or rewards: rotary positions of every layout, the
norm of queries and keys with that rotation, a preference loss over pairs of sequences and a clipped policy
loss over sampled tokens, each forward and backward.

``listed()`` gives calls that trainers make, ``draw(rng)`` others of the same ranges.  ``prepare`` makes what a
program holds before the call, ``run`` is one training pass (outputs and gradients): with ``own`` through
``pfeife_b200.ops``, else by elementary torch operations in 32 bits (64 where a sum, a logarithm or a
difference of near values needs them).  ``work`` counts the bytes and operations that no implementation can do
without, ``exact`` gives the same values from the definitions in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def listed():
    return [
        # rotary positions of the smallest configured decoder: launches and host time count, not bytes
        {"name": "rope_tiny", "op": "rope", "batch": 2, "seq": 32, "heads": 4, "dim": 16, "rotary": 16,
         "interleaved": False, "shared_positions": False, "scaling": 1.0, "dtype": "bf16"},
        # keys of one long sequence, pairs side by side, tables stretched to eight times their context
        {"name": "rope_long", "op": "rope", "batch": 1, "seq": 32768, "heads": 8, "dim": 128, "rotary": 128,
         "interleaved": True, "shared_positions": True, "scaling": 8.0, "dtype": "bf16"},
        # a quarter of each head rotates, several documents of odd lengths in a row
        {"name": "rope_quarter", "op": "rope", "batch": 3, "seq": 1027, "heads": 16, "dim": 96, "rotary": 24,
         "interleaved": False, "shared_positions": False, "scaling": 1.0, "dtype": "fp16"},
        # normed queries and keys of the smallest configured decoder, on its fused projection
        {"name": "qk_tiny", "op": "qk_packed", "batch": 2, "seq": 32, "heads": 4, "kv_heads": 4, "dim": 16,
         "rotary": 16, "interleaved": False, "shared_positions": True, "scaling": 1.0, "dtype": "bf16"},
        # one decoder layer of 4096 channels over 2048 tokens, on its fused projection
        {"name": "qk_layer", "op": "qk_packed", "batch": 1, "seq": 2048, "heads": 32, "kv_heads": 32, "dim": 128,
         "rotary": 128, "interleaved": False, "shared_positions": True, "scaling": 1.0, "dtype": "bf16"},
        # four query heads to a key head, slices of a projection, half of each head rotates
        {"name": "qk_shared", "op": "qk_heads", "batch": 2, "seq": 4096, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 64, "interleaved": True, "shared_positions": False, "scaling": 4.0, "dtype": "bf16"},
        # full precision and a head width that is no power of two
        {"name": "qk_fp32", "op": "qk_heads", "batch": 5, "seq": 301, "heads": 6, "kv_heads": 2, "dim": 72,
         "rotary": 72, "interleaved": False, "shared_positions": True, "scaling": 1.0, "dtype": "fp32"},
        # one pair of short sequences over the smallest configured vocabulary
        {"name": "preference_tiny", "op": "preference", "sequences": 2, "seq": 32, "classes": 256, "counted": 0.6,
         "smoothing": 0.0, "scale": 1.0, "dtype": "bf16"},
        # four pairs of 1024 tokens over 32000 words, the prompts and the padding not counted: the largest case
        {"name": "preference_pairs", "op": "preference", "sequences": 8, "seq": 1024, "classes": 32000,
         "counted": 0.5, "smoothing": 0.1, "scale": 1.0, "dtype": "bf16"},
        # eight samples of one prompt with an advantage each, held near a reference
        {"name": "policy_group", "op": "policy", "sequences": 8, "seq": 512, "classes": 32000, "counted": 0.7,
         "kl": 0.04, "per_token": False, "temperature": 1.0, "scale": 1.0, "dtype": "bf16"},
        # rows of an odd length in fp16 under a loss scale, an advantage for each token
        {"name": "policy_odd", "op": "policy", "sequences": 3, "seq": 333, "classes": 32003, "counted": 0.8,
         "kl": 0.1, "per_token": True, "temperature": 0.7, "scale": 1024.0, "dtype": "fp16"},
        # a few tokens in full precision, without a reference
        {"name": "policy_few", "op": "policy", "sequences": 1, "seq": 16, "classes": 32000, "counted": 1.0,
         "kl": 0.0, "per_token": True, "temperature": 1.0, "scale": 1.0, "dtype": "fp32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "qk_packed", "qk_heads", "preference", "policy"])
    c = {"op": op, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if op in ("rope", "qk_packed", "qk_heads"):
        dim = rng.choice([16, 32, 64, 64, 72, 80, 96, 128, 128, 128, 192, 256, 2 * rng.randint(5, 128)])
        rotary = rng.choice([dim, dim, dim, dim // 4 * 2, max(2, dim // 8 * 2)])
        kv = rng.choice([1, 2, 3, 4, 8])
        heads = kv * rng.choice([1, 2, 4, 6])
        if op == "rope":
            heads = rng.randint(1, 32)
        elif op == "qk_packed":
            heads = kv = rng.randint(2, 32)
        tokens = _log(rng, 17, min(65536, ((20 if c["dtype"] == "fp32" else 40) << 20) // ((heads + kv) * dim)))
        batch = rng.choice([1, 1, 2, 3, 5])
        c.update(batch=batch, seq=max(1, tokens // batch), heads=heads, dim=dim, rotary=rotary,
                 interleaved=rng.random() < 0.4, shared_positions=rng.random() < 0.5,
                 scaling=rng.choice([1.0, 1.0, 4.0, 8.0]))
        if op != "rope":
            c["kv_heads"] = kv
        return c
    classes = rng.choice([256, 32000, 32000, _log(rng, 500, 65000)])
    rows = _log(rng, 8, min(8192, (180 << 20) // (classes * (2 if c["dtype"] == "fp32" else 1))))
    sequences = 2 * rng.randint(1, 4) if op == "preference" else rng.randint(1, 8)
    c.update(sequences=sequences, seq=max(4, rows // sequences), classes=classes,
             counted=round(rng.uniform(0.3, 1.0), 2), scale=1024.0 if c["dtype"] == "fp16" else 1.0)
    if op == "preference":
        c.update(smoothing=rng.choice([0.0, 0.0, 0.1]))
    else:
        c.update(kl=rng.choice([0.0, 0.04, 0.1]), per_token=rng.random() < 0.5,
                 temperature=rng.choice([1.0, 1.0, 0.7]))
    return c


# ------------------------------------------------------------------------------ inputs
BETA, CLIP_LOW, CLIP_HIGH = 0.1, 0.2, 0.28


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", dtype=dtype, generator=g)


def _tables(rows, rotary, scaling):
    """Cosines and sines of `rows` positions.  A scaled table stretches the slow frequencies and leaves those that
    turn often within 2048 positions (a ramp between 1 and 32 turns), its values grown by 0.1 ln(scaling) + 1."""
    inv = 10000.0 ** -(torch.arange(0, rotary, 2, device="cuda", dtype=torch.float64) / rotary)
    if scaling != 1.0:
        turns = 2048 * inv / (2 * math.pi)
        kept = ((turns - 1) / 31).clamp(0, 1)
        inv = inv * (kept + (1 - kept) / scaling)
    angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * inv
    grown = 0.1 * math.log(scaling) + 1 if scaling != 1.0 else 1.0
    return (angle.cos() * grown).float(), (angle.sin() * grown).float()


def _positions(g, c):
    """Documents of random lengths in a row, each counting from 0: [seq] for all sequences, or [batch, seq]."""
    B, S = c["batch"], c["seq"]
    n = 1 if c["shared_positions"] else B
    starts = torch.rand(n, S, device="cuda", generator=g) < 4.0 / S
    starts[:, 0] = True
    at = torch.arange(S, device="cuda").expand(n, S)
    pos = at - torch.where(starts, at, torch.zeros_like(at)).cummax(1).values
    return pos[0].contiguous() if c["shared_positions"] else pos


def _spans(c):
    """(first, end) of the counted tokens of each sequence: a prompt before them, padding behind.  The same for every
    seed up to their order, so that the work of a case is known without its data."""
    rng = random.Random(c["seq"] * 131 + c["sequences"])
    n, spans = c["seq"], []
    while len(spans) < c["sequences"]:
        if c["op"] == "preference" and len(spans) % 2:       # the other answer to the same prompt
            first = spans[-1][0]
        else:
            first = int((1 - c["counted"]) * n * rng.uniform(0.5, 1.0))
        end = min(n, max(first + 1, first + int(c["counted"] * n * rng.uniform(0.8, 1.1))))
        spans.append((first, end))
    return spans


def _prepare_heads(c, seed):
    g, dtype = _gen(seed), DTYPES[c["dtype"]]
    B, S, H, D = c["batch"], c["seq"], c["heads"], c["dim"]
    s = {"case": c, "positions": _positions(g, c)}
    s["cos"], s["sin"] = _tables(S, c["rotary"], c["scaling"])
    if c["op"] == "rope":
        wide = _randn(g, B, S, H + 2, D, dtype=dtype)             # the heads of a projection that holds more
        s["x"] = wide[:, :, 1:H + 1].detach().requires_grad_()
        s["dy"] = _randn(g, B, S, H, D, dtype=dtype)
        return s
    K = c["kv_heads"]
    s["wq"] = (1 + 0.2 * _randn(g, D)).requires_grad_()
    s["wk"] = (1 + 0.2 * _randn(g, D)).requires_grad_()
    if c["op"] == "qk_packed":
        s["qkv"] = _randn(g, B, S, 3, H, D, dtype=dtype).requires_grad_()
        s["dy"] = _randn(g, B, S, 3, H, D, dtype=dtype)
    else:
        wide = _randn(g, B, S, H + 2 * K, D, dtype=dtype)
        s["q"] = wide[:, :, :H].detach().requires_grad_()
        s["k"] = wide[:, :, H:H + K].detach().requires_grad_()
        s["dq"] = _randn(g, B, S, H, D, dtype=dtype)
        s["dk"] = _randn(g, B, S, K, D, dtype=dtype)
    return s


def _log_prob(rows, tokens, temperature):
    """log softmax(rows / temperature)[tokens] in 64 bits, a sequence at a time"""
    out = []
    for r, t in zip(rows, tokens):
        z = r.double() / temperature
        out.append(z.gather(1, t[:, None])[:, 0] - z.logsumexp(-1))
    return torch.stack(out)


def _prepare_loss(c, seed):
    g, dtype = _gen(seed), DTYPES[c["dtype"]]
    N, T, V = c["sequences"], c["seq"], c["classes"]
    temperature = c.get("temperature", 1.0)
    logits = torch.empty(N, T, V, device="cuda", dtype=dtype)
    tokens = torch.empty(N, T, device="cuda", dtype=torch.int64)
    for n in range(N):                       # tokens drawn from the model, as answers are
        logits[n] = _randn(g, T, V) * 2.5
        noise = torch.rand(T, V, device="cuda", generator=g).clamp_(min=1e-20).log_().neg_().log_()
        tokens[n] = (logits[n].float() / temperature - noise).argmax(-1)
    logp = _log_prob(logits, tokens, temperature)
    spans = _spans(c)
    order = list(range(N // 2)) if c["op"] == "preference" else list(range(N))
    random.Random(seed).shuffle(order)
    if c["op"] == "preference":              # the chosen answers, then the rejected ones
        spans = [spans[2 * p] for p in order] + [spans[2 * p + 1] for p in order]
    else:
        spans = [spans[n] for n in order]
    at = torch.arange(T, device="cuda")
    first, end = (torch.tensor([x[i] for x in spans], device="cuda")[:, None] for i in (0, 1))
    counted = (at >= first) & (at < end)
    s = {"case": c, "logits": logits.requires_grad_(), "labels": tokens.masked_fill(~counted, -100),
         "grad": torch.tensor(c["scale"], device="cuda")}
    if c["op"] == "preference":
        s["ref"] = ((logp * counted).sum(1) + 5.0 * _randn(g, N)).float()
        return s
    # tokens were sampled by a policy some steps older; none lies on a border of the clipping, where the last bit
    # of a 32-bit ratio would decide on which side it is
    old = (logp + 0.15 * _randn(g, N, T)).float()
    ratio = (logp - old.double()).exp()
    near = ((ratio - (1 - CLIP_LOW)).abs() < 1e-3) | ((ratio - (1 + CLIP_HIGH)).abs() < 1e-3)
    s["old"] = torch.where(near, logp.float(), old)
    s["advantages"] = _randn(g, N, T) if c["per_token"] else _randn(g, N, 1)
    s["ref"] = (logp + 0.1 * _randn(g, N, T)).float() if c["kl"] else None
    return s


def prepare(case, seed):
    return (_prepare_loss if case["op"] in ("preference", "policy") else _prepare_heads)(case, seed)


# ------------------------------------------------------------------------------ one pass
def _rotated(x, cos, sin, positions, interleaved):
    """x [B, S, H, D] in 32 bits"""
    c, s = cos[positions].unsqueeze(-2), sin[positions].unsqueeze(-2)
    half = cos.shape[1]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([turned, rest], -1)


def _normed(x, weight):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight


def _plain_logps(logits, labels, temperature):
    """log softmax(logits / temperature) at the labels, 0 where there is none"""
    counted = (labels >= 0) & (labels < logits.shape[-1])
    z = logits.float()
    if temperature != 1.0:
        z = z / temperature
    z = z - z.detach().amax(-1, keepdim=True)
    total = z.exp().sum(-1)
    picked = z.gather(-1, labels.clamp(min=0).unsqueeze(-1)).squeeze(-1)
    return torch.where(counted, picked.double() - total.double().log(), 0.0), counted


def _plain_preference(logits, labels, ref, smoothing):
    logp = _plain_logps(logits, labels, 1.0)[0].sum(1)
    rewards = BETA * (logp - ref.double())
    chosen, rejected = rewards.chunk(2)
    margin = chosen - rejected
    loss = (1 - smoothing) * torch.log1p(torch.exp(-margin)) + smoothing * torch.log1p(torch.exp(margin))
    return loss.mean().float(), rewards.detach().float()


def _plain_policy(logits, actions, old, advantages, ref, kl_coef, temperature):
    logp, counted = _plain_logps(logits, actions, temperature)
    ratio = torch.exp(logp - old.double())
    free = ratio * advantages
    held = ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * advantages
    term = -torch.minimum(free, held)
    n = counted.sum().clamp(min=1)
    kl = torch.zeros((), device=logits.device)
    if ref is not None:
        d = ref.double() - logp
        each = d.exp() - d - 1
        term = term + kl_coef * each
        kl = (each.detach() * counted).sum() / n
    loss = (term * counted).sum() / n
    clipped = ((free > held) & counted).sum() / n
    return loss.float(), logp.detach().float(), kl.float(), clipped.float()


def run(state):
    c = state["case"]
    if own:
        from pfeife_b200 import ops
        if c["op"] in ("rope", "qk_packed", "qk_heads"):
            where = {"positions": state["positions"], "interleaved": c["interleaved"]}
        if c["op"] == "rope":
            y = ops.rope(state["x"], state["cos"], state["sin"], **where)
        elif c["op"] == "qk_packed":
            y = ops.qk_norm_rope_qkv(state["qkv"], state["wq"], state["wk"], state["cos"], state["sin"], EPS, **where)
        elif c["op"] == "qk_heads":
            q, k = ops.qk_norm_rope(state["q"], state["k"], state["wq"], state["wk"], state["cos"], state["sin"], EPS,
                                    **where)
        elif c["op"] == "preference":
            out = ops.preference_loss(state["logits"], state["labels"], state["ref"], beta=BETA,
                                      label_smoothing=c["smoothing"])
        else:
            out = ops.policy_loss(state["logits"], state["labels"], state["old"], state["advantages"],
                                  ref_logps=state["ref"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=c["kl"],
                                  temperature=c["temperature"])
    else:
        turn = lambda x: _rotated(x, state["cos"], state["sin"], state["positions"], c["interleaved"])  # noqa: E731
        if c["op"] == "rope":
            y = turn(state["x"].float()).to(state["x"].dtype)
        elif c["op"] == "qk_packed":
            x = state["qkv"].float()
            y = torch.stack([turn(_normed(x[:, :, 0], state["wq"])), turn(_normed(x[:, :, 1], state["wk"])),
                             x[:, :, 2]], 2).to(state["qkv"].dtype)
        elif c["op"] == "qk_heads":
            q = turn(_normed(state["q"].float(), state["wq"])).to(state["q"].dtype)
            k = turn(_normed(state["k"].float(), state["wk"])).to(state["k"].dtype)
        elif c["op"] == "preference":
            out = _plain_preference(state["logits"], state["labels"], state["ref"], c["smoothing"])
        else:
            out = _plain_policy(state["logits"], state["labels"], state["old"], state["advantages"], state["ref"],
                                c["kl"], c["temperature"])
    if c["op"] == "rope":
        return [y.detach(), *torch.autograd.grad(y, state["x"], state["dy"])]
    if c["op"] == "qk_packed":
        return [y.detach(), *torch.autograd.grad(y, [state["qkv"], state["wq"], state["wk"]], state["dy"])]
    if c["op"] == "qk_heads":
        grads = torch.autograd.grad([q, k], [state["q"], state["k"], state["wq"], state["wk"]],
                                    [state["dq"], state["dk"]])
        return [q.detach(), k.detach(), *grads]
    grads = torch.autograd.grad(out[0], state["logits"], state["grad"])
    return [out[0].detach(), *out[1:], *grads]


def work(case):
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    if c["op"] in ("rope", "qk_packed", "qk_heads"):
        heads = {"rope": c["heads"], "qk_packed": 3 * c["heads"]}.get(c["op"], c["heads"] + c.get("kv_heads", 0))
        n = c["batch"] * c["seq"] * heads * c["dim"]
        small = c["seq"] * c["rotary"] * 4 + c["seq"] * (1 if c["shared_positions"] else c["batch"]) * 8
        # read: the values and the gradient that arrives; written: the result and the gradient that leaves
        return {"bytes": 4 * n * size + small, "flops": n * (6 if c["op"] == "rope" else 20)}
    counted = sum(end - first for first, end in _spans(c))
    rows, V = c["sequences"] * c["seq"], c["classes"]
    # read: the logits of the rows that count, labels and the values beside them; written: the whole gradient
    return {"bytes": (counted + rows) * V * size + rows * (8 if c["op"] == "preference" else 24),
            "flops": counted * V * 9}


# ------------------------------------------------------------------------------ the same in 64 bits
def _turn64(x, cos, sin, positions, interleaved, sign):
    """Pairs as complex numbers times the tables' (conjugated for sign -1)"""
    half = cos.shape[1]
    turn = torch.complex(cos.double(), sign * sin.double())[positions]
    turn = turn[:, :, None] if turn.dim() == 3 else turn[None, :, None]
    out = x.clone()
    if interleaved:
        z = torch.complex(x[..., 0:2 * half:2], x[..., 1:2 * half:2]) * turn
        out[..., 0:2 * half:2], out[..., 1:2 * half:2] = z.real, z.imag
    else:
        z = torch.complex(x[..., :half], x[..., half:2 * half]) * turn
        out[..., :half], out[..., half:2 * half] = z.real, z.imag
    return out


def _heads64(x, w, dy, where):
    """-> (output, gradient, weight gradient) of one normed and rotated tensor"""
    D = x.shape[-1]
    r = 1 / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS)
    y = _turn64(x * r * w, *where, 1)
    g = _turn64(dy, *where, -1)
    gw = g * w
    dx = r * gw - x * r ** 3 * (gw * x).sum(-1, keepdim=True) / D
    return y, dx, (g * x * r).sum((0, 1, 2))


def exact(case, seed):
    c, s = case, prepare(case, seed)
    with torch.no_grad():
        if c["op"] in ("rope", "qk_packed", "qk_heads"):
            where = (s["cos"], s["sin"], s["positions"], c["interleaved"])
            if c["op"] == "rope":
                return [_turn64(s["x"].double(), *where, 1), _turn64(s["dy"].double(), *where, -1)]
            wq, wk = s["wq"].double(), s["wk"].double()
            if c["op"] == "qk_packed":
                x, dy = s["qkv"].double(), s["dy"].double()
                q, dq, dwq = _heads64(x[:, :, 0], wq, dy[:, :, 0], where)
                k, dk, dwk = _heads64(x[:, :, 1], wk, dy[:, :, 1], where)
                return [torch.stack([q, k, x[:, :, 2]], 2), torch.stack([dq, dk, dy[:, :, 2]], 2), dwq, dwk]
            q, dq, dwq = _heads64(s["q"].double(), wq, s["dq"].double(), where)
            k, dk, dwk = _heads64(s["k"].double(), wk, s["dk"].double(), where)
            return [q, k, dq, dk, dwq, dwk]
        logits, labels, scale = s["logits"], s["labels"], c["scale"]
        N, T, V = logits.shape
        temperature = c.get("temperature", 1.0)
        counted = labels != -100
        tokens = labels.clamp(min=0)
        logp = _log_prob(logits, tokens, temperature) * counted
        if c["op"] == "preference":
            rewards = BETA * (logp.sum(1) - s["ref"].double())
            P, e = N // 2, c["smoothing"]
            margin = rewards[:P] - rewards[P:]
            logsig = torch.nn.functional.logsigmoid
            loss = (-(1 - e) * logsig(margin) - e * logsig(-margin)).sum() / P
            slope = -BETA / P * ((1 - e) / (1 + margin.exp()) - e / (1 + (-margin).exp()))
            coef = torch.cat([slope, -slope])[:, None].expand(N, T)
            first = [loss, rewards]
        else:
            n = max(1, int(counted.sum()))
            A = s["advantages"].double().expand(N, T)
            r = (logp - s["old"].double()).exp()
            # which way the clipping holds a ratio depends on the sign of its advantage
            held = ((A > 0) & (r > 1 + CLIP_HIGH)) | ((A < 0) & (r < 1 - CLIP_LOW))
            most = torch.where(A > 0, 1 + CLIP_HIGH, 1 - CLIP_LOW).double()
            term = -torch.where(held, most, r) * A
            coef = torch.where(held, 0.0, -A * r)
            kl = torch.zeros((), device="cuda", dtype=torch.float64)
            if s["ref"] is not None:
                d = s["ref"].double() - logp
                each = torch.expm1(d) - d
                term, coef = term + c["kl"] * each, coef - c["kl"] * torch.expm1(d)
                kl = (each * counted).sum() / n
            coef = coef / (n * temperature)
            first = [(term * counted).sum() / n, logp, kl, (held & counted).sum().double() / n]
        grad = torch.zeros(N, T, V, device="cuda", dtype=torch.float64)
        for i in range(N):
            p = torch.softmax(logits[i].double() / temperature, -1).neg_()
            p.scatter_add_(1, tokens[i][:, None], torch.ones(T, 1, device="cuda", dtype=torch.float64))
            grad[i] = p * (coef[i] * counted[i] * scale)[:, None]
        return [*first, grad]
