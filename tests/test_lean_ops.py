"""Scaled embeddings, the gated feed-forward block and the head with its loss against their formulas in 64 bits.

Bounds.  u is half a step of the result's type, 2^-24 half a step of fp32.  The tensor cores' sums of n products are off by
a whole step (2^-23) of the sum of magnitudes for each of the n + 16 additions at most (they may cut bits off instead
of rounding).  An activation is off by 1e-6 (1 + |z|), and changes by no more than 1.2 times its argument's error, its
derivative by no more than 0.8 times.  Errors go through each formula by its partial derivatives, in magnitudes."""
import math
import threading

import pytest
import torch

from pfeife_b200 import ops
from pfeife_b200.ops import _lib
from test_kernel_calls import calls  # noqa: F401

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}
E = 2.0 ** -24


def within(got, want, error):
    """|got - want| <= error in the values, and half a step of got's type"""
    bound = error + U[got.dtype] * (want.abs() + error) + TINY[got.dtype]
    off = (got.double() - want).abs()
    assert got.shape == want.shape and torch.isfinite(got).all()
    assert (off <= bound).all(), float((off / bound).max())


def sums(n):
    return (n + 16) * 2.0 ** -23


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(*shape, device, dtype, seed, std=1.0):
    return (torch.randn(*shape, generator=gen(seed)) * std).to(device=device, dtype=dtype)


# ------------------------------------------------------------------------------ embedding
def tokens(kind, N, V, seed=0):
    ids = torch.randint(0, V, (N,), generator=gen(seed))
    if kind == "one":
        ids[:] = V - 1
    elif kind == "padded":
        ids[N // 3:] = 0
        ids[: N // 5] = -1
    elif kind == "outside":
        ids[::3] = V
        ids[1::7] = -(1 << 40)
        ids[2::11] = 1 << 40
    elif kind == "few":
        ids %= 3
    return ids


EMBED = [(1, 1, 1, "any"), (5, 7, 16, "any"), (64, 256, 64, "any"), (33, 9, 13, "few"), (1027, 3001, 77, "padded"),
         (2049, 512, 1032, "any"), (300, 4, 8, "one"), (4096, 40, 24, "few"), (4097, 33000, 8, "outside"),
         (9001, 300, 136, "padded"), (70001, 262145, 8, "any"), (20000, 70000, 5, "one")]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,wide", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32),
                                        (torch.bfloat16, torch.float32), (torch.float32, torch.float32),
                                        (torch.float16, torch.float16)], ids=str)
@pytest.mark.parametrize("N,V,D,kind", EMBED, ids=str)
def test_scaled_embedding(N, V, D, kind, dtype, wide, device):
    scale = 1.0 if N == 64 else 5.37
    ids = tokens(kind, N, V).to(device)
    table = normal(V, D, device=device, dtype=wide, seed=1).requires_grad_()
    dy = normal(N, D, device=device, dtype=dtype, seed=2)
    y = ops.scaled_embedding(ids, table, scale, out_dtype=dtype)
    (g,) = torch.autograd.grad(y, table, dy)
    assert y.dtype == dtype and g.dtype == wide
    inside = (ids >= 0) & (ids < V)
    at = ids.masked_fill(~inside, 0)
    want = table.detach().double()[at].masked_fill(~inside[:, None], 0.0) * scale
    within(y.detach(), want, E * want.abs())
    total, mag = (torch.zeros(V, D, dtype=torch.float64, device=device) for _ in range(2))
    total.index_add_(0, ids[inside], dy[inside].double())
    mag.index_add_(0, ids[inside], dy[inside].double().abs())
    times = torch.zeros(V, dtype=torch.float64, device=device).index_add_(0, ids[inside], torch.ones(
        int(inside.sum()), dtype=torch.float64, device=device))
    within(g, total * scale, (times[:, None] + 2) * E * mag * scale)
    assert not g[times == 0].any()


@pytest.mark.gpu
@pytest.mark.parametrize("N", [130, 4096, 50000])
def test_sums_of_tokens_go_in_their_order(N):
    """In the order of the tokens, in windows: the same bits every time, and exact sums where all partial sums are."""
    ids = tokens("padded", N, 50).cuda()
    table = torch.zeros(50, 32, device="cuda", requires_grad=True)
    dy = torch.randint(-8, 9, (N, 32), generator=gen(3)).cuda().to(torch.bfloat16)
    g = [torch.autograd.grad(ops.scaled_embedding(ids, table, 2.0, out_dtype=dy.dtype), table, dy)[0] for _ in range(3)]
    want = torch.zeros(50, 32, dtype=torch.float64, device="cuda").index_add_(0, ids.clamp(min=0), torch.where(
        ids[:, None] >= 0, dy.double(), 0.0)) * 2.0
    assert torch.equal(g[0].double(), want) and torch.equal(g[0], g[1]) and torch.equal(g[0], g[2])
    dy = normal(N, 32, device="cuda", dtype=torch.bfloat16, seed=4)
    g = [torch.autograd.grad(ops.scaled_embedding(ids, table, 2.0, out_dtype=dy.dtype), table, dy)[0] for _ in range(3)]
    assert torch.equal(g[0], g[1]) and torch.equal(g[0], g[2])


@pytest.mark.parametrize("device", DEVICES)
def test_embedded_tokens_of_any_shape(device):
    """Ids of several dimensions, types and strides, a table and a gradient that are views."""
    big = normal(40, 48, device=device, dtype=torch.bfloat16, seed=1)
    for table in (big[:, 8:40], big[::2], big.t()):
        V, D = table.shape
        table = table.detach().requires_grad_()
        ids = torch.randint(0, V, (6, 10), generator=gen(1)).to(device)
        for i in (ids, ids.t(), ids.int(), ids.to(torch.int16)[:, 1::2], ids[:0], ids[0, 0]):
            y = ops.scaled_embedding(i, table, 0.5)
            assert y.shape == i.shape + (D,) and torch.equal(y, (table[i.long()] * 0.5).detach())
            dy = normal(*i.shape, 2 * D, device=device, dtype=y.dtype, seed=2)[..., ::2]
            (g,) = torch.autograd.grad(y, table, dy)
            n = max(1, i.numel())
            want, mag = (torch.zeros(V, D, dtype=torch.float64, device=device) for _ in range(2))
            want.index_add_(0, i.long().reshape(-1), dy.double().reshape(-1, D))
            mag.index_add_(0, i.long().reshape(-1), dy.double().abs().reshape(-1, D))
            within(g, want * 0.5, (n + 2) * E * mag)
    y = ops.scaled_embedding(ids, table, 0.5)
    (g,) = torch.autograd.grad(y.sum(), table)            # a gradient that is broadcast
    assert torch.equal(g[:, 0].float(), torch.bincount(ids.reshape(-1), minlength=V).to(g.dtype).float() * 0.5)


# ------------------------------------------------------------------------------ gated feed-forward block
def act64(z, kind):
    if kind == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * (1 - s)
    if kind == "gelu":
        phi = 0.5 * torch.special.erfc(-z * math.sqrt(0.5))
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    q = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    s = torch.sigmoid(q)
    return z * s, s + z * s * (1 - s) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)


def mlp64(x, w1, b1, w2, b2, res, dy, kind, u):
    """((value, its error) of y, dx, dw1, db1, dw2, db2) with 16-bit values of half a step u in between"""
    x, w1, w2, dy = (t.detach().double() for t in (x, w1, w2, dy))
    K, H, N, M = x.shape[1], w2.shape[1], w2.shape[0], x.shape[0]
    z, zm = x @ w1.t(), x.abs() @ w1.abs().t()
    if b1 is not None:
        z, zm = z + b1.detach().double(), zm + b1.detach().double().abs()
    ez = sums(K) * zm
    gate, up, eg, eu = z[:, :H], z[:, H:], ez[:, :H], ez[:, H:]
    a, slope = act64(gate, kind)

    def hidden(eg, eu):
        ea = 1.2 * eg + 1e-6 * (1 + gate.abs())
        e = ea * (up.abs() + eu) + a.abs() * eu
        return e + u * (a * up).abs() + u * e
    h, eh = a * up, hidden(eg, eu)
    y, ey = h @ w2.t(), eh @ w2.abs().t() + sums(H) * (h.abs() + eh) @ w2.abs().t()
    for t in (b2, res):
        if t is not None:
            y, ey = y + t.detach().double(), ey + E * (y.abs() + t.detach().double().abs())
    eg, eu = (e + u * (t.abs() + e) for e, t in ((eg, gate), (eu, up)))       # as they were kept
    dh, dhm = dy @ w2, dy.abs() @ w2.abs()
    edh = sums(N) * dhm
    dg, du = dh * up * slope, dh * a
    es = 0.8 * eg + 1e-6 * (1 + gate.abs())
    ea = 1.2 * eg + 1e-6 * (1 + gate.abs())
    edg = edh * ((up.abs() + eu) * 1.2) + (dh.abs() + edh) * (eu * 1.2 + (up.abs() + eu) * es)
    edu = edh * a.abs() + (dh.abs() + edh) * ea
    d = torch.cat([dg, du], 1)
    ed = torch.cat([edg, edu], 1)
    ed = ed + u * (d.abs() + ed)
    eh = hidden(eg, eu)
    dx, edx = d @ w1, ed @ w1.abs() + sums(2 * H) * (d.abs() + ed) @ w1.abs()
    dw1, edw1 = d.t() @ x, ed.t() @ x.abs() + sums(M) * (d.abs() + ed).t() @ x.abs()
    dw2, edw2 = dy.t() @ h, dy.abs().t() @ eh + sums(M) * dy.abs().t() @ (h.abs() + eh)
    return ((y, ey), (dx, edx), (dw1, edw1), (dw2, edw2), (d.sum(0), ed.sum(0) + sums(M) * (d.abs() + ed).sum(0)),
            (dy.sum(0), sums(M) * dy.abs().sum(0)))


MLP = [(1, 8, 8, 8, "silu", False, False), (3, 16, 24, 8, "gelu", True, False), (64, 64, 128, 64, "silu", False, True),
       (129, 72, 136, 40, "gelu_tanh", True, True), (257, 264, 520, 264, "gelu", True, True),
       (7, 128, 1000, 72, "silu", True, False), (300, 40, 64, 1032, "gelu_tanh", False, False),
       (2500, 128, 648, 128, "silu", False, True),       # tiles of pairs, the last of them ragged
       (1, 2048, 1024, 2056, "gelu", True, True), (130, 1032, 2048, 520, "silu", True, False),    # products in parts
       (300, 4096, 2560, 1024, "gelu_tanh", False, True),
       (5, 20, 30, 12, "silu", True, True), (33, 24, 27, 16, "gelu", False, True), (2, 3, 1, 1, "silu", False, False)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("M,K,H,N,kind,biases,residual", MLP, ids=str)
def test_gated_mlp(M, K, H, N, kind, biases, residual, dtype, device):
    new = lambda *s, seed, std=1.0: normal(*s, device=device, dtype=dtype, seed=seed, std=std)
    x, w1 = new(M, K, seed=1), new(2 * H, K, seed=2, std=1.5 * K ** -0.5)
    w2, dy = new(N, H, seed=3, std=H ** -0.5), new(M, N, seed=4)
    b1, b2 = (new(2 * H, seed=5, std=0.3), new(N, seed=6)) if biases else (None, None)
    res = new(M, N, seed=7) if residual else None
    leaves = [t.requires_grad_() for t in (x, w1, w2, b1, b2, res) if t is not None]
    y = ops.gated_mlp(x, w1, b1, w2, b2, kind, res)
    grads = dict(zip(map(id, leaves), torch.autograd.grad(y, leaves, dy)))
    want = mlp64(x, w1, b1, w2, b2, res, dy, kind, U[dtype])
    within(y.detach(), *want[0])
    for t, w in zip((x, w1, w2, b1, b2), want[1:]):
        if t is not None:
            assert grads[id(t)].dtype == dtype
            within(grads[id(t)], *w)
    if residual:
        assert torch.equal(grads[id(res)], dy)
    with torch.no_grad():
        assert torch.equal(ops.gated_mlp(x, w1, b1, w2, b2, kind, res), y)
    again = torch.autograd.grad(ops.gated_mlp(x, w1, b1, w2, b2, kind, res), leaves, dy)
    assert all(torch.equal(a, grads[id(t)]) for a, t in zip(again, leaves))


@pytest.mark.parametrize("device", DEVICES)
def test_gated_mlp_of_views(device):
    """Rows, weights and gradients that are slices, transposed or off their vectors; dims in front; some gradients."""
    new = lambda *s, seed: normal(*s, device=device, dtype=torch.bfloat16, seed=seed, std=0.3)
    x = new(2, 5, 72, seed=1)[:, 1:4, 4:36]
    w1 = new(65, 32, seed=2)[1:].requires_grad_()
    w2 = new(32, 24, seed=3).t().requires_grad_()
    off = new(24 * 32 + 1, seed=3)[1:].view(24, 32)
    dy = new(3, 2, 24, seed=4).transpose(0, 1)
    for second in (w2, off):
        y = ops.gated_mlp(x, w1, None, second, None)
        want = mlp64(x.reshape(-1, 32), w1, None, second, None, None, dy.reshape(-1, 24), "silu", U[torch.bfloat16])
        within(y.detach().reshape(-1, 24), *want[0])
        (dw1,) = torch.autograd.grad(y, w1, dy)
        within(dw1, *want[2])
    x = x.detach().requires_grad_()
    y = ops.gated_mlp(x, w1.detach(), None, w2.detach(), None)
    within(torch.autograd.grad(y, x, dy)[0].reshape(-1, 32), *mlp64(
        x.reshape(-1, 32), w1, None, w2, None, None, dy.reshape(-1, 24), "silu", U[torch.bfloat16])[1])
    y = ops.gated_mlp(x[:, :0], w1, None, w2, None)
    dx, dw1, dw2 = torch.autograd.grad(y, [x, w1, w2], y)
    assert y.shape == (2, 0, 24) and not dx.any() and not dw1.any() and not dw2.any()


@pytest.mark.parametrize("device", DEVICES)
def test_large_gates(device):
    """Gates far out: the activation is the gate or nothing, its derivative one or nothing, and nothing is a NaN."""
    for dtype, far in ((torch.bfloat16, 1e18), (torch.float16, 6e4)):
        for kind in ("silu", "gelu", "gelu_tanh"):
            if device == "cpu" and kind == "gelu_tanh":
                far = min(far, 1e12)                  # whose cube fp32 has
            gates = torch.tensor([far, -far, 200.0, -200.0, 88.5, -88.5, -12.0, 0.0])
            x = torch.ones(1, 8, device=device, dtype=dtype, requires_grad=True)
            w1 = torch.zeros(16, 8, device=device, dtype=dtype)
            w1[:8, 0], w1[8:, 1] = gates.to(device, dtype), 1.0
            w1.requires_grad_()
            y = ops.gated_mlp(x, w1, None, torch.eye(8, device=device, dtype=dtype), None, kind)
            (dw1,) = torch.autograd.grad(y, w1, torch.ones_like(y))
            a, slope = act64(w1[:8, 0].detach().double().clamp(-1e4, 1e4), kind)
            a = torch.where(w1[:8, 0] > 1e4, w1[:8, 0].double(), a)
            within(y.detach()[0], a, 1e-6 * (1 + a.abs()) + U[dtype] * a.abs())
            within(dw1[:8, 0], slope, 1e-5 + U[dtype] * slope.abs())


# ------------------------------------------------------------------------------ head and loss
def head64(x, w, target, g, reduction, u, unit, ignore=-100):
    """((value, error) of the loss, dx, dw), rows that count only"""
    x, w, g = x.detach().double(), w.detach().double(), g.double()
    counted = (target >= 0) & (target < w.shape[0]) & (target != ignore)
    rows = counted.nonzero().squeeze(1)
    xr, t, at = x[rows], target[rows].long(), torch.arange(len(rows), device=x.device)
    z, ez = xr @ w.t(), sums(x.shape[1]) * (xr.abs() @ w.abs().t())
    logp = torch.log_softmax(z, -1)
    p, most = logp.exp(), ez.amax(-1, keepdim=True) if len(rows) else ez.new_zeros(0, 1)
    each = -logp[at, t]
    e_each = 2 * most.squeeze(1) + 1e-6 + 2 * E * (z.abs().amax(-1) if len(rows) else 0)
    n = max(1, len(rows)) if reduction == "mean" else 1
    if reduction == "none":
        loss, e_loss = (torch.zeros(len(x), dtype=torch.float64, device=x.device).index_copy(0, rows, v)
                        for v in (each, e_each))
        coef = g[rows][:, None]
    else:
        loss, e_loss = each.sum() / n, e_each.sum() / n
        coef = g / n
    d = p.clone()
    d[at, t] -= 1
    ed = p * (2 * (most + ez) + 4e-6)
    ed = ed + u * (d.abs() + ed) + 2.0 ** -25 / unit       # 16 bits of dz, before its factor
    c = coef.abs() * (1 + 4 * E)
    dx, dw = torch.zeros_like(x), (coef * d).t() @ xr
    edx = torch.zeros_like(x)
    dx[rows] = coef * d @ w
    edx[rows] = c * (ed + sums(w.shape[0]) * (d.abs() + ed)) @ w.abs()
    edw = (c * (ed + sums(len(rows)) * (d.abs() + ed))).t() @ xr.abs()
    return (loss, e_loss), (dx, edx), (dw, edw)


HEAD = [(1, 8, 1, 1.0, "mean"), (3, 16, 9, 1.0, "none"), (64, 64, 256, 0.7, "mean"), (300, 264, 1001, 0.7, "none"),
        (130, 100, 129, 0.5, "sum"), (257, 72, 5000, 0.9, "mean"), (1000, 40, 301, 0.2, "none"), (9, 3, 65, 1.0, "sum"),
        (100, 64, 70, 0.0, "mean"), (700, 136, 4097, 1.0, "mean")]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("N,D,V,part,reduction", HEAD, ids=str)
def test_head(N, D, V, part, reduction, dtype, device):
    x = normal(N, D, device=device, dtype=dtype, seed=1).requires_grad_()
    w = normal(V, D, device=device, dtype=dtype, seed=2, std=2.0 * D ** -0.5).requires_grad_()
    target = torch.randint(0, V, (N,), generator=gen(3))
    target[torch.rand(N, generator=gen(4)) >= part] = -100
    target[N // 2:: 17] = V                               # outside the vocabulary
    target = target.to(device)
    g = torch.randn(N, generator=gen(5)).to(device) if reduction == "none" else torch.tensor(0.37, device=device)
    loss = ops.linear_cross_entropy(x, w, target, reduction=reduction)
    dx, dw = torch.autograd.grad(loss, [x, w], g)
    unit = 2.0 ** 15 if dtype == torch.float16 else 2.0 ** 100
    if reduction == "none":
        unit /= 2 * float(g.abs().max())                  # rows' factors are divided by a power of two near the largest
        unit = unit * float(g.abs().min())
    want = head64(x, w, target, g, reduction, U[dtype], unit)
    assert loss.dtype == torch.float32 and dx.dtype == dw.dtype == dtype
    within(loss.detach(), *want[0])
    within(dx, *want[1])
    within(dw, *want[2])
    counted = (target >= 0) & (target < V)
    assert not dx[~counted].any()
    if reduction == "none":
        assert not loss[~counted].any()
    again = torch.autograd.grad(ops.linear_cross_entropy(x, w, target, reduction=reduction), [x, w], g)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])
    with torch.no_grad():
        assert torch.equal(ops.linear_cross_entropy(x, w, target, reduction=reduction), loss)


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_head_in_pieces(reduction):
    """More rows and words than one piece of the backward has: the last piece is ragged."""
    N, D, V = 33000, 16, 9000
    x = normal(N, D, device="cuda", dtype=torch.bfloat16, seed=1).requires_grad_()
    w = normal(V, D, device="cuda", dtype=torch.bfloat16, seed=2, std=0.5).requires_grad_()
    target = torch.randint(0, V, (N,), generator=gen(3)).cuda()
    g = torch.rand(N, generator=gen(5)).cuda() + 0.1 if reduction == "none" else torch.tensor(1.0, device="cuda")
    dx, dw = torch.autograd.grad(ops.linear_cross_entropy(x, w, target, reduction=reduction), [x, w], g)
    want = head64(x, w, target, g, reduction, U[torch.bfloat16], 2.0 ** 100)
    within(dx, *want[1])
    within(dw, *want[2])


@pytest.mark.gpu
@pytest.mark.parametrize("N", [4095, 4097, 9000])
def test_many_rows_of_which_some_count(N):
    """Beyond the calls in which every CTA looks at all labels, too."""
    D, V = 24, 70
    x = normal(N, D, device="cuda", dtype=torch.float16, seed=1).requires_grad_()
    w = normal(V, D, device="cuda", dtype=torch.float16, seed=2, std=0.4).requires_grad_()
    target = torch.randint(0, V, (N,), generator=gen(3))
    target[torch.rand(N, generator=gen(4)) < 0.4] = -100
    target[100:1300], target[-70:] = -1, V
    target = target.cuda()
    g = torch.rand(N, generator=gen(5)).cuda() + 0.1
    loss = ops.linear_cross_entropy(x, w, target, reduction="none")
    dx, dw = torch.autograd.grad(loss, [x, w], g)
    want = head64(x, w, target, g, "none", U[torch.float16], 2.0 ** 15 / 2 * float(g.min() / g.max()))
    within(loss.detach(), *want[0])
    within(dx, *want[1])
    within(dw, *want[2])
    out = (target < 0) | (target >= V)
    assert not loss[out].any() and not dx[out].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("N,D,V,part", [(5000, 24, 40000, 0.03), (5000, 24, 40000, 0.5), (5200, 264, 40000, 0.002),
                                        (6000, 72, 2000, 0.9), (6000, 72, 2000, 0.02), (9000, 20, 300, 0.3),
                                        (9000, 20, 300, 0.0), (4800, 1032, 130, 1.0), (300, 520, 9001, 0.1)], ids=str)
def test_parts_by_the_rows_there_are(N, D, V, part, dtype):
    """The parts of dx follow the rows that count: one or more of them, in one piece of the vocabulary or several."""
    x = normal(N, D, device="cuda", dtype=dtype, seed=1).requires_grad_()
    w = normal(V, D, device="cuda", dtype=dtype, seed=2, std=2.0 * D ** -0.5).requires_grad_()
    target = torch.randint(0, V, (N,), generator=gen(3))
    target[torch.rand(N, generator=gen(4)) >= part] = -100
    target = target.cuda()
    g = torch.tensor(0.37, device="cuda")
    loss = ops.linear_cross_entropy(x, w, target)
    dx, dw = torch.autograd.grad(loss, [x, w], g, retain_graph=True)
    want = head64(x, w, target, g, "mean", U[dtype], 2.0 ** 15 if dtype == torch.float16 else 2.0 ** 100)
    within(loss.detach(), *want[0])
    within(dx, *want[1])
    within(dw, *want[2])
    assert not dx[target < 0].any()
    again = torch.autograd.grad(loss, [x, w], g)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])


@pytest.mark.parametrize("device", DEVICES)
def test_rows_that_do_not_count_reach_nothing(device):
    """Whatever they hold: infinities and NaN, in rows between others and behind the last."""
    N, D, V = 150, 24, 40
    target = torch.randint(0, V, (N,), generator=gen(1))
    target[::3], target[140:] = -100, -1
    target = target.to(device)
    x = normal(N, D, device=device, dtype=torch.bfloat16, seed=1)
    w = normal(V, D, device=device, dtype=torch.bfloat16, seed=2).requires_grad_()
    bad = x.clone()
    bad[target < 0] = torch.tensor([math.nan, math.inf, -math.inf], device=device).repeat(8).to(x.dtype)
    out = []
    for t in (x, bad):
        t = t.requires_grad_()
        loss = ops.linear_cross_entropy(t, w, target)
        out.append((loss.detach(), *torch.autograd.grad(loss, [t, w])))
    assert all(torch.equal(a, b) for a, b in zip(*out)) and torch.isfinite(out[0][0])
    assert not out[1][1][target < 0].any()
    # a row that counts keeps its NaN to itself, but for the weights
    bad = x.detach().clone()
    bad[1, 0] = math.nan
    bad.requires_grad_()
    each = ops.linear_cross_entropy(bad, w, target, reduction="none")
    (dx,) = torch.autograd.grad(each.sum(), bad)
    assert each.isnan().nonzero().squeeze(1).tolist() == [1]
    assert torch.equal(dx[2:], out[0][1][2:] * 0 + torch.autograd.grad(ops.linear_cross_entropy(
        x, w, target, reduction="none").sum(), x)[0][2:])


@pytest.mark.parametrize("device", DEVICES)
def test_head_of_views_and_frozen_parts(device):
    x = normal(4, 9, 48, device=device, dtype=torch.float16, seed=1)[:, 1:, 3:35].requires_grad_()
    wide = normal(60, 41, device=device, dtype=torch.float16, seed=2, std=0.4)
    target = torch.randint(0, 60, (8, 4), generator=gen(3)).to(device).t()
    g = torch.tensor(0.5, device=device)
    for w in (wide[:, 1:33], wide[:, :32].t().contiguous().t(), wide[::2, 8:40].detach()):
        w = w.detach().requires_grad_()
        flat = (x.reshape(-1, 32), w, target.reshape(-1))
        want = head64(*flat, g, "mean", U[torch.float16], 2.0 ** 15)
        loss = ops.linear_cross_entropy(x, w, target.to(torch.int32))
        within(loss.detach(), *want[0])
        dx, dw = torch.autograd.grad(loss, [x, w], g)
        within(dx.reshape(-1, 32), *want[1])
        within(dw, *want[2])
        (only,) = torch.autograd.grad(ops.linear_cross_entropy(x.detach(), w, target), w, g)
        assert torch.equal(only, dw)
        (only,) = torch.autograd.grad(ops.linear_cross_entropy(x, w.detach(), target), x, g)
        assert torch.equal(only, dx)
    each = ops.linear_cross_entropy(x, w, target, reduction="none")
    assert each.shape == target.shape
    (a,) = torch.autograd.grad(each.sum(), x, retain_graph=True)      # one value for all rows
    (b,) = torch.autograd.grad(each, x, torch.ones_like(each))
    assert torch.equal(a, b)
    other = ops.linear_cross_entropy(x, w, target.where(target != 7, -5), ignore_index=3)
    want = head64(x.reshape(-1, 32), w, target.where(target != 7, -5).reshape(-1), g, "mean", U[torch.float16],
                  2.0 ** 15, ignore=3)
    within(other.detach(), *want[0])
    none = x.detach()[:, :0].requires_grad_()
    loss = ops.linear_cross_entropy(none, w, target[:, :0])
    dx, dw = torch.autograd.grad(loss, [none, w])
    assert float(loss.detach()) == 0.0 and dx.shape == none.shape and not dw.any()


@pytest.mark.parametrize("device", DEVICES)
def test_small_gradients_of_a_loss(device):
    """The mean over many rows and a vocabulary of small probabilities: fp16 would lose them without their factor."""
    N, D, V = 2048, 64, 3000
    x = normal(N, D, device=device, dtype=torch.float16, seed=1).requires_grad_()
    w = normal(V, D, device=device, dtype=torch.float16, seed=2, std=0.02).requires_grad_()
    target = torch.zeros(N, dtype=torch.int64, device=device)
    g = torch.tensor(65536.0, device=device)
    loss = ops.linear_cross_entropy(x, w, target)
    dx, dw = torch.autograd.grad(loss, [x, w], g)
    want = head64(x, w, target, g, "mean", U[torch.float16], 2.0 ** 15)
    within(dw, *want[2])
    rest = want[2][0][1:]                                  # words that are no label
    assert float((dw[1:].double() - rest).norm() / rest.norm()) < 2e-3


# ------------------------------------------------------------------------------ differences, refusals
def test_gradients_are_those_of_differences():
    """In 64 bits, where the formulas are the kernels' (the kernels have no such type)."""
    f64 = lambda *s, seed: torch.randn(*s, dtype=torch.float64, generator=gen(seed)).requires_grad_()
    x, w1, w2, res = f64(3, 4, 6, seed=1), f64(14, 6, seed=2), f64(5, 7, seed=3), f64(3, 4, 5, seed=4)
    b1, b2 = f64(14, seed=5), f64(5, seed=6)
    for kind in ("silu", "gelu", "gelu_tanh"):
        assert torch.autograd.gradcheck(lambda *a: ops.gated_mlp(*a[:5], kind, a[5]), [x, w1, b1, w2, b2, res])
    w, target = f64(9, 6, seed=7), torch.randint(0, 9, (3, 4), generator=gen(8))
    target[0, 1], target[2, 2] = -100, 9
    for reduction in ("mean", "sum", "none"):
        assert torch.autograd.gradcheck(lambda a, b: ops.linear_cross_entropy(a, b, target, reduction=reduction), [x, w])
    ids = torch.tensor([[0, 2, 2], [4, -1, 7]])
    assert torch.autograd.gradcheck(lambda t: ops.scaled_embedding(ids, t, 1.7), [f64(5, 4, seed=9)])


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    new = lambda *s: torch.zeros(*s, device=device, dtype=torch.bfloat16)
    for bad in (lambda: ops.gated_mlp(new(4, 8), new(16, 9), None, new(8, 8), None),
                lambda: ops.gated_mlp(new(4, 8), new(15, 8), None, new(8, 8), None),
                lambda: ops.gated_mlp(new(4, 8), new(16, 8), None, new(8, 9), None),
                lambda: ops.gated_mlp(new(4, 8), new(16, 8), new(8), new(8, 8), None),
                lambda: ops.gated_mlp(new(4, 8), new(16, 8), None, new(8, 8), new(4)),
                lambda: ops.gated_mlp(new(4, 8), new(16, 8), None, new(8, 8), None, residual=new(8)),
                lambda: ops.gated_mlp(new(4, 8), new(16, 8), None, new(8, 8), None, "relu"),
                lambda: ops.gated_mlp(new(4, 8), new(0, 8), None, new(8, 0), None),
                lambda: ops.linear_cross_entropy(new(4, 8), new(9, 7), new(4).long()),
                lambda: ops.linear_cross_entropy(new(4, 8), new(0, 8), new(4).long()),
                lambda: ops.linear_cross_entropy(new(4, 8), new(9, 8), new(5).long()),
                lambda: ops.linear_cross_entropy(new(4, 8), new(9, 8), new(4)),
                lambda: ops.linear_cross_entropy(new(4, 8), new(9, 8), new(4).long(), reduction="max"),
                lambda: ops.scaled_embedding(new(4), new(9, 8)),
                lambda: ops.scaled_embedding(new(4) > 0, new(9, 8)),
                lambda: ops.scaled_embedding(new(4).long(), new(9)),
                lambda: ops.scaled_embedding(new(4).long(), new(9, 8), math.inf),
                lambda: ops.scaled_embedding(new(4).long(), new(9, 8), out_dtype=torch.int32)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """A table, and gate and up, of more than 2^31 values: what lies at their end, against small calls."""
    V, D, N = 270000, 8192, 300
    table = torch.zeros(V, D, device="cuda", dtype=torch.bfloat16)
    table[-9:] = normal(9, D, device="cuda", dtype=torch.bfloat16, seed=1)
    table.requires_grad_()
    ids = torch.randint(V - 9, V, (N,), generator=gen(2)).cuda()
    small = table.detach()[-9:].clone().requires_grad_()
    y, want = ops.scaled_embedding(ids, table, 2.0), ops.scaled_embedding(ids - (V - 9), small, 2.0)
    assert torch.equal(y, want)
    (g,), (gw,) = torch.autograd.grad(y, table, y.detach()), torch.autograd.grad(want, small, y.detach())
    assert torch.equal(g[-9:], gw) and not g[:-9].any()
    del table, g
    M, D, H, N = 106000, 64, 10240, 64
    x, dy = (normal(M, D, device="cuda", dtype=torch.bfloat16, seed=s).requires_grad_() for s in (3, 4))
    w1, w2 = (normal(*s, device="cuda", dtype=torch.bfloat16, seed=5, std=0.05) for s in ((2 * H, D), (N, H)))
    y = ops.gated_mlp(x, w1, None, w2, None)
    (g,) = torch.autograd.grad(y, x, dy.detach())
    part = x.detach()[-2048:].clone().requires_grad_()
    want = ops.gated_mlp(part, w1, None, w2, None)
    (gw,) = torch.autograd.grad(want, part, dy.detach()[-2048:])
    # the same sums, in another order where a reduction is split
    for a, b in ((y[-2048:], want), (g[-2048:], gw)):
        assert float((a - b).detach().float().norm()) <= 4 * 2.0 ** -8 * float(b.detach().float().norm())


@pytest.mark.gpu
def test_operands_of_two_devices_are_refused():
    new = lambda *s, d="cuda": torch.zeros(*s, device=d, dtype=torch.bfloat16)
    for bad in (lambda: ops.gated_mlp(new(4, 8), new(16, 8, d="cpu"), None, new(8, 8), None),
                lambda: ops.gated_mlp(new(4, 8), new(16, 8), None, new(8, 8), None, residual=new(4, 8, d="cpu")),
                lambda: ops.linear_cross_entropy(new(4, 8), new(9, 8, d="cpu"), new(4).long()),
                lambda: ops.linear_cross_entropy(new(4, 8), new(9, 8), new(4, d="cpu").long()),
                lambda: ops.scaled_embedding(new(4, d="cpu").long(), new(9, 8))):
        with pytest.raises(ValueError):
            bad()


BF16, F32 = _lib.PF_BF16, _lib.PF_F32
# Entry points with operands of 16 bytes a time: arguments of a call that is all right but for what is put in place of one,
# and the positions of those operands.  None of them reaches a device: the first that is wrong is refused.
ENTRIES = {
    "pf_gated_mlp_fwd": (lambda t: [t, t, None, 0, t, None, 0, t, t, t, t, None, 0, 4, 8, 8, 8, 8, 8, 8, 8, 3, BF16, None,
                                    148, None], (0, 4, 7, 8, 9, 10)),
    "pf_gated_mlp_bwd": (lambda t: [t, t, t, t, t, t, t, t, t, t, None, None, None, 0, 4, 8, 8, 8, 8, 8, 8, 8, 3, BF16,
                                    BF16, BF16, 0, 0, 0, None, 148, None], range(10)),
    "pf_head_fwd": (lambda t: [t, t, t, t, t, t, t, t, t, 4, 8, 8, 8, 8, 8, -100, 1, BF16, None, 148, None], (1, 3, 8)),
    "pf_head_bwd": (lambda t: [t, t, t, t, t, t, t, t, t, t, None, 4, 8, 8, 8, 0, 8, 8, 0, 0, BF16, BF16, None, 148, None],
                    (2, 3, 7, 8, 9)),
    "pf_scaled_embed_bwd": (lambda t: [t, t, t, t, 4, 8, 8, 1.0, 0, BF16, BF16, None], (3,)),
}


@pytest.mark.parametrize("name", ENTRIES)
def test_operands_off_their_boundaries(name, calls):
    make, places = ENTRIES[name]
    t = torch.zeros(4096, dtype=torch.bfloat16)
    for i in places:
        args = make(t.data_ptr())
        args[i] = t.data_ptr() + 2
        assert getattr(calls, name)(*args) == -2, i


def test_entry_points_refuse(calls):
    t = torch.zeros(4096, dtype=torch.bfloat16).data_ptr()

    def answer(name, **put):
        args = ENTRIES[name][0](t)
        for i, v in put.items():
            args[int(i[1:])] = v
        return getattr(calls, name)(*args)
    fwd, bwd = "pf_gated_mlp_fwd", "pf_gated_mlp_bwd"
    assert answer(fwd, _22=F32) == answer(bwd, _23=F32) == -1
    assert answer(fwd, _21=0) == answer(fwd, _21=4) == answer(bwd, _22=7) == -1
    assert answer(fwd, _14=0) == answer(fwd, _13=-1) == answer(bwd, _16=0) == -3
    assert answer(fwd, _14=12) == answer(fwd, _15=9) == answer(bwd, _17=20) == answer(fwd, _17=12) == answer(bwd, _18=9) == -2
    assert answer(fwd, _13=0) == 0
    assert answer(bwd, _28=1) == -1                          # 16-bit gradients are not added to
    assert answer(bwd, _24=_lib.PF_F16) == -1
    for name, dtype in (("pf_head_fwd", 17), ("pf_head_bwd", 20)):
        assert answer(name, **{f"_{dtype}": F32}) == -1
        at = 9 if name == "pf_head_fwd" else 11
        assert answer(name, **{f"_{at}": -1}) == answer(name, **{f"_{at + 1}": 0}) == -3
        assert answer(name, **{f"_{at}": (1 << 28) + 1}) == -3
        assert answer(name, **{f"_{at + 3}": 12}) == answer(name, **{f"_{at + 5}": 12}) == -2
    assert answer("pf_head_bwd", _19=1) == -1 == answer("pf_head_bwd", _21=_lib.PF_F16)
    assert calls.pf_head_index(-1) == calls.pf_head_scratch(4, 0) == calls.pf_head_words(-1, 4) == -3
    assert calls.pf_head_scratch(1 << 28, 1 << 28) == -3     # more KiB than an int has
    assert calls.pf_scaled_embed_scratch(-1, 8, 8) == calls.pf_scaled_embed_scratch(8, 8, 1 << 30) == -3
    assert answer("pf_scaled_embed_bwd", _4=-1) == -3 and answer("pf_scaled_embed_bwd", _8=1) == -1
    assert answer("pf_scaled_embed_bwd", _3=t + 16) == -2 and answer("pf_scaled_embed_bwd", _6=0) == 0


@pytest.mark.parametrize("N,V", [(1, 8), (256, 32000), (8192, 32000), (4095, 128011), (1 << 20, 50257)])
def test_pieces_of_the_vocabulary(calls, N, V):
    """Whole tiles of words, no more of them alive than 2^27 values unless a piece would have fewer than 4096 words, and all
    of a vocabulary of that size in one piece."""
    words, rows = calls.pf_head_words(N, V), (N + 255) // 256 * 256
    assert words % 256 == 0 and 0 < words
    assert words * rows <= 2 ** 27 or words <= 4096
    assert words >= V or words >= 2048


# ------------------------------------------------------------------------------ how a program uses them
def _all(device, dtype, seed=0, N=70):
    """(leaves, a function that takes them through embedding, block and head to a loss)"""
    table = normal(50, 32, device=device, dtype=dtype, seed=seed + 1)
    w1, w2 = (normal(*s, device=device, dtype=dtype, seed=seed + i, std=0.2) for s, i in (((96, 32), 2), ((32, 48), 3)))
    head = normal(50, 32, device=device, dtype=dtype, seed=seed + 4, std=0.3)
    leaves = [t.requires_grad_() for t in (table, w1, w2, head)]

    def run(ids, labels):
        h = ops.scaled_embedding(ids, leaves[0], 1.5)
        h = ops.gated_mlp(h, leaves[1], None, leaves[2], None, residual=h)
        return ops.linear_cross_entropy(h, leaves[3], labels)
    return leaves, run


def _data(device, seed, N=70):
    ids = torch.randint(0, 50, (N,), generator=gen(seed))
    labels = torch.randint(0, 50, (N,), generator=gen(seed + 1))
    labels[::5] = -100
    return ids.to(device), labels.to(device)


@pytest.mark.gpu
def test_captured_and_replayed():
    """A forward and backward in a graph, replayed on other data beside a second graph and eager calls."""
    leaves, run = _all("cuda", torch.bfloat16)
    graphs = []
    for seed in (10, 20):
        ids, labels = _data("cuda", seed)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(2):
                torch.autograd.grad(run(ids, labels), leaves)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            loss = run(ids, labels)
            grads = torch.autograd.grad(loss, leaves)
        graphs.append((graph, ids, labels, loss, grads))
    for seed in (30, 40, 50):
        for i, (graph, ids, labels, loss, grads) in enumerate(graphs):
            new = _data("cuda", seed + 5 * i)
            ids.copy_(new[0])
            labels.copy_(new[1] if seed != 40 else torch.full_like(new[1], -100))
            graph.replay()
        for graph, ids, labels, loss, grads in graphs:
            want = run(ids, labels)
            assert torch.equal(want, loss)
            assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(want, leaves), grads))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64], ids=str)
def test_captured_in_full_precision(dtype):
    """PyTorch's own products ask the host for nothing either, and which rows count may differ from replay to replay."""
    leaves, run = _all("cuda", dtype)
    ids, labels = _data("cuda", 10)
    for _ in range(2):
        torch.autograd.grad(run(ids, labels), leaves)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = run(ids, labels)
        grads = torch.autograd.grad(loss, leaves)
    for seed in (30, 40):
        new = _data("cuda", seed)
        ids.copy_(new[0].masked_fill(new[0] < 5, -1))
        labels.copy_(new[1].masked_fill(new[1] < seed - 20, -100))
        graph.replay()
        want = run(ids, labels)
        assert abs(float(loss) - float(want)) <= 1e-5 * float(want)
        for a, b in zip(torch.autograd.grad(want, leaves), grads):
            assert float((a - b).norm()) <= 1e-5 * float(a.norm())


@pytest.mark.gpu
def test_no_rows_leave_buckets_as_they_are():
    leaves, run = _all("cuda", torch.float32)
    biases = [torch.randn(96, device="cuda").requires_grad_(), torch.randn(32, device="cuda").requires_grad_()]
    every = leaves[:3] + biases
    buckets = [torch.full(t.shape, 3.0, device="cuda") for t in every]
    try:
        for t, b in zip(every, buckets):
            ops.register_param(t, t.detach().to(torch.bfloat16), b)
        ids = torch.zeros(0, dtype=torch.long, device="cuda")
        with torch.autocast("cuda", dtype=torch.bfloat16):
            h = ops.scaled_embedding(ids, leaves[0], 1.5)
            y = ops.gated_mlp(h, leaves[1], biases[0], leaves[2], biases[1])
        assert y.shape == (0, 32)
        assert all(g is None for g in torch.autograd.grad(y.float().sum(), every, allow_unused=True))
        assert all((b == 3.0).all() for b in buckets)
    finally:
        ops.unregister_params()


@pytest.mark.gpu
def test_streams_and_threads():
    leaves, run = _all("cuda", torch.bfloat16)
    data = [_data("cuda", 10 * i, N=70 + 300 * i) for i in range(4)]
    want = [(l, torch.autograd.grad(l, leaves)) for l in (run(*d) for d in data)]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                loss = run(*data[i])
                got[i] = (loss, torch.autograd.grad(loss, leaves))
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for (a, ga), (b, gb) in zip(want, got):
        assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in zip(ga, gb))


@pytest.mark.gpu
def test_registered_weights_get_their_gradients_in_their_buckets():
    """16-bit shadows are read and fp32 buckets added to, tied weights included, as gradients of autograd would be."""
    leaves, run = _all("cuda", torch.float32)
    ids, labels = _data("cuda", 10)
    try:
        low = [t.detach().to(torch.bfloat16).requires_grad_() for t in leaves]
        h = ops.scaled_embedding(ids, low[0], 1.5)
        h = ops.gated_mlp(h, low[1], None, low[2], None, residual=h)
        want = torch.autograd.grad(ops.linear_cross_entropy(h, low[3], labels), low)
        buckets = [torch.full(t.shape, 3.0, device="cuda") for t in leaves]
        for t, b in zip(leaves, buckets):
            ops.register_param(t, t.detach().to(torch.bfloat16), b)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss = run(ids, labels)
        grads = torch.autograd.grad(loss, leaves, allow_unused=True)
        assert all(g is None for g in grads)
        for b, w in zip(buckets, want):
            # the bucket's 3.0 takes bits of small gradients; the 16-bit gradient is rounded
            assert ((b - 3.0).double() - w.double()).abs().le(2.0 ** -8 * w.double().abs() + 2.0 ** -21).all()
        ops.unregister_params()
        tied = normal(50, 32, device="cuda", dtype=torch.float32, seed=9, std=0.3).requires_grad_()
        bucket = torch.zeros_like(tied)
        low = tied.detach().to(torch.bfloat16)
        ops.register_param(tied, low, bucket)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss = ops.linear_cross_entropy(ops.scaled_embedding(ids, tied, 2.0), tied, labels)
        torch.autograd.grad(loss, tied, allow_unused=True)
        ops.unregister_params()
        low = low.requires_grad_()
        (w,) = torch.autograd.grad(ops.linear_cross_entropy(ops.scaled_embedding(ids, low, 2.0), low, labels), low)
        # autograd adds two 16-bit gradients in 16 bits
        assert (bucket.double() - w.double()).abs().max() <= 2.0 ** -7 * float(w.abs().max())
    finally:
        ops.unregister_params()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
def test_autocast_and_full_precision(device, dtype):
    """fp32 leaves under autocast, or without it in PyTorch's own products."""
    leaves, run = _all(device, torch.float32)
    ids, labels = _data(device, 10)
    with torch.autocast(device, dtype=dtype, enabled=dtype != torch.float32):
        loss = run(ids, labels)
    grads = torch.autograd.grad(loss, leaves)
    wide = [t.detach().double().cpu().requires_grad_() for t in leaves]
    h = ops.scaled_embedding(ids.cpu(), wide[0], 1.5)
    h = ops.gated_mlp(h, wide[1], None, wide[2], None, residual=h)
    want = ops.linear_cross_entropy(h, wide[3], labels.cpu())
    # some ten roundings lie between a leaf and its gradient; a gradient as a whole is off by no more than they add up to
    assert abs(float(loss) - float(want)) <= 16 * U[dtype] * float(want) + 2e-6
    for g, w in zip(grads, torch.autograd.grad(want, wide)):
        assert g.dtype == torch.float32 and float((g.cpu().double() - w).norm() / w.norm()) <= 16 * U[dtype] + 2e-5


def test_shapes_without_data():
    """What a trace sees: shapes and types of every output, and a gradient through the registered ops."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    leaves, run = _all("cpu", torch.bfloat16)
    ids, labels = _data("cpu", 10)
    with FakeTensorMode() as mode:
        low = [mode.from_tensor(t) for t in leaves]
        h = ops.scaled_embedding(mode.from_tensor(ids), low[0], 1.5)
        h = ops.gated_mlp(h, low[1], None, low[2], None, residual=h)
        loss = ops.linear_cross_entropy(h, low[3], mode.from_tensor(labels))
        assert h.shape == (70, 32) and loss.shape == () and loss.dtype == torch.float32
    compiled = torch.compile(run, backend="eager")
    a, b = run(ids, labels), compiled(ids, labels)
    assert torch.equal(a, b)
    for x, y in zip(torch.autograd.grad(a, leaves), torch.autograd.grad(b, leaves)):
        assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("case", ["embedding", "wide table", "block", "biases", "head", "rows"])
def test_native_calls_equal_those_through_python(case, monkeypatch):
    """Eager calls and their backwards in C++: the same bits, and no Python on the way."""
    from pfeife_b200.ops import _lib
    if _lib.eager() is None:
        pytest.skip("the module of eager calls is not built")
    new = lambda *s, seed: normal(*s, device="cuda", dtype=torch.bfloat16, seed=seed, std=0.5)
    ids, labels = _data("cuda", 3)
    if case in ("embedding", "wide table"):
        table = new(50, 24, seed=1).to(torch.float32 if case == "wide table" else torch.bfloat16).requires_grad_()
        leaves, call = [table], lambda: ops.scaled_embedding(ids.view(7, 10), table, 3.0, out_dtype=torch.bfloat16)
    elif case in ("block", "biases"):
        leaves = [new(*s, seed=i).requires_grad_() for i, s in enumerate(((7, 10, 32), (96, 32), (40, 48), (7, 10, 40)))]
        b1, b2 = (new(n, seed=n).requires_grad_() if case == "biases" else None for n in (96, 40))
        x, w1, w2, res = leaves
        leaves = leaves + [b for b in (b1, b2) if b is not None]
        call = lambda: ops.gated_mlp(x, w1, b1, w2, b2, "gelu", res)
    else:
        leaves = [new(*s, seed=i).requires_grad_() for i, s in enumerate(((7, 10, 32), (50, 32)))]
        call = lambda: ops.linear_cross_entropy(*leaves, labels.view(7, 10),
                                                reduction="none" if case == "rows" else "mean")

    def both():
        y = call()
        return (y, *torch.autograd.grad(y, leaves, torch.ones_like(y)))
    before = _lib._eager.launches()
    native = both()
    assert _lib._eager.launches() > before + 1
    launches = _lib._launches
    both()
    assert _lib._launches == launches                     # none went through Python
    with torch.no_grad():
        assert torch.equal(call(), native[0])
    monkeypatch.setattr(_lib, "_eager", None)
    monkeypatch.setattr(_lib, "eager", lambda: None)
    for a, b in zip(native, both()):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)


@pytest.mark.gpu
def test_saved_tensors_may_come_back_otherwise():
    """Hooks that unpack what was saved in another place or order of memory, in C++ and through Python."""
    from pfeife_b200.ops import _lib
    leaves, run = _all("cuda", torch.bfloat16)
    ids, labels = _data("cuda", 10)
    want = torch.autograd.grad(run(ids, labels), leaves)

    def moved(t):
        if t.dim() == 2 and t.is_floating_point():
            big = torch.empty(t.shape[1], t.shape[0] + 1, dtype=t.dtype, device=t.device)
            big[:, 1:] = t.t()
            return big[:, 1:].t()                         # the same values, columns innermost and off their vectors
        return t.clone()
    for through in ("C++", "Python"):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, moved):
            if through == "Python":
                held, _lib._eager = _lib._eager, None
                tried, _lib.eager = _lib.eager, lambda: None
            try:
                got = torch.autograd.grad(run(ids, labels), leaves)
            finally:
                if through == "Python":
                    _lib._eager, _lib.eager = held, tried
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_checkpoints_and_second_backwards():
    from torch.utils.checkpoint import checkpoint
    leaves, run = _all("cuda", torch.bfloat16)
    ids, labels = _data("cuda", 10)
    loss = run(ids, labels)
    want = torch.autograd.grad(loss, leaves, retain_graph=True)
    again = torch.autograd.grad(loss, leaves)
    through = torch.autograd.grad(checkpoint(run, ids, labels, use_reentrant=False), leaves)
    for a, b, c in zip(want, again, through):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_no_rows(reduction, dtype, device):
    """The losses of no rows are none, and have no address; a sum over them is 0."""
    x = torch.zeros(3, 0, 24, device=device, dtype=dtype, requires_grad=True)
    w = normal(40, 24, device=device, dtype=dtype, seed=1).requires_grad_()
    target = torch.zeros(3, 0, device=device, dtype=torch.int64)
    with torch.no_grad():
        loss = ops.linear_cross_entropy(x, w, target, reduction=reduction)
    assert loss.shape == ((3, 0) if reduction == "none" else ()) and not loss.any()
    loss = ops.linear_cross_entropy(x, w, target, reduction=reduction)
    dx, dw = torch.autograd.grad(loss, [x, w], torch.ones_like(loss))
    assert dx.shape == x.shape and not dw.any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float64], ids=str)
@pytest.mark.parametrize("M,D,H,N", [(4, 8, 16, 8), (4, 6, 5, 7), (0, 8, 16, 8)], ids=str)
def test_what_a_tracer_is_told(M, D, H, N, dtype, device):
    """Shapes and types of the registered ops' outputs without data are those with it: whole widths and odd ones, no rows,
    operands of two types, transposed weights, any gradients."""
    from torch.library import opcheck
    from pfeife_b200.ops import functional as Fn
    tests = ("test_schema", "test_autograd_registration", "test_faketensor")
    new = lambda *s, d=dtype: normal(*s, device=device, dtype=d, seed=len(s))
    other = torch.float32 if dtype != torch.float32 else torch.bfloat16
    for wide in (dtype, other):
        x, w1, b1, w2, b2 = new(M, D), new(2 * H, D, d=wide), new(2 * H, d=wide), new(H, N, d=wide).t(), new(N, d=wide)
        dy, gu = new(M, N), new(M, 2 * H)
        for keep in (True, False):
            opcheck(Fn.gated_mlp_fwd, (x, w1, b1, w2, b2, dy, 3, keep), test_utils=tests)
        for need in ((True,) * 5, (False, True, True, False, False), (True, False, False, True, True)):
            for p, q in ((b1, b2), (b1, None), (None, None)):
                want = need[:2] + (need[2] and p is not None, need[3], need[4] and q is not None)
                opcheck(Fn.gated_mlp_bwd, (dy, x, w1, w2, gu, 3, *want, p, q), test_utils=tests)
        w, target = new(D, H, d=wide).t(), torch.arange(M, device=device) % (H + 1)
        for reduction in range(3):
            opcheck(Fn.head_loss_fwd, (x, w, target, -100, reduction), test_utils=tests)
            loss, *kept = Fn.head_loss_fwd(x, w, target, -100, reduction)
            for need in ((True, True), (False, True), (True, False)):
                opcheck(Fn.head_loss_bwd, (torch.ones_like(loss), *kept, w, M, reduction == 0, *need), test_utils=tests)
        opcheck(Fn.scaled_embed_fwd, (target, w, 2.0, dtype), test_utils=tests)
        opcheck(Fn.scaled_embed_bwd, (x, target, w, 2.0), test_utils=tests)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_head_in_64_bits(reduction, device):
    """Gradients as exact as their type, the mean's factor among them."""
    x, w = (torch.randn(s, 6, dtype=torch.float64, generator=gen(s)).to(device).requires_grad_() for s in (7, 9))
    target = torch.tensor([0, 3, -100, 8, 3, 9, 1], device=device)
    g = torch.randn(7 if reduction == "none" else (), dtype=torch.float64, generator=gen(3)).to(device)
    got = torch.autograd.grad(ops.linear_cross_entropy(x, w, target, reduction=reduction), [x, w], g)
    coef = torch.where((target >= 0) & (target < 9), g / 5 if reduction == "mean" else g, 0.0)
    d = torch.softmax(x.detach() @ w.detach().t(), -1)
    d -= torch.nn.functional.one_hot(target.clamp(0, 8), 9)
    d *= coef[:, None]
    for a, b in zip(got, (d @ w.detach(), d.t() @ x.detach())):
        assert float((a - b).norm()) <= 1e-13 * float(b.norm())      # some hundred roundings of 2^-53


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D", [8, 9, 2048], ids=["whole", "odd", "parts"])
@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh"])
def test_gates_beyond_fp16(kind, D, device):
    """Gates and up values that fp16 does not have, of hidden values that it has: they are kept as its largest, and
    gradients are those of that."""
    H, top = 8, 65504.0
    gates = torch.tensor([7e4, 1.3e5, -7e4, -1.3e5, 3e4, 0.25, 7e4, 1e5])
    ups = torch.tensor([0.5, 0.25, 0.5, -0.25, 2.0, 1.3e5, -0.5, 7e4 / 2 ** 17])
    x = torch.zeros(1, D, device=device, dtype=torch.float16)
    x[0, :2] = 2.0
    w1 = torch.zeros(2 * H, D, device=device, dtype=torch.float16)
    w1[:H, 0], w1[H:, 1] = (gates / 2).to(w1), (ups / 2).to(w1)
    x, w1, w2 = x.requires_grad_(), w1.requires_grad_(), torch.eye(H, device=device, dtype=torch.float16).requires_grad_()
    gate, up = (2 * w1.detach()[i * H:i * H + H, i].double() for i in range(2))
    dy = torch.full((1, H), 2.0 ** -6, device=device, dtype=torch.float16)
    y = ops.gated_mlp(x, w1, None, w2, None, kind)
    within(y.detach()[0], act64(gate.clamp(-1e4, 1e4), kind)[0].where(gate < 1e4, gate) * up, 1e-6 * (1 + gate.abs()) * up.abs())
    dx, dw1, dw2 = torch.autograd.grad(y, [x, w1, w2], dy)
    gate, up = gate.clamp(-top, top), up.clamp(-top, top)
    a, slope = act64(gate.clamp(-1e4, 1e4), kind)
    a = a.where(gate < 1e4, gate)
    u = U[torch.float16]
    within(dw1[:H, 0], 2.0 ** -5 * up * slope, 2.0 ** -5 * up.abs() * (1e-6 + u) + 2.0 ** -24)
    within(dw1[H:, 1], 2.0 ** -5 * a, 2.0 ** -5 * a.abs() * u + 1e-6)
    within(dw2[0], 2.0 ** -6 * a * up, 2.0 ** -6 * (a * up).abs() * u + 1e-3)
    assert torch.isfinite(dx).all()


@pytest.mark.gpu
def test_products_take_the_sms_that_a_call_is_given(monkeypatch, tmp_path):
    """Whatever calls before it were given: CTAs of pairs of a gated block and of a plain product."""
    import json
    from torch.profiler import ProfilerActivity, profile
    from pfeife_b200.ops import kernels as kx
    new = lambda *s: normal(*s, device="cuda", dtype=torch.bfloat16, seed=1, std=0.1)
    x, w1, w2 = new(2048, 256), new(4096, 256), new(256, 2048)
    grids, out = {}, []
    for sms in (148, 16, 132, 24):
        monkeypatch.setattr(kx, "sm_count", lambda device: sms)
        grids[sms] = []
        for _ in range(8):                               # a profiler may lose records, never of all calls
            with profile(activities=[ProfilerActivity.CUDA]) as p:
                out.append((kx.gated_mlp_fwd(x, w1, None, w2, None, None, 3, False)[0], kx.gemm(x, w1)))
                torch.cuda.synchronize()
            p.export_chrome_trace(str(tmp_path / "trace.json"))
            events = json.loads((tmp_path / "trace.json").read_text())["traceEvents"]
            grids[sms] += [e["args"]["grid"][0] for e in events if "gemm" in e.get("name", "") and "grid" in e.get("args", {})]
    # 128 tiles of a pair each: as many pairs as there may be, where the device takes that many
    assert all(g and max(g) <= sms for sms, g in grids.items()), grids
    assert max(grids[16]) == 16 and max(grids[24]) == 24 and max(grids[148]) > 100 and max(grids[132]) > 100, grids
    for y, z in out[1:]:
        assert torch.equal(z, out[0][1]) and float((y - out[0][0]).float().norm()) <= 2.0 ** -8 * float(y.float().norm())


@pytest.mark.parametrize("N,D,V,rows", [(128, 4096, 300, 128), (2048, 4096, 32000, 256), (9000, 8192, 32000, 256),
                                        (16384, 4096, 32000, 256), (16385, 4096, 32000, 256), (32768, 4096, 32000, 256),
                                        (1 << 18, 8192, 128011, 256)], ids=str)
def test_tiles_of_many_rows(calls, N, D, V, rows):
    """Tiles of pairs however many outputs there are; what bounds memory are the parts, and there only their number."""
    parts = calls.pf_head_parts(N, V, D, 148)
    assert calls.pf_head_tile(N, V, D, 148) == rows and (parts == 1 or parts * N * D <= 2 ** 26)
    assert calls.pf_head_tile(-1, V, D, 148) == calls.pf_head_tile(N, 0, D, 148) == -3


@pytest.mark.gpu
@pytest.mark.parametrize("N,D,V", [(17000, 4096, 300), (33000, 2056, 4500)])
def test_more_outputs_than_parts_may_have(N, D, V):
    """Gradients of so many rows that they come in one part, in one piece of the vocabulary and in two."""
    x = normal(N, D, device="cuda", dtype=torch.bfloat16, seed=1).requires_grad_()
    w = normal(V, D, device="cuda", dtype=torch.bfloat16, seed=2, std=2.0 * D ** -0.5).requires_grad_()
    target = torch.randint(0, V, (N,), generator=gen(3)).cuda()
    target[::9] = -100
    g = torch.tensor(2.0 ** 10, device="cuda")
    loss = ops.linear_cross_entropy(x, w, target)
    dx, dw = torch.autograd.grad(loss, [x, w], g)
    assert not dx[::9].any()
    rows = torch.cat([torch.arange(0, 300), torch.arange(N - 300, N)]).cuda()      # each row's own, the mean over all
    n = int((target >= 0).sum())
    want = head64(x[rows], w, target[rows], g / n, "sum", U[torch.bfloat16], 2.0 ** 100)
    within(dx[rows], *want[1])
    part = ops.linear_cross_entropy(x.detach()[:N // 2].requires_grad_(), w, target[:N // 2], reduction="sum")
    rest = ops.linear_cross_entropy(x.detach()[N // 2:].requires_grad_(), w, target[N // 2:], reduction="sum")
    total = sum(torch.autograd.grad(s, w)[0].double() for s in (part, rest)) * (2.0 ** 10 / n)
    assert float((dw.double() - total).norm()) <= 4 * 2.0 ** -8 * float(total.norm())


def _bytes(call, leaves, grad):
    """Bytes asked for beside what was there before: (kept from forward to backward, the most at one time in the forward, in
    the backward, those of the gradients)"""
    of = lambda what: torch.cuda.memory_stats()[f"requested_bytes.all.{what}"]
    torch.cuda.synchronize()
    before = of("current")
    torch.cuda.reset_peak_memory_stats()
    y = call()
    kept, top = of("current") - before, of("peak") - before
    torch.cuda.reset_peak_memory_stats()
    grads = torch.autograd.grad(y, leaves, grad)
    return kept, top, of("peak") - before, sum(t.numel() * t.element_size() for t in grads)


@pytest.mark.gpu
@pytest.mark.parametrize("N,D,V,reduction", [(8192, 256, 32000, "mean"), (40000, 64, 32000, "none"), (2048, 512, 4000, "mean")],
                         ids=str)
def test_memory_of_a_head(N, D, V, reduction):
    """Kept: the rows, their index and 8 bytes of each.  Alive beside that: forward 8 bytes of each row and 64 words;
    backward dz of a piece, of 2^27 values or 4096 words, and the parts of dx in fp32."""
    x = normal(N, D, device="cuda", dtype=torch.bfloat16, seed=1).requires_grad_()
    w = normal(V, D, device="cuda", dtype=torch.bfloat16, seed=2, std=0.1).requires_grad_()
    target = torch.randint(0, V, (N,), generator=gen(3)).cuda()
    g = torch.ones(N if reduction == "none" else (), device="cuda")
    call = lambda: ops.linear_cross_entropy(x, w, target, reduction=reduction)
    torch.autograd.grad(call(), [x, w], g)               # what is made once for the device
    kept, forward, backward, size = _bytes(call, [x, w], g)
    rows = (N + 255) // 256 * 256
    slack = 16 * 1024                                    # words that stand by themselves, KiB rounded up
    least = rows * D * 2 + rows * 12 + N * 4
    assert kept <= least + N * 4 + rows * 8 + slack
    assert forward <= kept + rows * ((V + 63) // 64 * 8 + 4 + 1) + slack
    piece = max(min(rows * (V + 255), 2 ** 27), rows * 4096)
    assert backward <= kept + size + piece * 2 + max(rows * D, 2 ** 26) * 4 + rows * 4 + slack
    if N > 2048:                                         # 2 bytes a logit, and as many for the gradient
        assert backward < N * V * 2


@pytest.mark.gpu
def test_memory_of_a_gated_block():
    """Kept: gate and up.  Alive beside them: h in either direction, gate's and up's gradients in the backward, and the
    parts of products that are split, which the workspace's size says."""
    M, D, H = 4096, 256, 2048
    x, w1, w2 = (normal(*s, device="cuda", dtype=torch.bfloat16, seed=1, std=0.1).requires_grad_()
                 for s in ((M, D), (2 * H, D), (D, H)))
    call = lambda: ops.gated_mlp(x, w1, None, w2, None)
    dy = torch.ones(M, D, device="cuda", dtype=torch.bfloat16)
    torch.autograd.grad(call(), [x, w1, w2], dy)
    kept, forward, backward, size = _bytes(call, [x, w1, w2], dy)
    slack = 16 * 1024
    assert kept <= (M * 2 * H + M * D) * 2 + slack       # with the result
    parts = _lib.calls().pf_gated_mlp_scratch(M, D, H, D, 0) * 1024
    assert forward <= kept + M * H * 2 + parts + slack and backward <= kept + size + M * 3 * H * 2 + parts + slack
    assert parts <= 2 ** 28                              # 2^26 sums


@pytest.mark.gpu
def test_memory_of_embedded_tokens():
    """Nothing is kept; beside the gradient there are 12 bytes a token, 8 a word and the windows' parts."""
    N, V, D = 8192, 30000, 512
    table = torch.zeros(V, D, device="cuda", requires_grad=True)
    ids = tokens("any", N, V).cuda()
    call = lambda: ops.scaled_embedding(ids, table, 2.0, out_dtype=torch.bfloat16)
    dy = torch.ones(N, D, device="cuda", dtype=torch.bfloat16)
    torch.autograd.grad(call(), table, dy)
    kept, forward, backward, size = _bytes(call, [table], dy)
    slack = 16 * 1024
    assert kept <= N * D * 2 + slack and forward <= kept + slack
    assert backward <= kept + size + 12 * N + 8 * V + N // 8 * 2 * D * 4 + slack


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan], ids=str)
def test_a_gradient_that_is_no_number_stays_with_its_row(bad, device):
    """Rows' gradients are divided by a power of two near the largest: of those that are numbers."""
    N, D, V = 40, 16, 50
    x = normal(N, D, device=device, dtype=torch.float16, seed=1).requires_grad_()
    w = normal(V, D, device=device, dtype=torch.float16, seed=2, std=0.3)
    target = torch.randint(0, V, (N,), generator=gen(3)).to(device)
    g = torch.linspace(500.0, 1000.0, N, device=device)
    want = head64(x, w, target, g, "none", U[torch.float16], 2.0 ** 13)[1]
    g[7] = bad
    (dx,) = torch.autograd.grad(ops.linear_cross_entropy(x, w, target, reduction="none"), x, g)
    rest = torch.arange(N, device=device) != 7
    assert not torch.isfinite(dx[7]).any()
    within(dx[rest], want[0][rest], want[1][rest])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D", [8, 9], ids=["whole", "odd"])
@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh"])
def test_gates_whose_square_fp32_does_not_have(kind, D, device):
    gates = torch.tensor([1e30, -1e30, 2e19, -2e19, 1e13, -1e13, 1e38, -1e38])
    x = torch.ones(1, D, device=device, dtype=torch.bfloat16)
    w1 = torch.zeros(16, D, device=device, dtype=torch.bfloat16)
    w1[:8, 0], w1[8:, 1] = gates.to(w1), 2.0 ** -10
    w1.requires_grad_()
    y = ops.gated_mlp(x, w1, None, torch.eye(8, device=device, dtype=torch.bfloat16), None, kind)
    gate = w1.detach()[:8, 0]
    assert torch.equal(y.detach()[0], gate.clamp(min=0) * 2.0 ** -10)
    (dw1,) = torch.autograd.grad(y, w1, torch.ones_like(y))
    assert torch.equal(dw1[:8, 0], (gate > 0).to(gate) * 2.0 ** -10) and torch.equal(dw1[8:, 1], gate.clamp(min=0))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("through", ["C++", "Python"])
@pytest.mark.parametrize("M,H", [(1, 24), (3, 24), (1, 11), (3, 20)])
def test_rows_that_start_anywhere(M, H, through, device, monkeypatch):
    """Rows, residual and gradient of a block and rows of a head that are contiguous but off their vectors, or one row of a
    matrix whose rows are."""
    if through == "Python":
        monkeypatch.setattr(_lib, "_eager", None)
        monkeypatch.setattr(_lib, "eager", lambda: None)
    new = lambda *s, seed: normal(*s, device=device, dtype=torch.bfloat16, seed=seed, std=0.5)
    w1, w2, w3 = new(2 * H, 16, seed=1), new(32, H, seed=2), new(20, 16, seed=3)
    places = [lambda t: t,
              lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape),
              lambda t: torch.cat([t.new_zeros(M, 3), t], 1)[:, 3:]]
    x, res, dy, target = new(M, 16, seed=4), new(M, 32, seed=5), new(M, 32, seed=6), torch.arange(M, device=device)
    want = None
    for place in places:
        a, r = (place(t).detach().requires_grad_() for t in (x, res))
        y = ops.gated_mlp(a, w1, None, w2, None, "silu", r)
        got = [y.detach(), *torch.autograd.grad(y, [a, r], place(dy))]
        loss = ops.linear_cross_entropy(a, w3, target)
        got += [loss.detach(), *torch.autograd.grad(loss, a)]
        want = want or got
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("M,K,H,N", [(2, 65, 109, 430), (1413, 4, 4, 35), (70, 24, 27, 16), (9, 5, 16, 13), (40, 12, 33, 2050)],
                         ids=str)
def test_gradients_of_odd_widths(M, K, H, N, device):
    """The gradient of h is not rounded on its way to gate's and up's, whatever the widths."""
    new = lambda *s, seed, std=1.0: normal(*s, device=device, dtype=torch.bfloat16, seed=seed, std=std).requires_grad_()
    x, w1, w2 = new(M, K, seed=1), new(2 * H, K, seed=2, std=1.5 * K ** -0.5), new(N, H, seed=3, std=H ** -0.5)
    dy = new(M, N, seed=4).detach()
    u = U[torch.bfloat16]
    want = mlp64(x, w1, None, w2, None, None, dy, "silu", u)
    y = ops.gated_mlp(x, w1, None, w2, None)
    for got, w in zip(torch.autograd.grad(y, [x, w1, w2], dy), want[1:]):
        within(got, *w)
    # of one row that has one value, 1: gate and up are columns of w1, exactly, and gradients of biases those of gate and up
    one = torch.zeros(1, K, device=device, dtype=torch.bfloat16)
    one[0, K // 2] = 1.0
    b1 = torch.zeros(2 * H, device=device, dtype=torch.bfloat16, requires_grad=True)
    (db,) = torch.autograd.grad(ops.gated_mlp(one, w1, b1, w2, None), b1, dy[:1])
    dh, dhm = ((f(dy[:1].double()) @ f(w2.detach().double()))[0] for f in (lambda t: t, torch.abs))
    gate, up = w1.detach()[:, K // 2].double().view(2, H)
    a, slope = act64(gate, "silu")
    edh = sums(N) * dhm
    within(db, torch.cat([dh * up * slope, dh * a]), torch.cat([
        up.abs() * (edh * 1.2 + dh.abs() * 1e-6 * (1 + gate.abs())), edh * a.abs() + dh.abs() * 1e-6 * (1 + gate.abs())]))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("K,H,N", [(16, 24, 32), (88, 33, 896), (13, 16, 24), (24, 9, 5)], ids=str)
def test_weights_that_lie_anywhere(K, H, N, device):
    """Transposed ones, every other row of a matrix, and ones that start off 16 bytes."""
    new = lambda *s, seed: normal(*s, device=device, dtype=torch.bfloat16, seed=seed, std=0.2)
    x, w1, w2, dy = new(5, K, seed=1), new(2 * H, K, seed=2), new(N, H, seed=3), new(5, N, seed=4)
    x.requires_grad_()
    places = [lambda t: t, lambda t: t.t().contiguous().t(),
              lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape),
              lambda t: torch.stack([t, t], 1).view(-1, t.shape[1])[::2],
              lambda t: torch.cat([t, t], 1)[:, :t.shape[1]]]
    want = None
    for place in places:
        a, b = (place(t).detach().requires_grad_() for t in (w1, w2))
        y = ops.gated_mlp(x, a, None, b, None)
        got = [y.detach(), *torch.autograd.grad(y, [x, a, b], dy)]
        want = want or got
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("through", ["C++", "Python"])
def test_rows_that_stand_for_several(through, device, monkeypatch):
    """Operands that are one row, expanded, or rows that overlap: as the rows written out."""
    if through == "Python":
        monkeypatch.setattr(_lib, "_eager", None)
        monkeypatch.setattr(_lib, "eager", lambda: None)
    new = lambda *s, seed: normal(*s, device=device, dtype=torch.bfloat16, seed=seed, std=0.3)
    wide = lambda n, d, seed: new(8 * n + d, seed=seed).as_strided((n, d), (8, 1))
    one = lambda n, d, seed: new(1, d, seed=seed).expand(n, d)
    target = torch.arange(6, device=device)
    for make in (wide, one):
        ops_in = [make(*s, seed=i) for i, s in enumerate(((6, 32), (48, 32), (16, 24), (6, 16), (40, 32)))]
        got = []
        for x, w1, w2, res, head in (ops_in, [t.contiguous() for t in ops_in]):
            x, w1, w2, res, head = (t.detach().requires_grad_() for t in (x, w1, w2, res, head))
            y = ops.gated_mlp(x, w1, None, w2, None, "silu", res)
            loss = ops.linear_cross_entropy(x, head, target)
            got.append([y.detach(), loss.detach(), *torch.autograd.grad(y, [x, w1, w2, res], one(6, 16, 9)),
                        *torch.autograd.grad(loss, [x, head])])
        assert all(torch.equal(a, b) for a, b in zip(*got))
