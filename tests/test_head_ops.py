"""Rotations of every layout and the norm of queries and keys in front of them, against their formulas in 64 bits.

Bounds.  u is half a step of the result's type; an fp32 operation is off by 2^-24 of its value.  A rotated value
a c - b s is two products and a sum: 3 * 2^-24 (|a c| + |b s|) at most before it is rounded.  Normed values carry the
error of a mean over D squares, at most (D + 8) 2^-24 of the value.  A gradient has two such factors, a mean over D
products and a rotation before them: (3 D + 32) 2^-24 of the sum of the magnitudes of its terms.  Sums over n rows
add n 2^-24 of the sum of magnitudes."""
import math

import pytest
import torch

from pfeife_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}
E = 2.0 ** -24
EPS = 1e-6


def within(got, want, magnitude, factor):
    """|got - want| <= u |want| + factor 2^-24 magnitude, element by element"""
    u = U[got.dtype]
    bound = u * want.abs() + (1 + u) * factor * E * magnitude + TINY[got.dtype]
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all() and (off <= bound).all(), float((off / bound).max())


def turned(x, cos, sin, pos, interleaved, sign=1, magnitude=False):
    """The rotation in 64 bits by indexing each pair; with `magnitude` the sums of magnitudes."""
    half = cos.shape[1]
    rows = pos if pos.dim() == 2 else pos.expand(x.shape[0], -1)
    c, s = cos.double()[rows][:, :, None], sign * sin.double()[rows][:, :, None]
    i = torch.arange(half, device=x.device)
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    out = x.abs().clone() if magnitude else x.clone()
    a, b = x[..., ia], x[..., ib]
    if magnitude:
        out[..., ia], out[..., ib] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    else:
        out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
    return out


def norm_turn(x, w, g, *where):
    """(y, its magnitudes, dx, its magnitudes, dw, its magnitudes) in 64 bits"""
    x, w, g = x.double(), w.double(), g.double()
    r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
    xh = x * r
    back, mag = turned(g, *where, sign=-1), turned(g, *where, sign=-1, magnitude=True)
    gw, gm = back * w, mag * w.abs()
    dx = r * (gw - xh * (gw * xh).mean(-1, keepdim=True))
    dxm = r * (gm + xh.abs() * (gm * xh.abs()).mean(-1, keepdim=True))
    return (turned(xh * w, *where), turned(xh * w, *where, magnitude=True), dx, dxm, (back * xh).sum((0, 1, 2)),
            (mag * xh.abs()).sum((0, 1, 2)))


def heads(B, S, H, D, device, dtype, seed, layout="packed"):
    """Normal values [B, S, H, D] in several orders of memory."""
    g = torch.Generator().manual_seed(seed)
    new = lambda *s: torch.randn(*s, generator=g).to(device=device, dtype=dtype)
    if layout == "slice":                        # some heads of a wider projection
        return new(B, S, H + 3, D)[:, :, 2:2 + H]
    if layout == "heads first":
        return new(B, H, S, D).transpose(1, 2)
    if layout == "seq first":
        return new(S, B, H, D).transpose(0, 1)
    if layout == "off by one":                   # on no boundary but the elements'
        return new(B * S * H * D + 1)[1:].view(B, S, H, D)
    if layout == "columns":                      # D is not innermost
        return new(B, S, D, H).transpose(2, 3)
    return new(B, S, H, D)


def angles(rows, half, device, seed=0):
    a = torch.rand(rows, half, generator=torch.Generator().manual_seed(seed)) * 6.3
    return a.cos().to(device), a.sin().to(device)


def rows_of(kind, B, S, T, device):
    g = torch.Generator().manual_seed(S)
    if kind == "each":
        return torch.randint(0, T, (B, S), generator=g).to(device)
    if kind == "int32":
        return torch.randint(0, T, (S,), generator=g).to(device=device, dtype=torch.int32)
    if kind == "strided":
        return torch.randint(0, T, (S, B), generator=g).to(device).t()
    return None


# (B, S, H, D, R): whole and partial heads of every vector width, odd D, one token, more heads than an item
SHAPES = [(1, 1, 1, 2, 2), (2, 5, 3, 7, 4), (1, 3, 2, 16, 16), (2, 33, 5, 64, 64), (1, 17, 9, 96, 24),
          (3, 7, 2, 72, 72), (2, 9, 4, 36, 36), (1, 11, 6, 88, 40), (1, 4, 1, 256, 256), (1, 3, 2, 250, 6),
          (2, 130, 13, 128, 64), (1, 5, 2, 300, 300)]
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
LAYOUTS = ["packed", "slice", "heads first", "seq first", "off by one", "columns"]


def _cases():
    kinds = [None, "each", "int32", "strided"]
    out, n = [], 0
    for shape in SHAPES:
        for dtype in DTYPES:
            for interleaved in (False, True):
                out.append((*shape, dtype, interleaved, LAYOUTS[n % 6], kinds[n // 2 % 4]))
                n += 1
    return out


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("B,S,H,D,R,dtype,interleaved,layout,kind", _cases(), ids=str)
def test_rope_of_every_layout(B, S, H, D, R, dtype, interleaved, layout, kind, device):
    T = S + 6
    cos, sin = angles(T, R // 2, device)
    x = heads(B, S, H, D, device, dtype, 1, layout).requires_grad_()
    dy = heads(B, S, H, D, device, dtype, 2, LAYOUTS[(LAYOUTS.index(layout) + 1) % 6])
    pos = rows_of(kind, B, S, T, device)
    at = torch.arange(S, device=device) if pos is None else pos.long()
    y = ops.rope(x, cos, sin, positions=pos, interleaved=interleaved)
    (dx,) = torch.autograd.grad(y, x, dy)
    assert y.dtype == dx.dtype == dtype and y.is_contiguous()
    where = (cos, sin, at, interleaved)
    within(y.detach(), turned(x.detach().double(), *where), turned(x.detach().double(), *where, magnitude=True), 3)
    within(dx, turned(dy.double(), *where, sign=-1), turned(dy.double(), *where, sign=-1, magnitude=True), 3)
    assert torch.equal(y[..., R:], x[..., R:]) and torch.equal(dx[..., R:], dy[..., R:])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("B,S,H,D,R,dtype,interleaved,layout,kind", _cases()[::2] + _cases()[1::6], ids=str)
def test_qk_norm_rope(B, S, H, D, R, dtype, interleaved, layout, kind, device):
    """Queries of more heads than keys."""
    T = S + 6
    cos, sin = angles(T, R // 2, device)
    q = heads(B, S, 2 * H + 1, D, device, dtype, 1, layout).requires_grad_()
    k = heads(B, S, H, D, device, dtype, 2, layout).requires_grad_()
    gq, gk = (heads(*t.shape, device, dtype, 5 + i, "slice") for i, t in enumerate((q, k)))
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=torch.Generator().manual_seed(i))).to(device).requires_grad_()
              for i in (3, 4))
    pos = rows_of(kind, B, S, T, device)
    at = torch.arange(S, device=device) if pos is None else pos.long()
    out = ops.qk_norm_rope(q, k, wq, wk, cos, sin, EPS, positions=pos, interleaved=interleaved)
    grads = torch.autograd.grad(out, [q, k, wq, wk], [gq, gk])
    for i, (x, w, g) in enumerate(((q, wq, gq), (k, wk, gk))):
        y, ym, dx, dxm, dw, dwm = norm_turn(x.detach(), w.detach(), g, cos, sin, at, interleaved)
        within(out[i].detach(), y, ym, D + 8)
        within(grads[i], dx, dxm, 3 * D + 32)
        within(grads[2 + i], dw, dwm, B * S * x.shape[2] + D + 32)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("B,S,H,D,R,dtype,interleaved", [
    (2, 19, 3, 64, 64, torch.bfloat16, False), (1, 2, 1, 2, 2, torch.float16, True), (2, 70, 9, 128, 32, torch.bfloat16, True),
    (1, 33, 5, 72, 72, torch.float32, False), (3, 5, 2, 33, 32, torch.float16, False), (1, 4, 2, 264, 8, torch.bfloat16, True)], ids=str)
def test_fused_projections(norm, B, S, H, D, R, dtype, interleaved, device):
    """The values of a projection and of its gradient keep their bits, infinities and NaN among them."""
    cos, sin = angles(S, R // 2, device)
    pos = torch.randint(0, S, (B, S), generator=torch.Generator().manual_seed(1)).to(device)
    qkv, dy = (heads(B, S, 3 * H, D, device, dtype, i).view(B, S, 3, H, D) for i in (1, 2))
    for t in (qkv, dy):
        t[:, :, 2, :, 0], t[:, 0, 2, 0, 1] = math.inf, math.nan
    qkv.requires_grad_()
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=torch.Generator().manual_seed(i))).to(device).requires_grad_()
              for i in (3, 4))
    if norm:
        y = ops.qk_norm_rope_qkv(qkv, wq, wk, cos, sin, EPS, positions=pos, interleaved=interleaved)
        grads = torch.autograd.grad(y, [qkv, wq, wk], dy)
    else:
        y = ops.rope_qkv(qkv, cos, sin, positions=pos, interleaved=interleaved)
        grads = torch.autograd.grad(y, [qkv], dy)
    same = lambda a, b: torch.equal(torch.nan_to_num(a, nan=7.0), torch.nan_to_num(b, nan=7.0))
    assert same(y[:, :, 2], qkv[:, :, 2]) and same(grads[0][:, :, 2], dy[:, :, 2])
    where = (cos, sin, pos, interleaved)
    for i, w in enumerate((wq, wk)):
        x, g = qkv.detach()[:, :, i], dy[:, :, i]
        if norm:
            want, mag, dx, dxm, dw, dwm = norm_turn(x, w.detach(), g, *where)
            within(grads[1 + i], dw, dwm, B * S * H + D + 32)
        else:
            want, mag = turned(x.double(), *where), turned(x.double(), *where, magnitude=True)
            dx, dxm = turned(g.double(), *where, sign=-1), turned(g.double(), *where, sign=-1, magnitude=True)
        within(y.detach()[:, :, i], want, mag, D + 8 if norm else 3)
        within(grads[0][:, :, i], dx, dxm, 3 * D + 32 if norm else 3)


def test_gradients_are_those_of_differences():
    """In 64 bits, where the formulas are the kernels' (the kernels have no such type)."""
    torch.manual_seed(0)
    cos, sin = (t.double() for t in angles(9, 3, "cpu"))
    pos = torch.tensor([[0, 8, 2], [5, 5, 1]])
    q, k = (torch.randn(2, 3, h, 8, dtype=torch.float64, requires_grad=True) for h in (4, 2))
    wq, wk = (torch.randn(8, dtype=torch.float64, requires_grad=True) for _ in range(2))
    for interleaved in (False, True):
        assert torch.autograd.gradcheck(lambda x: ops.rope(x, cos, sin, pos, interleaved), [q])
        assert torch.autograd.gradcheck(
            lambda *a: ops.qk_norm_rope(*a, cos, sin, 1e-3, pos, interleaved), [q, k, wq, wk])
        qkv = torch.randn(2, 3, 3, 2, 8, dtype=torch.float64, requires_grad=True)
        assert torch.autograd.gradcheck(
            lambda x, a, b: ops.qk_norm_rope_qkv(x, a, b, cos, sin, 1e-3, pos, interleaved), [qkv, wq, wk])


@pytest.mark.parametrize("device", DEVICES)
def test_heads_of_zeros_and_of_large_values(device):
    """A head of zeros has r = eps^-1/2; squares of fp16's largest values do not overflow the sums."""
    cos, sin = angles(4, 8, device)
    x = torch.zeros(1, 4, 2, 16, device=device, dtype=torch.float16)
    x[:, 1] = 65504.0
    x[:, 2] = -65504.0
    x.requires_grad_()
    w = torch.ones(16, device=device)
    y, _ = ops.qk_norm_rope(x, x, w, w, cos, sin, EPS)
    g = torch.ones_like(y)
    (dx,) = torch.autograd.grad(y, x, g)
    assert not y[:, 0].any() and not y[:, 3].any()
    want = norm_turn(x.detach(), w, g, cos, sin, torch.arange(4, device=device), False)
    within(y.detach(), want[0], want[1], 24)
    within(dx, want[2], want[3], 80)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shape", [(0, 3, 2, 16), (2, 0, 2, 16), (2, 3, 0, 16)])
def test_no_heads_at_all(device, shape):
    cos, sin = angles(4, 8, device)
    x = torch.zeros(shape, device=device, dtype=torch.bfloat16).requires_grad_()
    k = torch.zeros(*shape[:2], 1, 16, device=device, dtype=torch.bfloat16).requires_grad_()
    w = torch.ones(16, device=device, requires_grad=True)
    y = ops.rope(x, cos, sin, interleaved=True)
    assert y.shape == shape and torch.autograd.grad(y, x, y)[0].shape == shape
    q, k2 = ops.qk_norm_rope(x, k, w, w, cos, sin)
    dx, dw = torch.autograd.grad([q, k2], [x, w], [torch.ones_like(q), torch.zeros_like(k2)])
    assert dx.shape == shape and not dw.any()
    none = x[:, :, :0]
    q, k2 = ops.qk_norm_rope(none, none, w, w, cos, sin)
    assert not torch.autograd.grad([q, k2], w, [q, k2])[0].any()


@pytest.mark.parametrize("device", DEVICES)
def test_one_gradient_of_two_and_gradients_that_are_broadcast(device):
    cos, sin = angles(6, 8, device)
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    q, k = (heads(2, 6, h, 16, device, dtype, h).requires_grad_() for h in (4, 2))
    w = (torch.rand(16) + 0.5).to(device).requires_grad_()          # one gain for both
    for use in ((1, 0), (0, 1), (1, 1)):
        out = ops.qk_norm_rope(q, k, w, w, cos, sin)
        loss = sum(u * t.float().sum() for u, t in zip(use, out) if u)
        dq, dk, dw = torch.autograd.grad(loss, [q, k, w], allow_unused=True)
        total, most = 0.0, 0.0
        for u, x, d in ((use[0], q, dq), (use[1], k, dk)):
            g = torch.full_like(x, float(u))
            want = norm_turn(x.detach(), w.detach(), g, cos, sin, torch.arange(6, device=device), False)
            within(d, want[2], want[3], 80)
            total, most = total + want[4], most + want[5]
        within(dw, total, most, 2 * 6 * 4 + 50)


@pytest.mark.parametrize("device", DEVICES)
def test_tables_that_are_longer_or_in_another_order(device):
    dtype = torch.float32 if device == "cpu" else torch.float16
    cos, sin = angles(40, 8, device)
    x = heads(2, 9, 3, 16, device, dtype, 1)
    want = ops.rope(x, cos[:9].contiguous(), sin[:9].contiguous(), interleaved=True)
    assert torch.equal(ops.rope(x, cos, sin, interleaved=True), want)
    assert torch.equal(ops.rope(x, cos.t().contiguous().t(), sin.half().float().copy_(sin), interleaved=True), want)
    wide = torch.cat([cos, sin], 1)
    assert torch.equal(ops.rope(x, wide[:, :8], wide[:, 8:], interleaved=True), want)
    odd = torch.cat([cos.new_zeros(1), cos.flatten()])[1:].view(40, 8)          # 4 bytes off a vector
    assert torch.equal(ops.rope(x, odd, sin, interleaved=True), want)
    # the first rows, by number
    assert torch.equal(ops.rope(x, cos, sin, torch.arange(9, device=device), True), want)
    assert torch.equal(ops.rope(x, cos, sin), ops.rope(x, cos, sin, torch.arange(9, device=device)))


def test_positions_outside_the_tables_on_the_cpu():
    cos, sin = angles(5, 8, "cpu")
    x = torch.zeros(1, 3, 2, 16)
    for bad in (-1, 5, 1 << 40):
        with pytest.raises(IndexError, match="outside"):
            ops.rope(x, cos, sin, positions=torch.tensor([0, bad, 1]))


@pytest.mark.gpu
def test_positions_outside_the_tables_on_cuda():
    """The kernel looks at them before it reads: NaN in those tokens, every other one as it was."""
    cos, sin = angles(5, 4, "cuda")
    x = heads(2, 3, 2, 16, "cuda", torch.bfloat16, 1)
    pos = torch.tensor([[0, 5, 1], [4, -1, 1 << 40]], device="cuda")
    y = ops.rope(x, cos, sin, positions=pos)
    bad = (pos < 0) | (pos > 4)
    assert torch.isnan(y[bad][..., :8]).all() and torch.equal(y[bad][..., 8:], x[bad][..., 8:])
    good = ops.rope(x, cos, sin, positions=pos.clamp(0, 4))
    assert torch.equal(y[~bad], good[~bad])


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    cos, sin = angles(8, 8, device)
    x = torch.zeros(2, 4, 2, 16, device=device, dtype=torch.bfloat16)
    w = torch.ones(16, device=device)
    other = "meta" if device == "cpu" else "cpu"
    for tables, pos in (((cos[:3], sin[:3]), None), ((cos, sin[:7]), None), ((cos.flatten(), sin.flatten()), None),
                        ((torch.zeros(8, 9, device=device),) * 2, None), ((cos[:, :0], sin[:, :0]), None),
                        ((cos.to(other), sin.to(other)), None), ((cos, sin), torch.zeros(3, dtype=torch.int64)),
                        ((cos, sin), torch.zeros(4)), ((cos, sin), torch.zeros(1, 4, dtype=torch.int64)),
                        ((cos, sin), torch.zeros(4, dtype=torch.int64, device=other))):
        if pos is not None and pos.device.type == "cpu" and pos.device.type != other:
            pos = pos.to(device)
        with pytest.raises(ValueError):
            ops.rope(x, *tables, positions=pos, interleaved=True)
        with pytest.raises(ValueError):
            ops.qk_norm_rope(x, x, w, w, *tables, positions=pos)
    for q, k in ((x, x[:1]), (x, x[:, :3]), (x, x[..., :8]), (x, x.float()), (x[0], x[0])):
        with pytest.raises(ValueError):
            ops.qk_norm_rope(q, k, w, w, cos, sin)
    with pytest.raises(ValueError):
        ops.qk_norm_rope(x, x, w, w[:8], cos, sin)
    with pytest.raises(ValueError):
        ops.qk_norm_rope(x, x, w, w.to(other), cos, sin)
    with pytest.raises(ValueError):
        ops.qk_norm_rope_qkv(torch.stack([x, x], 2), w, w, cos, sin)
    with pytest.raises(ValueError):
        ops.rope(x, cos[:, :4], sin[:3, :4])                     # a partial rotation of too few rows
    with pytest.raises(ValueError):
        ops.rope(x, cos[:0], sin[:0], torch.zeros(4, dtype=torch.int64, device=device))
    packed = torch.stack([x, x, x], 2)
    for wrong, call in ((packed, ops.rope), (x, ops.rope_qkv), (packed[:, :, :2], ops.rope_qkv), (x[0], ops.rope)):
        with pytest.raises(ValueError):
            call(wrong, cos, sin, interleaved=True)
    from pfeife_b200.models.llama import Llama, llama_config
    for dim in (7, 0, 18):
        with pytest.raises(ValueError):
            Llama(llama_config("llama_tiny", rope_dim=dim))


# ------------------------------------------------------------------------------ scaled tables
def _frequency(kind, i, R, theta, factor, L):
    f = theta ** (-2.0 * i / R)
    if kind == "linear":
        return f / factor
    if kind == "ntk":
        return (theta * factor ** (R / (R - 2))) ** (-2.0 * i / R)
    if kind == "yarn":
        at = lambda turns: R * math.log(L / (2 * math.pi * turns)) / (2 * math.log(theta))
        low, high = max(0, math.floor(at(32))), min(R - 1, math.ceil(at(1)))
        ramp = min(1.0, max(0.0, (i - low) / max(high - low, 1e-3)))
        return f / factor * ramp + f * (1 - ramp)
    wave = 2 * math.pi / f
    if wave < L / 4:
        return f
    if wave > L:
        return f / factor
    smooth = (L / wave - 1) / 3
    return (1 - smooth) * f / factor + smooth * f


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["linear", "ntk", "yarn", "bands"])
@pytest.mark.parametrize("R,factor,L", [(64, 4.0, 512), (128, 8.0, 2048), (6, 1.0, 16)])
def test_scaled_tables(kind, R, factor, L, device):
    """Far positions too: angles of thousands of radians keep their cosines."""
    rows = 40000
    cos, sin = ops.rope_tables(rows, R, 1e4, device, ops.RopeScaling(kind, factor, L))
    assert cos.shape == sin.shape == (rows, R // 2) and cos.dtype == torch.float32
    grown = 0.1 * math.log(factor) + 1 if kind == "yarn" else 1.0
    for p in (0, 1, L - 1, 39999):
        for i in range(R // 2):
            a = p * _frequency(kind, i, R, 1e4, factor, L)
            # an angle of 4e4 radians is off by 4e4 * 2^-50 in 64 bits, the value then rounded to 32
            assert abs(float(cos[p, i]) - grown * math.cos(a)) < 1.3 * 2 ** -24 * grown + 1e-9
            assert abs(float(sin[p, i]) - grown * math.sin(a)) < 1.3 * 2 ** -24 * grown + 1e-9


def test_scalings_that_are_refused():
    for bad in (ops.RopeScaling("cubic", 2.0), ops.RopeScaling("linear", 0.5), ops.RopeScaling("yarn", 2.0, 0),
                ops.RopeScaling("bands", 2.0, slow=0.0), ops.RopeScaling("yarn", 2.0, fast=1.0)):
        with pytest.raises(ValueError):
            ops.rope_tables(8, 16, scaling=bad)
    with pytest.raises(ValueError):
        ops.rope_tables(8, 2, scaling=ops.RopeScaling("ntk", 2.0))
    plain = ops.rope_tables(8, 16)
    assert all(torch.equal(a, b) for a, b in zip(plain, ops.rope_tables(8, 16, scaling=None)))


# ------------------------------------------------------------------------------ where and how it runs
@pytest.mark.gpu
def test_other_streams_and_graphs():
    """On a stream of its own, and captured with its backward and replayed on new data."""
    cos, sin = angles(64, 32, "cuda")
    w = torch.rand(64, device="cuda") + 0.5
    pos = torch.randint(0, 64, (2, 64), device="cuda")
    x, dy = (heads(2, 64, 3 * 5, 64, "cuda", torch.bfloat16, i).view(2, 64, 3, 5, 64) for i in (1, 2))

    def both(x, dy):
        from pfeife_b200.ops import functional as f
        y = ops.qk_norm_rope_qkv(x, w, w, cos, sin, EPS, positions=pos)
        return y, *f.qk_norm_rope_qkv_bwd(dy, x, w, w, cos, sin, pos, EPS, False)

    with torch.no_grad():
        want = both(x, dy)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = both(x, dy)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        sx, sdy = torch.zeros_like(x), torch.zeros_like(dy)
        graphs = []
        for _ in range(2):                       # two that do not share anything
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = both(sx, sdy)
            graphs.append((g, out))
        sx.copy_(x)
        sdy.copy_(dy)
        for g, _ in graphs + graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
def test_registered_gains_and_bits_that_repeat():
    """Gradients of registered gains are added to their buckets; the sums are made in a fixed order."""
    cos, sin = angles(700, 32, "cuda")
    q, k = (heads(3, 700, h, 64, "cuda", torch.bfloat16, h).requires_grad_() for h in (8, 4))
    wq, wk = (torch.rand(64, device="cuda").requires_grad_() for _ in range(2))
    grads = lambda: torch.autograd.grad(ops.qk_norm_rope(q, k, wq, wk, cos, sin), [q, k, wq, wk], [q.detach(), k.detach()],
                                        allow_unused=True)
    first = grads()
    assert all(torch.equal(a, b) for a, b in zip(first, grads()))
    buckets = [torch.full((64,), 3.0, device="cuda") for _ in range(2)]
    try:
        for w, b in zip((wq, wk), buckets):
            ops.register_param(w, None, b)
        again = grads()
    finally:
        ops.unregister_params()
    assert again[2] is None and again[3] is None
    for b, d in zip(buckets, first[2:]):
        assert torch.equal(b, 3.0 + d)
    assert all(torch.equal(a, b) for a, b in zip(again[:2], first[:2]))


@pytest.mark.gpu
def test_one_registered_gain_for_queries_and_keys():
    """Both sums reach the one gradient, neither overtaken by the other."""
    cos, sin = angles(300, 32, "cuda")
    q, k = (heads(2, 300, h, 64, "cuda", torch.bfloat16, h) for h in (8, 4))
    w = torch.rand(64, device="cuda").requires_grad_()
    def grad():
        out = ops.qk_norm_rope(q, k, w, w, cos, sin)
        return torch.autograd.grad(out, w, [q, k])[0]
    want = grad()
    bucket = torch.zeros(64, device="cuda")
    try:
        ops.register_param(w, None, bucket)
        got = [grad() for _ in range(3)]
    finally:
        ops.unregister_params()
    assert not bucket.any() and all(torch.equal(g, want) for g in got)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,heads_q", [(1, 1), (3, 2), (131072, 1), (4097, 33)])
def test_many_tokens_and_many_heads(tokens, heads_q):
    """Every item of the grid and of the backward's walks, one CTA to many."""
    cos, sin = angles(tokens, 8, "cuda")
    q = torch.randn(1, tokens, heads_q, 16, device="cuda").bfloat16().requires_grad_()
    k = torch.randn(1, tokens, 1, 16, device="cuda").bfloat16().requires_grad_()
    w = torch.ones(16, device="cuda", requires_grad=True)
    out = ops.qk_norm_rope(q, k, w, w, cos, sin)
    g = [torch.randn_like(t) for t in out]
    dq, dk, dw = torch.autograd.grad(out, [q, k, w], g)
    at, total, most = torch.arange(tokens, device="cuda"), 0.0, 0.0
    for x, y, d, go in ((q, out[0], dq, g[0]), (k, out[1], dk, g[1])):
        want = norm_turn(x.detach(), w.detach(), go, cos, sin, at, False)
        within(y.detach(), want[0], want[1], 24)
        within(d, want[2], want[3], 80)
        total, most = total + want[4], most + want[5]
    within(dw, total, most, tokens * (heads_q + 1) + 80)


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Heads of a projection whose elements lie further than 2^31 apart."""
    S, H, D = 33000, 520, 128                    # 2.2e9 elements
    wide = torch.empty(1, S, H, D, device="cuda", dtype=torch.bfloat16)
    x = wide[:, :, H - 3:]
    x.normal_()
    cos, sin = angles(S, 64, "cuda")
    y = ops.rope(x, cos, sin, interleaved=True)
    tail = slice(S - 50, S)
    want = ops.rope(x[:, tail].contiguous(), cos[tail], sin[tail], interleaved=True)
    assert torch.equal(y[:, tail], want)


@pytest.mark.parametrize("device", DEVICES)
def test_ops_are_seen_by_tracers_and_modes(device):
    """The registered ops pass PyTorch's checks of schemas, fakes and autograd formulas, and a compiled call is
    one of them."""
    from pfeife_b200.ops import functional as f
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    cos, sin = angles(6, 4, device)
    w = torch.ones(16, device=device)
    pos = torch.arange(6, device=device).flip(0)
    x = heads(2, 6, 4, 16, device, dtype, 1).requires_grad_()
    qkv = heads(2, 6, 6, 16, device, dtype, 2).view(2, 6, 3, 2, 16).requires_grad_()
    checks = ("test_schema", "test_faketensor", "test_autograd_registration")
    torch.library.opcheck(f.rope_at, (x, cos, sin, pos, True, False), test_utils=checks)
    torch.library.opcheck(f.rope_qkv_at, (qkv, cos, sin, None, False, False), test_utils=checks)
    torch.library.opcheck(f.qk_norm_rope_fwd, (x, x, w, w, cos, sin, pos, EPS, True), test_utils=checks)
    torch.library.opcheck(f.qk_norm_rope_qkv_fwd, (qkv, w, w, cos, sin, None, EPS, False), test_utils=checks)
    fn = lambda t: ops.qk_norm_rope_qkv(t, w, w, cos, sin, EPS, positions=pos, interleaved=True)
    want = fn(qkv)
    got = torch.compile(fn, backend="eager", fullgraph=True)(qkv)
    assert torch.equal(got, want)
    g = torch.ones_like(want)
    assert torch.equal(torch.autograd.grad(got, qkv, g)[0], torch.autograd.grad(want, qkv, g)[0])
    gm = torch.fx.symbolic_trace(lambda t: ops.rope(t, cos, sin, pos, True))
    assert torch.equal(gm(x), ops.rope(x, cos, sin, pos, True))


# ------------------------------------------------------------------------------ calls that do not go the usual way
class Watch(torch.utils._python_dispatch.TorchDispatchMode):
    """Lets every op be seen, which keeps all calls on the dispatcher."""

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


def _functions(device):
    """name -> (function of the leaves, leaves)"""
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    cos, sin = angles(16, 8, device)
    pos = torch.randint(0, 16, (2, 16), generator=torch.Generator().manual_seed(1)).to(device)
    new = lambda h, seed: heads(2, 16, h, 16, device, dtype, seed)
    gain = lambda seed: (torch.rand(16, generator=torch.Generator().manual_seed(seed)) + 0.5).to(device)
    return {
        "rope": (lambda x: ops.rope(x, cos, sin, pos), [new(3, 1)]),
        "interleaved": (lambda x: ops.rope(x, cos, sin, interleaved=True), [new(3, 1)]),
        "partial": (lambda x: ops.rope(x, cos[:, :3].contiguous(), sin[:, :3].contiguous()), [new(3, 1)]),
        "rope_qkv": (lambda x: ops.rope_qkv(x, cos, sin, pos, True), [new(6, 1).view(2, 16, 3, 2, 16)]),
        "qk_norm_rope": (lambda q, k, a, b: torch.cat(ops.qk_norm_rope(q, k, a, b, cos, sin, 1e-5, pos), 2),
                         [new(4, 1), new(2, 2), gain(1), gain(2)]),
        "qk_norm_rope_qkv": (lambda x, a, b: ops.qk_norm_rope_qkv(x, a, b, cos, sin, 1e-5, pos, True),
                             [new(6, 1).view(2, 16, 3, 2, 16), gain(1), gain(2)]),
    }


NAMES = ["rope", "interleaved", "partial", "rope_qkv", "qk_norm_rope", "qk_norm_rope_qkv"]


@pytest.fixture(params=DEVICES)
def direct_device(request, monkeypatch):
    """On the CPU the direct way is switched on too."""
    from pfeife_b200.ops import functional
    monkeypatch.setattr(functional, "_FIRST_DEVICE", -1 if request.param == "cpu" else 0)
    return request.param


@pytest.mark.parametrize("name", NAMES)
def test_direct_calls_and_the_dispatcher_agree(name, direct_device):
    fn, leaves = _functions(direct_device)[name]
    leaves = [t.requires_grad_() for t in leaves]
    y = fn(*leaves)
    g = torch.randn(y.shape, generator=torch.Generator().manual_seed(3)).to(y)
    want = torch.autograd.grad(y, leaves, g, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, g), want))     # a second time
    with Watch():
        seen = fn(*leaves)
        got = torch.autograd.grad(seen, leaves, g)
    assert torch.equal(y, seen) and all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad():
        assert torch.equal(fn(*leaves), y) and not fn(*leaves).requires_grad
    y = fn(*leaves)
    y.mul_(2.0)                                    # no view to autograd: may be changed in place
    for a, b in zip(torch.autograd.grad(y, leaves, g / 2), want):
        assert torch.allclose(a, b, rtol=2e-2, atol=2e-2)


@pytest.mark.parametrize("name", NAMES)
def test_saved_tensors_of_other_types_and_orders(name, direct_device):
    """Hooks on saved tensors may return any tensor of the same values."""
    fn, leaves = _functions(direct_device)[name]
    leaves = [t.requires_grad_() for t in leaves]
    y = fn(*leaves)
    g = torch.ones_like(y)
    want = torch.autograd.grad(y, leaves, g)

    def unpack(t):
        if t.is_floating_point():                  # every second element of a wider tensor, or 64 bits
            return torch.stack([t, t], -1)[..., 0] if t.dim() > 1 else t.double()
        return t

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        y = fn(*leaves)
    for a, b in zip(torch.autograd.grad(y, leaves, g), want):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)
    from torch.utils.checkpoint import checkpoint
    y = checkpoint(fn, *leaves, use_reentrant=False)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, g), want))


def test_entry_points_refuse_what_they_cannot_read():
    """Before anything touches a device."""
    import ctypes
    from pfeife_b200.csrc import build
    from pfeife_b200.ops import _lib
    if not build.KERNEL_LIB.exists():
        pytest.skip("the kernel library is not built")
    calls = _lib.load_calls(ctypes.CDLL(str(build.KERNEL_LIB), mode=ctypes.RTLD_GLOBAL))
    t = torch.zeros(64).data_ptr()
    z = (64, 64, 16)

    def fwd(q=t, B=1, S=1, Hq=1, Hk=0, D=16, R=16, cos=t, pos=None, dtype=2):
        return calls.pf_heads_fwd(q, None, None, t, None, None, None, None, cos, t, pos, B, S, Hq, Hk, D, R, z, None,
                                  z, None, (0, 1), 1, 0, 0, 1e-6, dtype, 148, None)
    assert fwd(dtype=5) == -1
    for bad in (dict(D=257), dict(D=300, R=300), dict(R=17), dict(R=18), dict(R=0), dict(D=0), dict(S=1 << 30, B=4),
                dict(S=1 << 24, Hq=256)):
        assert fwd(**bad) == -3, bad
    for bad in (dict(q=t + 1), dict(cos=t + 2), dict(pos=t + 4), dict(q=t + 2, dtype=0)):
        assert fwd(**bad) == -2, bad
    for empty in (dict(B=0), dict(S=0), dict(Hq=0)):
        assert fwd(**empty) == 0, empty
    assert calls.pf_heads_bwd_rows(32, 8, 148) >= 2 * 148


def test_scalings_whose_ramp_would_run_backwards():
    """The defaults of ``fast`` are held to the same order as a value that is given, and nothing that is no number
    becomes a table."""
    S = ops.RopeScaling
    for bad in (S("bands", 2.0, slow=8.0), S("bands", 2.0, slow=4.0), S("yarn", 2.0, slow=64.0), S("yarn", 2.0, slow=32.0),
                S("bands", 2.0, fast=0.0), S("linear", math.nan), S("ntk", math.inf), S("yarn", 2.0, fast=math.nan),
                S("yarn", 2.0, grown=math.inf), S("bands", 2.0, slow=math.nan), S("linear", 2.0, math.nan)):
        with pytest.raises(ValueError, match="RopeScaling"):
            ops.rope_tables(8, 16, scaling=bad)
    for kind, theta in (("yarn", 1.0), ("yarn", 0.5), ("linear", 0.0), ("bands", -2.0), ("ntk", math.nan)):
        with pytest.raises(ValueError, match="base"):
            ops.rope_tables(8, 16, theta, scaling=S(kind, 2.0))
    # an order that is right, with a value given or not: the fastest pair is kept, the slowest divided
    for good in (S("bands", 2.0, 64), S("bands", 2.0, 64, slow=3.5), S("bands", 2.0, 64, fast=8.0, slow=6.0)):
        cos, _ = ops.rope_tables(8, 16, scaling=good)
        assert abs(float(cos[1, 0]) - math.cos(1.0)) < 1e-7
        assert abs(float(cos[1, 7]) - math.cos(_frequency("linear", 7, 16, 1e4, 2.0, 64))) < 1e-7


@pytest.mark.parametrize("device", DEVICES)
def test_tables_that_want_a_gradient(device):
    """They get none, and are told so; where nothing is recorded they are tables as any other."""
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    tables = angles(6, 8, device)
    x = heads(2, 6, 3, 16, device, dtype, 1)
    qkv = heads(2, 6, 6, 16, device, dtype, 2).view(2, 6, 3, 2, 16)
    w, pos = torch.ones(16, device=device), torch.arange(6, device=device)
    calls = [lambda c, s: ops.rope(x, c, s, pos), lambda c, s: ops.rope(x, c, s, interleaved=True),
             lambda c, s: ops.rope(x, c[:, :4], s[:, :4]), lambda c, s: ops.rope_qkv(qkv, c, s, pos),
             lambda c, s: ops.qk_norm_rope(x, x, w, w, c, s), lambda c, s: ops.qk_norm_rope_qkv(qkv, w, w, c, s)]
    for i in range(2):
        wanted = [t.clone().requires_grad_(i == j) for j, t in enumerate(tables)]
        for call in calls:
            for leaf in (x, qkv):
                leaf.requires_grad_(i == 1)
            with pytest.raises(ValueError, match="no gradient"):
                call(*wanted)
            with torch.no_grad():
                got, want = call(*wanted), call(*tables)
            for a, b in zip(got, want):
                assert torch.equal(a, b) and not a.requires_grad


def test_the_backward_entry_point_refuses_what_it_cannot_write():
    """Both gains' gradients and the rows that their sums need are the caller's; a part without heads has no row."""
    import ctypes
    from pfeife_b200.csrc import build
    from pfeife_b200.ops import _lib
    if not build.KERNEL_LIB.exists():
        pytest.skip("the kernel library is not built")
    calls = _lib.load_calls(ctypes.CDLL(str(build.KERNEL_LIB), mode=ctypes.RTLD_GLOBAL))
    t = torch.zeros(64).data_ptr()
    z = (64, 64, 16)

    def bwd(wq=t, wk=t, dwq=t, dwk=t, scratch=t, D=16, R=16, q=t, dtype=2):
        return calls.pf_heads_bwd(t, t, None, q, t, t, t, None, wq, wk, dwq, dwk, scratch, t, t, None, 1, 1, 1, 1, D, R,
                                  z, z, z, z, z, z, (0, 1), 1, 0, 1e-6, 0, dtype, 148, None)
    for missing in ("wq", "wk", "dwq", "dwk", "scratch"):
        assert bwd(**{missing: None}) == -3, missing
    assert bwd(dtype=4) == -1 and bwd(q=t + 1) == -2 and bwd(R=18) == -3 and bwd(D=258, R=2) == -3
    rows = [calls.pf_heads_bwd_rows(h, k, 148) for h, k in ((32, 8), (32, 0), (0, 0))]
    assert rows == [rows[2] + 2, rows[2] + 1, 2 * 148]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,hq,hk,D,R,dtype,interleaved,packed", [
    (131072, 1, 1, 16, 16, torch.bfloat16, False, False), (4097, 33, 1, 16, 16, torch.bfloat16, True, False),
    (2048, 32, 8, 128, 128, torch.bfloat16, False, False), (2049, 24, 6, 128, 64, torch.float16, True, False),
    (5003, 6, 2, 72, 72, torch.float32, False, False), (3001, 16, 16, 64, 64, torch.bfloat16, False, True),
    (1777, 9, 9, 90, 90, torch.float16, True, True)], ids=str)
def test_gains_gradients_over_many_rows(tokens, hq, hk, D, R, dtype, interleaved, packed):
    """The sums over all heads of long sequences, whose rounding grows with their depth and not with the number of
    rows.  A lane adds up its group's heads: at most two CTAs an SM, shared by queries and keys by their numbers, of 8
    groups or more; then 5 sums across a warp, 8 of warps, one for each 32 CTAs and 5 across a warp.  A term is off by
    D + 32 parts of 2^-24 of its magnitude, as elsewhere.  Rows are normal, so that a sum lies as far from 0 as the
    root of their number, beyond the bound: one that misses a CTA or a share of the fold does not pass."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    cos, sin = angles(tokens, R // 2, "cuda")
    torch.manual_seed(tokens)
    new = lambda *s: torch.randn(*s, device="cuda").to(dtype)
    wq, wk = ((1 + 0.3 * torch.randn(D, device="cuda")).requires_grad_() for _ in range(2))
    if packed:
        qkv, g = new(1, tokens, 3, hq, D), new(1, tokens, 3, hq, D)
        y = ops.qk_norm_rope_qkv(qkv, wq, wk, cos, sin, EPS, interleaved=interleaved)
        got = torch.autograd.grad(y, [wq, wk], g)
        parts = [(qkv[:, :, i], g[:, :, i]) for i in range(2)]
    else:
        parts = [(new(1, tokens, h, D), new(1, tokens, h, D)) for h in (hq, hk)]
        out = ops.qk_norm_rope(parts[0][0], parts[1][0], wq, wk, cos, sin, EPS, interleaved=interleaved)
        got = torch.autograd.grad(out, [wq, wk], [g for _, g in parts])
    total = hq + hk + (2 / 3 * hk if packed else 0)              # the values of a projection take CTAs too
    at = torch.arange(tokens, device="cuda")
    for (x, g), w, d in zip(parts, (wq, wk), got):
        want, most = norm_turn(x, w.detach(), g, cos, sin, at, interleaved)[4:]
        heads_here = x.shape[2]
        ctas = max(1.0, 2 * sms * heads_here / total - 1)
        depth = tokens * heads_here / (ctas * 8) + 1 + 5 + 8 + 2 * sms / 32 + 1 + 5
        within(d, want, most, depth + D + 32)
        # what would not pass: nothing at all, the other sign, and the sum without one token in six hundred
        bound = U[d.dtype] * want.abs() + (1 + U[d.dtype]) * (depth + D + 32) * E * most
        few = slice(0, max(1, tokens // 600))
        where = tuple(t[few] for t in (cos, sin, at)) + (interleaved,)
        missing = norm_turn(x[:, few], w.detach(), g[:, few], *where)[4]
        assert float((want.abs() > bound).double().mean()) > 0.8
        assert float((missing.abs() > 2 * bound).double().mean()) > 0.5
