"""Preference and policy losses, forward and backward, against their formulas in 64 bits.

Bounds.  u is half a step of a type, E = 2^-24 that of fp32.  A row's sum of exponentials: each exponent k z - M is
rounded twice (k and the difference) at the size of the largest |k z|, each exponential is off by 2^-22 of its value,
and a thread adds up at most V / 32 + 64 of them one after the other, so the sum is off by
R = (V / 32 + 68 + 4 max |k z|) E + 2^-22, and a log-probability l by R + E (|z| + |l|).  A gradient
g (onehot - p) has p off by 2 R and g by what its loss makes of the error of l."""
import math

import pytest
import torch

from pfeife_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}
E = 2.0 ** -24


def near(got, want, off):
    """|got - want| <= u |want| + off"""
    got64 = got.double()
    assert torch.isfinite(got).all()
    bound = U[got.dtype] * want.abs() + 1.01 * off + TINY[got.dtype]
    worst = ((got64 - want).abs() / bound).max() if got.numel() else 0.0
    assert worst <= 1.0, float(worst)


def batch(N, T, V, device, dtype, seed, layout="packed", masked=0.4):
    g = torch.Generator().manual_seed(seed)
    new = lambda *s: (torch.randn(*s, generator=g) * 2).to(device=device, dtype=dtype)
    if layout == "shifted":                      # all but the last position of longer sequences
        z = new(N, T + 1, V)[:, :-1]
    elif layout == "seq first":
        z = new(T, N, V).transpose(0, 1)
    elif layout == "columns":                    # V is not innermost
        z = new(N, V, T).transpose(1, 2)
    elif layout == "wide":                       # some words of a padded vocabulary, off the vectors
        z = new(N, T, V + 5)[..., 3:3 + V]
    else:
        z = new(N, T, V)
    labels = torch.randint(0, V, (N, T), generator=g)
    labels[torch.rand(N, T, generator=g) < masked] = -100
    return z, labels.to(device)


def rows64(z, labels, temperature):
    """(l, its error bound, softmax, its relative error bound, which rows count) in 64 bits"""
    V = z.shape[-1]
    counted = (labels >= 0) & (labels < V)
    x = z.double() / temperature
    lse = x.logsumexp(-1)
    zl = x.gather(-1, labels.clamp(0, V - 1).unsqueeze(-1))[..., 0]
    l = (zl - lse).masked_fill(~counted, 0.0)
    big = x.masked_fill(x.isinf(), 0.0).abs().amax(-1) * 1.4427
    rel = (V / 32 + 68 + 4 * big) * E + 2.0 ** -22
    return l, (rel + E * (zl.abs() + l.abs())).masked_fill(~counted, 0.0), torch.softmax(x, -1), 2 * rel, counted


def gradient(g, dg, p, rel, labels, counted):
    """(g (onehot - p), its error bound), zero where nothing counts"""
    hot = torch.zeros_like(p).scatter_(-1, labels.masked_fill(~counted, 0).unsqueeze(-1), 1.0)
    g, dg = (t.masked_fill(~counted, 0.0).unsqueeze(-1) for t in (g, dg))
    off = dg * (hot + p) + g.abs() * p * rel.unsqueeze(-1) + 4 * E * g.abs() * (hot + p)
    at = counted.unsqueeze(-1)
    return (g * (hot - p)).masked_fill(~at, 0.0), off.masked_fill(~at, 0.0)


# rows of a warp, of a CTA and of a wide CTA; odd lengths, fewer words than a vector
SIZES = [(2, 1, 1), (2, 3, 7), (4, 5, 256), (2, 9, 1000), (6, 30, 1025), (2, 33, 2049), (2, 2, 9001), (4, 60, 8192),
         (2, 40, 32003)]
LAYOUTS = ["packed", "shifted", "seq first", "columns", "wide"]


def _cases():
    out = []
    for i, size in enumerate(SIZES):
        for j, dtype in enumerate(DTYPES):
            out.append((*size, dtype, LAYOUTS[(3 * i + j) % 5]))
    return out


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("N,T,V,dtype,layout", _cases(), ids=str)
def test_preference_loss(N, T, V, dtype, layout, device):
    for seed, (beta, smoothing) in enumerate(((0.1, 0.0), (0.5, 0.2))):
        z, labels = batch(N, T, V, device, dtype, seed, layout)
        z.requires_grad_()
        l, dl, p, rel, counted = rows64(z.detach(), labels, 1.0)
        ref = (l.sum(1) + torch.randn(N, generator=torch.Generator().manual_seed(9)).to(device) * 3).float()
        out = ops.preference_loss(z, labels, ref, beta=beta, label_smoothing=smoothing)
        gout = torch.tensor(2.5, device=device)
        (dz,) = torch.autograd.grad(out.loss, z, gout)
        assert dz.shape == z.shape and dz.dtype == dtype and not out.rewards.requires_grad
        P = N // 2
        r, dr = beta * (l.sum(1) - ref.double()), beta * dl.sum(1) + 2 * E * beta * (l.sum(1).abs() + ref.abs())
        near(out.rewards, r, dr)
        m, dm = r[:P] - r[P:], dr[:P] + dr[P:]
        sig = lambda t: 1 / (1 + (-t).exp())
        want = -(1 - smoothing) * sig(m).log() - smoothing * sig(-m).log()
        near(out.loss.detach(), want.mean(), dm.mean() + 4 * E * want.mean())
        c = -beta / P * ((1 - smoothing) * sig(-m) - smoothing * sig(m))
        c = torch.cat([c, -c])[:, None].expand(N, T) * 2.5
        dc = (2.5 * beta / P * torch.cat([dm, dm]) / 4)[:, None].expand(N, T)     # sig' <= 1/4
        near(dz, *gradient(c, dc + 4 * E * 2.5 * beta / P, p, rel, labels, counted))
        assert not dz[~counted].any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("N,T,V,dtype,layout", _cases(), ids=str)
def test_policy_loss(N, T, V, dtype, layout, device):
    for seed, (kl, temperature, lo, hi, per_token) in enumerate(((0.0, 1.0, 0.2, 0.2, True), (0.3, 0.7, 0.1, 0.3, False))):
        z, actions = batch(N, T, V, device, dtype, seed, layout)
        z.requires_grad_()
        l, dl, p, rel, counted = rows64(z.detach(), actions, temperature)
        g = torch.Generator().manual_seed(3)
        noise = lambda *s: torch.randn(*s, generator=g).to(device)
        old = (l + 0.2 * noise(N, T)).float()
        r = (l - old.double()).exp()
        # no ratio so near a border that the error of l could carry it over
        for border in (1 - lo, 1 + hi):
            old = torch.where((r - border).abs() < 4e-3 + 4 * dl, l.float(), old)
        r = (l - old.double()).exp()
        adv = noise(N, T) if per_token else noise(N, 1)
        ref = (l + 0.3 * noise(N, T)).float() if kl else None
        out = ops.policy_loss(z, actions, old, adv, ref, lo, hi, kl, temperature)
        (dz,) = torch.autograd.grad(out.loss, z)
        assert dz.shape == z.shape and dz.dtype == dtype and not any(t.requires_grad for t in out[1:])
        near(out.logps, l, dl)
        n, A = max(1, int(counted.sum())), adv.double().expand(N, T)
        held = ((A > 0) & (r > 1 + hi)) | ((A < 0) & (r < 1 - lo))
        term = -torch.where(held, torch.where(A > 0, 1 + hi, 1 - lo).double(), r) * A
        c, off = torch.where(held, 0.0, -A * r), (A * r).abs() * (dl * 1.1 + 8 * E)
        dc = off.clone()
        if kl:
            d = ref.double() - l
            term, c = term + kl * (torch.expm1(d) - d), c - kl * torch.expm1(d)
            off = off + kl * (torch.expm1(d).abs() * 1.1 * dl + 4 * E * (torch.expm1(d).abs() + d.abs()))
            dc = dc + kl * d.exp() * 1.1 * dl + 4 * E * kl * torch.expm1(d).abs()
            each = (torch.expm1(d) - d)
            near(out.kl, each[counted].sum() / n, (torch.expm1(d).abs() * 1.1 * dl + 2 * E * each)[counted].sum() / n)
        else:
            assert float(out.kl) == 0.0
        off = off + 4 * E * term.abs()
        near(out.loss.detach(), term[counted].sum() / n, off[counted].sum() / n)
        near(out.clipped, (held & counted).sum().double() / n, torch.zeros((), device=device))
        near(dz, *gradient(c / (n * temperature), (dc + 4 * E * c.abs()) / (n * temperature), p, rel, actions, counted))
        assert not dz[~counted].any()


def test_gradients_are_those_of_differences():
    torch.manual_seed(1)
    z = torch.randn(4, 3, 6, dtype=torch.float64, requires_grad=True)
    labels = torch.tensor([[0, 5, -100], [1, 1, 2], [3, -1, 6], [0, 2, 4]])
    ref = torch.tensor([-3.0, -5.0, -4.0, -6.0])
    # losses are rounded to 32 bits: differences of 1e-2 and a tolerance of their curvature and that rounding
    check = lambda f: torch.autograd.gradcheck(f, [z], eps=1e-2, atol=2e-4, rtol=1e-3)
    assert check(lambda x: ops.preference_loss(x, labels, ref, 0.5, 0.1).loss.double())
    lp = torch.log_softmax(z.detach(), -1).gather(-1, labels.clamp(0, 5).unsqueeze(-1))[..., 0]
    old = (lp + torch.tensor([0.4, -0.05, 0.05])).float()          # held or not by a wide margin
    adv = torch.tensor([[1.0], [-1.0], [2.0], [0.5]])
    assert check(lambda x: ops.policy_loss(x, labels, old, adv, old, kl_coef=0.5).loss.double())
    assert check(lambda x: ops.policy_loss(x, labels, old.flip(1), adv, temperature=2.0).loss.double())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [40, 3001])
def test_masked_words_and_what_stands_in_rows_that_do_not_count(V, dtype, device):
    """Logits of -inf and of the type's lowest value have no probability and no gradient; NaN and infinities in rows
    that do not count reach nothing; labels beyond the vocabulary count as little as the ignored one."""
    z, labels = batch(4, 6, V, device, dtype, 5, masked=0.0)
    z[..., V // 2:] = -math.inf
    z[..., V // 4:V // 2] = torch.finfo(dtype).min
    labels = labels % (V // 4)
    labels[0, 1], labels[1, :], labels[2, 3], labels[3, 0] = -100, V, -1, 1 << 40
    counted = (labels >= 0) & (labels < V)
    clean = z.clone()
    z[~counted] = torch.tensor([math.nan, math.inf, -math.inf, 1.0], dtype=dtype).repeat(V // 4 + 1)[:V].to(device)
    got, want = [], []
    for values, to in ((z, got), (clean, want)):
        values = values.detach().requires_grad_()
        a = ops.preference_loss(values, labels, torch.zeros(4, device=device))
        old = torch.full((4, 6), -3.0, device=device)
        b = ops.policy_loss(values, labels, old, torch.ones(4, 1, device=device), old - 1, kl_coef=0.1)
        to += [a.loss, a.rewards, *b, *torch.autograd.grad(a.loss + b.loss, values)]
    for a, b in zip(got, want):
        assert torch.isfinite(a).all() and torch.equal(a, b)
    assert not got[-1][..., V // 4:].any() and not got[-1][~counted].any() and got[-1][counted].any()


@pytest.mark.parametrize("device", DEVICES)
def test_a_row_that_counts_keeps_its_nan(device):
    """A NaN logit, and a row of -inf alone, which has no softmax, are not smoothed over."""
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    for V in (9, 2500):
        for fill in (math.nan, -math.inf):
            z, labels = batch(2, 3, V, device, dtype, 1, masked=0.0)
            z[0, 1] = fill
            if fill != fill:
                z[0, 1, : V - 1] = 0.0
            labels[0, 1] = 0
            out = ops.policy_loss(z, labels, torch.zeros(2, 3, device=device), torch.ones(2, 3, device=device))
            assert torch.isnan(out.loss) and torch.isnan(out.logps[0, 1]) and torch.isfinite(out.logps[1]).all()
            assert torch.isnan(ops.preference_loss(z, labels, torch.zeros(2, device=device)).loss)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V,T", [(9, 4), (260, 6), (260, 3000), (2500, 3), (40001, 3)])
def test_rows_far_from_zero(V, T, dtype, device):
    """Rows that count though a mask of the type's lowest value, or of another large one, has left them nothing: the
    softmax of their differences.  Per row: everything masked; all but the label, the label alone; in the first half
    only; a large positive mask; next to words of ordinary size; -inf beside it.

    Differences of such values are 0 or so large that the exponential is 0, where nothing is rounded but the sum:
    l is off by R of the module's bound without its |k z|, and by E |l|."""
    low = torch.finfo(dtype).min
    z, _ = batch(2, T, V, device, dtype, 3)
    labels = torch.full((2, T), 1, device=device)
    rows = z.view(-1, V)
    for i in range(0, 2 * T):
        fill, kind = (low, -1e9, -1e30, 1e12, -5e6, 3e38)[i % 6], i % 7
        if kind < 5:
            rows[i] = fill
        if kind == 1:
            rows[i, 1] = fill * 1.5 if abs(fill) < 1e38 else fill / 2
        elif kind == 2:
            rows[i, V // 2:] = -math.inf
        elif kind == 3:
            rows[i, V // 2:] = low
        elif kind == 4:
            rows[i, V // 2:] = -7.0
        elif kind == 5:
            rows[i, V // 2:] = min(fill, -fill)
    z.requires_grad_()
    x = z.detach().double()
    l = torch.log_softmax(x, -1)[..., 1]
    p = torch.softmax(x, -1)
    ok = l > -50
    # words of ordinary size are the only ones whose differences have a rounding, of |k z| < 24
    R = (V / 32 + 68 + 4 * 24) * E + 2.0 ** -22
    out = ops.policy_loss(z, labels, torch.where(ok, l.float(), -3.0), torch.ones(2, 1, device=device))
    near(out.logps, l, R + 2 * E * l.abs())
    # old = l: the ratio is 1 but for l's rounding, and the gradient -(onehot - p) / (2 T); 0 for the impossible
    (dz,) = torch.autograd.grad(out.loss, z)
    g = torch.where(ok, -1.0, 0.0).double() / (2 * T)
    dg = (R + 3 * E * l.abs() + 2.0 ** -20) / (2 * T)
    bound = gradient(g, dg, p, torch.full_like(l, 2 * R), labels, torch.ones_like(ok))
    near(dz[ok], bound[0][ok], bound[1][ok])
    assert torch.isfinite(dz).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("V", [65, 3001])
def test_temperatures_of_all_sizes(V, device):
    """From the largest word alone to all words alike.  z / temperature is rounded twice, and its difference to the
    largest once: l is off by 4 E of it besides R.  What fp32 cannot invert is refused."""
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    z, labels = batch(2, 4, V, device, dtype, 8, masked=0.0)
    v = torch.full((2, 4), -3.0, device=device)
    for temperature in (1e-30, 1e-12, 1e-6, 1e-3, 1e6, 1e30):
        x = z.double() / temperature
        far = (x - x.amax(-1, keepdim=True)).gather(-1, labels.unsqueeze(-1))[..., 0].abs()
        l = torch.log_softmax(x, -1).gather(-1, labels.unsqueeze(-1))[..., 0]
        big = x.abs().amax(-1).clamp(max=2.0 ** 22) * 1.4427      # beyond it there is no rounded reference
        R = (V / 32 + 68 + 4 * big) * E + 2.0 ** -22
        near(ops.policy_loss(z, labels, v, v + 1, temperature=temperature).logps, l, R + 4 * E * far + E * l.abs())
    for temperature in (1e-31, 1e-320, 1e31):
        with pytest.raises(ValueError, match="temperature"):
            ops.policy_loss(z, labels, v, v, temperature=temperature)


@pytest.mark.parametrize("device", DEVICES)
def test_certain_words(device):
    """A word that has all the probability, alone in its vocabulary or not: no log-probability above 0."""
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    for V in (1, 2, 70, 3000):
        z = torch.full((4, 50, V), -300.0, device=device)
        z[..., 0] = torch.linspace(-90, 90, 200, device=device).view(4, 50)
        z, labels = z.to(dtype).requires_grad_(), torch.zeros(4, 50, dtype=torch.int64, device=device)
        v = torch.zeros(4, 50, device=device)
        out = ops.policy_loss(z, labels, v, v + 1)
        assert (out.logps <= 0).all() and (out.logps > -1e-6).all() and abs(float(out.loss.detach()) + 1) < 1e-6
        (dz,) = torch.autograd.grad(out.loss, z)
        assert (dz.abs() <= 1e-6 / 200).all()


@pytest.mark.parametrize("device", DEVICES)
def test_an_impossible_token_beside_a_reference(device):
    """A sampled word that a mask has taken since: its estimate of the KL is infinite, and reaches neither the loss
    nor a gradient where the coefficient is 0."""
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    z, labels = batch(2, 3, 40, device, dtype, 2, masked=0.0)
    labels[0, 1] = 7
    z[0, 1, 7] = -math.inf
    z.requires_grad_()
    old, adv = torch.full((2, 3), -3.0, device=device), torch.ones(2, 3, device=device)
    alone = ops.policy_loss(z, labels, old, adv)
    for ref in (old, old - 800):
        out = ops.policy_loss(z, labels, old, adv, ref)
        assert out.kl == math.inf and out.logps[0, 1] == -math.inf
        assert torch.equal(out.loss, alone.loss) and torch.isfinite(out.loss)
        for a, b in zip(torch.autograd.grad(out.loss, z), torch.autograd.grad(alone.loss, z, retain_graph=True)):
            assert torch.equal(a, b) and torch.isfinite(a).all()
        assert ops.policy_loss(z, labels, old, adv, ref, kl_coef=0.1).loss == math.inf


@pytest.mark.parametrize("device", DEVICES)
def test_nothing_counts(device):
    dtype = torch.float32 if device == "cpu" else torch.float16
    z, labels = batch(2, 4, 33, device, dtype, 1)
    labels.fill_(-100)
    z.requires_grad_()
    zeros = torch.zeros(2, 4, device=device)
    out = ops.policy_loss(z, labels, zeros, zeros + 1, zeros, kl_coef=1.0)
    assert float(out.loss.detach()) == float(out.kl) == float(out.clipped) == 0.0 and not out.logps.any()
    assert not torch.autograd.grad(out.loss, z)[0].any()
    pref = ops.preference_loss(z, labels, torch.tensor([1.0, 3.0], device=device), beta=0.5)
    assert torch.allclose(pref.rewards, torch.tensor([-0.5, -1.5], device=device))
    assert abs(float(pref.loss.detach()) - math.log1p(math.exp(-1.0))) < 1e-6
    assert not torch.autograd.grad(pref.loss, z)[0].any()
    # no tokens at all
    empty = torch.zeros(2, 0, 33, device=device, dtype=dtype).requires_grad_()
    none = torch.zeros(2, 0, dtype=torch.int64, device=device)
    out = ops.policy_loss(empty, none, none.float(), none.float())
    assert float(out.loss.detach()) == 0.0 and torch.autograd.grad(out.loss, empty)[0].shape == (2, 0, 33)
    pref = ops.preference_loss(empty, none, torch.zeros(2, device=device))
    assert abs(float(pref.loss.detach()) - math.log(2)) < 1e-6
    assert torch.autograd.grad(pref.loss, empty)[0].shape == (2, 0, 33)


@pytest.mark.parametrize("device", DEVICES)
def test_far_margins_do_not_overflow(device):
    """Margins of hundreds of nats, and an impossible token: -log sig(m) is 0 or -m."""
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    z, labels = batch(2, 4, 50, device, dtype, 1, masked=0.0)
    z.requires_grad_()
    for ref, want in (((0.0, 5000.0), 0.0), ((5000.0, 0.0), None)):
        ref = torch.tensor(ref, device=device)
        out = ops.preference_loss(z, labels, ref, beta=1.0)
        m = float(out.rewards[0] - out.rewards[1])
        assert abs(float(out.loss.detach()) - max(-m, 0.0)) <= 1e-5 * abs(m)
        (dz,) = torch.autograd.grad(out.loss, z)
        assert torch.isfinite(dz).all() and (dz.any() if want is None else True)
    with torch.no_grad():
        z[1, 2, labels[1, 2]] = -math.inf
    assert float(ops.preference_loss(z, labels, torch.zeros(2, device=device)).loss.detach()) == 0.0


@pytest.mark.parametrize("device", DEVICES)
def test_shapes_types_and_an_ignored_word(device):
    """One dimension of tokens or three, labels of 32 bits, a word of the vocabulary that does not count, advantages
    and log-probabilities of other types."""
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    z, labels = batch(6, 4, 33, device, dtype, 1, masked=0.0)
    labels[2, 1] = 0
    old, adv = torch.full((6, 4), -3.0, device=device), torch.linspace(-1, 1, 24, device=device).view(6, 4)
    z.requires_grad_()
    def both(z, labels, old, adv, ref=None):
        out = ops.policy_loss(z, labels, old, adv, ref, ignore_index=0, kl_coef=0.1)
        return out.loss, out.logps.reshape(6, 4), torch.autograd.grad(out.loss, z)[0].reshape(6, 4, 33)
    want = both(z, labels, old, adv)
    flat = z.detach().view(24, 33).requires_grad_()
    deep = z.detach().view(2, 3, 4, 33).requires_grad_()
    for got in (both(flat, labels.view(24), old.view(24), adv.view(24)),
                both(deep, labels.view(2, 3, 4), old.view(2, 3, 4), adv.view(2, 3, 4)),
                both(z, labels.int(), old.double(), adv.double())):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert not want[1][labels == 0].any() and not want[2][labels == 0].any()
    some = torch.linspace(-1, 1, 6, device=device)[:, None]
    a, b = (both(z, labels, old, t, old) for t in (some, some.expand(6, 4).contiguous()))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    pa, pb = (ops.preference_loss(z, t, torch.zeros(6, device=device).to(r), ignore_index=0) for t, r in
              ((labels, torch.float32), (labels.int(), torch.float64)))
    assert torch.equal(pa.loss, pb.loss) and torch.equal(pa.rewards, pb.rewards)


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    z, labels = batch(2, 3, 9, device, torch.float32, 1)
    v, ref = torch.zeros(2, 3, device=device), torch.zeros(2, device=device)
    other = "meta" if device == "cpu" else "cpu"
    for bad in (dict(logits=z[:1], labels=labels[:1], ref_logps=ref[:1]), dict(logits=z[0], labels=labels[0]),
                dict(labels=labels[:, :2]), dict(labels=v), dict(labels=labels.to(other)), dict(ref_logps=v),
                dict(ref_logps=ref.to(other)), dict(ref_logps=ref.clone().requires_grad_()), dict(label_smoothing=-0.1),
                dict(label_smoothing=1.5), dict(logits=z[..., :0])):
        with pytest.raises(ValueError):
            ops.preference_loss(**{**dict(logits=z, labels=labels, ref_logps=ref), **bad})
    for bad in (dict(logits=z[0, 0], actions=labels[0, 0]), dict(actions=labels[:, :2]), dict(old_logps=v[:1]),
                dict(ref_logps=v[:, :1]), dict(advantages=v[:, :2]), dict(advantages=ref), dict(temperature=0.0),
                dict(temperature=-1.0), dict(temperature=math.inf), dict(temperature=math.nan), dict(clip_high=math.nan),
                dict(clip_low=1.5), dict(clip_high=-0.1), dict(old_logps=v.to(other)),
                dict(advantages=v.clone().requires_grad_()), dict(actions=v)):
        with pytest.raises(ValueError):
            ops.policy_loss(**{**dict(logits=z, actions=labels, old_logps=v, advantages=v), **bad})


@pytest.mark.gpu
@pytest.mark.parametrize("pad,off", [(0, 0), (5, 0), (61, 3), (2000, 1), (3, 3)])
@pytest.mark.parametrize("V", [259, 4099])
def test_some_words_of_a_padded_vocabulary(pad, off, V):
    """The gradient of rows with space between them has the same values wherever it lies."""
    g = torch.Generator().manual_seed(V)
    wide = torch.randn(2, 5, V + pad + off, generator=g).cuda().half()
    labels = torch.randint(0, V, (2, 5), generator=g).cuda()
    labels[0, 2] = -100
    z = wide[..., off:off + V].detach().requires_grad_()
    packed = z.detach().clone().requires_grad_()
    def grad(t):
        return torch.autograd.grad(ops.preference_loss(t, labels, torch.zeros(2, device="cuda")).loss, t)[0]
    a, b = grad(z), grad(packed)
    assert a.shape == b.shape and torch.equal(a, b) and not a[0, 2].any()
    whole = wide.requires_grad_()                  # and reaches the whole of it
    (c,) = torch.autograd.grad(ops.preference_loss(whole[..., off:off + V], labels, torch.zeros(2, device="cuda")).loss,
                               whole)
    assert torch.equal(c[..., off:off + V], b) and not c[..., :off].any() and not c[..., off + V:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,V", [(70001, 33), (9000, 1500)])
def test_many_rows(rows, V):
    z, labels = batch(1, rows, V, "cuda", torch.bfloat16, 1)
    z.requires_grad_()
    l, dl, p, rel, counted = rows64(z.detach(), labels, 1.0)
    old = l.float()
    adv = torch.rand(1, rows, device="cuda") + 0.5
    out = ops.policy_loss(z, labels, old, adv)
    n = int(counted.sum())
    near(out.logps, l, dl)
    near(out.loss.detach(), -(adv.double() * counted).sum() / n, (adv * (1.1 * dl + 8 * E) * counted).sum() / n)
    two = torch.cat([z, z.flip(1)]).detach().requires_grad_()
    ref = torch.stack([l.sum(), l.sum() - 1]).float()[0].reshape(1, -1)[0]
    pref = ops.preference_loss(two, torch.cat([labels, labels.flip(1)]), torch.cat([ref, ref - 1]))
    near(pref.rewards, 0.1 * torch.tensor([0.0, 1.0], device="cuda", dtype=torch.float64),
         (0.1 * dl.sum() + 4 * E * l.sum().abs()).expand(2))
    (dz,) = torch.autograd.grad(pref.loss, two)
    assert torch.isfinite(dz).all() and not dz[0][~counted[0]].any()


@pytest.mark.gpu
def test_other_streams_graphs_and_bits_that_repeat():
    from pfeife_b200.ops import functional as f
    z, labels = batch(4, 37, 5001, "cuda", torch.bfloat16, 1)
    old = torch.full((4, 37), -9.0, device="cuda")
    adv, ref, one = torch.randn(4, 1, device="cuda"), torch.zeros(4, device="cuda"), torch.ones((), device="cuda")

    def both(z):
        a = f.policy_fwd(z, labels, old, adv.expand(4, 37), old, 0.2, 0.2, 0.1, 1.0, -100)
        b = f.preference_fwd(z, labels, ref, 0.1, 0.1, -100)
        da = f.token_loss_bwd(one, z, labels, a[4], a[5], a[6], -100, 1.0)
        db = f.token_loss_bwd(one, z, labels, b[2], b[3], None, -100, 1.0)
        return [*a[:4], b[0], b[1], da, db]

    with torch.no_grad():
        want = both(z)
        assert all(torch.equal(a, b) for a, b in zip(both(z), want))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = both(z)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        static = torch.zeros_like(z)
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = both(static)
            graphs.append((g, out))
        static.copy_(z)
        for g, _ in graphs + graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Rows whose logits lie further than 2^31 elements in, and whose gradient does."""
    N, T, V = 2, 35000, 32000                    # 2.2e9 elements
    z = torch.zeros(N, T, V, device="cuda", dtype=torch.bfloat16)
    z[1, T - 3:].normal_()
    labels = torch.full((N, T), -100, device="cuda")
    labels[0, 5], labels[1, T - 3:] = 3, 7
    z.requires_grad_()
    out = ops.preference_loss(z, labels, torch.zeros(2, device="cuda"))
    (dz,) = torch.autograd.grad(out.loss, z)
    l, dl, p, rel, counted = rows64(z.detach()[1:, T - 3:], labels[1:, T - 3:], 1.0)
    near(out.rewards[1], 0.1 * l.sum(), 0.1 * dl.sum() + 4 * E * l.sum().abs())
    m = (out.rewards[0] - out.rewards[1]).double()
    c = (0.1 * torch.sigmoid(-m)).expand(1, 3)
    near(dz[1:, T - 3:], *gradient(c, c * 1e-5, p, rel, labels[1:, T - 3:], counted))
    assert int(dz.count_nonzero(-1).ne(0).sum()) == 4


@pytest.mark.parametrize("device", DEVICES)
def test_ops_are_seen_by_tracers_and_modes(device):
    from pfeife_b200.ops import functional as f
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    z, labels = batch(4, 5, 12, device, dtype, 1)
    z.requires_grad_()
    v, ref = torch.zeros(4, 5, device=device), torch.zeros(4, device=device)
    checks = ("test_schema", "test_faketensor", "test_autograd_registration")
    torch.library.opcheck(f.preference_fwd, (z, labels, ref, 0.1, 0.0, -100), test_utils=checks)
    torch.library.opcheck(f.policy_fwd, (z, labels, v, v, None, 0.2, 0.2, 0.0, 1.0, -100), test_utils=checks)
    fn = lambda t: ops.preference_loss(t, labels, ref).loss + ops.policy_loss(t, labels, v, v + 1, v, kl_coef=0.1).loss
    want = fn(z)
    got = torch.compile(fn, backend="eager", fullgraph=True)(z)
    assert torch.equal(got, want)
    assert torch.equal(torch.autograd.grad(got, z)[0], torch.autograd.grad(want, z)[0])


# ------------------------------------------------------------------------------ calls that do not go the usual way
class Watch(torch.utils._python_dispatch.TorchDispatchMode):
    """Lets every op be seen, which keeps all calls on the dispatcher."""

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("loss", ["preference", "policy"])
def test_direct_calls_and_the_dispatcher_agree(loss, device, monkeypatch):
    from pfeife_b200.ops import functional
    monkeypatch.setattr(functional, "_FIRST_DEVICE", -1 if device == "cpu" else 0)
    z, labels = batch(4, 7, 300, device, torch.float32 if device == "cpu" else torch.bfloat16, 3)
    z.requires_grad_()
    v = torch.full((4, 7), -5.0, device=device)

    def fn(t):
        if loss == "preference":
            return ops.preference_loss(t, labels, v[:, 0], 0.3, 0.1)
        return ops.policy_loss(t, labels, v, v[:, :1] + 6, v + 1, kl_coef=0.2, temperature=1.3)

    out = fn(z)
    g = torch.tensor(3.0, device=device)
    (want,) = torch.autograd.grad(out.loss, z, g, retain_graph=True)
    assert torch.equal(torch.autograd.grad(out.loss, z, g)[0], want)
    with Watch():
        seen = fn(z)
        (got,) = torch.autograd.grad(seen.loss, z, g)
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(out, seen))
    with torch.no_grad():
        assert all(torch.equal(a, b) and not b.requires_grad for a, b in zip(out, fn(z)))

    def unpack(t):                                 # every second element of a wider tensor, or another type
        return torch.stack([t, t], -1)[..., 0] if t.dim() != 1 else t.double() if t.is_floating_point() else t
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        hooked = fn(z).loss
    assert torch.equal(torch.autograd.grad(hooked, z, g)[0], want)
    from torch.utils.checkpoint import checkpoint
    again = checkpoint(lambda t: fn(t).loss, z, use_reentrant=False)
    assert torch.equal(torch.autograd.grad(again, z, g)[0], want)
    # the other outputs are constants
    assert not any(t.requires_grad for t in fn(z)[1:])


def test_entry_points_refuse_what_they_cannot_read():
    """Before anything touches a device."""
    import ctypes
    from pfeife_b200.csrc import build
    from pfeife_b200.ops import _lib
    if not build.KERNEL_LIB.exists():
        pytest.skip("the kernel library is not built")
    calls = _lib.load_calls(ctypes.CDLL(str(build.KERNEL_LIB), mode=ctypes.RTLD_GLOBAL))
    t = torch.zeros(64).data_ptr()

    def preference(z=t, N=2, T=1, V=4, dtype=2):
        return calls.pf_preference_fwd(z, t, t, t, t, t, t, t, N, T, V, 4, 4, -100, 0.1, 0.0, dtype, 148, None)

    def policy(z=t, N=2, T=1, V=4, dtype=2):
        return calls.pf_policy_fwd(z, t, t, None, t, t, t, t, t, t, t, t, t, N, T, V, 4, 4, 1, 0, -100, 0.2, 0.2, 0.0,
                                   1.0, dtype, 148, None)

    def backward(z=t, N=2, T=1, V=4, dtype=2, row=4):
        return calls.pf_token_loss_bwd(z, t, t, t, t, None, t, row, N, T, V, 4, 4, -100, 1, 1.0, dtype, 148, None)
    for call in (preference, policy, backward):
        assert call(dtype=3) == -1 and call(z=t + 1) == -2 and call(z=t + 2, dtype=0) == -2
        assert call(V=0) == -3 and call(N=1 << 20, T=1 << 20) == -3 and call(N=-2) == -3
    assert preference(N=3) == -3 and preference(N=0) == -3 and backward(T=0) == 0 and backward(row=3) == -3
    # several parts of a row only where rows are few: two floats for each part and one for each row, beside the sums
    few, many = (calls.pf_token_loss_scratch(1, n, 32000, 2, 148) for n in (16, 16384))
    assert few >= 16 * 4 + 8 and 16384 + 8192 <= many < 2 * 16384


# ------------------------------------------------------------------------------ together
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("loss", ["preference", "policy"])
def test_a_decoder_with_normed_heads_tuned_on_a_loss(loss, device):
    """One step of a decoder with normed queries and keys and a scaled, partial, interleaved rotation: the loss and
    every gradient against the same model in plain 64-bit PyTorch."""
    from pfeife_b200.models.llama import Llama, llama_config
    torch.manual_seed(0)
    cfg = llama_config("llama_tiny", qk_norm=True, rope_dim=8, rope_interleaved=True, num_layers=2,
                       rope_scaling=ops.RopeScaling("yarn", 2.0, 16))
    model = Llama(cfg)
    with torch.no_grad():
        for name, p in model.named_parameters():
            if name.endswith("norm"):
                p.add_(0.3 * torch.randn_like(p))
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    model = model.to(device)
    for p in model.parameters():
        if p.dim() > 1:
            p.data = p.data.to(dtype)
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 256, (4, 24), generator=g).to(device)
    labels = torch.cat([ids[:, 1:], ids.new_full((4, 1), -100)], 1)
    labels[:, :5] = -100
    labels[1, 15:] = -100
    ref, old = torch.randn(4, generator=g).to(device) - 80, torch.full((4, 24), -5.4, device=device)
    adv = torch.tensor([[1.0], [-0.5], [0.7], [-1.2]], device=device)

    def tuned(logits):
        if loss == "preference":
            return ops.preference_loss(logits, labels, ref).loss
        return ops.policy_loss(logits, labels, old, adv, old, 0.6, 0.8, kl_coef=0.1).loss

    got = tuned(model(ids))
    names = [n for n, _ in model.named_parameters()]
    grads = torch.autograd.grad(got, list(model.parameters()))

    w = {n: p.detach().double().requires_grad_() for n, p in model.named_parameters()}
    def norm(x, gain, eps=cfg.rms_eps):
        return x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * gain
    x = w["embed.weight"][ids]
    for i in range(cfg.num_layers):
        at = lambda n: w[f"layers.{i}.{n}"]
        qkv = (norm(x, at("input_norm")) @ at("qkv.weight").t()).view(4, 24, 3, 4, 16)
        where = (model.rope_cos.double()[:24, None], model.rope_sin.double()[:24, None])
        def turn(t):
            a, b = t[..., 0:8:2], t[..., 1:8:2]
            c, s = where
            return torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), t[..., 8:]], -1)
        q, k = turn(norm(qkv[:, :, 0], at("q_norm"))), turn(norm(qkv[:, :, 1], at("k_norm")))
        scores = torch.einsum("bqhd,bkhd->bhqk", q, k) / 4
        scores = scores.masked_fill(torch.ones(24, 24, dtype=torch.bool, device=device).triu(1), -math.inf)
        a = torch.einsum("bhqk,bkhd->bqhd", scores.softmax(-1), qkv[:, :, 2]).reshape(4, 24, 64)
        x = x + a @ at("o_proj.weight").t()
        gate, up = (norm(x, at("post_norm")) @ at("gate_up.weight").t()).chunk(2, -1)
        x = x + (torch.nn.functional.silu(gate) * up) @ at("down.weight").t()
    z = norm(x, w["norm"]) @ w["lm_head.weight"].t()
    l = torch.log_softmax(z, -1).gather(-1, labels.clamp(min=0).unsqueeze(-1))[..., 0] * (labels >= 0)
    if loss == "preference":
        r = 0.1 * (l.sum(1) - ref)
        want = -torch.nn.functional.logsigmoid(r[:2] - r[2:]).mean()
    else:
        ratio, d = (l - old).exp(), old - l
        term = -torch.minimum(ratio * adv, ratio.clamp(0.4, 1.8) * adv) + 0.1 * (d.exp() - d - 1)
        want = (term * (labels >= 0)).sum() / (labels >= 0).sum()
    exact = torch.autograd.grad(want, list(w.values()))
    # some 40 roundings of 2^-8 lie between a weight and the loss in 16 bits, 2^-24 in 32; they add up at random
    rel = 40 * (2.0 ** -24 * 8 if device == "cpu" else 2.0 ** -8 / 2)
    got, want = float(got.detach()), float(want.detach())
    assert abs(got - want) < rel * abs(want) + rel * 0.1
    for name, a, b in zip(names, grads, exact):
        assert (a.double() - b).norm() <= rel * b.norm() + 1e-12, name


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.int32, torch.int16, torch.int8, torch.uint8])
def test_labels_of_small_types(dtype, device):
    """Numbers are read as 64 bits before they are compared: a vocabulary or an ignored number beyond the labels' type
    is neither an error nor wrapped around."""
    kind = torch.float32 if device == "cpu" else torch.bfloat16
    z, _ = batch(4, 5, 400, device, kind, 4)
    z.requires_grad_()
    labels = torch.arange(20, device=device).view(4, 5) * 6            # up to 114
    v, ref = torch.full((4, 5), -5.0, device=device), torch.zeros(4, device=device)
    for ignore in (-100, 6, 300):
        got, want = [], []
        for t, to in ((labels.to(dtype), got), (labels, want)):
            a = ops.preference_loss(z, t, ref, ignore_index=ignore)
            b = ops.policy_loss(z, t, v, v + 6, v, kl_coef=0.1, ignore_index=ignore)
            to += [a.loss, a.rewards, *b, *torch.autograd.grad(a.loss + b.loss, z)]
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert bool(want[-1][0, 1].any()) == (ignore != 6)
    for wrong in (labels.float(), labels.to(torch.complex64)):
        with pytest.raises(ValueError, match="labels"):
            ops.preference_loss(z, wrong, ref)
        with pytest.raises(ValueError, match="labels"):
            ops.policy_loss(z, wrong, v, v)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("V", [2, 300, 5000, 40001])
def test_rows_far_from_zero_hide_nothing(V, device):
    """The exponential of the largest word is 1 there without a rounding, and so are those of all that are alike: a
    word that has all the probability has a log-probability of 0, V words alike -ln V to its rounding in 32 bits."""
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    for value in (1e8, -1e30):
        z = torch.full((2, 3, V), value, device=device)
        z[:, 1:, V // 2] = value * (1.5 if value > 0 else 0.5)
        z, labels = z.to(dtype), torch.full((2, 3), V // 2, dtype=torch.int64, device=device)
        v = torch.zeros(2, 3, device=device)
        logps = ops.policy_loss(z, labels, v, v).logps
        assert not logps[:, 1:].any()
        # half a step of a value between 2^k and 2^(k+1), beside 64-bit logarithms
        assert ((logps[:, 0].double() + math.log(V)).abs() <= 2.0 ** (math.floor(math.log2(math.log(V))) - 24) + 1e-12).all()
        rewards = ops.preference_loss(z[:, 1:], labels[:, 1:], torch.zeros(2, device=device)).rewards
        assert not rewards.any()


@pytest.mark.parametrize("device", DEVICES)
def test_borders_of_the_clipping_in_64_bits(device):
    """A certain word has a log-probability of 0 and a ratio of exp(-old), which 64 bits place on the right side of a
    border 1e-9 away; the borders, which have no 32 bits, are not rounded to them, nor are coefficients below their
    range taken for 0."""
    dtype = torch.float32 if device == "cpu" else torch.bfloat16
    z = torch.full((1, 1, 40), -1e30, device=device)
    z[..., 3] = -1e29
    z, actions = z.to(dtype), torch.full((1, 1), 3, dtype=torch.int64, device=device)
    for i in range(32):
        old = torch.tensor([[(-1) ** i * (0.05 + 0.005 * i)]], dtype=torch.float32)
        ratio = math.exp(-float(old))
        for off in (-1e-9, 1e-9):
            if ratio > 1:
                a, clip, held = 1.0, dict(clip_low=0.5, clip_high=ratio - 1 + off), off < 0
            else:
                a, clip, held = -1.0, dict(clip_low=1 - ratio + off, clip_high=0.5), off < 0
            adv = torch.full((1, 1), a, device=device)
            assert float(ops.policy_loss(z, actions, old.to(device), adv, **clip).clipped) == held, (i, off)
    adv = torch.ones(1, 1, device=device)
    far = ops.policy_loss(z, actions, adv * 0, adv * 0, adv * 60, kl_coef=1e-50).loss         # 1e-50 exp(60)
    assert float(far) == pytest.approx(1e-50 * math.exp(60), rel=1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V,T", [(32000, 2048), (2000, 4096), (256, 16384)])
def test_errors_of_rows_that_have_one_sign(V, T, dtype):
    """A reward is a sum over a sequence less another, which keeps what is off by the same part in every row: over rows
    of normal logits that may be 1e-8 a row, 1e-5 in a thousand tokens, beside
      * k = log2(e) to 24 bits, a temperature that is off by 1.3e-8: the sums are those of that temperature, whose
        log-probability lies 1.3e-8 (z_label - mean of z) from the other;
      * what is left of the rows' own errors in the mean of 2 T of them, five times 8e-8 / sqrt(2 T): a row's sum is off
        by 4e-8 (one standard deviation) around its average, by twice that where a few words make it up.
    The exponential's average error alone is 3.7e-8."""
    g = torch.Generator(device="cuda").manual_seed(V)
    z = (torch.randn(2, T, V, device="cuda", generator=g) * 2.5).to(dtype)
    labels = torch.randint(0, V, (2, T), device="cuda", generator=g)
    k = float(torch.tensor(1.44269504088896341, dtype=torch.float32)) * math.log(2)
    l, lk, mean = (torch.stack(t) for t in zip(*(
        (torch.log_softmax(x, -1).gather(-1, t[:, None])[:, 0], torch.log_softmax(x * k, -1).gather(-1, t[:, None])[:, 0],
         (torch.softmax(x, -1) * x).sum(-1)) for x, t in ((z[i].double(), labels[i]) for i in range(2)))))
    ref = l.sum(1).float()
    rewards = ops.preference_loss(z, labels, ref, beta=1.0).rewards.double() + ref.double()
    bound = 1e-8 + 5 * 8e-8 / math.sqrt(2 * T)
    assert abs(float((rewards - lk.sum(1)).mean())) / T < bound
    far = (z.double().gather(-1, labels.unsqueeze(-1))[..., 0] - mean).sum() / (2 * T)
    assert abs(float((rewards - l.sum(1)).mean()) / T - (k - 1) * float(far)) < bound
    assert bound < 2e-8


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V,T", [(1, 4096), (256, 8192), (32000, 1024)])
def test_certain_words_over_a_sequence(V, T, dtype):
    """One exponential is the whole sum, and what is above 0 is cut off: a log-probability of 0 comes out below it by
    less than half a step of 1 in fp32 on average."""
    g = torch.Generator(device="cuda").manual_seed(V + 1)
    z = torch.full((2, T, V), -math.inf, device="cuda", dtype=dtype)
    labels = torch.randint(0, V, (2, T), device="cuda", generator=g)
    z.scatter_(2, labels.unsqueeze(-1), (torch.rand(2, T, 1, device="cuda", generator=g) * 40 - 20).to(dtype))
    rewards = ops.preference_loss(z, labels, torch.zeros(2, device="cuda"), beta=1.0).rewards.double()
    assert (rewards <= 0).all() and (rewards / T > -2.0 ** -24).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [32000, 256])
def test_rows_of_two_values(V, dtype):
    """All of a row's exponentials have one of two errors, which nothing but references that differ from lane to lane
    averages: in 128 sequences of four such rows each, a log-probability is off by less than half a step of 1 in fp32
    (root mean square; with one reference for all lanes 7.6e-8 in bf16)."""
    g = torch.Generator(device="cuda").manual_seed(1)
    values = torch.rand(128, 1, 2, device="cuda", generator=g) * 2
    pick = torch.randint(0, 2, (1, 4, V), device="cuda", generator=g).expand(128, 4, V)
    z = torch.gather(values.expand(128, 4, 2), 2, pick).to(dtype)
    labels = torch.zeros(128, 4, dtype=torch.int64, device="cuda")
    l = torch.log_softmax(z.double(), -1)[..., 0].sum(1)          # k's 24 bits: 1.3e-8 of 2 and less
    rewards = ops.preference_loss(z, labels, l.float(), beta=1.0).rewards.double()
    off = (rewards - (l - l.float().double())) / 4
    assert float(off.square().mean().sqrt()) < 2.0 ** -24


@pytest.mark.gpu
def test_numbers_arrive_through_ctypes_too(monkeypatch):
    """Where there is no module of the entry points, numbers in 64 bits reach them by the same declarations."""
    import ctypes
    from pfeife_b200.csrc import build
    from pfeife_b200.ops import _lib
    z, labels = batch(4, 7, 300, "cuda", torch.bfloat16, 3)
    z.requires_grad_()
    v = torch.full((4, 7), -5.0, device="cuda")

    def values():
        with Watch():                              # through the registered ops, not the eager module
            a = ops.preference_loss(z, labels, v[:, 0], 0.3, 0.1)
            b = ops.policy_loss(z, labels, v, v[:, :1] + 6, v + 1, 0.1, 0.3, kl_coef=0.2, temperature=1.3)
            return [*a, *b, *torch.autograd.grad(a.loss + b.loss, z)]
    want = values()
    through = _lib._CtypesCalls(ctypes.CDLL(str(build.KERNEL_LIB), mode=ctypes.RTLD_GLOBAL))
    monkeypatch.setattr(_lib, "_calls", through)
    assert _lib.calls() is through
    assert all(torch.equal(a, b) for a, b in zip(values(), want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,T", [(131072, 2), (151936, 40), (200019, 3)])
def test_large_vocabularies(V, T, dtype):
    """Rows of 128 thousand words and more, in many parts where they are few, some of them masked."""
    z, labels = batch(2, T, V, "cuda", dtype, 6, masked=0.2)
    z[0, 0, 1000:] = torch.finfo(dtype).min
    labels[0, 0], labels[1, 0] = 17, V - 1
    z.requires_grad_()
    l, dl, p, rel, counted = rows64(z.detach(), labels, 1.0)
    l0 = torch.log_softmax(z.detach()[0, 0, :1000].double(), -1)[17]     # the masked row's bound is that of its words
    R = (V / 32 + 68 + 4 * 24) * E + 2.0 ** -22
    dl[0, 0], rel[0, 0] = R + 2 * E * l0.abs(), 2 * R
    out = ops.policy_loss(z, labels, l.float(), torch.ones(2, 1, device="cuda"))
    near(out.logps, l, dl)
    (dz,) = torch.autograd.grad(out.loss, z)
    n = int(counted.sum())
    g = torch.full_like(l, -1.0 / n)
    near(dz, *gradient(g, (1.1 * dl + 8 * E * l.abs().clamp(min=1)) / n, p, rel, labels, counted))
    pref = ops.preference_loss(z, labels, l.sum(1).float(), beta=0.5)
    near(pref.rewards, 0.5 * (l.sum(1) - l.sum(1).float().double()), 0.5 * dl.sum(1) + 4 * E * l.sum(1).abs())
