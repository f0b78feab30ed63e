"""GPU checks of the losses on next-token logits against 64-bit forms: token
log-probabilities, the clipped policy loss, the preference loss, and their
gradients."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


@pytest.fixture(scope="module")
def L():
    from provenloop_b200 import losses
    return losses


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rows(n, v, dt, seed=0, std=3.0):
    """Logits [n, v] and targets, about a third of which do not count."""
    g = _gen(seed)
    z = (torch.randn((n, v), generator=g, device="cuda") * std).to(TYPES[dt])
    y = torch.randint(0, v, (n,), generator=g, device="cuda")
    y[torch.rand((n,), generator=g, device="cuda") < 0.3] = -100
    y[0] = v - 1
    return z, y


# ---------------------------------------------------------------- 64-bit forms


def _forms(z, y, counts=None):
    """(log-probabilities, p, p's allowed relative error, the
    log-probabilities' allowed error, the rows that count) in 64 bits.

    An exp(z - m) is off by a relative 2^-22 for the instruction and 2^-22
    |z - m| for its argument (three roundings of half a step and less, and the
    constant).  A row's sum goes through one exp for each change of the
    reference value: one for each 32 elements of a thread at most, and for each
    of 12 joins of threads and CTAs; their arguments add up to |z - m|.  Its
    additions, at most 16 for each 32 elements and for each join, are off by
    2^-24 each, all of one sign.  The argument's part enters the sum weighted
    by p."""
    d = z.double()
    v = d.shape[1]
    m = d.amax(1, keepdim=True)
    off = torch.where(d == m, 0.0, (m - d).clamp_max(700.0))
    e = torch.exp(d - m)
    e = torch.where(d == m, 1.0, e)
    s = e.sum(1, keepdim=True)
    p = e / s
    counts = (y >= 0) & (y < v) if counts is None else counts & (y >= 0) & (y < v)
    yy = torch.where(counts, y, 0).long()
    l = torch.where(counts, (d.gather(1, yy[:, None]) - m)[:, 0] - s[:, 0].log(), 0.0)
    l = torch.where(counts & (d.gather(1, yy[:, None])[:, 0] == -math.inf), -math.inf, l)
    groups = math.ceil(v / (256 * 4 * 4)) + 2
    rel = 2.0 ** -22 * ((groups + 12) * (1 + 16 / 4) + 2 * (p * off).sum(1))
    p_rel = 2.0 ** -22 * (3 + 2 * off) + rel[:, None]
    return l, p, p_rel, rel, counts


def _near(got, want, tol, what=""):
    got, want = got.double(), want.double()
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)), what
    assert torch.equal(torch.isnan(want), torch.isnan(got)), what
    assert torch.equal(want[~fine & ~torch.isnan(want)], got[~fine & ~torch.isnan(want)]), what
    if not isinstance(tol, torch.Tensor):
        tol = torch.full_like(want, tol)
    off = ((got - want).abs() - tol)[fine]
    assert off.numel() == 0 or off.max() <= 0, f"{what}: worst excess {off.max().item():.3g} of {tol[fine][off.argmax()].item():.3g} allowed"


def _near_logprobs(got, z, y, counts=None):
    l, _, _, rel, _ = _forms(z, y, counts)
    _near(got.view(-1), l, 2.0 ** -24 * l.abs().clamp_max(1e30) + rel, "log-probabilities")


def _near_gradient(got, z, y, g, g_tol, counts=None):
    """got against g ([v = y] - p), g (64 bits) being off by g_tol at most."""
    _, p, p_rel, _, counts = _forms(z, y, counts)
    eps = torch.finfo(z.dtype).eps
    one = torch.zeros_like(p)
    one[torch.arange(len(y), device=y.device), torch.where(counts, y, 0).long()] = 1.0
    g, g_tol = torch.where(counts, g, 0.0)[:, None], torch.where(counts, g_tol, 0.0)[:, None]
    want = torch.where(g == 0, 0.0, g * (one - p))
    # g's own error and rounding, p's, the difference's rounding, half a step of the result's type or of its least values
    tiny = 2.0 ** -25 if z.dtype is torch.float16 else 2.0 ** -125 * (1 + g.abs())
    tol = (g_tol + 2.0 ** -24 * g.abs()) * (one - p).abs() + g.abs() * p * (p_rel + 2.0 ** -23) + 2.0 ** -24 * want.abs()
    _near(got.view(p.shape), want, tol * (1 + eps) + eps / 2 * want.abs() + tiny, "gradient")


def _policy64(l, counts, seq, old, adv, ref, low, high, kl, kind, sequences):
    """(loss, its allowed error for an error of 1 in each l, g, the same for g) for advantages by row."""
    zero = torch.zeros_like(l)
    per = torch.zeros(sequences, dtype=torch.float64, device=l.device).index_add_(0, seq.clamp_min(0), counts.double())
    w = {"token": lambda: counts / per.sum().clamp_min(1), "sequence": lambda: counts / (per[seq.clamp_min(0)].clamp_min(1) * sequences),
         "sum": lambda: counts.double()}[kind]()
    a = adv.double()
    rho = torch.exp(l - old.double()) if old is not None else torch.ones_like(l)
    # as the C entry point takes them: the borders in 32 bits
    low, high, kl = (float(torch.tensor(x, dtype=torch.float32)) for x in (low, high, kl))
    cut = rho.clamp(float(torch.tensor(1.0) - torch.tensor(low)), float(torch.tensor(1.0) + torch.tensor(high)))
    clipped = rho * a > cut * a
    term, by = -torch.where(clipped, cut * a, rho * a), -torch.where(clipped, zero, rho * a)
    more = torch.where(clipped, zero, (rho * a).abs())
    if ref is not None and kl:
        d = ref.double() - l
        term, by, more = term + kl * (torch.expm1(d) - d), by - kl * torch.expm1(d), more + kl * torch.exp(d)
    pick = lambda x: torch.where(counts, w * x, zero)  # noqa: E731
    return pick(term).sum(), pick(by.abs()), pick(by), pick(more)


def _check_policy(L, z, y, old, adv, ref, starts=None, low=0.2, high=0.2, kl=0.0, kind="token", scale=None, **kw):
    shape = y.shape
    sequences = (starts.numel() - 1) if starts is not None else (shape[0] if len(shape) > 1 else 1)
    zz = z.reshape(-1, z.shape[-1]).clone()
    loss, logp, grad = L.policy_loss(z, y, old, adv, ref_logprobs=ref, starts=starts, clip=(low, high), kl=kl, reduction=kind,
                                     grad_scale=scale, **kw)
    yy = y.reshape(-1)
    n = yy.numel()
    at = torch.arange(n, device="cuda")
    if starts is None:
        seq = at // max(1, n // sequences)
        inside = torch.ones(n, dtype=torch.bool, device="cuda")
    else:
        seq = torch.searchsorted(starts.long(), at, right=True) - 1
        inside = (seq >= 0) & (seq < sequences)
        seq = torch.where(inside, seq, 0)
    l, _, _, rel, counts = _forms(zz, yy, inside)
    flat = lambda t: None if t is None else t.reshape(-1)  # noqa: E731
    a = adv.reshape(-1) if adv.shape == y.shape else adv[seq]
    want, dloss, g, dg = _policy64(l, counts, seq, flat(old), a, flat(ref), low, high, kl, kind, sequences)
    _near_logprobs(logp, zz, yy, inside)
    _near(loss.view(1), want.view(1), 2.0 ** -24 * want.abs().item() + (dloss * rel * 1.01).sum().item() + 1e-44, "loss")
    if grad is not None:
        k = 1.0 if scale is None else scale.double()
        _near_gradient(grad, zz, yy, g * k, dg * rel * 1.01 * k + 2.0 ** -50 * g.abs() * k, inside)
    return loss, logp, grad


def _check_preference(L, z, y, ref, starts=None, beta=0.1, kind="sigmoid", smoothing=0.0, average=False, scale=None, **kw):
    shape = y.shape
    sequences = (starts.numel() - 1) if starts is not None else shape[0]
    pairs = sequences // 2
    zz = z.reshape(-1, z.shape[-1]).clone()
    loss, margins, logp, grad = L.preference_loss(z, y, ref, starts=starts, beta=beta, kind=kind, smoothing=smoothing, average=average,
                                                  grad_scale=scale, **kw)
    yy = y.reshape(-1)
    n = yy.numel()
    at = torch.arange(n, device="cuda")
    if starts is None:
        member = (at // max(1, n // sequences) == torch.arange(sequences, device="cuda")[:, None])
    else:
        member = (at >= starts[:-1, None]) & (at < starts[1:, None])
    inside = member.any(0)
    l, _, _, rel, counts = _forms(zz, yy, inside)
    member = (member & counts).double()
    if average:
        member = member / member.sum(1, keepdim=True).clamp_min(1)
    lead = torch.where(counts, l - (ref.reshape(-1).double() if ref is not None else 0.0), 0.0)
    lead, off = member @ lead, member @ (rel + 2.0 ** -50 * lead.abs())
    d, d_off = lead[:pairs] - lead[pairs:], off[:pairs] + off[pairs:]
    b, e = (float(torch.tensor(x, dtype=torch.float32)) for x in (beta, smoothing))
    h = b * d
    sig = torch.sigmoid
    if kind == "sigmoid":
        part = -(1 - e) * torch.nn.functional.logsigmoid(h) - e * torch.nn.functional.logsigmoid(-h)
        slope, curve = b * (e * sig(h) - (1 - e) * sig(-h)), b * b * sig(h) * sig(-h) + 1e-18 * b
    elif kind == "hinge":
        part, slope, curve = (1 - h).clamp_min(0), -b * (h < 1).double(), 0.0 * h
    else:
        part, slope, curve = (d - 0.5 / b) ** 2, 2 * (d - 0.5 / b), 2.0 + 0.0 * h
    _near_logprobs(logp, zz, yy, inside)
    _near(margins, h, 2.0 ** -24 * h.abs() + b * d_off, "margins")
    # to second order: the slope, and half the curve of the error's square
    _near(loss.view(1), part.mean().view(1), 2.0 ** -23 * part.mean().item() + ((slope.abs() + curve * d_off) * d_off).mean().item(), "loss")
    if grad is not None:
        k = 1.0 if scale is None else scale.double()
        g = torch.cat([slope, -slope]) @ member / pairs * k
        g_off = torch.cat([curve * d_off * 1.01] * 2) @ member / pairs * k + 2.0 ** -24 * g.abs()
        _near_gradient(grad, zz, yy, g, g_off, inside)
    return loss, margins, logp, grad


# ---------------------------------------------------------------- sizes and types

SIZES = [(1, 151936), (1, 1), (2, 7), (3, 31), (5, 1000), (40, 4097), (7, 50257), (160, 9001), (31, 151936), (701, 2049), (3, 400003)]


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("n,v", SIZES)
def test_token_logprobs_and_gradient(L, n, v, dt):
    z, y = _rows(n, v, dt, seed=n + v)
    got = L.token_logprobs(z, y)
    assert got.dtype == torch.float32 and got.shape == y.shape
    _near_logprobs(got, z, y)
    g = torch.randn((n,), generator=_gen(1), device="cuda")
    if n > 4:
        g[3] = 0.0
    grad = L.token_logprobs_backward(g, z, y)
    assert grad.dtype == z.dtype and grad.shape == z.shape
    _near_gradient(grad, z, y, g.double(), torch.zeros_like(g.double()))


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("pad,cut", [(0, 1), (3, 0), (5, 2), (8, 0)])
def test_rows_off_16_bytes(L, dt, pad, cut):
    """Strided rows, the gradient's rows on another phase than the logits'."""
    n, v = 23, 1537
    whole, y = _rows(n, v + pad + cut, dt, seed=pad)
    z = whole[:, cut:cut + v]
    y = y.clamp_max(v - 1)
    _near_logprobs(L.token_logprobs(z, y), z, y)
    g = torch.randn((n,), generator=_gen(2), device="cuda")
    for out in (None, torch.full((n, v + 1), 7.0, dtype=z.dtype, device="cuda")[:, 1:], torch.full((n, v + 9), 7.0, dtype=z.dtype, device="cuda")[:, 1:v + 1]):
        got = L.token_logprobs_backward(g, z, y, out=out)
        assert out is None or got is out
        _near_gradient(got, z, y, g.double(), torch.zeros_like(g.double()))
        if out is not None:
            assert (out._base[:, 0] == 7).all() and (out._base[:, v + 1:] == 7).all()
    keep, before = z.clone(), whole.clone()
    assert L.token_logprobs_backward(g, z, y, out=z) is z
    _near_gradient(z, keep, y, g.double(), torch.zeros_like(g.double()))
    assert torch.equal(whole[:, :cut], before[:, :cut]) and torch.equal(whole[:, cut + v:], before[:, cut + v:])


@pytest.mark.parametrize("ints", [torch.int32, torch.int64])
def test_targets_outside_the_vocabulary(L, ints):
    z, _ = _rows(6, 100, "bf16")
    y = torch.tensor([0, -1, 100, 99, -100, 2 ** 31 - 1], device="cuda", dtype=ints)
    if ints is torch.int64:
        y[1], y[2] = 2 ** 32 + 5, -2 ** 63
    z[1], z[2], z[4] = math.nan, math.inf, -math.inf  # rows that do not count may hold anything
    got, grad = L.token_logprobs(z, y), L.token_logprobs_backward(torch.ones(6, device="cuda"), z, y)
    assert (got[[1, 2, 4, 5]] == 0).all() and (grad[[1, 2, 4, 5]] == 0).all()
    keep = torch.tensor([0, 3], device="cuda")
    _near_logprobs(got[keep], z[keep], y[keep])
    _near_gradient(grad[keep], z[keep], y[keep], torch.ones(2, device="cuda").double(), torch.zeros(2, device="cuda").double())


def _policy_inputs(z, y, seed=3, per_row=False):
    """Old log-probabilities near the present ones, reference ones a little further, none of the ratios on a border."""
    g = _gen(seed)
    l = _forms(z.reshape(-1, z.shape[-1]), y.reshape(-1))[0]
    moved = 0.25 * torch.randn(l.shape, generator=g, device="cuda", dtype=torch.float64)
    for border in (math.log(0.8), math.log(1.2), math.log(0.9), math.log(1.3)):
        moved = torch.where((moved - border).abs() < 1e-3, border + 2e-3, moved)
    old = (l - moved).float().view(y.shape)
    ref = (l + 0.3 * torch.randn(l.shape, generator=g, device="cuda")).float().view(y.shape)
    adv = torch.randn(y.shape if per_row else y.shape[:1], generator=g, device="cuda")
    return old, adv, ref


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("kind", ["token", "sequence", "sum"])
@pytest.mark.parametrize("s,t,v", [(1, 1, 151936), (3, 5, 997), (4, 33, 4099), (11, 20, 50257), (40, 30, 300)])
def test_policy_loss(L, s, t, v, dt, kind):
    z, y = _rows(s * t, v, dt, seed=s + v)
    z, y = z.view(s, t, v), y.view(s, t)
    if s > 2:
        y[1] = -100  # a sequence in which no row counts
    old, adv, ref = _policy_inputs(z, y)
    scale = torch.tensor(3.0, device="cuda")
    _check_policy(L, z, y, old, adv, ref, kl=0.04, kind=kind, scale=scale)
    _check_policy(L, z, y, old, adv, None, kind=kind, low=0.1, high=0.3)
    old, adv, ref = _policy_inputs(z, y, per_row=True)
    _check_policy(L, z, y, None, adv, ref, kl=0.2, kind=kind, need_grad=False)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("kind", ["token", "sequence"])
@pytest.mark.parametrize("cuts", [[0, 3, 3, 17, 40], [2, 9, 38, 38], [0, 0], [5, 40], [0, 41], [0] + list(range(1, 41))])
def test_policy_loss_of_packed_sequences(L, cuts, dt, kind):
    z, y = _rows(41, 1111, dt, seed=9)
    starts = torch.tensor(cuts, dtype=torch.int32, device="cuda")
    old, _, ref = _policy_inputs(z, y)
    adv = torch.randn((len(cuts) - 1,), generator=_gen(4), device="cuda")
    loss, logp, grad = _check_policy(L, z, y, old, adv, ref, starts=starts, kl=0.1, kind=kind)
    outside = torch.ones(41, dtype=torch.bool)
    outside[cuts[0]:cuts[-1]] = False
    assert (grad[outside.cuda()] == 0).all() and (logp[outside.cuda()] == 0).all()


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("kind,smoothing", [("sigmoid", 0.0), ("sigmoid", 0.2), ("hinge", 0.0), ("squared", 0.0)])
@pytest.mark.parametrize("s,t,v", [(2, 1, 151936), (6, 13, 997), (4, 70, 4099), (16, 300, 260)])
def test_preference_loss(L, s, t, v, dt, kind, smoothing):
    z, y = _rows(s * t, v, dt, seed=s + v)
    z, y = z.view(s, t, v), y.view(s, t)
    if s > 2:
        y[2] = -100
    l = _forms(z.reshape(-1, v), y.reshape(-1))[0].view(s, t)
    ref = (l + 0.1 * torch.randn((s, t), generator=_gen(5), device="cuda")).float()
    scale = torch.tensor([0.5], device="cuda")
    _check_preference(L, z, y, ref, kind=kind, smoothing=smoothing, beta=0.3, scale=scale)
    _check_preference(L, z, y, ref, kind=kind, smoothing=smoothing, average=True)
    _check_preference(L, z, y, None, kind=kind, smoothing=smoothing, beta=0.01, need_grad=False)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("cuts", [[0, 3, 17], [4, 4, 19, 30, 41], [0, 0, 0], [0, 10, 10, 12, 40]])
def test_preference_loss_of_packed_pairs(L, cuts, average, dt):
    z, y = _rows(41, 1111, dt, seed=11)
    starts = torch.tensor(cuts, dtype=torch.int32, device="cuda")
    ref = torch.randn((41,), generator=_gen(6), device="cuda") - 9
    _, _, logp, grad = _check_preference(L, z, y, ref, starts=starts, average=average)
    outside = torch.ones(41, dtype=torch.bool)
    outside[cuts[0]:cuts[-1]] = False
    assert (grad[outside.cuda()] == 0).all() and (logp[outside.cuda()] == 0).all()


# ---------------------------------------------------------------- values out of the ordinary


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("v", [33, 1000, 151936])
def test_masked_and_extreme_logits(L, v, dt):
    """Rows masked by -inf or by the type's lowest value, in part or throughout, rows of large values, of one
    value, and rows whose target is masked."""
    t, g = TYPES[dt], _gen(12)
    low, big = torch.finfo(t).min, torch.finfo(t).max
    z = (torch.randn((10, v), generator=g, device="cuda") * 3).to(t)
    y = torch.randint(0, v, (10,), generator=g, device="cuda")
    z[0, torch.arange(v, device="cuda") != y[0]] = -math.inf  # one token left
    z[1, : v // 2], y[1] = -math.inf, v - 1
    z[2] = low  # uniform
    z[3, : v // 2], y[3] = low, v - 1
    z[4] = big
    z[5] = 0.0
    z[6, 5] = big
    z[7, y[7]] = -math.inf  # the target masked
    z[8, y[8]] = low
    z[9] *= 100
    got = L.token_logprobs(z, y)
    _near_logprobs(got, z, y)
    assert got[7] == -math.inf and got[0] == 0
    grad = L.token_logprobs_backward(torch.ones(10, device="cuda"), z, y)
    _near_gradient(grad, z, y, torch.ones(10, device="cuda").double(), torch.zeros(10, device="cuda").double())
    assert (grad[0] == 0).all() and (grad[1, : v // 2] == 0).all()


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_not_numbers_stay_in_their_rows(L, dt):
    z, y = _rows(12, 5000, dt)
    y = y.clamp_min(0)
    z[2, 77], z[5, 4321], z[8] = math.nan, math.inf, -math.inf
    got = L.token_logprobs(z, y)
    assert torch.isnan(got[2]) and torch.isnan(got[5]) and got[8] == -math.inf
    others = torch.tensor([0, 1, 3, 4, 6, 7, 9, 10, 11], device="cuda")
    _near_logprobs(got[others], z[others], y[others])
    g = torch.ones(12, device="cuda")
    grad = L.token_logprobs_backward(g, z, y)
    assert torch.isnan(grad[2]).all() and torch.isnan(grad[5, 4321])
    _near_gradient(grad[others], z[others], y[others], g[others].double(), torch.zeros_like(g[others].double()))
    g[2] = g[5] = g[8] = 0.0  # not wanted: zeros
    grad = L.token_logprobs_backward(g, z, y)
    assert (grad[[2, 5, 8]] == 0).all()
    loss, logp, grad = L.policy_loss(z, y, None, torch.ones(12, device="cuda"))
    assert torch.isnan(loss) and torch.isnan(grad[2]).all() and torch.isfinite(grad[others]).all()
    loss, margins, logp, grad = L.preference_loss(z.view(12, 1, 5000), y.view(12, 1))
    assert torch.isnan(loss) and torch.isnan(margins[2]) and torch.isnan(margins[5])
    keep = torch.tensor([0, 1, 3, 4, 6, 7, 9, 10], device="cuda")  # pairs 0, 1, 3 and 4
    assert torch.isfinite(margins[[0, 1, 3, 4]]).all() and torch.isfinite(grad.view(12, -1)[keep]).all()


def test_policy_ratios_far_off(L):
    """Ratios of 0 and beyond the range, advantages of both signs and 0; borders count as not clipped."""
    z, y = _rows(8, 300, "fp32")
    y = y.clamp_min(0)
    l = L.token_logprobs(z, y)
    old = l.clone()
    old[0], old[1], old[2], old[3] = l[0] + 200, l[1] + 200, l[2] - 60, l[3] - 60
    adv = torch.tensor([1.0, -1.0, 1.0, -1.0, 0.0, 2.0, -2.0, 1.0], device="cuda")
    _check_policy(L, z, y, old, adv, None)
    # clipping of width 0: rho = 1 lies on both borders
    loss, _, grad = L.policy_loss(z, y, None, adv, clip=(0.0, 0.0), reduction="sum")
    _near(loss.view(1), -adv.double().sum().view(1), 1e-6)
    _near_gradient(grad, z, y, -adv.double(), torch.zeros(8, device="cuda").double())


def test_nothing_counts(L):
    z, y = _rows(12, 500, "bf16")
    z[:] = math.nan
    y[:] = -100
    adv = torch.ones(12, device="cuda")
    for kind in ("token", "sequence", "sum"):
        loss, logp, grad = L.policy_loss(z, y, None, adv, reduction=kind)
        assert loss == 0 and (logp == 0).all() and (grad == 0).all()
    loss, margins, logp, grad = L.preference_loss(z.view(4, 3, 500), y.view(4, 3))
    _near(loss.view(1), torch.tensor([math.log(2.0)], device="cuda"), 1e-7)
    assert (margins == 0).all() and (logp == 0).all() and (grad == 0).all()


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_no_rows(L, dt):
    z, y = torch.empty((0, 100), dtype=TYPES[dt], device="cuda"), torch.empty((0,), dtype=torch.int64, device="cuda")
    assert L.token_logprobs(z, y).shape == (0,)
    assert L.token_logprobs_backward(torch.empty(0, device="cuda"), z, y).shape == (0, 100)
    for shape in ((0,), (3, 0), (0, 5)):
        zz, yy = z.view(*shape, 100), y.view(shape)
        loss, logp, grad = L.policy_loss(zz, yy, None, torch.empty(shape, device="cuda"))
        assert loss == 0 and logp.shape == shape and grad.shape == zz.shape
    loss, margins, _, _ = L.preference_loss(z.view(4, 0, 100), y.view(4, 0))
    _near(loss.view(1), torch.tensor([math.log(2.0)], device="cuda"), 1e-7)
    assert (margins == 0).all() and margins.shape == (2,)
    loss, margins, _, _ = L.preference_loss(z.view(0, 7, 100), y.view(0, 7))
    assert loss == 0 and margins.shape == (0,)


# ---------------------------------------------------------------- calls out of the ordinary


def _everything(L, s):
    """One call of each, on new results."""
    out = [L.token_logprobs(s["z"], s["y"]), L.token_logprobs_backward(s["g"], s["z"], s["y"])]
    out += L.policy_loss(s["z"], s["y"], s["old"], s["adv"], s["ref"], kl=0.1, reduction="sequence")
    out += L.preference_loss(s["z"], s["y"], s["ref"], average=True)
    return out


def _everything_inputs(dt, seed, s=6, t=17, v=3001):
    z, y = _rows(s * t, v, dt, seed=seed)
    z, y = z.view(s, t, v), y.view(s, t)
    old, adv, ref = _policy_inputs(z, y, seed=seed)
    return dict(z=z, y=y, old=old, adv=adv, ref=ref, g=torch.randn((s, t), generator=_gen(seed), device="cuda"))


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_same_bits_every_time_and_on_every_stream(L, dt):
    s = _everything_inputs(dt, 1)
    want = _everything(L, s)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for stream in streams:
            with torch.cuda.stream(stream):
                got.append(_everything(L, s))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_captured_calls_read_new_values(L, dt):
    live = _everything_inputs(dt, 1)
    other = _everything_inputs(dt, 2)
    want = [[t.clone() for t in _everything(L, s)] for s in (live, other)]
    first = {k: v.clone() for k, v in live.items()}
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):  # two graphs of one pool
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append(_everything(L, live))
        graphs.append(graph)
    for k, s in ((1, other), (0, first), (1, other)):
        for name, t in s.items():
            live[name].copy_(t)
        for graph, out in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want[k]))


def test_calls_queued_one_behind_the_other(L):
    """Many calls of changing sizes, faster than the GPU works them off, each result as when it is alone."""
    data = [_everything_inputs("bf16", k, s=2 + 2 * (k % 3), t=3 + 5 * k, v=1000 + 777 * k) for k in range(4)]
    want = []
    for s in data:
        want.append([t.clone() for t in _everything(L, s)])
        torch.cuda.synchronize()
    busy = torch.randn((4096, 4096), device="cuda")
    got = []
    for _ in range(4):
        busy @ busy
        got += [_everything(L, s) for s in data]
    torch.cuda.synchronize()
    for k, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[k % 4]))


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_gradient_in_place_of_the_logits(L, dt):
    s = _everything_inputs(dt, 3)
    policy = L.policy_loss(s["z"], s["y"], s["old"], s["adv"], s["ref"], kl=0.1)
    prefer = L.preference_loss(s["z"], s["y"], s["ref"])
    for call, want in ((lambda z: L.policy_loss(z, s["y"], s["old"], s["adv"], s["ref"], kl=0.1, out=z), policy),
                       (lambda z: L.preference_loss(z, s["y"], s["ref"], out=z), prefer)):
        z = s["z"].clone()
        version = z._version
        got = call(z)
        assert got[-1] is z and z._version > version
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_rows_beyond_32_bits(L):
    """Rows further apart than 2^31 elements."""
    v, stride = 1000, 2 ** 31 + 8
    whole = torch.empty((stride + v,), dtype=torch.bfloat16, device="cuda")
    z = whole.as_strided((2, v), (stride, 1))
    z.copy_(_rows(2, v, "bf16")[0])
    y = torch.tensor([5, 999], device="cuda")
    keep = z.clone()
    _near_logprobs(L.token_logprobs(z, y), keep, y)
    adv = torch.tensor([1.0, -2.0], device="cuda")
    _check_policy(L, z, y, None, adv, None)
    L.token_logprobs_backward(adv, z, y, out=z)
    _near_gradient(z, keep, y, adv.double(), torch.zeros(2, device="cuda").double())


@pytest.mark.parametrize("dt,v", [("bf16", 1200000), ("fp32", 600011)])
def test_long_rows(L, dt, v):
    z, y = _rows(3, v, dt, seed=1)
    y = y.clamp_min(0)
    _near_logprobs(L.token_logprobs(z, y), z, y)
    _check_policy(L, z, y, None, torch.tensor([1.0, -0.5, 2.0], device="cuda"), None)


def test_gradients_against_differences(L):
    """Loss differences along a direction, in 32 bits: each loss is off by 2^-24 of
    itself and by its rows' errors times their slopes (half of the gradient's sum
    of absolute values at most), the difference by h^2 / 6 of the third derivative,
    which along a unit direction is below three times the loss's size here."""
    s, t, v = 4, 5, 50
    z, y = _rows(s * t, v, "fp32", seed=20, std=1.0)
    z, y = z.view(s, t, v), y.view(s, t).clamp_min(0)
    _, adv, ref = _policy_inputs(z, y)
    old = L.token_logprobs(z, y) + 0.05  # ratios far from the borders
    h = 2.0 ** -6
    rel = _forms(z.reshape(-1, v), y.reshape(-1))[3].max().item()
    calls = [lambda x: L.policy_loss(x, y, old, adv, ref, clip=(0.5, 0.5), kl=0.1, reduction="sum"),
             lambda x: L.preference_loss(x, y, ref, beta=0.5), lambda x: L.preference_loss(x, y, ref, beta=0.5, kind="squared", average=True)]
    for call in calls:
        out = call(z)
        grad = out[-1].double()
        u = torch.randn(z.shape, generator=_gen(21), device="cuda").double()
        u = (u / u.norm() + grad / grad.norm())
        u /= u.norm()
        up, down = (call((z.double() + k * u).float())[0].double() for k in (h, -h))
        size = 1.0 + abs(out[0].item())
        tol = (2.0 ** -23 * size + grad.abs().sum().item() * (rel + 2.0 ** -22)) / h + 3 * size * h * h
        assert abs((up - down) / (2 * h) - (grad * u).sum()) <= tol and tol < 0.05 * (grad * u).sum().abs()


# ---------------------------------------------------------------- rows by the hundred, which persistent clusters share


def _padded(s, t, v, dt, seed=0):
    """Sequences of ragged lengths behind prompts, padded: about half of the rows count."""
    z, y = _rows(s * t, v, dt, seed=seed)
    z, y = z.view(s, t, v), torch.randint(0, v, (s, t), generator=_gen(seed), device="cuda")
    at = torch.arange(t, device="cuda")
    ends = torch.randint(1, t + 1, (s, 1), generator=_gen(seed + 1), device="cuda")
    prompts = (ends * torch.rand((s, 1), generator=_gen(seed + 2), device="cuda") * 0.6).long()
    return z, torch.where((at >= prompts) & (at < ends), y, -100)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("s,t,v", [(6, 300, 5003), (40, 31, 9001), (3, 111, 33001), (2, 100, 151936)])
def test_padded_batches(L, s, t, v, dt):
    z, y = _padded(s, t, v, dt, seed=s)
    old, adv, ref = _policy_inputs(z, y)
    flat, yy = z.view(-1, v), y.view(-1)
    _near_logprobs(L.token_logprobs(z, y), flat, yy)
    g = torch.randn((s, t), generator=_gen(7), device="cuda")
    g[0, :5] = 0.0
    _near_gradient(L.token_logprobs_backward(g, z, y), flat, yy, g.double().view(-1), torch.zeros_like(g).double().view(-1))
    out = torch.full_like(z, 7.0)
    _check_policy(L, z, y, old, adv, ref, kl=0.04, kind="sequence", out=out)
    if s % 2 == 0:
        _check_preference(L, z, y, ref, average=True, out=out)
        _check_preference(L, z, y, ref, kind="squared", beta=0.3, out=z)  # in place


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("count", ["none", "one", "all"])
def test_batches_in_which_few_or_all_rows_count(L, count, dt):
    n, v = 1300, 5000
    z, y = _rows(n, v, dt, seed=3)
    y = y.clamp_min(0)
    if count != "all":
        keep = y[777].item()
        z[:777], z[778:] = math.nan, math.nan
        y[:] = -1
        if count == "one":
            y[777] = keep
    adv = torch.ones((n,), device="cuda")
    loss, logp, grad = L.policy_loss(z, y, None, adv)
    used = (y >= 0).nonzero()[:, 0]
    assert loss == (-1 if len(used) else 0) and (logp[y < 0] == 0).all() and (grad[y < 0] == 0).all()
    _near_logprobs(logp[used], z[used], y[used])
    one = torch.full((len(used),), -1.0 / max(1, len(used)), dtype=torch.float64, device="cuda")
    if len(used):
        _near_gradient(grad[used], z[used], y[used], one, 2.0 ** -24 * one.abs())


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [3, 300, 700])
@pytest.mark.parametrize("v", [2040, 2041, 4088, 4089, 8188, 8189, 16376, 16377, 20472, 20480, 40945, 81920, 163840])
def test_where_the_kernels_change(L, v, n, dt):
    """Vocabularies at the lengths that threads, CTAs and clusters can hold."""
    if n * v > 60e6:
        n = 150
    z, y = _rows(n, v + 3, dt, seed=v)
    z, y = z[:, 3:], y.clamp_max(v - 1)  # rows off 16-byte boundaries
    g = torch.randn((n,), generator=_gen(8), device="cuda")
    _near_logprobs(L.token_logprobs(z, y), z, y)
    _near_gradient(L.token_logprobs_backward(g, z, y), z, y, g.double(), torch.zeros(n, device="cuda").double())


@pytest.mark.parametrize("n", [1023, 1024, 1025, 4097, 262147, 1050001])
def test_losses_of_many_rows(L, n):
    """Losses that are sums of sums: of groups of rows or pairs, and of groups of those."""
    z, y = _rows(n, 8, "bf16", seed=n)
    old, adv, ref = _policy_inputs(z, y, per_row=True)
    for kind in ("token", "sum"):
        _check_policy(L, z, y, old, adv, ref, kl=0.1, kind=kind)
    starts = torch.cat([torch.arange(0, n, 7, device="cuda"), torch.tensor([n], device="cuda")]).int()
    _check_policy(L, z, y, old, adv, None, starts=starts, kind="sequence")
    # as pairs of single tokens: the loss is the margins' mean form
    z, y = z[:n // 2 * 2], y[:n // 2 * 2]
    loss, margins, logp, _ = L.preference_loss(z.view(-1, 1, 8), y.view(-1, 1), beta=0.5)
    _near_logprobs(logp, z, y)
    h = 0.5 * (logp[:n // 2].double() - logp[n // 2:].double()).view(-1)
    _near(margins, h, 2.0 ** -24 * (logp[:n // 2].abs() + logp[n // 2:].abs()).view(-1).double() + 2.0 ** -24 * h.abs(), "margins")
    want = torch.nn.functional.softplus(-margins.double()).mean()
    _near(loss.view(1), want.view(1), 2.0 ** -24 * (want.item() + margins.double().abs().mean().item()), "loss")


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("n,v", [(2, 5), (1185, 1017), (1185, 2041), (9001, 500), (19001, 1016), (19001, 2040), (18945, 4088)])
def test_many_short_rows(L, n, v, dt):
    """As many as a warp, or a CTA, takes each, and more of them than run at once; rows off 16-byte boundaries too."""
    z, y = _rows(n, v + 3, dt, seed=v)
    wide, y = torch.empty_like(z), y.clamp_max(v - 1)
    z, out = z[:, 3:], wide[:, 1:v + 1]  # not the same offset
    g = torch.randn((n,), generator=_gen(8), device="cuda")
    g[n // 2] = 0.0
    _near_logprobs(L.token_logprobs(z, y), z, y)
    _near_gradient(L.token_logprobs_backward(g, z, y, out=out), z, y, g.double(), torch.zeros(n, device="cuda").double())
    starts = torch.tensor(sorted([1, n // 3, n // 3, n // 2, n]), dtype=torch.int32, device="cuda")  # ascending with two rows too
    adv = torch.randn((4,), generator=_gen(9), device="cuda")
    old, _, ref = _policy_inputs(z, y)
    for kind in ("token", "sequence"):
        _check_policy(L, z, y, old, adv, ref, starts=starts, kl=0.1, kind=kind)
    _check_preference(L, z, y, ref, starts=starts, average=True)
    mine = z.contiguous()  # the sums' order goes by the rows' offsets from 16-byte boundaries: the same tensor twice
    want = L.preference_loss(mine, y, ref, starts=starts, average=True)
    loss, _, _, grad = L.preference_loss(mine, y, ref, starts=starts, average=True, out=mine)
    assert grad is mine and torch.equal(loss, want[0]) and torch.equal(mine, want[3])


@pytest.mark.parametrize("n,v,dt", [(18945, 4088, "fp32"), (6000, 8000, "bf16"), (3000, 20000, "fp16"), (2000, 50257, "fp32"), (900, 151936, "bf16")])
def test_same_bits_however_the_copies_arrive(L, n, v, dt):
    """Many rows through the slots of a ring, many times: each load of a slot is done before the next copy into it."""
    z, y = _rows(n, v, dt, seed=n)
    adv = torch.randn((n,), generator=_gen(1), device="cuda")
    starts = torch.tensor([1, n // 3, n // 3, n // 2, n], dtype=torch.int32, device="cuda")

    def everything():
        return (L.token_logprobs(z, y), L.token_logprobs_backward(adv, z, y), *L.policy_loss(z, y, None, adv),
                *L.preference_loss(z, y, starts=starts, average=True))

    want = everything()
    _near_logprobs(want[0][:300], z[:300], y[:300])
    bad = sum((~(a == b)).sum() for _ in range(20) for a, b in zip(everything(), want))
    assert bad == 0


def test_no_wait_ran_out():
    from provenloop_b200 import adapters
    assert adapters.expired_waits() == 0
