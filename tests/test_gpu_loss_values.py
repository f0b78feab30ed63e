"""GPU checks of the losses at values where a formula's parts are infinite or
cancel, against its limits and 64-bit forms."""
import math

import pytest
import torch

from tests.test_gpu_losses import TYPES, L, _device, _gen  # noqa: F401

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- preference losses of masked targets

# a pair's loss by its margin h = beta d, and the loss's slope by d, at d = inf and d = -inf
LIMITS = {("sigmoid", 0.0): ((0.0, 0.0), (math.inf, -1.0)), ("sigmoid", 0.25): ((math.inf, 0.25), (math.inf, -0.75)),
          ("hinge", 0.0): ((0.0, 0.0), (math.inf, -1.0)), ("squared", 0.0): ((math.inf, math.inf), (math.inf, -math.inf))}


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("kind,smoothing", LIMITS)
@pytest.mark.parametrize("average", [False, True])
def test_preference_loss_of_masked_targets(L, kind, smoothing, average, dt):  # noqa: F811
    """Pairs of three tokens, one target masked by -inf in the rejected sequence, in the chosen one, in both, in none."""
    beta, pairs, t, v = 0.5, 4, 3, 300
    z = (torch.randn((2 * pairs, t, v), generator=_gen(3), device="cuda") * 2).to(TYPES[dt])
    y = torch.randint(0, v, (2 * pairs, t), generator=_gen(4), device="cuda")
    masked = ((pairs + 0, 1), (1, 2), (2, 0), (pairs + 2, 2))
    for s, i in masked:
        z[s, i, y[s, i]] = -math.inf
    loss, margins, logp, grad = L.preference_loss(z, y, beta=beta, kind=kind, smoothing=smoothing, average=average)
    assert torch.isnan(loss) and margins[0] == math.inf and margins[1] == -math.inf and torch.isnan(margins[2]) and torch.isfinite(margins[3])
    assert all(logp[s, i] == -math.inf for s, i in masked) and torch.isfinite(logp).sum() == 2 * pairs * t - 4
    # without the pair of both: its loss is no number by its formula
    keep = [0, 1, 3]
    both = keep + [pairs + p for p in keep]
    rest, _, _, grad = L.preference_loss(z[both], y[both], beta=beta, kind=kind, smoothing=smoothing, average=average)
    up, down = LIMITS[kind, smoothing]
    assert rest == max(up[0], down[0]) and not torch.isnan(rest)
    for k, (_, slope) in ((0, up), (1, down)):
        one = [keep[k], pairs + keep[k]]
        loss, margins, _, grad = L.preference_loss(z[one], y[one], beta=beta, kind=kind, smoothing=smoothing, average=average)
        assert loss == (up, down)[k][0]
        if not math.isfinite(slope):
            continue
        g = slope * (1.0 if kind == "squared" else beta) / (t if average else 1)
        p = torch.softmax(z[one].double(), 2)
        want = torch.stack([torch.full((t,), g), torch.full((t,), -g)]).to(p)[:, :, None] * (torch.nn.functional.one_hot(y[one], v) - p)
        # p by 2^-17 of itself (sums of a row and distances up to 20), the type's rounding, fp16's least values
        assert ((grad.double() - want).abs() <= torch.finfo(z.dtype).eps / 2 * want.abs() + 2.0 ** -17 * abs(g) * p + 2.0 ** -24 * abs(g) + 2.0 ** -25).all()


# ---------------------------------------------------------------- f32: as near as 32 bits allow


@pytest.mark.parametrize("n,v", [(1, 40), (3, 2041), (40, 9001), (3, 151936), (300, 20000), (40, 400003)])
def test_exponentials_far_from_the_maximum(L, n, v):  # noqa: F811
    """Gradients of f32 logits, which are multiples of 1/8 here, so that their differences are exact: warps,
    CTAs and clusters to a row, and the ring.

    -g p is an exp by ex2.approx (2^-22), corrected by a constant's 2^-28 |d| and rounded (2^-24), times -g / s,
    rounded (2^-24).  The rest is s, which all of a row's elements share: their quotients by p lie within those
    3 2^-23 + 80 2^-28 of one value.  s >= 1 is a sum of the maximum's 1 and of exps off by 2^-22 (1 + |d|) each, and
    of additions that are off by half a step of s, 2^-24 of it, each.  Those that the 1 goes through: six in a
    group of 16 elements, one for each later group of the thread (of 256 threads or more), and at most 42 for the
    warps, lanes and CTAs.  -g / s is off by 2^-24 more."""
    g = _gen(v)
    z = -torch.randint(80, 640, (n, v), generator=g, device="cuda").float() / 8  # 10 to 80 below the maximum
    y = torch.randint(0, v, (n,), generator=g, device="cuda")
    top = torch.randint(0, v, (n,), generator=g, device="cuda")
    z[torch.arange(n, device="cuda"), top] = 0.0
    grad = L.token_logprobs_backward(torch.ones(n, device="cuda"), z, y)
    logp = L.token_logprobs(z, y)
    d = z.double()
    s = torch.exp(d).sum(1, keepdim=True)
    p = torch.exp(d) / s
    exp_off = 3 * 2.0 ** -23 + 80 * 2.0 ** -28
    s_off = (p * torch.where(d < 0, 1 - d, 0.0)).sum(1, keepdim=True) * 2.0 ** -22 + (v / 4096 + 48) * 2.0 ** -24
    off = torch.arange(v, device="cuda") != y[:, None]
    by = -grad.double() / p
    assert ((by - 1).abs() <= s_off + 2.0 ** -24 + exp_off)[off].all()
    high, low = torch.where(off, by, 0.0).amax(1), torch.where(off, by, 2.0).amin(1)
    assert (high - low <= 2 * exp_off * high).all()
    at = torch.arange(n, device="cuda")
    want = d[at, y] - s.log()[:, 0]
    assert ((logp.double() - want).abs() <= 2.0 ** -24 * want.abs() + s_off[:, 0] + 2.0 ** -24).all()


# ---------------------------------------------------------------- the policy loss's ratio and KL term: 64 bits


def _two(n, dt="fp32"):
    """Logits of two tokens that are alike: every log-probability is -log 2, every probability a half."""
    z = torch.randn((n, 1), generator=_gen(5), device="cuda").to(TYPES[dt]).expand(n, 2).contiguous()
    return z, torch.randint(0, 2, (n,), generator=_gen(6), device="cuda")


def _row_by_row(L, n, one, want, slope):
    """Each row's loss by a call of its own, and all gradients by one.  The loss and g are
    rounded to 32 bits (2^-24), g p and g - g p too."""
    z, y = _two(n)
    for i in range(n):
        assert abs(L.policy_loss(z[i:i + 1], y[i:i + 1], reduction="sum", need_grad=False, **one(slice(i, i + 1)))[0].double() - want[i]) <= 2.0 ** -23.99 * want[i].abs()
    grad = L.policy_loss(z, y, reduction="sum", **one(slice(0, n)))[2].double()
    sign = torch.where(torch.arange(2, device="cuda") == y[:, None], 0.5, -0.5)
    assert ((grad - slope[:, None] * sign).abs() <= 2.0 ** -22.9 * 0.5 * slope[:, None].abs()).all()


def test_policy_ratios_in_64_bits(L):  # noqa: F811
    """Ratios between exp(-60) and exp(60) that nothing clips."""
    n = 48
    old = -math.log(2) - 60 * (2 * torch.rand((n,), generator=_gen(7), device="cuda") - 1)
    rho = torch.exp(-math.log(2) - old.double())
    adv = torch.where(rho > 1, -1.0, 1.0).float()  # a ratio above 1 counts whole where it harms, one below where it helps
    _row_by_row(L, n, lambda at: dict(old_logprobs=old[at], advantages=adv[at]), -rho * adv, -rho * adv)


def test_policy_divergence_in_64_bits(L):  # noqa: F811
    """exp(d) - 1 - d on both sides of the place where its series takes over, and far off."""
    d = torch.tensor([1e-6, -3e-4, 0.01, -0.1, 0.2, 0.249, 0.251, -0.249, -0.251, 0.26, 0.3, -0.3, 0.5, -0.7, 1.0, -2.0, 5.0, -9.0, 30.0, -50.0], device="cuda")
    ref = -math.log(2) + d
    d = ref.double() + math.log(2)
    # exp(d) - 1 - d as a sum of its series' terms where it cancels
    want, term = torch.zeros_like(d), d.clone()
    for k in range(2, 60):
        term = term * d / k
        want += term
    want = torch.where(d.abs() < 2, want, torch.expm1(d) - d)
    zero = torch.zeros(len(d), device="cuda")
    _row_by_row(L, len(d), lambda at: dict(old_logprobs=None, advantages=zero[at], ref_logprobs=ref[at], kl=0.5), 0.5 * want, -0.5 * torch.expm1(d))


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_policy_loss_of_masked_targets(L, dt):  # noqa: F811
    """A target masked by -inf: the ratio is 0, or 1 without old log-probabilities; the KL term is infinite for a finite
    reference, as its limit is, and finite slopes give finite gradients."""
    n, v = 4, 300
    z = torch.randn((n, v), generator=_gen(11), device="cuda").to(TYPES[dt])
    y = torch.randint(0, v, (n,), generator=_gen(12), device="cuda")
    z[1, y[1]] = -math.inf
    adv, ref = torch.ones(n, device="cuda"), torch.full((n,), -2.0, device="cuda")
    for old in (None, torch.full((n,), -6.0, device="cuda")):
        loss, logp, grad = L.policy_loss(z, y, old, adv)
        assert torch.isfinite(loss) and logp[1] == -math.inf and torch.isfinite(grad).all()
        if old is not None:
            assert (grad[1] == 0).all()
        loss, logp, grad = L.policy_loss(z, y, old, adv, ref, kl=0.1)
        assert loss == math.inf and torch.isfinite(grad[[0, 2, 3]]).all()


# ---------------------------------------------------------------- targets shifted in place of sliced logits


def test_next_token_targets(L):  # noqa: F811
    """All of the logits with targets that are shifted, the last of each sequence -100, as against slices."""
    s, t, v = 5, 19, 1003
    z = (torch.randn((s, t, v), generator=_gen(8), device="cuda") * 3).bfloat16()
    ids = torch.randint(0, v, (s, t), generator=_gen(9), device="cuda")
    targets = torch.nn.functional.pad(ids[:, 1:], (0, 1), value=-100)
    logp = L.token_logprobs(z, targets)
    want = torch.log_softmax(z[:, :-1].double(), 2).gather(2, ids[:, 1:, None])[:, :, 0]
    assert (logp[:, -1] == 0).all() and ((logp[:, :-1] - want).abs() <= 2.0 ** -17 * want.abs().clamp_min(1)).all()
    adv = torch.randn((s,), generator=_gen(10), device="cuda")
    cut = z[:, :-1].contiguous()
    for kind in ("token", "sequence"):
        loss, _, grad = L.policy_loss(z, targets, None, adv, reduction=kind)
        less, _, part = L.policy_loss(cut, ids[:, 1:].contiguous(), None, adv, reduction=kind)
        # the rows' offsets from 16 bytes differ, and with them the order of their sums
        assert abs(loss - less) <= 2.0 ** -20 * less.abs().clamp_min(1)
        assert (grad[:, -1] == 0).all() and ((grad[:, :-1] - part).abs() <= 2.0 ** -7 * part.abs() + 2.0 ** -30).all()
    for call in (lambda: L.token_logprobs(z[:, :-1], targets[:, :-1].contiguous()), lambda: L.token_logprobs(cut, ids[:, 1:])):
        with pytest.raises(ValueError, match="one stride|contiguous"):
            call()
