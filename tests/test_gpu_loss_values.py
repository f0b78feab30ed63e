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
