"""GPU checks of the losses on rows that clusters of CTAs share."""
import os
import re

import pytest
import torch

from provenloop_b200 import build
from tests.test_gpu_losses import (TYPES, L, _check_policy, _check_preference, _device, _gen, _near_gradient, _near_logprobs,  # noqa: F401
                                   _padded, _policy_inputs)

pytestmark = pytest.mark.gpu


def _behind_parts(v):
    """Targets around the ends of the parts that 2, 4 and 8 CTAs have of a row, most of them just behind."""
    ends = {-(-(-(-v // c)) // 128) * 128 * r for c in (2, 4, 8) for r in range(1, c)}
    return [y for e in sorted(ends) for y in (e, e + 1, e + 127, e + 1000, e - 1) if y < v]


@pytest.mark.parametrize("dt,n,v", [("fp32", 2406, 230000), ("fp32", 24, 230000), ("fp32", 16, 230000), ("bf16", 222, 151936), ("fp16", 40, 400003)])
def test_gradient_in_place_with_targets_behind_a_part(L, dt, n, v):  # noqa: F811
    """Few rows to a cluster, and more than the 32 that it looks ahead.  All the bits of the gradient elsewhere."""
    z = torch.empty((n, v), dtype=TYPES[dt], device="cuda")
    for rows in z.split(256):
        rows.copy_(torch.randn(rows.shape, generator=_gen(len(rows)), device="cuda") * 3)
    at = torch.tensor(_behind_parts(v), device="cuda")
    y = at[torch.arange(n, device="cuda") % len(at)].view(2, n // 2)
    z = z.view(2, n // 2, v)
    loss, _, logp, want = L.preference_loss(z, y, beta=0.01, average=True)
    p = torch.exp(logp.double())
    part = -0.01 * torch.sigmoid(0.01 * (logp[1].double().mean() - logp[0].double().mean())) / (n // 2)
    g = (1 - p) * torch.stack([part, -part])[:, None]
    got = want.gather(2, y[:, :, None])[:, :, 0].double()
    # the slope and 1 - p in 32 bits, p off by its log's 2^-17 (twenty and less), the result's type
    assert ((got - g).abs() <= (torch.finfo(z.dtype).eps / 2 + 2.0 ** -16) * g.abs() + 2.0 ** -25).all()
    for _ in range(3):
        mine = z.clone()
        again, _, _, grad = L.preference_loss(mine, y, beta=0.01, average=True, out=mine)
        assert grad is mine and torch.equal(again, loss) and torch.equal(mine, want)


with open(os.path.join(build.CSRC, "k_loss.cu")) as _f:
    OWN_ORDER = int(re.search(r"kOwnOrder = (\d+)", _f.read())[1])


@pytest.mark.parametrize("s,t,v,dt", [(6, 350, 20000, "bf16"), (6, 350, 20000, "fp16"), (70, 31, 50257, "fp32"), (6, 350, 60001, "fp16"),
                                      (6, 350, 151936, "bf16"), (30, 71, 70001, "fp32"), (2, 1200, 9001, "fp32")])
def test_padded_batches_that_a_launch_puts_in_order(L, s, t, v, dt):  # noqa: F811
    """More rows than CTAs put in order by themselves; rows of a slot, of several, of parts that are copied
    again; short ones as they come, longer ones in order for gradients, the longest for all."""
    assert s * t > OWN_ORDER
    z, y = _padded(s, t, v, dt, seed=s)
    old, adv, ref = _policy_inputs(z, y)
    flat, yy = z.view(-1, v), y.view(-1)
    _near_logprobs(L.token_logprobs(z, y), flat, yy)
    g = torch.randn((s, t), generator=_gen(7), device="cuda")
    g[0, :5] = 0.0
    _near_gradient(L.token_logprobs_backward(g, z, y), flat, yy, g.double().view(-1), torch.zeros_like(g).double().view(-1))
    out = torch.full_like(z, 7.0)
    _check_policy(L, z, y, old, adv, ref, kl=0.04, kind="sequence", out=out)
    _check_preference(L, z, y, ref, average=True, out=out)
    mine = z.clone()
    _check_policy(L, mine, y, old, adv, ref, kl=0.04, out=mine)
    _check_preference(L, z, y, ref, kind="squared", beta=0.3, out=z)
