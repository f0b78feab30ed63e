"""GPU checks of the losses on rows that clusters of CTAs share."""
import pytest
import torch

from tests.test_gpu_losses import TYPES, L, _device, _gen  # noqa: F401

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
