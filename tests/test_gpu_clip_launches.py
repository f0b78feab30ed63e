"""GPU checks of the clipping of more tensors than one launch takes."""
import os
import re

import pytest
import torch

from provenloop_b200 import build
from tests.test_gpu_clip import A, TYPES, _check, _device, _gen  # noqa: F401

pytestmark = pytest.mark.gpu

with open(os.path.join(build.CSRC, "k_clip.cu")) as _f:
    _source = _f.read()
MOST = max(int(n) for n in re.findall(r"clip<(\d+)>\(a, s\)", _source))  # tensors of a launch
CHUNK, FOLD = (int(re.search(rf"{name} = (\d+)", _source)[1]) for name in ("kChunk", "kFold"))


@pytest.mark.parametrize("count", [MOST, MOST + 1, 2 * MOST, 2 * MOST + 5])
def test_one_norm_over_several_launches(A, count):  # noqa: F811
    """Tensors of three types, up to three launches of the squares and as many of the scaling, in place and apart."""
    g = _gen(count)
    grads = [torch.randn((1 + 37 * k % 501,), generator=g, device="cuda").to(list(TYPES.values())[k % 3]) for k in range(count)]
    grads[-1] = grads[-1] * 100  # the last launch has its part of the norm
    outs = [torch.empty_like(t) for t in grads]
    _check(A.clip_gradients(grads, 1.0, out=outs), outs, grads, 1.0)
    keep = [t.clone() for t in grads]
    _check(A.clip_gradients(grads, 1.0), grads, keep, 1.0)
    assert all(torch.equal(a, b) for a, b in zip(grads, outs))
    _check(A.clip_gradients(keep, 1e9), keep, [t.clone() for t in keep], 1e9)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_each_adapter_over_several_launches(A, dt):  # noqa: F811
    g = _gen(2)
    grads = [torch.randn((3, 1 + 11 * k % 97, 5), generator=g, device="cuda").to(TYPES[dt]) for k in range(2 * MOST + 77)]
    keep = [t.clone() for t in grads]
    most = torch.tensor([1.0, 1e9, 30.0], device="cuda")
    _check(A.clip_gradients(grads, most, adapters=3), grads, keep, most, 3)
    assert all(torch.equal(t[1], k[1]) for t, k in zip(grads, keep))


def test_sums_that_a_launch_of_their_own_adds_up(A):  # noqa: F811
    """More chunks of a group than every CTA of the scaling adds up by itself, from three launches."""
    count = 2 * MOST + 3
    each = FOLD // count + 1  # chunks of a tensor's part
    g = _gen(3)
    grads = [torch.randn((2, each * CHUNK // 4 - k % 5), generator=g, device="cuda") for k in range(count)]
    grads[0][1] *= 3
    assert sum(-(-t[0].numel() * 4 // CHUNK) for t in grads) > FOLD
    keep = [t.clone() for t in grads]
    most = torch.tensor([10.0, 20.0], device="cuda")
    _check(A.clip_gradients(grads, most, adapters=2), grads, keep, most, 2)
