"""GPU checks of the gradients' norms and clipping against 64-bit forms."""
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
def A():
    from provenloop_b200 import adapters
    return adapters


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _norms64(grads, adapters):
    n = adapters or 1
    return torch.stack([t.double().reshape(n, -1).square().sum(1) for t in grads]).sum(0).sqrt()


def _check(norms, outs, grads, max_norm, adapters=None):
    """Norms: sums of up to 64 squares in 32 bits, all of one sign, are off by
    2^-24 for each addition, the rest is in 64 bits; half of that in the root,
    which is rounded once.  Results: the factor's rounding, the norm's error, the product's
    rounding, half a step of the type (of its least values, for tiny ones)."""
    want = _norms64(grads, adapters)
    off = 2.0 ** -24 * (64 / 2 + 1)
    assert norms.dtype == torch.float32 and norms.shape == ((adapters,) if adapters else ())
    assert ((norms.double().view(-1) - want).abs() <= off * want).all()
    most = torch.as_tensor(max_norm, dtype=torch.float64, device="cuda").expand(want.shape)
    by = torch.where(want > most, most / want, 1.0)
    for o, t in zip(outs, grads):
        w = t.double() * by.view(-1, *[1] * (t.dim() - 1)) if adapters else t.double() * by
        eps, tiny = torch.finfo(o.dtype).eps, 2.0 ** -25 if o.dtype is torch.float16 else 2.0 ** -127
        assert ((o.double() - w).abs() <= (eps / 2 + off + 2.0 ** -23) * w.abs() + tiny).all()


def _stack(adapters, dt, seed, shapes=((16, 257), (33, 7), (5, 1024), (1, 1), (40, 1536)), std=1.0):
    g = _gen(seed)
    return [(torch.randn((adapters, *s), generator=g, device="cuda") * std).to(TYPES[dt]) for s in shapes]


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("adapters", [1, 3, 7, 64])
@pytest.mark.parametrize("most", [0.0, 1.0, 200.0, 1e9])
def test_each_adapter(A, adapters, dt, most):
    grads = _stack(adapters, dt, adapters)
    grads = [(t * torch.linspace(0.1, 3, adapters, device="cuda").view(-1, 1, 1)).to(t.dtype) for t in grads]
    keep = [t.clone() for t in grads]
    norms = A.clip_gradients(grads, most, adapters=adapters)
    _check(norms, grads, keep, most, adapters)
    each = torch.linspace(0.0, 400.0, adapters, device="cuda")
    grads = [t.clone() for t in keep]
    norms = A.clip_gradients(grads, each, adapters=adapters)
    _check(norms, grads, keep, each, adapters)
    free = (_norms64(keep, adapters) < each).cpu()
    for t, k in zip(grads, keep):
        assert torch.equal(t[free], k[free])


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shapes", [((1,),), ((0,), (3,)), ((), (17,)), ((5, 7, 11), (16385,), (8, 8)), ((3000017,), (70000, 3))])
def test_one_norm(A, shapes, dt):
    g = _gen(3)
    grads = [torch.randn(s, generator=g, device="cuda").to(TYPES[dt]) for s in shapes]
    keep = [t.clone() for t in grads]
    _check(A.clip_gradients(grads, 0.5), grads, keep, 0.5)
    most = torch.tensor([2.0], device="cuda")
    outs = [torch.empty_like(t) for t in keep]
    versions = [t._version for t in outs]
    _check(A.clip_gradients(keep, most, out=outs), outs, keep, 2.0)
    assert all(t._version > v for t, v in zip(outs, versions))
    wide = [torch.empty(t.shape, device="cuda") for t in keep]
    _check(A.clip_gradients(tuple(keep), 3.0, out=wide), wide, keep, 3.0)


def test_many_tensors_of_mixed_types(A):
    """More tensors than one launch takes, some empty, some not there."""
    g = _gen(4)
    grads = [torch.randn((1 + 37 * k % 501,), generator=g, device="cuda").to(list(TYPES.values())[k % 3]) for k in range(411)]
    grads[5] = grads[5][:0]
    keep = [t.clone() for t in grads]
    _check(A.clip_gradients(grads[:200] + [None] + grads[200:], 1.0), grads, keep, 1.0)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("cut,cut_out", [(0, 0), (1, 1), (1, 2), (3, 0), (7, 5)])
def test_off_16_bytes(A, dt, cut, cut_out):
    g = _gen(5)
    whole = torch.randn((3 * 10007 + 16,), generator=g, device="cuda").to(TYPES[dt])
    grad = whole[cut:cut + 3 * 10007].view(3, 10007)
    for ot in {TYPES[dt], torch.float32}:
        room = torch.full((3 * 10007 + 16,), 7.0, device="cuda").to(ot)
        out = room[cut_out:cut_out + 3 * 10007].view(3, 10007)
        _check(A.clip_gradients([grad], 1.0, adapters=3, out=[out]), [out], [grad], 1.0, 3)
        assert (room[:cut_out] == 7).all() and (room[cut_out + 3 * 10007:] == 7).all()
    before = whole.clone()
    keep = grad.clone()
    _check(A.clip_gradients([grad], 1.0, adapters=3), [grad], [keep], 1.0, 3)
    assert torch.equal(whole[:cut], before[:cut]) and torch.equal(whole[cut + 3 * 10007:], before[cut + 3 * 10007:])


def test_dense_layouts(A):
    g = _gen(6)
    x = torch.randn((30, 50, 4), generator=g, device="cuda")
    grads = [x.permute(2, 0, 1), torch.randn((6, 4), generator=g, device="cuda").t()]
    keep = [t.clone() for t in grads]
    _check(A.clip_gradients(grads, 1.0), grads, keep, 1.0)
    outs = [torch.empty_like(t) for t in keep]
    assert outs[0].stride() == keep[0].stride()
    _check(A.clip_gradients(keep, 1.0, out=outs), outs, keep, 1.0)


def test_a_tensor_twice_counts_twice(A):
    x = torch.full((4,), 2.0, device="cuda")
    outs = [torch.empty_like(x) for _ in range(2)]
    # 32 is exact, its root (no number of 32 bits) is rounded once
    assert A.clip_gradients([x, x], 1e9, out=outs).cpu() == torch.tensor(math.sqrt(32), dtype=torch.float32)
    with pytest.raises(ValueError, match="overlap"):
        A.clip_gradients([x, x], 1.0)
    with pytest.raises(ValueError, match="overlap"):
        A.clip_gradients([x, x[:2]], 1.0)
    with pytest.raises(ValueError, match="overlap"):
        A.clip_gradients([x, x.clone()], 1.0, out=[outs[0], outs[0]])


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_not_finite(A, dt):
    """An adapter with an infinity or a NaN is left as it is, the others are clipped."""
    grads = _stack(5, dt, 7)
    grads[0][1, 3, 5], grads[4][3, 39, 1535], grads[2][4, 0, 0] = math.inf, math.nan, -math.inf
    keep = [t.clone() for t in grads]
    outs = [torch.empty_like(t) for t in grads]
    for to in (outs, grads):
        norms = A.clip_gradients(grads, 1.0, adapters=5, out=None if to is grads else to)
        assert norms[1] == math.inf and torch.isnan(norms[3]) and norms[4] == math.inf
        for o, k in zip(to, keep):
            same = lambda x, y: torch.equal(torch.nan_to_num(x, nan=7.0), torch.nan_to_num(y, nan=7.0))  # noqa: E731
            assert all(same(o[e], k[e]) for e in (1, 3, 4))
        good = [0, 2]
        _check(norms[good], [o[good] for o in to], [k[good] for k in keep], 1.0, 2)


@pytest.mark.parametrize("dt,size", [("bf16", 1e-30), ("bf16", 1e30), ("fp32", 1e-30), ("fp32", 1e30), ("fp16", 6e-8), ("fp16", 60000.0),
                                     ("fp32", 1e-38), ("bf16", 0.0)])
def test_sizes_out_of_the_ordinary(A, dt, size):
    """Squares below and above the range of 32 bits."""
    g = _gen(8)
    sign = torch.randint(0, 2, (2, 20003), generator=g, device="cuda") * 2 - 1
    grads = [(sign * size).to(TYPES[dt])]
    keep = [t.clone() for t in grads]
    most = size * 3
    _check(A.clip_gradients(grads, most, adapters=2), grads, keep, float(torch.tensor(most, dtype=torch.float32)), 2)


def test_norm_beyond_32_bits_is_not_finite(A):
    x = torch.full((1000,), 3e38, device="cuda")
    assert A.clip_gradients([x], 1.0).item() == math.inf and (x == 3e38).all()


def test_least_values(A):
    """Gradients of the types' least values have a norm, and are clipped by it."""
    for dt, least in ((torch.float32, -149), (torch.float32, -134), (torch.bfloat16, -133), (torch.float16, -24)):
        t = torch.full((16,), 2.0 ** least, dtype=dt, device="cuda")
        want = t.double().norm()
        norm = A.clip_gradients([t], 0.0)
        assert abs(norm.item() - want.item()) <= 2.0 ** -24 * want.item() + 2.0 ** -150 and (t == 0).all()


def test_large_stack(A):
    """A part of more than 2^31 bytes."""
    x = torch.empty((2, 1 << 30), dtype=torch.bfloat16, device="cuda")
    x[0], x[1] = 2.0 ** -15, 2.0 ** -16  # norms 1 and a half
    x[1, -1] = 1.0
    norms = A.clip_gradients([x], 0.5, adapters=2)
    assert norms[0] == 1.0 and abs(norms[1].item() - math.sqrt(1.25)) < 2.0 ** -24 * 33 * 1.2
    assert (x[0] == 2.0 ** -16).all() and abs(x[1, -1].item() - 0.5 / math.sqrt(1.25)) < 2.0 ** -9


def test_same_bits_on_every_stream_and_captured(A):
    grads = _stack(3, "bf16", 9)
    other = _stack(3, "bf16", 10, std=0.001)
    want = []
    for s in (grads, other):
        outs = [torch.empty_like(t) for t in s]
        want.append([A.clip_gradients(s, 1.0, adapters=3, out=outs).clone(), *outs])
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for _ in range(3):
            outs = [torch.empty_like(t) for t in grads]
            norms = A.clip_gradients(grads, 1.0, adapters=3, out=outs)
            stream.synchronize()
            assert all(torch.equal(a, b) for a, b in zip([norms, *outs], want[0]))
    live = [t.clone() for t in grads]
    outs = [torch.empty_like(t) for t in grads]
    most = torch.tensor(1.0, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norms = A.clip_gradients(live, most, adapters=3, out=outs)
    for k, s in ((1, other), (0, grads)):
        for t, v in zip(live, s):
            t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip([norms, *outs], want[k]))
    most.fill_(0.0)
    graph.replay()
    torch.cuda.synchronize()
    assert all((o == 0).all() for o in outs)
