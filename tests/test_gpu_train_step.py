"""GPU check of a training step of adapters made of the plaintext operators:
projection with adapters, logits, loss, gradients, clipping."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _batch(seed=0, s=6, t=21, d=256, o=320, v=9001, r=8, e=3, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)

    b = dict(x=normal(s, t, d), w=normal(o, d, std=d ** -0.5), a=normal(e, r, d, std=d ** -0.5), b=normal(e, o, r, std=0.3), head=normal(v, o, std=2 * o ** -0.5),
             adapter=torch.tensor([0, 1, 2, -1, 1, 0], dtype=torch.int32, device="cuda")[:s], scale=torch.tensor([1.0, 0.5, 2.0], device="cuda"))
    y = torch.randint(0, v, (s, t), generator=g, device="cuda")
    at = torch.arange(t, device="cuda")
    b["y"] = torch.where((at >= 4) & (at < torch.tensor([t, 9, t, 13, t, t - 2], device="cuda")[:s, None]), y, -100)
    b["adv"] = torch.randn((s,), generator=g, device="cuda")
    return b


def _step(b, old, ref, kind, limit):
    """(loss, clipped gradients of A and B, norms) by the framework's calls; the head's product is the host framework's."""
    from provenloop_b200.adapters import adapter_project, adapter_project_backward, clip_gradients
    from provenloop_b200.losses import policy_loss, preference_loss
    h = adapter_project(b["x"], b["a"], b["b"], b["adapter"], weight=b["w"], scale=b["scale"])
    z = h @ b["head"].T
    if kind == "policy":
        loss, _, dz = policy_loss(z, b["y"], old, b["adv"], ref_logprobs=ref, kl=0.05, reduction="sequence", out=z)
    else:
        loss, _, _, dz = preference_loss(z, b["y"], ref, beta=0.2, average=True, out=z)
    _, da, db = adapter_project_backward(dz @ b["head"], b["x"], b["a"], b["b"], b["adapter"], scale=b["scale"], need_x=False)
    norms = clip_gradients([da, db], limit, adapters=b["a"].shape[0])
    return loss, da, db, norms


def _step64(b, old, ref, kind, limit):
    """The same by autograd in 64 bits."""
    x, w, head = (b[k].double() for k in ("x", "w", "head"))
    a, bb = (b[k].double().requires_grad_() for k in ("a", "b"))
    h = torch.stack([x[k] @ w.T + (b["scale"][e].double() * (x[k] @ a[e].T) @ bb[e].T if e >= 0 else 0.0) for k, e in enumerate(b["adapter"].tolist())])
    counts = b["y"] >= 0
    l = torch.log_softmax(h @ head.T, -1).gather(-1, b["y"].clamp_min(0)[..., None])[..., 0]
    mean = lambda t: (torch.where(counts, t, 0.0).sum(1) / counts.sum(1))  # noqa: E731
    if kind == "policy":
        rho, adv, lead = torch.exp(l - old.double()), b["adv"].double()[:, None], ref.double() - l
        loss = mean(0.05 * (torch.expm1(lead) - lead) - torch.minimum(rho * adv, rho.clamp(0.8, 1.2) * adv)).mean()
    else:
        lead = mean(l - ref.double())
        loss = torch.nn.functional.softplus(-0.2 * (lead[:len(lead) // 2] - lead[len(lead) // 2:])).mean()
    da, db = torch.autograd.grad(loss, (a, bb))
    norms = torch.stack([torch.cat([da[e].flatten(), db[e].flatten()]).norm() for e in range(len(da))])
    by = torch.where(norms > limit, limit / norms, 1.0)[:, None, None]
    return loss.detach(), da * by, db * by, norms


@pytest.mark.parametrize("kind", ["policy", "preference"])
def test_step_in_32_bits(kind):
    """In f32.  Every stage is within 2^-24 times the square root of its sums' lengths of what it
    is given (and below 2^-17 of its terms at worst); six stages, the longest sum 9001, and a
    loss whose slope for a log-probability's error is of the size of its gradient: 2^-12 of
    the gradients' norm bounds all of it by far, and a wrong term is seen."""
    torch.backends.cuda.matmul.allow_tf32 = False
    b = _batch()
    from provenloop_b200.adapters import adapter_project
    from provenloop_b200.losses import token_logprobs
    now = token_logprobs(adapter_project(b["x"], b["a"], b["b"], b["adapter"], weight=b["w"], scale=b["scale"]) @ b["head"].T, b["y"])
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    old, ref = now + 0.05 * torch.randn(now.shape, generator=g, device="cuda"), now + 0.3 * torch.randn(now.shape, generator=g, device="cuda")
    want = _step64(b, old, ref, kind, 1e9)
    limit = want[3].median().item() * 0.9  # some adapters are clipped, some are not
    want = _step64(b, old, ref, kind, limit)
    got = _step(b, old, ref, kind, limit)
    for w, h in zip(want, got):
        assert (w - h.double()).norm() <= 2.0 ** -12 * w.norm()
    again = _step(b, old, ref, kind, limit)
    assert all(torch.equal(p, q) for p, q in zip(got, again))


def test_captured_step_follows_its_inputs():
    b, other = _batch(1), _batch(2)
    old, ref = torch.full(b["y"].shape, -9.0, device="cuda"), torch.full(b["y"].shape, -9.5, device="cuda")
    want = [[t.clone() for t in _step(q, old, ref, "policy", 0.01)] for q in (b, other)]
    live = {k: t.clone() for k, t in b.items()}
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        _step(live, old, ref, "policy", 0.01)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = _step(live, old, ref, "policy", 0.01)
    for k, q in ((1, other), (0, b)):
        for name, t in q.items():
            live[name].copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, w) for p, w in zip(got, want[k]))


def test_losses_in_an_autograd_function():
    """The loss as a step of autograd's: forward keeps the gradient, backward scales it."""
    from provenloop_b200.losses import policy_loss

    class Policy(torch.autograd.Function):
        @staticmethod
        def forward(ctx, z, y, adv):
            loss, logp, grad = policy_loss(z, y, None, adv)
            ctx.save_for_backward(grad)
            return loss, logp

        @staticmethod
        def backward(ctx, dloss, _):
            return ctx.saved_tensors[0] * dloss, None, None

    b = _batch(3)
    h = torch.randn((6, 21, 320), device="cuda", requires_grad=True)
    z = h @ b["head"].T
    loss, logp = Policy.apply(z, b["y"], b["adv"])
    (loss * 3).backward()
    _, _, grad = policy_loss((h @ b["head"].T).detach(), b["y"], None, b["adv"])
    assert torch.equal(h.grad, (grad * 3) @ b["head"])
    with pytest.raises(ValueError, match="no_grad"):
        policy_loss(z, b["y"], None, b["adv"])
