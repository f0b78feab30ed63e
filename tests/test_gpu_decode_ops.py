"""GPU checks of the plaintext decode-step operators against 64-bit forms:
low-rank adapters beside a shared projection, their gradients, and the rules
on next-token logits."""
import numpy as np
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


@pytest.fixture(scope="module")
def R():
    from provenloop_b200 import logits
    return logits


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ids(n, adapters, layout, g):
    if layout == "mixed":  # each token its own, some none (-1) and some outside the range
        return torch.randint(-1, adapters + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
    if layout == "none":
        return torch.full((n,), -1, device="cuda", dtype=torch.int32)
    if layout == "one":
        return torch.full((n,), adapters - 1, device="cuda", dtype=torch.int32)
    cuts = torch.randint(0, n, (max(1, n // 50),), generator=g, device="cuda").sort().values  # ragged requests
    which = torch.randint(-1, adapters, (cuts.numel() + 1,), generator=g, device="cuda", dtype=torch.int32)
    return which[torch.searchsorted(cuts, torch.arange(n, device="cuda"), right=True)]


def _inputs(n, i, o, r, e, dt, layout, seed=0):
    g, t = _gen(seed), TYPES[dt]

    def normal(*s, std=1.0):
        return (torch.randn(s, generator=g, device="cuda") * std).to(t)

    return dict(x=normal(n, i), a=normal(e, r, i, std=i ** -0.5), b=normal(e, o, r, std=0.7 * r ** -0.5),
                w=normal(o, i, std=i ** -0.5), bias=normal(o), base=normal(n, o), dy=normal(n, o), ids=_ids(n, e, layout, g),
                scale=0.5 + torch.rand((e,), generator=g, device="cuda"))


def _low64(x, a, s, ids):
    """s_e x a_e^T per token (zero without an adapter), and the sum of its terms' absolute values."""
    out, mag = (torch.zeros((x.shape[0], a.shape[1]), dtype=torch.float64, device="cuda") for _ in range(2))
    for k in range(a.shape[0]):
        rows = (ids == k).nonzero()[:, 0]
        out[rows] = s[k].double() * (x[rows].double() @ a[k].double().T)
        mag[rows] = s[k].double() * (x[rows].double().abs() @ a[k].double().abs().T)
    return out, mag


def _high64(low, mag, g, ids):
    """low_m g_e (g [adapters, r, d]) per token, and the terms' absolute values."""
    y, ymag = (torch.zeros((low.shape[0], g.shape[2]), dtype=torch.float64, device="cuda") for _ in range(2))
    for k in range(g.shape[0]):
        rows = (ids == k).nonzero()[:, 0]
        y[rows] = low[rows] @ g[k].double()
        ymag[rows] = mag[rows] @ g[k].double().abs()
    return y, ymag


def _allow(value, t, low_mag, low_len, main_mag, main_len):
    """Half a step of the result's type; the low-rank intermediate may be
    rounded once to 11 significant bits (half a step of 2^-10) where the inputs
    have 16 bits; sums of k terms in 32 bits are off by less than (k + 8) 2^-23
    of the terms' absolute sum (each addition at most a whole step)."""
    eps = torch.finfo(t).eps
    low = (0.0 if t is torch.float32 else 2.0 ** -11) + (low_len + 8) * 2.0 ** -23
    tiny = 2.0 ** -25 if t is torch.float16 else 1e-38  # half a step of fp16's subnormals
    tol = eps / 2 * value.abs() + low * low_mag * (1 + eps) + tiny
    if main_mag is not None:
        tol = tol + (main_len + 8) * 2.0 ** -23 * main_mag * (1 + eps)
    return tol


def _within(got, value, tol):
    off = (got.double() - value).abs() - tol
    assert torch.isfinite(got).all()
    assert (off <= 0).all(), f"worst excess {off.max().item():.3g}, allowed there {tol.flatten()[off.argmax()].item():.3g}"


def _check_project(A, s, weight=True, bias=True, base=False, scale=True, **kw):
    ids, t = s["ids"], s["x"].dtype
    sc = s["scale"] if scale else torch.ones_like(s["scale"])
    y = A.adapter_project(s["x"], s["a"], s["b"], ids, weight=s["w"] if weight else None, bias=s["bias"] if bias else None,
                          base=s["base"] if base else None, scale=s["scale"] if scale else None, **kw)
    low, lmag = _low64(s["x"], s["a"], sc, ids)
    ref, dmag = _high64(low, lmag, s["b"].transpose(1, 2), ids)
    main = torch.zeros_like(ref)
    if weight:
        ref = ref + s["x"].double() @ s["w"].double().T
        main = main + s["x"].double().abs() @ s["w"].double().abs().T
    if bias:
        ref, main = ref + s["bias"].double(), main + s["bias"].double().abs()
    if base:
        ref, main = ref + s["base"].double(), main + s["base"].double().abs()
    i, r = s["x"].shape[1], s["a"].shape[1]
    _within(y, ref, _allow(ref, t, dmag, i + r, main + dmag, i + r))
    return y


def _check_backward(A, s, weight=True, scale=True, **kw):
    ids, t, x, dy, a, b = s["ids"], s["x"].dtype, s["x"], s["dy"], s["a"], s["b"]
    sc = s["scale"] if scale else torch.ones_like(s["scale"])
    dx, da, db = A.adapter_project_backward(dy, x, a, b, ids, weight=s["w"] if weight else None,
                                            scale=s["scale"] if scale else None, **kw)
    n, i = x.shape
    o, r = b.shape[1], a.shape[1]
    u, umag = _low64(dy, b.transpose(1, 2), sc, ids)
    low, lmag = _low64(x, a, sc, ids)
    if dx is not None:
        ref, mag = _high64(u, umag, a, ids)
        main = mag
        if weight:
            ref = ref + dy.double() @ s["w"].double()
            main = mag + dy.double().abs() @ s["w"].double().abs()
        _within(dx, ref, _allow(ref, t, mag, o + r, main, o + r))
    if da is not None:
        for k in range(a.shape[0]):
            rows = (ids == k).nonzero()[:, 0]
            ref = u[rows].T @ x[rows].double()
            _within(da[k], ref, _allow(ref, t, umag[rows].T @ x[rows].double().abs(), o + n, None, 0))
            ref = dy[rows].double().T @ low[rows]
            _within(db[k], ref, _allow(ref, t, dy[rows].double().abs().T @ lmag[rows], i + n, None, 0))
    return dx, da, db


SHAPES = [  # n, d_in, d_out, r, adapters, layout
    (1, 1536, 1536, 16, 3, "one"),
    (1, 1, 1, 1, 1, "one"),
    (2, 9, 7, 3, 2, "mixed"),
    (3, 33, 65, 5, 4, "mixed"),
    (16, 1536, 256, 30, 64, "mixed"),
    (17, 520, 136, 16, 1, "one"),
    (63, 256, 1536, 256, 2, "mixed"),
    (64, 1537, 1535, 8, 3, "mixed"),
    (65, 64, 8, 16, 3, "none"),
    (129, 1536, 1536, 16, 3, "ragged"),
    (200, 104, 333, 30, 40, "mixed"),
    (300, 8960, 256, 64, 5, "ragged"),
    (513, 1001, 770, 7, 3, "ragged"),
    (1100, 1536, 264, 16, 200, "mixed"),
    (2300, 1536, 4104, 32, 5, "ragged"),
    (1500, 4104, 4096, 16, 3, "none"),
    (1300, 4104, 1000, 17, 40, "mixed"),
    (4099, 200, 2056, 16, 2, "one"),
]


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_project(A, shape, dt):
    s = _inputs(*shape[:5], dt, shape[5])
    _check_project(A, s)
    _check_project(A, s, weight=False, bias=False, base=True, scale=False)


@pytest.mark.parametrize("weight,bias,base,scale", [(True, False, False, True), (True, True, True, True), (False, True, False, False),
                                                    (False, False, False, True)])
@pytest.mark.parametrize("n", [5, 150])
def test_project_optional_terms(A, n, weight, bias, base, scale):
    _check_project(A, _inputs(n, 264, 200, 16, 3, "bf16", "mixed", seed=3), weight, bias, base, scale)


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_backward(A, shape, dt):
    s = _inputs(*shape[:5], dt, shape[5], seed=1)
    _check_backward(A, s)
    _check_backward(A, s, weight=False, scale=False)


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", [(900, 1536, 300, 64, 40, "mixed"), (1878, 90, 84, 64, 41, "mixed"), (72, 1536, 520, 64, 42, "mixed"),
                                   (217, 1536, 8960, 64, 14, "one"), (1024, 300, 1537, 16, 4, "ragged"), (129, 136, 40, 33, 500, "mixed"),
                                   (640, 1001, 256, 2, 9, "mixed")], ids=lambda s: "x".join(map(str, s)))
def test_many_adapters_and_ranks(A, shape, dt):
    """Sizes at which the rules by adapters, rank and tiles go the other way than above."""
    s = _inputs(*shape[:5], dt, shape[5], seed=5)
    _check_project(A, s)
    _check_project(A, s, weight=False, bias=False, base=True, scale=False)
    _check_backward(A, s)
    _check_backward(A, s, weight=False, scale=False)


@pytest.mark.parametrize("need", ["x", "adapters"])
def test_backward_parts(A, need):
    s = _inputs(140, 256, 328, 16, 3, "bf16", "ragged", seed=2)
    full = A.adapter_project_backward(s["dy"], s["x"], s["a"], s["b"], s["ids"], weight=s["w"], scale=s["scale"])
    part = A.adapter_project_backward(s["dy"], s["x"], s["a"], s["b"], s["ids"], weight=s["w"], scale=s["scale"],
                                      need_x=need == "x", need_adapters=need == "adapters")
    for p, f, wanted in zip(part, full, (need == "x", need == "adapters", need == "adapters")):
        assert (p is None) != wanted and (p is None or torch.equal(p, f))


def test_backward_against_differences(A):
    """The gradients are the slopes of the forward call: fp32, a loss linear
    in y, central differences.  y is bilinear in (A, B) and linear in each, so
    central differences are exact up to rounding."""
    s = _inputs(20, 24, 18, 4, 3, "fp32", "mixed", seed=5)
    dx, da, db = A.adapter_project_backward(s["dy"], s["x"], s["a"], s["b"], s["ids"], weight=s["w"], scale=s["scale"])

    def loss(**kw):
        q = {**s, **kw}
        y = A.adapter_project(q["x"], q["a"], q["b"], q["ids"], weight=q["w"], scale=q["scale"])
        return (y.double() * s["dy"].double()).sum().item()

    g = _gen(6)
    for name, grad in (("x", dx), ("a", da), ("b", db)):
        v = torch.randn(grad.shape, generator=g, device="cuda")
        slope = (loss(**{name: s[name] + v}) - loss(**{name: s[name] - v})) / 2
        want = (grad.double() * v.double()).sum().item()
        # each of the 360 outputs is off by at most (24 + 4 + 16) 2^-23 of its
        # terms' absolute sum (a few tens), weighted by dy (at most about 4)
        assert abs(slope - want) < 360 * 44 * 2.0 ** -23 * 50 * 4


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [6, 140])
def test_strided_rows_and_in_place(A, n, dt):
    s = _inputs(n, 264, 200, 16, 3, dt, "mixed", seed=7)
    plain = A.adapter_project(s["x"], s["a"], s["b"], s["ids"], weight=s["w"], base=s["base"], scale=s["scale"])

    def padded(t, left, right):
        big = torch.full((t.shape[0], t.shape[1] + left + right), 77.0, dtype=t.dtype, device="cuda")
        view = big[:, left:left + t.shape[1]]
        view.copy_(t)
        return big, view

    for left, right in ((0, 8), (8, 24), (3, 2)):
        _, x = padded(s["x"], left, right)
        _, w = padded(s["w"], left, right)
        big, base = padded(s["base"], left, right)
        got = A.adapter_project(x, s["a"], s["b"], s["ids"], weight=w, base=base, scale=s["scale"], out=base)
        assert got is base
        _within(got, plain.double(), 2 * _allow(plain.double(), plain.dtype, plain.double().abs() * 0 + 40, 280, plain.double().abs() * 0 + 40, 280))
        assert (big[:, :left] == 77).all() and (big[:, left + 200:] == 77).all()
        _, dy = padded(s["dy"], left, right)
        one = A.adapter_project_backward(s["dy"], s["x"], s["a"], s["b"], s["ids"], weight=s["w"], scale=s["scale"])
        two = A.adapter_project_backward(dy, x, s["a"], s["b"], s["ids"], weight=w, scale=s["scale"])
        for p, q in zip(one, two):
            mag = torch.full_like(p, 40.0 * max(1.0, n ** 0.5), dtype=torch.float64)
            _within(q, p.double(), 2 * _allow(p.double(), p.dtype, mag, 480, mag, 480))


def test_last_token_of_each_request(A):
    """x = h[:, -1, :], one index per request; and x [requests, tokens, d]."""
    s = _inputs(12, 256, 128, 16, 3, "bf16", "mixed", seed=8)
    h = s["x"].view(3, 4, 256)
    ids = s["ids"][:3].contiguous()
    rep = ids.repeat_interleave(4)
    y = A.adapter_project(h, s["a"], s["b"], ids, weight=s["w"])
    assert y.shape == (3, 4, 128)
    assert torch.equal(y.view(12, 128), A.adapter_project(s["x"], s["a"], s["b"], rep, weight=s["w"]))
    last = A.adapter_project(h[:, -1, :], s["a"], s["b"], ids, weight=s["w"])
    assert torch.equal(last, A.adapter_project(h[:, -1, :].contiguous(), s["a"], s["b"], ids, weight=s["w"]))
    g = A.adapter_project_backward(s["dy"][:, :128].reshape(3, 4, 128), h, s["a"], s["b"], ids, weight=s["w"])
    f = A.adapter_project_backward(s["dy"][:, :128].contiguous(), s["x"], s["a"], s["b"], rep, weight=s["w"])
    assert g[0].shape == h.shape and all(torch.equal(p.view(-1), q.view(-1)) for p, q in zip(g, f))


def test_no_tokens(A):
    s = _inputs(4, 64, 40, 8, 2, "bf16", "one")
    ids = s["ids"][:0]
    y = A.adapter_project(s["x"][:0], s["a"], s["b"], ids, weight=s["w"])
    assert y.shape == (0, 40)
    dx, da, db = A.adapter_project_backward(s["dy"][:0], s["x"][:0], s["a"], s["b"], ids, weight=s["w"])
    assert dx.shape == (0, 64) and not da.any() and not db.any()


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("n,i,o", [(8, 264, 200), (40, 264, 200), (200, 264, 200), (300, 264, 4000), (300, 4000, 264)])
@pytest.mark.parametrize("weight", [True, False])
def test_a_request_is_not_touched_by_the_others(A, n, i, o, weight, dt):
    """NaN and infinities in one adapter, or in one request's rows, stay with
    the tokens that use them, forward and backward."""
    s = _inputs(n, i, o, 16, 3, dt, "mixed", seed=9)
    s["ids"] = (torch.arange(n, device="cuda") % 4 - 1).to(torch.int32)
    kw = dict(weight=s["w"] if weight else None, scale=s["scale"])
    clean = A.adapter_project(s["x"], s["a"], s["b"], s["ids"], **kw)
    cback = A.adapter_project_backward(s["dy"], s["x"], s["a"], s["b"], s["ids"], **kw)
    hit = s["ids"] == 1
    for name, where, value in (("a", (1, 3, 7), float("nan")), ("b", (1, 11, 2), float("inf")), ("x", None, float("inf")),
                               ("dy", None, float("nan")), ("scale", (1,), float("inf"))):
        q = dict(s)
        q[name] = s[name].clone()
        if where is None:
            q[name][hit] = value
        else:
            q[name][where] = value
        k2 = dict(weight=kw["weight"], scale=q["scale"])
        y = A.adapter_project(q["x"], q["a"], q["b"], q["ids"], **k2)
        assert torch.equal(y[~hit], clean[~hit]), name
        dx, da, db = A.adapter_project_backward(q["dy"], q["x"], q["a"], q["b"], q["ids"], **k2)
        assert torch.equal(dx[~hit], cback[0][~hit]), name
        for e in (0, 2):
            assert torch.equal(da[e], cback[1][e]) and torch.equal(db[e], cback[2][e]), name
        if name == "b":
            assert not torch.isfinite(y[hit][:, 11]).any()


def test_large_intermediates_stay_finite(A):
    """fp16: x A^T beyond 65504 is no overflow where the result is in range."""
    n, i, o, r = 70, 512, 64, 8
    x = torch.full((n, i), 16.0, dtype=torch.float16, device="cuda")
    a = torch.full((1, r, i), 16.0, dtype=torch.float16, device="cuda")       # x A^T = 131072
    b = torch.full((1, o, r), 2.0 ** -12, dtype=torch.float16, device="cuda")  # y = 8 * 131072 / 4096 = 256
    for m in (1, n):
        y = A.adapter_project(x[:m], a, b, torch.zeros(m, dtype=torch.int32, device="cuda"))
        assert (y == 256).all()


@pytest.mark.parametrize("n", [4, 200])
def test_streams_and_graphs(A, n):
    """Another stream, and two captured graphs of the same tensors replayed
    on two streams at once, give what the plain call gives."""
    s = _inputs(n, 520, 264, 16, 3, "bf16", "mixed", seed=10)

    def both():
        y = A.adapter_project(s["x"], s["a"], s["b"], s["ids"], weight=s["w"], bias=s["bias"], scale=s["scale"])
        return (y, *A.adapter_project_backward(s["dy"], s["x"], s["a"], s["b"], s["ids"], weight=s["w"], scale=s["scale"]))

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = both()
        graphs.append((g, out, torch.cuda.Stream()))
    fresh = torch.randn_like(s["x"])
    s["x"].copy_(fresh)
    want = both()
    torch.cuda.synchronize()
    for _ in range(3):
        for g, out, st in graphs:
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for _, out, _ in graphs:
        assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_same_inputs_same_bits(A):
    s = _inputs(777, 520, 328, 30, 5, "bf16", "mixed", seed=11)
    runs = [A.adapter_project_backward(s["dy"], s["x"], s["a"], s["b"], s["ids"], weight=s["w"], scale=s["scale"]) for _ in range(4)]
    for r in runs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(r, runs[0]))


# ---------------------------------------------------------------- rules


def _rules_ref(x, tokens=None, lengths=None, prompt=None, rho=None, f=None, p=None, bias_ids=None, bias=None, mask=None, dtype=np.float64):
    """The rules in numpy, row by row, in `dtype`; (z, picks, magnitude of the intermediate values)."""
    z = x.astype(dtype).copy()
    mag = np.abs(z)
    n, v = z.shape
    for i in range(n):
        if tokens is not None:
            m = tokens.shape[1] if lengths is None else min(max(int(lengths[i]), 0), tokens.shape[1])
            q = 0 if prompt is None else max(int(prompt[i]), 0)
            ids = [t for t in tokens[i, :m] if 0 <= t < v]
            r = dtype(1 if rho is None else rho[i])
            for t in set(ids):
                z[i, t] = z[i, t] / r if z[i, t] > 0 else z[i, t] * r
                mag[i, t] = max(mag[i, t], abs(z[i, t]))
            said, times = np.unique([t for t in tokens[i, q:m] if 0 <= t < v], return_counts=True)
            for t, c in zip(said.astype(int), times):
                a, b = dtype(0 if f is None else f[i]) * dtype(c), dtype(0 if p is None else p[i])
                z[i, t] = (z[i, t] - a) - b
                mag[i, t] += abs(a) + abs(b)
        if bias_ids is not None:
            row = bias_ids if bias_ids.ndim == 1 else bias_ids[i]
            val = bias if bias.ndim == 1 else bias[i]
            for t, c in {int(t): c for t, c in zip(row, val) if 0 <= t < v}.items():
                z[i, t] = z[i, t] + dtype(c)
                mag[i, t] += abs(c)
        if mask is not None:
            row = (mask if mask.ndim == 1 else mask[i]).view(np.uint32)
            ok = (row[np.arange(v) // 32] >> (np.arange(v) % 32).astype(np.uint32)) & 1
            z[i, ok == 0] = -np.inf
            mag[i, ok == 0] = 0
    picks = np.array([-1 if (r == -np.inf).all() else int(np.argmax(r)) for r in z])
    return z, picks, mag


def _rules_case(n, v, dt, hist, biases, masked, seed, wide=False):
    rng = np.random.default_rng(seed)
    x = torch.from_numpy((rng.standard_normal((n, v)) * 3).astype(np.float32)).to(TYPES[dt])
    ref, kw = {}, {}
    it = np.int64 if wide else np.int32
    if hist:
        ref["tokens"] = rng.integers(-2, v + 2, (n, hist)).astype(it)
        ref["tokens"][:, : hist // 2] %= max(1, min(v, 9))  # many repeats
        ref["lengths"] = rng.integers(-1, hist + 2, n).astype(np.int32)
        ref["lengths"][0] = hist
        ref["prompt"] = rng.integers(-1, hist + 2, n).astype(np.int32)
        ref["rho"] = (1 + rng.random(n)).astype(np.float32)
        ref["f"], ref["p"] = rng.random(n).astype(np.float32), rng.random(n).astype(np.float32)
    if biases:
        ref["bias_ids"] = rng.integers(-3, v + 3, (n, biases)).astype(it)
        ref["bias_ids"][:, biases // 2:] = ref["bias_ids"][:, : biases - biases // 2]  # each id twice
        ref["bias"] = (4 * rng.standard_normal((n, biases))).astype(np.float32)
    if masked:
        words = [rng.integers(-2 ** 31, 2 ** 31, (n, (v + 31) // 32)) for _ in range(2)]
        ref["mask"] = (words[0] & words[1]).astype(np.int32)
        if n > 1:
            ref["mask"][n // 2] = 0
    names = dict(tokens="tokens", lengths="lengths", prompt="prompt_lengths", rho="repetition", f="frequency", p="presence",
                 bias_ids="bias_ids", bias="bias_values", mask="mask")
    for k, t in ref.items():
        kw[names[k]] = torch.from_numpy(t).cuda()
    return x.cuda(), kw, ref


def _check_rules(R, x, kw, ref, **more):
    z, pick = R.apply_rules(x, **kw, **more)
    xf = x.float().cpu().numpy()
    want32, pick32, _ = _rules_ref(xf, **ref, dtype=np.float32)
    assert np.array_equal(pick.cpu().numpy(), pick32)
    if z is not None:
        # the same roundings in the same order: the same values
        assert torch.equal(z.cpu(), torch.from_numpy(want32).to(z.dtype))
        # and near the 64-bit value: at most five roundings of 32 bits, one to the type
        want, _, mag = _rules_ref(xf, **ref)
        fine = np.isfinite(want)
        tol = 5 * 2.0 ** -24 * mag + torch.finfo(z.dtype).eps / 2 * np.abs(np.where(fine, want, 0)) * (1 + 2.0 ** -20) + 1e-7 * (z.dtype == torch.float16)
        got = z.double().cpu().numpy()
        assert np.array_equal(fine, np.isfinite(got)) and (np.abs(got - want)[fine] <= tol[fine]).all()
    return z, pick


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("n,v,hist,biases,masked,wide", [
    (1, 1, 3, 2, True, False), (2, 31, 5, 3, True, True), (3, 33, 0, 0, True, False), (1, 1000, 64, 0, False, True),
    (5, 1023, 200, 17, True, True), (7, 50257, 300, 40, True, True), (2, 151936, 4096, 300, True, True),
    (3, 151936, 1, 1, False, False), (9, 4099, 0, 5, False, False), (2, 200003, 100, 10, True, False), (4, 257, 0, 0, False, False)])
def test_rules(R, n, v, hist, biases, masked, wide, dt):
    _check_rules(R, *_rules_case(n, v, dt, hist, biases, masked, seed=n + v, wide=wide))


def test_rules_each_alone(R):
    x, kw, ref = _rules_case(3, 777, "bf16", 50, 9, True, seed=1)
    one = dict(repetition="rho", frequency="f", presence="p")
    for k, q in one.items():
        _check_rules(R, x, dict(tokens=kw["tokens"], **{k: kw[k]}), dict(tokens=ref["tokens"], **{q: ref[q]}))
    for keys in (("bias_ids", "bias_values"), ("mask",), ("tokens",), ("tokens", "lengths", "repetition")):
        names = dict(bias_values="bias", repetition="rho")
        _check_rules(R, x, {k: kw[k] for k in keys}, {names.get(k, k): ref[names.get(k, k)] for k in keys})


def test_rules_shared_rows_out_and_strides(R):
    x, kw, ref = _rules_case(5, 1001, "bf16", 60, 12, True, seed=2)
    for k, q in (("bias_ids", "bias_ids"), ("bias_values", "bias"), ("mask", "mask")):
        kw[k], ref[q] = kw[k][1].contiguous(), ref[q][1]
    z, pick = _check_rules(R, x, kw, ref)
    z32, pick32 = R.apply_rules(x, **kw, out=torch.empty((5, 1001), device="cuda"))
    assert z32.dtype == torch.float32 and torch.equal(z32.to(torch.bfloat16), z) and torch.equal(pick, pick32)
    none, only = R.apply_rules(x, **kw, write=False)
    assert none is None and torch.equal(only, pick)
    nopick = R.apply_rules(x, **kw, pick=False)
    assert nopick[1] is None and torch.equal(nopick[0], z)
    for left, right in ((0, 23), (5, 2)):
        big = torch.full((5, 1001 + left + right), 7.0, dtype=x.dtype, device="cuda")
        view = big[:, left:left + 1001]
        view.copy_(x)
        got, p2 = R.apply_rules(view, **kw)
        assert torch.equal(got, z) and torch.equal(p2, pick)
        got, p2 = R.apply_rules(view, **kw, out=view)  # in place
        assert got is view and torch.equal(view, z) and torch.equal(p2, pick)
        assert (big[:, :left] == 7).all() and (big[:, left + 1001:] == 7).all()
        dst = torch.full((5, 1001 + left + right), 7.0, device="cuda")
        R.apply_rules(x, **kw, out=dst[:, left:left + 1001])
        assert torch.equal(dst[:, left:left + 1001], z32) and (dst[:, :left] == 7).all() and (dst[:, left + 1001:] == 7).all()
    h = torch.randn((5, 3, 1001), device="cuda").to(torch.bfloat16)
    a, b = R.apply_rules(h[:, -1, :], **kw), R.apply_rules(h[:, -1, :].contiguous(), **kw)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("n,v,hist,biases,dt", [(300, 40000, 30, 3, "bf16"), (40, 300007, 700, 33, "fp16"), (150, 60000, 20, 0, "fp32"),
                                                (2, 300007, 60000, 4095, "bf16"), (160, 50001, 40000, 60, "fp32"),
                                                (160, 50001, 40000, 60, "bf16"), (1, 2100001, 9, 3, "bf16")])
def test_rules_splits(R, n, v, hist, biases, dt):
    """Few and many rows (each row on one to eight CTAs, one or more segments
    and blocks of the vocabulary), short and very long lists."""
    g = torch.Generator(device="cuda")
    g.manual_seed(n + v)

    def ints(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.int64)

    x = (torch.randn((n, v), generator=g, device="cuda") * 3).to(TYPES[dt])
    kw = dict(tokens=ints(-1, v, n, hist), lengths=ints(0, hist + 1, n).int(), prompt_lengths=ints(0, hist + 1, n).int(),
              repetition=1 + torch.rand(n, generator=g, device="cuda"), frequency=torch.rand(n, generator=g, device="cuda"),
              presence=torch.rand(n, generator=g, device="cuda"))
    if biases:
        kw.update(bias_ids=ints(0, v, n, biases), bias_values=torch.randn((n, biases), generator=g, device="cuda") * 4)
    mask = ints(-2 ** 31, 2 ** 31, n, (v + 31) // 32).int()
    z, pick = R.apply_rules(x, **kw, mask=mask, out=torch.empty((n, v), device="cuda"))
    # the same steps over whole rows, in 32 bits
    col = torch.arange(hist, device="cuda")
    tok = kw["tokens"]
    used = (col < kw["lengths"][:, None]) & (tok >= 0)
    spare = torch.where(used, tok, v)
    seen = torch.zeros((n, v + 1), dtype=torch.int32, device="cuda").scatter_add_(1, spare, used.int())[:, :v] > 0
    said = used & (col >= kw["prompt_lengths"][:, None])
    count = torch.zeros((n, v + 1), dtype=torch.int32, device="cuda").scatter_add_(1, torch.where(said, tok, v), said.int())[:, :v]
    rho, f, p = (kw[k][:, None] for k in ("repetition", "frequency", "presence"))
    w = x.float()
    w = torch.where(seen, torch.where(w > 0, w / rho, w * rho), w)
    w = torch.where(count > 0, w - f * count - p, w)
    if biases:
        last = torch.full((n, v), -1, device="cuda", dtype=torch.int64)
        last.scatter_reduce_(1, kw["bias_ids"], torch.arange(biases, device="cuda").expand(n, biases), "amax")
        w = torch.where(last >= 0, w + kw["bias_values"].gather(1, last.clamp_min(0)), w)
    at = torch.arange(v, device="cuda")
    w = torch.where((mask[:, at // 32] >> (at % 32)) & 1 != 0, w, float("-inf"))
    assert torch.equal(z, w)
    best = w.amax(1, keepdim=True)
    assert torch.equal(pick, torch.where(w == best, at, v).amin(1))
    inplace = x.clone()
    same, pick2 = R.apply_rules(inplace, **kw, mask=mask, out=inplace)
    assert torch.equal(same, w.to(x.dtype)) and torch.equal(pick2, pick)


def test_rules_ties_and_special_values(R):
    inf, nan = float("inf"), float("nan")
    rows = torch.zeros((7, 300), device="cuda")
    rows[1, [17, 250]] = 5.0                     # a tie: the lowest id
    rows[2] = -inf                               # nothing left
    rows[3, 100] = nan                           # NaN counts as the greatest
    rows[3, 200] = inf
    rows[4, 5] = inf
    rows[5] = -3.4028234663852886e38             # the type's lowest value is still a value
    rows[6, :150], rows[6, 150:] = -0.0, 0.0     # equal zeros
    z, pick = R.apply_rules(rows)
    assert pick.tolist() == [0, 17, -1, 100, 5, 0, 0]
    assert torch.equal(z.nan_to_num(nan=9.0), rows.nan_to_num(nan=9.0))
    mask = torch.full((10,), -1, dtype=torch.int32, device="cuda")
    mask[100 // 32] &= ~(1 << 100 % 32)
    mask[0] &= ~(1 << 5)
    z, pick = R.apply_rules(rows, mask=mask)
    assert pick.tolist() == [0, 17, -1, 200, 0, 0, 0] and z[3, 100] == -inf and z[4, 5] == -inf
    _, pick = R.apply_rules(rows, mask=torch.zeros(10, dtype=torch.int32, device="cuda"))
    assert (pick == -1).all()


def test_rules_empty(R):
    z, pick = R.apply_rules(torch.zeros((0, 100), device="cuda"))
    assert z.shape == (0, 100) and pick.shape == (0,)
    x = torch.randn((2, 100), device="cuda")
    empty = torch.zeros((2, 0), dtype=torch.int64, device="cuda")
    z, pick = R.apply_rules(x, tokens=empty, repetition=torch.full((2,), 2.0, device="cuda"), bias_ids=empty,
                            bias_values=torch.zeros((2, 0), device="cuda"))
    assert torch.equal(z, x) and torch.equal(pick, x.argmax(1))


def test_rules_captured(R):
    """A captured call reads lengths and tokens anew at each replay, also two
    graphs at once."""
    x, kw, ref = _rules_case(4, 1500, "bf16", 40, 6, True, seed=3, wide=True)
    R.apply_rules(x, **kw)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = R.apply_rules(x, **kw)
        graphs.append((g, out, torch.cuda.Stream()))
    for step in (1, 7, 40):
        kw["lengths"].fill_(step)
        kw["tokens"][:, :step] = step
        torch.cuda.synchronize()
        for g, _, st in graphs:
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        ref["lengths"], ref["tokens"] = kw["lengths"].cpu().numpy(), kw["tokens"].cpu().numpy()
        want, picks, _ = _rules_ref(x.float().cpu().numpy(), **ref, dtype=np.float32)
        for _, (z, pick), _ in graphs:
            assert torch.equal(z.cpu(), torch.from_numpy(want).to(z.dtype)) and np.array_equal(pick.cpu().numpy(), picks)


def test_training_step_of_two_layers(A, R):
    """Forward through two projections, the rules' pick on the result, the
    gradients back through both, an update, and forward again."""
    first, second = _inputs(230, 520, 264, 16, 3, "bf16", "ragged", seed=21), _inputs(230, 264, 1000, 30, 3, "bf16", "ragged", seed=22)
    second["ids"] = first["ids"]
    for _ in range(2):
        second["x"] = _check_project(A, first)
        y = _check_project(A, second)
        z, pick = R.apply_rules(y, mask=torch.full((32,), 0x5555_5555, dtype=torch.int32, device="cuda"))
        want = y.clone()
        want[:, 1::2] = -float("inf")
        assert torch.equal(z, want) and torch.equal(pick, want.float().argmax(1))
        first["dy"], da2, db2 = _check_backward(A, second)
        _, da1, db1 = _check_backward(A, first)
        for s, da, db in ((first, da1, db1), (second, da2, db2)):
            s["a"], s["b"] = s["a"] - 1e-3 * da, s["b"] - 1e-3 * db


def _model():
    from provenloop_b200.decode_step import build_model
    return build_model(layers=2)


def _layers(model, rank, experts, seed):
    rng, cfg = np.random.default_rng(seed), model.config
    d, dv = cfg.hidden_size, cfg.num_key_value_heads * (cfg.hidden_size // cfg.num_attention_heads)
    shapes = ((experts, rank, d), (experts, rank, d), (experts, d, rank), (experts, dv, rank))
    return [tuple((0.05 * rng.standard_normal(s)).astype(np.float32) for s in shapes) for _ in range(cfg.num_hidden_layers)]


def test_lora_batch_decodes_under_rules():
    """A batch of requests, each with its own adapter: every projection of
    every step and every pick against the 64-bit forms."""
    from types import SimpleNamespace
    from provenloop_b200.decode_step import LoraBatch
    model, n, k, steps = _model(), 5, 7, 4
    weights, v = _layers(model, 16, 3, 4), model.config.vocab_size
    plain = model.model.layers[0].self_attn.q_proj.forward
    batch = LoraBatch(model, weights)
    seen, logits, hooks = [], [], []
    for layer, (aq, av, bq, bv) in zip(model.model.layers, weights):
        for module, a, b in ((layer.self_attn.q_proj, aq, bq), (layer.self_attn.v_proj, av, bv)):
            a, b = (torch.from_numpy(w).cuda().bfloat16() for w in (a, b))
            hooks.append(module.register_forward_hook(lambda m, i, o, a=a, b=b: seen.append((m, i[0].clone(), o.clone(), a, b))))
    hooks.append(model.lm_head.register_forward_hook(lambda m, i, o: logits.append(o[:, -1].detach().clone())))
    rng = np.random.default_rng(8)
    prompt = rng.integers(0, v, (n, k))
    adapter = [0, 2, -1, 1, 0]
    ref = dict(rho=(1 + rng.random(n)).astype(np.float32), f=rng.random(n).astype(np.float32), p=rng.random(n).astype(np.float32),
               bias_ids=rng.integers(0, v, (n, 3)), bias=rng.standard_normal((n, 3)).astype(np.float32),
               mask=rng.integers(-2 ** 31, 2 ** 31, (n, (v + 31) // 32)).astype(np.int32))
    ref["mask"][3] = 0  # this request ends at once
    names = dict(rho="repetition", f="frequency", p="presence", bias="bias_values")
    got = batch.generate(prompt, adapter, tokens=steps, rules={names.get(q, q): torch.from_numpy(t).cuda() for q, t in ref.items()}).cpu().numpy()
    for h in hooks:
        h.remove()
    assert got.shape == (n, steps) and len(logits) == steps and len(seen) == steps * 4
    history = prompt
    for i in range(steps):
        lengths = np.full(n, history.shape[1], np.int32)
        picks = _rules_ref(logits[i].float().cpu().numpy(), tokens=history, lengths=lengths, prompt=np.full(n, k, np.int32), **ref,
                           dtype=np.float32)[1]
        assert np.array_equal(got[:, i], picks) and picks[3] == -1
        history = np.concatenate([history, picks[:, None]], axis=1)
    for module, x, y, a, b in seen:
        ids = torch.tensor(adapter, dtype=torch.int32, device="cuda").repeat_interleave(x.shape[1])
        s = dict(x=x.flatten(0, 1), a=a, b=b, ids=ids, w=module.weight.detach(), bias=module.bias.detach(), scale=torch.ones(3, device="cuda"))
        _check_project(SimpleNamespace(adapter_project=lambda *_, **__: y.flatten(0, 1)), s, scale=False)
    batch.remove()
    assert model.model.layers[0].self_attn.q_proj.forward == plain


def test_encrypted_decode_under_rules():
    """Eager and captured: three biased tokens in the order of their biases
    (a token once picked loses more than any bias), the rest within the mask."""
    from provenloop_b200 import tensafe_he
    from provenloop_b200.decode_step import HeLoraDecoder
    model, ctx = _model(), tensafe_he.CkksContext(16384)
    dec = HeLoraDecoder(model, ctx, ctx.keygen(0), rank=16, experts=3, seed=2)
    mask = torch.full(((model.config.vocab_size + 31) // 32,), 0x0F0F_0F0F, dtype=torch.int32, device="cuda")
    rules = dict(presence=torch.full((1,), 1000.0, device="cuda"), bias_ids=torch.tensor([3, 9, 11], device="cuda"),
                 bias_values=torch.tensor([300.0, 200.0, 100.0], device="cuda"), mask=mask)
    run = dec.capture(max_len=8, rules=rules)
    for decode, n in ((lambda p, n: dec.generate([p], tokens=n, rules=rules), 5), (run, 5), (run, 8)):
        out = decode(151643, n)
        torch.cuda.synchronize()  # run works on a stream of its own
        ids = out[0].tolist()
        assert ids[:3] == [3, 9, 11] and len(set(ids)) == len(ids)
        assert all(t >= 0 and t % 8 < 4 for t in ids)
    dec.remove()


def test_no_wait_ran_out():
    """Collected last: none of the calls above gave up a wait in a kernel."""
    import ctypes as C
    from provenloop_b200._lib import check, lib
    v = C.c_uint64(1)
    check(lib().ts_expired_waits(0, C.byref(v)))
    assert v.value == 0
