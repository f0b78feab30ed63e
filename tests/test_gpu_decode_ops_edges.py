"""GPU checks of the plaintext decode-step operators where launches, memory or
values are out of the ordinary."""
import ctypes as C

import pytest
import torch

from tests.test_gpu_decode_ops import TYPES, _check_backward, _check_project, _high64, _inputs, _low64

pytestmark = pytest.mark.gpu


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


def _c_args(A, s, back, out, da=None, db=None, ws=None):
    """ts_adapter_args for contiguous tensors."""
    p = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    n, i = s["x"].shape
    e, r, _ = s["a"].shape
    o = s["b"].shape[1]
    return A._ARGS.pack({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[s["x"].dtype], 0,
                        torch.cuda.current_stream().cuda_stream, n, 1, i, o, r, e, p(s["x"]), i, p(s["w"]), i, 0, 0, 0, p(s["a"]), p(s["b"]),
                        p(s["ids"]), p(s["scale"]), p(s["dy"]) if back else 0, o, p(out), i if back else o, p(da), p(db), p(ws),
                        0 if ws is None else ws.numel())


def _c_results(s, back):
    if back:
        return [torch.empty_like(s[q]) for q in ("x", "a", "b")]
    return [torch.empty((s["x"].shape[0], s["b"].shape[1]), dtype=s["x"].dtype, device="cuda")]


def _c_room(A, s, back):
    from provenloop_b200._lib import check, lib
    v = C.c_uint64()
    check(lib().ts_adapter_workspace(_c_args(A, s, back, *_c_results(s, back)), int(back), C.byref(v)))
    return v.value


def _c_call(A, s, back, ws):
    """One call through the C entry point in the given workspace; its results."""
    from provenloop_b200._lib import check, lib
    outs = _c_results(s, back)
    args = _c_args(A, s, back, *outs, *(() if back else (None, None)), ws)
    check((lib().ts_adapter_project_backward if back else lib().ts_adapter_project)(args))
    return outs


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("shapes", [
    ((12, 1537, 1535, 16, 3, "mixed"), (40, 521, 777, 8, 3, "mixed")),          # contractions shared by clusters, low token by token
    ((200, 4105, 1001, 16, 3, "ragged"), (700, 4105, 333, 33, 9, "ragged")),    # the same, low on the tensor cores
    ((2300, 521, 1537, 16, 3, "ragged"), (1300, 1001, 2057, 17, 20, "ragged")),  # persistent tiles after both kinds of low
], ids=["few", "split", "tiles"])
def test_rows_off_16_bytes_queued_one_behind_the_other(A, shapes, dt, back, captured):
    """Operands that are copied to the workspace first: calls with new values
    in the same tensors, of two shapes in turn, in one workspace that holds
    NaNs before each of them, queued faster than the GPU works them off."""
    sets = 3
    data = [[_inputs(*shape[:5], dt, shape[5], seed=40 + k) for k in range(sets)] for shape in shapes]
    want = []
    for k in range(sets):
        for d in data:
            if back:
                want.append([t.clone() for t in _check_backward(A, d[k])])
            else:
                want.append([_check_project(A, d[k], bias=False).clone()])
            torch.cuda.synchronize()
    live = [{q: t.clone() for q, t in d[0].items()} for d in data]
    ws = torch.empty(max(_c_room(A, s, back) for s in live), dtype=torch.uint8, device="cuda")
    busy = torch.randn((4096, 4096), device="cuda")

    def queue():
        got = []
        for _ in range(4):
            busy @ busy
        for k in range(sets):
            for s, d in zip(live, data):
                for q in ("x", "w", "dy", "a", "b", "ids", "scale"):
                    s[q].copy_(d[k][q])
                ws.fill_(0xff)
                got.append(_c_call(A, s, back, ws))
        return got

    if captured:
        queue()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = queue()
        for _ in range(3):
            graph.replay()
    else:
        got = queue()
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(g, w))


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("vocab", [1, 127, 130, 700, 1024])
def test_rules_rows_shorter_than_their_cluster(R, vocab, dt):
    """One row is split over eight CTAs, most of which get no token of a small
    vocabulary and bring their (empty) pick at once: the pick is the row's
    wherever it lies, also on a busy GPU."""
    rows = torch.full((vocab, vocab), -1.0, dtype=TYPES[dt], device="cuda")
    rows.fill_diagonal_(1.0)
    mask = torch.full(((vocab + 31) // 32,), -1, dtype=torch.int32, device="cuda")
    busy = torch.randn((2048, 2048), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            busy @ busy
    at = list(range(vocab)) if vocab < 200 else list(range(0, vocab, 7)) + [vocab - 1]
    picks = [R.apply_rules(rows[i:i + 1], mask=mask if i % 2 else None, write=False)[1] for i in at]
    torch.cuda.synchronize()
    assert torch.cat(picks).tolist() == at


def _special64(s, weight):
    """y, dx, da and db in 64 bits, with the terms' absolute sums, of 16 or 32
    bit inputs that hold infinities."""
    x, dy, a, b, ids = s["x"].double(), s["dy"].double(), s["a"].double(), s["b"].double(), s["ids"]
    low, lmag = _low64(x, a, s["scale"], ids)
    u, umag = _low64(dy, b.transpose(1, 2), s["scale"], ids)
    y, ymag = _high64(low, lmag, b.transpose(1, 2), ids)
    dx, dxmag = _high64(u, umag, a, ids)
    if weight:
        w = s["w"].double()
        y, ymag, dx, dxmag = y + x @ w.T, ymag + x.abs() @ w.T.abs(), dx + dy @ w, dxmag + dy.abs() @ w.abs()
    own = [(ids == e).nonzero()[:, 0] for e in range(a.shape[0])]
    da, damag = (torch.stack([p[r].T @ q[r] for r in own]) for p, q in ((u, x), (umag, x.abs())))
    db, dbmag = (torch.stack([p[r].T @ q[r] for r in own]) for p, q in ((dy, low), (dy.abs(), lmag)))
    return (y, dx, da, db), (ymag, dxmag, damag, dbmag)


def _same_where_special(got, want, mag, terms):
    """Infinities and NaNs where the 64-bit values have them, and the other
    values near those: half a step of the type, the intermediate's 11 bits at
    least, and sums of `terms` in 32 bits."""
    t, got = got.dtype, got.double()
    special = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[special].nan_to_num(0.0), want[special].nan_to_num(0.0))
    tol = torch.finfo(t).eps / 2 * want.abs() + ((0 if t is torch.float32 else 2.0 ** -11) + (terms + 8) * 2.0 ** -23) * 1.01 * mag + 2.0 ** -25
    assert ((got - want).abs() <= tol)[~special].all()


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("weight", [True, False])
@pytest.mark.parametrize("n,i,o,r", [(9, 264, 200, 16), (70, 136, 328, 30), (300, 264, 136, 64), (700, 4104, 264, 16), (2400, 264, 7176, 1)])
def test_infinities_stay_infinities(A, n, i, o, r, weight, dt):
    """An infinity in an input makes those results infinite (or, where
    infinities of both signs or a zero meet it, not a number) that it makes so in
    64 bits, of the adapters' gradients too."""
    s = _inputs(n, i, o, r, 3, dt, "mixed", seed=60)
    s["ids"] = torch.where(torch.arange(n, device="cuda") == n // 2, 1, torch.arange(n, device="cuda") % 2 * 2).int()
    m, inf = n // 2, float("inf")
    puts = (("x", (m, 5), inf), ("dy", (m, 7), -inf), ("a", (1, r - 1, 3), inf), ("b", (1, 130, 0), -inf), ("scale", (1,), inf))
    for names in (("x",), ("dy",), ("a",), ("b",), ("scale",), ("x", "b"), ("a", "dy")):
        q = dict(s)
        for name, at, value in puts:
            if name in names:
                q[name] = s[name].clone()
                q[name][at] = value
        y = A.adapter_project(q["x"], q["a"], q["b"], q["ids"], weight=q["w"] if weight else None, scale=q["scale"])
        got = (y, *A.adapter_project_backward(q["dy"], q["x"], q["a"], q["b"], q["ids"], weight=q["w"] if weight else None, scale=q["scale"]))
        want, mags = _special64(q, weight)
        for g, w, mag, terms in zip(got, want, mags, (i + r, o + r, o + n, i + n)):
            _same_where_special(g, w, mag, terms)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [1, 33, 200])
def test_largest_values_stay_finite(A, n, dt):
    """Gradients of the largest inputs and intermediates, which round to
    infinity in fewer bits than they have, are finite where they are in 64 bits."""
    s = _inputs(n, 72, 40, 16, 1, dt, "one", seed=61)
    s["x"].zero_(), s["a"].zero_(), s["dy"].mul_(2.0 ** -8)
    s["x"][:, 3] = torch.finfo(TYPES[dt]).max if n == 1 else 2.0 ** 120
    s["a"][:, :, 3] = 1.0
    s["scale"].fill_(1.003 if dt == "bf16" else 1.0)  # bf16: the intermediate is behind the type's largest value
    got = A.adapter_project_backward(s["dy"], s["x"], s["a"], s["b"], s["ids"], scale=s["scale"])
    want, mags = _special64(s, False)
    for g, w, mag, terms in zip(got, want[1:], mags[1:], (56, 40 + n, 72 + n)):
        assert torch.isfinite(g).all()
        _same_where_special(g, w, mag, terms)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("n,i,o,r,weight", [(1, 16, 200, 1, True), (16, 8, 200, 3, False), (40, 16, 333, 2, True),
                                            (300, 24, 1001, 1, False), (300, 16, 264, 3, True), (200, 9, 520, 2, True)])
def test_intermediate_keeps_its_bits(A, n, i, o, r, weight, dt):
    """Where the other terms cancel the adapter's but for a rounding, the
    result shows the intermediate's last bits: sums of k terms in 32 bits are
    off by less than (k + 8) 2^-23 of the terms' absolute sum, and nothing else is
    rounded before the result."""
    s = _inputs(n, i, o, r, 3, dt, "ragged", seed=70)
    low, lmag = _low64(s["x"], s["a"], s["scale"], s["ids"])
    y, mag = _high64(low, lmag, s["b"].transpose(1, 2), s["ids"])
    if weight:
        y, mag = y + s["x"].double() @ s["w"].double().T, mag + s["x"].double().abs() @ s["w"].double().abs().T
    base = (-y).to(s["x"].dtype)
    got = A.adapter_project(s["x"], s["a"], s["b"], s["ids"], weight=s["w"] if weight else None, base=base, scale=s["scale"])
    want, mag = y + base.double(), mag + base.double().abs()
    tol = torch.finfo(got.dtype).eps / 2 * want.abs() + (2 * i + r + 8) * 2.0 ** -23 * mag + 2.0 ** -25
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dt,bits", [("bf16", 15), ("fp16", 20), ("fp32", 22)])
@pytest.mark.parametrize("n,i,o,r", [(2, 72, 40, 3), (40, 264, 200, 16), (500, 264, 136, 64), (3000, 4104, 40, 16)])
def test_gradients_keep_the_intermediates_bits(A, n, i, o, r, dt, bits):
    """Pairs of tokens whose terms cancel but for a small difference of their
    intermediates, which hold to a relative 2^-bits; sums of n terms in 32 bits."""
    s = _inputs(n, i, o, r, 1, dt, "one", seed=71)
    s["x"][1::2] = s["x"][::2]
    s["x"][1::2, :3] += 2.0 ** -6
    s["dy"][1::2] = -s["dy"][::2]
    s["dy"][1::2, :3] += 2.0 ** -6
    _, da, db = A.adapter_project_backward(s["dy"], s["x"], s["a"], s["b"], s["ids"], scale=s["scale"])
    (_, _, wa, wb), (_, _, ma, mb) = _special64(s, False)
    low = _low64(s["x"], s["a"], s["scale"], s["ids"])[0].abs()
    u = _low64(s["dy"], s["b"].transpose(1, 2), s["scale"], s["ids"])[0].abs()
    held = (u.T @ s["x"].double().abs(), s["dy"].double().abs().T @ low)  # of the products with the intermediates
    for g, w, mag, h, k in zip((da, db), (wa, wb), (ma, mb), held, (o, i)):
        tol = torch.finfo(g.dtype).eps / 2 * w.abs() + 2.0 ** -bits * h + (k + 8) * 2.0 ** -23 * mag + (n + 8) * 2.0 ** -23 * h + 2.0 ** -25
        assert ((g.double() - w).abs() <= tol * 1.01).all()


def test_autograd_sees_what_is_overwritten(A, R):
    """A tensor that autograd has saved and a call writes over makes the
    backward pass an error, not a wrong gradient."""
    s = _inputs(6, 64, 40, 8, 2, "fp32", "one")
    w = torch.ones(40, device="cuda", requires_grad=True)
    for write in (lambda t: A.adapter_project(s["x"], s["a"], s["b"], s["ids"], out=t),
                  lambda t: A.adapter_project(s["x"], s["a"], s["b"], s["ids"], base=t, out=t),
                  lambda t: R.apply_rules(t, out=t), lambda t: R.apply_rules(s["base"], out=t[:, :])):
        saved = s["base"].clone()
        loss = (saved * w).sum()
        with torch.no_grad():
            write(saved)
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()
    with torch.inference_mode():  # tensors that count no versions
        made = torch.zeros((6, 40), device="cuda")
    assert A.adapter_project(s["x"], s["a"], s["b"], s["ids"], out=made) is made and made.any()


def test_expired_waits_are_counted_behind_the_work():
    """ts_expired_waits waits for streams that the legacy stream does not."""
    from provenloop_b200._lib import check, lib
    busy, v = torch.randn((8192, 8192), device="cuda"), C.c_uint64(1)
    check(lib().ts_expired_waits(0, C.byref(v)))
    side, done = torch.cuda.Stream(), torch.cuda.Event()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            busy @ busy
        done.record()
    assert not done.query()
    check(lib().ts_expired_waits(0, C.byref(v)))
    assert done.query() and v.value == 0


def test_captured_decode_sees_rules_changed_before_it():
    """New values of the rules' tensors, queued on the current stream behind
    other work, are the ones that the replay reads."""
    from provenloop_b200 import tensafe_he
    from provenloop_b200.decode_step import HeLoraDecoder, build_model
    model, ctx = build_model(layers=1), tensafe_he.CkksContext(16384)
    dec = HeLoraDecoder(model, ctx, ctx.keygen(0), rank=16, experts=3, seed=2)
    mask = torch.zeros(((model.config.vocab_size + 31) // 32,), dtype=torch.int32, device="cuda")
    run = dec.capture(max_len=4, rules=dict(mask=mask))
    busy = torch.randn((8192, 8192), device="cuda")
    torch.cuda.synchronize()
    for allowed in (5, 77):
        for _ in range(20):
            busy @ busy
        mask.zero_()
        mask[allowed // 32:allowed // 32 + 1].fill_(1 << allowed % 32)
        out = run(1, 3)
        torch.cuda.synchronize()
        assert out.tolist() == [[allowed] * 3]
    dec.remove()


def test_no_wait_ran_out():
    """Collected last: none of the calls above gave up a wait in a kernel."""
    from provenloop_b200._lib import check, lib
    v = C.c_uint64(1)
    check(lib().ts_expired_waits(0, C.byref(v)))
    assert v.value == 0
