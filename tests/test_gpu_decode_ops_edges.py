"""GPU checks of the plaintext decode-step operators where launches, memory or
values are out of the ordinary."""
import ctypes as C

import pytest
import torch

from tests.test_gpu_decode_ops import TYPES, _check_backward, _check_project, _inputs

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


def test_no_wait_ran_out():
    """Collected last: none of the calls above gave up a wait in a kernel."""
    from provenloop_b200._lib import check, lib
    v = C.c_uint64(1)
    check(lib().ts_expired_waits(0, C.byref(v)))
    assert v.value == 0
