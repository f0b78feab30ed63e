"""CPU checks of the plaintext decode-step operators' refusals: the Python
entry points on CPU tensors, and the C entry points' own checks, which come
before any CUDA call."""
import ctypes as C

import numpy as np
import pytest
import torch

from provenloop_b200 import _lib, adapters, logits


def _tensors(n=4, i=16, o=24, r=4, e=3, t=torch.float32):
    return dict(x=torch.zeros(n, i, dtype=t), lora_a=torch.zeros(e, r, i, dtype=t), lora_b=torch.zeros(e, o, r, dtype=t),
                adapter=torch.zeros(n, dtype=torch.int32))


@pytest.mark.parametrize("change,match", [
    (dict(x=torch.zeros(16)), "two dimensions"),
    (dict(x=torch.zeros(4, 16, dtype=torch.float64)), "dtype"),
    (dict(x=torch.zeros(16, 4).T), "contiguous"),
    (dict(x=torch.zeros(4, 3, 16)[:, :2]), "one stride"),
    (dict(lora_a=torch.zeros(3, 4, 15)), "lora_a"),
    (dict(lora_a=torch.zeros(4, 16)), "lora_a must be"),
    (dict(lora_a=torch.zeros(3, 16, 4).transpose(1, 2)), "contiguous"),
    (dict(lora_b=torch.zeros(2, 24, 4)), "lora_b"),
    (dict(lora_b=torch.zeros(3, 24, 4, dtype=torch.bfloat16)), "lora_b"),
    (dict(adapter=torch.zeros(4, dtype=torch.int64)), "int32"),
    (dict(adapter=torch.zeros(5, dtype=torch.int32)), "adapter"),
    (dict(adapter=torch.tensor(0, dtype=torch.int32)), "adapter"),
    (dict(weight=torch.zeros(24, 17)), "weight"),
    (dict(weight=torch.zeros(16, 24).T), "weight"),
    (dict(bias=torch.zeros(23)), "bias"),
    (dict(base=torch.zeros(4, 23)), "base"),
    (dict(scale=torch.zeros(3, dtype=torch.float64)), "scale"),
    (dict(scale=torch.zeros(4)), "scale"),
    (dict(out=torch.zeros(4, 24, dtype=torch.bfloat16)), "out"),
    (dict(x=torch.zeros(4, 16, requires_grad=True)), "no_grad"),
    (dict(weight=torch.zeros(24, 16, requires_grad=True)), "no_grad"),
    (dict(), "CUDA"),
])
def test_project_refusals(change, match):
    with pytest.raises(ValueError, match=match):
        adapters.adapter_project(**{**_tensors(), **change})


@pytest.mark.parametrize("change,match", [
    (dict(grad=torch.zeros(4, 23)), "grad"), (dict(grad=torch.zeros(4, 24, dtype=torch.float16)), "grad"),
    (dict(need_x=False, need_adapters=False), "no gradient"), (dict(grad=torch.zeros(4, 24, requires_grad=True)), "no_grad"),
    (dict(), "CUDA")])
def test_backward_refusals(change, match):
    with pytest.raises(ValueError, match=match):
        adapters.adapter_project_backward(**{"grad": torch.zeros(4, 24), **_tensors(), **change})


@pytest.mark.parametrize("change,match", [
    (dict(logits=torch.zeros(100)), "logits"), (dict(logits=torch.zeros(2, 100, dtype=torch.float64)), "dtype"),
    (dict(logits=torch.zeros(100, 2).T), "contiguous"), (dict(logits=torch.zeros(2, 0)), "empty"),
    (dict(tokens=torch.zeros(3, 5, dtype=torch.int64)), "tokens"), (dict(tokens=torch.zeros(2, 5)), "tokens"),
    (dict(tokens=torch.zeros(5, dtype=torch.int64)), "tokens"),
    (dict(tokens=torch.zeros(2, 1048576, dtype=torch.int32)), "1048575"),
    (dict(lengths=torch.zeros(2, dtype=torch.int32)), "needs tokens"), (dict(repetition=torch.ones(2)), "needs tokens"),
    (dict(tokens=torch.zeros(2, 5, dtype=torch.int64), lengths=torch.zeros(2, dtype=torch.int64)), "lengths"),
    (dict(tokens=torch.zeros(2, 5, dtype=torch.int64), frequency=torch.zeros(3)), "frequency"),
    (dict(bias_ids=torch.zeros(2, 5, dtype=torch.int64)), "together"),
    (dict(bias_ids=torch.zeros(2, 5, dtype=torch.int64), bias_values=torch.zeros(2, 4)), "bias_values"),
    (dict(bias_ids=torch.zeros(4096, dtype=torch.int64), bias_values=torch.zeros(4096)), "4095"),
    (dict(mask=torch.zeros(2, 3, dtype=torch.int32)), "mask"), (dict(mask=torch.zeros(2, 4, dtype=torch.int64)), "mask"),
    (dict(mask=torch.zeros(3, 4, dtype=torch.int32)), "mask"),
    (dict(out=torch.zeros(2, 100, dtype=torch.float16)), "out"), (dict(out=torch.zeros(2, 100), write=False), "write"),
    (dict(write=False, pick=False), "neither"), (dict(logits=torch.zeros(2, 100, requires_grad=True)), "no_grad"),
    (dict(), "CUDA")])
def test_rules_refusals(change, match):
    with pytest.raises(ValueError, match=match):
        logits.apply_rules(**{"logits": torch.zeros(2, 100), **change})


_RULES = dict(tokens=torch.zeros(2, 5, dtype=torch.int64), repetition=torch.ones(2), frequency=torch.ones(2), presence=torch.ones(2),
              bias_ids=torch.zeros(2, 3, dtype=torch.int64), bias_values=torch.zeros(2, 3))


@pytest.mark.parametrize("name", ["repetition", "frequency", "presence", "bias_values"])
def test_rules_refuse_parameters_that_want_gradients(name):
    change = {name: _RULES[name].clone().requires_grad_()}
    with pytest.raises(ValueError, match="no_grad"):
        logits.apply_rules(**{"logits": torch.zeros(2, 100), **_RULES, **change})
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        logits.apply_rules(**{"logits": torch.zeros(2, 100), **_RULES, **change})


def test_forward_mode_tangents_are_refused():
    import torch.autograd.forward_ad as fw
    scale, bias, base = torch.ones(3), torch.zeros(24), torch.zeros(4, 24)
    project = {**_tensors(), "scale": scale, "bias": bias, "base": base, "weight": torch.zeros(24, 16), "out": torch.zeros(4, 24)}
    back = {**_tensors(), "grad": torch.zeros(4, 24), "scale": scale, "weight": torch.zeros(24, 16)}
    rules = {"logits": torch.zeros(2, 100), **_RULES, "out": torch.zeros(2, 100)}
    with fw.dual_level():
        for call, args in ((adapters.adapter_project, project), (adapters.adapter_project_backward, back), (logits.apply_rules, rules)):
            for name, t in args.items():
                if t.is_floating_point():
                    with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
                        call(**{**args, name: fw.make_dual(t, torch.ones_like(t))})
            with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
                call(**args)


def test_flags_without_a_truth_value():
    both = torch.ones(2, dtype=torch.bool)
    for name in ("need_x", "need_adapters"):
        with pytest.raises(RuntimeError, match="ambiguous"):
            adapters.adapter_project_backward(grad=torch.zeros(4, 24), **_tensors(), **{name: both})
    for name in ("write", "pick"):
        with pytest.raises(RuntimeError, match="ambiguous"):
            logits.apply_rules(torch.zeros(2, 100), **{name: both})


def test_expired_waits_reach_python(monkeypatch):
    asked = []

    class Fake:
        @staticmethod
        def ts_expired_waits(device, out):
            asked.append(device)
            C.cast(out, C.POINTER(C.c_uint64))[0] = 5 + device
            return 0
    monkeypatch.setattr(adapters, "lib", lambda: Fake)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    assert [adapters.expired_waits(d) for d in (None, 2, "cuda", "cuda:1", torch.device("cuda", 4))] == [8, 7, 8, 6, 9]
    assert asked == [3, 2, 3, 1, 4]
    with pytest.raises(ValueError, match="cpu"):
        adapters.expired_waits("cpu")


# ---------------------------------------------------------------- C entry points

_A = ("dtype device stream n per d_in d_out r adapters x x_stride weight w_stride bias base base_stride lora_a lora_b adapter scale "
      "grad grad_stride out out_stride grad_a grad_b workspace workspace_bytes").split()
_R = ("dtype out_dtype device ids64 stream n vocab token_cols bias_cols reserved logits logits_stride tokens tokens_stride lengths "
      "prompt repetition frequency presence bias_ids bi_stride bias_values bv_stride mask mask_stride out out_stride pick").split()
G = 1 << 32  # fake, far apart device addresses


def _adapter_args(**kw):
    d = dict.fromkeys(_A, 0)
    d.update(dtype=1, n=4, per=1, d_in=16, d_out=24, r=4, adapters=3, x=1 * G, x_stride=16, weight=2 * G, w_stride=16, lora_a=3 * G,
             lora_b=4 * G, adapter=5 * G, out=6 * G, out_stride=24)
    d.update(kw)
    return adapters._ARGS.pack(*(d[k] for k in _A))


BACK = dict(grad=7 * G, grad_stride=24, grad_a=8 * G, grad_b=9 * G, out_stride=16)


@pytest.mark.parametrize("change,match", [
    (dict(dtype=3), "dtype"), (dict(d_in=0), "d_in"), (dict(d_out=1 << 25), "d_out"), (dict(r=0), "rank"), (dict(r=257), "rank"),
    (dict(adapters=0), "adapters"), (dict(adapters=65536), "adapters"), (dict(n=1 << 31), "tokens"), (dict(per=0), "tokens_per_id"),
    (dict(x_stride=-1), "stride"), (dict(out_stride=1 << 41), "stride"), (dict(x=0), "NULL"), (dict(lora_a=0), "NULL"),
    (dict(lora_b=0), "NULL"), (dict(adapter=0), "NULL"), (dict(out=0), "NULL"), (dict(x=G + 1), "aligned"), (dict(adapter=G + 2), "aligned"),
    (dict(scale=G + 2), "aligned"), (dict(out_stride=23), "rows of out"), (dict(out=G + 32), "overlaps"), (dict(out=2 * G), "overlaps"),
    (dict(out=5 * G), "overlaps"), (dict(base=6 * G, base_stride=25), "overlaps"), (dict(base=6 * G + 2, base_stride=24), "overlaps"),
    (dict(grad=7 * G), "forward"), (dict(grad_a=7 * G), "forward"), (dict(), "workspace"),
    (dict(workspace=10 * G + 8, workspace_bytes=1 << 20), "workspace"), (dict(workspace=10 * G, workspace_bytes=8), "workspace"),
    (dict(workspace=G, workspace_bytes=1 << 20), "overlaps"), (dict(workspace=6 * G, workspace_bytes=1 << 20), "overlap")])
def test_c_project_refusals(change, match):
    assert _lib.lib().ts_adapter_project(_adapter_args(**change)) == _lib.TS_ERR_ARG
    assert match in _lib.last_error()


@pytest.mark.parametrize("change,match", [
    (dict(out=0, grad_a=0, grad_b=0), "no gradient"), (dict(grad_a=0), "together"), (dict(bias=11 * G), "no place"),
    (dict(base=11 * G), "no place"), (dict(grad=0), "NULL"), (dict(grad_stride=-5), "stride"), (dict(grad_a=7 * G), "overlaps"),
    (dict(grad_b=8 * G + 64), "overlap"), (dict(grad_a=3 * G), "overlaps"), (dict(out_stride=15), "rows of out"), (dict(), "workspace")])
def test_c_backward_refusals(change, match):
    assert _lib.lib().ts_adapter_project_backward(_adapter_args(**{**BACK, **change})) == _lib.TS_ERR_ARG
    assert match in _lib.last_error()


def test_c_columns_of_one_buffer_do_not_overlap():
    # x in columns 0..15 and out in columns 16..39 of one [n][40] buffer: only the missing workspace is refused
    args = _adapter_args(x_stride=40, out=G + 32, out_stride=40)
    assert _lib.lib().ts_adapter_project(args) == _lib.TS_ERR_ARG and "workspace" in _lib.last_error()
    args = _adapter_args(x_stride=40, out=G + 30, out_stride=40)
    assert _lib.lib().ts_adapter_project(args) == _lib.TS_ERR_ARG and "overlaps" in _lib.last_error()


def test_c_workspace_size():
    v = C.c_uint64()
    assert _lib.lib().ts_adapter_workspace(_adapter_args(), 0, C.byref(v)) == 0 and v.value >= 4 * 4 * 4
    one = v.value
    assert _lib.lib().ts_adapter_workspace(_adapter_args(**BACK), 1, C.byref(v)) == 0 and v.value >= one
    assert _lib.lib().ts_adapter_workspace(_adapter_args(), 0, None) == _lib.TS_ERR_ARG
    assert _lib.lib().ts_adapter_workspace(None, 0, C.byref(v)) == _lib.TS_ERR_ARG


def test_c_nothing_to_do_is_ok():
    assert _lib.lib().ts_adapter_project(_adapter_args(n=0)) == 0
    assert _lib.lib().ts_adapter_project(None) == _lib.TS_ERR_ARG
    assert _lib.lib().ts_adapter_project_backward(None) == _lib.TS_ERR_ARG
    assert _lib.lib().ts_logit_rules(None) == _lib.TS_ERR_ARG
    assert _lib.lib().ts_logit_rules(_rules_args(n=0)) == 0


def _rules_args(**kw):
    d = dict.fromkeys(_R, 0)
    d.update(dtype=1, out_dtype=1, n=2, vocab=100, logits=G, logits_stride=100, out=2 * G, out_stride=100, pick=3 * G)
    d.update(kw)
    return logits._ARGS.pack(*(d[k] for k in _R))


@pytest.mark.parametrize("change,match", [
    (dict(dtype=-1), "dtype"), (dict(out_dtype=2), "out_dtype"), (dict(reserved=1), "reserved"), (dict(vocab=0), "vocab"),
    (dict(vocab=(1 << 30) + 1), "vocab"), (dict(n=1 << 28), "rows"), (dict(tokens=4 * G, token_cols=1 << 20), "history"),
    (dict(bias_ids=4 * G, bias_values=5 * G, bias_cols=4096), "biases"), (dict(bias_ids=4 * G), "together"),
    (dict(token_cols=4), "history"), (dict(out=0, pick=0), "neither"),
    (dict(logits=0), "NULL"), (dict(logits_stride=-1), "stride"), (dict(mask=4 * G, mask_stride=-1), "stride"),
    (dict(logits=G + 1), "aligned"), (dict(out=2 * G + 2, out_dtype=0), "aligned"), (dict(pick=3 * G + 4), "aligned"),
    (dict(tokens=4 * G + 4, token_cols=3, tokens_stride=3, ids64=1), "aligned"), (dict(mask=4 * G + 2), "aligned"),
    (dict(out_stride=99), "rows of out"), (dict(out=G, out_dtype=0), "overlaps"), (dict(out=G, out_stride=101), "overlaps"),
    (dict(out=G + 2), "overlaps"), (dict(pick=G + 8), "overlaps"), (dict(pick=2 * G + 8), "overlaps"),
    (dict(mask=2 * G, mask_stride=4), "overlaps"), (dict(tokens=3 * G, token_cols=2, tokens_stride=2), "overlaps")])
def test_c_rules_refusals(change, match):
    assert _lib.lib().ts_logit_rules(_rules_args(**change)) == _lib.TS_ERR_ARG
    assert match in _lib.last_error()


def test_lora_batch_refusals():
    from types import SimpleNamespace as N
    from provenloop_b200.decode_step import LoraBatch
    linear = torch.nn.Linear(4, 4)
    layers = [N(self_attn=N(q_proj=linear, v_proj=torch.nn.Linear(4, 2)))]
    model = N(parameters=linear.parameters, model=N(layers=layers))
    one = tuple(np.zeros(s, np.float32) for s in ((2, 3, 4), (2, 3, 4), (2, 4, 3), (2, 2, 3)))
    with pytest.raises(ValueError, match="layers"):
        LoraBatch(model, [one, one])
    batch = LoraBatch(model, [one])
    x = torch.ones(1, 4)
    assert torch.equal(layers[0].self_attn.q_proj(x), torch.nn.functional.linear(x, linear.weight, linear.bias))  # outside of generate
    for ids, adapter in (([1, 2], [0]), ([[1, 2]], [0, 1]), ([[1, 2]], 0)):
        with pytest.raises(ValueError, match="requests"):
            batch.generate(ids, adapter)
    batch.remove()
    assert "forward" not in linear.__dict__


def _one_layer():
    from types import SimpleNamespace as N
    from provenloop_b200.decode_step import LoraBatch
    linear = torch.nn.Linear(4, 4)
    model = N(parameters=linear.parameters, model=N(layers=[N(self_attn=N(q_proj=linear, v_proj=torch.nn.Linear(4, 2)))]))
    return linear, lambda: LoraBatch(model, [tuple(np.zeros(s, np.float32) for s in ((2, 3, 4), (2, 3, 4), (2, 4, 3), (2, 2, 3)))])


def test_lora_batch_removed_does_not_decode():
    _, make = _one_layer()
    batch = make()
    batch.remove()
    with pytest.raises(RuntimeError, match="removed"):
        batch.generate([[1]], [0])


def test_lora_batches_leave_a_model_in_turn():
    linear, make = _one_layer()
    first, second = make(), make()
    over = linear.forward
    with pytest.raises(RuntimeError, match="first"):
        first.remove()
    assert linear.forward is over  # the second one's adapters are still there
    second.remove()
    first.remove()
    assert "forward" not in linear.__dict__
    first.remove()


def test_lora_batch_on_two_threads(monkeypatch):
    """The batch of one thread keeps its adapters when another one's ends."""
    import threading
    from types import SimpleNamespace as N
    from provenloop_b200 import decode_step
    linear = torch.nn.Linear(4, 4)
    model = N(parameters=linear.parameters, model=N(layers=[N(self_attn=N(q_proj=linear, v_proj=torch.nn.Linear(4, 2)))]))
    batch = decode_step.LoraBatch(model, [tuple(np.zeros(s, np.float32) for s in ((2, 3, 4), (2, 3, 4), (2, 4, 3), (2, 2, 3)))])
    used, both, ended = {}, threading.Barrier(2, timeout=20), threading.Event()
    monkeypatch.setattr(decode_step, "adapter_project", lambda x, a, b, adapter, **kw: used[len(adapter)].append(adapter.tolist()))

    def decode(model, ids, *_):
        n = ids.shape[0]
        used[n] = []
        both.wait()
        if n == 2:
            assert ended.wait(20)
        linear(torch.zeros(n, 1, 4))

    def first():
        batch.generate([[1]], [1])
        ended.set()

    monkeypatch.setattr(decode_step, "_generate", decode)
    thread = threading.Thread(target=first)
    thread.start()
    batch.generate([[1], [2]], [0, -1])
    thread.join()
    assert used == {1: [[1]], 2: [[0, -1]]}
    batch.remove()
