"""CPU checks of the training operators' refusals: the Python entry points on
CPU tensors, and the C entry points' own checks, which come before any CUDA
call."""
import ctypes as C
import math
import struct

import pytest
import torch

from provenloop_b200 import _lib, adapters, losses

Z, Y = torch.zeros(4, 6, 100), torch.zeros(4, 6, dtype=torch.int64)
ROW, SEQ = torch.zeros(4, 6), torch.zeros(4)
FLAT = dict(logits=torch.zeros(24, 100), targets=torch.zeros(24, dtype=torch.int64))
STARTS = torch.tensor([0, 5, 24], dtype=torch.int32)


def _grads(t):
    return t.clone().requires_grad_()


ROWS = [
    (dict(logits=torch.zeros(100)), "two dimensions"), (dict(logits=Z.double()), "dtype"), (dict(logits=torch.zeros(4, 100, 6).transpose(1, 2)), "contiguous"),
    (dict(logits=torch.zeros(4, 9, 100)[:, :6]), "one stride"), (dict(logits=torch.zeros(4, 6, 0)), "empty"), (dict(targets=Y.int().short()), "targets"),
    (dict(targets=Y[:3]), "targets"), (dict(targets=Y.view(24)), "targets"), (dict(targets=torch.zeros(6, 4, dtype=torch.int64).t()), "contiguous"),
    (dict(targets=ROW), "targets"), (dict(logits=_grads(Z)), "no_grad"), (dict(logits=None), "tensor"), (dict(), "CUDA")]


@pytest.mark.parametrize("change,match", ROWS)
def test_logprobs_refusals(change, match):
    with pytest.raises(ValueError, match=match):
        losses.token_logprobs(**{**dict(logits=Z, targets=Y), **change})


OUT = [(dict(out=torch.zeros(4, 6, 99)), "out"), (dict(out=Z.half()), "out"), (dict(out=torch.zeros(4, 100, 6).transpose(1, 2)), "contiguous"),
       (dict(out=_grads(Z)), "no_grad")]


@pytest.mark.parametrize("change,match", ROWS + OUT[:2] + [(dict(grad=ROW.half()), "grad"), (dict(grad=SEQ), "grad"), (dict(grad=_grads(ROW)), "no_grad")])
def test_logprobs_backward_refusals(change, match):
    with pytest.raises(ValueError, match=match):
        losses.token_logprobs_backward(**{**dict(grad=ROW, logits=Z, targets=Y), **change})


@pytest.mark.parametrize("change,match", ROWS + [
    (dict(old_logprobs=ROW[:2]), "old_logprobs"), (dict(old_logprobs=ROW.double()), "old_logprobs"), (dict(ref_logprobs=SEQ), "ref_logprobs"),
    (dict(advantages=torch.zeros(3)), "advantages"), (dict(advantages=SEQ.half()), "advantages"), (dict(advantages=None), "tensor"),
    (dict(starts=STARTS), "starts"), (dict(FLAT, old_logprobs=None, starts=STARTS.long()), "starts"),
    (dict(FLAT, old_logprobs=None, starts=STARTS[:1]), "starts"), (dict(FLAT, old_logprobs=None, starts=STARTS, advantages=SEQ[:3]), "advantages"),
    (dict(reduction="mean"), "reduction"), (dict(grad_scale=SEQ), "grad_scale"), (dict(grad_scale=torch.tensor(1.0, dtype=torch.float64)), "grad_scale"),
    (dict(old_logprobs=_grads(ROW)), "no_grad"), (dict(ref_logprobs=_grads(ROW)), "no_grad"), (dict(advantages=_grads(SEQ)), "no_grad"),
    (dict(grad_scale=torch.tensor(1.0, requires_grad=True)), "no_grad"), (dict(FLAT, old_logprobs=None, starts=STARTS, advantages=SEQ[:2]), "CUDA")])
def test_policy_refusals(change, match):
    with pytest.raises(ValueError, match=match):
        losses.policy_loss(**{**dict(logits=Z, targets=Y, old_logprobs=ROW, advantages=SEQ), **change})


def test_policy_arguments_that_are_no_numbers():
    for bad in (dict(clip=(0.2, "x")), dict(kl="x"), dict(kl=None)):
        with pytest.raises(TypeError):
            losses.policy_loss(Z, Y, ROW, SEQ, **bad)
    with pytest.raises(TypeError):
        losses.policy_loss(Z, Y, ROW, SEQ, clip=0.2)


@pytest.mark.parametrize("change,match", ROWS + [
    (dict(ref_logprobs=SEQ), "ref_logprobs"), (dict(logits=Z[:3], targets=Y[:3]), "rejected"), (dict(FLAT), "rejected"), (dict(kind="ipo"), "kind"),
    (dict(FLAT, starts=torch.zeros(4, dtype=torch.int32)), "rejected"), (dict(grad_scale=SEQ), "grad_scale"), (dict(FLAT, starts=STARTS), "CUDA")])
def test_preference_refusals(change, match):
    with pytest.raises(ValueError, match=match):
        losses.preference_loss(**{**dict(logits=Z, targets=Y), **change})


def test_forward_mode_tangents_are_refused():
    import torch.autograd.forward_ad as fw
    policy = dict(logits=Z, targets=Y, old_logprobs=ROW, advantages=SEQ, ref_logprobs=ROW.clone(), grad_scale=torch.tensor(1.0))
    calls = [(losses.token_logprobs, dict(logits=Z, targets=Y)), (losses.token_logprobs_backward, dict(grad=ROW, logits=Z, targets=Y)),
             (losses.policy_loss, policy), (losses.preference_loss, dict(logits=Z, targets=Y, ref_logprobs=ROW, grad_scale=torch.tensor(1.0)))]
    with fw.dual_level():
        for call, args in calls:
            for name, t in args.items():
                if t.is_floating_point():
                    with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
                        call(**{**args, name: fw.make_dual(t, torch.ones_like(t))})
        with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
            adapters.clip_gradients([fw.make_dual(ROW, ROW)], 1.0)


@pytest.mark.parametrize("change,match", [
    (dict(grads=[]), "no tensors"), (dict(grads=[None]), "no tensors"), (dict(grads=ROW), "list"), (dict(grads=3), "list"), (dict(grads=[ROW, 3]), "tensor"),
    (dict(grads=[ROW.double()]), "dtype"), (dict(grads=[ROW[:, ::2]]), "dense"), (dict(grads=[torch.zeros(1, 5).expand(4, 5)]), "dense"),
    (dict(adapters=0), "adapters"), (dict(adapters=65536), "adapters"), (dict(adapters=3), "leading"), (dict(grads=[ROW.t()], adapters=6), "contiguous"),
    (dict(grads=[torch.tensor(1.0)], adapters=1), "leading"), (dict(out=[]), "as many"), (dict(out=[ROW.half()]), "out"), (dict(out=[SEQ]), "out"),
    (dict(out=[torch.zeros(6, 4).t()]), "layout"), (dict(max_norm=-1.0), "negative"), (dict(max_norm=math.nan), "negative"),
    (dict(max_norm=torch.zeros(4)), "max_norm"), (dict(max_norm=torch.tensor(1.0, dtype=torch.float64)), "max_norm"),
    (dict(max_norm=torch.zeros(3), adapters=4), "max_norm"), (dict(max_norm=torch.zeros(4), adapters=4), "CUDA"),
    (dict(grads=[_grads(ROW)]), "no_grad"), (dict(), "CUDA")])
def test_clip_refusals(change, match):
    with pytest.raises(ValueError, match=match):
        adapters.clip_gradients(**{**dict(grads=[ROW], max_norm=1.0), **change})


# ---------------------------------------------------------------- C entry points

_F = ("dtype device stream n vocab targets64 logits logits_stride targets grad_logprobs sequences kind starts old ref advantages advantage_rows "
      "average clip_low clip_high kl beta smoothing reserved grad_scale loss margins logprobs grad grad_stride workspace workspace_bytes").split()
G = 1 << 32  # fake, far apart device addresses
OPS = ["ts_token_logprobs", "ts_token_logprobs_backward", "ts_policy_loss", "ts_preference_loss"]


def _loss_args(op, **kw):
    d = dict.fromkeys(_F, 0)
    d.update(dtype=1, n=4, vocab=100, logits=1 * G, logits_stride=100, targets=2 * G)
    if op != 1:
        d.update(logprobs=3 * G)
    if op:
        d.update(grad=4 * G, grad_stride=100)
    if op == 1:
        d.update(grad_logprobs=5 * G)
    if op > 1:
        d.update(sequences=2, loss=6 * G, ref=7 * G)
    if op == 2:
        d.update(old=8 * G, advantages=9 * G, clip_low=0.2, clip_high=0.2)
    if op == 3:
        d.update(margins=10 * G, beta=0.1)
    d.update(kw)
    return losses._ARGS.pack(*(d[k] for k in _F))


def _refused(op, match, **kw):
    assert getattr(_lib.lib(), OPS[op])(_loss_args(op, **kw)) == _lib.TS_ERR_ARG
    assert match in _lib.last_error()


@pytest.mark.parametrize("op", range(4))
@pytest.mark.parametrize("change,match", [
    (dict(dtype=3), "dtype"), (dict(vocab=0), "vocab"), (dict(vocab=(1 << 30) + 1), "vocab"), (dict(n=1 << 28), "rows"), (dict(reserved=1), "reserved"),
    (dict(logits_stride=-1), "stride"), (dict(logits=0), "NULL"), (dict(targets=0), "NULL"), (dict(logits=G + 1), "aligned"),
    (dict(targets=2 * G + 4, targets64=1), "aligned")])
def test_c_row_refusals(op, change, match):
    _refused(op, match, **change)


@pytest.mark.parametrize("op,change,match", [
    (0, dict(logprobs=0), "NULL"), (0, dict(grad=4 * G), "no place"), (0, dict(loss=6 * G), "no place"), (0, dict(grad_logprobs=5 * G), "no place"),
    (0, dict(logprobs=2 * G), "overlaps"), (0, dict(logprobs=G + 400), "overlaps"), (1, dict(grad=0), "NULL"), (1, dict(grad_logprobs=0), "NULL"),
    (1, dict(logprobs=3 * G), "no place"), (1, dict(sequences=2), "no place"), (1, dict(grad_stride=99), "rows of grad"),
    (1, dict(grad=G, grad_stride=101), "overlaps"), (1, dict(grad=G + 2), "overlaps"), (1, dict(grad=5 * G), "overlaps"),
    (2, dict(loss=0), "NULL"), (2, dict(advantages=0), "NULL"), (2, dict(sequences=3), "divide"), (2, dict(sequences=0), "divide"),
    (2, dict(kind=3), "reduction"), (2, dict(kind=-1), "reduction"), (2, dict(clip_low=1.5), "clip_low"), (2, dict(clip_low=-0.1), "clip_low"),
    (2, dict(clip_high=math.nan), "clip_low"), (2, dict(kl=math.inf), "kl"), (2, dict(margins=10 * G), "no place"), (2, dict(loss=4 * G + 8), "overlap"),
    (2, dict(grad_scale=3 * G), "overlaps"), (2, dict(starts=11 * G, sequences=0), "starts"), (2, dict(advantages=9 * G + 2), "aligned"), (2, dict(), "workspace"),
    (2, dict(workspace=12 * G + 8, workspace_bytes=1 << 20), "workspace"), (2, dict(workspace=12 * G, workspace_bytes=8), "workspace"),
    (2, dict(workspace=3 * G, workspace_bytes=1 << 20), "overlap"), (3, dict(sequences=1), "pairs"), (3, dict(kind=3), "kind"), (3, dict(beta=0.0), "beta"),
    (3, dict(beta=math.inf), "beta"), (3, dict(smoothing=0.6), "smoothing"), (3, dict(smoothing=0.1, kind=1), "smoothing"), (3, dict(old=8 * G), "no place"),
    (3, dict(advantages=9 * G), "no place"), (3, dict(margins=6 * G), "overlap"), (3, dict(), "workspace")])
def test_c_loss_refusals(op, change, match):
    _refused(op, match, **change)


def test_c_loss_workspace():
    v = C.c_uint64()
    L = _lib.lib()
    for op in (0, 1):
        assert L.ts_loss_workspace(_loss_args(op), op, C.byref(v)) == 0 and v.value == 0
    for op in (2, 3):
        assert L.ts_loss_workspace(_loss_args(op), op, C.byref(v)) == 0 and v.value > 0
        assert L.ts_loss_workspace(_loss_args(op, beta=-1.0, kind=9), op, C.byref(v)) == _lib.TS_ERR_ARG
    assert L.ts_loss_workspace(_loss_args(0), 4, C.byref(v)) == _lib.TS_ERR_ARG
    assert L.ts_loss_workspace(_loss_args(0), 0, None) == _lib.TS_ERR_ARG
    assert L.ts_loss_workspace(None, 0, C.byref(v)) == _lib.TS_ERR_ARG
    for name in OPS:
        assert getattr(L, name)(None) == _lib.TS_ERR_ARG
    for op in (0, 1):
        assert getattr(L, OPS[op])(_loss_args(op, n=0)) == 0


def _clip_args(tensors, **kw):
    blob = b"".join(adapters._CLIP_TENSOR.pack(*t) for t in tensors)
    d = dict(device=0, groups=3, stream=0, count=len(tensors), tensors=0, max_norms=0, max_norm=1.0, one_max=0, norms=9 * G, workspace=0, workspace_bytes=0)
    d.update(kw)
    keep = C.create_string_buffer(blob, max(1, len(blob)))
    if tensors:
        d["tensors"] = C.addressof(keep)
    return adapters._CLIP_ARGS.pack(*d.values()), keep


def _tensor(grad=1 * G, out=None, elements=300, dtype=1, out_dtype=None):
    return grad, grad if out is None else out, elements, dtype, dtype if out_dtype is None else out_dtype


@pytest.mark.parametrize("tensors,change,match", [
    ([_tensor()], dict(groups=0), "groups"), ([_tensor()], dict(groups=65536), "groups"), ([_tensor()], dict(norms=0), "norms"),
    ([_tensor()], dict(max_norm=-1.0), "max_norm"), ([_tensor()], dict(max_norm=math.nan), "max_norm"), ([], dict(count=2), "tensors"),
    ([_tensor(dtype=3)], {}, "dtype"), ([_tensor(out=2 * G, out_dtype=2)], {}, "out_dtype"), ([_tensor(elements=301)], {}, "divide"),
    ([_tensor(grad=0)], {}, "NULL"), ([_tensor(grad=G + 1)], {}, "aligned"), ([_tensor(out_dtype=0)], {}, "overlap"),
    ([_tensor(), _tensor()], {}, "overlap"), ([_tensor(), _tensor(grad=G + 598)], {}, "overlap"), ([_tensor(out=G + 2)], {}, "overlap"),
    ([_tensor(out=2 * G), _tensor(grad=3 * G, out=2 * G + 598)], {}, "overlap"), ([_tensor(grad=9 * G - 596)], {}, "overlap"),
    ([_tensor()], dict(max_norms=9 * G), "overlap"), ([_tensor()], dict(max_norms=G), "overlap"), ([_tensor()], {}, "workspace"),
    ([_tensor()], dict(workspace=8 * G + 8, workspace_bytes=1 << 20), "workspace"), ([_tensor()], dict(workspace=8 * G, workspace_bytes=8), "workspace"),
    ([_tensor()], dict(workspace=G, workspace_bytes=1 << 20), "overlap"), ([_tensor(elements=3 << 40)], {}, "elements"),
    ([_tensor(grad=(k + 1) << 44, elements=1 << 40, dtype=0) for k in range(9)], dict(groups=1, norms=G), "too many")])
def test_c_clip_refusals(tensors, change, match):
    args, keep = _clip_args(tensors, **change)
    assert _lib.lib().ts_clip_gradients(args) == _lib.TS_ERR_ARG
    assert match in _lib.last_error()


def test_c_clip_workspace():
    v = C.c_uint64()
    L = _lib.lib()
    for tensors in ([], [_tensor(elements=0)], [_tensor()], [_tensor(out=2 * G), _tensor(out=3 * G)]):
        args, keep = _clip_args(tensors)
        assert L.ts_clip_workspace(args, C.byref(v)) == 0 and v.value > 0
        assert L.ts_clip_workspace(args, None) == _lib.TS_ERR_ARG
    assert L.ts_clip_workspace(None, C.byref(v)) == _lib.TS_ERR_ARG
    assert L.ts_clip_gradients(None) == _lib.TS_ERR_ARG


def test_blocks_have_the_headers_sizes(tmp_path):
    """What the Python side packs is what a C compiler lays out."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "tsgpu.h"\nint main(void) { printf("%zu %zu %zu", sizeof(ts_loss_args), sizeof(ts_clip_args), '
                   'sizeof(ts_clip_tensor)); }\n')
    subprocess.check_call(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "sizes")])
    sizes = subprocess.check_output([str(tmp_path / "sizes")]).split()
    assert [int(s) for s in sizes] == [struct.calcsize(s.format) for s in (losses._ARGS, adapters._CLIP_ARGS, adapters._CLIP_TENSOR)]
