"""Plaintext low-rank adapters of many requests at once.

The plaintext branch of ``_he_lora_delta`` (demonstrator/server/
inference_engine.py:1234-1242), for any number of tokens, each with its own
adapter or none, beside the projection that the adapters belong to:

* ``adapter_project`` -- ``y = x W^T + bias + scale_e (x A_e^T) B_e^T``, or the
  same delta added to a projection that has been computed already;
* ``adapter_project_backward`` -- the gradients for x and for the adapters
  (the projection is frozen), with which adapters are trained.

Both take CUDA tensors, run on torch's current stream of their device and
return without waiting; the workspace comes from torch's allocator, so calls
may be captured in CUDA graphs and run on several streams.  They do not
record autograd history and refuse inputs that ask for it: call them under
``torch.no_grad()``, or from the two halves of a ``torch.autograd.Function``.
"""
from __future__ import annotations

import ctypes as C
import struct

from ._lib import check, lib

_ARGS = struct.Struct("@2iP2Q4IPqPqPPqPPPPPqPqPPPQ")  # ts_adapter_args
_types = {}  # torch dtype -> TS_DTYPE_*
_torch = None


def _load():
    """torch, imported by the first call; the dtype codes."""
    global _torch
    if _torch is None:
        import torch
        _types.update({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2})
        _torch = torch
    return _torch


def _dtype_code(t):
    code = _types.get(t)
    if code is None:
        raise ValueError(f"dtype must be float32, bfloat16 or float16, not {t}")
    return code


def _current_stream(index):
    return _torch._C._cuda_getCurrentRawStream(index)


def _rows(t, name):
    """(n, stride between rows) of t [..., d] seen as [n, d]."""
    dim = t.dim()
    if dim != 2:
        if dim < 2:
            raise ValueError(f"{name} must be [..., d] with at least two dimensions, not {tuple(t.shape)}")
        try:
            t = t.view(-1, t.shape[-1])
        except RuntimeError:
            raise ValueError(f"the leading dimensions of {name} do not form rows of one stride") from None
    row, col = t.stride()
    n, d = t.shape
    if col != 1 and d > 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")
    return n, row


def _same(t, name, dtype, device, shape):
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, not {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, not {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, x on {device}")


def _whole(t, name, dtype, device, shape):
    _same(t, name, dtype, device, shape)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _no_history():
    raise ValueError("an input requires a gradient, which this call does not record: call it under torch.no_grad() and use "
                     "adapter_project_backward")


_sizes = {}  # what the size of a workspace goes by -> bytes


def _workspace_bytes(key, packed, backward):
    size = _sizes.get(key)
    if size is None:
        v = C.c_uint64()
        check(lib().ts_adapter_workspace(packed, backward, C.byref(v)), "ts_adapter_workspace")
        if len(_sizes) > 4096:
            _sizes.clear()
        size = _sizes[key] = v.value
    return size


def _common(x, lora_a, lora_b, adapter, weight, scale):
    """Checks shared by both directions; (code, n, x stride, d_in, d_out, r, adapters, tokens per id, weight stride)."""
    dtype, lead = x.dtype, x.shape
    code = _types.get(dtype)
    if code is None:
        _dtype_code(dtype)
    if len(lead) == 2 and (x.stride(1) == 1 or lead[1] == 1):
        n, x_stride = lead[0], x.stride(0)
    else:
        n, x_stride = _rows(x, "x")
    d_in, lead = lead[-1], lead[:-1]
    a_shape, b_shape, ids = lora_a.shape, lora_b.shape, adapter.shape
    if len(a_shape) != 3 or len(b_shape) != 3:
        raise ValueError("lora_a must be [adapters, r, d_in] and lora_b [adapters, d_out, r]")
    adapters, r, _ = a_shape
    d_out = b_shape[1]
    at, int32 = x.get_device(), _torch.int32
    # accepted at one go; what is not goes through the checks that say why
    if not (lora_a.dtype is dtype and lora_b.dtype is dtype and adapter.dtype is int32 and a_shape[2] == d_in and
            b_shape == (adapters, d_out, r) and lora_a.get_device() == at and lora_b.get_device() == at and adapter.get_device() == at and
            lora_a.is_contiguous() and lora_b.is_contiguous() and adapter.is_contiguous() and ids and ids == lead[:len(ids)]):
        device = x.device
        _whole(lora_a, "lora_a", dtype, device, (adapters, r, d_in))
        _whole(lora_b, "lora_b", dtype, device, (adapters, d_out, r))
        if not ids or ids != lead[:len(ids)]:
            raise ValueError(f"adapter must hold one index per leading entry of x {tuple(lead)}, not {tuple(ids)}")
        _whole(adapter, "adapter", int32, device, ids)
    per = 1
    for s in lead[len(ids):]:
        per *= s
    w_stride = 0
    if weight is not None:
        if not (weight.dtype is dtype and weight.shape == (d_out, d_in) and weight.get_device() == at):
            _same(weight, "weight", dtype, x.device, (d_out, d_in))
        w_stride, col = weight.stride()
        if col != 1 and d_in > 1:
            raise ValueError("the last dimension of weight must be contiguous")
    if scale is not None and not (scale.dtype is _torch.float32 and scale.shape == (adapters,) and scale.get_device() == at and
                                  scale.is_contiguous()):
        _whole(scale, "scale", _torch.float32, x.device, (adapters,))
    if _torch.is_grad_enabled() and (x.requires_grad or lora_a.requires_grad or lora_b.requires_grad or
                                     (weight is not None and weight.requires_grad) or (scale is not None and scale.requires_grad)):
        _no_history()
    return code, n, x_stride, d_in, d_out, r, adapters, per or 1, w_stride


def _call(entry, backward, like, *args):
    """The C call with `args` (the fields of ts_adapter_args but for stream, device and workspace), on like's device."""
    index = like.get_device()
    if index < 0 or not like.is_cuda:
        raise ValueError("the tensors must be on a CUDA device: there is no CPU form")
    code, x, x_stride, w, w_stride, a, grad, grad_stride = args[0], args[7], args[8], args[9], args[10], args[14], args[18], args[19]
    # sizes, strides, alignment and which results are wanted
    key = (code, args[1], args[3], args[4], args[5], args[6], x_stride, w_stride, grad_stride, x & 15, a & 15, grad & 15, w & 15 if w else -1,
           backward and args[20] != 0, args[22] != 0)
    size = _sizes.get(key)
    if size is None:
        size = _workspace_bytes(key, _ARGS.pack(code, index, 0, *args[1:], 0, 0), backward)
    ws = like.new_empty(size, dtype=_torch.uint8)
    rc = entry(_ARGS.pack(code, index, _current_stream(index), *args[1:], ws.data_ptr(), size))
    if rc:
        check(rc, "ts_adapter_project")


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def adapter_project(x, lora_a, lora_b, adapter, weight=None, bias=None, base=None, scale=None, out=None):
    """``base + x W^T + bias + scale_e (x A_e^T) B_e^T``, e the token's adapter.

    x: [..., d_in]; lora_a: [adapters, r, d_in]; lora_b: [adapters, d_out, r];
    adapter: int32, of x's leading shape or a leading part of it (an index per
    request for x [requests, tokens, d_in]); an index outside [0, adapters),
    such as -1, means none.  weight: [d_out, d_in]; bias: [d_out]; base:
    [..., d_out] (each optional, base may be ``out``); scale: float32
    [adapters].  All but adapter and scale share one dtype: float32, bfloat16
    or float16.  Rows may be strided, their elements are contiguous.  A
    NaN or an infinity in one adapter or one token's row stays with the tokens
    that use it.
    Returns ``out`` [..., d_out], allocated unless given."""
    if _torch is None:
        _load()
    code, n, x_stride, d_in, d_out, r, adapters, per, w_stride = _common(x, lora_a, lora_b, adapter, weight, scale)
    shape = (*x.shape[:-1], d_out)
    if bias is not None:
        if not (bias.dtype is x.dtype and bias.shape == (d_out,) and bias.get_device() == x.get_device() and bias.is_contiguous()):
            _whole(bias, "bias", x.dtype, x.device, (d_out,))
        if bias.requires_grad and _torch.is_grad_enabled():
            _no_history()
    base_stride = 0
    if base is not None:
        _same(base, "base", x.dtype, x.device, shape)
        base_stride = _rows(base, "base")[1]
        if base.requires_grad and _torch.is_grad_enabled():
            _no_history()
    if out is None:
        out, out_stride = x.new_empty(shape), d_out
    else:
        _same(out, "out", x.dtype, x.device, shape)
        out_stride = _rows(out, "out")[1]
    _call(lib().ts_adapter_project, 0, x,
          code, n, per, d_in, d_out, r, adapters, x.data_ptr(), x_stride, _ptr(weight), w_stride, _ptr(bias), _ptr(base),
          base_stride, lora_a.data_ptr(), lora_b.data_ptr(), adapter.data_ptr(), _ptr(scale), 0, 0, out.data_ptr(), out_stride, 0, 0)
    return out


def adapter_project_backward(grad, x, lora_a, lora_b, adapter, weight=None, scale=None, need_x=True, need_adapters=True):
    """Gradients of ``adapter_project`` for ``grad`` = d loss / d out, weight,
    bias and scale held fixed: (d x [..., d_in], d lora_a, d lora_b), in the
    inputs' dtype, None where not needed.  An adapter without tokens gets
    zeros.  (The gradient of base is ``grad`` itself.)  The order of every sum
    depends on the sizes and indexes alone."""
    if _torch is None:
        _load()
    code, n, x_stride, d_in, d_out, r, adapters, per, w_stride = _common(x, lora_a, lora_b, adapter, weight, scale)
    if grad.requires_grad and _torch.is_grad_enabled():
        _no_history()
    _same(grad, "grad", x.dtype, x.device, (*x.shape[:-1], d_out))
    grad_stride = _rows(grad, "grad")[1]
    if not need_x and not need_adapters:
        raise ValueError("no gradient is asked for")
    dx = x.new_empty(x.shape) if need_x else None
    da, db = (lora_a.new_empty(lora_a.shape), lora_b.new_empty(lora_b.shape)) if need_adapters else (None, None)
    _call(lib().ts_adapter_project_backward, 1, x,
          code, n, per, d_in, d_out, r, adapters, x.data_ptr(), x_stride, _ptr(weight), w_stride, 0, 0, 0, lora_a.data_ptr(),
          lora_b.data_ptr(), adapter.data_ptr(), _ptr(scale), grad.data_ptr(), grad_stride, _ptr(dx), d_in, _ptr(da), _ptr(db))
    return dx, da, db
