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
import functools
import struct

from ._lib import check, lib

_ARGS = struct.Struct("@2iP2Q4IPqPqPPqPPPPPqPqPPPQ")  # ts_adapter_args
_types = {}  # torch dtype -> TS_DTYPE_*


def _dtype_code(t):
    if not _types:
        import torch
        _types.update({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2})
    code = _types.get(t)
    if code is None:
        raise ValueError(f"dtype must be float32, bfloat16 or float16, not {t}")
    return code


def _rows(t, name):
    """(n, stride between rows) of t [..., d] seen as [n, d]."""
    if t.dim() < 2:
        raise ValueError(f"{name} must be [..., d] with at least two dimensions, not {tuple(t.shape)}")
    if t.dim() > 2:
        try:
            t = t.view(-1, t.shape[-1])
        except RuntimeError:
            raise ValueError(f"the leading dimensions of {name} do not form rows of one stride") from None
    if t.stride(1) != 1 and t.shape[1] > 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")
    return t.shape[0], t.stride(0)


def _same(t, name, dtype, device, shape):
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, not {t.dtype}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {shape}, not {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, x on {device}")


def _whole(t, name, dtype, device, shape):
    _same(t, name, dtype, device, shape)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _no_history(*tensors):
    import torch
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError("an input requires a gradient, which this call does not record: call it under "
                                 "torch.no_grad() and use adapter_project_backward")


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(packed: bytes, backward: int) -> int:
    v = C.c_uint64()
    check(lib().ts_adapter_workspace(packed, backward, C.byref(v)), "ts_adapter_workspace")
    return v.value


def _common(x, lora_a, lora_b, adapter, weight, scale):
    """Checks shared by both directions; (code, n, x stride, d_in, d_out, r, adapters, tokens per id, weight stride)."""
    import torch
    dtype, device = x.dtype, x.device
    code = _dtype_code(dtype)
    n, x_stride = _rows(x, "x")
    d_in = x.shape[-1]
    if lora_a.dim() != 3 or lora_b.dim() != 3:
        raise ValueError("lora_a must be [adapters, r, d_in] and lora_b [adapters, d_out, r]")
    adapters, r, _ = lora_a.shape
    d_out = lora_b.shape[1]
    _whole(lora_a, "lora_a", dtype, device, (adapters, r, d_in))
    _whole(lora_b, "lora_b", dtype, device, (adapters, d_out, r))
    lead, k = x.shape[:-1], adapter.dim()
    if k == 0 or adapter.shape != lead[:k]:
        raise ValueError(f"adapter must hold one index per leading entry of x {tuple(lead)}, not {tuple(adapter.shape)}")
    _whole(adapter, "adapter", torch.int32, device, tuple(lead[:k]))
    per = 1
    for s in lead[k:]:
        per *= s
    w_stride = 0
    if weight is not None:
        _same(weight, "weight", dtype, device, (d_out, d_in))
        if weight.stride(1) != 1 and d_in > 1:
            raise ValueError("the last dimension of weight must be contiguous")
        w_stride = weight.stride(0)
    if scale is not None:
        _whole(scale, "scale", torch.float32, device, (adapters,))
    return code, n, x_stride, d_in, d_out, r, adapters, max(per, 1), w_stride


def _call(entry, backward, device, fields):
    import torch
    if device.type != "cuda":
        raise ValueError("the tensors must be on a CUDA device: there is no CPU form")
    code, rest = fields[0], fields[1:]
    size = _workspace_bytes(_ARGS.pack(code, 0, 0, *rest, 0, 0), backward)
    ws = torch.empty(size, dtype=torch.uint8, device=device)
    index = device.index
    stream = torch.cuda.current_stream(index).cuda_stream
    check(entry(_ARGS.pack(code, index, stream, *rest, ws.data_ptr(), size)), entry.__name__)


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
    code, n, x_stride, d_in, d_out, r, adapters, per, w_stride = _common(x, lora_a, lora_b, adapter, weight, scale)
    _no_history(x, lora_a, lora_b, weight, bias, base, scale)
    dtype, device, shape = x.dtype, x.device, (*x.shape[:-1], d_out)
    if bias is not None:
        _whole(bias, "bias", dtype, device, (d_out,))
    base_stride = 0
    if base is not None:
        _same(base, "base", dtype, device, shape)
        base_stride = _rows(base, "base")[1]
    if out is None:
        out, out_stride = x.new_empty(shape), d_out
    else:
        _same(out, "out", dtype, device, shape)
        out_stride = _rows(out, "out")[1]
    _call(lib().ts_adapter_project, 0, device,
          (code, n, per, d_in, d_out, r, adapters, x.data_ptr(), x_stride, _ptr(weight), w_stride, _ptr(bias), _ptr(base),
           base_stride, lora_a.data_ptr(), lora_b.data_ptr(), adapter.data_ptr(), _ptr(scale), 0, 0, out.data_ptr(), out_stride,
           0, 0))
    return out


def adapter_project_backward(grad, x, lora_a, lora_b, adapter, weight=None, scale=None, need_x=True, need_adapters=True):
    """Gradients of ``adapter_project`` for ``grad`` = d loss / d out, weight,
    bias and scale held fixed: (d x [..., d_in], d lora_a, d lora_b), in the
    inputs' dtype, None where not needed.  An adapter without tokens gets
    zeros.  (The gradient of base is ``grad`` itself.)  The order of every sum
    depends on the sizes and indexes alone."""
    code, n, x_stride, d_in, d_out, r, adapters, per, w_stride = _common(x, lora_a, lora_b, adapter, weight, scale)
    _no_history(grad, x, lora_a, lora_b, weight, scale)
    _same(grad, "grad", x.dtype, x.device, (*x.shape[:-1], d_out))
    grad_stride = _rows(grad, "grad")[1]
    if not need_x and not need_adapters:
        raise ValueError("no gradient is asked for")
    dx = x.new_empty(x.shape) if need_x else None
    da, db = (lora_a.new_empty(lora_a.shape), lora_b.new_empty(lora_b.shape)) if need_adapters else (None, None)
    _call(lib().ts_adapter_project_backward, 1, x.device,
          (code, n, per, d_in, d_out, r, adapters, x.data_ptr(), x_stride, _ptr(weight), w_stride, 0, 0, 0, lora_a.data_ptr(),
           lora_b.data_ptr(), adapter.data_ptr(), _ptr(scale), grad.data_ptr(), grad_stride, _ptr(dx), d_in, _ptr(da), _ptr(db)))
    return dx, da, db
