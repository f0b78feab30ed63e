"""Plaintext low-rank adapters of many requests at once.

The plaintext branch of ``_he_lora_delta`` (demonstrator/server/
inference_engine.py:1234-1242), for any number of tokens, each with its own
adapter or none, beside the projection that the adapters belong to:

* ``adapter_project`` -- ``y = x W^T + bias + scale_e (x A_e^T) B_e^T``, or the
  same delta added to a projection that has been computed already;
* ``adapter_project_backward`` -- the gradients for x and for the adapters
  (the projection is frozen), with which adapters are trained;
* ``clip_gradients`` -- the norm of an adapter's gradients over all tensors,
  for each adapter of a stack, and their clipping;
* ``expired_waits`` -- whether a kernel has given up.

The first three take CUDA tensors, run on torch's current stream of their device and
return without waiting; the workspace comes from torch's allocator, so calls
may be captured in CUDA graphs and run on several streams.  They do not
record autograd history and refuse inputs that ask for it: call them under
``torch.no_grad()``, or from the two halves of a ``torch.autograd.Function``.
"""
from __future__ import annotations

import ctypes as C
import os
import struct

from . import build
from ._lib import HERE, check, lib

_ARGS = struct.Struct("@2iP2Q4IPqPqPPqPPPPPqPqPPPQ")  # ts_adapter_args, for callers of the C entry points
_CLIP_ARGS = struct.Struct("@iIPQPPfiPPQ")  # ts_clip_args
_CLIP_TENSOR = struct.Struct("@PPQ2i")  # ts_clip_tensor
_ops = None


def _load():
    """The compiled checks (csrc/torch_ops.cpp), bound to the library that ``_lib`` loads."""
    global _ops
    if _ops is None:
        import torch  # noqa: F401  (its libraries have to be there first)
        path = os.path.join(HERE, "_torch_ops.so")
        if not os.path.exists(path):
            raise ImportError(f"{path} not found; build it with `python -m provenloop_b200.build`")
        if not build.torch_ops_fits():
            raise ImportError(f"{path} was not built for {build.torch_tag()}; build it with `python -m provenloop_b200.build`")
        from . import _torch_ops
        L = lib()
        entries = (L.ts_adapter_workspace, L.ts_adapter_project, L.ts_adapter_project_backward, L.ts_logit_rules, L.ts_loss_workspace,
                   L.ts_token_logprobs, L.ts_token_logprobs_backward, L.ts_policy_loss, L.ts_preference_loss, L.ts_clip_workspace,
                   L.ts_clip_gradients)
        _torch_ops.bind(*(C.cast(f, C.c_void_p).value for f in entries), check)
        _ops = _torch_ops
    return _ops


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
    return (_ops or _load()).project(x, lora_a, lora_b, adapter, weight, bias, base, scale, out)


def adapter_project_backward(grad, x, lora_a, lora_b, adapter, weight=None, scale=None, need_x=True, need_adapters=True):
    """Gradients of ``adapter_project`` for ``grad`` = d loss / d out, weight,
    bias and scale held fixed: (d x [..., d_in], d lora_a, d lora_b), in the
    inputs' dtype, None where not needed.  An adapter without tokens gets
    zeros.  (The gradient of base is ``grad`` itself.)  The order of every sum
    depends on the sizes, the indexes and the kind of GPU alone."""
    return (_ops or _load()).backward(grad, x, lora_a, lora_b, adapter, weight, scale, need_x, need_adapters)


def clip_gradients(grads, max_norm, adapters=None, out=None):
    """Scales gradients so that their norm is at most ``max_norm``, in place
    or to ``out``; returns the norm from before.

    grads: a list of CUDA tensors of any shapes (float32, bfloat16, float16, also
    mixed; dense in memory), None entries are skipped.  The norm is the root of
    the sum of all their squares: a 0-dim float32 tensor.  With ``adapters``
    given, every tensor is a stack [adapters, ...] (contiguous), as
    ``adapter_project_backward`` returns them, and each adapter has a norm over its part of
    all tensors and is clipped by itself: float32 [adapters].  max_norm: a
    number, or a float32 tensor with one value or one for each adapter, which is
    read on the device.  out: a list of tensors like grads, each of its gradient's
    dtype or float32; gradients that are only read may occur twice and then count twice.

    Values are multiplied in 32 bits by min(1, max_norm / norm) and rounded
    once.  What has a norm that is not finite is left as it is (or copied to ``out``): look
    at the norm before the step.  The order of the sums depends on the sizes alone."""
    return (_ops or _load()).clip(grads, max_norm, adapters, out)


def expired_waits(device=None) -> int:
    """How many waits inside kernels of this module, ``logits`` and ``losses`` have run
    out (after two seconds) on ``device`` (default: the current one) since the
    library was loaded.  Anything but 0 means that a kernel or the device is
    broken and that some call's results are incomplete: the calls themselves do
    not wait and cannot say so.  Waits for the device."""
    import torch
    d = torch.device("cuda", device) if isinstance(device, int) else torch.device("cuda" if device is None else device)
    if d.type != "cuda":
        raise ValueError(f"{d} is not a CUDA device")
    v = C.c_uint64()
    check(lib().ts_expired_waits(torch.cuda.current_device() if d.index is None else d.index, C.byref(v)), "ts_expired_waits")
    return v.value
