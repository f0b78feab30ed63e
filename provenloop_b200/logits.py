"""Rules applied to next-token logits before a token is picked.

``apply_rules`` computes, in one pass over the logits, the penalties for
repeated tokens, the per-request biases and the grammar mask of a batch of
requests, and the greedy pick.  It takes CUDA tensors, runs on torch's current
stream of their device and returns without waiting.  The history, its lengths
and all parameters are read on the device, so that a captured decode step
that extends its own history replays with the new tokens.
"""
from __future__ import annotations

import struct

from ._lib import check, lib
from .adapters import _current_stream, _dtype_code, _load, _ptr

_ARGS = struct.Struct("@4iPQ4IPqPq5PPqPqPqPqP")  # ts_rules_args

MAX_HISTORY, MAX_BIASES = 1048575, 4095


def _per_row(t, name, dtype, n, device):
    if t.dtype is dtype and t.shape == (n,) and t.device == device and t.is_contiguous():
        return
    if t.dtype != dtype or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape ({n},)")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, logits on {device}")


def _table(t, name, dtypes, n, device, cols=None):
    """Stride between rows of t [n, cols], or 0 for one row [cols] for all."""
    shape = t.shape
    if len(shape) == 2 and shape[0] == n and t.dtype in dtypes and t.device == device and cols in (None, shape[1]):
        row, col = t.stride()
        if col == 1:
            return row
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be one of {[str(d) for d in dtypes]}, not {t.dtype}")
    if t.dim() not in (1, 2) or (t.dim() == 2 and t.shape[0] != n) or (cols is not None and t.shape[-1] != cols):
        raise ValueError(f"{name} must be [{n}, {'k' if cols is None else cols}] or one such row, not {tuple(t.shape)}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, logits on {device}")
    return t.stride(0) if t.dim() == 2 else 0


def apply_rules(logits, tokens=None, lengths=None, prompt_lengths=None, repetition=None, frequency=None, presence=None,
                bias_ids=None, bias_values=None, mask=None, out=None, write=True, pick=True):
    """(processed logits [n, vocab] or None, picks int64 [n] or None).

    Per row of ``logits`` [n, vocab] (float32, bfloat16 or float16; rows may
    be strided), in 32 bits and in this order:

    * ``tokens`` [n, k] (int32 or int64): the row's history, of which the first
      ``lengths[i]`` entries count (int32 [n]; default all) and the first
      ``prompt_lengths[i]`` are the prompt (default none); ids outside the
      vocabulary are skipped.  A token of the history has its logit divided by
      ``repetition[i]`` where it is positive and multiplied by it elsewhere;
      one that occurs c > 0 times behind the prompt then loses
      ``frequency[i] * c`` and ``presence[i]`` (float32 [n] each).
    * ``bias_ids`` / ``bias_values`` [n, m] or [m] (int32 or int64 / float32)
      are added; ids outside the vocabulary (padding) are skipped; of an id
      listed twice the last entry counts.
    * ``mask`` (int32 [n, ceil(vocab / 32)] or one row): a token whose bit
      ``v % 32`` of word ``v // 32`` is 0 becomes -inf, whatever it was.

    The result is rounded to ``out``'s type: ``out`` may be given (of the
    logits' dtype or float32; ``logits`` itself for in-place work) and is
    allocated in the logits' dtype otherwise; ``write=False`` leaves it out.
    The pick is the lowest id of the greatest unrounded value (a NaN counts as
    the greatest, as in ``torch.argmax``), -1 for a row that is -inf
    throughout.  At most 1048575 tokens and 4095 biases a row."""
    torch = _load()
    code, device = _dtype_code(logits.dtype), logits.device
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits must be [n, vocab] with contiguous rows")
    n, vocab = logits.shape
    if vocab == 0:
        raise ValueError("the vocabulary is empty")
    ints, ids64 = (torch.int64, torch.int32), 0
    cols = t_stride = 0
    if tokens is not None:
        if tokens.dim() != 2:
            raise ValueError("tokens must be [n, k]")
        t_stride = _table(tokens, "tokens", ints, n, device)
        cols = tokens.shape[1]
        ids64 = int(tokens.dtype == torch.int64)
        if cols > MAX_HISTORY:
            raise ValueError(f"the history is longer than {MAX_HISTORY}")
    for t, name, dt in ((lengths, "lengths", torch.int32), (prompt_lengths, "prompt_lengths", torch.int32),
                        (repetition, "repetition", torch.float32), (frequency, "frequency", torch.float32),
                        (presence, "presence", torch.float32)):
        if t is not None:
            if tokens is None:
                raise ValueError(f"{name} needs tokens")
            _per_row(t, name, dt, n, device)
    b_cols = bi_stride = bv_stride = 0
    if (bias_ids is None) != (bias_values is None):
        raise ValueError("bias_ids and bias_values come together")
    if bias_ids is not None:
        b_cols = bias_ids.shape[-1] if bias_ids.dim() else 0
        bi_stride = _table(bias_ids, "bias_ids", ints, n, device)
        bv_stride = _table(bias_values, "bias_values", (torch.float32,), n, device, b_cols)
        ids64 |= int(bias_ids.dtype == torch.int64) << 1
        if b_cols > MAX_BIASES:
            raise ValueError(f"more than {MAX_BIASES} biases in a row")
    m_stride = 0 if mask is None else _table(mask, "mask", (torch.int32,), n, device, (vocab + 31) // 32)
    if logits.requires_grad and torch.is_grad_enabled():
        raise ValueError("logits require a gradient, which this call does not record: call it under torch.no_grad()")
    if not write and out is not None:
        raise ValueError("out is given, but write is false")
    out_code, o_stride = code, 0
    if out is not None:
        if out.dtype not in (logits.dtype, torch.float32) or out.shape != logits.shape or out.device != device:
            raise ValueError(f"out must be {tuple(logits.shape)} on {device}, {logits.dtype} or float32")
        if vocab > 1 and out.stride(1) != 1:
            raise ValueError("the rows of out must be contiguous")
        out_code, o_stride = _dtype_code(out.dtype), out.stride(0)
    elif not write and not pick:
        raise ValueError("neither logits nor picks are asked for")
    if device.type != "cuda":
        raise ValueError("logits must be on a CUDA device: there is no CPU form")
    if write and out is None:
        out, o_stride = logits.new_empty((n, vocab)), vocab
    picks = torch.empty(n, dtype=torch.int64, device=device) if pick else None
    index = device.index
    rc = lib().ts_logit_rules(_ARGS.pack(
        code, out_code, index, ids64, _current_stream(index), n, vocab, cols, b_cols, 0, logits.data_ptr(),
        logits.stride(0), _ptr(tokens), t_stride, _ptr(lengths), _ptr(prompt_lengths), _ptr(repetition), _ptr(frequency),
        _ptr(presence), _ptr(bias_ids), bi_stride, _ptr(bias_values), bv_stride, _ptr(mask), m_stride, _ptr(out), o_stride,
        _ptr(picks)))
    if rc:
        check(rc, "ts_logit_rules")
    return out, picks
