"""Rules applied to next-token logits before a token is picked.

``apply_rules`` computes, in one pass over the logits, the penalties for
repeated tokens, the per-request biases and the grammar mask of a batch of
requests, and the greedy pick.  It takes CUDA tensors, runs on torch's current
stream of their device and returns without waiting.  The history, its lengths
and all parameters are read on the device, so that a captured decode step
that extends its own history replays with the new tokens.
``adapters.expired_waits`` tells whether a kernel has given up a wait.
"""
from __future__ import annotations

import struct

from . import adapters

_ARGS = struct.Struct("@4iPQ4IPqPq5PPqPqPqPqP")  # ts_rules_args, for callers of the C entry point


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
    return (adapters._ops or adapters._load()).rules(logits, tokens, lengths, prompt_lengths, repetition, frequency, presence, bias_ids,
                                                     bias_values, mask, out, write, pick)
