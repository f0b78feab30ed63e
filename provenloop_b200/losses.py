"""Losses on next-token logits, for the training of adapters.

* ``token_logprobs`` / ``token_logprobs_backward`` -- log-probabilities of given
  tokens and their gradient: scoring, supervised training, and the old and
  reference log-probabilities of the two losses;
* ``policy_loss`` -- the clipped policy loss with a KL term;
* ``preference_loss`` -- the loss of pairs of a chosen and a rejected sequence.

Both losses give the gradient for the logits in the same call.  They take
CUDA tensors, run on torch's current stream of their device and return
without waiting; the workspace comes from torch's allocator, so calls may be
captured in CUDA graphs and run on several streams.  They record no autograd
history and refuse inputs that ask for it: call them under ``torch.no_grad()``
or in a ``torch.autograd.Function``.  ``adapters.adapter_project_backward`` takes
the gradient on to the adapters, ``adapters.clip_gradients`` clips theirs.

Logits are [..., vocab] (float32, bfloat16 or float16; rows may be strided), targets
their leading shape (int32 or int64): row i's target is the token that its
log-probability is taken of.  Next-token targets are shifted by the caller, with
the logits left whole (rows of ``logits[:, :-1]`` do not have one stride):
``targets = torch.nn.functional.pad(ids[:, 1:], (0, 1), value=-100)``.  A
target outside the vocabulary, such as -100, means that the row does not count: its
log-probability is 0 and its gradient zeros, whatever its logits are; it is not read.
Log-probabilities are float32.  Sums are held in 32 bits, what is computed
from a row's log-probability and sums over rows in 64; gradients are rounded once, and
probabilities below 2^-126 count as 0 in them.
A target whose logit is -inf has the log-probability -inf; a row with a NaN
or +inf has NaN.
"""
from __future__ import annotations

import struct

from . import adapters

_ARGS = struct.Struct("@2iPQIiPqPPIi4P2i6f5PqPQ")  # ts_loss_args, for callers of the C entry points
_REDUCTIONS = {"token": 0, "sequence": 1, "sum": 2}
_KINDS = {"sigmoid": 0, "hinge": 1, "squared": 2}


def _code(codes, value, name):
    if value not in codes:
        raise ValueError(f"{name} must be one of {', '.join(codes)}, not {value!r}")
    return codes[value]


def token_logprobs(logits, targets):
    """log softmax(logits)[target] for each row: float32, of targets' shape."""
    return (adapters._ops or adapters._load()).logprobs(logits, targets)


def token_logprobs_backward(grad, logits, targets, out=None):
    """Gradient for logits of ``token_logprobs``, given ``grad`` (float32, of targets'
    shape) for its result: grad ([v = target] - softmax(logits)[v]), in the
    logits' dtype.  ``out`` may be given, also ``logits`` itself.  Rows whose grad
    is 0 get zeros."""
    return (adapters._ops or adapters._load()).logprobs_backward(grad, logits, targets, out)


def policy_loss(logits, targets, old_logprobs, advantages, ref_logprobs=None, starts=None, clip=(0.2, 0.2), kl=0.0, reduction="token",
                grad_scale=None, need_grad=True, out=None):
    """(loss, logprobs, gradient for logits or None).

    With l a row's log-probability, rho = exp(l - old) and A its advantage, the
    row's loss is -min(rho A, clamp(rho, 1 - clip[0], 1 + clip[1]) A) + kl (exp(ref - l) - (ref - l) - 1).

    Sequences are the leading dimension of targets [sequences, tokens]; targets
    [n] are one sequence, or with ``starts`` (int32 [sequences + 1], ascending,
    on the device) packed ones: sequence s has the rows starts[s] to starts[s + 1];
    rows outside of them do not count.
    old_logprobs, ref_logprobs: float32 of targets' shape; old_logprobs None:
    rho is 1; ref_logprobs None: no KL term.  advantages: float32 of targets' shape or
    [sequences] (where both are the same, by row).  reduction: "token", the mean over all rows that count;
    "sequence", the mean over the sequences of their means (0 where no row counts);
    "sum".  grad_scale: a float32 tensor with one value, which multiplies the
    gradient (not the loss).  out: where the gradient goes, ``logits``
    itself included.  A ratio on a border of the clipping counts as not clipped."""
    low, high = clip
    return (adapters._ops or adapters._load()).policy(logits, targets, old_logprobs, advantages, ref_logprobs, starts, low, high, kl,
                                                      _code(_REDUCTIONS, reduction, "reduction"), grad_scale, need_grad, out)


def preference_loss(logits, targets, ref_logprobs=None, starts=None, beta=0.1, kind="sigmoid", smoothing=0.0, average=False,
                    grad_scale=None, need_grad=True, out=None):
    """(loss, margins, logprobs, gradient for logits or None).

    The sequences (as in ``policy_loss``) are the chosen ones and then as many
    rejected ones; sequence p and sequence pairs + p are a pair.  With D the sum
    over the chosen sequence's rows of l - ref, less that over the rejected one's
    (``average``: means in place of sums; 0 for a sequence without rows that
    count), and h = beta D the margin, a pair's loss is

    * "sigmoid": -(1 - smoothing) log sigmoid(h) - smoothing log sigmoid(-h),
    * "hinge": max(0, 1 - h),
    * "squared": (D - 1 / (2 beta))^2;

    the loss is the mean over the pairs.  margins: float32 [pairs].  ref_logprobs
    None: 0.  grad_scale, need_grad and out as in ``policy_loss``."""
    return (adapters._ops or adapters._load()).preference(logits, targets, ref_logprobs, starts, beta, _code(_KINDS, kind, "kind"), smoothing,
                                                          average, grad_scale, need_grad, out)
