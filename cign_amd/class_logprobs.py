"""What a row of logits says, in one pass over it: the log probability of a
given class, the entropy and the top classes, with the gradient of the first
two (cign_class_logprobs_fwd / cign_class_logprobs_bwd).

The reference takes these from torch, one pass each: cross-entropy over
logits gathered by the train mask (generic_engine/train_cign.py:2123), argmax
and softmax for its metrics (:1774-1817). Here a training loss is
``-class_logprobs(logits, labels).logprob`` over labels whose rows outside the
mask are ``ignore_index``, without gathering logits, and an evaluation reads
prediction, confidence and uncertainty from one call.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from ._rows import check_rows, output_ops

MAX_CLASSES = 1 << 20
MAX_TOP_K = 128


class ClassLogprobs(NamedTuple):
    logprob: Optional[torch.Tensor]       # [...] float32; None without labels
    entropy: torch.Tensor                 # [...] float32, in nats
    top_logprobs: Optional[torch.Tensor]  # [..., top_k] float32, falling; None without top_k
    top_index: Optional[torch.Tensor]     # [..., top_k] int64


def check_temperature(temperature) -> float:
    t = float(temperature)
    # the kernels take 1 / T in float32
    if not (1e-30 < t < 1e30):
        raise ValueError(f"temperature must be between 1e-30 and 1e30, got {temperature}")
    return t


def check_index(t, name: str, shape, device) -> torch.Tensor:
    """t as contiguous int64 of this shape on this device."""
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{name} must be an int64 or int32 tensor")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    return (t if t.dtype == torch.int64 else t.to(torch.int64)).contiguous()


def class_logprobs(logits, labels=None, top_k=0, temperature=1.0, ignore_index=-100) -> ClassLogprobs:
    """For each row of logits ([..., V], float32 or bfloat16, 1 <= V <=
    1048576; row-strided views are read in place), with l = logits /
    temperature (between 1e-30 and 1e30) and log p = l - logsumexp(l):

    - logprob: log p of labels ([...], int64 or int32); 0, without gradient,
      where the label is ignore_index, NaN where it is another value outside
      [0, V) (its row of the gradient too);
    - entropy: -sum p log p;
    - top_logprobs, top_index: the top_k (0 to 128, at most V) most likely
      classes, the lowest index first among equal logits; a NaN logit ranks as
      -inf. Not differentiable.

    A logit of -inf masks its class. A row without any class left has logprob
    -inf, entropy 0, no gradient, and its lowest indices as top classes. Sums
    are float32; the gradient has the logits' type and is once
    differentiable."""
    V = check_rows(logits, "logits", MAX_CLASSES)
    top_k = int(top_k)
    if not (0 <= top_k <= min(V, MAX_TOP_K)):
        raise ValueError(f"top_k must be in [0, min(V, {MAX_TOP_K})], got {top_k} for V = {V}")
    temperature = check_temperature(temperature)
    if labels is not None:
        labels = check_index(labels, "labels", logits.shape[:-1], logits.device)
    return ClassLogprobs(*output_ops().class_logprobs(logits, labels, top_k, temperature, int(ignore_index)))
