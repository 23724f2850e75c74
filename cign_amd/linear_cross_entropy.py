"""Cross entropy of a linear classifier over many classes, the logits never
stored, with the gradients of rows, weight and bias (cign_linear_xent_fwd /
cign_linear_xent_bwd).

The reference forms the logits with nn.Linear and takes torch's cross-entropy of
them (generic_engine/model_cign.py:1199, train_cign.py:2123): N x V values that
are kept for the backward, and their gradient beside them. Here a tile's logits
live in registers; what a training step holds over the classes is a piece of the
gradient at a time.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from ._rows import check_rows, output_ops
from .class_logprobs import MAX_CLASSES, check_index

MAX_WIDTH = 65536
MAX_ROWS = 1 << 23


class LinearCrossEntropy(NamedTuple):
    loss: torch.Tensor       # [...] float32
    logsumexp: torch.Tensor  # [...] float32


def linear_cross_entropy(x, weight, labels, bias=None, ignore_index=-100) -> LinearCrossEntropy:
    """For the logits z = x weight^T + bias of each row of x ([..., D], float32 or
    bfloat16, 1 <= D <= 65536, at most 2^23 rows; row-strided views are read in
    place), weight [V, D] of x's type, 1 <= V <= 1048576, bias [V] float32 or of
    x's type or None, labels [...] int64 or int32:

    - loss: logsumexp(z) - z[label]; 0, without gradient, where the label is
      ignore_index, NaN where it is another value outside [0, V) (its row of the
      gradient too, and with it the gradients of weight and bias);
    - logsumexp: log sum_v e^z of every row, differentiable (a penalty on it keeps
      the logits' scale).

    A bias of -inf masks its class, whatever its row of weight holds. A row
    without any class left has logsumexp -inf, loss inf and no gradient. Rows
    whose gradients are zero, an ignored label's among them, take no part in any
    gradient, whatever they hold.

    Products of bfloat16 are exact, of float32 within 2^-22; sums are float32;
    with bfloat16 rows the gradient of the logits is rounded to bfloat16 before
    its products with weight and rows. Gradients have their inputs' types and are
    once differentiable; the same call gives the same bits."""
    D = check_rows(x, "x", MAX_WIDTH)
    if x.numel() // D > MAX_ROWS:
        raise ValueError(f"x must have at most {MAX_ROWS} rows, got {tuple(x.shape)}")
    if not isinstance(weight, torch.Tensor) or weight.dtype != x.dtype:
        raise TypeError(f"weight must be a tensor of x's type ({x.dtype})")
    if weight.dim() != 2 or weight.size(1) != D or not (1 <= weight.size(0) <= MAX_CLASSES):
        raise ValueError(f"weight must be [V, {D}] with 1<=V<={MAX_CLASSES}, got {tuple(weight.shape)}")
    V = weight.size(0)
    if weight.device != x.device:
        raise ValueError(f"weight must be on {x.device}, got {weight.device}")
    if bias is not None:
        if not isinstance(bias, torch.Tensor) or bias.dtype not in (torch.float32, x.dtype):
            raise TypeError("bias must be a tensor, float32 or of x's type")
        if bias.shape != (V,):
            raise ValueError(f"bias must have shape [{V}], got {tuple(bias.shape)}")
        if bias.device != x.device:
            raise ValueError(f"bias must be on {x.device}, got {bias.device}")
    labels = check_index(labels, "labels", x.shape[:-1], x.device)
    return LinearCrossEntropy(*output_ops().linear_xent(x, weight, labels, bias, int(ignore_index)))
