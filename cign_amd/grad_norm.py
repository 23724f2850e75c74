"""The global norm of gradients, and clipping to it (cign_grad_norm,
cign_clip_grad_norm): two kernels for up to 128 tensors, two more for each
further 128. The reference's step does not clip
(generic_engine/train_cign.py:2103-2148).
"""
from __future__ import annotations

import torch

from ._rows import ROW_DTYPES, output_ops


def _listed(tensors, name: str) -> list:
    """The tensors as a list that is not empty; the first one checked here, where
    no device need be present, the others by the operators."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not tensors:
        raise ValueError(f"{name} must not be empty")
    t = tensors[0]
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in ROW_DTYPES:
        raise TypeError(f"{name} must be CUDA float32 or bfloat16 tensors")
    return tensors


def global_grad_norm(grads) -> torch.Tensor:
    """sqrt of the sum of all squares over the tensors (float32 and bfloat16, of
    any shapes and strides, on one device), a float32 scalar on their device:
    squares and sums in float64, in an order that depends on the sizes alone. Not
    differentiable."""
    grads = _listed(grads, "grads")
    return output_ops().global_grad_norm(grads)


def clip_grad_norm(grads, max_norm, out=None) -> torch.Tensor:
    """Multiplies the tensors by min(1, max_norm / (norm + 1e-6)), norm their
    global_grad_norm, which is returned: in place, or into the tensors `out` (of
    the gradients' shapes and types). The factor stays on the device: no
    synchronisation. A norm of NaN makes every gradient NaN, an infinite one makes
    finite values 0 and the others NaN: the returned norm tells.

    Tensors that are written must not share memory with each other or with
    another gradient (from the first to the last value of each); out[i] may be
    grads[i]. max_norm >= 0, taken as float32 (inf: no clipping)."""
    grads = _listed(grads, "grads")
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    if out is not None:
        out = [out] if isinstance(out, torch.Tensor) else list(out)
    return output_ops().clip_grad_norm(grads, max_norm, out)
