"""Tensors as rows of their last axis, for the operators at the model's output
(fused_block_ops.fused_layernorm, class_logprobs, distill): what they share in
checks, strides and devices."""
from __future__ import annotations

import contextlib

import torch
from torch.autograd.function import once_differentiable

ROW_DTYPES = (torch.float32, torch.bfloat16)
_HERE = contextlib.nullcontext()


def check_rows(t, name: str, max_width: int) -> int:
    """TypeError / ValueError unless t is a float32 or bfloat16 GPU tensor
    whose last axis has 1 to max_width values; returns that width."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in ROW_DTYPES:
        raise TypeError(f"{name} must be CUDA float32 or bfloat16")
    if t.dim() < 1 or not (1 <= t.size(-1) <= max_width):
        raise ValueError(f"{name} must be [..., D] with 1<=D<={max_width}, got {tuple(t.shape)}")
    return int(t.size(-1))


def as_rows(t: torch.Tensor):
    """(t as [rows, width] with values next to each other, elements from one
    row to the next). Copies only where the leading axes do not collapse to one
    or the last one is strided."""
    if t.dim() != 2:
        t = t.reshape(-1, t.size(-1))
    if t.stride(1) != 1 and t.size(1) > 1:
        t = t.contiguous()
    return t, t.stride(0)


def new_like(t: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of t's shape and type (empty_like takes half the
    time of empty)."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def once(backward):
    """once_differentiable of a backward, at the price of one look at the grad
    mode where no graph of the gradient is asked for."""
    slow = once_differentiable(backward)

    def run(ctx, *grads):
        return slow(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run


def on_device_of(t: torch.Tensor):
    """The context in which kernels are launched for t: its own device, where
    that is not the current one."""
    return _HERE if t.get_device() == torch.cuda.current_device() else torch.cuda.device(t.device)
