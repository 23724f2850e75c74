"""What the operators at the model's output (fused_block_ops.fused_layernorm,
class_logprobs, distill) share on the host: checks of rows, and _cign_ops.so
(csrc/python/output_ops.cpp), which holds their autograd nodes."""
from __future__ import annotations

import torch

from . import _lib

ROW_DTYPES = (torch.float32, torch.bfloat16)
_OPS = None


def output_ops():
    """The module of the autograd nodes. Raises RuntimeError if it or the
    library is not built, or if no HIP device is visible."""
    _lib.load_library()
    return _OPS or load_output_ops()


def load_output_ops():
    """The same without a device: the operators torch.ops.cign_amd.*, on meta
    tensors."""
    global _OPS
    if _OPS is None:
        _lib.load_library(require_gpu=False)
        try:
            from . import _cign_ops
        except ImportError as exc:
            raise RuntimeError(f"{_lib.LIB_PATH.with_name('_cign_ops.so')} is not built; run "
                               "`python -m cign_amd._build`") from exc
        _OPS = _cign_ops
    return _OPS


def check_rows(t, name: str, max_width: int) -> int:
    """TypeError / ValueError unless t is a float32 or bfloat16 GPU tensor
    whose last axis has 1 to max_width values; returns that width."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in ROW_DTYPES:
        raise TypeError(f"{name} must be CUDA float32 or bfloat16")
    if t.dim() < 1 or not (1 <= t.size(-1) <= max_width):
        raise ValueError(f"{name} must be [..., D] with 1<=D<={max_width}, got {tuple(t.shape)}")
    return int(t.size(-1))
