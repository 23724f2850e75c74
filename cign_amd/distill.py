"""Distillation: the loss of a student's logits against a teacher's top
classes, and its gradient (cign_distill_topk_fwd / cign_distill_topk_bwd).

A teacher's distribution over many classes is kept as a short list a row, what
``class_logprobs(teacher_logits, top_k=K, temperature=T)`` returns as
top_logprobs and top_index; the student's logits are read once forward, and
once for their gradient. The reference has no counterpart: it trains on
labels alone (generic_engine/train_cign.py:2123).
"""
from __future__ import annotations

import torch

from ._rows import check_rows, output_ops
from .class_logprobs import MAX_CLASSES, check_index, check_temperature

MAX_LIST = 128


def distill_topk_loss(logits, teacher_logprobs, teacher_index, temperature=1.0, tail=False) -> torch.Tensor:
    """temperature^2 KL(p || q) of each row ([...] float32): q = softmax(logits
    / temperature) over the V classes of logits ([..., V], float32 or bfloat16,
    1 <= V <= 1048576; row-strided views are read in place), p the teacher's
    list: teacher_index ([..., K], int64 or int32, 1 <= K <= 128) and
    teacher_logprobs ([..., K], float32 or bfloat16), the teacher's log
    probabilities of those classes at the same temperature.

    tail False: p is the list renormalised, so any constant may be added to a
    row of teacher_logprobs (logits divided by the temperature do). tail True:
    the list holds sum e^teacher_logprobs of the teacher's mass, and what is
    left of one is a further class, against the mass the student leaves
    outside the list; nothing is left where the list names every class.

    A negative index marks an empty place, whose teacher_logprobs is not
    looked at. A row without a listed class has loss 0 and no gradient; an
    index of V or more makes its row's loss and gradient NaN. The divergence is
    summed over places, p_i (log p_i - log q of the place's class): a class named
    twice counts with both masses, place by place, which is less than the KL of
    its joined mass P by the sum of p_i log(P / p_i) over its places (the loss may
    be negative then) and has the same gradient. The loss's gradient is that of
    the logits (their type, once differentiable); the teacher's tensors are
    constants."""
    check_rows(logits, "logits", MAX_CLASSES)
    if not isinstance(teacher_logprobs, torch.Tensor) or teacher_logprobs.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError("teacher_logprobs must be a float32 or bfloat16 tensor")
    K = teacher_logprobs.size(-1) if teacher_logprobs.dim() else 0
    if teacher_logprobs.shape[:-1] != logits.shape[:-1] or not (1 <= K <= MAX_LIST):
        raise ValueError(f"teacher_logprobs must be {(*logits.shape[:-1], 'K')} with 1<=K<={MAX_LIST}, got "
                         f"{tuple(teacher_logprobs.shape)}")
    if teacher_logprobs.device != logits.device:
        raise ValueError(f"teacher_logprobs must be on {logits.device}, got {teacher_logprobs.device}")
    if torch.is_grad_enabled() and teacher_logprobs.requires_grad:
        raise ValueError("teacher_logprobs is a constant of the loss: detach it")
    teacher_index = check_index(teacher_index, "teacher_index", teacher_logprobs.shape, logits.device)
    temperature = check_temperature(temperature)
    if teacher_logprobs.dtype != torch.float32:
        teacher_logprobs = teacher_logprobs.to(torch.float32)
    return output_ops().distill_topk(logits, teacher_logprobs.contiguous(), teacher_index, temperature, bool(tail))
