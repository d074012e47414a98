"""A student from a teacher: the teacher's top logits, and the loss against them, on the HIP kernels.

``top_logits`` keeps the k largest logits of every row with their ids; ``distillation_loss`` is the divergence of a student's
distribution from the teacher's over those, with the gradient of the student's logits.  ``CDSSMLMHeadModel.top_logits`` and
``CDSSMLMHeadModel.distill_loss`` put them behind the model.  (The reference trains on labels alone, trainer.py:228-247.)
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib

Tensor = torch.Tensor

MAX_TOP = 128     # of top_logits
MAX_LIST = 256    # entries of a teacher's list

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}

_nodes = None


def _native():
    """The host side and the autograd node (csrc/compress_nodes.cpp), working on the loaded library."""
    global _nodes
    if _nodes is None:
        _nodes = _lib.native("compress_nodes")
    return _nodes


def _check_logits(op: str, logits: Tensor) -> None:
    if not logits.is_cuda:
        raise RuntimeError(f"{op} runs on the GPU only")
    if logits.dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"{op}: logits must be float32 or bfloat16, got {logits.dtype}")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{op}: logits must be (..., V) with V >= 1, got {tuple(logits.shape)}")


def top_logits(logits: Tensor, k: int) -> tuple:
    """The k largest of logits (..., V) fp32 or bf16 in each row, largest first, and their ids: (values (..., k) in
    logits' dtype, ids (..., k) int64), 1 <= k <= min(V, 128).

    Of equal logits the lowest id comes first; -0 equals 0, and NaN counts as the largest.  Without a gradient: refused
    where one would be followed."""
    _check_logits("top_logits", logits)
    if not 1 <= k <= min(MAX_TOP, logits.shape[-1]):
        raise ValueError(f"top_logits: k must be within 1 .. min(V, {MAX_TOP}), got {k} for V {logits.shape[-1]}")
    return _native().top_logits(logits, k)


def _check_loss(logits: Tensor, teacher_logits: Tensor, teacher_ids: Tensor, temperature: float, reduction: str) -> int:
    op = "distillation_loss"
    _check_logits(op, logits)
    if not teacher_logits.is_cuda or teacher_logits.device != logits.device or teacher_ids.device != logits.device:
        raise RuntimeError(f"{op}: logits are on {logits.device}, teacher_logits on {teacher_logits.device}, teacher_ids on "
                           f"{teacher_ids.device}")
    if teacher_logits.dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"{op}: teacher_logits must be float32 or bfloat16, got {teacher_logits.dtype}")
    if teacher_ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{op}: teacher_ids must be int64 or int32, got {teacher_ids.dtype}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"{op}: reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}")
    if not 1e-4 <= temperature <= 1e4:
        raise ValueError(f"{op}: temperature must be within 1e-4 .. 1e4, got {temperature}")
    if teacher_logits.shape != teacher_ids.shape or teacher_logits.dim() != logits.dim() \
            or teacher_logits.shape[:-1] != logits.shape[:-1] or not 1 <= teacher_logits.shape[-1] <= MAX_LIST:
        raise ValueError(f"{op}: teacher_logits and teacher_ids must be (*logits.shape[:-1], K) with K of 1 .. {MAX_LIST}, "
                         f"got {tuple(teacher_logits.shape)} and {tuple(teacher_ids.shape)} for {tuple(logits.shape)}")
    return _REDUCTIONS[reduction]


def distillation_loss(logits: Tensor, teacher_logits: Tensor, teacher_ids: Tensor, temperature: float = 1.0,
                      reduction: str = "mean") -> Tensor:
    """t^2 KL(p || q) of a student's logits (..., V) against a teacher's top logits (..., K) and their ids (..., K):
    p = softmax(teacher_logits / t) over the K entries, q = softmax(logits / t) over all V words, t the temperature
    (1e-4 .. 1e4; t^2 keeps the gradients' size).

    logits and teacher_logits fp32 or bf16 (each its own), ids int64 or int32, 1 <= K <= 256; fp32 loss: a number for
    ``reduction`` "mean" (over the tokens that take part; NaN if there is none) or "sum", (...) for "none".
    Differentiable in logits, once; teacher_logits must not ask for a gradient.

    An entry whose teacher logit is -inf takes no part, whatever its id: lists may be shorter than K.  A token without any
    other entry takes no part either, whatever its logits hold: its loss and its gradient are 0.  A word listed twice counts
    with the sum of its probabilities.  An id outside [0, V) makes its token's loss and gradient NaN; nothing outside the
    logits is read.  A word of student logit -inf has probability 0 (the loss is infinite if the teacher gives it one that
    fp32 holds); a token whose logits are all -inf, or hold +inf or NaN, has NaN, and so has one whose teacher's do."""
    return _native().distill(logits, teacher_logits, teacher_ids, temperature,
                             _check_loss(logits, teacher_logits, teacher_ids, temperature, reduction))


def distillation_loss_fwd(logits: Tensor, teacher_logits: Tensor, teacher_ids: Tensor, temperature: float = 1.0,
                          reduction: str = "mean") -> tuple:
    """The loss as ``distillation_loss`` returns it, without autograd, and the workspace that ``distillation_loss_bwd`` reads."""
    return _native().distill_fwd(logits, teacher_logits, teacher_ids, temperature,
                                 _check_loss(logits, teacher_logits, teacher_ids, temperature, reduction))


def distillation_loss_bwd(grad: Tensor, logits: Tensor, teacher_logits: Tensor, teacher_ids: Tensor,
                          workspace: Optional[Tensor], temperature: float = 1.0, reduction: str = "mean") -> Tensor:
    """The gradient of logits, in their dtype, from the gradient of the loss, the forward's arguments and its workspace."""
    return _native().distill_bwd(grad, logits, teacher_logits, teacher_ids, workspace, temperature,
                                 _check_loss(logits, teacher_logits, teacher_ids, temperature, reduction))
