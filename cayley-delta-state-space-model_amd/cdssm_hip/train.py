"""The two ends of a training step around the model's blocks, on the HIP kernels.

``token_embedding`` turns token ids into hidden states and sums the table's gradient by sorted tokens;
``linear_cross_entropy`` turns hidden states into the loss of the (tied) head without keeping the logits, with the
gradients of both operands; ``global_grad_norm`` / ``clip_grads`` / ``clip_grad_norm_`` bound the gradients before the
optimizer (the reference's trainer.py:228-247 with model.py:37-51, where torch's embedding, linear, cross_entropy and
clip_grad_norm_ do it).  ``CDSSMLMHeadModel.loss`` puts the first two around the blocks.
"""

from __future__ import annotations

import math
from typing import Iterable, Optional, Sequence, Union

import torch

from . import _lib

Tensor = torch.Tensor

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}
_INDEX = (torch.int64, torch.int32)

_nodes = None


def _native():
    """The host side and the autograd nodes (csrc/train_nodes.cpp), working on the loaded library."""
    global _nodes
    if _nodes is None:
        _nodes = _lib.native("train_nodes")
    return _nodes


def _check_float(op: str, name: str, t: Tensor) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{op} runs on the GPU only")
    if t.dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"{op}: {name} must be float32 or bfloat16, got {t.dtype}")


def _check_index(op: str, name: str, t: Tensor, device: torch.device) -> None:
    if t.dtype not in _INDEX:
        raise TypeError(f"{op}: {name} must be int64 or int32, got {t.dtype}")
    if t.device != device:
        raise RuntimeError(f"{op}: {name} is on {t.device}, the other tensors on {device}")


# ---------------------------------------------------------------------------------------------------------
# embedding
# ---------------------------------------------------------------------------------------------------------

def _check_embedding(ids: Tensor, weight: Tensor) -> None:
    op = "token_embedding"
    _check_float(op, "weight", weight)
    _check_index(op, "ids", ids, weight.device)
    if weight.dim() != 2 or 0 in weight.shape:
        raise ValueError(f"{op}: weight must be (V, C) with V, C >= 1, got {tuple(weight.shape)}")


def token_embedding_fwd(ids: Tensor, weight: Tensor, scale: float = 1.0) -> Tensor:
    """scale * weight[ids] (..., C) in weight's dtype (cdssm_token_embedding_fwd)."""
    _check_embedding(ids, weight)
    return _native().embedding_fwd(ids, weight, scale)


def token_embedding_bwd(grad: Tensor, ids: Tensor, num_rows: int, scale: float = 1.0,
                        padding_idx: Optional[int] = None) -> Tensor:
    """The table's gradient (num_rows, C) in grad's dtype from grad (..., C): every row the fp32 sum of its tokens'
    gradients in the tokens' order, rounded once; rows without a token, and the padding row, zero
    (cdssm_token_embedding_bwd)."""
    op = "token_embedding"
    _check_float(op, "grad", grad)
    _check_index(op, "ids", ids, grad.device)
    if grad.shape[:-1] != ids.shape or grad.dim() < 1 or num_rows < 1:
        raise ValueError(f"{op}: grad must be (*ids.shape, C), got {tuple(grad.shape)} for ids {tuple(ids.shape)}")
    return _native().embedding_bwd(grad, ids, num_rows, scale, _padding(op, padding_idx, num_rows))


def _padding(op: str, padding_idx: Optional[int], rows: int) -> int:
    """The row without a gradient, -1 for none."""
    if padding_idx is None:
        return -1
    if not -rows <= padding_idx < rows:
        raise ValueError(f"{op}: padding_idx must be within the {rows} rows, got {padding_idx}")
    return padding_idx % rows


def token_embedding(ids: Tensor, weight: Tensor, scale: float = 1.0, padding_idx: Optional[int] = None) -> Tensor:
    """scale * weight[ids]: ids (...) int64 or int32, weight (V, C) fp32 or bf16 -> (..., C).

    Differentiable in ``weight`` (``token_embedding_bwd``: deterministic).  ``padding_idx`` (negative: from the end)
    names a row that takes no gradient.  An id outside [0, V) gives a row of NaN and no gradient; nothing outside the
    table is read."""
    _check_embedding(ids, weight)
    padding = _padding("token_embedding", padding_idx, weight.shape[0])
    return _native().embedding(weight, ids, scale, padding)


# ---------------------------------------------------------------------------------------------------------
# the head's loss
# ---------------------------------------------------------------------------------------------------------

def _check_loss(x: Tensor, weight: Tensor, labels: Tensor, reduction: str) -> int:
    op = "linear_cross_entropy"
    _check_float(op, "x", x)
    _check_float(op, "weight", weight)
    if x.dtype != weight.dtype or x.device != weight.device:
        raise TypeError(f"{op}: x and weight must share dtype and device, got {x.dtype} on {x.device} and "
                        f"{weight.dtype} on {weight.device}")
    _check_index(op, "labels", labels, x.device)
    if reduction not in _REDUCTIONS:
        raise ValueError(f"{op}: reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}")
    if weight.dim() != 2 or x.dim() < 1 or 0 in weight.shape or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"{op}: x must be (..., d) and weight (V, d), got {tuple(x.shape)} and {tuple(weight.shape)}")
    if labels.shape != x.shape[:-1]:
        raise ValueError(f"{op}: labels must be {tuple(x.shape[:-1])}, got {tuple(labels.shape)}")
    return _REDUCTIONS[reduction]


def linear_cross_entropy_fwd(x: Tensor, weight: Tensor, labels: Tensor, ignore_index: int = -100,
                             reduction: str = "mean") -> tuple:
    """The loss as ``linear_cross_entropy`` returns it, and the workspace that ``linear_cross_entropy_bwd`` reads."""
    return _native().loss_fwd(x, weight, labels, ignore_index, _check_loss(x, weight, labels, reduction))


def linear_cross_entropy_bwd(grad: Tensor, weight: Tensor, workspace: Optional[Tensor], x_shape: Sequence[int],
                             reduction: str = "mean", need_x: bool = True, need_weight: bool = True) -> tuple:
    """(dx, dW) in weight's dtype from the gradient of the loss and the workspace of the forward over x of that shape, the
    same weight and reduction; None in the place of one that is not needed."""
    op = "linear_cross_entropy_bwd"
    _check_float(op, "weight", weight)
    if reduction not in _REDUCTIONS:
        raise ValueError(f"{op}: reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}")
    if weight.dim() != 2 or len(x_shape) < 1 or x_shape[-1] != weight.shape[1] or grad.device != weight.device \
            or grad.numel() != (math.prod(x_shape[:-1]) if reduction == "none" else 1):
        raise ValueError(f"{op}: the gradient of a {reduction} over x {tuple(x_shape)} and weight {tuple(weight.shape)} on "
                         f"{weight.device}, got {tuple(grad.shape)} on {grad.device}")
    return _native().loss_bwd(grad, weight, workspace, x_shape, _REDUCTIONS[reduction], need_x, need_weight)


def linear_cross_entropy(x: Tensor, weight: Tensor, labels: Tensor, ignore_index: int = -100,
                         reduction: str = "mean") -> Tensor:
    """Softmax cross entropy of the logits x @ weight^T against ``labels``, the logits never stored.

    x (..., d) and weight (V, d) fp32 or bf16, labels (...) int64 or int32; fp32 loss: a number for ``reduction``
    "mean" (over the labels that are not ``ignore_index``; NaN if there is none) or "sum", (...) for "none" (0 where
    ignored).  Differentiable in x and weight.  Rows whose label is ``ignore_index`` take no part, whatever they hold: their
    gradient is 0.  Any other label outside [0, V) makes its row's loss, and the gradients, NaN.  A logit over an infinite
    operand is what the products give (-inf: a word of probability 0) in bf16, and NaN in fp32, whose parts of a number may be
    0 where it is not.  fp32 operands are taken to 2^-24 of themselves, but not below 2^-126: smaller parts count as 0."""
    return _native().loss(x, weight, labels, ignore_index, _check_loss(x, weight, labels, reduction))


# ---------------------------------------------------------------------------------------------------------
# gradient norm and clipping
# ---------------------------------------------------------------------------------------------------------

def _list(ts: Union[Tensor, Iterable[Tensor]]) -> list:
    return [ts] if torch.is_tensor(ts) else list(ts)


def global_grad_norm(grads: Union[Tensor, Iterable[Tensor]]) -> Tensor:
    """The 2-norm over all elements of the given tensors (fp32 and bf16 may be mixed), as one fp32 number on their
    device: squares added in fp64, the same bits every time."""
    return _native().global_norm(_list(grads))


def clip_grads(grads: Union[Tensor, Iterable[Tensor]], max_norm: float,
               out: Optional[Sequence[Tensor]] = None) -> Tensor:
    """Scales the given tensors by min(1, max_norm / (norm + 1e-6)), norm the 2-norm over all of them, which it returns
    (one fp32 number on their device; nothing waits for it).  In place, or into ``out``: as many tensors of the same
    sizes, fp32 or bf16 (fp32 copies of bf16 gradients for an optimizer that keeps fp32 weights, rounded nowhere).
    A tensor may be given once, and must not share memory with another; a norm that is infinite or NaN scales as
    torch's clip_grad_norm_ does."""
    return _native().clip(_list(grads), max_norm, None if out is None else _list(out))


def clip_grad_norm_(parameters: Union[Tensor, Iterable[Tensor]], max_norm: float) -> Tensor:
    """``clip_grads`` of the parameters' gradients, in place (trainer.py:242-243); parameters without a gradient are
    left out."""
    return _native().clip_parameters(_list(parameters), max_norm)
