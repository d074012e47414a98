"""The two ends of a training step around the model's blocks, on the HIP kernels.

``token_embedding`` turns token ids into hidden states and sums the table's gradient by sorted tokens;
``linear_cross_entropy`` turns hidden states into the loss of the (tied) head without keeping the logits, with the
gradients of both operands; ``global_grad_norm`` / ``clip_grads`` / ``clip_grad_norm_`` bound the gradients before the
optimizer (the reference's trainer.py:228-247 with model.py:37-51, where torch's embedding, linear, cross_entropy and
clip_grad_norm_ do it).  ``CDSSMLMHeadModel.loss`` puts the first two around the blocks.
"""

from __future__ import annotations

import array
import math
import operator
from typing import Iterable, Optional, Sequence, Union

import torch

from . import _lib

Tensor = torch.Tensor

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}
_DTYPES = frozenset(_lib.DTYPE_CODE)
_INDEX_BYTES = {torch.int64: 8, torch.int32: 4}


def _call(name: str, device: torch.device, *args) -> None:
    """Entry point ``name`` on ``device``'s current stream, with that device as the current one."""
    fn = getattr(_lib.load(), name)
    if device.index == torch.cuda.current_device():
        st = fn(*args, _lib.stream_of(device))
    else:
        with torch.cuda.device(device):
            st = fn(*args, _lib.stream_of(device))
    if st != 0:
        _lib.check(st, name)


def _check_float(op: str, name: str, t: Tensor) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{op} runs on the GPU only")
    if t.dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"{op}: {name} must be float32 or bfloat16, got {t.dtype}")


def _check_index(op: str, name: str, t: Tensor, device: torch.device) -> None:
    if t.dtype not in _INDEX_BYTES:
        raise TypeError(f"{op}: {name} must be int64 or int32, got {t.dtype}")
    if t.device != device:
        raise RuntimeError(f"{op}: {name} is on {t.device}, the other tensors on {device}")


def _row_stride(t: Tensor) -> int:
    """Row stride of a (rows, columns) tensor with dense columns; any row stride will do for a single row."""
    return max(t.stride(0), t.shape[1]) if t.shape[0] == 1 else t.stride(0)


def _rows(t: Tensor) -> Tensor:
    """t (..., C) as (rows, C) with dense columns and a row stride of at least C, copied only where it has to be."""
    r = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
    if r.is_contiguous():
        return r
    ok = (r.shape[1] == 1 or r.stride(1) == 1) and (r.shape[0] <= 1 or r.stride(0) >= r.shape[1])
    return r if ok else r.contiguous()


# ---------------------------------------------------------------------------------------------------------
# embedding
# ---------------------------------------------------------------------------------------------------------

def token_embedding_fwd(ids: Tensor, weight: Tensor, scale: float = 1.0) -> Tensor:
    """scale * weight[ids] (..., C) in weight's dtype (cdssm_token_embedding_fwd)."""
    op = "token_embedding"
    _check_float(op, "weight", weight)
    _check_index(op, "ids", ids, weight.device)
    if weight.dim() != 2 or 0 in weight.shape:
        raise ValueError(f"{op}: weight must be (V, C) with V, C >= 1, got {tuple(weight.shape)}")
    w, i = _rows(weight.detach()), ids.contiguous()
    V, C = w.shape
    y = torch.empty(*ids.shape, C, dtype=w.dtype, device=w.device)
    n = i.numel()
    if n:
        _call("cdssm_token_embedding_fwd", w.device, _lib.DTYPE_CODE[w.dtype], _INDEX_BYTES[i.dtype], i.data_ptr(),
              w.data_ptr(), _row_stride(w), scale, y.data_ptr(), n, V, C)
    return y


def token_embedding_bwd(grad: Tensor, ids: Tensor, num_rows: int, scale: float = 1.0,
                        padding_idx: Optional[int] = None) -> Tensor:
    """The table's gradient (num_rows, C) in grad's dtype from grad (..., C): every row the fp32 sum of its tokens'
    gradients in the tokens' order, rounded once; rows without a token, and the padding row, zero
    (cdssm_token_embedding_bwd)."""
    op = "token_embedding"
    _check_float(op, "grad", grad)
    _check_index(op, "ids", ids, grad.device)
    if grad.shape[:-1] != ids.shape or num_rows < 1:
        raise ValueError(f"{op}: grad must be (*ids.shape, C), got {tuple(grad.shape)} for ids {tuple(ids.shape)}")
    return _table_gradient(grad, ids, num_rows, scale, _padding(op, padding_idx, num_rows))


def _table_gradient(grad: Tensor, ids: Tensor, rows: int, scale: float, padding_idx: int) -> Tensor:
    g, i = _rows(grad), ids.contiguous()
    T, C = g.shape
    device = g.device
    if T == 0:
        return torch.zeros(rows, C, dtype=g.dtype, device=device)
    dw = torch.empty(rows, C, dtype=g.dtype, device=device)
    nb = _lib.load().cdssm_token_embedding_bwd_workspace_bytes(T, rows, C)
    if nb < 0:
        raise ValueError(f"token_embedding: {_lib.last_error()}")
    ws = torch.empty(nb, dtype=torch.uint8, device=device)
    _call("cdssm_token_embedding_bwd", device, _lib.DTYPE_CODE[g.dtype], _INDEX_BYTES[i.dtype], i.data_ptr(), g.data_ptr(),
          _row_stride(g), scale, padding_idx, dw.data_ptr(), ws.data_ptr(), T, rows, C)
    return dw


def _padding(op: str, padding_idx: Optional[int], rows: int) -> int:
    """The row without a gradient, -1 for none."""
    if padding_idx is None:
        return -1
    if not -rows <= padding_idx < rows:
        raise ValueError(f"{op}: padding_idx must be within the {rows} rows, got {padding_idx}")
    return padding_idx % rows


class TokenEmbeddingFn(torch.autograd.Function):
    """``token_embedding`` as an autograd node: (weight, ids, scale, padding_idx as ``_padding`` gives it) -> rows."""

    @staticmethod
    def forward(ctx, weight, ids, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.meta = (weight.shape[0], scale, padding_idx)
        return token_embedding_fwd(ids, weight, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        (ids,) = ctx.saved_tensors
        return _table_gradient(grad, ids, *ctx.meta), None, None, None


def token_embedding(ids: Tensor, weight: Tensor, scale: float = 1.0, padding_idx: Optional[int] = None) -> Tensor:
    """scale * weight[ids]: ids (...) int64 or int32, weight (V, C) fp32 or bf16 -> (..., C).

    Differentiable in ``weight`` (``token_embedding_bwd``: deterministic).  ``padding_idx`` (negative: from the end)
    names a row that takes no gradient.  An id outside [0, V) gives a row of NaN and no gradient; nothing outside the
    table is read."""
    if weight.requires_grad and torch.is_grad_enabled() and weight.dim() == 2:
        return TokenEmbeddingFn.apply(weight, ids, scale, _padding("token_embedding", padding_idx, weight.shape[0]))
    if padding_idx is not None and weight.dim() == 2:
        _padding("token_embedding", padding_idx, weight.shape[0])
    return token_embedding_fwd(ids, weight, scale)


# ---------------------------------------------------------------------------------------------------------
# the head's loss
# ---------------------------------------------------------------------------------------------------------

def linear_cross_entropy_fwd(x: Tensor, weight: Tensor, labels: Tensor, ignore_index: int = -100,
                             reduction: str = "mean") -> tuple:
    """The loss as ``linear_cross_entropy`` returns it, and the workspace that ``linear_cross_entropy_bwd`` reads."""
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
    if tuple(labels.shape) != tuple(x.shape[:-1]):
        raise ValueError(f"{op}: labels must be {tuple(x.shape[:-1])}, got {tuple(labels.shape)}")
    x2, w, y = _rows(x.detach()), _rows(weight.detach()), labels.contiguous()
    T, d = x2.shape
    V = w.shape[0]
    if T == 0:
        empty = float("nan") if reduction == "mean" else 0.0
        loss = torch.full(labels.shape if reduction == "none" else (), empty, dtype=torch.float32, device=x.device)
        return loss, None
    lib, code, ldw = _lib.load(), _lib.DTYPE_CODE[x.dtype], _row_stride(w)
    nb = lib.cdssm_linear_cross_entropy_workspace_bytes(code, _lib.ptr(w), ldw, T, V, d)
    if nb < 0:
        raise ValueError(f"{op}: {_lib.last_error()}")
    ws = torch.empty(nb, dtype=torch.uint8, device=x.device)
    loss = torch.empty(labels.shape if reduction == "none" else (), dtype=torch.float32, device=x.device)
    _call("cdssm_linear_cross_entropy_fwd", x.device, code, _INDEX_BYTES[y.dtype], x2.data_ptr(), _row_stride(x2),
          w.data_ptr(), ldw, y.data_ptr(), ignore_index, _REDUCTIONS[reduction], loss.data_ptr(), ws.data_ptr(), T, V, d)
    return loss, ws


def linear_cross_entropy_bwd(grad: Tensor, weight: Tensor, workspace: Tensor, x_shape: Sequence[int],
                             reduction: str = "mean", need_x: bool = True, need_weight: bool = True) -> tuple:
    """(dx, dW) in weight's dtype from the gradient of the loss and the workspace of the forward over x of that shape, the
    same weight and reduction; None in the place of one that is not needed."""
    op = "linear_cross_entropy_bwd"
    _check_float(op, "weight", weight)
    if reduction not in _REDUCTIONS:
        raise ValueError(f"{op}: reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}")
    if weight.dim() != 2 or len(x_shape) < 1:
        raise ValueError(f"{op}: x must be (..., d) and weight (V, d), got {tuple(x_shape)} and {tuple(weight.shape)}")
    w = _rows(weight.detach())
    V, d = w.shape
    T = math.prod(x_shape[:-1])
    if x_shape[-1] != d or grad.device != w.device or grad.numel() != (T if reduction == "none" else 1):
        raise ValueError(f"{op}: the gradient of a {reduction} over x {tuple(x_shape)} and weight {tuple(w.shape)} on "
                         f"{w.device}, got {tuple(grad.shape)} on {grad.device}")
    g = grad.detach().to(torch.float32).contiguous()
    dx = torch.empty(*x_shape, dtype=w.dtype, device=w.device) if need_x else None
    dw = torch.empty(V, d, dtype=w.dtype, device=w.device) if need_weight else None
    if T == 0:
        return dx, None if dw is None else dw.zero_()
    if dx is None and dw is None:
        return None, None
    lib, code, ldw = _lib.load(), _lib.DTYPE_CODE[w.dtype], _row_stride(w)
    if workspace is None or workspace.device != w.device or workspace.numel() != (
            lib.cdssm_linear_cross_entropy_workspace_bytes(code, _lib.ptr(w), ldw, T, V, d)):
        raise ValueError(f"{op}: not the workspace of a forward over x {tuple(x_shape)} and this weight")
    ws = torch.empty(lib.cdssm_linear_cross_entropy_bwd_workspace_bytes(code, _lib.ptr(w), ldw, T, V, d),
                     dtype=torch.uint8, device=w.device)
    _call("cdssm_linear_cross_entropy_bwd", w.device, code, w.data_ptr(), ldw, _REDUCTIONS[reduction], g.data_ptr(),
          workspace.data_ptr(), _lib.ptr(dx), d, _lib.ptr(dw), d, ws.data_ptr(), T, V, d)
    return dx, dw


class LinearCrossEntropyFn(torch.autograd.Function):
    """``linear_cross_entropy`` as an autograd node: (x, weight, labels, ignore_index, reduction) -> loss.  Keeps the
    packed rows of x and their log sums, not the logits; the backward forms those again."""

    @staticmethod
    def forward(ctx, x, weight, labels, ignore_index, reduction):
        loss, ws = linear_cross_entropy_fwd(x, weight, labels, ignore_index, reduction)
        ctx.save_for_backward(weight, ws)
        ctx.meta = (tuple(x.shape), reduction)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        weight, ws = ctx.saved_tensors
        shape, reduction = ctx.meta
        dx, dw = linear_cross_entropy_bwd(grad, weight, ws, shape, reduction, ctx.needs_input_grad[0],
                                          ctx.needs_input_grad[1])
        return dx, dw, None, None, None


def linear_cross_entropy(x: Tensor, weight: Tensor, labels: Tensor, ignore_index: int = -100,
                         reduction: str = "mean") -> Tensor:
    """Softmax cross entropy of the logits x @ weight^T against ``labels``, the logits never stored.

    x (..., d) and weight (V, d) fp32 or bf16, labels (...) int64 or int32; fp32 loss: a number for ``reduction``
    "mean" (over the labels that are not ``ignore_index``; NaN if there is none) or "sum", (...) for "none" (0 where
    ignored).  Differentiable in x and weight.  Rows whose label is ``ignore_index`` take no part, whatever they hold: their
    gradient is 0.  Any other label outside [0, V) makes its row's loss, and the gradients, NaN.  A logit over an infinite
    operand is what the products give (-inf: a word of probability 0) in bf16, and NaN in fp32, whose parts of a number may be
    0 where it is not."""
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        return LinearCrossEntropyFn.apply(x, weight, labels, ignore_index, reduction)
    return linear_cross_entropy_fwd(x, weight, labels, ignore_index, reduction)[0]


# ---------------------------------------------------------------------------------------------------------
# gradient norm and clipping
# ---------------------------------------------------------------------------------------------------------

def _is_dense(t: Tensor) -> bool:
    """Whether t's elements fill one stretch of memory, in any order of its dimensions."""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != want:
            return False
        want *= size
    return True


_DTYPE_OF = operator.attrgetter("dtype")


def _list(ts: Union[Tensor, Iterable[Tensor]]) -> list:
    return [ts] if torch.is_tensor(ts) else list(ts)


def _table(op: str, what: str, ts: Sequence[Tensor]) -> tuple:
    """Addresses, dtype codes and sizes of the tensors as host arrays, and whether all are contiguous; raises for one that
    the kernels do not take.  The whole list at a time: a model has hundreds of gradients, and a loop of checks for each
    took longer than the kernels."""
    codes = list(map(_lib.DTYPE_CODE.get, map(_DTYPE_OF, ts)))
    if None in codes or len(set(map(Tensor.get_device, ts))) > 1 or (ts and not ts[0].is_cuda):
        for t in ts:
            _check_float(op, what, t)
            if t.device != ts[0].device:
                raise RuntimeError(f"{op}: tensors on {ts[0].device} and {t.device}")
    dense = all(map(Tensor.is_contiguous, ts))
    if not dense:
        for t in ts:
            if not _is_dense(t):
                raise ValueError(f"{op}: {what} of shape {tuple(t.shape)} and strides {t.stride()} has gaps or overlaps")
    return array.array("Q", map(Tensor.data_ptr, ts)), array.array("i", codes), array.array("q", map(Tensor.numel, ts)), dense


def _at(a: array.array) -> int:
    return a.buffer_info()[0]


def global_grad_norm(grads: Union[Tensor, Iterable[Tensor]]) -> Tensor:
    """The 2-norm over all elements of the given tensors (fp32 and bf16 may be mixed), as one fp32 number on their
    device: squares added in fp64, the same bits every time."""
    ts = _list(grads)
    if not ts:
        return torch.zeros(())
    ptrs, codes, sizes, _ = _table("global_grad_norm", "a gradient", ts)
    dev = ts[0].device
    lib, n = _lib.load(), len(ts)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    ws = torch.empty(lib.cdssm_grad_norm_workspace_bytes(n), dtype=torch.uint8, device=dev)
    _call("cdssm_grad_norm", dev, n, _at(ptrs), _at(codes), _at(sizes), norm.data_ptr(), ws.data_ptr())
    return norm


def clip_grads(grads: Union[Tensor, Iterable[Tensor]], max_norm: float,
               out: Optional[Sequence[Tensor]] = None) -> Tensor:
    """Scales the given tensors by min(1, max_norm / (norm + 1e-6)), norm the 2-norm over all of them, which it returns
    (one fp32 number on their device; nothing waits for it).  In place, or into ``out``: as many tensors of the same
    sizes, fp32 or bf16 (fp32 copies of bf16 gradients for an optimizer that keeps fp32 weights, rounded nowhere).
    A tensor may be given once, and must not share memory with another; a norm that is infinite or NaN scales as
    torch's clip_grad_norm_ does."""
    op = "clip_grads"
    ts = _list(grads)
    if not max_norm >= 0:
        raise ValueError(f"{op}: max_norm must be at least 0, got {max_norm}")
    outs = ts if out is None else _list(out)
    if len(outs) != len(ts):
        raise ValueError(f"{op}: {len(ts)} gradients, {len(outs)} outputs")
    if not ts:
        return torch.zeros(())
    dev = ts[0].device
    ptrs, codes, sizes, dense = _table(op, "a gradient", ts)
    optrs, ocodes, osizes, odense = (ptrs, codes, sizes, dense) if out is None else _table(op, "an output", outs)
    if out is not None and (sizes != osizes or outs[0].device != dev or not (dense and odense)):
        for t, o in zip(ts, outs):
            if (o.numel() != t.numel() or o.device != t.device
                    or not (t.is_contiguous() and o.is_contiguous() or (o.shape, o.stride()) == (t.shape, t.stride()))):
                raise ValueError(f"{op}: an output must have its gradient's size, layout and device, got "
                                 f"{tuple(o.shape)} {o.stride()} for {tuple(t.shape)} {t.stride()}")
    if len(set(optrs)) < len(optrs) and len({p for p, k in zip(optrs, sizes) if k}) < sum(1 for k in sizes if k):
        raise ValueError(f"{op}: a tensor is given twice")
    if out is not None and any(o != p for o, p in zip(optrs, ptrs)):
        given = set(ptrs)
        if any(o != p and k and o in given for o, p, k in zip(optrs, ptrs, sizes)):
            raise ValueError(f"{op}: an output is another gradient's tensor")
    lib, n = _lib.load(), len(ts)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    ws = torch.empty(lib.cdssm_grad_norm_workspace_bytes(n), dtype=torch.uint8, device=dev)
    _call("cdssm_clip_grads", dev, n, _at(ptrs), _at(codes), _at(optrs), _at(ocodes), _at(sizes), float(max_norm),
          norm.data_ptr(), ws.data_ptr())
    torch.autograd.graph.increment_version(outs)  # a graph that saved one of them has to notice
    return norm


def clip_grad_norm_(parameters: Union[Tensor, Iterable[Tensor]], max_norm: float) -> Tensor:
    """``clip_grads`` of the parameters' gradients, in place (trainer.py:242-243); parameters without a gradient are
    left out."""
    ps = [parameters] if torch.is_tensor(parameters) else list(parameters)
    return clip_grads([p.grad for p in ps if p.grad is not None], max_norm)
