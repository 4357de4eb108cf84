"""Embedding lookup with scaling, and the gradient of the table, on the device.

:func:`embedding` is differentiable in the table; :func:`embedding_backward`
gives the gradient by itself, or adds it to one that is there (the
micro-batches of an accumulated step then touch only the rows of their own
tokens, where autograd writes and adds whole tables).  The rows of equal
tokens are summed in fp32 in ascending position, so the gradient repeats bit
for bit.

A token outside the table gives a row of zeros and no gradient, and sets
``ERR_BAD_INDEX`` in the int32 error word ``err`` where one is given (as the
blocks' error words; reading it waits for the device, so the caller chooses
when).
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import call_on, differentiated, ptr

MAX_WIDTH = 1 << 22


def _check_ids(ids: torch.Tensor, of: torch.Tensor) -> torch.Tensor:
    if ids.dtype is not torch.int64 and ids.dtype is not torch.int32:
        raise TypeError(f"ids: expected int32 or int64, got {ids.dtype}")
    if ids.get_device() != of.get_device():
        raise ValueError(f"ids: expected on {of.device}, got {ids.device}")
    return ids.contiguous()


def _err_at(err: Optional[torch.Tensor], of: torch.Tensor) -> Optional[int]:
    if err is None:
        return None
    if err.dtype is not torch.int32 or err.numel() < 1 or err.get_device() != of.get_device():
        raise ValueError(f"err: expected an int32 word on {of.device}")
    return err.data_ptr()


def _padding(padding_idx: Optional[int], V: int) -> int:
    if padding_idx is None:
        return -1
    if not -V <= padding_idx < V:
        raise ValueError(f"padding_idx {padding_idx} outside a table of {V} rows")
    return padding_idx % V


def embedding_forward(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0,
                      err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``scale * table[ids]``, rounded once to the table's type."""
    if table.dim() != 2 or table.shape[1] < 1:
        raise ValueError(f"table: expected [rows, width], got {tuple(table.shape)}")
    if table.shape[1] > MAX_WIDTH:
        raise ValueError(f"rows of {table.shape[1]} values; at most {MAX_WIDTH} are handled")
    if not table.is_contiguous():
        raise ValueError("table: must be contiguous")
    ids = _check_ids(ids, table)
    err_at = _err_at(err, table)
    code = _lib.dtype_code(table.dtype)
    at = ptr(table)               # on a CUDA device, and so are the others
    V, H = table.shape
    out = table.new_empty((*ids.shape, H))
    call_on(table.get_device(), "usaf_embedding_fwd", ids.data_ptr(), 8 * ids.element_size(), ids.numel(), at, code, V, H,
            float(scale), out.data_ptr(), err_at)
    return out


def embedding_backward(dout: torch.Tensor, ids: torch.Tensor, num_embeddings: int, scale: float = 1.0,
                       padding_idx: Optional[int] = None, grad: Optional[torch.Tensor] = None,
                       err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of the table: ``scale`` times the sum of ``dout``'s rows at each
    token's positions, zeros in the other rows and in ``padding_idx``'s.  With
    ``grad`` ([num_embeddings, width], ``dout``'s type or fp32) the sums are
    added into it instead, and rows without tokens are not touched."""
    V = int(num_embeddings)
    if V < 0:
        raise ValueError(f"num_embeddings: expected >= 0, got {V}")
    shape = dout.shape
    if not shape or shape[:-1] != ids.shape or shape[-1] < 1:
        raise ValueError(f"dout: expected shape {tuple(ids.shape)} + (width,), got {tuple(shape)}")
    H = shape[-1]
    if H > MAX_WIDTH:
        raise ValueError(f"rows of {H} values; at most {MAX_WIDTH} are handled")
    ids = _check_ids(ids, dout)
    err_at = _err_at(err, dout)
    pad = _padding(padding_idx, V)
    dout = dout.contiguous()
    code = g_code = _lib.dtype_code(dout.dtype)
    at = ptr(dout)                # on a CUDA device, and so are the others
    adds = grad is not None
    if adds:
        if tuple(grad.shape) != (V, H):
            raise ValueError(f"grad: expected shape {(V, H)}, got {tuple(grad.shape)}")
        if grad.dtype is not dout.dtype and grad.dtype is not torch.float32:
            raise TypeError(f"grad: expected {dout.dtype} or torch.float32, got {grad.dtype}")
        if grad.get_device() != dout.get_device() or not grad.is_contiguous():
            raise ValueError(f"grad: must be contiguous, on {dout.device}")
        g_code = _lib.dtype_code(grad.dtype)
    else:
        grad = dout.new_empty((V, H))
    n = ids.numel()
    ws = dout.new_empty(_lib.LIB.usaf_embedding_workspace_bytes(n, V, H), dtype=torch.uint8)
    if adds:
        torch.autograd.graph.increment_version(grad)      # a graph that saved it finds it changed
    call_on(dout.get_device(), "usaf_embedding_bwd", at, ids.data_ptr(), 8 * ids.element_size(), n, code, V, H,
            float(scale), pad, int(adds), grad.data_ptr(), g_code, ws.data_ptr(), err_at)
    return grad


def _add_at_the_end(table: torch.Tensor, dout: torch.Tensor, ids: torch.Tensor, *args) -> None:
    """Adds to ``table.grad`` when the backward pass is through, on the stream
    that backward() was called on: autograd has made it wait for the leaves'
    gradients there, and neither another lookup of the table on a stream of its
    own nor the table's use elsewhere in the model adds at the same time."""
    dev = dout.get_device()
    stream = torch.cuda.current_stream(dev)

    def add() -> None:
        caller = torch.cuda.current_stream(dev)
        if caller != stream:
            caller.wait_stream(stream)
            dout.record_stream(caller)
            ids.record_stream(caller)
        if _can_add(table.grad, dout):
            embedding_backward(dout, ids, *args, grad=table.grad)
        else:
            new = embedding_backward(dout, ids, *args)
            table.grad = new if table.grad is None else table.grad + new

    torch.autograd.Variable._execution_engine.queue_callback(add)


def _can_add(held: Optional[torch.Tensor], dout: torch.Tensor) -> bool:
    return held is not None and held.is_contiguous() and held.dtype in (dout.dtype, torch.float32)


def _adds_to(leaf_node) -> bool:
    """Whether the backward pass that runs now adds to this leaf's ``.grad``;
    ``torch.autograd.grad`` hands the gradient out instead (the engine then
    refuses the question for a leaf)."""
    try:
        return torch._C._will_engine_execute_node(leaf_node)
    except RuntimeError:
        return False


class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale, padding_idx, err, into_grad):
        ctx.save_for_backward(ids)
        ctx.args = (table.shape[0], scale, padding_idx)
        ctx.into = table if into_grad else None
        return embedding_forward(ids, table, scale, err)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        (ids,) = ctx.saved_tensors
        # next_functions: of the tensors among the inputs, ids and the table first
        if ctx.into is not None and _can_add(ctx.into.grad, dout) and _adds_to(ctx.next_functions[1][0]):
            _add_at_the_end(ctx.into, dout, ids, *ctx.args)
            return None, None, None, None, None, None
        return None, embedding_backward(dout, ids, *ctx.args), None, None, None, None


def embedding(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0, padding_idx: Optional[int] = None,
              err: Optional[torch.Tensor] = None, into_grad: bool = False) -> torch.Tensor:
    """``scale * table[ids]`` (any shape of ``ids``), differentiable in the
    table, once and backward (forward mode is refused); ``padding_idx``'s row
    gets no gradient.

    ``into_grad``: ``backward()`` adds the gradient to ``table.grad`` itself, where
    the table (a leaf) has one, when the pass is through (on the stream that it
    was called on), and autograd is given nothing, so the table's hooks do not see
    it: for loops that accumulate micro-batches.  ``torch.autograd.grad`` gets its
    gradient as ever."""
    _padding(padding_idx, table.shape[0])
    if differentiated(table):
        if into_grad and table.requires_grad and not table.is_leaf:
            raise ValueError("into_grad: the table must be a leaf")
        return _EmbeddingFn.apply(ids, table, scale, padding_idx, err, into_grad)
    return embedding_forward(ids, table, scale, err)
