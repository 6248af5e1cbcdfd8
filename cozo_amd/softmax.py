"""Softmax cross entropy over a whole table of vectors, and its gradient (cz_softmax_xent* of include/cozo_gpu.h): the loss that
trains the vectors an index holds.  Row targets[t] of `table` is the answer to queries[t]; every other row speaks against it.

Arrays are numpy on the host (a call is synchronous; bfloat16 as uint16 bits) or torch tensors on the GPU (a call only enqueues
work, on torch's current stream unless told otherwise, and may be captured into a graph).  A target of -1 (0xFFFFFFFF) is no answer:
loss and gradient of that query are 0.  The calls are no part of an autograd graph: tensors that require a gradient are taken under
torch.no_grad() only.
"""
from __future__ import annotations

import numpy as np

from . import _lib
from ._device import all_on_gpu, no_graph, on_stream
from ._lib import CZ_DEVICE_PTRS, check, ptr
from .quantized import _elem_of, _rows


def _targets(targets, T: int, gpu: bool):
    if gpu:
        import torch
        if targets.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"targets are int32 or int64, not {targets.dtype}")
        if targets.dtype == torch.int64:  # what does not fit 31 bits is no row
            targets = torch.where((targets >= -1) & (targets < 2**31), targets, torch.full_like(targets, 2**31 - 1)).to(torch.int32)
        targets = targets.contiguous()
    else:
        t = np.asarray(targets)
        if t.dtype.kind not in "iu":
            raise ValueError("targets are whole numbers")
        if t.size and (int(t.min()) < -1 or int(t.max()) > 0xFFFFFFFF):
            raise ValueError("a target is a row number or -1")
        targets = np.ascontiguousarray(t.astype(np.int64) & 0xFFFFFFFF, dtype=np.uint32)
    if tuple(targets.shape) != (T,):
        raise ValueError("targets must be [queries]")
    return targets


def _inputs(queries, table, *more):
    no_graph(queries, table, *more)
    gpu = all_on_gpu(queries, table, *more)
    if not gpu:
        queries, table = (a if isinstance(a, np.ndarray) else np.asarray(a, dtype=np.float32) for a in (queries, table))
    elem = _elem_of(table)
    if _elem_of(queries) != elem:
        raise ValueError("queries and table are of one type")
    if queries.ndim != 2 or table.ndim != 2 or queries.shape[1] != table.shape[1]:
        raise ValueError("queries [T][dim] and table [V][dim] have one dim")
    return gpu, elem


def softmax_xent(queries, table, targets, scale: float = 1.0, stream=None):
    """(loss [T] f32, lse [T] f32) of logits scale * queries . table^T; lse is what the gradient asks for"""
    L = _lib.lib()
    gpu, elem = _inputs(queries, table, targets)
    T, V, dim = int(queries.shape[0]), int(table.shape[0]), int(table.shape[1])
    if not gpu:
        (q, ldq), (w, ldw) = _rows(queries, "queries"), _rows(table, "table")
        y = _targets(targets, T, False)
        loss, lse = np.empty(T, dtype=np.float32), np.empty(T, dtype=np.float32)
        check(L.cz_softmax_xent(ptr(q), ldq, ptr(w), ldw, elem, T, V, dim, ptr(y), scale, ptr(loss), ptr(lse), None, 0, 0, None))
        return loss, lse
    import torch
    with on_stream(table, stream) as s:
        (q, ldq), (w, ldw) = _rows(queries, "queries"), _rows(table, "table")
        y = _targets(targets, T, True)
        loss = torch.empty(T, dtype=torch.float32, device=w.device)
        lse = torch.empty(T, dtype=torch.float32, device=w.device)
        need = L.cz_softmax_xent_workspace(T, V, dim, elem, 0)
        ws = torch.empty(need, dtype=torch.uint8, device=w.device)
        check(L.cz_softmax_xent(ptr(q), ldq, ptr(w), ldw, elem, T, V, dim, ptr(y), scale, ptr(loss), ptr(lse), ptr(ws), need,
                                CZ_DEVICE_PTRS, s))
        return loss, lse


def softmax_xent_grad(queries, table, targets, lse, grad_loss, scale: float = 1.0, want_queries: bool = True, want_table: bool = True,
                      stream=None):
    """(grad_queries [T][dim], grad_table [V][dim]) of sum_t grad_loss[t] * loss[t], in the inputs' type; None where not wanted"""
    L = _lib.lib()
    gpu, elem = _inputs(queries, table, targets, lse, grad_loss)
    T, V, dim = int(queries.shape[0]), int(table.shape[0]), int(table.shape[1])
    if tuple(lse.shape) != (T,) or tuple(grad_loss.shape) != (T,):
        raise ValueError("lse and grad_loss must be [queries]")
    if not gpu:
        (q, ldq), (w, ldw) = _rows(queries, "queries"), _rows(table, "table")
        y = _targets(targets, T, False)
        lse, g = (np.ascontiguousarray(a, dtype=np.float32) for a in (lse, grad_loss))
        dq = np.empty((T, dim), dtype=q.dtype) if want_queries else None
        dw = np.empty((V, dim), dtype=w.dtype) if want_table else None
        check(L.cz_softmax_xent_grad(ptr(q), ldq, ptr(w), ldw, elem, T, V, dim, ptr(y), scale, ptr(lse), ptr(g), ptr(dq), ptr(dw),
                                     None, 0, 0, None))
        return dq, dw
    import torch
    if lse.dtype != torch.float32 or grad_loss.dtype != torch.float32:
        raise ValueError("lse and grad_loss are float32")
    with on_stream(table, stream) as s:
        (q, ldq), (w, ldw) = _rows(queries, "queries"), _rows(table, "table")
        y, lse, g = _targets(targets, T, True), lse.contiguous(), grad_loss.contiguous()
        dq = torch.empty((T, dim), dtype=q.dtype, device=w.device) if want_queries else None
        dw = torch.empty((V, dim), dtype=w.dtype, device=w.device) if want_table else None
        need = L.cz_softmax_xent_workspace(T, V, dim, elem, 1)
        ws = torch.empty(need, dtype=torch.uint8, device=w.device)
        check(L.cz_softmax_xent_grad(ptr(q), ldq, ptr(w), ldw, elem, T, V, dim, ptr(y), scale, ptr(lse), ptr(g), ptr(dq), ptr(dw),
                                     ptr(ws), need, CZ_DEVICE_PTRS, s))
        return dq, dw

