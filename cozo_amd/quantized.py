"""4-bit rows: a table of vectors in an eighth of its f32 bytes (cz_q4_* of include/cozo_gpu.h).

`quantize` makes a `Q4Table` of vectors; the table answers `dots` (products of queries with every row), `knn` (exhaustive k-NN
over the rows as they stand) and `dequantize`.  Arrays are numpy on the host (a call is synchronous) or torch tensors on the GPU
(a call only enqueues work, on torch's current stream unless told otherwise, and may be captured into a graph).  On the host
bfloat16 is held as uint16 bits; row numbers in results are uint32 on the host and int32 on the GPU (a missing one is 0xFFFFFFFF / -1).
Results are no part of an autograd graph: queries that require a gradient are taken under torch.no_grad() only (`quantize`, whose codes have none,
takes any vectors).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Any, Optional

import numpy as np

from . import _lib
from ._device import all_on_gpu, no_graph, on_stream
from ._lib import CZ_DEVICE_PTRS, CZ_ELEM_BF16, CZ_ELEM_F32, check, ptr
from .hnsw import DISTANCES


def _elem_of(a) -> int:
    name = str(a.dtype).replace("torch.", "")
    if name == "float32":
        return CZ_ELEM_F32
    if name == "bfloat16" or (isinstance(a, np.ndarray) and a.dtype == np.uint16):
        return CZ_ELEM_BF16
    raise ValueError(f"vectors are float32 or bfloat16, not {a.dtype}")


def _rows(a, what: str):
    """a 2-D array whose rows are contiguous, and the distance between rows in elements"""
    if a.ndim != 2:
        raise ValueError(f"{what} must be [rows][dim]")
    if isinstance(a, np.ndarray):
        a = np.ascontiguousarray(a)
        return a, a.shape[1]
    if a.shape[1] > 1 and a.stride(1) != 1 or a.stride(0) < a.shape[1]:  # transposed or broadcast rows
        a = a.contiguous()
    return a, max(int(a.stride(0)), a.shape[1])


@dataclass
class Q4Table:
    """codes u8 [n][groups * group / 2], scales bf16 [n][groups], sqnorms f32 [n] (needed by `knn` only)"""
    codes: Any
    scales: Any
    sqnorms: Any
    dim: int

    def __post_init__(self):
        if self.codes.ndim != 2 or self.scales.ndim != 2 or self.codes.shape[0] != self.scales.shape[0]:
            raise ValueError("codes and scales must be [rows][..]")
        groups, width = self.scales.shape[1], self.codes.shape[1]
        self.group = 2 * width // groups if groups else 0
        if self.group not in (32, 64, 128) or groups * self.group != 2 * width:
            raise ValueError("codes and scales belong to no group of 32, 64 or 128")
        if -(-self.dim // self.group) != groups:
            raise ValueError(f"{groups} groups of {self.group} do not hold rows of {self.dim}")
        if self.sqnorms is not None and tuple(self.sqnorms.shape) != (self.codes.shape[0],):
            raise ValueError("sqnorms must be [rows]")
        types = [str(a.dtype).replace("torch.", "") for a in (self.codes, self.scales, self.sqnorms) if a is not None]
        if types[0] != "uint8" or types[1] not in ("bfloat16", "uint16") or types[2:] not in ([], ["float32"]):
            raise ValueError("codes are uint8, scales bfloat16 (uint16 bits on the host), sqnorms float32")
        self._gpu = all_on_gpu(self.codes, self.scales, self.sqnorms)
        contiguous = (lambda a: a.is_contiguous()) if self._gpu else (lambda a: a.flags.c_contiguous)
        if not all(contiguous(a) for a in (self.codes, self.scales, self.sqnorms) if a is not None):
            raise ValueError("the table's arrays must be contiguous")

    @property
    def n(self) -> int:
        return int(self.codes.shape[0])

    def __len__(self) -> int:
        return self.n

    @property
    def nbytes(self) -> int:
        return sum(int(np.prod(a.shape)) * w for a, w in ((self.codes, 1), (self.scales, 2), (self.sqnorms, 4)) if a is not None)

    def _queries(self, queries):
        gpu = all_on_gpu(self.codes, queries)
        no_graph(queries, self.scales)
        if not gpu:
            queries = np.ascontiguousarray(queries, dtype=np.float32)
        elif str(queries.dtype) != "torch.float32":
            raise ValueError(f"queries are float32, not {queries.dtype}")
        if queries.ndim == 1:
            queries = queries[None, :]
        if queries.ndim != 2 or queries.shape[1] != self.dim:
            raise ValueError("query vector dimension mismatch")
        return queries.contiguous() if gpu else queries

    def dequantize(self, rows=None, stream=None):
        """f32 rows: those that `rows` names (a number that is no row: refused on the host, NaN on the GPU), or all"""
        L = _lib.lib()
        no_graph(self.scales)
        if not self._gpu:
            r = None if rows is None else np.asarray(rows).reshape(-1)
            if r is not None:
                if r.size and (r.dtype.kind not in "iu" or int(r.min()) < 0 or int(r.max()) >= self.n):
                    raise ValueError("rows are numbers of rows of the table")
                r = np.ascontiguousarray(r, dtype=np.uint32)
            m = self.n if r is None else r.size
            out = np.empty((m, self.dim), dtype=np.float32)
            check(L.cz_q4_dequantize(ptr(self.codes), ptr(self.scales), self.n, self.dim, self.group, ptr(r), m, ptr(out), 0, None))
            return out
        import torch
        with on_stream(self.codes, stream) as s:
            r = None
            if rows is not None:
                all_on_gpu(self.codes, rows)
                if rows.dtype not in (torch.int32, torch.int64):
                    raise ValueError(f"rows are int32 or int64, not {rows.dtype}")
                r = rows.reshape(-1)
                if r.dtype == torch.int64:  # what does not fit 31 bits is no row
                    r = torch.where((r >= 0) & (r < 2**31), r, torch.full_like(r, -1)).to(torch.int32)
                r = r.contiguous()
            m = self.n if r is None else r.numel()
            out = torch.empty((m, self.dim), dtype=torch.float32, device=self.codes.device)
            check(L.cz_q4_dequantize(ptr(self.codes), ptr(self.scales), self.n, self.dim, self.group, ptr(r), m, ptr(out),
                                     CZ_DEVICE_PTRS, s))
            return out

    def dots(self, queries, stream=None):
        """f32 [B][n]: the products of every query with every row"""
        L = _lib.lib()
        if not self._gpu:
            q = self._queries(queries)
            out = np.empty((q.shape[0], self.n), dtype=np.float32)
            check(L.cz_q4_dots(ptr(self.codes), ptr(self.scales), self.n, self.dim, self.group, ptr(q), q.shape[0], ptr(out), None, 0,
                               0, None))
            return out
        import torch
        with on_stream(self.codes, stream) as s:
            q = self._queries(queries)
            B, dev = q.shape[0], self.codes.device
            out = torch.empty((B, self.n), dtype=torch.float32, device=dev)
            need = L.cz_q4_workspace(self.n, self.dim, self.group, B, 0)
            ws = torch.empty(need, dtype=torch.uint8, device=dev)
            check(L.cz_q4_dots(ptr(self.codes), ptr(self.scales), self.n, self.dim, self.group, ptr(q), B, ptr(out), ptr(ws), need,
                               CZ_DEVICE_PTRS, s))
            return out

    def knn(self, queries, k: int, distance: str = "Cosine", radius: Optional[float] = None, poison=None, stream=None):
        """(ids [B][k], distances [B][k] f64, count [B]): the k rows nearest to each query among all rows, ascending, ties to the
        lower row; distances are the reference's (runtime/hnsw.rs:66-109) from the rows as they stand."""
        L = _lib.lib()
        if self.sqnorms is None:
            raise ValueError("knn needs the table's sqnorms")
        metric, args = DISTANCES[distance], (int(radius is not None), float(radius or 0.0))
        if not self._gpu:
            q = self._queries(queries)
            B = q.shape[0]
            ids = np.empty((B, k), dtype=np.uint32)
            dist = np.empty((B, k), dtype=np.float64)
            cnt = np.empty(B, dtype=np.uint32)
            check(L.cz_q4_knn(metric, ptr(self.codes), ptr(self.scales), ptr(self.sqnorms), self.n, self.dim, self.group, ptr(q), B, k,
                              *args, ptr(ids), ptr(dist), ptr(cnt), None, 0, ptr(poison), 0, None))
            return ids, dist, cnt
        import torch
        with on_stream(self.codes, stream) as s:
            q = self._queries(queries)
            B, dev = q.shape[0], self.codes.device
            ids = torch.empty((B, k), dtype=torch.int32, device=dev)
            dist = torch.empty((B, k), dtype=torch.float64, device=dev)
            cnt = torch.empty(B, dtype=torch.int32, device=dev)
            need = L.cz_q4_workspace(self.n, self.dim, self.group, B, k)
            ws = torch.empty(need, dtype=torch.uint8, device=dev)
            check(L.cz_q4_knn(metric, ptr(self.codes), ptr(self.scales), ptr(self.sqnorms), self.n, self.dim, self.group, ptr(q), B, k,
                              *args, ptr(ids), ptr(dist), ptr(cnt), ptr(ws), need, ptr(poison), CZ_DEVICE_PTRS, s))
            return ids, dist, cnt


def quantize(vectors, group: int = 64, stream=None) -> Q4Table:
    """the 4-bit form of f32 or bf16 rows (cz_q4_quantize)"""
    L = _lib.lib()
    gpu = all_on_gpu(vectors)
    if not gpu and not isinstance(vectors, np.ndarray):
        vectors = np.asarray(vectors, dtype=np.float32)
    elem = _elem_of(vectors)
    if vectors.ndim != 2 or vectors.shape[1] == 0:
        raise ValueError("vectors must be [rows][dim]")
    if group not in (32, 64, 128):
        raise ValueError(f"group is 32, 64 or 128, not {group}")
    n, dim = int(vectors.shape[0]), int(vectors.shape[1])
    groups = -(-dim // group)
    if not gpu:
        vectors, ld = _rows(vectors, "vectors")
        codes = np.empty((n, groups * group // 2), dtype=np.uint8)
        scales = np.empty((n, groups), dtype=np.uint16)
        sq = np.empty(n, dtype=np.float32)
        check(L.cz_q4_quantize(ptr(vectors), elem, n, dim, ld, group, ptr(codes), ptr(scales), ptr(sq), 0, None))
        return Q4Table(codes, scales, sq, dim)
    import torch
    with on_stream(vectors, stream) as s:
        vectors, ld = _rows(vectors, "vectors")
        codes = torch.empty((n, groups * group // 2), dtype=torch.uint8, device=vectors.device)
        scales = torch.empty((n, groups), dtype=torch.bfloat16, device=vectors.device)
        sq = torch.empty(n, dtype=torch.float32, device=vectors.device)
        check(L.cz_q4_quantize(ptr(vectors), elem, n, dim, ld, group, ptr(codes), ptr(scales), ptr(sq), CZ_DEVICE_PTRS, s))
        return Q4Table(codes, scales, sq, dim)
