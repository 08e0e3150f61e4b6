"""Rows of the key / value cache put elsewhere, on the GPU and in place.

    reorder(tensors, index, dim)                         t[i] = t[index[i]] along dim, in every tensor
    evict(k, v, weights, positions, n, budget, recent)   a cache cut to a budget of rows per KV head

The reference's cache only grows (HF's DynamicCache, gemma_npu.py:278-300); these are for decoding that
does otherwise: beams (ops.beam_select gives the index), drafted tokens (attention.decode_tree; the
accepted path's rows are moved up), and caches of bounded size (attention.add_key_weights gives the
weights).  Everything runs on torch's current stream of the tensors' device; there is no CPU fallback.
"""
import torch

from ._lib import Rows, call_on, lib
from .ops import _native, _stream


def _runs(t, dim, name):
    """The tensor as w8a8_rows: dims before `dim` as one, those behind it as runs of contiguous bytes."""
    es = t.element_size()
    outer, outer_stride = 1, 0
    for d in range(dim - 1, -1, -1):
        size, stride = t.shape[d], t.stride(d)
        if size == 1:
            continue
        if outer == 1:
            outer_stride = stride
        elif stride != outer * outer_stride:
            raise ValueError(f"reorder: {name}: the dimensions before {dim} are not evenly spaced, strides {t.stride()}")
        outer *= size
    run, runs, run_stride = 1, 1, 0
    for d in range(t.dim() - 1, dim, -1):
        size, stride = t.shape[d], t.stride(d)
        if size == 1:
            continue
        if runs == 1 and stride == run:
            run *= size
        elif runs == 1:
            runs, run_stride = size, stride
        elif stride == runs * run_stride:
            runs *= size
        else:
            raise ValueError(f"reorder: {name}: the dimensions after {dim} are not evenly spaced, strides {t.stride()}")
    if t.numel() == 0:
        runs = 0
    return outer, Rows(t.data_ptr(), outer_stride * es, t.stride(dim) * es, run_stride * es, runs, run * es)


def reorder(tensors, index, dim=0):
    """t.select(dim, i) = t.select(dim, index[i]) for i < len(index), in place, in each of `tensors` (one or a
    list; any types and shapes, the same size along dim), all in one launch: the beams' keys and values in
    the order that ops.beam_select chose, or an accepted path's rows moved up.

    index: int64 GPU tensor [n], n <= 64 and at most the size of dim (rows past n are left as they are), or
    [outer, n] with one row per entry of the dimensions before dim.  Every row is read before any is written:
    rows may be exchanged, repeated and dropped.  An index outside the dimension leaves its row as it is.
    Views are taken as they are, so k[:, :, :length] moves the live rows only; the tensors must not overlap
    (one given twice, as a cache that two layers share, is refused), and the index is none of them: a copy of it
    reorders the tensor it was taken from."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if _native is not None and _native.reorder(tensors, index, dim):
        return
    if not isinstance(index, torch.Tensor) or index.dtype != torch.int64 or index.dim() not in (1, 2):
        raise TypeError("reorder: index must be an int64 GPU tensor [n] or [outer, n]")
    if index.device.type != "cuda":
        raise ValueError("reorder: index must be on the GPU")
    n = index.shape[-1]
    if n > 1 and index.stride(-1) != 1:
        raise ValueError("reorder: index must have contiguous rows")
    if not tensors:
        return
    rows, size, outer = [], None, None
    for i, t in enumerate(tensors):
        if not isinstance(t, torch.Tensor) or t.device != index.device:
            raise ValueError(f"reorder: tensor {i} must be on {index.device}")
        d = dim + t.dim() if dim < 0 else dim
        if not 0 <= d < t.dim():
            raise ValueError(f"reorder: tensor {i} has no dimension {dim}, shape {tuple(t.shape)}")
        if any(s > 1 and st <= 0 for s, st in zip(t.shape, t.stride())):
            raise ValueError(f"reorder: tensor {i} overlaps itself, strides {t.stride()}")
        o, r = _runs(t, d, f"tensor {i}")
        if size is not None and (t.shape[d] != size or o != outer):
            raise ValueError(f"reorder: tensor {i} has {t.shape[d]} rows in {o} entries, the first {size} in {outer}")
        size, outer = t.shape[d], o
        rows.append(r)
    if n > 64 or n > size:
        raise ValueError(f"reorder: an index of {n} for {size} rows (at most 64)")
    if index.dim() == 2 and index.shape[0] != outer:
        raise ValueError(f"reorder: index {tuple(index.shape)} for {outer} entries before dimension {dim}")
    if n == 0 or outer == 0:
        return
    call_on(index, "w8a8_reorder_rows", (Rows * len(rows))(*rows), len(rows), index.data_ptr(),
            index.stride(0) if index.dim() == 2 and outer > 1 else 0, n, size, outer, _stream(index))


def evict_workspace_bytes(KV, n, budget):
    """Bytes of scratch evict() needs (w8a8_evict_workspace_bytes)."""
    b = lib().w8a8_evict_workspace_bytes(int(KV), int(n), int(budget))
    if b < 0:
        raise ValueError(f"evict: KV={KV} n={n} budget={budget} (1 <= budget <= n)")
    return b


def evict(k, v, weights, positions, n, budget, recent=0, out=None, workspace=None):
    """Cut a cache of n rows to `budget` rows per KV head, in place: kept are the rows within `recent` of the
    head's newest position, then those of the largest weight (NaN the largest; ties: the lower row).

    k / v: [KV, Tk, D] with Tk >= n (bf16, or any type with rows of a multiple of 16 bytes), weights fp32
    [KV, >= n] (attention.add_key_weights), positions int32 [KV, >= n].  Kept rows below the budget stay where
    they are, the others move in order into the places that became free; rows from the budget on are left as
    they were.  Attention over the rows 0 .. budget - 1 (attention.decode without a window) does not depend
    on their order.  Returns (kept int32, weights fp32, positions int32), each [KV, budget]: the row that each
    row came from, and its weight and position; out: the three tensors to write them to, of which the
    latter two may be weights[:, :budget] and positions[:, :budget] themselves."""
    if _native is not None and out is None and workspace is None:
        r = _native.evict(k, v, weights, positions, n, budget, recent)
        if r is not None:
            return r
    n, budget, recent = int(n), int(budget), int(recent)
    for t, name in ((k, "k"), (v, "v")):
        if not isinstance(t, torch.Tensor) or t.device.type != "cuda" or t.dim() != 3:
            raise ValueError(f"evict: {name} must be a GPU tensor [KV, rows, head_dim]")
        if t.shape[2] > 1 and t.stride(2) != 1:
            raise ValueError(f"evict: {name}: the last dimension must be contiguous, got strides {t.stride()}")
    KV, Tk, D = k.shape
    if tuple(v.shape) != (KV, Tk, D) or v.dtype != k.dtype:
        raise ValueError(f"evict: k {tuple(k.shape)} {k.dtype} and v {tuple(v.shape)} {v.dtype} do not match")
    if not 1 <= budget <= n <= Tk or not 0 <= recent <= budget:
        raise ValueError(f"evict: n={n} of {Tk} rows, budget={budget}, recent={recent} (recent <= budget <= n)")
    for t, name, dt in ((weights, "weights", torch.float32), (positions, "positions", torch.int32)):
        if not isinstance(t, torch.Tensor) or t.dtype != dt or t.dim() != 2 or t.shape[0] != KV or t.shape[1] < n:
            raise ValueError(f"evict: {name} must be a GPU tensor [{KV}, at least {n}] of {dt}")
        if t.shape[1] > 1 and t.stride(1) != 1:
            raise ValueError(f"evict: {name} must have contiguous rows")
    if out is None:
        out = (torch.empty((KV, budget), dtype=torch.int32, device=k.device),
               torch.empty((KV, budget), dtype=torch.float32, device=k.device),
               torch.empty((KV, budget), dtype=torch.int32, device=k.device))
    else:
        for t, name, dt in zip(out, ("kept", "weights", "positions"), (torch.int32, torch.float32, torch.int32)):
            if tuple(t.shape) != (KV, budget) or t.dtype != dt or (budget > 1 and t.stride(1) != 1):
                raise ValueError(f"evict: out's {name} must be {dt} [{KV}, {budget}] with contiguous rows")
    kept, w_out, p_out = out
    if len({t.device for t in (k, v, weights, positions, kept, w_out, p_out)}) != 1:
        raise ValueError("evict: all tensors must be on one device")
    ws = workspace
    if ws is None:
        ws = torch.empty(evict_workspace_bytes(KV, n, budget), dtype=torch.uint8, device=k.device)
    elif ws.device != k.device or not ws.is_contiguous():
        raise ValueError(f"evict: the workspace must be a contiguous tensor on {k.device}")
    es = k.element_size()
    ld = lambda t: t.stride(0) if KV > 1 else t.shape[1]
    call_on(k, "w8a8_evict", k.data_ptr(), k.stride(0) * es if KV > 1 else 0, k.stride(1) * es if Tk > 1 else D * es,
            v.data_ptr(), v.stride(0) * es if KV > 1 else 0, v.stride(1) * es if Tk > 1 else D * es, D * es, KV, n,
            weights.data_ptr(), ld(weights), positions.data_ptr(), ld(positions), budget, recent, kept.data_ptr(), ld(kept),
            w_out.data_ptr(), ld(w_out), p_out.data_ptr(), ld(p_out), ws.data_ptr(), ws.numel() * ws.element_size(),
            _stream(k))
    return kept, w_out, p_out
