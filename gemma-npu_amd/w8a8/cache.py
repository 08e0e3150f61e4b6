"""Rows of the key / value cache put elsewhere, on the GPU and in place, and caches of 8-bit codes.

    reorder(tensors, index, dim)                         t[i] = t[index[i]] along dim, in every tensor
    evict(k, v, weights, positions, n, budget, recent)   a cache cut to a budget of rows per KV head
    BlockCache(KV, capacity, D, dtype)                   a cache of 8-bit codes with a scale per block of 64 rows
    append(c, k, v, n), read(c, start, n)                rows put into it and read back

The reference's cache only grows (HF's DynamicCache, gemma_npu.py:278-300); these are for decoding that
does otherwise: beams (ops.beam_select gives the index), drafted tokens (attention.decode_tree; the
accepted path's rows are moved up), and caches of bounded size (attention.add_key_weights gives the
weights).  Everything runs on torch's current stream of the tensors' device; there is no CPU fallback.
"""
import torch

from ._lib import Rows, call_on, lib
from .ops import _native, _stream

BLOCK = 64  # rows of a BlockCache that share a scale


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


class BlockCache:
    """The keys and values of one layer in 8 bits: `capacity` rows of KV heads, D values each (128, 256, 512).

    Every whole block of 64 rows is held as int8 codes (dtype torch.float8_e4m3fn: e4m3) with one fp32 scale per KV
    head, for keys and for values: max |x| / 127 (times 1 / 448), as the engine quantises activations.  The rows of the block
    that is not whole yet stay bf16, so what it holds depends on the rows alone, not on how they were appended.  Holds
    half a bf16 cache's bytes; attention.block_attention attends to it.  `data` is opaque (the order in which the
    matrix instructions take the codes).

    bf16 rows are held of two blocks: of the even and of the odd ones that which append() last put rows into, as one of
    its last two blocks.  A length that append(), read() or block_attention() is given has to be a multiple of 64 or lie
    in one of these.  Lengths given as ints are checked against the ints given before; once a length came from device
    memory, or an append was captured into a graph, nothing is known on the host and nothing is checked."""

    __slots__ = ("data", "KV", "capacity", "D", "dtype", "_ring", "_made")

    def __init__(self, KV, capacity, D, dtype=torch.int8, device="cuda"):
        if dtype not in (torch.int8, torch.float8_e4m3fn):
            raise TypeError(f"BlockCache: codes are torch.int8 or torch.float8_e4m3fn, got {dtype}")
        n = lib().w8a8_block_cache_bytes(int(KV), int(capacity), int(D))
        if n < 0:
            raise ValueError(f"BlockCache: invalid shape KV={KV} capacity={capacity} D={D} (D: 128, 256, 512)")
        self.KV, self.capacity, self.D, self.dtype = int(KV), int(capacity), int(D), dtype
        with torch.inference_mode(False):  # (a tensor that counts what torch writes to it)
            self.data = torch.empty(n, dtype=torch.uint8, device=device)
        if self.data.device.type != "cuda":
            raise ValueError(f"BlockCache: expected a GPU, got device {device}")
        # the even and the odd block whose rows are held (None: unknown), data's version at that time, whether this is kept
        self._ring, self._made = [None, None, self.data._version, True], self.data

    @property
    def device(self):
        return self.data.device

    @property
    def e4m3(self):
        return 1 if self.dtype == torch.float8_e4m3fn else 0

    def _lost(self, n):
        """Why there are no n rows, or None: the bf16 rows of n's block have made way for another's."""
        if type(n) is not int:
            if isinstance(n, torch.Tensor):
                return None
            n = int(n)
        b, r = n // BLOCK, self._ring
        if n % BLOCK == 0 or r[b & 1] is None or r[b & 1] == b or not self._known():
            return None
        if torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
            return None
        return (f"{n} rows: those of block {b} ({BLOCK * b} ..) are not held in bf16 any more, block {r[b & 1]}'s came in "
                f"their place; a multiple of {BLOCK} is possible")

    def _appended(self, n, m):
        """m rows were appended to n."""
        r = self._ring
        if not r[3]:
            return
        if torch.cuda.is_current_stream_capturing() or (type(n) is not int and isinstance(n, torch.Tensor)):
            r[3] = False
            return
        if not self._known():
            r[0] = r[1] = None
            r[2] = self.data._version if self.data is self._made else -1
        first, last = int(n) // BLOCK, (int(n) + m - 1) // BLOCK
        r[last & 1] = last
        if first < last:
            r[last - 1 & 1] = last - 1

    def _known(self):
        """Whether the ring is what the calls made it: `data` is the tensor it was, and torch has written nothing to it (as
        where one cache is copied over another)."""
        return self._ring[3] and self.data is self._made and self._ring[2] == self.data._version


def append(c, k, v, n):
    """Rows n .. n + m - 1 of BlockCache c: k / v bf16 [KV, m, D] (any strides with a contiguous last dimension).

    n: the rows that are there, an int, or an int32 GPU tensor of one element (the launch then does not depend on it,
    so a captured step replays at each new length).  n may be less than before, as where drafted tokens are taken
    back: rows from n on are written anew.  It has to be a multiple of 64 then, or lie in one of the two blocks whose
    rows are held in bf16 (BlockCache): in the newest two, as long as it did not go back from further on before.  After 600
    rows and 10 put to 128, for instance, 100 is refused: of the odd blocks the ring holds the rows from 576 on."""
    if not isinstance(c, BlockCache):
        raise TypeError(f"append: expected a BlockCache, got {type(c).__name__}")
    lost = c._lost(n)
    if lost is None and _native is not None and _native.block_append(c.data, c.KV, c.capacity, c.D, c.e4m3, k, v, n):
        c._appended(n, k.shape[1])
        return
    for t, name in ((k, "k"), (v, "v")):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.bfloat16 or t.device != c.device:
            raise TypeError(f"append: {name} must be a bf16 tensor on {c.device}")
        if t.dim() != 3 or t.shape[0] != c.KV or t.shape[2] != c.D or t.shape[1] != k.shape[1]:
            raise ValueError(f"append: {name} must be [{c.KV}, rows, {c.D}], got {tuple(t.shape)}")
        if t.stride(2) != 1:
            raise ValueError(f"append: {name}: the last dimension must be contiguous, got strides {t.stride()}")
    m, dev = k.shape[1], None
    if isinstance(n, torch.Tensor):
        if n.dtype != torch.int32 or n.numel() != 1 or n.device != c.device:
            raise ValueError("append: n must be an int or an int32 tensor of one element on the cache's device")
        dev, n = n, -1
    elif not 0 <= int(n) <= c.capacity - m:
        raise ValueError(f"append: {m} rows from {n} on in a cache of {c.capacity}")
    if m == 0:
        return
    if lost is not None:
        raise ValueError(f"append: {lost}")
    call_on(k, "w8a8_block_append", c.data.data_ptr(), c.KV, c.capacity, c.D, c.e4m3, k.data_ptr(), k.stride(0) if c.KV > 1 else 0,
            k.stride(1) if m > 1 else c.D, v.data_ptr(), v.stride(0) if c.KV > 1 else 0, v.stride(1) if m > 1 else c.D, m, int(n),
            None if dev is None else dev.data_ptr(), _stream(k))
    c._appended(n if dev is None else dev, m)


def read(c, start, n):
    """(k, v) bf16 [KV, n - start, D]: what rows start .. n - 1 of BlockCache c, which holds n rows (or more, if n is one of the
    lengths that append() may go back to), stand for, rounded to bf16 (for attention.attention over what came before,
    or to put the rows elsewhere)."""
    if not isinstance(c, BlockCache):
        raise TypeError(f"read: expected a BlockCache, got {type(c).__name__}")
    lost = c._lost(n)
    if lost is None and _native is not None:
        r = _native.block_read(c.data, c.KV, c.capacity, c.D, c.e4m3, start, n)
        if r is not None:
            return r
    start, n = int(start), int(n)
    if not 0 <= start <= n <= c.capacity:
        raise ValueError(f"read: rows {start} .. {n} of a cache of {c.capacity}")
    if lost is not None and n > start:
        raise ValueError(f"read: {lost}")
    k = torch.empty((c.KV, n - start, c.D), dtype=torch.bfloat16, device=c.device)
    v = torch.empty_like(k)
    if n > start:
        call_on(k, "w8a8_block_read", c.data.data_ptr(), c.KV, c.capacity, c.D, c.e4m3, start, n, k.data_ptr(), v.data_ptr(), _stream(k))
    return k, v
