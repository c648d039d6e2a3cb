"""The state cache: rows of K and V held in 4 bits in HBM and read by id, the attention over them,
and eviction of rows by accumulated attention weight.

It stands beside the feature server as a cache of rows: with pages of one slot a page is a graph
node and a table row holds a seed's sampled neighbours; with larger pages a table row is a
sequence.  Serving only: no gradients flow through a cache (tensors that require grad are refused).
All calls run on the current stream of their tensors' device, neither synchronise nor allocate
outside torch's allocator (but for the report words, once a process), and can be captured into a
graph.  An id or length outside the cache or its table is left out or clamped by the kernel, and the
next gather or state call (or dgs.ops._check_async_errors) raises.
"""
import contextlib
import ctypes
import math

import torch

from ._lib import c_i64, c_vp, check, lib, stream_ptr

__all__ = ["StateCache", "evict_rows", "neighbour_table"]

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # DGS_STATE_* (dgs_amd.h)


class _CCache(ctypes.Structure):
    _fields_ = [("k_codes", c_vp), ("k_scales", c_vp), ("v_codes", c_vp), ("v_scales", c_vp),
                ("pages", c_i64), ("page_size", ctypes.c_int32), ("heads", ctypes.c_int32),
                ("head_dim", ctypes.c_int32), ("group", ctypes.c_int32)]


_HERE = contextlib.nullcontext()
_current = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _on(index):
    """Makes device `index` the current one for the call: the library launches on that."""
    return _HERE if _current() == index else torch.cuda.device(index)


def _require(cond, msg):
    if not cond:
        raise RuntimeError(msg)


def _ids(t, name):
    if t.dtype is not torch.int32 and t.dtype is not torch.int64:
        raise RuntimeError(f"{name}: ID can only be int32 or int64")
    return t if t.is_contiguous() else t.contiguous()


def _no_grad(*tensors):
    for t in tensors:
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("the state cache has no backward: detach the tensor or use "
                               "torch.no_grad()")


def _same_device(index, *tensors):
    """Every tensor lies on CUDA device `index` (the cache's, or the weights')."""
    for t in tensors:
        if t.get_device() != index or not t.is_cuda:
            raise RuntimeError(f"every tensor of a call must be a CUDA tensor on device {index}, "
                               f"not on {t.device}")


def _rows16(t):
    """t [n, heads, dim] with contiguous channels and 16-byte aligned rows (copied if need be)."""
    e = t.element_size()
    s0, s1, s2 = t.stride()
    if s2 == 1 and (t.data_ptr() | s0 * e | s1 * e) % 16 == 0:
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


class StateCache:
    """K and V rows of `heads` heads x `head_dim` channels in 4 bits, in `num_pages` pages of
    `page_size` slots (a power of two; a slot holds one row of every head).

    A group of `group` channels (a multiple of 8 that divides head_dim; by default 64 if that
    divides it, else all of them) shares a bfloat16 scale s and base b, value = s * code + b with
    codes 0..15.  The buffers are the attributes k_codes, v_codes (uint8 [pages, heads, page_size,
    head_dim / 2], two channels a byte, the even one low) and k_scales, v_scales (bfloat16 [pages,
    heads, page_size, head_dim / group, 2]).  A flat slot is page * page_size + offset."""

    def __init__(self, num_pages, page_size, heads, head_dim, group=None, device=None):
        if group is None:
            group = 64 if head_dim % 64 == 0 else head_dim
        self._check_shape(num_pages, page_size, heads, head_dim, group)
        dev = torch.device("cuda" if device is None else device)
        _require(dev.type == "cuda", "the state cache lives on a CUDA device")
        lead = (num_pages, heads, page_size)

        def codes():
            return torch.zeros(lead + (head_dim // 2,), dtype=torch.uint8, device=dev)

        def scales():
            return torch.zeros(lead + (head_dim // group, 2), dtype=torch.bfloat16, device=dev)

        self._adopt(codes(), scales(), codes(), scales())

    @classmethod
    def wrap(cls, k_codes, k_scales, v_codes, v_scales):
        """A cache over the caller's own buffers (of the shapes above; not copied)."""
        self = cls.__new__(cls)
        _require(k_codes.dim() == 4 and k_scales.dim() == 5, "codes need 4 dimensions, scales 5")
        pages, heads, page_size, half = k_codes.shape
        ng = k_scales.shape[3]
        _require(ng > 0 and (2 * half) % ng == 0, "scales do not fit the codes")
        cls._check_shape(pages, page_size, heads, 2 * half, 2 * half // ng)
        for name, t in (("k_codes", k_codes), ("v_codes", v_codes)):
            _require(t.dtype == torch.uint8 and t.shape == k_codes.shape,
                     f"{name} must be uint8 of shape {tuple(k_codes.shape)}")
        for name, t in (("k_scales", k_scales), ("v_scales", v_scales)):
            _require(t.dtype == torch.bfloat16 and
                     tuple(t.shape) == (pages, heads, page_size, ng, 2),
                     f"{name} must be bfloat16 of shape {(pages, heads, page_size, ng, 2)}")
        for name, t in (("k_codes", k_codes), ("k_scales", k_scales), ("v_codes", v_codes),
                        ("v_scales", v_scales)):
            _require(t.is_contiguous() and t.data_ptr() % 16 == 0,
                     f"{name} must be contiguous and 16-byte aligned")
        _require(k_codes.is_cuda, "the state cache lives on a CUDA device")
        _same_device(k_codes.get_device(), k_scales, v_codes, v_scales)
        self._adopt(k_codes, k_scales, v_codes, v_scales)
        return self

    @staticmethod
    def _check_shape(pages, page_size, heads, head_dim, group):
        _require(pages > 0 and heads > 0, "a state cache needs pages and heads")
        _require(page_size > 0 and page_size & (page_size - 1) == 0 and page_size < 2 ** 31,
                 "page_size must be a power of two")
        _require(0 < head_dim <= 256 and head_dim % 8 == 0,
                 "head_dim must be a multiple of 8 up to 256")
        _require(group > 0 and group % 8 == 0 and head_dim % group == 0,
                 "group must be a multiple of 8 that divides head_dim")
        _require(heads * head_dim <= 2 ** 30, "heads * head_dim must be at most 2^30")

    # read-only: the library holds their addresses
    k_codes = property(lambda self: self._buffers[0])
    k_scales = property(lambda self: self._buffers[1])
    v_codes = property(lambda self: self._buffers[2])
    v_scales = property(lambda self: self._buffers[3])

    def _adopt(self, k_codes, k_scales, v_codes, v_scales):
        self._buffers = (k_codes, k_scales, v_codes, v_scales)
        self.num_pages, self.heads, self.page_size = k_codes.shape[:3]
        self.head_dim = 2 * k_codes.shape[3]
        self.group = self.head_dim // k_scales.shape[3]
        self.device = k_codes.device
        self._index = k_codes.get_device()
        self._c = _CCache(k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(),
                          v_scales.data_ptr(), self.num_pages, self.page_size, self.heads,
                          self.head_dim, self.group)
        self._ref = ctypes.addressof(self._c)
        self._room = {}
        with _on(self._index):
            check(lib.dgs_check_async_errors())  # makes the report words

    def _rows(self, k, v):
        shape = k.shape
        if len(shape) != 3 or shape[1] != self.heads or shape[2] != self.head_dim:
            raise RuntimeError(f"k must be [tokens, {self.heads}, {self.head_dim}]")
        if k.dtype not in _DTYPES:
            raise RuntimeError("k must be float32, bfloat16 or float16")
        if v.shape != shape or v.dtype is not k.dtype:
            raise RuntimeError("k and v must be alike")
        _no_grad(k, v)
        _same_device(self._index, k, v)
        return _rows16(k), _rows16(v)

    def write(self, k, v, slots):
        """Rows k[t], v[t] ([tokens, heads, head_dim]) go to flat slot slots[t]; a negative slot
        is skipped.  What a slot holds that a call names twice is not defined."""
        if slots.dim() != 1 or slots.numel() != k.shape[0]:
            raise RuntimeError("slots must be [tokens]")
        slots = _ids(slots, "slots")
        k, v = self._rows(k, v)
        _same_device(self._index, slots)
        with _on(self._index):
            s = slots if slots.dtype == torch.int64 else slots.long()
            check(lib.dgs_state_write(self._ref, k.data_ptr(), v.data_ptr(), _DTYPES[k.dtype],
                                      k.shape[0], k.stride(0), k.stride(1), v.stride(0),
                                      v.stride(1), s.data_ptr(), stream_ptr(self._index)))

    def append(self, k, v, table, lens):
        """One new row per sequence: k[i], v[i] go to slot lens[i] of table row i (page ids
        [sequences, pages]; lens is not changed).  Returns the flat slots (int64)."""
        n = k.shape[0]
        if table.dim() != 2 or table.shape[0] != n:
            raise RuntimeError("table must be [tokens, pages]")
        if n > 0 and table.shape[1] == 0:
            raise RuntimeError("the table has no columns")
        if lens.dim() != 1 or lens.numel() != n:
            raise RuntimeError("lens must be [tokens]")
        table, lens = _ids(table, "table"), _ids(lens, "lens")
        k, v = self._rows(k, v)
        _same_device(self._index, table, lens)
        with _on(self._index):
            slots = torch.empty_like(lens, dtype=torch.int64)
            check(lib.dgs_state_append(self._ref, k.data_ptr(), v.data_ptr(), _DTYPES[k.dtype],
                                       n, k.stride(0), k.stride(1), v.stride(0), v.stride(1),
                                       table.data_ptr(), table.element_size(), table.shape[1],
                                       lens.data_ptr(), lens.element_size(), slots.data_ptr(),
                                       stream_ptr(self._index)))
        return slots

    def read(self, slots, dtype=torch.float32):
        """The rows' values as (k, v), each [n, heads, head_dim]; a negative slot gives zeros."""
        if slots.dim() != 1:
            raise RuntimeError("slots must have one dimension")
        if dtype not in _DTYPES:
            raise RuntimeError("rows are read as float32, bfloat16 or float16")
        slots = _ids(slots, "slots")
        _same_device(self._index, slots)
        with _on(self._index):
            s = slots if slots.dtype == torch.int64 else slots.long()
            k = torch.empty((s.numel(), self.heads, self.head_dim), dtype=dtype,
                            device=self.device)
            v = torch.empty_like(k)
            check(lib.dgs_state_read(self._ref, s.data_ptr(), s.numel(), _DTYPES[dtype],
                                     k.data_ptr(), v.data_ptr(), stream_ptr(self._index)))
        return k, v

    def attend(self, q, table, lens, scale=None, weights=None, decay=1.0):
        """Attention of q [rows, q_heads, head_dim] (one query token a row; q_heads a multiple of
        heads, neighbouring query heads share a head) over the first lens[i] slots of table row i
        -> [rows, q_heads, head_dim]; a row of length 0, or with all its pages outside the cache,
        gives zeros.  scale: 1 / sqrt(head_dim) by default.  weights (float32 [rows, heads, >= pages *
        page_size], updated in place): weights[i, h, j] = decay * weights[i, h, j] + the probabilities
        of head h's query heads, for j < lens[i].  Several query tokens of one sequence are several
        rows with the same table row, each with the length that it may see."""
        if q.dim() != 3 or q.shape[2] != self.head_dim:
            raise RuntimeError(f"q must be [rows, q_heads, {self.head_dim}]")
        rows, q_heads = q.shape[0], q.shape[1]
        if q.dtype not in _DTYPES:
            raise RuntimeError("q must be float32, bfloat16 or float16")
        if q_heads == 0 or q_heads % self.heads:
            raise RuntimeError(f"q_heads must be a multiple of {self.heads}")
        if table.dim() != 2 or table.shape[0] != rows:
            raise RuntimeError("table must be [rows, pages]")
        if lens.dim() != 1 or lens.numel() != rows:
            raise RuntimeError("lens must be [rows]")
        table, lens = _ids(table, "table"), _ids(lens, "lens")
        width = table.shape[1]
        _no_grad(q)
        if weights is not None:
            if (weights.dtype != torch.float32 or weights.dim() != 3 or
                    weights.shape[:2] != (rows, self.heads) or
                    weights.shape[2] < width * self.page_size):
                raise RuntimeError(f"weights must be float32 [rows, {self.heads}, >= pages * "
                                   "page_size]")
            if not weights.is_contiguous():
                raise RuntimeError("weights must be contiguous (updated in place)")
            _no_grad(weights)
            _same_device(self._index, weights)
        _same_device(self._index, q, table, lens)
        scale = 1.0 / math.sqrt(self.head_dim) if scale is None else float(scale)
        q = _rows16(q)
        dt = _DTYPES[q.dtype]
        with _on(self._index):
            out = torch.empty((rows, q_heads, self.head_dim), dtype=q.dtype, device=self.device)
            if rows == 0:
                return out
            key = (rows, q_heads, width, weights is None, dt)
            room = self._room.get(key)
            if room is None:
                n = c_i64()
                check(lib.dgs_state_attend_workspace(self._ref, rows, q_heads, width,
                                                     int(weights is not None), dt,
                                                     ctypes.byref(n)))
                if len(self._room) >= 1024:
                    self._room.clear()
                room = self._room[key] = n.value
            ws = torch.empty(room, dtype=torch.uint8, device=self.device) if room else None
            check(lib.dgs_state_attend(
                self._ref, q.data_ptr(), dt, rows, q_heads, q.stride(0), q.stride(1),
                table.data_ptr(), table.element_size(), width, lens.data_ptr(),
                lens.element_size(), scale, None if weights is None else weights.data_ptr(),
                0 if weights is None else weights.shape[2], float(decay), out.data_ptr(),
                None if ws is None else ws.data_ptr(), room, stream_ptr(self._index)))
        return out

    def evict(self, weights, positions, table, lens, budget, sinks=0, recent=0):
        """evict_rows over this cache's buffers."""
        return evict_rows(self._buffers, weights, positions, table, lens, budget, sinks=sinks,
                          recent=recent)


_evict_room = {}  # workspace bytes by (rows, heads, cols, budget)


def evict_rows(stores, weights, positions, table, lens, budget, sinks=0, recent=0):
    """Eviction from a paged cache by accumulated attention weight.

    Every (row, head) with n = lens[row] > budget slots keeps the `budget` slots that come first by
    (protected, weight descending, slot ascending).  A slot is protected when its position is below
    `sinks` or among the `recent` highest (position >= highest + 1 - recent); sinks + recent may
    not exceed budget (positions may repeat: of more protected slots than stay the heaviest do).
    A NaN weight counts as the lowest.  The i-th dropped slot below budget
    receives the row of the i-th kept slot at or past it, in every tensor of `stores` ([pages,
    heads, page_size, ...], contiguous, any type; in place, at most 8).  Rows whose pages move must
    not share them: this is for sequences; tables of sampled neighbours share their nodes' pages.

    weights: float32 [rows, heads, cols], positions: int32 of that shape or None (position = slot),
    cols >= table.shape[1] * page_size.  Returns new (weights, positions, lens): the kept slots'
    weights and positions in their new order, 0 and -1 behind them, min(n, budget)."""
    if weights.dim() != 3 or weights.dtype != torch.float32:
        raise RuntimeError("weights must be float32 [rows, heads, slots]")
    rows, heads, cols = weights.shape
    if heads == 0:
        raise RuntimeError("weights must have heads")
    if positions is not None and (positions.dtype != torch.int32 or
                                  positions.shape != weights.shape):
        raise RuntimeError("positions must be int32 of the weights' shape")
    if table.dim() != 2 or table.shape[0] != rows:
        raise RuntimeError("table must be [rows, pages]")
    if lens.dim() != 1 or lens.numel() != rows:
        raise RuntimeError("lens must be [rows]")
    table, lens = _ids(table, "table"), _ids(lens, "lens")
    budget, sinks, recent = int(budget), int(sinks), int(recent)
    if budget <= 0:
        raise RuntimeError("budget must be positive")
    if sinks < 0 or recent < 0 or sinks + recent > budget:
        raise RuntimeError("sinks + recent must lie between 0 and budget")
    stores = list(stores)
    if not 0 < len(stores) <= 8:
        raise RuntimeError("evict_rows takes one to eight stores")
    lead = stores[0].shape[:3]
    if len(lead) != 3 or lead[0] == 0 or lead[1] != heads or lead[2] == 0:
        raise RuntimeError(f"a store must be [pages, {heads}, page_size, ...]")
    pages, _, page = lead
    slots, width = pages * heads * page, table.shape[1]
    ptrs, nbytes = [], []
    for s in stores:
        if s.shape[:3] != lead:
            raise RuntimeError("the stores must have the same pages")
        size = s.numel()
        if size == 0 or not s.is_contiguous():
            raise RuntimeError("a store must be contiguous and not empty")
        ptrs.append(s.data_ptr())
        nbytes.append(size // slots * s.element_size())
    if cols < width * page:
        raise RuntimeError("weights need a column for every slot of the table")
    _no_grad(weights, *stores)
    if not weights.is_cuda:
        raise RuntimeError("weights must be a CUDA tensor")
    index, device = weights.get_device(), weights.device
    _same_device(index, table, lens, *stores)
    if positions is not None:
        _same_device(index, positions)
    with _on(index):
        w = weights if weights.is_contiguous() else weights.contiguous()
        p = positions
        if p is not None and not p.is_contiguous():
            p = p.contiguous()
        new_w = torch.empty_like(w)
        new_p = torch.empty_like(w, dtype=torch.int32) if p is None else torch.empty_like(p)
        new_lens = torch.empty_like(lens)
        if rows == 0:
            return new_w, new_p, new_lens
        key = (rows, heads, cols, budget)
        room = _evict_room.get(key)
        if room is None:
            n = c_i64()
            check(lib.dgs_evict_workspace(rows, heads, cols, budget, ctypes.byref(n)))
            if len(_evict_room) >= 1024:
                _evict_room.clear()
            room = _evict_room[key] = n.value
        ws = torch.empty(room, dtype=torch.uint8, device=device) if room else None
        n = len(stores)
        check(lib.dgs_evict_rows(
            (c_vp * n)(*ptrs), (c_i64 * n)(*nbytes), n, pages, heads, page, w.data_ptr(),
            None if p is None else p.data_ptr(), new_w.data_ptr(), new_p.data_ptr(), rows, cols,
            table.data_ptr(), table.element_size(), width, lens.data_ptr(),
            lens.element_size(), new_lens.data_ptr(), budget, sinks, recent,
            None if ws is None else ws.data_ptr(), room, stream_ptr(index)))
    return new_w, new_p, new_lens


def neighbour_table(block, fan_out):
    """The table and lengths that StateCache.attend takes (pages of one slot, page = node id) for a
    block of the sampler (seeds, frontier, coo_row, coo_col): table row i = the sampled neighbours
    of the block's i-th target node, the first `fan_out` if there are more, -1 behind them.  No
    synchronisation."""
    seeds, frontier, row, col = block
    _require(fan_out > 0, "fan_out must be positive")
    row, col = row.long(), col.long()
    lens = torch.zeros(seeds.numel(), dtype=torch.int64, device=row.device)
    lens.scatter_add_(0, row, torch.ones_like(row))
    # a block's edges are grouped by target, in target order; what passes fan_out goes to a column
    # that is cut off
    at = torch.arange(row.numel(), device=row.device) - (lens.cumsum(0) - lens)[row]
    table = torch.full((seeds.numel(), fan_out + 1), -1, dtype=torch.int64, device=row.device)
    table[row, at.clamp(max=fan_out)] = frontier.long()[col]
    return table[:, :fan_out].contiguous(), lens.clamp(max=fan_out)
