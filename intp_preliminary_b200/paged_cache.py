"""A paged cache of a decoder's own keys and values, and attention over it.

The cache is a pool of pages, each ``page_size`` states of every key head; a page
table names each sequence's pages, so sequences grow without moving and may share
pages.  State p of sequence b is row ``p % page_size`` of page
``page_table[b, p // page_size]``.  Entries that are no page of the pool (-1 for
instance) hold nothing: rows that belong there are not written and states there
take no part in the attention.

The cache does not know how many states a sequence has: a program keeps each
sequence's length and passes it as ``start``, the position of the first new row.
A step appends its keys and values there and attends from there:

    q = cache.append(k, v, page_table=table, start=length, rotary=rotary, q=q)
    out = paged_attention(q, cache, page_table=table, start=length, scale=scale)

The operators take no part in autograd.  An append is one CUDA kernel of
``libintp_b200.so``, an attention one or two (see ``paged_attention``), on the
current stream; inputs that are not laid out for them are copied first, and int64
``start``, ``counts`` and ``page_table`` converted to 32 bits (values past those
become the nearest) in every call.  CPU tensors raise ``ValueError``.
"""

from __future__ import annotations

import struct

import torch

from . import _lib
from .cross_attention import (_HALF, _MAX_STRIDE, _call, _check_counts, _check_scale, _keep, _laid_out, _output, _plans,
                              _ready, _refuse_grad, _scratch_bytes)
from .look_attention import _DTYPE_CODE
from .rotary import (_POINTERS, RotaryAxes, _check_heads, _check_positions, _check_rotary, _grad_enabled, _rows_laid_out,
                     _set_rotary, _unusual)

_ATTENTION_POINTERS = struct.Struct("9Q")  # paged_attention_args up to the sizes
_MAX_STATES = 1 << 30
_MAX_SPAN = 1 << 35  # elements: 2^32 units of 16 bytes
_KERNELS = {"auto": _lib.PAGED_KERNEL_AUTO, "joined": _lib.PAGED_KERNEL_JOINED, "parts": _lib.PAGED_KERNEL_PARTS}


def _check_cache(keys, values) -> None:
    for t in (keys, values):
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise ValueError("a paged cache requires CUDA tensors")
    if keys.ndim != 4 or keys.shape != values.shape:
        raise ValueError("keys and values must share shape (pages, G, page_size, D)")
    if keys.dtype not in _HALF or values.dtype != keys.dtype:
        raise ValueError("keys and values must be bfloat16 or float16 and share a dtype")
    if keys.device != values.device:
        raise ValueError("all tensors must be on the same CUDA device")
    if min(keys.shape[:3]) < 1:
        raise ValueError("a paged cache needs a page, a key head and a state")
    if keys.shape[3] % 8 or not 8 <= keys.shape[3] <= 128:
        raise ValueError("head_dim must be a multiple of 8 up to 128")
    if keys.requires_grad or values.requires_grad:
        raise ValueError("a paged cache takes no part in autograd: detach its tensors")
    if not (_ready(keys) and _ready(values)):
        raise ValueError("the cache's tensors need unit stride on head_dim and 16-byte aligned rows")
    if keys.stride() != values.stride():
        raise ValueError("keys and values must share their strides")
    if sum((n - 1) * s for n, s in zip(keys.shape, keys.stride())) >= _MAX_SPAN:
        raise ValueError("a paged cache's keys may span 64 GB at most, and its values too")


class PagedCache:
    """``keys`` and ``values`` ``(pages, G, page_size, D)`` bf16 or f16 of the pool's
    pages, any page size from one up, D a multiple of 8 up to 128.  Outer strides are free
    (multiples of 16 bytes, the same for both): a pool laid out ``(pages, page_size, G, D)``
    is passed transposed.  The tensors may be written to but not replaced."""

    def __init__(self, keys, values) -> None:
        _check_cache(keys, values)
        self._keys, self._values = keys, values
        # what calls know the pool by
        self._layout = (keys.shape, keys.stride(), keys.dtype, keys.device)

    def __setstate__(self, state: dict) -> None:
        """A copy, and what is loaded from a file, is checked again: its tensors may lie elsewhere."""
        self.__dict__.update(state)
        PagedCache.__init__(self, self._keys, self._values)

    # read only: a call takes the layout that was checked above
    keys = property(lambda self: self._keys)
    values = property(lambda self: self._values)
    layout = property(lambda self: self._layout)

    @classmethod
    def empty(cls, pages: int, groups: int, page_size: int, head_dim: int, *, dtype=torch.bfloat16,
              device) -> "PagedCache":
        """A pool of zeros."""
        return cls(*(torch.zeros(pages, groups, page_size, head_dim, dtype=dtype, device=device) for _ in range(2)))

    @property
    def device(self) -> torch.device:
        return self._keys.device

    @property
    def shape(self) -> tuple[int, ...]:
        return tuple(self._keys.shape)

    def _append_plan(self, q, k, v, page_table, start, counts, rotary, positions) -> bytes:
        """Checks an append of laid out tensors; its argument block behind the pointers."""
        args = _lib.RotaryArgs()
        args.batch, args.groups, args.rows, args.head_dim = k.shape
        args.k_stride, args.v_stride = k.stride(), v.stride()
        args.k_out_stride = args.v_out_stride = self._keys.stride()
        if q is not None:
            args.heads = q.shape[1]
            args.q_stride, args.q_out_stride = q.stride(), torch.empty_like(q, device="meta").stride()
        args.pages, _, args.page_size, _ = self._keys.shape
        args.table_width, args.table_stride = page_table.shape[1], page_table.stride(0)
        args.dtype = _DTYPE_CODE[k.dtype]
        if rotary is not None:
            _set_rotary(args, rotary, positions)
        return bytes(args)[_POINTERS.size:]

    def _append_inputs(self, q, k, v, page_table, start, counts, rotary, positions):
        """Checks a call and returns its tensors as the kernel takes them."""
        what = "a paged cache"
        _, groups, page_size, head_dim = self._keys.shape
        for name, t in (("k", k), ("v", v), ("q", q)):
            if t is None:
                continue
            _check_heads(t, name, what, _HALF)
            if t.dtype != self._keys.dtype or t.device != self._keys.device:
                raise ValueError(f"{name} must have the cache's dtype and device")
            if t.shape[0] != k.shape[0] or t.shape[2:] != (k.shape[2], head_dim) or (name != "q" and t.shape[1] != groups):
                raise ValueError("k and v must have shape (B, G, n, D) and q (B, H, n, D) with the cache's G and D")
        batch, device = k.shape[0], k.device
        page_table = _table(page_table, batch, page_size, device)
        if rotary is not None:
            _check_rotary(rotary, head_dim, device)
            if positions is not None:
                _check_positions(positions, batch, k.shape[2], max(rotary.axes) + 1, device)
        elif q is not None or positions is not None:
            raise ValueError("q and positions are for a rotation: pass rotary too")
        return (None if q is None else _rows_laid_out(q), _rows_laid_out(k), _rows_laid_out(v), page_table,
                _check_counts(start, batch, device, "start"), _check_counts(counts, batch, device, "counts"))

    def append(self, k, v, *, page_table, start, counts=None, rotary=None, positions=None, q=None):
        """Row i of ``k``, ``v`` ``(B, G, n, D)`` to state ``start[b] + i`` of sequence b for
        ``i < counts[b]`` (all n without it); rows outside the table or without a page are
        skipped, and every other row of the pool is left as it was.

        With ``rotary`` (a :class:`~intp_preliminary_b200.RotaryAxes`) the keys are turned
        on the way, by ``positions`` ``(B, n, axes)`` or ``(n, axes)``, or without them by
        the state's number on every axis; ``q`` ``(B, H, n, D)`` is turned likewise, every
        row of it, and returned.  Two rows that go to the same row of the pool leave it
        unspecified, and so do inputs that overlap the rows they are written to."""
        if rotary is not None and not isinstance(rotary, RotaryAxes):
            raise ValueError("rotary must be a RotaryAxes")
        try:
            if _unusual() or (_grad_enabled() and (k.requires_grad or v.requires_grad or (q is not None and q.requires_grad)
                                                   or (positions is not None and positions.requires_grad)
                                                   or self._keys.requires_grad or self._values.requires_grad)):
                _refuse_grad("a paged cache", k, v, q, positions, self._keys, self._values)
            key = ("append", self._layout, k.shape, k.stride(), k.dtype, k.device, v.shape, v.stride(), v.dtype, v.device,
                   page_table.shape, page_table.stride(), page_table.dtype, page_table.device, start.shape,
                   start.stride(), start.dtype, start.device,
                   None if q is None else (q.shape, q.stride(), q.dtype, q.device),
                   None if counts is None else (counts.shape, counts.stride(), counts.dtype, counts.device),
                   None if rotary is None else rotary._layout,
                   None if positions is None else (positions.shape, positions.stride(), positions.dtype, positions.device))
        except (AttributeError, TypeError):
            _check_tensors("a paged cache", k, v, page_table, start, q, counts, positions)
            raise
        tail = _plans.get(key)
        k_at, v_at, q_at = k.data_ptr(), v.data_ptr(), 0 if q is None else q.data_ptr()
        if tail is None or (k_at | v_at | q_at) & 15:
            given = (q, k, v, page_table, start, counts)
            taken = self._append_inputs(*given, rotary, positions)
            if any([a is not b for a, b in zip(given, taken)]):
                q, k, v, page_table, start, counts = taken
                return self.append(k, v, page_table=page_table, start=start, counts=counts, rotary=rotary,
                                   positions=positions, q=q)
            tail = _keep(key, self._append_plan(*given, rotary, positions))
        q_out, q_to = None, 0
        if q is not None:
            q_out = torch.empty_like(q)
            q_to = q_out.data_ptr()
        turns, axis = (0, 0) if rotary is None else rotary._launch_pointers()
        block = _POINTERS.pack(q_at, k_at, v_at, q_to, self._keys.data_ptr(), self._values.data_ptr(), turns, axis,
                               0 if positions is None else positions.data_ptr(), start.data_ptr(),
                               0 if counts is None else counts.data_ptr(), page_table.data_ptr()) + tail
        _call(_lib.load().paged_cache_append, block, self._keys.device.index, "paged cache append")
        return q_out


def _check_tensors(what: str, *tensors) -> None:
    """Says which of a call's arguments is no tensor; from the fifth on they may be None."""
    what = f"{what} requires CUDA tensors"
    messages = (what, what, "page_table must be an int32 or int64 tensor of shape (B, width)",
                "start must be an int32 or int64 tensor of shape (B,)", what,
                "counts must be an int32 or int64 tensor of shape (B,)", "positions must be a tensor")
    for i, (t, message) in enumerate(zip(tensors, messages)):
        if not (isinstance(t, torch.Tensor) or (i > 3 and t is None)):
            raise ValueError(message)


def _table(page_table, batch: int, page_size: int, device) -> torch.Tensor:
    """The page table as the kernels take it: int32, unit stride along a sequence's pages."""
    if page_table.ndim != 2 or page_table.dtype not in (torch.int32, torch.int64):
        raise ValueError("page_table must be an int32 or int64 tensor of shape (B, width)")
    if page_table.shape[0] != batch:
        raise ValueError("page_table must have a row for each sequence")
    if page_table.shape[1] < 1 or page_table.shape[1] * page_size > _MAX_STATES:
        raise ValueError("page_table must name at least one page and at most 2^30 states a sequence")
    if page_table.device != device:
        raise ValueError("page_table must be on the same CUDA device as q")
    if page_table.dtype == torch.int64:
        page_table = page_table.clamp(-1, 2147483647).to(torch.int32)
    strides = page_table.stride()
    if (strides[1] != 1 and page_table.shape[1] > 1) or not 0 <= strides[0] < _MAX_STRIDE:
        page_table = page_table.contiguous()
    return page_table


def _attention_inputs(q, cache: PagedCache, page_table, start, counts, out):
    """Checks a call and returns its tensors as the kernels take them."""
    what = "paged attention"
    _check_heads(q, "q", what, _HALF)
    _, groups, page_size, head_dim = cache._keys.shape
    if q.dtype != cache._keys.dtype or q.device != cache._keys.device:
        raise ValueError("q must have the cache's dtype and device")
    if q.shape[3] != head_dim:
        raise ValueError("q and the cache must share head_dim")
    if q.shape[1] < 1 or q.shape[1] % groups:
        raise ValueError("the query heads must be a multiple of the key heads")
    if out is not None:
        _output(q, out)
    return (_laid_out(q), _table(page_table, q.shape[0], page_size, q.device),
            _check_counts(start, q.shape[0], q.device, "start"), _check_counts(counts, q.shape[0], q.device, "counts"))


def _attention_plan(q, cache: PagedCache, page_table, scale, window, sinks, kernel, out):
    """Checks the numbers of a call; its argument block behind the pointers, its scratch bytes."""
    if window is not None and not 1 <= window <= _MAX_STATES:
        raise ValueError("window must be at least 1 (None: the whole sequence)")
    if not 0 <= sinks <= _MAX_STATES:
        raise ValueError("sinks must not be negative")
    if sinks and window is None:
        raise ValueError("sinks are the states that stay visible beside a window: pass window too")
    if kernel not in _KERNELS:
        raise ValueError(f"kernel must be one of {sorted(_KERNELS)}")
    args = _lib.PagedAttentionArgs()
    args.batch, args.heads, args.queries, args.head_dim = q.shape
    args.pages, args.groups, args.page_size, _ = cache._keys.shape
    args.q_stride = q.stride()
    args.out_stride = (torch.empty_like(q, device="meta") if out is None else out).stride()
    args.cache_stride = cache._keys.stride()
    args.table_width, args.table_stride = page_table.shape[1], page_table.stride(0)
    args.window, args.sinks = window or 0, sinks
    args.scale = _check_scale(scale)
    args.dtype = _DTYPE_CODE[q.dtype]
    args.kernel = _KERNELS[kernel]
    scratch = _scratch_bytes(_lib.load().paged_attention_workspace, args, "paged attention")
    return bytes(args)[_ATTENTION_POINTERS.size:], scratch


def paged_attention(q, cache, *, page_table, start, scale, counts=None, window=None, sinks: int = 0,
                    kernel: str = "auto", out=None):
    """Attention of the new tokens ``q`` ``(B, H, M, D)`` over a :class:`PagedCache`.

    Row m of sequence b stands at position ``start[b] + m`` and sees the states up to
    and with its own; with ``window`` only the last ``window`` of them, and the
    sequence's first ``sinks`` states.  Query head h reads key head ``h // (H / G)``.
    Rows from ``counts[b]`` on (all M count without it) and rows that see nothing give
    zeros; states that a row does not see take no part whatever they hold.  The result
    is laid out like ``q`` unless ``out`` is given.

    Made for few rows: the states are read once for every 16 rows (tokens times
    ``H / G``) of a key head.  fp32 sums and statistics; the result is rounded once.
    ``kernel``: ``"auto"`` chooses; ``"joined"`` (a cluster of CTAs for each sequence and key
    head, one launch) and ``"parts"`` (equal shares of the batch's states, joined by a second
    launch; at most 16 rows) force one of the two."""
    what = "paged attention"
    if not isinstance(cache, PagedCache):
        raise ValueError("cache must be a PagedCache")
    try:
        if _unusual() or (_grad_enabled() and (q.requires_grad or cache._keys.requires_grad or cache._values.requires_grad
                                               or (out is not None and out.requires_grad))):
            _refuse_grad(what, q, cache._keys, cache._values, out)
        device = q.device
        key = ("attend", cache._layout, q.shape, q.stride(), q.dtype, device, page_table.shape, page_table.stride(),
               page_table.dtype, page_table.device, start.shape, start.stride(), start.dtype, start.device,
               None if counts is None else (counts.shape, counts.stride(), counts.dtype, counts.device), float(scale),
               None if window is None else int(window), int(sinks), kernel,
               None if out is None else (out.shape, out.stride(), out.dtype, out.device))
    except (AttributeError, TypeError):
        _check_tensors(what, q, q, page_table, start, None, counts)
        if out is not None:
            _output(q, out)
        raise
    plan = _plans.get(key)
    if plan is None or (q.data_ptr() | (0 if out is None else out.data_ptr())) & 15:
        given = (q, page_table, start, counts)
        taken = _attention_inputs(q, cache, page_table, start, counts, out)
        if any([a is not b for a, b in zip(given, taken)]):
            q, page_table, start, counts = taken
            return paged_attention(q, cache, page_table=page_table, start=start, scale=scale, counts=counts, window=window,
                                   sinks=sinks, kernel=kernel, out=out)
        plan = _keep(key, _attention_plan(q, cache, page_table, float(scale), None if window is None else int(window),
                                          int(sinks), kernel, out))
    tail, scratch_bytes = plan
    if out is None:
        out = torch.empty_like(q)
    space = 0
    if scratch_bytes:
        scratch = torch.empty(scratch_bytes, dtype=torch.uint8, device=device)  # from the current stream's pool
        space = scratch.data_ptr()
    block = _ATTENTION_POINTERS.pack(q.data_ptr(), cache._keys.data_ptr(), cache._values.data_ptr(), out.data_ptr(),
                                     page_table.data_ptr(), start.data_ptr(), 0 if counts is None else counts.data_ptr(),
                                     space, scratch_bytes) + tail
    _call(_lib.load().paged_attention, block, device.index, what)
    return out
