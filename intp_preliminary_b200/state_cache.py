"""The 8-bit cache of an encoder's key / value states, and attention over it.

A state's row of D values (one sequence, one key head) is held as e4m3 codes
and one exponent byte (1 to 254) and stands for ``code * 2^(byte - 127)``; the power of
two is the smallest whose 448-fold (e4m3's largest value) reaches the row's
largest finite value, no smaller than 2^-126.  So a value that is normal in
e4m3 is off by at most 2^-4 of itself, and a row costs D + 1 bytes instead of
2 D.  Infinities and NaN become NaN.
"""

from __future__ import annotations

import struct

import torch

from . import _lib
from .cross_attention import (_base_args, _call, _check_counts, _check_query, _check_scale, _finish_plan, _keep,
                              _laid_out, _launch, _lengths_pointer, _output, _plans, _ready, _refuse_grad)
from .look_attention import _DTYPE_CODE, _refuse_transforms

_POINTERS = struct.Struct("8Q")  # state_cache_args up to the sizes
_HALF = (torch.bfloat16, torch.float16)


def _check_tensors(keys, key_exponents, values, value_exponents) -> None:
    tensors = (keys, values, key_exponents, value_exponents)
    if not all(t.is_cuda for t in tensors):
        raise ValueError("a state cache requires CUDA tensors")
    if keys.ndim != 4 or keys.shape != values.shape:
        raise ValueError("keys and values must share shape (B, G, C, D)")
    if key_exponents.shape != keys.shape[:3] or value_exponents.shape != keys.shape[:3]:
        raise ValueError("the exponents must have shape (B, G, C)")
    if keys.dtype != torch.float8_e4m3fn or values.dtype != torch.float8_e4m3fn:
        raise ValueError("keys and values must be float8_e4m3fn")
    if key_exponents.dtype != torch.uint8 or value_exponents.dtype != torch.uint8:
        raise ValueError("the exponents must be uint8")
    if keys.shape[3] % 16 or not 16 <= keys.shape[3] <= 128:
        raise ValueError("head_dim must be a multiple of 16 up to 128")
    if not all(t.is_contiguous() for t in tensors):
        raise ValueError("the cache's tensors must be contiguous, codes 16-byte aligned")
    if len({t.device for t in tensors}) != 1:
        raise ValueError("all tensors must be on the same CUDA device")


class StateCache:
    """Codes ``keys``, ``values`` ``(B, G, C, D)`` float8_e4m3fn and exponent bytes
    ``key_exponents``, ``value_exponents`` ``(B, G, C)`` uint8, all contiguous, of
    C states per sequence and key head; D a multiple of 16 up to 128.

    The cache does not know how many of its states are filled: a program keeps
    its sequences' lengths and passes them (``start`` of a write, ``lengths`` of
    the attention).  Its tensors may be written to but not replaced: other tensors
    are another ``StateCache``, which costs no copy."""

    def __init__(self, keys, key_exponents, values, value_exponents) -> None:
        for t in (keys, key_exponents, values, value_exponents):
            if not isinstance(t, torch.Tensor):
                raise ValueError("a state cache requires CUDA tensors")
        # what the tensors' layout decides is checked once and known by it
        self._layout = (keys.shape, keys.stride(), keys.dtype, keys.device, values.shape, values.stride(), values.dtype,
                       values.device, key_exponents.shape, key_exponents.stride(), key_exponents.dtype,
                       key_exponents.device, value_exponents.shape, value_exponents.stride(), value_exponents.dtype,
                       value_exponents.device)
        if self._layout not in _plans:
            _check_tensors(keys, key_exponents, values, value_exponents)
            _keep(self._layout, None)
        if (keys.data_ptr() | values.data_ptr()) & 15:
            raise ValueError("the cache's tensors must be contiguous, codes 16-byte aligned")
        self._keys, self._values = keys, values
        self._key_exponents, self._value_exponents = key_exponents, value_exponents

    # read only: a call takes the layout that was checked above
    keys = property(lambda self: self._keys)
    values = property(lambda self: self._values)
    key_exponents = property(lambda self: self._key_exponents)
    value_exponents = property(lambda self: self._value_exponents)
    layout = property(lambda self: self._layout)

    @classmethod
    def empty(cls, batch: int, groups: int, capacity: int, head_dim: int, *, device) -> "StateCache":
        """A cache of zeros."""
        shape = (batch, groups, capacity, head_dim)
        codes = [torch.zeros(shape, dtype=torch.float8_e4m3fn, device=device) for _ in range(2)]
        exponents = [torch.full(shape[:3], 127, dtype=torch.uint8, device=device) for _ in range(2)]
        return cls(codes[0], exponents[0], codes[1], exponents[1])

    @property
    def device(self) -> torch.device:
        return self.keys.device

    @property
    def shape(self) -> tuple[int, ...]:
        return tuple(self.keys.shape)

    def _tail(self, k, v, key) -> bytes:
        """The argument block of a copy between ``k``, ``v`` and this cache, behind its pointers."""
        args = _lib.StateCacheArgs()
        args.batch, args.groups, args.capacity, args.head_dim = self.keys.shape
        args.count = k.shape[2]
        args.dtype = _DTYPE_CODE[k.dtype]
        args.k_stride, args.v_stride = k.stride(), v.stride()
        return _keep(key, bytes(args)[_POINTERS.size:])

    def _copy(self, fn, tail: bytes, k, v, start, counts, what: str) -> None:
        keys = self.keys
        device = keys.device
        start_p = counts_p = 0
        if start is not None:
            start = _check_counts(start, keys.shape[0], device, "start")
            start_p = start.data_ptr()
        if counts is not None:
            counts = _check_counts(counts, keys.shape[0], device, "counts")
            counts_p = counts.data_ptr()
        block = _POINTERS.pack(k.data_ptr(), v.data_ptr(), start_p, counts_p, keys.data_ptr(),
                               self.key_exponents.data_ptr(), self.values.data_ptr(), self.value_exponents.data_ptr())
        _call(fn, block + tail, device.index, what)

    def _check_pair(self, k, v) -> None:
        batch, groups, _, head_dim = self.keys.shape
        for t in (k, v):
            if not isinstance(t, torch.Tensor) or not t.is_cuda:
                raise ValueError("a state cache requires CUDA tensors")
            if t.ndim != 4 or t.shape != k.shape or (t.shape[0], t.shape[1], t.shape[3]) != (batch, groups, head_dim):
                raise ValueError("k and v must share shape (B, G, n, D) with the cache's B, G and D")
            if t.dtype not in _HALF or t.dtype != k.dtype:
                raise ValueError("k and v must be bfloat16 or float16 and share a dtype")
            if t.device != self.keys.device:
                raise ValueError("all tensors must be on the same CUDA device")

    def write(self, k, v, *, start=None, counts=None) -> None:
        """Quantise ``k``, ``v`` ``(B, G, n, D)`` (bf16 or f16) into the cache: row i of
        sequence b goes to state ``start[b] + i`` (``start`` ``(B,)``, zero without
        it) for ``i < counts[b]`` (all n without it).  Rows that fall outside the
        cache are skipped; every other state is left as it was."""
        if not (isinstance(k, torch.Tensor) and isinstance(v, torch.Tensor)):
            raise ValueError("a state cache requires CUDA tensors")
        _refuse_grad("a state cache", k, v)
        key = (self.layout, k.shape, k.stride(), k.dtype, k.device, v.shape, v.stride(), v.dtype, v.device)
        tail = _plans.get(key)
        if tail is None or (k.data_ptr() | v.data_ptr()) & 15:
            self._check_pair(k, v)
            k, v = _laid_out(k), _laid_out(v)
            key = (self.layout, k.shape, k.stride(), k.dtype, k.device, v.shape, v.stride(), v.dtype, v.device)
            tail = _plans.get(key) or self._tail(k, v, key)
        self._copy(_lib.load().state_cache_write, tail, k, v, start, counts, "state cache write")

    def read(self, count: int | None = None, *, start=None, counts=None, dtype=torch.bfloat16):
        """The values of ``count`` states per sequence (all C without it) from state
        ``start[b]`` on, as ``(k, v)`` ``(B, G, count, D)``: exact, but for what lies
        past the dtype's range (its largest value instead) or below it.  States past
        ``counts[b]`` or outside the cache read as zero."""
        _refuse_transforms("a state cache")
        batch, groups, capacity, head_dim = self.keys.shape
        count = capacity if count is None else int(count)
        if count < 0:
            raise ValueError("count must not be negative")
        if dtype not in _HALF:
            raise ValueError("dtype must be bfloat16 or float16")
        shape, device = (batch, groups, count, head_dim), self.keys.device
        k = torch.empty(shape, dtype=dtype, device=device)
        v = torch.empty(shape, dtype=dtype, device=device)
        key = (self.layout, count, dtype)
        tail = _plans.get(key) or self._tail(k, v, key)
        self._copy(_lib.load().state_cache_read, tail, k, v, start, counts, "state cache read")
        return k, v

    def _set_states(self, args) -> None:
        _, args.groups, args.states, _ = self.keys.shape
        args.k_stride, args.v_stride = self.keys.stride(), self.values.stride()
        args.eight_bit = 1
        strides = self.key_exponents.stride()
        args.exponent_stride[0], args.exponent_stride[1] = strides[0], strides[1]


def _cached_plan(q, cache: StateCache, scale, out_stride):
    key = (cache.layout, q.shape, q.stride(), q.dtype, q.device, scale, out_stride)
    plan = _plans.get(key)
    if plan is None:
        _check_query(q, cache.keys.shape[1], cache.keys.shape[3], "cached cross attention", 16)
        if q.device != cache.device:
            raise ValueError("all tensors must be on the same CUDA device")
        if q.shape[0] != cache.keys.shape[0]:
            raise ValueError("q and the cache must share the batch size")
        if cache.keys.shape[2] < 1:
            raise ValueError("the cache must hold at least one state")
        scale = _check_scale(scale)
        if not _ready(q):
            return None
        args = _base_args(q, scale, out_stride, "auto")
        cache._set_states(args)
        plan = _keep(key, _finish_plan(args, q, "cached cross attention"))
    return plan


def cached_cross_attention(q, cache, *, scale, lengths=None, out=None):
    """``cross_attention`` of ``q`` ``(B, H, M, D)`` over a :class:`StateCache`, whose
    codes are widened inside the kernel: a state is read once for every 16 rows of
    its key head.  Made for new tokens (few rows); inference only.  ``lengths``
    counts each sequence's filled states (the whole capacity without it)."""
    what = "cached cross attention"
    if not isinstance(cache, StateCache):
        raise ValueError("cache must be a StateCache")
    if not isinstance(q, torch.Tensor):
        raise ValueError(f"{what} requires CUDA tensors")
    _refuse_grad(what, q)
    scale = float(scale)
    out_stride = None
    if out is not None:
        out_stride = _output(q, out).stride()
    elif q.ndim == 4:
        _, h, m, d = q.shape
        out_stride = (h * m * d, m * d, d, 1)
    plan = _cached_plan(q, cache, scale, out_stride)
    if plan is None or q.data_ptr() & 15:
        q = _laid_out(q)
        plan = _cached_plan(q, cache, scale, out_stride)
    lengths, lengths_p = _lengths_pointer(lengths, plan, "lengths")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=plan.device)
    _launch(plan, what, q.data_ptr(), cache.keys.data_ptr(), cache.values.data_ptr(), cache.key_exponents.data_ptr(),
            cache.value_exponents.data_ptr(), 0, 0, lengths_p, out.data_ptr(), 0)
    return out
