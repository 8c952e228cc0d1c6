"""Queries and keys turned by their positions, which may have several axes.

``RotaryAxes`` says which axis turns each pair of a head's columns and how fast;
``rotate_positions(q, k, rotary=..., positions=...)`` turns the pairs:

    t = positions[b, n, axes[i]] * frequencies[i]                 (64 bits)
    y1 = x1 cos t - x2 sin t,   y2 = x2 cos t + x1 sin t          (32 bits), cast to x.dtype

Pair i of the first R = 2 * len(frequencies) columns is columns i and R/2 + i, or
2i and 2i + 1 with ``interleaved``; columns past R pass unchanged.  An axis is
whatever the positions count: a token's place in its sequence, a video's time,
height and width, the coordinates of a patch on the hex lattice.

The operator is differentiable in q and k, any number of times (a gradient is
turned back by the same angles); results repeat bit for bit.  Forward-mode
tangents and ``torch.jit.trace`` are refused.  Every call runs one CUDA kernel of
``libintp_b200.so`` on the current stream of the inputs' device, behind a copy of
each input whose rows are not laid out for it; there is no CPU path, CPU tensors
raise ``ValueError``.
"""

from __future__ import annotations

import math
import struct

import torch
from torch.autograd import forward_ad

from . import _lib
from .cross_attention import _MAX_STRIDE, _call, _current_stream, _keep, _plans
from .look_attention import _DTYPE_CODE, _refuse_transforms

_POINTERS = struct.Struct("12Q")  # rotary_args up to the sizes
_POSITION_TYPES = {torch.int32: _lib.ROTARY_INT32, torch.int64: _lib.ROTARY_INT64, torch.float32: _lib.ROTARY_FLOAT32}
_MAX_PAIRS = 64
_grad_enabled = torch.is_grad_enabled
_tracing = torch._C._get_tracing_state


def _unusual() -> bool:
    """Whether forward-mode tangents or a trace may be about, which the kernels know nothing of."""
    return forward_ad._current_level >= 0 or _tracing() is not None


class RotaryAxes:
    """The turning of a head's pairs: ``frequencies[i]`` radians for each step along
    axis ``axes[i]``, of as many pairs as there are entries, a multiple of 4 up to 64.
    The axes are numbered from 0 without gaps; ``interleaved`` pairs neighbouring
    columns.  The object holds its tables on ``device`` and does not change; a copy, or one that
    is unpickled, has tables of its own.  A CUDA graph that was captured with it reads them:
    keep it as long."""

    def __init__(self, frequencies, axes, *, interleaved: bool = False, device) -> None:
        frequencies, axes = [float(f) for f in frequencies], [int(a) for a in axes]
        if len(frequencies) != len(axes):
            raise ValueError("frequencies and axes must have the same length")
        if len(axes) % 4 or not 4 <= len(axes) <= _MAX_PAIRS:
            raise ValueError(f"the number of pairs must be a multiple of 4 up to {_MAX_PAIRS}")
        if not all(math.isfinite(f) for f in frequencies):
            raise ValueError("frequencies must be finite")
        if min(axes) < 0 or set(axes) != set(range(max(axes) + 1)):
            raise ValueError("axes must be numbered from 0 without gaps")
        self._device = torch.device(device)
        if self._device.type != "cuda":
            raise ValueError("rotary positions require a CUDA device")
        self._frequencies, self._axes = tuple(frequencies), tuple(axes)
        self._interleaved = bool(interleaved)
        self._lay_out()

    def _lay_out(self) -> None:
        """The tables on the device, in one copy: turns (64 bits), then axes (32 bits)."""
        pairs = len(self._axes)
        tables = bytearray(struct.pack(f"{pairs}d{pairs}i", *(f / (2 * math.pi) for f in self._frequencies), *self._axes))
        self._tables = torch.frombuffer(tables, dtype=torch.uint8).to(self._device)
        self._device = self._tables.device
        self._index, self._turn_bytes = self._device.index, 8 * pairs
        # streams that the tables' memory is held for: the one it was allocated on
        self._streams = {_current_stream(self._index)} if self._tables.is_cuda else set()
        # what a call's checks and argument block depend on
        self._layout = (pairs, max(self._axes) + 1, self._interleaved, self._device)

    @property
    def _pointers(self) -> tuple[int, int]:
        at = self._tables.data_ptr()
        return at, at + self._turn_bytes

    def _launch_pointers(self) -> tuple[int, int]:
        """The tables' addresses for a launch on the device's current stream: should the object go while
        the launch is pending, its memory waits for that stream."""
        stream = _current_stream(self._index)
        if stream not in self._streams:
            self._tables.record_stream(torch.cuda.current_stream(self._device))
            self._streams.add(stream)
        at = self._tables.data_ptr()
        return at, at + self._turn_bytes

    # A copy, and what is unpickled, lays out tables of its own from the numbers.
    def __getstate__(self) -> dict:
        return {name: value for name, value in self.__dict__.items() if name not in ("_tables", "_streams", "_layout")}

    def __setstate__(self, state: dict) -> None:
        self.__dict__.update(state)
        self._lay_out()

    @classmethod
    def sections(cls, sections, *, base: float = 10000.0, apart: bool = False, interleaved: bool = False,
                 device) -> "RotaryAxes":
        """``sections[a]`` consecutive pairs for axis a, with frequencies ``base ** (-i / n)``:
        i counts all n pairs of the head, or with ``apart`` those of each axis."""
        sections = [int(s) for s in sections]
        if not sections or min(sections) < 1:
            raise ValueError("every axis needs at least one pair")
        if not (base > 0 and math.isfinite(base)):
            raise ValueError("base must be positive and finite")
        axes = [a for a, s in enumerate(sections) for _ in range(s)]
        if apart:
            frequencies = [base ** (-i / s) for s in sections for i in range(s)]
        else:
            frequencies = [base ** (-i / len(axes)) for i in range(len(axes))]
        return cls(frequencies, axes, interleaved=interleaved, device=device)

    # read only: calls take the layout that was checked above
    frequencies = property(lambda self: self._frequencies)
    axes = property(lambda self: self._axes)
    interleaved = property(lambda self: self._interleaved)
    device = property(lambda self: self._device)

    @property
    def rotary_dim(self) -> int:
        """Columns that turn."""
        return 2 * len(self._axes)


def _rows_ready(t: torch.Tensor) -> bool:
    """Unit stride along D, 16-byte rows, outer strides multiples of 16 bytes, zero (a broadcast) among them."""
    strides = t.stride()
    if strides[-1] != 1 or t.data_ptr() % 16:
        return False
    unit = 16 // t.element_size()
    for size, stride in zip(t.shape[:-1], strides[:-1]):
        if size > 1 and (stride < 0 or stride % unit or stride >= _MAX_STRIDE):
            return False
    return True


def _rows_laid_out(t: torch.Tensor) -> torch.Tensor:
    return t if _rows_ready(t) else t.clone(memory_format=torch.contiguous_format)


def _check_rotary(rotary, head_dim: int, device) -> None:
    if not isinstance(rotary, RotaryAxes):
        raise ValueError("rotary must be a RotaryAxes")
    if rotary.rotary_dim > head_dim:
        raise ValueError("rotary turns more columns than head_dim")
    if rotary.device != device:
        raise ValueError("rotary must be on the same CUDA device as the inputs")


def _check_positions(positions, batch: int, rows: int, axes: int, device) -> None:
    if not isinstance(positions, torch.Tensor) or positions.shape not in ((batch, rows, axes), (rows, axes)):
        raise ValueError(f"positions must have shape (B, n, {axes}) or (n, {axes})")
    if positions.dtype not in _POSITION_TYPES:
        raise ValueError("positions must be int32, int64 or float32")
    if positions.device != device:
        raise ValueError("positions must be on the same CUDA device as the inputs")


def _position_stride(positions) -> tuple[int, ...]:
    strides = positions.stride()
    return strides if len(strides) == 3 else (0, *strides)


def _check_heads(t, name: str, what: str, dtypes) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{what} requires CUDA tensors")
    if t.ndim != 4:
        raise ValueError(f"{name} must have shape (B, heads, n, D)")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be " + " or ".join(str(d).removeprefix("torch.") for d in dtypes))
    if t.shape[3] % 8 or not 8 <= t.shape[3] <= 128:
        raise ValueError("head_dim must be a multiple of 8 up to 128")


def _set_rotary(args, rotary, positions) -> None:
    args.rotary_dim, args.axes = rotary.rotary_dim, max(rotary.axes) + 1
    args.interleaved = int(rotary.interleaved)
    if positions is not None:
        args.position_type = _POSITION_TYPES[positions.dtype]
        args.position_stride[:] = _position_stride(positions)


_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _turn_plan(q, k, rotary, positions, inverse: bool):
    """Checks a call and returns its argument block behind the pointers, or None when a tensor has to
    be laid out first."""
    what = "rotate_positions"
    _check_heads(q, "q", what, _DTYPES)
    if k is not None:
        _check_heads(k, "k", what, _DTYPES)
        if (k.shape[0], *k.shape[2:]) != (q.shape[0], *q.shape[2:]) or k.dtype != q.dtype or k.device != q.device:
            raise ValueError("q and k must share B, n, D, dtype and device")
    _check_rotary(rotary, q.shape[3], q.device)
    _check_positions(positions, q.shape[0], q.shape[2], max(rotary.axes) + 1, q.device)
    if not (_rows_ready(q) and (k is None or _rows_ready(k))):
        return None
    args = _lib.RotaryArgs()
    args.batch, args.heads, args.rows, args.head_dim = q.shape
    args.q_stride, args.q_out_stride = q.stride(), torch.empty_like(q, device="meta").stride()
    if k is not None:
        args.groups = k.shape[1]
        args.k_stride, args.k_out_stride = k.stride(), torch.empty_like(k, device="meta").stride()
    args.dtype = _DTYPE_CODE[q.dtype]
    args.inverse = int(inverse)
    _set_rotary(args, rotary, positions)
    return bytes(args)[_POINTERS.size:]


def _rotate(q, k, rotary, positions, inverse: bool):
    """q and k (or None) turned: one launch.  What sizes, strides and types decide is kept by those alone."""
    try:
        device = q.device
        key = ("rotate", rotary._layout, q.shape, q.stride(), q.dtype, device, positions.shape, positions.stride(),
               positions.dtype, positions.device, inverse,
               None if k is None else (k.shape, k.stride(), k.dtype, k.device))
    except (AttributeError, TypeError):
        if not isinstance(q, torch.Tensor) or not (k is None or isinstance(k, torch.Tensor)):
            raise ValueError("rotate_positions requires CUDA tensors") from None
        if not isinstance(rotary, RotaryAxes):
            raise ValueError("rotary must be a RotaryAxes") from None
        if not isinstance(positions, torch.Tensor):
            raise ValueError("positions must be a tensor") from None
        raise
    tail = _plans.get(key)
    q_at, k_at = q.data_ptr(), 0 if k is None else k.data_ptr()
    if tail is None or (q_at | k_at) & 15:
        tail = _turn_plan(q, k, rotary, positions, inverse)
        if tail is None:
            return _rotate(_rows_laid_out(q), None if k is None else _rows_laid_out(k), rotary, positions, inverse)
        _keep(key, tail)
    q_out = torch.empty_like(q)
    k_out, k_to = None, 0
    if k is not None:
        k_out = torch.empty_like(k)
        k_to = k_out.data_ptr()
    block = _POINTERS.pack(q_at, k_at, 0, q_out.data_ptr(), k_to, 0, *rotary._launch_pointers(), positions.data_ptr(), 0, 0, 0) + tail
    _call(_lib.load().rotary_positions, block, device.index, "rotate_positions")
    return q_out, k_out


class _RotatePositions(torch.autograd.Function):
    """Linear in q and k: the gradient is turned back by the same angles.  A result whose input
    needs no gradient needs none."""

    @staticmethod
    def forward(ctx, q, k, rotary, positions, inverse):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions)
        ctx.rotary, ctx.inverse = rotary, inverse
        outs = _rotate(q, k, rotary, positions, inverse)
        # the result of an input that needs no gradient needs none either
        ctx.mark_non_differentiable(*(y for y, needs in zip(outs, ctx.needs_input_grad) if y is not None and not needs))
        return outs

    @staticmethod
    def backward(ctx, grad_q, grad_k):
        positions, = ctx.saved_tensors
        if grad_q is not None:
            grad_q, grad_k = _back(ctx, grad_q, grad_k, positions)
        elif grad_k is not None:
            grad_k, _ = _back(ctx, grad_k, None, positions)
        return grad_q, grad_k, None, None, None


def _back(ctx, one, two, positions):
    if _grad_enabled():  # create_graph: the gradient has one of its own
        return rotate_positions(one, two, rotary=ctx.rotary, positions=positions, inverse=not ctx.inverse)
    return _rotate(one, two, ctx.rotary, positions, not ctx.inverse)


def rotate_positions(q, k=None, *, rotary, positions, inverse: bool = False):
    """``(q, k)`` turned by ``positions`` (see the module's text); ``k`` may be left out
    and is then None.

    ``q`` ``(B, H, n, D)`` and ``k`` ``(B, G, n, D)`` bf16, f16 or f32, D a multiple of 8
    up to 128; ``positions`` ``(B, n, axes)`` or, for every sequence, ``(n, axes)``,
    int32, int64 or float32 with any strides.  ``inverse`` turns by the negative angles.
    Inputs whose rows are not 16-byte aligned with unit stride along D are copied
    first; broadcast ones (stride zero) are not."""
    if _unusual():
        _refuse_transforms("rotate_positions", q, k, positions)
    if _grad_enabled():
        if isinstance(positions, torch.Tensor) and positions.requires_grad:
            raise ValueError("positions have no gradient: detach them")
        if (isinstance(q, torch.Tensor) and q.requires_grad) or (isinstance(k, torch.Tensor) and k.requires_grad):
            return _RotatePositions.apply(q, k, rotary, positions, bool(inverse))
    return _rotate(q, k, rotary, positions, bool(inverse))
