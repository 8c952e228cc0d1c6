"""Cross attention to an encoder's states on B200.

``cross_attention(q, k, v, *, scale, lengths=None)`` for a decoder (or pooling
queries) that reads the encoder's states:

    S = scale * q @ k^T                     (fp32; query head h reads key head h // (H / G))
    out = softmax(S over the sequence's states, -1) @ v      cast to q.dtype

with ``q`` ``(B, H, M, D)`` and ``k``, ``v`` ``(B, G, N, D)``, H a multiple of
G, bf16 or f16, ``D`` a multiple of 8 up to 128, M and N from one up.
``lengths`` ``(B,)`` counts each sequence's states (all N without it; values
are clamped to 0..N); states past it take no part whatever they hold, NaN
included, and a sequence without states gives zeros.  A row whose every score
is -inf gives zeros too.  The operator is differentiable in q, k and v
(``cross_attention_forward`` / ``cross_attention_backward`` are its two
halves); results and gradients repeat bit for bit.

Many rows per key head run on 128-row tensor-core tiles, few (single tokens)
on a kernel that streams the states once for every 16 rows; ``kernel`` selects.

``shared_prefix_attention(q, prefix_k, prefix_v, k, v, *, scale, lengths=None)``
is the same softmax over a prefix ``(G, P, D)`` that every sequence shares and
then the sequence's own states (a 16-bit pair, or a ``StateCache``): the
prefix's part is computed for the rows of the whole batch at once.

Inputs without unit stride along D, or with rows that are not 16-byte aligned,
are copied first; nothing else is.  Every call runs the CUDA kernels of
``libintp_b200.so`` on the current stream of the inputs' device; there is no CPU
path, CPU tensors raise ``ValueError``.  Calls can be captured into a CUDA graph
once one call has run on the device.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .look_attention import _DTYPE_CODE, _status_word, _status_words

_KERNELS = {"auto": _lib.XATTN_KERNEL_AUTO, "rows": _lib.XATTN_KERNEL_ROWS, "tiles": _lib.XATTN_KERNEL_TILES}
_HALF = (torch.bfloat16, torch.float16)
_MAX_STRIDE = 1 << 39  # elements: 2^40 bytes


def _ready(t: torch.Tensor) -> bool:
    """Unit stride along D, 16-byte rows, outer strides positive multiples of 16 bytes."""
    strides = t.stride()
    if strides[-1] != 1 or t.data_ptr() % 16:
        return False
    unit = 16 // t.element_size()
    for size, stride in zip(t.shape[:-1], strides[:-1]):
        if size > 1 and (stride <= 0 or stride % unit or stride >= _MAX_STRIDE):
            return False
    return True


def _laid_out(t: torch.Tensor) -> torch.Tensor:
    return t if _ready(t) else t.clone(memory_format=torch.contiguous_format)


def _check_scale(scale) -> float:
    scale = float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError("scale must be positive and finite")
    return scale


def _check_query(q, groups: int, head_dim: int, what: str, unit: int) -> None:
    if not isinstance(q, torch.Tensor) or not q.is_cuda:
        raise ValueError(f"{what} requires CUDA tensors")
    if q.ndim != 4:
        raise ValueError("q must have shape (B, H, M, D)")
    if q.dtype not in _HALF:
        raise ValueError("q must be bfloat16 or float16")
    if q.shape[3] != head_dim:
        raise ValueError("q and the states must share head_dim")
    if head_dim % unit or not unit <= head_dim <= 128:
        raise ValueError(f"head_dim must be a multiple of {unit} up to 128")
    if groups < 1 or q.shape[1] < 1 or q.shape[1] % groups:
        raise ValueError("the query heads must be a multiple of the key heads")


def _check_pair(q, k, v, shape_text: str, what: str) -> None:
    for t in (k, v):
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise ValueError(f"{what} requires CUDA tensors")
        if t.ndim != len(shape_text.split(",")):
            raise ValueError(f"k and v must share shape {shape_text}")
    if k.shape != v.shape:
        raise ValueError(f"k and v must share shape {shape_text}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must share a dtype")
    if k.device != q.device or v.device != q.device:
        raise ValueError("all tensors must be on the same CUDA device")


def _check_counts(t, batch: int, device, name: str):
    """A per-sequence int32 vector (int64 is converted), or None."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.shape != (batch,) or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be an int32 or int64 tensor of shape (B,)")
    if t.device != device:
        raise ValueError(f"{name} must be on the same CUDA device as q")
    if t.dtype == torch.int64:
        t = t.clamp(-2147483648, 2147483647).to(torch.int32)
    return t.contiguous()


def _check_states(q, k, v, lengths):
    """The checks of ``cross_attention``; returns the lengths as the kernels take them."""
    what = "cross attention"
    if not isinstance(q, torch.Tensor) or not q.is_cuda:
        raise ValueError(f"{what} requires CUDA tensors")
    _check_pair(q, k, v, "(B, G, N, D)", what)
    _check_query(q, k.shape[1], k.shape[3], what, 8)
    if k.shape[0] != q.shape[0]:
        raise ValueError("q, k and v must share the batch size")
    if k.shape[2] < 1:
        raise ValueError("k and v must hold at least one state (use lengths for empty sequences)")
    return _check_counts(lengths, q.shape[0], q.device, "lengths")


def _status(device) -> torch.Tensor:
    word = _status_words.get(device.index)
    if word is None:
        if torch.cuda.is_current_stream_capturing():
            # the word would live in the graph's memory and stay unset until its first replay
            raise RuntimeError("run one call on this device before capturing one into a CUDA graph")
        word = _status_word(device)
    return word


def _call(fn, args, device) -> int:
    """One library call on the device's current stream."""
    index = device.index
    if torch.cuda.current_device() == index:
        return fn(ctypes.addressof(args), torch.cuda.current_stream(index).cuda_stream)
    with torch.cuda.device(index):
        return fn(ctypes.addressof(args), torch.cuda.current_stream(index).cuda_stream)


def _base_args(q, scale: float, lengths, out, lse, kernel: str) -> _lib.XattnArgs:
    batch, heads, queries, head_dim = q.shape
    args = _lib.XattnArgs()
    args.batch, args.heads, args.queries, args.head_dim = batch, heads, queries, head_dim
    args.scale = scale
    args.dtype = _DTYPE_CODE[q.dtype]
    args.q, args.q_stride = q.data_ptr(), q.stride()
    args.out, args.out_stride = out.data_ptr(), out.stride()
    if lengths is not None:
        args.lengths = lengths.data_ptr()
    if lse is not None:
        args.lse = lse.data_ptr()
    if kernel not in _KERNELS:
        raise ValueError(f"kernel must be one of {sorted(_KERNELS)}")
    args.kernel = _KERNELS[kernel]
    args.status = _status(q.device).data_ptr()
    return args


def _set_states(args, k, v) -> None:
    args.groups, args.states = k.shape[1], k.shape[2]
    args.k, args.k_stride = k.data_ptr(), k.stride()
    args.v, args.v_stride = v.data_ptr(), v.stride()


def _workspace(fn, args, fwd_args, device, what: str):
    """Scratch memory for one call, from the current stream's allocator."""
    size = ctypes.c_int64()
    _lib.check(fn(ctypes.addressof(args), ctypes.byref(size)), what)
    if size.value == 0:
        return None
    space = torch.empty(size.value, dtype=torch.uint8, device=device)
    fwd_args.workspace, fwd_args.workspace_bytes = space.data_ptr(), size.value
    return space


def _run_forward(args, device, what: str) -> None:
    lib = _lib.load()
    space = _workspace(lib.xattn_forward_workspace, args, args, device, what)
    status = _call(lib.xattn_forward, args, device)
    del space
    if status == _lib.INTP_ERR_UNSUPPORTED:
        raise ValueError(f"{what}: the selected kernel does not take these inputs")
    _lib.check(status, what)


def _output(q, out):
    if out is None:
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if not isinstance(out, torch.Tensor) or out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
        raise ValueError("out must match q in shape, dtype and device")
    if not _ready(out):
        raise ValueError("out needs unit stride on head_dim and 16-byte aligned rows")
    return out


def cross_attention_forward(q, k, v, *, scale, lengths=None, want_lse: bool = False, kernel: str = "auto", out=None):
    """Forward only.  Returns ``(out, lse_or_None)``; ``lse`` ``(B, H, M)`` float32 is
    the natural log of the row sums (-inf for a row without states).

    ``kernel``: ``"auto"`` chooses by the number of rows that share a key head
    (``M * H / G``), ``"rows"`` and ``"tiles"`` force one of the two kernels."""
    lengths = _check_states(q, k, v, lengths)
    scale = _check_scale(scale)
    out = _output(q, out)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device) if want_lse else None
    q, k, v = _laid_out(q), _laid_out(k), _laid_out(v)
    args = _base_args(q, scale, lengths, out, lse, kernel)
    _set_states(args, k, v)
    _run_forward(args, q.device, "cross attention")
    return out, lse


def cross_attention_backward(q, k, v, out, lse, grad_out, *, scale, lengths=None, needs=(True, True, True)):
    """Gradients ``(dq, dk, dv)`` of ``cross_attention_forward`` from its ``out`` and
    ``lse``, contiguous and in the inputs' dtype; None where ``needs`` is False.
    States past a sequence's length get zeros."""
    lengths = _check_states(q, k, v, lengths)
    scale = _check_scale(scale)
    for name, t in (("out", out), ("grad_out", grad_out)):
        if not isinstance(t, torch.Tensor) or t.shape != q.shape or t.device != q.device:
            raise ValueError(f"{name} must match q in shape and device")
    if out.dtype != q.dtype:
        raise ValueError("out must match q in dtype")
    if (not isinstance(lse, torch.Tensor) or lse.shape != q.shape[:3] or lse.dtype != torch.float32
            or lse.device != q.device):
        raise ValueError("lse must be the forward's (B, H, M) float32 row sums")
    device = q.device
    empty = q.numel() == 0
    make = torch.zeros if empty else torch.empty
    dq = make(q.shape, dtype=q.dtype, device=device) if needs[0] else None
    dk = make(k.shape, dtype=q.dtype, device=device) if needs[1] else None
    dv = make(v.shape, dtype=q.dtype, device=device) if needs[2] else None
    if empty or not any(needs):
        return dq, dk, dv
    q, k, v, out, lse = _laid_out(q), _laid_out(k), _laid_out(v), _laid_out(out), lse.contiguous()
    grad_out = _laid_out(grad_out.to(q.dtype))
    args = _lib.XattnBackwardArgs()
    args.fwd = _base_args(q, scale, lengths, out, lse, "auto")
    _set_states(args.fwd, k, v)
    args.grad_out, args.grad_out_stride = grad_out.data_ptr(), grad_out.stride()
    for name, t in (("grad_q", dq), ("grad_k", dk), ("grad_v", dv)):
        if t is not None:
            setattr(args, name, t.data_ptr())
    lib = _lib.load()
    what = "cross attention backward"
    space = _workspace(lib.xattn_backward_workspace, args, args.fwd, device, what)
    status = _call(lib.xattn_backward, args, device)
    del space
    _lib.check(status, what)
    return dq, dk, dv


class _CrossAttention(torch.autograd.Function):
    """The forward keeps its row sums; the backward recomputes the probabilities from them."""

    @staticmethod
    def forward(ctx, q, k, v, lengths, scale):
        out, lse = cross_attention_forward(q, k, v, scale=scale, lengths=lengths, want_lse=True)
        ctx.scale = scale
        ctx.save_for_backward(q, k, v, lengths, out, lse)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        q, k, v, lengths, out, lse = ctx.saved_tensors
        dq, dk, dv = cross_attention_backward(q, k, v, out, lse, grad_out, scale=ctx.scale, lengths=lengths,
                                              needs=ctx.needs_input_grad[:3])
        return dq, dk, dv, None, None


def cross_attention(q, k, v, *, scale, lengths=None):
    """Attention of ``q`` to the states ``k``, ``v`` (see the module's text)."""
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (q, k, v)):
        return _CrossAttention.apply(q, k, v, lengths, _check_scale(scale))
    return cross_attention_forward(q, k, v, scale=scale, lengths=lengths)[0]


def _refuse_grad(what: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors):
        raise ValueError(f"{what} has no backward pass: call it under torch.no_grad() or detach its inputs")


def shared_prefix_attention(q, prefix_k, prefix_v, k, v=None, *, scale, lengths=None, out=None):
    """Attention of every sequence's ``q`` ``(B, H, M, D)`` to the prefix ``prefix_k``,
    ``prefix_v`` ``(G, P, D)`` and then to its own states: ``k``, ``v`` ``(B, G, N, D)``
    (N may be zero), or a :class:`~intp_preliminary_b200.StateCache` as ``k``.
    ``lengths`` counts a sequence's own states.  Inference only."""
    from .state_cache import StateCache

    what = "shared-prefix attention"
    _refuse_grad(what, q, prefix_k, prefix_v, k, v)
    if not isinstance(q, torch.Tensor) or not q.is_cuda:
        raise ValueError(f"{what} requires CUDA tensors")
    _check_pair(q, prefix_k, prefix_v, "(G, P, D)", what)
    groups, prefix, head_dim = prefix_k.shape
    if prefix < 1:
        raise ValueError("the prefix must hold at least one state")
    scale = _check_scale(scale)
    cached = isinstance(k, StateCache)
    _check_query(q, groups, head_dim, what, 16 if cached else 8)
    if cached:
        if v is not None:
            raise ValueError("a StateCache holds both keys and values: leave v out")
        own_shape = k.keys.shape
        if k.device != q.device:
            raise ValueError("all tensors must be on the same CUDA device")
    else:
        _check_pair(q, k, v, "(B, G, N, D)", what)
        own_shape = k.shape
    if own_shape[0] != q.shape[0] or own_shape[1] != groups or own_shape[3] != head_dim:
        raise ValueError("the sequences' own states must have shape (B, G, N, D) like q and the prefix")
    lengths = _check_counts(lengths, q.shape[0], q.device, "lengths")
    out = _output(q, out)
    q, prefix_k, prefix_v = _laid_out(q), _laid_out(prefix_k), _laid_out(prefix_v)
    args = _base_args(q, scale, lengths, out, None, "auto")
    if cached:
        k._set_states(args)
    else:
        k, v = _laid_out(k), _laid_out(v)
        _set_states(args, k, v)
    args.prefix = prefix
    args.prefix_k, args.prefix_k_stride = prefix_k.data_ptr(), prefix_k.stride()
    args.prefix_v, args.prefix_v_stride = prefix_v.data_ptr(), prefix_v.stride()
    _run_forward(args, q.device, what)
    return out
