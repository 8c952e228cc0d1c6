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
halves); results and gradients repeat bit for bit.  Reverse mode, once: a second
derivative, forward-mode tangents and ``torch.jit.trace`` are refused, and the
operators over a cache or a prefix take no part in autograd at all.

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
import struct

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .look_attention import _DTYPE_CODE, _refuse_transforms, _status_word, _status_words

_KERNELS = {"auto": _lib.XATTN_KERNEL_AUTO, "rows": _lib.XATTN_KERNEL_ROWS, "tiles": _lib.XATTN_KERNEL_TILES}
_HALF = (torch.bfloat16, torch.float16)
_INTEGERS = (torch.int32, torch.int64)
_MAX_STRIDE = 1 << 39  # elements: 2^40 bytes


# torch's own accessors, without the lazy initialisation that a CUDA tensor's existence has done.
_current_device = torch._C._cuda_getDevice
_current_stream = torch._C._cuda_getCurrentRawStream


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
    if not isinstance(t, torch.Tensor) or t.shape != (batch,) or t.dtype not in _INTEGERS:
        raise ValueError(f"{name} must be an int32 or int64 tensor of shape (B,)")
    if t.device != device:
        raise ValueError(f"{name} must be on the same CUDA device as q")
    if t.dtype == torch.int64:
        t = t.clamp(-2147483648, 2147483647).to(torch.int32)
    return t if t.is_contiguous() else t.contiguous()


def _check_states(q, k, v) -> None:
    what = "cross attention"
    if not isinstance(q, torch.Tensor) or not q.is_cuda:
        raise ValueError(f"{what} requires CUDA tensors")
    _check_pair(q, k, v, "(B, G, N, D)", what)
    _check_query(q, k.shape[1], k.shape[3], what, 8)
    if k.shape[0] != q.shape[0]:
        raise ValueError("q, k and v must share the batch size")
    if k.shape[2] < 1:
        raise ValueError("k and v must hold at least one state (use lengths for empty sequences)")


def _status(device) -> torch.Tensor:
    word = _status_words.get(device.index)
    if word is None:
        if torch.cuda.is_current_stream_capturing():
            # the word would live in the graph's memory and stay unset until its first replay
            raise RuntimeError("run one call on this device before capturing one into a CUDA graph")
        word = _status_word(device)
    return word


# What a call's sizes, strides and types decide, kept by those alone: its checks have
# passed, the library's argument block is filled but for the pointers, its scratch size known.
_POINTERS = struct.Struct("13Q")   # xattn_args up to workspace_bytes
_BACKWARD_POINTERS = struct.Struct("4Q")
_POINTER_BYTES = _POINTERS.size
_FORWARD_BYTES = ctypes.sizeof(_lib.XattnArgs)
_MAX_PLANS = 1024


class _Plan:
    # backward: by the output gradient's strides, (the argument block's end, scratch bytes)
    # layout: of q, k, v and out (_layout), for the tensors that a backward gets back
    __slots__ = ("tail", "scratch", "status", "index", "batch", "device", "empty", "out_shape", "lse_shape", "dtype",
                 "args", "backward", "layout", "scale")


_plans: dict = {}


def _keep(key, plan):
    if len(_plans) >= _MAX_PLANS:
        _plans.clear()
    _plans[key] = plan
    return plan


def _base_args(q, scale: float, out_stride, kernel: str) -> _lib.XattnArgs:
    if kernel not in _KERNELS:
        raise ValueError(f"kernel must be one of {sorted(_KERNELS)}")
    args = _lib.XattnArgs()
    args.batch, args.heads, args.queries, args.head_dim = q.shape
    args.scale = scale
    args.dtype = _DTYPE_CODE[q.dtype]
    args.q_stride, args.out_stride = q.stride(), out_stride
    args.kernel = _KERNELS[kernel]
    return args


def _set_pair(args, k, v) -> None:
    args.groups, args.states = k.shape[1], k.shape[2]
    args.k_stride, args.v_stride = k.stride(), v.stride()


def _scratch_bytes(fn, args, what: str) -> int:
    size = ctypes.c_int64()
    status = fn(ctypes.addressof(args), ctypes.byref(size))
    if status == _lib.INTP_ERR_UNSUPPORTED:
        raise ValueError(f"{what}: the selected kernel does not take these inputs")
    _lib.check(status, what)
    return size.value


def _finish_plan(args, q, what: str) -> _Plan:
    """Scratch size and argument block of a filled ``XattnArgs``."""
    plan = _Plan()
    plan.scratch = _scratch_bytes(_lib.load().xattn_forward_workspace, args, what)
    plan.device, plan.index, plan.batch, plan.dtype = q.device, q.device.index, q.shape[0], q.dtype
    plan.out_shape, plan.lse_shape = q.shape, q.shape[:3]
    plan.status = _status(q.device).data_ptr()
    plan.empty = q.numel() == 0
    plan.tail = bytes(args)[_POINTER_BYTES:]
    plan.args, plan.backward = args, {}
    return plan


def _call(fn, block, index: int, what: str) -> None:
    """One library call on the device's current stream."""
    if _current_device() == index:
        status = fn(block, _current_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(block, _current_stream(index))
    if status:
        _lib.check(status, what)


def _launch(plan: _Plan, what: str, q, k, v, k_exponents, v_exponents, prefix_k, prefix_v, lengths, out, lse) -> None:
    if plan.empty:
        return
    space = 0
    if plan.scratch:
        scratch = torch.empty(plan.scratch, dtype=torch.uint8, device=plan.device)  # from the current stream's pool
        space = scratch.data_ptr()
    block = _POINTERS.pack(q, k, v, k_exponents, v_exponents, prefix_k, prefix_v, lengths, out, lse, space, plan.status,
                           plan.scratch) + plan.tail
    _call(_lib.load().xattn_forward, block, plan.index, what)


def _output(q, out):
    if out is None:
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if not isinstance(out, torch.Tensor) or out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
        raise ValueError("out must match q in shape, dtype and device")
    if not _ready(out):
        raise ValueError("out needs unit stride on head_dim and 16-byte aligned rows")
    return out


def _lengths_pointer(lengths, plan: _Plan, name: str):
    """``(tensor to keep, its address)`` of a per-sequence count."""
    if lengths is None:
        return None, 0
    lengths = _check_counts(lengths, plan.batch, plan.device, name)
    return lengths, lengths.data_ptr()


def _layout(t: torch.Tensor):
    return t.shape, t.stride(), t.dtype


def _forward_plan(q, k, v, scale, out_stride, kernel):
    """The plan for these tensors, or None when one has to be laid out first."""
    key = (q.shape, q.stride(), k.shape, k.stride(), v.shape, v.stride(), q.dtype, k.dtype, v.dtype, q.device,
           k.device, v.device, scale, out_stride, kernel)
    plan = _plans.get(key)
    if plan is None:
        _check_states(q, k, v)
        args = _base_args(q, _check_scale(scale), out_stride, kernel)
        if not (_ready(q) and _ready(k) and _ready(v)):
            return None
        _set_pair(args, k, v)
        plan = _finish_plan(args, q, "cross attention")
        plan.layout = (_layout(q), _layout(k), _layout(v), (q.shape, out_stride, q.dtype))
        plan.scale = scale
        _keep(key, plan)
    return plan


def _forward(q, k, v, scale, lengths, want_lse: bool, kernel: str, out):
    """``(out, lse, plan, q, k, v, lengths)``, the last four as the kernels took them."""
    if not (isinstance(q, torch.Tensor) and isinstance(k, torch.Tensor) and isinstance(v, torch.Tensor)):
        raise ValueError("cross attention requires CUDA tensors")
    scale = float(scale)
    out_stride = None
    if out is not None:
        out_stride = _output(q, out).stride()
    elif q.ndim == 4:
        _, h, m, d = q.shape
        out_stride = (h * m * d, m * d, d, 1)
    plan = _forward_plan(q, k, v, scale, out_stride, kernel)
    qp, kp, vp = q.data_ptr(), k.data_ptr(), v.data_ptr()
    if plan is None or (qp | kp | vp) & 15:
        q, k, v = _laid_out(q), _laid_out(k), _laid_out(v)
        plan = _forward_plan(q, k, v, scale, out_stride, kernel)
        qp, kp, vp = q.data_ptr(), k.data_ptr(), v.data_ptr()
    lengths, lengths_p = _lengths_pointer(lengths, plan, "lengths")
    if out is None:
        out = torch.empty(plan.out_shape, dtype=plan.dtype, device=plan.device)
    lse, lse_p = None, 0
    if want_lse:
        lse = torch.empty(plan.lse_shape, dtype=torch.float32, device=plan.device)
        lse_p = lse.data_ptr()
    _launch(plan, "cross attention", qp, kp, vp, 0, 0, 0, 0, lengths_p, out.data_ptr(), lse_p)
    return out, lse, plan, q, k, v, lengths


def cross_attention_forward(q, k, v, *, scale, lengths=None, want_lse: bool = False, kernel: str = "auto", out=None):
    """Forward only.  Returns ``(out, lse_or_None)``; ``lse`` ``(B, H, M)`` float32 is
    the natural log of the row sums (-inf for a row without states).

    ``kernel``: ``"auto"`` chooses by the number of rows that share a key head
    (``M * H / G``), ``"rows"`` and ``"tiles"`` force one of the two kernels."""
    _refuse_transforms("cross attention", q, k, v)
    return _forward(q, k, v, scale, lengths, want_lse, kernel, out)[:2]


def _backward(plan: _Plan, q, k, v, lengths, out, lse, grad_out, needs):
    """The gradients; every tensor but ``grad_out`` as ``_forward`` took or made it."""
    if plan.empty or not any(needs):
        return tuple(torch.zeros(t.shape, dtype=t.dtype, device=t.device) if n else None
                     for t, n in zip((q, k, v), needs))
    if grad_out.dtype != plan.dtype:
        grad_out = grad_out.to(plan.dtype)
    grad_stride = grad_out.stride()
    known = plan.backward.get(grad_stride)
    if known is None or grad_out.data_ptr() & 15:
        grad_out = _laid_out(grad_out)
        grad_stride = grad_out.stride()
        args = _lib.XattnBackwardArgs()
        args.fwd = plan.args
        args.grad_out_stride = grad_stride
        scratch = _scratch_bytes(_lib.load().xattn_backward_workspace, args, "cross attention backward")
        known = plan.backward[grad_stride] = (bytes(args)[_FORWARD_BYTES + _BACKWARD_POINTERS.size:], scratch)
    end, scratch_bytes = known
    dq, dk, dv = (torch.empty(t.shape, dtype=plan.dtype, device=plan.device) if n else None
                  for t, n in zip((q, k, v), needs))
    scratch = torch.empty(scratch_bytes, dtype=torch.uint8, device=plan.device)
    block = _POINTERS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), 0, 0, 0, 0,
                           0 if lengths is None else lengths.data_ptr(), out.data_ptr(), lse.data_ptr(),
                           scratch.data_ptr(), plan.status, scratch_bytes) + plan.tail
    block += _BACKWARD_POINTERS.pack(grad_out.data_ptr(), 0 if dq is None else dq.data_ptr(),
                                     0 if dk is None else dk.data_ptr(), 0 if dv is None else dv.data_ptr()) + end
    _call(_lib.load().xattn_backward, block, plan.index, "cross attention backward")
    return dq, dk, dv


def cross_attention_backward(q, k, v, out, lse, grad_out, *, scale, lengths=None, needs=(True, True, True)):
    """Gradients ``(dq, dk, dv)`` of ``cross_attention_forward`` from its ``out`` and
    ``lse``, contiguous and in the inputs' dtype; None where ``needs`` is False.
    States past a sequence's length get zeros."""
    _refuse_transforms("cross attention backward", q, k, v, out, lse, grad_out)
    _check_states(q, k, v)
    scale = _check_scale(scale)
    for name, t in (("out", out), ("grad_out", grad_out)):
        if not isinstance(t, torch.Tensor) or t.shape != q.shape or t.device != q.device:
            raise ValueError(f"{name} must match q in shape and device")
    if out.dtype != q.dtype:
        raise ValueError("out must match q in dtype")
    if (not isinstance(lse, torch.Tensor) or lse.shape != q.shape[:3] or lse.dtype != torch.float32
            or lse.device != q.device):
        raise ValueError("lse must be the forward's (B, H, M) float32 row sums")
    q, k, v, out, lse = _laid_out(q), _laid_out(k), _laid_out(v), _laid_out(out), lse.contiguous()
    plan = _forward_plan(q, k, v, scale, out.stride(), "auto")
    lengths, _ = _lengths_pointer(lengths, plan, "lengths")
    return _backward(plan, q, k, v, lengths, out, lse, grad_out, needs)


class _CrossAttention(torch.autograd.Function):
    """The forward keeps its row sums; the backward recomputes the probabilities from them."""

    @staticmethod
    def forward(ctx, q, k, v, lengths, scale):
        out, lse, ctx.plan, q, k, v, lengths = _forward(q, k, v, scale, lengths, True, "auto", None)
        ctx.save_for_backward(q, k, v, lengths, out, lse)
        return out

    @staticmethod
    def backward(ctx, grad_out):
        if torch.is_grad_enabled():  # create_graph: refuse a second derivative in so many words
            return _CrossAttention._once(ctx, grad_out)
        return _CrossAttention._first(ctx, grad_out)

    @staticmethod
    def _first(ctx, grad_out):
        q, k, v, lengths, out, lse = ctx.saved_tensors
        plan, needs = ctx.plan, ctx.needs_input_grad[:3]
        if ((_layout(q), _layout(k), _layout(v), _layout(out)) != plan.layout
                or (q.data_ptr() | k.data_ptr() | v.data_ptr() | out.data_ptr()) & 15 or not lse.is_contiguous()):
            # hooks on saved tensors (offloading, compression) return the values, not always the strides
            return (*cross_attention_backward(q, k, v, out, lse, grad_out, scale=plan.scale, lengths=lengths,
                                              needs=needs), None, None)
        return (*_backward(plan, q, k, v, lengths, out, lse, grad_out, needs), None, None)

    _once = staticmethod(once_differentiable(_first))


def cross_attention(q, k, v, *, scale, lengths=None):
    """Attention of ``q`` to the states ``k``, ``v`` (see the module's text)."""
    _refuse_transforms("cross attention", q, k, v)
    if torch.is_grad_enabled() and any([isinstance(t, torch.Tensor) and t.requires_grad for t in (q, k, v)]):
        return _CrossAttention.apply(q, k, v, lengths, _check_scale(scale))
    return _forward(q, k, v, scale, lengths, False, "auto", None)[0]


def _refuse_grad(what: str, *tensors) -> None:
    _refuse_transforms(what, *tensors)
    if torch.is_grad_enabled() and any([isinstance(t, torch.Tensor) and t.requires_grad for t in tensors]):
        raise ValueError(f"{what} has no backward pass: call it under torch.no_grad() or detach its inputs")


def _prefix_plan(q, prefix_k, prefix_v, k, v, cache, scale, out_stride):
    """The plan of a shared-prefix call, or None when a tensor has to be laid out first."""
    own = cache.layout if cache is not None else (k.shape, k.stride(), v.shape, v.stride(), k.dtype, v.dtype, k.device,
                                                  v.device)
    key = (q.shape, q.stride(), q.dtype, q.device, prefix_k.shape, prefix_k.stride(), prefix_v.shape,
           prefix_v.stride(), prefix_k.dtype, prefix_v.dtype, prefix_k.device, prefix_v.device, own, scale, out_stride)
    plan = _plans.get(key)
    if plan is not None:
        return plan
    what = "shared-prefix attention"
    if not q.is_cuda:
        raise ValueError(f"{what} requires CUDA tensors")
    _check_pair(q, prefix_k, prefix_v, "(G, P, D)", what)
    groups, prefix, head_dim = prefix_k.shape
    if prefix < 1:
        raise ValueError("the prefix must hold at least one state")
    scale = _check_scale(scale)
    _check_query(q, groups, head_dim, what, 8 if cache is None else 16)
    if cache is not None:
        own_shape = cache.keys.shape
        if cache.device != q.device:
            raise ValueError("all tensors must be on the same CUDA device")
    else:
        _check_pair(q, k, v, "(B, G, N, D)", what)
        own_shape = k.shape
    if own_shape[0] != q.shape[0] or own_shape[1] != groups or own_shape[3] != head_dim:
        raise ValueError("the sequences' own states must have shape (B, G, N, D) like q and the prefix")
    if not all(_ready(t) for t in (q, prefix_k, prefix_v) + (() if cache is not None else (k, v))):
        return None
    args = _base_args(q, scale, out_stride, "auto")
    if cache is not None:
        cache._set_states(args)
    else:
        _set_pair(args, k, v)
    args.prefix = prefix
    args.prefix_k_stride, args.prefix_v_stride = prefix_k.stride(), prefix_v.stride()
    return _keep(key, _finish_plan(args, q, what))


def shared_prefix_attention(q, prefix_k, prefix_v, k, v=None, *, scale, lengths=None, out=None):
    """Attention of every sequence's ``q`` ``(B, H, M, D)`` to the prefix ``prefix_k``,
    ``prefix_v`` ``(G, P, D)`` and then to its own states: ``k``, ``v`` ``(B, G, N, D)``
    (N may be zero), or a :class:`~intp_preliminary_b200.StateCache` as ``k``.
    ``lengths`` counts a sequence's own states.  Inference only."""
    from .state_cache import StateCache

    what = "shared-prefix attention"
    cache = k if isinstance(k, StateCache) else None
    if cache is not None and v is not None:
        raise ValueError("a StateCache holds both keys and values: leave v out")
    if not all(isinstance(t, torch.Tensor) for t in (q, prefix_k, prefix_v) + (() if cache is not None else (k, v))):
        raise ValueError(f"{what} requires CUDA tensors")
    _refuse_grad(what, q, prefix_k, prefix_v, k, v)
    scale = float(scale)
    out_stride = None
    if out is not None:
        out_stride = _output(q, out).stride()
    elif q.ndim == 4:
        _, h, m, d = q.shape
        out_stride = (h * m * d, m * d, d, 1)
    plan = _prefix_plan(q, prefix_k, prefix_v, k, v, cache, scale, out_stride)
    own = (cache.keys, cache.values) if cache is not None else (k, v)
    if plan is None or (q.data_ptr() | prefix_k.data_ptr() | prefix_v.data_ptr() | own[0].data_ptr()
                        | own[1].data_ptr()) & 15:
        q, prefix_k, prefix_v = _laid_out(q), _laid_out(prefix_k), _laid_out(prefix_v)
        if cache is None:
            k, v = own = _laid_out(k), _laid_out(v)
        plan = _prefix_plan(q, prefix_k, prefix_v, k, v, cache, scale, out_stride)
    exponents = (0, 0)
    if cache is not None and cache.keys.shape[2] > 0:
        exponents = (cache.key_exponents.data_ptr(), cache.value_exponents.data_ptr())
    lengths, lengths_p = _lengths_pointer(lengths, plan, "lengths")
    if out is None:
        out = torch.empty(plan.out_shape, dtype=plan.dtype, device=plan.device)
    _launch(plan, what, q.data_ptr(), own[0].data_ptr(), own[1].data_ptr(), *exponents, prefix_k.data_ptr(),
            prefix_v.data_ptr(), lengths_p, out.data_ptr(), 0)
    return out
