"""Cross attention, the state cache and shared prefixes without a GPU: the C ABI's
structs, refusals and workspace sizes, CPU tensors, and the oracle itself."""

import ctypes
import re
import sys
from pathlib import Path

import pytest
import torch

from intp_preliminary_b200 import (StateCache, _lib, cached_cross_attention, cross_attention,
                                   cross_attention_backward, cross_attention_forward, shared_prefix_attention)
from oracle import cross_attention as oracle

HEADER = Path(__file__).resolve().parent.parent / "include" / "intp_b200.h"
FAKE = 1 << 20  # never dereferenced: every call below is refused before a launch


@pytest.mark.parametrize("name,mirror", [("xattn_args", _lib.XattnArgs), ("xattn_backward_args", _lib.XattnBackwardArgs),
                                         ("state_cache_args", _lib.StateCacheArgs)])
def test_struct_layout_matches_header_field_order(name, mirror):
    text = HEADER.read_text()
    body = text[text.index(f"typedef struct {name} {{"):text.index(f"}} {name};")]
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    assert re.findall(r"(\w+)(?:\[\d\])?\s*[;,]", body) == [f[0] for f in mirror._fields_]


def _args(**over):
    a = _lib.XattnArgs()
    a.batch, a.heads, a.groups, a.queries, a.states, a.head_dim = 2, 4, 2, 3, 100, 64
    a.scale, a.dtype = 0.125, _lib.INTP_BF16
    a.q = a.k = a.v = a.out = a.status = FAKE
    a.q_stride = a.out_stride = _lib._Stride(768, 192, 64, 1)
    a.k_stride = a.v_stride = _lib._Stride(12800, 6400, 64, 1)
    for key, value in over.items():
        setattr(a, key, value)
    return a


@pytest.mark.parametrize("over,status", [
    ({"heads": 3}, _lib.INTP_ERR_SHAPE),                       # not a multiple of the key heads
    ({"head_dim": 60}, _lib.INTP_ERR_SHAPE),
    ({"head_dim": 136}, _lib.INTP_ERR_SHAPE),
    ({"batch": -1}, _lib.INTP_ERR_SHAPE),
    ({"batch": 1 << 29, "queries": 1 << 29}, _lib.INTP_ERR_SHAPE),
    ({"states": 0}, _lib.INTP_ERR_SHAPE),                      # nothing to attend to, and no prefix
    ({"dtype": _lib.INTP_F32}, _lib.INTP_ERR_DTYPE),
    ({"scale": 0.0}, _lib.INTP_ERR_ARGUMENT),
    ({"scale": float("inf")}, _lib.INTP_ERR_ARGUMENT),
    ({"scale": float("nan")}, _lib.INTP_ERR_ARGUMENT),
    ({"kernel": 7}, _lib.INTP_ERR_ARGUMENT),
    ({"q": None}, _lib.INTP_ERR_ARGUMENT),
    ({"status": None}, _lib.INTP_ERR_ARGUMENT),
    ({"eight_bit": 1, "k_exponents": FAKE}, _lib.INTP_ERR_ARGUMENT),  # one of the two
    ({"k_exponents": FAKE, "v_exponents": FAKE}, _lib.INTP_ERR_ARGUMENT),  # of 16-bit states
    ({"eight_bit": 1, "kernel": _lib.XATTN_KERNEL_TILES}, _lib.INTP_ERR_UNSUPPORTED),
    ({"eight_bit": 1, "head_dim": 40}, _lib.INTP_ERR_SHAPE),
    ({"eight_bit": 2}, _lib.INTP_ERR_ARGUMENT),
    ({"prefix": 5}, _lib.INTP_ERR_ARGUMENT),                   # no prefix tensors
    ({"q": FAKE + 8}, _lib.INTP_ERR_LAYOUT),
    ({"k_stride": _lib._Stride(12800, 6400, 68, 1)}, _lib.INTP_ERR_LAYOUT),
    ({"v_stride": _lib._Stride(12800, 6400, 64, 2)}, _lib.INTP_ERR_LAYOUT),
    ({"k_stride": _lib._Stride(0, 6400, 64, 1)}, _lib.INTP_ERR_LAYOUT),
    ({"states": 100_000, "k_stride": _lib._Stride(12_800_000, 6_400_000, 64, 1),
      "v_stride": _lib._Stride(12_800_000, 6_400_000, 64, 1)}, _lib.INTP_ERR_ARGUMENT),  # no workspace
])
def test_forward_refuses_before_a_launch(over, status):
    args = _args(**over)
    assert _lib.load().xattn_forward(ctypes.addressof(args), None) == status


def test_backward_refuses_before_a_launch():
    lib = _lib.load()
    assert lib.xattn_backward(None, None) == lib.xattn_forward(None, None) == _lib.INTP_ERR_ARGUMENT
    b = _lib.XattnBackwardArgs()
    b.fwd = _args()
    b.grad_q = FAKE
    assert lib.xattn_backward(ctypes.addressof(b), None) == _lib.INTP_ERR_ARGUMENT  # no row sums
    b.fwd.lse, b.grad_out = FAKE, FAKE
    assert lib.xattn_backward(ctypes.addressof(b), None) == _lib.INTP_ERR_LAYOUT    # strides of grad_out
    b.grad_out_stride = b.fwd.q_stride
    assert lib.xattn_backward(ctypes.addressof(b), None) == _lib.INTP_ERR_ARGUMENT  # no workspace
    b.fwd.prefix, b.fwd.prefix_k, b.fwd.prefix_v = 4, FAKE, FAKE
    assert lib.xattn_backward(ctypes.addressof(b), None) == _lib.INTP_ERR_UNSUPPORTED


def test_cache_refuses_before_a_launch():
    lib = _lib.load()
    a = _lib.StateCacheArgs()
    a.batch, a.groups, a.capacity, a.count, a.head_dim, a.dtype = 1, 2, 16, 4, 64, _lib.INTP_F16
    assert lib.state_cache_write(ctypes.addressof(a), None) == _lib.INTP_ERR_ARGUMENT
    for name in ("k", "v", "k_codes", "v_codes", "k_exponents", "v_exponents"):
        setattr(a, name, FAKE)
    assert lib.state_cache_write(ctypes.addressof(a), None) == _lib.INTP_ERR_LAYOUT
    a.head_dim = 40
    assert lib.state_cache_read(ctypes.addressof(a), None) == _lib.INTP_ERR_SHAPE
    a.head_dim, a.dtype = 64, _lib.INTP_F32
    assert lib.state_cache_read(ctypes.addressof(a), None) == _lib.INTP_ERR_DTYPE
    a.dtype, a.count = _lib.INTP_F16, 0
    assert lib.state_cache_read(ctypes.addressof(a), None) == _lib.INTP_OK  # nothing to do
    assert lib.state_cache_write(None, None) == _lib.INTP_ERR_ARGUMENT


@pytest.mark.parametrize("batch,heads,groups,queries,states,prefix", [
    (1, 3, 3, 1, 196, 0), (64, 32, 8, 1, 4096, 0), (1, 1, 1, 1, 1 << 20, 0), (4, 3, 3, 1, 33, 196),
    (1, 8, 8, 2048, 512, 0), (2, 8, 2, 100, 5000, 0), (64, 32, 8, 1, 0, 16384)])
def test_workspace_holds_every_part(batch, heads, groups, queries, states, prefix):
    """The parts of a split pass, their row sums, and nothing for a pass in one piece."""
    a = _args(batch=batch, heads=heads, groups=groups, queries=queries, states=states, prefix=prefix)
    size = ctypes.c_int64(-1)
    assert _lib.load().xattn_forward_workspace(ctypes.addressof(a), ctypes.byref(size)) == _lib.INTP_OK
    part = batch * heads * queries * (64 + 1) * 4
    assert size.value == 0 or size.value >= 2 * part
    if states and prefix > 1024:
        assert size.value >= 2 * part
    b = _lib.XattnBackwardArgs()
    b.fwd = a
    assert _lib.load().xattn_backward_workspace(ctypes.addressof(b), ctypes.byref(size)) == _lib.INTP_OK
    assert size.value >= (batch * heads * queries * 2 * 4 if states else 0)


def test_operators_refuse_cpu_tensors():
    q = torch.randn(1, 2, 3, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        cross_attention(q, q, q, scale=0.25)
    with pytest.raises(ValueError, match="CUDA"):
        cross_attention(q.requires_grad_(), q, q, scale=0.25)
    q = q.detach()
    with pytest.raises(ValueError, match="CUDA"):
        cross_attention_forward(q, q, q, scale=0.25)
    with pytest.raises(ValueError, match="CUDA"):
        cross_attention_backward(q, q, q, q, q[..., 0].float(), q, scale=0.25)
    with pytest.raises(ValueError, match="CUDA"):
        shared_prefix_attention(q, q[0], q[0], q, q, scale=0.25)
    with pytest.raises(ValueError, match="CUDA"):
        StateCache.empty(1, 2, 8, 16, device="cpu")
    with pytest.raises(ValueError, match="StateCache"):
        cached_cross_attention(q, q, scale=0.25)


def test_oracle_gradients_match_differences():
    """The gradient formulas against central differences of the forward, in float64."""
    g = torch.Generator().manual_seed(5)
    q, k, v, grad = (torch.randn(s, generator=g, dtype=torch.float64).half()
                     for s in ((2, 4, 3, 8), (2, 2, 5, 8), (2, 2, 5, 8), (2, 4, 3, 8)))
    lengths = [5, 3]
    grads, _ = oracle.cross_attention_gradients(q, k, v, grad, scale=0.3, lengths=lengths)

    def loss(tensors):
        out, _, _ = oracle.cross_attention(*tensors, scale=0.3, lengths=lengths, out_dtype=torch.float16,
                                           p_dtype=torch.float16)
        return float((out * grad.double()).sum())

    step = 1e-5
    for which in range(3):
        base = [t.double() for t in (q, k, v)]
        flat = grads[which].reshape(-1)
        for i in range(0, flat.numel(), 7):
            moved = []
            for sign in (1, -1):
                t = base[which].clone()
                t.view(-1)[i] += sign * step
                moved.append(loss([t if j == which else base[j] for j in range(3)]))
            # central differences: O(step^2) truncation and 1e-15 / step cancellation
            assert abs((moved[0] - moved[1]) / (2 * step) - float(flat[i])) < 1e-7


def test_oracle_e4m3_table_matches_torch():
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(codes, oracle.e4m3_values())
    x = torch.randn(7, 33, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    values, exponents = oracle.quantise_rows(x)
    again = (x.double() / torch.exp2(exponents.double())[:, None]).to(torch.float8_e4m3fn).double()
    assert torch.equal(values, again * torch.exp2(exponents.double())[:, None])


def test_statistics_are_read_behind_their_writer():
    """The gradient kernels start while the kernel that writes the row statistics may still run: a
    read-only load could be moved before the wait or hit an old line, and dk / dv, which does not
    wait itself, relies on dq's wait and fence standing before dq lets it start."""
    text = (HEADER.parent.parent / "intp_preliminary_b200" / "csrc" / "cross_attention_backward.cu").read_text()
    body = text[text.index("xattn_grad_kernel(const"):text.index("split sums")]
    pointer = re.search(r"const float\* (\w+) = a\.stats", body).group(1)
    loads = re.findall(rf"(\w+)\({pointer}\b", body)
    assert loads and set(loads) == {"__ldcg"}
    assert re.search(r"if \(!KV\) \{\s*wait_previous_kernel\(\);[^}]*__threadfence\(\);[^}]*\}", body)
    assert body.index("wait_previous_kernel();") < body.index("__threadfence();") < body.index("allow_next_kernel();")
    assert body.count("allow_next_kernel();") == 1 and "a.after_stats = bp.dq == nullptr;" in text


@pytest.mark.parametrize("heads,queries,status", [
    (2, (1 << 30) - 1, _lib.INTP_ERR_SHAPE),    # 2^31 - 2 rows of a key head: their last tile ends past 2^31
    (2, (1 << 30) - 128, _lib.INTP_ERR_SHAPE),
    (2, (1 << 30) - 129, _lib.INTP_OK),         # the last tile of 256 rows ends at 2^31 - 256
    (1, 1 << 30, _lib.INTP_OK),
])
def test_rows_whose_last_tile_leaves_32_bits_are_refused(heads, queries, status):
    a = _args(batch=1, heads=heads, groups=1, queries=queries, states=300)
    size = ctypes.c_int64()
    assert _lib.load().xattn_forward_workspace(ctypes.addressof(a), ctypes.byref(size)) == status
    b = _lib.XattnBackwardArgs()
    b.fwd = a
    assert _lib.load().xattn_backward_workspace(ctypes.addressof(b), ctypes.byref(size)) == status


def test_a_write_to_a_cache_without_room_has_nothing_to_do():
    """Rows outside the cache are skipped, and all are; a cache of no states has no memory."""
    a = _lib.StateCacheArgs()
    a.batch, a.groups, a.capacity, a.count, a.head_dim, a.dtype = 1, 2, 0, 4, 64, _lib.INTP_F16
    a.k = a.v = FAKE
    a.k_stride = a.v_stride = _lib._Stride(512, 256, 64, 1)
    assert _lib.load().state_cache_write(ctypes.addressof(a), None) == _lib.INTP_OK
    a.capacity = 1
    assert _lib.load().state_cache_write(ctypes.addressof(a), None) == _lib.INTP_ERR_ARGUMENT


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("states,dim", [(5, 16), (17, 16), (60, 16), (17, 64)])
def test_two_part_bound_tells_one_rounding_of_the_probabilities_from_two_parts(states, dim, dtype):
    """The bound that the few-rows kernel is held to fails for probabilities rounded to 16 bits, and
    for low parts that miss their place, and holds for two parts."""
    g = torch.Generator().manual_seed(states)
    q, k, v = (torch.randn(s, generator=g).to(dtype) for s in ((4, 4, 4, dim), (4, 4, states, dim), (4, 4, states, dim)))
    want, _, bound = oracle.cross_attention(q, k, v, scale=dim ** -0.5, two_part=True)
    s = (q.double() @ k.double().transpose(-1, -2)) * dim ** -0.5
    p = torch.exp(s - s.amax(-1, keepdim=True))
    high = p.to(dtype).double()
    low = (p - high).to(dtype).double()
    for operand, holds in ((high, False), (high + low, True), (high + low.flip(-1), False)):
        got = ((operand @ v.double()) / p.sum(-1, keepdim=True)).to(dtype).double()
        assert bool(((got - want).abs() <= bound).all()) == holds


def _operator_calls(make):
    """Every operator's call on the tensors that ``make(shape)`` gives, one of them marked by it."""
    plain = torch.zeros(1, 2, 3, 16, dtype=torch.bfloat16)
    marked = make(plain)
    lse = torch.zeros(1, 2, 3)
    return [lambda: cross_attention(marked, plain, plain, scale=0.25),
            lambda: cross_attention(plain, plain, marked, scale=0.25),
            lambda: cross_attention(plain.clone().requires_grad_(), marked, plain, scale=0.25),
            lambda: cross_attention_forward(plain, marked, plain, scale=0.25),
            lambda: cross_attention_backward(plain, plain, plain, plain, lse, marked, scale=0.25),
            lambda: shared_prefix_attention(plain, plain[0], marked[0], plain, plain, scale=0.25),
            lambda: shared_prefix_attention(plain, plain[0], plain[0], marked, plain, scale=0.25)]


def test_tangents_are_refused():
    """A forward-mode tangent would be lost: the kernels know nothing of it."""
    forward_ad = torch.autograd.forward_ad
    with forward_ad.dual_level():
        for call in _operator_calls(lambda t: forward_ad.make_dual(t, torch.ones_like(t))):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
        for call in _operator_calls(lambda t: t):  # the primal alone gets as far as before
            with pytest.raises(ValueError, match="CUDA"):
                call()


def test_tracing_is_refused():
    """A trace would hold the output's allocation and not the kernel that fills it."""
    for call in _operator_calls(lambda t: t):
        with pytest.raises(ValueError, match="traced"):
            torch.jit.trace(lambda t: (call(), t)[1], torch.zeros(1), check_trace=False)


@pytest.fixture
def recorded(monkeypatch):
    """The operators on CPU tensors with every library call recorded instead of made: what a call's
    argument block says can be compared with the tensors it points to."""
    module = sys.modules["intp_preliminary_b200.cross_attention"]
    blocks = []
    monkeypatch.setattr(module, "_check_states", lambda q, k, v: None)
    monkeypatch.setattr(module, "_status", lambda device: torch.zeros(1, dtype=torch.int32))
    monkeypatch.setattr(module, "_plans", {})
    monkeypatch.setattr(module, "_call", lambda fn, block, index, what: blocks.append(block))
    return blocks


def _strided_leaves():
    q = torch.randn(2, 7, 4, 16).bfloat16().requires_grad_()
    kv = torch.randn(2, 30, 2, 2, 16).bfloat16().requires_grad_()
    return q.transpose(1, 2), kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)


@pytest.mark.parametrize("form", ["same", "contiguous", "padded", "unaligned"])
def test_backward_describes_the_tensors_that_hooks_return(recorded, form):
    """Hooks on saved tensors (offloading, compression) may return other strides than were saved: the
    backward's block must hold the strides and the 16-byte rows of what it points to."""
    held = {}

    def pack(t):
        if form == "same" or t.dtype != torch.bfloat16:
            kept = t
        elif form == "contiguous":
            kept = t.clone(memory_format=torch.contiguous_format)
        else:
            wide = torch.empty(*t.shape[:-1], t.shape[-1] + 8, dtype=t.dtype)
            kept = wide[..., 8:] if form == "padded" else wide[..., 1:t.shape[-1] + 1]
            kept.copy_(t)
        held[kept.data_ptr()] = kept
        return kept

    q, k, v = _strided_leaves()
    lengths = torch.tensor([30, 11], dtype=torch.int32)
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        out = cross_attention(q, k, v, scale=0.25, lengths=lengths)
    torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
    args = _lib.XattnBackwardArgs.from_buffer_copy(recorded[-1])
    f = args.fwd
    assert (f.batch, f.heads, f.groups, f.queries, f.states, f.head_dim) == (2, 4, 2, 7, 30, 16)
    for pointer, stride in ((f.q, f.q_stride), (f.k, f.k_stride), (f.v, f.v_stride), (f.out, f.out_stride)):
        assert pointer % 16 == 0
        if form == "unaligned":
            assert pointer not in held and list(stride[2:]) == [16, 1]
        else:
            assert tuple(stride) == held[pointer].stride()
    assert f.lengths in held and f.lse in held


def test_a_cache_keeps_its_tensors(monkeypatch):
    """Calls take the layout that was checked when the cache was made: its tensors cannot be replaced."""
    module = sys.modules["intp_preliminary_b200.state_cache"]
    monkeypatch.setattr(module, "_check_tensors", lambda *tensors: None)
    monkeypatch.setattr(module, "_keep", lambda key, plan: plan)
    cache = StateCache.empty(2, 2, 8, 16, device="cpu")
    for name in ("keys", "values", "key_exponents", "value_exponents", "layout"):
        with pytest.raises(AttributeError):
            setattr(cache, name, getattr(cache, name)[:1])
    assert cache.shape == tuple(cache.keys.shape) == (2, 2, 8, 16)
