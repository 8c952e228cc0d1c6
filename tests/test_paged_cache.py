"""Positions, the paged cache and attention over it without a GPU: the C ABI's structs and
refusals, CPU tensors, and the oracle itself."""

import ctypes
import re
from pathlib import Path

import pytest
import torch

from intp_preliminary_b200 import PagedCache, RotaryAxes, _lib, paged_attention, rotate_positions
from oracle import cross_attention as cross_oracle
from oracle import paged as oracle

HEADER = Path(__file__).resolve().parent.parent / "include" / "intp_b200.h"
FAKE = 1 << 20  # never dereferenced: every call below is refused before a launch


@pytest.mark.parametrize("name,mirror", [("rotary_args", _lib.RotaryArgs), ("paged_attention_args", _lib.PagedAttentionArgs)])
def test_struct_layout_matches_header_field_order(name, mirror):
    text = HEADER.read_text()
    body = text[text.index(f"typedef struct {name} {{"):text.index(f"}} {name};")]
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    assert re.findall(r"(\w+)(?:\[\d\])?\s*[;,]", body) == [f[0] for f in mirror._fields_]


def _rotary(**over):
    a = _lib.RotaryArgs()
    a.batch, a.heads, a.groups, a.rows, a.head_dim, a.rotary_dim, a.axes = 2, 4, 2, 3, 64, 64, 1
    a.dtype, a.position_type = _lib.INTP_BF16, _lib.ROTARY_INT32
    a.q = a.k = a.q_out = a.k_out = a.turns = a.axis = a.positions = FAKE
    a.q_stride = a.q_out_stride = _lib._Stride(768, 192, 64, 1)
    a.k_stride = a.k_out_stride = a.v_stride = a.v_out_stride = _lib._Stride(384, 192, 64, 1)
    for key, value in over.items():
        setattr(a, key, value)
    return a


def _append(**over):
    more = dict(v=FAKE, v_out=FAKE, page_table=FAKE, pages=10, page_size=16, table_width=4, table_stride=4,
                k_out_stride=_lib._Stride(2048, 1024, 64, 1), v_out_stride=_lib._Stride(2048, 1024, 64, 1))
    return _rotary(**{**more, **over})


COMMON = [
    ({"head_dim": 60}, _lib.INTP_ERR_SHAPE),
    ({"head_dim": 136}, _lib.INTP_ERR_SHAPE),
    ({"rotary_dim": 72}, _lib.INTP_ERR_SHAPE),                 # more than the head has
    ({"rotary_dim": 36}, _lib.INTP_ERR_SHAPE),
    ({"batch": -1}, _lib.INTP_ERR_SHAPE),
    ({"batch": 1 << 20, "rows": 1 << 20}, _lib.INTP_ERR_SHAPE),
    ({"position_type": 4}, _lib.INTP_ERR_ARGUMENT),
    ({"positions": None}, _lib.INTP_ERR_ARGUMENT),
    ({"turns": None}, _lib.INTP_ERR_ARGUMENT),
    ({"axis": None}, _lib.INTP_ERR_ARGUMENT),
    ({"q_out": None}, _lib.INTP_ERR_ARGUMENT),
    ({"q": FAKE + 8}, _lib.INTP_ERR_LAYOUT),
    ({"k_out": FAKE + 8}, _lib.INTP_ERR_LAYOUT),
    ({"q_stride": _lib._Stride(768, 192, 68, 1)}, _lib.INTP_ERR_LAYOUT),
    ({"q_stride": _lib._Stride(768, 192, 64, 2)}, _lib.INTP_ERR_LAYOUT),
    ({"q_stride": _lib._Stride(-768, 192, 64, 1)}, _lib.INTP_ERR_LAYOUT),
    ({"q_out_stride": _lib._Stride(0, 192, 64, 1)}, _lib.INTP_ERR_LAYOUT),  # results are not broadcast
    ({"k_out_stride": _lib._Stride(384, 0, 64, 1)}, _lib.INTP_ERR_LAYOUT),
    ({"batch": 0}, _lib.INTP_OK),
    ({"rows": 0}, _lib.INTP_OK),
]


@pytest.mark.parametrize("over,status", COMMON + [
    ({"dtype": 5}, _lib.INTP_ERR_DTYPE),
    ({"v": FAKE}, _lib.INTP_ERR_ARGUMENT),                     # of an append
    ({"page_table": FAKE}, _lib.INTP_ERR_ARGUMENT),
    ({"position_type": _lib.ROTARY_ROW}, _lib.INTP_ERR_ARGUMENT),
])
def test_rotation_refuses_before_a_launch(over, status):
    assert _lib.load().rotary_positions(ctypes.addressof(_rotary(**over)), None) == status
    assert _lib.load().rotary_positions(None, None) == _lib.INTP_ERR_ARGUMENT


@pytest.mark.parametrize("over,status", COMMON + [
    ({"dtype": _lib.INTP_F32}, _lib.INTP_ERR_DTYPE),
    ({"page_table": None}, _lib.INTP_ERR_ARGUMENT),
    ({"k": None}, _lib.INTP_ERR_ARGUMENT),
    ({"v": None}, _lib.INTP_ERR_ARGUMENT),
    ({"v_out": None}, _lib.INTP_ERR_ARGUMENT),
    ({"page_size": 0}, _lib.INTP_ERR_SHAPE),
    ({"pages": 1 << 31}, _lib.INTP_ERR_SHAPE),
])
def test_append_refuses_before_a_launch(over, status):
    assert _lib.load().paged_cache_append(ctypes.addressof(_append(**over)), None) == status
    assert _lib.load().paged_cache_append(None, None) == _lib.INTP_ERR_ARGUMENT


@pytest.mark.parametrize("over,status", [
    ({"heads": 3}, _lib.INTP_ERR_SHAPE),
    ({"head_dim": 60}, _lib.INTP_ERR_SHAPE),
    ({"head_dim": 136}, _lib.INTP_ERR_SHAPE),
    ({"batch": -1}, _lib.INTP_ERR_SHAPE),
    ({"pages": 0}, _lib.INTP_ERR_SHAPE),
    ({"page_size": 0}, _lib.INTP_ERR_SHAPE),
    ({"table_width": 0}, _lib.INTP_ERR_SHAPE),
    ({"table_width": 1 << 28, "page_size": 16}, _lib.INTP_ERR_SHAPE),  # positions leave 2^30
    ({"queries": 1 << 30}, _lib.INTP_ERR_SHAPE),
    ({"window": -1}, _lib.INTP_ERR_SHAPE),
    ({"sinks": -1}, _lib.INTP_ERR_SHAPE),
    ({"dtype": _lib.INTP_F32}, _lib.INTP_ERR_DTYPE),
    ({"scale": 0.0}, _lib.INTP_ERR_ARGUMENT),
    ({"scale": float("inf")}, _lib.INTP_ERR_ARGUMENT),
    ({"scale": float("nan")}, _lib.INTP_ERR_ARGUMENT),
    ({"q": None}, _lib.INTP_ERR_ARGUMENT),
    ({"v": None}, _lib.INTP_ERR_ARGUMENT),
    ({"page_table": None}, _lib.INTP_ERR_ARGUMENT),
    ({"start": None}, _lib.INTP_ERR_ARGUMENT),
    ({"q": FAKE + 8}, _lib.INTP_ERR_LAYOUT),
    ({"cache_stride": _lib._Stride(2048, 1024, 68, 1)}, _lib.INTP_ERR_LAYOUT),
    ({"cache_stride": _lib._Stride(2048, 0, 64, 1)}, _lib.INTP_ERR_LAYOUT),
    ({"cache_stride": _lib._Stride(1 << 32, 1024, 64, 1)}, _lib.INTP_ERR_LAYOUT),  # places leave 32 bits
    ({"out_stride": _lib._Stride(768, 192, 64, 2)}, _lib.INTP_ERR_LAYOUT),
    ({"kernel": 3}, _lib.INTP_ERR_ARGUMENT),
    ({"kernel": _lib.PAGED_KERNEL_PARTS}, _lib.INTP_ERR_ARGUMENT),              # no workspace
    ({"kernel": _lib.PAGED_KERNEL_PARTS, "queries": 9}, _lib.INTP_ERR_UNSUPPORTED),
    ({"kernel": _lib.PAGED_KERNEL_PARTS, "batch": 1025}, _lib.INTP_ERR_UNSUPPORTED),
    ({"batch": 0}, _lib.INTP_OK),
    ({"queries": 0}, _lib.INTP_OK),
])
def test_attention_refuses_before_a_launch(over, status):
    a = _lib.PagedAttentionArgs()
    a.batch, a.heads, a.groups, a.queries, a.head_dim = 2, 4, 2, 3, 64
    a.pages, a.page_size, a.table_width, a.table_stride = 10, 16, 4, 4
    a.scale, a.dtype = 0.125, _lib.INTP_BF16
    a.q = a.k = a.v = a.out = a.page_table = a.start = FAKE
    a.q_stride = a.out_stride = _lib._Stride(768, 192, 64, 1)
    a.cache_stride = _lib._Stride(2048, 1024, 64, 1)
    for key, value in over.items():
        setattr(a, key, value)
    assert _lib.load().paged_attention(ctypes.addressof(a), None) == status
    assert _lib.load().paged_attention(None, None) == _lib.INTP_ERR_ARGUMENT


def test_rotary_axes_refuse():
    for frequencies, axes, message in (
            ([1.0] * 4, [0] * 5, "length"), ([1.0] * 6, [0] * 6, "multiple of 4"), ([], [], "multiple of 4"),
            ([1.0] * 68, [0] * 68, "multiple of 4"), ([1.0, 1.0, 1.0, float("nan")], [0] * 4, "finite"),
            ([1.0] * 4, [0, 0, 2, 2], "without gaps"), ([1.0] * 4, [-1, 0, 0, 0], "without gaps"),
            ([1.0] * 4, [0] * 4, "CUDA")):
        with pytest.raises(ValueError, match=message):
            RotaryAxes(frequencies, axes, device="cpu")
    for sections, base, message in (([], 1e4, "at least one"), ([4, 0], 1e4, "at least one"), ([4], 0.0, "base"),
                                    ([4], float("inf"), "base")):
        with pytest.raises(ValueError, match=message):
            RotaryAxes.sections(sections, base=base, device="cpu")


def _fake_rotary(pairs=8, axes=1):
    r = RotaryAxes.__new__(RotaryAxes)
    r._axes, r._frequencies, r._interleaved, r._device = tuple(i % axes for i in range(pairs)), (1.0,) * pairs, False, torch.device("cpu")
    r._layout = (pairs, axes, False, r._device)
    return r


def test_operators_refuse_cpu_tensors():
    q, at = torch.zeros(1, 2, 3, 16, dtype=torch.bfloat16), torch.zeros(1, 3, 1, dtype=torch.int32)
    rotary = _fake_rotary()
    for k in (None, q):
        with pytest.raises(ValueError, match="CUDA"):
            rotate_positions(q, k, rotary=rotary, positions=at)
    with pytest.raises(ValueError, match="CUDA"):
        rotate_positions(q.clone().requires_grad_(), rotary=rotary, positions=at)
    with pytest.raises(ValueError, match="RotaryAxes"):
        rotate_positions(q, rotary=None, positions=at)
    with pytest.raises(ValueError, match="positions"):
        rotate_positions(q, rotary=rotary, positions=None)
    with pytest.raises(ValueError, match="gradient"):
        rotate_positions(q, rotary=rotary, positions=at.float().requires_grad_())
    with pytest.raises(ValueError, match="CUDA"):
        PagedCache(q, q)
    with pytest.raises(ValueError, match="CUDA"):
        PagedCache.empty(4, 2, 16, 16, device="cpu")
    with pytest.raises(ValueError, match="PagedCache"):
        paged_attention(q, q, page_table=at[0], start=at[0, 0], scale=0.25)


def test_tangents_and_traces_are_refused():
    forward_ad = torch.autograd.forward_ad
    q, at, rotary = torch.zeros(1, 2, 3, 16, dtype=torch.bfloat16), torch.zeros(3, 1), _fake_rotary()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        for a, b in ((dual, q), (q, dual), (dual, None)):
            with pytest.raises(ValueError, match="forward-mode"):
                rotate_positions(a, b, rotary=rotary, positions=at)
    with pytest.raises(ValueError, match="traced"):
        torch.jit.trace(lambda t: (rotate_positions(q, rotary=rotary, positions=at), t)[1], torch.zeros(1), check_trace=False)


@pytest.mark.parametrize("interleaved", [False, True])
def test_oracle_turns_as_complex_numbers(interleaved):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, 3, 5, 12, generator=g, dtype=torch.float64)
    positions = torch.randint(0, 1000, (2, 5, 2), generator=g).double()
    frequencies, axes = [1.0, 0.3, 0.01, 2.0], [0, 1, 1, 0]
    y, _ = oracle.turn(x, positions, frequencies, axes, interleaved=interleaved)
    pairs = [(2 * i, 2 * i + 1) if interleaved else (i, 4 + i) for i in range(4)]
    for i, (one, two) in enumerate(pairs):
        z = torch.complex(x[..., one], x[..., two]) * torch.exp(1j * frequencies[i] * positions[:, None, :, axes[i]])
        # a product of angles below 2000, rounded at 2^-53: 2e-13 each way
        assert (torch.complex(y[..., one], y[..., two]) - z).abs().max() < 1e-12
    assert torch.equal(y[..., 8:], x[..., 8:])
    back, _ = oracle.turn(y, positions, frequencies, axes, interleaved=interleaved, inverse=True)
    assert (back - x).abs().max() < 1e-14


def test_oracle_gradient_of_a_rotation_matches_differences():
    g = torch.Generator().manual_seed(2)
    x, grad = (torch.randn(1, 2, 3, 8, generator=g, dtype=torch.float64) for _ in range(2))
    at = torch.randn(1, 3, 1, generator=g)
    back, _ = oracle.turn(grad, at, [1.0, 0.5, 0.2, 0.1], [0] * 4, inverse=True)
    for i in range(0, x.numel(), 5):
        moved = []
        for step in (0.5, -0.5):  # linear: any step will do
            y = x.clone()
            y.view(-1)[i] += step
            moved.append(float((oracle.turn(y, at, [1.0, 0.5, 0.2, 0.1], [0] * 4)[0] * grad).sum()))
        assert abs(moved[0] - moved[1] - float(back.view(-1)[i])) < 1e-12


@pytest.mark.parametrize("page_size", [1, 3, 16])
def test_oracle_attends_like_cross_attention_over_the_gathered_states(page_size):
    """A sequence of n states read by its last token is cross attention to n states."""
    g = torch.Generator().manual_seed(page_size)
    k, v = (torch.randn(2, 2, 20, 8, generator=g).bfloat16() for _ in range(2))
    q = torch.randn(2, 4, 1, 8, generator=g).bfloat16()
    width = (20 + page_size - 1) // page_size
    table = torch.randperm(2 * width + 2, generator=g)[:2 * width].reshape(2, width).to(torch.int32)
    keys, values = (torch.full((2 * width + 2, 2, page_size, 8), float("nan")).bfloat16() for _ in range(2))
    lengths = [20, 7]
    oracle.append(keys, values, k, v, page_table=table, start=[0, 0], counts=lengths)
    got, bound = oracle.attend(q, keys, values, page_table=table, start=[x - 1 for x in lengths], scale=0.3)
    want, _, want_bound = cross_oracle.cross_attention(q, k, v, scale=0.3, lengths=lengths, two_part=True)
    assert (got - want).abs().max() < 1e-14
    # one more u^2 of the same sum that the other bound holds one of
    assert bool((bound >= want_bound).all()) and bool((bound <= 2 * want_bound).all())


def test_a_copied_rotary_points_into_its_own_tables():
    """Without a GPU, on a stand-in whose tables lie in the host's memory."""
    import copy
    import pickle

    rotary = _fake_rotary(axes=2)
    rotary._lay_out()
    layer = torch.nn.Module()
    layer.rotary = rotary
    for other in (copy.copy(rotary), copy.deepcopy(rotary), pickle.loads(pickle.dumps(rotary)), copy.deepcopy(layer).rotary):
        assert other._pointers == (other._tables.data_ptr(), other._tables.data_ptr() + 8 * 8)
        assert other._tables.data_ptr() != rotary._tables.data_ptr() and torch.equal(other._tables, rotary._tables)
        assert (other.frequencies, other.axes, other._layout) == (rotary.frequencies, rotary.axes, rotary._layout)
    assert b"_tables" not in pickle.dumps(rotary)


def test_a_cache_loaded_onto_the_host_is_refused():
    """Its calls take the layout and device that were checked when it was made, so loading checks again."""
    import io

    from intp_preliminary_b200 import StateCache

    half, byte = torch.zeros(2, 1, 4, 16, dtype=torch.bfloat16), torch.zeros(2, 1, 4, dtype=torch.uint8)
    paged, state = PagedCache.__new__(PagedCache), StateCache.__new__(StateCache)
    paged._keys = paged._values = half
    state._keys = state._values = half.to(torch.float8_e4m3fn)
    state._key_exponents = state._value_exponents = byte
    paged._layout = state._layout = ("as it was on a GPU",)
    for cache in (paged, state):
        file = io.BytesIO()
        torch.save(cache, file)
        file.seek(0)
        with pytest.raises(ValueError, match="CUDA"):
            torch.load(file, weights_only=False)


@pytest.mark.parametrize("which", ["_keys", "_values"])
def test_a_pool_that_comes_to_require_a_gradient_is_refused(which):
    """Not only when the cache is made: a tensor may be marked later."""
    cache = PagedCache.__new__(PagedCache)
    cache._keys, cache._values = (torch.zeros(2, 1, 4, 16, dtype=torch.bfloat16) for _ in range(2))
    cache._layout = ()
    q, start = torch.zeros(1, 1, 1, 16, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="no backward"):
        paged_attention(q, cache, page_table=start[None], start=start, scale=0.25, out=q.clone().requires_grad_())
    getattr(cache, which).requires_grad_()
    with pytest.raises(ValueError, match="no backward"):
        paged_attention(q, cache, page_table=start[None], start=start, scale=0.25)
    with pytest.raises(ValueError, match="no backward"):
        cache.append(q, q, page_table=start[None], start=start)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        paged_attention(q, cache, page_table=start[None], start=start, scale=0.25)


@pytest.mark.parametrize("needs_q,needs_k", [(True, True), (True, False), (False, True)])
@pytest.mark.parametrize("create_graph", [False, True])
def test_only_what_needs_a_gradient_gets_one(monkeypatch, needs_q, needs_k, create_graph):
    """The autograd node alone, over a stand-in for the kernel that doubles."""
    import importlib

    module = importlib.import_module("intp_preliminary_b200.rotary")
    turned = []

    def double(q, k, rotary, positions, inverse):
        turned.append((q is not None) + (k is not None))
        return q.detach() * 2, None if k is None else k.detach() * 2

    monkeypatch.setattr(module, "_rotate", double)
    q, k = (torch.ones(1, 2, 3, 8, requires_grad=needs) for needs in (needs_q, needs_k))
    outs = rotate_positions(q, k, rotary=_fake_rotary(4), positions=torch.zeros(3, 1))
    assert [t.requires_grad for t in outs] == [needs_q, needs_k]
    leaves = [t for t in (q, k) if t.requires_grad]
    grads = torch.autograd.grad(sum(t.sum() for t in outs), leaves, create_graph=create_graph)
    assert all(torch.equal(g, torch.full_like(g, 2)) for g in grads)
    assert turned == [2, len(leaves)]


def test_tables_are_held_for_every_stream_that_reads_them(monkeypatch):
    """Without a GPU: the launch's stream and the tables' allocator are stand-ins."""
    import importlib

    module = importlib.import_module("intp_preliminary_b200.rotary")
    held, now = [], [7]

    class Tables:
        def data_ptr(self):
            return 4096

        def record_stream(self, stream):
            held.append(stream)

    rotary = _fake_rotary()
    rotary._lay_out()
    rotary._tables, rotary._streams = Tables(), {7}
    monkeypatch.setattr(module, "_current_stream", lambda index: now[0])
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device: f"stream {now[0]}")
    for now[0] in (7, 9, 9, 7, 8, 9):
        assert rotary._launch_pointers() == (4096, 4096 + 8 * 8)
    assert held == ["stream 9", "stream 8"]
