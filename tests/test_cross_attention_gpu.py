"""Cross attention on the GPU against the float64 oracle, elementwise within the
oracle's error bounds (derived there from where the kernels round)."""

import ctypes

import pytest
import torch
import torch.utils.checkpoint

from intp_preliminary_b200 import (_lib, check_device_status, cross_attention, cross_attention_backward,
                                   cross_attention_forward, shared_prefix_attention)
from oracle import cross_attention as oracle

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _device_status(cuda_device):
    yield
    check_device_status(cuda_device)


def _normal(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def _inputs(batch, heads, groups, queries, states, dim, dtype, seed=0):
    return (_normal((batch, heads, queries, dim), dtype, seed + 1), _normal((batch, groups, states, dim), dtype, seed + 2),
            _normal((batch, groups, states, dim), dtype, seed + 3))


def _assert_within(got, want, bound):
    off = (got.detach().cpu().double() - want).abs()
    assert torch.isfinite(off).all()
    worst = (off / bound).max()
    assert (off <= bound).all(), f"error {float(worst):.2f} times the bound"


def _check_forward(q, k, v, lengths, device, kernel, scale=None):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    want, lse, bound = oracle.cross_attention(q, k, v, scale=scale, lengths=lengths)
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=device)
    out, got_lse = cross_attention_forward(q.to(device), k.to(device), v.to(device), scale=scale, lengths=lens,
                                           want_lse=True, kernel=kernel)
    _assert_within(out, want, bound)
    got_lse = got_lse.cpu().double()
    empty = torch.isinf(lse)
    assert torch.equal(torch.isinf(got_lse), empty)
    assert (got_lse - lse)[~empty].abs().max() <= oracle.LSE if (~empty).any() else True


SHAPES = [
    # batch, heads, groups, queries, states, dim, lengths
    (1, 1, 1, 1, 1, 8, None),
    (2, 3, 3, 5, 17, 64, None),
    (1, 4, 2, 3, 127, 40, None),
    (2, 2, 1, 64, 128, 64, [128, 77]),
    (3, 2, 2, 33, 129, 72, [0, 1, 129]),
    (2, 4, 4, 130, 300, 80, [299, 128]),
    (1, 6, 2, 100, 513, 128, [511]),
    (2, 2, 2, 257, 64, 96, None),
    (1, 8, 1, 70, 1000, 128, [999]),
    (4, 3, 3, 1, 196, 64, [196, 0, 63, 64]),
    (2, 8, 2, 1, 2500, 128, [2500, 1300]),
    (1, 16, 2, 2, 3001, 64, None),
]


@pytest.mark.parametrize("kernel", ["rows", "tiles", "auto"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_matches_oracle(cuda_device, shape, dtype, kernel):
    *sizes, lengths = shape
    q, k, v = _inputs(*sizes, dtype)
    _check_forward(q, k, v, lengths, cuda_device, kernel)


@pytest.mark.parametrize("kernel", ["rows", "tiles"])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), "lowest"])
def test_padded_states_never_show(cuda_device, kernel, poison):
    """Whatever sits past a length: NaN, infinities, the type's lowest value."""
    q, k, v = _inputs(3, 4, 2, 9, 700, 64, BF16, seed=9)
    lengths = [0, 333, 640]
    value = torch.finfo(BF16).min if poison == "lowest" else poison
    clean = [t.clone() for t in (k, v)]
    for b, n in enumerate(lengths):
        k[b, :, n:] = value
        v[b, :, n:] = value
        for t in clean:
            t[b, :, n:] = 0
    lens = torch.tensor(lengths, dtype=torch.int32, device=cuda_device)
    a, lse = cross_attention_forward(*(t.to(cuda_device) for t in (q, k, v)), scale=0.125, lengths=lens, want_lse=True,
                                     kernel=kernel)
    b, lse0 = cross_attention_forward(q.to(cuda_device), *(t.to(cuda_device) for t in clean), scale=0.125, lengths=lens,
                                      want_lse=True, kernel=kernel)
    assert torch.equal(a, b) and torch.equal(lse, lse0)
    assert a[0].abs().max() == 0 and torch.isinf(lse[0]).all()
    grad = torch.randn_like(a)
    got = cross_attention_backward(*(t.to(cuda_device) for t in (q, k, v)), a, lse, grad, scale=0.125, lengths=lens)
    ref = cross_attention_backward(q.to(cuda_device), *(t.to(cuda_device) for t in clean), a, lse, grad, scale=0.125,
                                   lengths=lens)
    for x, y in zip(got, ref):
        assert torch.equal(x, y)
    for x in got[1:]:
        for i, n in enumerate(lengths):
            assert x[i, :, n:].abs().sum() == 0


@pytest.mark.parametrize("kernel", ["rows", "tiles"])
def test_lengths_outside_the_range_are_clamped(cuda_device, kernel):
    q, k, v = (t.to(cuda_device) for t in _inputs(3, 2, 2, 4, 150, 64, BF16, seed=3))
    wild = torch.tensor([-5, 1000, 2 ** 40], device=cuda_device)
    got, _ = cross_attention_forward(q, k, v, scale=0.125, lengths=wild, kernel=kernel)
    tame = torch.tensor([0, 150, 150], dtype=torch.int32, device=cuda_device)
    assert torch.equal(got, cross_attention_forward(q, k, v, scale=0.125, lengths=tame, kernel=kernel)[0])


@pytest.mark.parametrize("kernel", ["rows", "tiles"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("states,queries,dim,flat", [(1, 1, 64, True), (300, 1, 64, True), (300, 6, 128, False),
                                                     (2500, 1, 128, False), (37, 3, 72, False)])
def test_an_infinite_value_makes_its_column_infinite(cuda_device, states, queries, dim, flat, dtype, kernel):
    """Every weight is positive, so p * inf is inf of the value's sign; the other columns do not see it."""
    q, k, v = _inputs(1, 2, 1, queries, states, dim, dtype, seed=states)
    if flat:
        q.zero_()
    want, _, bound = oracle.cross_attention(q, k, v, scale=dim ** -0.5)
    v[0, 0, states // 2, 3], v[0, 0, states - 1, dim - 1] = float("inf"), -float("inf")
    got, _ = cross_attention_forward(*(t.to(cuda_device) for t in (q, k, v)), scale=dim ** -0.5, kernel=kernel)
    assert (got[..., 3] == float("inf")).all() and (got[..., dim - 1] == -float("inf")).all()
    rest = [c for c in range(dim) if c not in (3, dim - 1)]
    _assert_within(got[..., rest], want[..., rest], bound[..., rest])


@pytest.mark.parametrize("kernel", ["rows", "tiles"])
def test_values_that_are_not_finite_spread_as_in_a_softmax(cuda_device, kernel):
    """A NaN score makes its row NaN; a key with -inf scores drops out; a row of them gives zeros."""
    q, k, v = _inputs(1, 1, 1, 6, 300, 64, BF16, seed=4)
    q = q.abs() + 0.1
    k[0, 0, 290] = -float("inf")
    got, lse = cross_attention_forward(*(t.to(cuda_device) for t in (q, k, v)), scale=0.125, want_lse=True, kernel=kernel)
    keep = [i for i in range(300) if i != 290]
    want, _, bound = oracle.cross_attention(q, k[:, :, keep], v[:, :, keep], scale=0.125)
    _assert_within(got, want, bound)
    k[:] = -float("inf")
    got, lse = cross_attention_forward(*(t.to(cuda_device) for t in (q, k, v)), scale=0.125, want_lse=True, kernel=kernel)
    assert got.abs().max() == 0 and torch.isinf(lse).all()
    q, k, v = _inputs(1, 1, 1, 6, 300, 64, BF16, seed=4)
    for at in (0, 150, 299):
        for e in range(8):
            broken = k.clone()
            broken[0, 0, (at + e) % 300, 3] = float("nan")
            got, _ = cross_attention_forward(*(t.to(cuda_device) for t in (q, broken, v)), scale=0.125, kernel=kernel)
            assert torch.isnan(got).all()


@pytest.mark.parametrize("kernel", ["rows", "tiles"])
def test_scores_of_any_size(cuda_device, kernel):
    """Peaked rows: the running maximum moves by hundreds from tile to tile."""
    q, k, v = _inputs(1, 2, 1, 40, 900, 64, BF16, seed=6)
    ramp = torch.linspace(0.1, 12.0, 900)[None, None, :, None]
    _check_forward(q, (k.float() * ramp).to(BF16), v, None, cuda_device, kernel, scale=0.5)
    _check_forward(q, (k.float() * ramp.flip(2)).to(BF16), v, None, cuda_device, kernel, scale=0.5)


@pytest.mark.parametrize("kernel", ["rows", "tiles"])
def test_strided_inputs(cuda_device, kernel):
    """(B, M, H, D) projections seen as (B, H, M, D), slices of a wider tensor, broadcast states, odd rows."""
    q = _normal((2, 37, 4, 64), BF16, 1).to(cuda_device).transpose(1, 2)
    kv = _normal((2, 210, 2, 2, 64), BF16, 2).to(cuda_device)
    k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    want, _ = cross_attention_forward(q.contiguous(), k.contiguous(), v.contiguous(), scale=0.125, kernel=kernel)
    got, _ = cross_attention_forward(q, k, v, scale=0.125, kernel=kernel)
    assert torch.equal(got, want)
    wide = torch.empty(2, 4, 37, 72, dtype=BF16, device=cuda_device)[..., 8:]
    got, _ = cross_attention_forward(q, k, v, scale=0.125, kernel=kernel, out=wide)
    assert got.data_ptr() == wide.data_ptr() and torch.equal(wide, want)
    odd = torch.empty(2, 4, 37, 67, dtype=BF16, device=cuda_device)[..., 1:65].copy_(q)  # not 16-byte aligned
    assert torch.equal(cross_attention_forward(odd, k, v, scale=0.125, kernel=kernel)[0], want)
    with pytest.raises(ValueError, match="16-byte"):
        cross_attention_forward(q, k, v, scale=0.125, out=odd)
    one = k[:1].expand(2, -1, -1, -1)
    got, _ = cross_attention_forward(q, one, v, scale=0.125, kernel=kernel)
    assert torch.equal(got, cross_attention_forward(q, one.contiguous(), v, scale=0.125, kernel=kernel)[0])


GRAD_SHAPES = [
    (1, 1, 1, 1, 16, 8, None),
    (2, 3, 3, 65, 64, 64, None),
    (2, 4, 2, 63, 130, 64, [129, 64]),
    (3, 4, 1, 40, 200, 80, [0, 200, 77]),
    (1, 2, 2, 129, 257, 128, [193]),
    (1, 2, 1, 300, 20, 96, None),
    (1, 1, 1, 20, 2000, 128, None),
    (1, 2, 1, 2000, 40, 64, [33]),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape", GRAD_SHAPES)
def test_gradients_match_oracle(cuda_device, shape, dtype):
    *sizes, lengths = shape
    q, k, v = _inputs(*sizes, dtype, seed=20)
    grad = _normal(q.shape, dtype, 31)
    scale = q.shape[-1] ** -0.5
    want, bounds = oracle.cross_attention_gradients(q, k, v, grad, scale=scale, lengths=lengths)
    leaves = [t.to(cuda_device).requires_grad_() for t in (q, k, v)]
    lens = None if lengths is None else torch.tensor(lengths, device=cuda_device)
    out = cross_attention(*leaves, scale=scale, lengths=lens)
    got = torch.autograd.grad(out, leaves, grad.to(cuda_device))
    for g, w, b, leaf in zip(got, want, bounds, leaves):
        assert g.shape == leaf.shape and g.dtype == dtype
        _assert_within(g, w, b)


def test_gradients_of_broadcast_and_strided_inputs(cuda_device):
    """Leaves that are expanded or transposed on their way in get their own shape's gradient."""
    q = _normal((2, 30, 4, 64), BF16, 1).to(cuda_device).requires_grad_()
    k = _normal((1, 2, 90, 64), BF16, 2).to(cuda_device).requires_grad_()
    v = _normal((2, 2, 90, 64), BF16, 3).to(cuda_device).requires_grad_()
    out = cross_attention(q.transpose(1, 2), k.expand(2, -1, -1, -1), v, scale=0.125)
    grad = torch.ones(1, dtype=BF16, device=cuda_device).expand(out.shape)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), grad)
    full = [t.detach().clone().requires_grad_() for t in (q.transpose(1, 2).contiguous(),
                                                          k.expand(2, -1, -1, -1).contiguous(), v)]
    ref = torch.autograd.grad(cross_attention(*full, scale=0.125), full, torch.ones_like(out))
    assert torch.equal(dq, ref[0].transpose(1, 2)) and torch.equal(dv, ref[2])
    assert dk.shape == k.shape and torch.equal(dk, ref[1].sum(0, keepdim=True))


def test_only_what_needs_a_gradient(cuda_device):
    q, k, v = (t.to(cuda_device) for t in _inputs(1, 2, 2, 20, 90, 64, BF16))
    out, lse = cross_attention_forward(q, k, v, scale=0.125, want_lse=True)
    grad = torch.randn_like(out)
    full = cross_attention_backward(q, k, v, out, lse, grad, scale=0.125)
    for i in range(3):
        needs = [j == i for j in range(3)]
        part = cross_attention_backward(q, k, v, out, lse, grad, scale=0.125, needs=needs)
        assert torch.equal(part[i], full[i]) and all(part[j] is None for j in range(3) if j != i)
    k.requires_grad_()
    (dk,) = torch.autograd.grad(cross_attention(q, k, v, scale=0.125), k, grad)
    assert torch.equal(dk, full[1])
    with pytest.raises(RuntimeError, match="once_differentiable"):
        twice = torch.autograd.grad(cross_attention(q, k, v, scale=0.125), k, grad.requires_grad_(), create_graph=True)
        twice[0].sum().backward()


def test_results_repeat_bit_for_bit(cuda_device):
    q, k, v = (t.to(cuda_device).requires_grad_() for t in _inputs(2, 4, 2, 300, 1000, 128, BF16))
    grad = torch.randn(q.shape, device=cuda_device).to(BF16)
    first = None
    for _ in range(5):
        out = cross_attention(q, k, v, scale=0.1)
        got = (out, *torch.autograd.grad(out, (q, k, v), grad))
        token = cross_attention_forward(q.detach()[:, :, :1], k.detach(), v.detach(), scale=0.1)[0]
        got = (*got, token)
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))


@pytest.mark.parametrize("queries", [1, 3, 40])
@pytest.mark.parametrize("prefix,states,lengths", [(1, 5, None), (196, 33, [33, 0, 17, 1]), (1500, 700, [700, 650, 3, 0]),
                                                   (300, 0, None)])
@pytest.mark.parametrize("heads,groups,dim,dtype", [(3, 3, 64, BF16), (8, 2, 128, BF16), (4, 1, 40, F16)])
def test_shared_prefix_matches_oracle(cuda_device, heads, groups, dim, dtype, prefix, states, lengths, queries):
    q, k, v = _inputs(4, heads, groups, queries, states, dim, dtype, seed=50)
    pk, pv = _normal((groups, prefix, dim), dtype, 61), _normal((groups, prefix, dim), dtype, 62)
    want, _, bound = oracle.cross_attention(q, k, v, scale=0.2, lengths=lengths, prefix=(pk, pv))
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=cuda_device)
    got = shared_prefix_attention(*(t.to(cuda_device) for t in (q, pk, pv, k, v)), scale=0.2, lengths=lens)
    _assert_within(got, want, bound)


def test_shared_prefix_equals_cross_attention_of_the_joined_states(cuda_device):
    q, k, v = (t.to(cuda_device) for t in _inputs(40, 8, 2, 1, 100, 64, BF16, seed=70))
    pk, pv = (_normal((2, 400, 64), BF16, s).to(cuda_device) for s in (71, 72))
    got = shared_prefix_attention(q, pk, pv, k, v, scale=0.125)
    joined = [torch.cat([p.expand(40, -1, -1, -1), t], 2) for p, t in ((pk, k), (pv, v))]
    want, _, bound = oracle.cross_attention(q, *joined, scale=0.125)
    _assert_within(got, want, bound)
    _assert_within(cross_attention(q, *joined, scale=0.125), want, bound)


def test_long_states_past_32_bit_offsets(cuda_device):
    """The last sequence's states start past 2^31 elements."""
    batch, states, dim = 9, 2_000_000, 128
    base = torch.zeros(batch, 1, states, dim, dtype=BF16, device=cuda_device)
    k, v = _normal((1, 1, 333, dim), BF16, 1), _normal((1, 1, 333, dim), BF16, 2)
    q = _normal((batch, 2, 1, dim), BF16, 3)
    base[-1, :, -333:] = k.to(cuda_device)[0]
    vals = torch.zeros_like(base)
    vals[-1, :, -333:] = v.to(cuda_device)[0]
    tail = [t[:, :, states - 333:] for t in (base, vals)]
    want, _, bound = oracle.cross_attention(q[-1:], k, v, scale=0.1)
    for kernel in ("rows", "tiles"):
        got, _ = cross_attention_forward(q.to(cuda_device), *tail, scale=0.1, kernel=kernel)
        _assert_within(got[-1:], want, bound)


def test_captured_and_replayed(cuda_device):
    """A training step and a token step in one graph each, replayed on new inputs."""
    q, k, v = (t.to(cuda_device) for t in _inputs(2, 4, 2, 50, 600, 64, BF16))
    grad = torch.randn_like(q)
    pk, pv = k[0, :, :100].contiguous(), v[0, :, :100].contiguous()

    def step():
        out, lse = cross_attention_forward(q, k, v, scale=0.125, want_lse=True)
        grads = cross_attention_backward(q, k, v, out, lse, grad, scale=0.125)
        return (out, *grads)

    def token():
        return (shared_prefix_attention(q[:, :, :1], pk, pv, k, v, scale=0.125),
                cross_attention(q[:, :, :1], k, v, scale=0.125))

    step(), token()
    torch.cuda.synchronize()
    graphs = []
    for fn in (step, token):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results = fn()
        graphs.append((graph, results, fn))
    for seed in (100, 200):
        for t, s in ((q, 1), (k, 2), (v, 3), (grad, 4)):
            t.copy_(_normal(t.shape, BF16, seed + s))
        for graph, results, fn in graphs:
            graph.replay()
            for a, b in zip(results, fn()):
                assert torch.equal(a, b)


def test_other_streams(cuda_device):
    """Two streams at once, each with its own inputs and workspace."""
    sets = [[t.to(cuda_device) for t in _inputs(1, 4, 4, 8, 5000, 64, BF16, seed=s)] for s in (1, 2)]
    want = [cross_attention(*s, scale=0.125) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(20):
        for i, (s, st) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(st):
                got[i].append(cross_attention(*s, scale=0.125))
    torch.cuda.synchronize()
    for outs, w in zip(got, want):
        assert all(torch.equal(o, w) for o in outs)


def test_refusals(cuda_device):
    q, k, v = (t.to(cuda_device) for t in _inputs(2, 4, 2, 3, 50, 64, BF16))
    ok = dict(scale=0.125)
    for args, kw, text in [
        ((q.float(), k.float(), v.float()), ok, "bfloat16 or float16"),
        ((q, k.half(), v), ok, "share a dtype"),
        ((q, k, v[:, :, :49]), ok, "share shape"),
        ((q[0], k, v), ok, "shape"),
        ((q[..., :60], k[..., :60], v[..., :60]), ok, "multiple of 8"),
        ((q, k[..., :32], v[..., :32]), ok, "head_dim"),
        ((q[:, :3], k, v), ok, "multiple of the key heads"),
        ((q[:1], k, v), ok, "batch"),
        ((q, k[:, :, :0], v[:, :, :0]), ok, "at least one state"),
        ((q, k, v), dict(scale=0.0), "scale"),
        ((q, k, v), dict(scale=float("nan")), "scale"),
        ((q, k, v.cpu()), ok, "CUDA"),
        ((q, k, v), dict(scale=0.125, lengths=torch.ones(3, dtype=torch.int32, device=cuda_device)), "lengths"),
        ((q, k, v), dict(scale=0.125, lengths=torch.ones(2, device=cuda_device)), "lengths"),
        ((q, k, v), dict(scale=0.125, lengths=torch.ones(2, dtype=torch.int32)), "lengths"),
    ]:
        with pytest.raises(ValueError, match=text):
            cross_attention(*args, **kw)
    with pytest.raises(ValueError, match="kernel"):
        cross_attention_forward(q, k, v, scale=0.125, kernel="simt")
    with pytest.raises(ValueError, match="out must match"):
        cross_attention_forward(q, k, v, scale=0.125, out=q[:, :, :2])
    with pytest.raises(ValueError, match="row sums"):
        cross_attention_backward(q, k, v, q, q[..., 0], q, scale=0.125)
    for args, text in [((q, k[0], v[0][:, :9], k, v), "share shape"), ((q, k[0][:, :0], v[0][:, :0], k, v), "prefix"),
                       ((q, k[0], v[0], k[:, :1], v[:, :1]), "own states"), ((q, k[0], v[0], k[:1], v[:1]), "own states")]:
        with pytest.raises(ValueError, match=text):
            shared_prefix_attention(*args, scale=0.125)
    with pytest.raises(ValueError, match="no backward"):
        shared_prefix_attention(q.requires_grad_(), k[0], v[0], k, v, scale=0.125)


def test_empty_batches_and_queries(cuda_device):
    k, v = (_normal((2, 2, 50, 64), BF16, s).to(cuda_device).requires_grad_() for s in (1, 2))
    q = torch.empty(2, 4, 0, 64, dtype=BF16, device=cuda_device, requires_grad=True)
    out = cross_attention(q, k, v, scale=0.125)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), torch.empty_like(out))
    assert out.shape == q.shape == dq.shape and dk.abs().sum() == 0 and dv.abs().sum() == 0
    none = cross_attention(q.detach()[:0].new_empty(0, 4, 3, 64), k.detach()[:0], v.detach()[:0], scale=0.125)
    assert none.shape == (0, 4, 3, 64)


def test_wait_budget_reports_and_the_next_call_is_clean(cuda_device):
    """Every wait of the tensor-core kernels is bounded: a 1 ns budget runs out at the first wait, the
    status word says so, and the next call with the usual budget is right."""
    lib = _lib.load()
    q, k, v = _inputs(4, 4, 4, 200, 700, 64, BF16, seed=80)
    dev = [t.to(cuda_device) for t in (q, k, v)]
    out, lse = cross_attention_forward(*dev, scale=0.125, want_lse=True, kernel="tiles")
    calls = [lambda: cross_attention_forward(*dev, scale=0.125, kernel="tiles"),
             lambda: cross_attention_backward(*dev, out, lse, dev[0], scale=0.125)]
    check_device_status(cuda_device)
    for call in calls:
        assert lib.intp_set_wait_budget_ns(ctypes.c_uint64(1)) == _lib.INTP_OK
        try:
            call()
            with pytest.raises(RuntimeError, match="device wait failed: code 0x10"):
                check_device_status(cuda_device)
        finally:
            assert lib.intp_set_wait_budget_ns(ctypes.c_uint64(1_000_000_000)) == _lib.INTP_OK
    _check_forward(q, k, v, None, cuda_device, "tiles", scale=0.125)


@pytest.mark.parametrize("dim,dtype", [(128, BF16), (64, F16), (40, BF16)])
@pytest.mark.parametrize("queries", [1, 3, 8])
@pytest.mark.parametrize("prefix,states,lengths", [(15, 1, None), (16, 16, [16, 0, 7]), (63, 65, [65, 64, 1]),
                                                   (257, 300, [0, 299, 128]), (900, 100, [100, 3, 99]), (1000, 40, None)])
def test_short_prefix_in_one_pass_and_in_three(cuda_device, prefix, states, lengths, queries, dim, dtype):
    """Around the border where a prefix is read by each sequence in one pass: slices of both
    segments end anywhere, and padded own states may hold NaN."""
    q, k, v = _inputs(3, 4, 2, queries, states, dim, dtype, seed=90)
    pk, pv = _normal((2, prefix, dim), dtype, 91), _normal((2, prefix, dim), dtype, 92)
    want, _, bound = oracle.cross_attention(q, k, v, scale=0.15, lengths=lengths, prefix=(pk, pv))
    if lengths is not None:
        for b, n in enumerate(lengths):
            k[b, :, n:] = float("nan")
            v[b, :, n:] = float("nan")
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=cuda_device)
    got = shared_prefix_attention(*(t.to(cuda_device) for t in (q, pk, pv, k, v)), scale=0.15, lengths=lens)
    _assert_within(got, want, bound)
    wide = torch.empty(2, prefix, 2 * dim, dtype=dtype, device=cuda_device)
    wide[..., :dim], wide[..., dim:] = pk.to(cuda_device), pv.to(cuda_device)
    again = shared_prefix_attention(q.to(cuda_device), wide[..., :dim], wide[..., dim:], k.to(cuda_device),
                                    v.to(cuda_device), scale=0.15, lengths=lens)
    assert torch.equal(got, again)


def test_autograd_step_in_a_graph(cuda_device):
    """Forward and autograd's backward captured together (fresh leaves), replayed on new values."""
    data = [t.to(cuda_device) for t in _inputs(2, 4, 2, 40, 300, 64, BF16, seed=120)]
    grad = torch.randn_like(data[0])

    def step():
        leaves = [t.detach().requires_grad_() for t in data]
        out = cross_attention(*leaves, scale=0.125)
        return (out.detach(), *torch.autograd.grad(out, leaves, grad))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = step()
    for t in data:
        t.mul_(-0.5)
    graph.replay()
    for a, b in zip(results, step()):
        assert torch.equal(a, b)


def test_calls_from_two_threads(cuda_device):
    """Calls of different sizes at once from two host threads, each on its own stream."""
    import threading

    sets = [[t.to(cuda_device) for t in _inputs(2, 4, 4, m, n, 64, BF16, seed=m)] for m, n in ((1, 3000), (200, 500))]
    want = [cross_attention(*s, scale=0.125) for s in sets]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                out = cross_attention(*sets[i], scale=0.125)
                if not torch.equal(out, want[i]):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_largest_and_smallest_magnitudes(cuda_device):
    """f16 at the ends of its range: outputs near its largest value, subnormal values."""
    q, k, v = _inputs(1, 2, 1, 33, 200, 64, F16, seed=130)
    for factor in (2.0 ** 13, 2.0 ** -20):
        for kernel in ("rows", "tiles"):
            _check_forward(q, k, (v.float() * factor).to(F16), [150], cuda_device, kernel)


def test_kernels_agree_on_which_rows_share_a_head(cuda_device):
    """H = 6 over G = 2 and 3: each query head reads the key head of its group."""
    for groups in (1, 2, 3, 6):
        q, k, v = _inputs(2, 6, groups, 5, 70, 64, BF16, seed=140)
        v = torch.arange(groups).view(1, groups, 1, 1).expand(2, groups, 70, 64).to(BF16).contiguous()
        for kernel in ("rows", "tiles"):
            out, _ = cross_attention_forward(*(t.to(cuda_device) for t in (q, k, v)), scale=0.125, kernel=kernel)
            want = torch.arange(6) // (6 // groups)
            assert (out.cpu().float().round() == want.view(1, 6, 1, 1)).all()


@pytest.mark.parametrize("kernel", ["rows", "tiles"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("states,queries,dim", [(1, 2, 64), (16, 2, 64), (40, 2, 128), (300, 6, 64), (300, 2, 128),
                                                (3000, 2, 64)])
def test_a_score_of_plus_infinity_makes_its_row_nan(cuda_device, states, queries, dim, dtype, kernel):
    """At every position of a group of 16 keys, in the first tile and in the last; a row to which
    the same key scores -inf does not see it."""
    batch = 32  # one position of the infinite key each
    q, k, v = _inputs(batch, 1, 1, queries, states, dim, dtype, seed=states + dim)
    q[..., 3] = 1.0
    q[:, :, 1, 3] = -1.0
    at = [(b if b < 16 else states - 1 - (b - 16)) % states for b in range(batch)]
    for b, i in enumerate(at):
        k[b, 0, i, 3] = float("inf")
    got, lse = cross_attention_forward(*(t.to(cuda_device) for t in (q, k, v)), scale=dim ** -0.5, want_lse=True,
                                       kernel=kernel)
    up = [m for m in range(queries) if m != 1]
    assert torch.isnan(got[:, :, up]).all() and torch.isnan(lse[:, :, up]).all()
    for b, i in enumerate(at):
        keep = [j for j in range(states) if j != i]
        want, _, bound = oracle.cross_attention(q[b:b + 1, :, 1:2], k[b:b + 1, :, keep], v[b:b + 1, :, keep],
                                                scale=dim ** -0.5)
        _assert_within(got[b:b + 1, :, 1:2], want, bound)


@pytest.mark.parametrize("kernel", ["rows", "tiles"])
def test_a_score_past_the_largest_number_makes_its_row_nan(cuda_device, kernel):
    """Finite operands whose product is not: 2^100 * 2^100 at each of 16 keys."""
    q, k, v = _inputs(16, 1, 1, 3, 40, 64, BF16, seed=5)
    q[..., 3] = 2.0 ** 100
    k[..., 3] = 0
    for b in range(16):
        k[b, 0, b, 3] = 2.0 ** 100
    got, lse = cross_attention_forward(*(t.to(cuda_device) for t in (q, k, v)), scale=0.125, want_lse=True, kernel=kernel)
    assert torch.isnan(got).all() and torch.isnan(lse).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("needs", [(True, True, True), (True, False, False), (False, True, True), (False, False, True)])
@pytest.mark.parametrize("sizes", [(2, 4, 2, 100, 196, 64), (1, 2, 2, 700, 300, 128), (1, 1, 1, 30, 2000, 64)])
def test_backwards_in_a_row_use_their_own_statistics(cuda_device, sizes, needs, dtype):
    """Calls that follow one another at once, on the same workspace memory with other values, give
    what each gives alone."""
    sets = []
    for seed in (150, 250):
        q, k, v = (t.to(cuda_device) for t in _inputs(*sizes, dtype, seed=seed))
        grad = _normal(q.shape, dtype, seed + 9).to(cuda_device)
        out, lse = cross_attention_forward(q, k, v, scale=0.125, want_lse=True)
        sets.append((q, k, v, out, lse, grad))
    torch.cuda.synchronize()
    want = []
    for s in sets:
        want.append(cross_attention_backward(*s, scale=0.125, needs=needs))
        torch.cuda.synchronize()
    got = [cross_attention_backward(*sets[i % 2], scale=0.125, needs=needs) for i in range(40)]
    for i, grads in enumerate(got):
        for a, b in zip(grads, want[i % 2]):
            assert a is b is None or torch.equal(a, b)


SCALED_GRADS = [
    # sizes, lengths, sizes of q, k, v and grad as powers of two
    ((1, 2, 1, 70, 4096, 64), None, (-8, 8, 0, -16)),        # dS far below f16's last step, dq is not
    ((1, 2, 1, 70, 4096, 64), None, (8, -8, 0, -16)),        # the same for dk
    ((2, 2, 2, 150, 1000, 128), [900, 77], (-8, 8, 0, -14)),
    ((2, 2, 2, 150, 1000, 128), [900, 77], (8, -8, 0, -14)),
    ((1, 4, 2, 33, 3000, 40), [2500], (-8, 8, -10, -4)),     # small values and small gradients
    ((1, 1, 1, 700, 20, 64), None, (-6, -10, 8, 8)),         # dS past f16's largest number
    ((1, 1, 1, 40, 20, 128), None, (-6, -10, 8, 8)),
    ((1, 1, 1, 2, 131072, 16), None, (0, 0, 0, 6)),          # P near 2^-17
    ((2, 3, 3, 65, 64, 64), None, (0, 0, 0, 0)),
]


def _powers(shape, dtype, seed, power):
    return (_normal(shape, torch.float32, seed) * 2.0 ** power).to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", SCALED_GRADS)
def test_gradients_keep_their_bits_at_any_size(cuda_device, case, dtype):
    """Bounds that know no absolute size but the result's own; values past the lengths are the
    type's largest, infinite and NaN, and play no part in a scale either."""
    (batch, heads, groups, queries, states, dim), lengths, powers = case
    q = _powers((batch, heads, queries, dim), dtype, 161, powers[0])
    k = _powers((batch, groups, states, dim), dtype, 162, powers[1])
    v = _powers((batch, groups, states, dim), dtype, 163, powers[2])
    grad = _powers((batch, heads, queries, dim), dtype, 164, powers[3])
    scale = dim ** -0.5
    want, bounds = oracle.cross_attention_gradients(q, k, v, grad, scale=scale, lengths=lengths, scaled=True)
    for b, n in enumerate(lengths or []):
        v[b, :, n:] = torch.finfo(dtype).max
        v[b, :, n + 1:] = float("inf")
        v[b, :, n + 2:] = float("nan")
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=cuda_device)
    dev = [t.to(cuda_device) for t in (q, k, v)]
    out, lse = cross_attention_forward(*dev, scale=scale, lengths=lens, want_lse=True)
    got = cross_attention_backward(*dev, out, lse, grad.to(cuda_device), scale=scale, lengths=lens)
    for g, w, b in zip(got, want, bounds):
        _assert_within(g, w, b)


@pytest.mark.parametrize("dim", [64, 128])
def test_query_rows_with_gradients_of_any_size_together(cuda_device, dim):
    """A row's dq keeps its bits beside rows whose gradients are 2^20 times as large, and zero."""
    q, k = _powers((1, 2, 90, dim), F16, 171, -8), _powers((1, 1, 2000, dim), F16, 172, 8)
    v = _powers((1, 1, 2000, dim), F16, 173, 0)
    power = torch.tensor([-16.0, 4.0, -8.0])[torch.arange(90) % 3][None, None, :, None]
    grad = _normal((1, 2, 90, dim), torch.float32, 174) * torch.exp2(power)
    grad[:, :, 7] = 0
    grad = grad.to(F16)
    want, bounds = oracle.cross_attention_gradients(q, k, v, grad, scale=0.125, scaled=True)
    dev = [t.to(cuda_device) for t in (q, k, v)]
    out, lse = cross_attention_forward(*dev, scale=0.125, want_lse=True)
    got = cross_attention_backward(*dev, out, lse, grad.to(cuda_device), scale=0.125)
    for g, w, b in zip(got, want, bounds):
        _assert_within(g, w, b)
    assert got[0][:, :, 7].abs().max() == 0


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_gradients_that_are_not_finite_stay_in_their_rows(cuda_device, bad, dtype):
    """A query row whose upstream gradient is not finite has no finite dq; the others keep theirs."""
    q, k, v = (t.to(cuda_device) for t in _inputs(1, 2, 2, 100, 300, 64, dtype, seed=181))
    grad = _normal(q.shape, dtype, 182).to(cuda_device)
    out, lse = cross_attention_forward(q, k, v, scale=0.125, want_lse=True)
    want = cross_attention_backward(q, k, v, out, lse, grad, scale=0.125)
    grad[0, 0, 41, 5] = bad
    got = cross_attention_backward(q, k, v, out, lse, grad, scale=0.125)
    rest = [m for m in range(100) if m != 41]
    assert not torch.isfinite(got[0][0, 0, 41]).any()
    assert torch.equal(got[0][0, 0, rest], want[0][0, 0, rest])
    for g, w in zip(got, want):
        assert torch.equal(g[0, 1], w[0, 1])
    assert not torch.isfinite(got[1][0, 0]).any() and not torch.isfinite(got[2][0, 0, :, 5]).any()
    others = [c for c in range(64) if c != 5]
    torch.testing.assert_close(got[2][0, 0][:, others], want[2][0, 0][:, others], rtol=0, atol=0)


@pytest.mark.parametrize("queries,batch", [(0, 2), (0, 0), (3, 2)])
def test_the_library_writes_every_gradient(cuda_device, queries, batch):
    """Through the C entry: without queries the states' gradients are zeros, not what the buffers held."""
    q, k, v = (t.to(cuda_device) for t in _inputs(batch, 4, 2, queries, 70, 64, BF16, seed=190))
    grads = [torch.full_like(t, float("nan")) for t in (q, k, v)]
    args = _lib.XattnBackwardArgs()
    f = args.fwd
    f.batch, f.heads, f.groups, f.queries, f.states, f.head_dim = batch, 4, 2, queries, 70, 64
    f.scale, f.dtype = 0.125, _lib.INTP_BF16
    if queries:
        out, lse = cross_attention_forward(q, k, v, scale=0.125, want_lse=True)
        status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
        f.q, f.k, f.v, f.out, f.lse, f.status = (t.data_ptr() for t in (q, k, v, out, lse, status))
        args.grad_out = q.data_ptr()
        f.q_stride = f.out_stride = args.grad_out_stride = _lib._Stride(*q.stride())
        f.k_stride = f.v_stride = _lib._Stride(*k.stride())
    args.grad_q, args.grad_k, args.grad_v = (t.data_ptr() or None for t in grads)
    size = ctypes.c_int64()
    lib = _lib.load()
    assert lib.xattn_backward_workspace(ctypes.addressof(args), ctypes.byref(size)) == _lib.INTP_OK
    space = torch.empty(size.value, dtype=torch.uint8, device=cuda_device)
    f.workspace, f.workspace_bytes = space.data_ptr() or None, size.value
    stream = torch.cuda.current_stream(cuda_device).cuda_stream
    assert lib.xattn_backward(ctypes.addressof(args), stream) == _lib.INTP_OK
    assert not any(torch.isnan(g).any() for g in grads)
    if queries == 0:
        assert all(g.abs().sum() == 0 for g in grads)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape", [
    (4, 4, 4, 4, 5, 16, None), (4, 4, 4, 4, 17, 16, None), (4, 8, 2, 1, 60, 16, [60, 17, 0, 33]), (4, 4, 4, 4, 17, 64, None),
    (2, 6, 2, 3, 129, 40, [129, 70]), (2, 8, 2, 4, 300, 128, [299, 128]), (1, 16, 4, 1, 3001, 64, None),
    (3, 4, 2, 8, 196, 64, None)])
def test_few_rows_carry_only_the_rounding_of_the_result(cuda_device, shape, dtype):
    """The few-rows kernel multiplies two parts of each probability: held to the bound of that."""
    *sizes, lengths = shape
    q, k, v = _inputs(*sizes, dtype, seed=200)
    scale = q.shape[-1] ** -0.5
    want, _, bound = oracle.cross_attention(q, k, v, scale=scale, lengths=lengths, two_part=True)
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=cuda_device)
    got, _ = cross_attention_forward(*(t.to(cuda_device) for t in (q, k, v)), scale=scale, lengths=lens, kernel="rows")
    _assert_within(got, want, bound)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("prefix,states,lengths,dim", [(3, 4, None, 16), (16, 17, [17, 0, 9], 16), (100, 33, [33, 1, 0], 64),
                                                       (600, 300, None, 64)])
def test_a_prefix_read_in_one_pass_carries_only_the_rounding_of_the_result(cuda_device, prefix, states, lengths, dim, dtype):
    q, k, v = _inputs(3, 8, 4, 2, states, dim, dtype, seed=210)
    pk, pv = _normal((4, prefix, dim), dtype, 211), _normal((4, prefix, dim), dtype, 212)
    scale = dim ** -0.5
    want, _, bound = oracle.cross_attention(q, k, v, scale=scale, lengths=lengths, prefix=(pk, pv), two_part=True)
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=cuda_device)
    got = shared_prefix_attention(*(t.to(cuda_device) for t in (q, pk, pv, k, v)), scale=scale, lengths=lens)
    _assert_within(got, want, bound)


def test_transforms_that_the_kernels_do_not_see_are_refused(cuda_device):
    """Forward-mode tangents, traces and functional transforms: an error each, not a lost derivative."""
    forward_ad = torch.autograd.forward_ad
    q, k, v = (t.to(cuda_device) for t in _inputs(2, 2, 2, 3, 20, 64, BF16, seed=220))

    def call(t):
        return cross_attention(t, k, v, scale=0.125)

    want = call(q)
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="forward-mode"):
            call(forward_ad.make_dual(q, torch.ones_like(q)))
        with pytest.raises(ValueError, match="forward-mode"):
            shared_prefix_attention(q, k[0], v[0], k, forward_ad.make_dual(v, torch.ones_like(v)), scale=0.125)
        assert torch.equal(call(q), want)
    with pytest.raises(ValueError, match="traced"):
        torch.jit.trace(call, q)
    for transform in (lambda: torch.func.jvp(call, (q,), (q,)), lambda: torch.func.vmap(call)(q[:, None]),
                      lambda: torch.func.grad(lambda t: call(t).float().sum())(q)):
        with pytest.raises((ValueError, RuntimeError)):
            transform()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("sizes,lengths", [((4, 12, 4, 1100, 77, 64), [77, 40, 0, 65]),      # 432 dq items
                                           ((3, 8, 8, 800, 150, 128), [150, 129, 3]),       # 168 dq, 48 dk / dv
                                           ((2, 64, 64, 60, 260, 64), [260, 200]),          # 384 dk / dv items
                                           ((2, 40, 40, 60, 300, 128), None)])
def test_gradients_of_more_items_than_ctas(cuda_device, sizes, lengths, dtype):
    """A CTA runs several items, whose gradients differ in size by up to 2^16 from row to row and head
    to head, and whose values do by 2^8: each item keeps its own scale."""
    batch, heads, groups, queries, states, dim = sizes
    q, k, v = _inputs(*sizes, dtype, seed=230)
    g = torch.Generator().manual_seed(231)
    rows = torch.randint(-8, 1, (batch, heads, queries, 1), generator=g) + torch.randint(-8, 1, (batch, heads, 1, 1), generator=g)
    grad = (torch.randn(q.shape, generator=g) * torch.exp2(rows.float())).to(dtype)
    v = (v.float() * torch.exp2(torch.randint(-8, 1, (batch, groups, 1, 1), generator=g).float())).to(dtype)
    scale = dim ** -0.5
    want, bounds = oracle.cross_attention_gradients(q, k, v, grad, scale=scale, lengths=lengths, scaled=True)
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=cuda_device)
    dev = [t.to(cuda_device) for t in (q, k, v)]
    out, lse = cross_attention_forward(*dev, scale=scale, lengths=lens, want_lse=True)
    for needs in ((True, True, True), (False, True, True)):
        got = cross_attention_backward(*dev, out, lse, grad.to(cuda_device), scale=scale, lengths=lens, needs=needs)
        for g, w, b in zip(got, want, bounds):
            if g is not None:
                _assert_within(g, w, b)


@pytest.mark.parametrize("form", ["contiguous", "padded", "unaligned", "cpu", "checkpoint"])
def test_gradients_through_hooks_on_saved_tensors(cuda_device, form):
    """Offloaded, copied and recomputed tensors come back in other layouts: the same gradients."""
    base = _normal((2, 37, 4, 64), BF16, 240).to(cuda_device)
    both = _normal((2, 210, 2, 2, 64), BF16, 241).to(cuda_device)
    grad = _normal((2, 4, 37, 64), BF16, 242).to(cuda_device)
    lengths = torch.tensor([210, 77], dtype=torch.int32, device=cuda_device)

    def pack(t):
        if form == "cpu":
            return t.cpu()
        if t.dtype != BF16:
            return t
        if form == "contiguous":
            return t.clone(memory_format=torch.contiguous_format)
        wide = torch.empty(*t.shape[:-1], t.shape[-1] + 8, dtype=t.dtype, device=t.device)
        return (wide[..., 8:] if form == "padded" else wide[..., 1:t.shape[-1] + 1]).copy_(t)

    def attend(x, kv):
        return cross_attention(x.transpose(1, 2), kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2), scale=0.125,
                               lengths=lengths)

    leaves = [base.clone().requires_grad_(), both.clone().requires_grad_()]
    want = torch.autograd.grad(attend(*leaves), leaves, grad)
    if form == "checkpoint":
        out = torch.utils.checkpoint.checkpoint(attend, *leaves, use_reentrant=False)
    else:
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.to(cuda_device)):
            out = attend(*leaves)
    for g, w in zip(torch.autograd.grad(out, leaves, grad), want):
        assert torch.equal(g, w)


@pytest.mark.parametrize("kernel", ["rows", "tiles"])
@pytest.mark.parametrize("value", [float("inf"), float("nan"), "largest"])
@pytest.mark.parametrize("states", [1, 40, 300, 3000])
def test_a_row_of_minus_infinite_scores_gives_zeros_whatever_the_values(cuda_device, states, value, kernel):
    """Its output is zero, not a sum of values times zero; the row beside it sees them."""
    q, k, v = _inputs(2, 2, 2, 2, states, 64, BF16, seed=250)
    q[..., 3], k[..., 3] = 1.0, -float("inf")
    q[:, :, 1, 3] = 0.0                    # 0 * -inf: a NaN row
    v[:, :, ::3] = torch.finfo(BF16).max if value == "largest" else value
    got, lse = cross_attention_forward(*(t.to(cuda_device) for t in (q, k, v)), scale=0.125, want_lse=True, kernel=kernel)
    assert (got[:, :, 0] == 0).all() and (lse[:, :, 0] == -float("inf")).all()
    assert torch.isnan(got[:, :, 1]).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("far", [1e3, 6e4])
@pytest.mark.parametrize("dim,states", [(64, 4096), (128, 1000)])
def test_a_large_value_that_is_hardly_read_costs_the_others_nothing(cuda_device, dim, states, far, dtype):
    """States with values far above the others' and probabilities near zero: dk of every other key
    keeps its bits, and dq loses 2^-39 of |dO| |v| per state."""
    q, k, v = _inputs(1, 2, 1, 100, states, dim, dtype, seed=260)
    q[..., 3] = 4.0
    hidden = list(range(5, states, 97))
    k[:, :, hidden, 3] = -60.0             # scores of -30 and below: probabilities near 2^-55
    v[:, :, hidden] = far
    grad = _normal(q.shape, dtype, 261)
    scale = dim ** -0.5
    want, bounds = oracle.cross_attention_gradients(q, k, v, grad, scale=scale, scaled=True)
    dev = [t.to(cuda_device) for t in (q, k, v)]
    out, lse = cross_attention_forward(*dev, scale=scale, want_lse=True)
    got = cross_attention_backward(*dev, out, lse, grad.to(cuda_device), scale=scale)
    for g, w, b in zip(got, want, bounds):
        _assert_within(g, w, b)
    # As a whole, too: dS and the result are rounded (u each), P is within 6.5e-4 (1.4 u in f16).  dq adds
    # 2^-39 |dO| |v| to each dS of about 2^-12 |dO|: 2^-27 |v|, 2^-14 for |v| = 8e3, ten times u for 5e5.
    for g, w in list(zip(got, want))[1 if far > 1e4 else 0:2]:
        off = (g.cpu().double() - w).norm() / w.norm()
        assert off <= 4 * torch.finfo(dtype).eps / 2, float(off)
