"""Queries and keys turned by positions of several axes on the GPU, against the float64 oracle."""

import pytest
import torch

from intp_preliminary_b200 import RotaryAxes, check_device_status, rotate_positions
from intp_preliminary_b200.share_vit import HexSupport
from oracle import paged as oracle

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _rand(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _axes(pairs, count):
    return sorted(i % count for i in range(pairs))


def _rotary(pairs, count, device, interleaved=False):
    return RotaryAxes([10000.0 ** (-i / pairs) for i in range(pairs)], _axes(pairs, count), interleaved=interleaved,
                      device=device)


def _positions(batch, rows, count, kind, seed, far=5000):
    g = torch.Generator().manual_seed(seed)
    if kind == torch.float32:
        return torch.randn(batch, rows, count, generator=g) * 100
    return torch.randint(-far, far, (batch, rows, count), generator=g).to(kind)


def _close(got, x, positions, rotary, inverse=False):
    want, bound = oracle.turn(x, positions, rotary.frequencies, rotary.axes, interleaved=rotary.interleaved,
                              inverse=inverse)
    worst = ((got.detach().cpu().double() - want).abs() - bound).max()
    assert got.dtype == x.dtype and worst <= 0, f"past the bound by {worst}"


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,pairs", [(8, 4), (16, 8), (24, 12), (40, 4), (64, 32), (72, 36), (72, 16), (80, 40), (96, 24),
                                       (120, 4), (128, 64), (128, 20)])
def test_matches_oracle(cuda_device, dtype, interleaved, dim, pairs):
    rotary = _rotary(pairs, 2, cuda_device, interleaved)
    q, k = _rand((2, 5, 7, dim), dtype, 1), _rand((2, 2, 7, dim), dtype, 2)
    at = _positions(2, 7, 2, torch.int32, 3)
    got = rotate_positions(q.to(cuda_device), k.to(cuda_device), rotary=rotary, positions=at.to(cuda_device))
    _close(got[0], q, at, rotary)
    _close(got[1], k, at, rotary)
    back = rotate_positions(q.to(cuda_device), rotary=rotary, positions=at.to(cuda_device), inverse=True)
    assert back[1] is None
    _close(back[0], q, at, rotary, inverse=True)


@pytest.mark.parametrize("batch,heads,rows", [(1, 1, 1), (1, 3, 196), (3, 1, 33), (1, 40, 1), (2, 9, 1000), (65, 12, 129)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_sizes(cuda_device, batch, heads, rows, dtype):
    rotary = _rotary(32, 3, cuda_device)
    q, k = _rand((batch, heads, rows, 64), dtype, 4), _rand((batch, heads + 1, rows, 64), dtype, 5)
    at = _positions(batch, rows, 3, torch.int64, 6)
    got = rotate_positions(q.to(cuda_device), k.to(cuda_device), rotary=rotary, positions=at.to(cuda_device))
    _close(got[0], q, at, rotary)
    _close(got[1], k, at, rotary)


@pytest.mark.parametrize("kind,values", [
    (torch.int32, [-2**31, 2**31 - 1, 10**9 + 7, 0]), (torch.int64, [2**40 + 1, -2**33, 10**12 + 39, -1]),
    (torch.float32, [1e6 + 0.25, -12345.678, 1e-30, 0.0])])
def test_far_positions_keep_their_angle(cuda_device, kind, values):
    rotary = _rotary(32, 1, cuda_device)
    x = _rand((1, 2, 4, 64), F32, 7)
    at = torch.tensor(values, dtype=kind)[None, :, None]
    got, _ = rotate_positions(x.to(cuda_device), rotary=rotary, positions=at.to(cuda_device))
    _close(got, x, at, rotary)


def test_quarter_turns(cuda_device):
    """Angles at and about the multiples of an eighth of a turn, where the reduction changes its case."""
    import math

    rotary = RotaryAxes([math.pi / 4, math.pi / 4 * (1 + 1e-9), math.pi / 4 * (1 - 1e-9), math.pi / 2], [0] * 4,
                        device=cuda_device)
    x = _rand((1, 1, 41, 8), F32, 8)
    at = torch.arange(-20, 21)[:, None]
    got, _ = rotate_positions(x.to(cuda_device), rotary=rotary, positions=at.to(cuda_device))
    _close(got, x, at, rotary)


def test_strided_and_broadcast_inputs(cuda_device):
    rotary = _rotary(32, 2, cuda_device)
    at = _positions(2, 9, 2, torch.int32, 9)
    moved = at.permute(2, 0, 1).contiguous().to(cuda_device).permute(1, 2, 0)  # (axes, B, n) in memory
    rows = _rand((2, 9, 3, 4, 64), BF16, 10).to(cuda_device)
    forms = {"a projection's slice": rows[:, :, 1].transpose(1, 2), "one sequence for all": rows[:1, :, 0].transpose(1, 2).expand(2, -1, -1, -1),
             "one head for all": rows[:, :, 2, :1].transpose(1, 2).expand(-1, 4, -1, -1),
             "every second column": _rand((2, 4, 9, 128), BF16, 11).to(cuda_device)[..., ::2],
             "unaligned": _rand((2, 4, 9, 65), BF16, 12).to(cuda_device)[..., 1:],
             "backwards": rows[:, :, 1].transpose(1, 2).flip(1)}
    for name, q in forms.items():
        got, other = rotate_positions(q, q[:, :1], rotary=rotary, positions=moved)
        _close(got, q.cpu(), at, rotary)
        _close(other, q[:, :1].cpu(), at, rotary)
    same = at[0]
    got, _ = rotate_positions(forms["unaligned"], rotary=rotary, positions=same.to(cuda_device))
    _close(got, forms["unaligned"].cpu(), same, rotary)


def test_gradients(cuda_device):
    rotary = _rotary(20, 3, cuda_device, interleaved=True)
    at = _positions(2, 11, 3, torch.float32, 13)
    on = at.to(cuda_device)
    q, k, gq, gk = (_rand((2, h, 11, 48), F32, 14 + i).to(cuda_device) for i, h in enumerate((4, 2, 4, 2)))
    leaves = [t.clone().requires_grad_() for t in (q, k)]
    out = rotate_positions(*leaves, rotary=rotary, positions=on)
    dq, dk = torch.autograd.grad(out, leaves, (gq, gk), retain_graph=True)
    _close(dq, gq.cpu(), at, rotary, inverse=True)
    _close(dk, gk.cpu(), at, rotary, inverse=True)
    # against differences: linear, so a step of one; 11 * 48 terms of two fp32 results with errors of 1e-6 each
    for i in range(0, 48, 7):
        step = torch.zeros_like(q)
        step[1, 2, 3, i] = 1.0
        change = (rotate_positions(q + step, rotary=rotary, positions=on)[0].double()
                  - rotate_positions(q - step, rotary=rotary, positions=on)[0].double())
        assert abs(float((change * gq.double()).sum()) / 2 - float(dq[1, 2, 3, i])) < 1e-5
    # only one of the two results, only one of the two inputs
    only, = torch.autograd.grad(out[1], [leaves[1]], gk, retain_graph=True)
    assert torch.equal(only, dk)
    mixed = rotate_positions(leaves[0], k, rotary=rotary, positions=on)
    assert torch.equal(torch.autograd.grad(mixed[0], leaves[0], gq)[0], dq)
    # a gradient of the gradient: the same turn again
    seed = gq.clone().requires_grad_()
    first, = torch.autograd.grad(rotate_positions(leaves[0], rotary=rotary, positions=on)[0], leaves[0], seed,
                                 create_graph=True)
    again, = torch.autograd.grad(first, seed, q)
    _close(again, q.cpu(), at, rotary)


def test_gradient_of_a_broadcast_input_is_summed(cuda_device):
    rotary = _rotary(8, 1, cuda_device)
    at = torch.arange(5)[:, None]
    q, grad = _rand((1, 1, 5, 16), F32, 20), _rand((3, 4, 5, 16), F32, 21)
    leaf = q.to(cuda_device).requires_grad_()
    out, _ = rotate_positions(leaf.expand(3, 4, 5, 16), rotary=rotary, positions=at.to(cuda_device))
    got, = torch.autograd.grad(out, leaf, grad.to(cuda_device))
    want, bound = oracle.turn(grad, at, rotary.frequencies, rotary.axes, inverse=True)
    # twelve fp32 numbers summed: their bounds and 11 roundings of partial sums
    limit = bound.sum((0, 1), keepdim=True) + 12 * 2.0 ** -24 * want.abs().sum((0, 1), keepdim=True)
    assert ((got.cpu().double() - want.sum((0, 1), keepdim=True)).abs() <= limit).all()


def test_patches_of_the_hex_lattice(cuda_device):
    """The encoder's own places: 195 lattice points and the CLS token at the origin."""
    places = torch.cat((torch.zeros(1, 2), HexSupport(24).unit_xy.float()))
    rotary = RotaryAxes.sections([16, 16], apart=True, base=100.0, device=cuda_device)
    assert rotary.axes == (0,) * 16 + (1,) * 16 and rotary.frequencies[16] == 1.0
    q = _rand((4, 3, 196, 64), BF16, 22)
    got, _ = rotate_positions(q.to(cuda_device), rotary=rotary, positions=places.to(cuda_device))
    _close(got, q, places, rotary)
    assert torch.equal(got[:, :, 0].cpu(), q[:, :, 0])


def test_values_that_are_not_finite_stay_in_their_pairs(cuda_device):
    rotary = _rotary(8, 1, cuda_device)
    x = _rand((1, 1, 3, 24), BF16, 23)
    clean, _ = rotate_positions(x.to(cuda_device), rotary=rotary, positions=torch.arange(3, device=cuda_device)[:, None])
    x[0, 0, 1, 2], x[0, 0, 2, 20] = float("inf"), float("nan")
    got, _ = rotate_positions(x.to(cuda_device), rotary=rotary, positions=torch.arange(3, device=cuda_device)[:, None])
    bad = torch.zeros(x.shape, dtype=torch.bool)
    bad[0, 0, 1, [2, 10]] = bad[0, 0, 2, 20] = True
    assert torch.equal(~torch.isfinite(got.cpu()), bad)
    assert torch.equal(got.cpu()[~bad], clean.cpu()[~bad])


def test_captured_replayed_other_streams_and_repeats(cuda_device):
    rotary = _rotary(32, 2, cuda_device)
    at = _positions(2, 300, 2, torch.int32, 24)
    on = at.to(cuda_device)
    q, k = _rand((2, 4, 300, 64), BF16, 25).to(cuda_device), _rand((2, 2, 300, 64), BF16, 26).to(cuda_device)
    first = rotate_positions(q, k, rotary=rotary, positions=on)
    stream = torch.cuda.Stream(cuda_device)
    stream.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(stream):
        other = rotate_positions(q, k, rotary=rotary, positions=on)
    torch.cuda.current_stream(cuda_device).wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        leaves = [t.detach().requires_grad_() for t in (q, k)]
        out = rotate_positions(*leaves, rotary=rotary, positions=on)
        grads = torch.autograd.grad(out, leaves, [t.detach() for t in out])
    q.copy_(_rand((2, 4, 300, 64), BF16, 27))
    on.copy_(_positions(2, 300, 2, torch.int32, 28))
    graph.replay()
    again = rotate_positions(q, k, rotary=rotary, positions=on)
    assert all(torch.equal(a, b) for a, b in zip(out, again))
    back = rotate_positions(*again, rotary=rotary, positions=on, inverse=True)
    assert all(torch.equal(a, b) for a, b in zip(grads, back))
    check_device_status(cuda_device)


def test_refusals(cuda_device):
    rotary = _rotary(32, 2, cuda_device)
    q = torch.zeros(2, 4, 5, 64, dtype=BF16, device=cuda_device)
    at = torch.zeros(2, 5, 2, dtype=torch.int32, device=cuda_device)
    good = dict(rotary=rotary, positions=at)
    for args, over, message in (
            ((q.double(),), {}, "must be bfloat16"), ((q[0],), {}, "shape"), ((q[..., :60],), {}, "multiple of 8"),
            ((torch.zeros(1, 1, 5, 136, dtype=BF16, device=cuda_device),), {}, "up to 128"),
            ((q[..., :32],), {}, "more columns"), ((q, q[:1]), {}, "share"), ((q, q.float()), {}, "share"),
            ((q, q[:, :, :4]), {}, "share"), ((q,), {"positions": at[:, :4]}, "positions"),
            ((q,), {"positions": at[..., :1]}, "positions"), ((q,), {"positions": at[:1]}, "positions"),
            ((q,), {"positions": at.double()}, "int32, int64 or float32"), ((q,), {"positions": at.cpu()}, "same CUDA device"),
            ((q, q.cpu()), {}, "CUDA")):
        with pytest.raises(ValueError, match=message):
            rotate_positions(*args, **{**good, **over})
    assert rotate_positions(q[:0], **{**good, "positions": at[:0]})[0].shape == (0, 4, 5, 64)
    assert rotate_positions(q[:, :, :0], q[:, :, :0], **{**good, "positions": at[:, :0]})[1].shape == (2, 4, 0, 64)


def test_rows_past_32_bit_offsets(cuda_device):
    """A tensor of more than 2^31 elements, its far rows checked against their own call."""
    rotary = _rotary(64, 1, cuda_device)
    rows = (1 << 24) + 5
    q = torch.empty(1, 1, rows, 128, dtype=BF16, device=cuda_device)
    for part in q[0, 0].split(1 << 20):
        part.normal_()
    at = torch.arange(rows, device=cuda_device)[:, None]
    got, _ = rotate_positions(q, rotary=rotary, positions=at)
    for where in (slice(0, 3), slice(rows - 7, rows)):
        want, _ = rotate_positions(q[:, :, where].clone(), rotary=rotary, positions=at[where].clone())
        assert torch.equal(got[:, :, where], want)


def test_copies_turn_alike_without_the_original(cuda_device):
    """A deep copy, a pickled object, copies inside a module: the same bits once the original is gone."""
    import copy
    import pickle

    q = _rand((1, 2, 9, 32), F32, 30).to(cuda_device)
    at = _positions(1, 9, 2, torch.int32, 31).to(cuda_device)
    rotary = _rotary(16, 2, cuda_device)
    layer = torch.nn.Linear(2, 2)
    layer.rotary = rotary
    want, _ = rotate_positions(q, rotary=rotary, positions=at)
    copies = [copy.copy(rotary), copy.deepcopy(rotary), pickle.loads(pickle.dumps(rotary)), copy.deepcopy(layer).rotary,
              pickle.loads(pickle.dumps(layer)).rotary]
    assert all(c.device == rotary.device for c in copies)
    del rotary, layer
    others = [RotaryAxes([0.0] * 16, [1, 0] * 8, device=cuda_device) for _ in range(8)]  # where the original's tables were
    for c in copies:
        assert torch.equal(rotate_positions(q, rotary=c, positions=at)[0], want)
    assert len(others) == 8


def test_a_rotary_dropped_while_another_stream_has_yet_to_read_it(cuda_device):
    """Its memory is not given to new work before that stream's launches are done."""
    from intp_preliminary_b200 import PagedCache

    q = _rand((1, 2, 9, 32), F32, 32).to(cuda_device)
    k = q.bfloat16()
    at = _positions(1, 9, 2, torch.int32, 33).to(cuda_device)
    table = torch.arange(2, dtype=torch.int32, device=cuda_device)[None]
    start = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    kept = _rotary(16, 2, cuda_device)
    want, _ = rotate_positions(q, rotary=kept, positions=at)
    pool, other = (PagedCache.empty(2, 2, 16, 32, device=cuda_device) for _ in range(2))
    pool.append(k, k, page_table=table, start=start, rotary=kept, positions=at)
    for append in (False, True):
        rotary = _rotary(16, 2, cuda_device)
        address = rotary._tables.data_ptr()
        torch.cuda.synchronize(cuda_device)
        stream, done = torch.cuda.Stream(cuda_device), torch.cuda.Event()
        with torch.cuda.stream(stream):
            torch.cuda._sleep(400_000_000)  # a fifth of a second
            if append:
                other.append(k, k, page_table=table, start=start, rotary=rotary, positions=at)
            else:
                got, _ = rotate_positions(q, rotary=rotary, positions=at)
            done.record()
        del rotary
        new = [torch.zeros(192, dtype=torch.uint8, device=cuda_device) for _ in range(20)]
        assert not done.query()
        assert address not in [t.data_ptr() for t in new]
        done.synchronize()
    assert torch.equal(got, want) and torch.equal(other.keys, pool.keys)
