"""The paged cache and attention over it on the GPU, against the float64 oracle."""

import pytest
import torch

from intp_preliminary_b200 import (PagedCache, RotaryAxes, check_device_status, cross_attention, paged_attention,
                                   rotate_positions)
from oracle import paged as oracle

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
KERNELS = ["joined", "parts"]
NAN, INF = float("nan"), float("inf")


@pytest.fixture(autouse=True)
def _device_status(cuda_device):
    yield
    check_device_status(cuda_device)


def _rand(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def _table(batch, width, spare, seed):
    """Shuffled pages, and how many the pool has."""
    pages = batch * width + spare
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
    return order[:batch * width].reshape(batch, width).to(torch.int32), pages


def _filled(batch, groups, states, dim, page_size, dtype, seed, spare=2, hole=NAN):
    """A pool whose sequences hold `states` states each; what they do not hold is `hole`."""
    width = -(-states // page_size)
    table, pages = _table(batch, width, spare, seed)
    keys, values = (torch.full((pages, groups, page_size, dim), hole).to(dtype) for _ in range(2))
    k, v = _rand((batch, groups, states, dim), dtype, seed + 1), _rand((batch, groups, states, dim), dtype, seed + 2)
    oracle.append(keys, values, k, v, page_table=table, start=[0] * batch)
    return keys, values, table


def _attend(device, q, keys, values, table, start, **more):
    cache = PagedCache(keys.to(device), values.to(device))
    on = {n: torch.tensor(x, device=device) if isinstance(x, list) else x for n, x in more.items()}
    return paged_attention(q.to(device), cache, page_table=table.to(device), start=torch.tensor(start, device=device),
                           **on)


def _check(device, q, keys, values, table, start, kernel="auto", **more):
    got = _attend(device, q, keys, values, table, start, kernel=kernel, **more).cpu().double()
    want, bound = oracle.attend(q, keys, values, page_table=table, start=start, **more)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    wrong = ~(((got - want).abs() <= bound) | torch.isnan(want) | (got == want))
    assert not wrong.any(), f"{int(wrong.sum())} past the bound, {float(((got - want).abs() / bound)[wrong].max())} times it"
    return got


# ------------------------------------------------------------------ appending
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("page_size", [1, 3, 16, 64])
@pytest.mark.parametrize("dim,pairs,interleaved", [(64, 32, False), (72, 36, True), (80, 8, False), (128, 64, False), (8, 4, True)])
def test_append_turns_and_places(cuda_device, dtype, page_size, dim, pairs, interleaved):
    batch, groups, heads, rows = 3, 2, 6, 21
    start, counts = [0, 5, 40], [21, 13, 21]
    width = -(-64 // page_size)
    table, pages = _table(batch, width, 3, 1)
    keys, values = _rand((pages, groups, page_size, dim), dtype, 2), _rand((pages, groups, page_size, dim), dtype, 3)
    q, k, v = _rand((batch, heads, rows, dim), dtype, 4), _rand((batch, groups, rows, dim), dtype, 5), _rand((batch, groups, rows, dim), dtype, 6)
    rotary = RotaryAxes([1000.0 ** (-i / pairs) for i in range(pairs)], [i % 2 for i in range(pairs)],
                        interleaved=interleaved, device=cuda_device)
    own = torch.randint(0, 900, (batch, rows, 2), generator=torch.Generator().manual_seed(7))
    for positions in (None, own):
        at = own if positions is not None else (torch.tensor(start)[:, None] + torch.arange(rows))[..., None].expand(-1, -1, 2)
        cache = PagedCache(keys.to(cuda_device), values.to(cuda_device))
        on = dict(page_table=table.to(cuda_device), start=torch.tensor(start, device=cuda_device),
                  counts=torch.tensor(counts, device=cuda_device), rotary=rotary,
                  positions=None if positions is None else positions.to(cuda_device))
        turned = cache.append(k.to(cuda_device), v.to(cuda_device), q=q.to(cuda_device), **on)
        want_q, bound_q = oracle.turn(q, at, rotary.frequencies, rotary.axes, interleaved=interleaved)
        assert ((turned.cpu().double() - want_q).abs() <= bound_q).all()
        want_k, bound_k = oracle.turn(k, at, rotary.frequencies, rotary.axes, interleaved=interleaved)
        want, want_v, bound = keys.double(), values.clone(), torch.zeros(keys.shape, dtype=torch.float64)
        oracle.append(want, want_v, want_k, v, page_table=table, start=start, counts=counts)
        oracle.append(bound, values.clone(), bound_k, v, page_table=table, start=start, counts=counts)
        assert ((cache.keys.cpu().double() - want).abs() <= bound).all()   # rows that are not written stay: bound 0
        assert torch.equal(cache.values.cpu(), want_v)
        # the keys in the pool and q are what rotate_positions gives, bit for bit
        again = rotate_positions(q.to(cuda_device), k.to(cuda_device), rotary=rotary, positions=at.to(cuda_device))
        assert torch.equal(again[0], turned)
        same = keys.clone()
        oracle.append(same, values.clone(), again[1].cpu(), v, page_table=table, start=start, counts=counts)
        assert torch.equal(cache.keys.cpu(), same)


def test_append_without_a_rotation_copies_bits(cuda_device):
    k, v = _rand((2, 2, 9, 16), BF16, 1), _rand((2, 2, 9, 16), BF16, 2)
    k[0, 0, 0, 0], k[1, 1, 8, 15], v[0, 1, 2, 3] = NAN, INF, -INF
    table, pages = _table(2, 3, 1, 3)
    keys, values = torch.zeros(pages, 2, 4, 16).bfloat16(), torch.zeros(pages, 2, 4, 16).bfloat16()
    cache = PagedCache(keys.to(cuda_device), values.to(cuda_device))
    assert cache.append(k.to(cuda_device), v.to(cuda_device), page_table=table.long().to(cuda_device),
                        start=torch.tensor([0, 3], dtype=torch.int64, device=cuda_device)) is None
    oracle.append(keys, values, k, v, page_table=table, start=[0, 3])
    assert torch.equal(cache.keys.cpu().view(torch.int16), keys.view(torch.int16))
    assert torch.equal(cache.values.cpu().view(torch.int16), values.view(torch.int16))


@pytest.mark.parametrize("start,counts", [([-3, 10, 2**31 - 1, -2**31, 0], None), ([0, 1, 2, 3, 4], [-1, 0, 99, 2, 2**31 - 1])])
def test_rows_without_a_place_are_skipped(cuda_device, start, counts):
    """Before the sequence, past the table, on entries that are no page, past the count."""
    k, v = _rand((5, 1, 6, 8), F16, 1), _rand((5, 1, 6, 8), F16, 2)
    table, pages = _table(5, 4, 2, 3)
    table[0, 0], table[1, 3], table[2, 1], table[3, 1] = -1, pages, 2**31 - 1, -2**31
    keys, values = _rand((pages, 1, 3, 8), F16, 4), _rand((pages, 1, 3, 8), F16, 5)
    # pages around the pool that nothing may touch
    guard = [torch.full((pages + 2, 1, 3, 8), 7.0, dtype=F16, device=cuda_device) for _ in range(2)]
    for g, x in zip(guard, (keys, values)):
        g[1:-1] = x.to(cuda_device)
    cache = PagedCache(guard[0][1:-1], guard[1][1:-1])
    rotary = RotaryAxes([0.0] * 4, [0] * 4, device=cuda_device)  # turns nothing, but through the rotation
    more = {} if counts is None else {"counts": torch.tensor(counts, device=cuda_device)}
    cache.append(k.to(cuda_device), v.to(cuda_device), page_table=table.to(cuda_device), rotary=rotary,
                 start=torch.tensor(start, device=cuda_device), **more)
    oracle.append(keys, values, k, v, page_table=table, start=start, counts=counts)
    for g, x in zip(guard, (keys, values)):
        assert torch.equal(g[1:-1].cpu(), x) and bool((g[0] == 7).all()) and bool((g[-1] == 7).all())


def test_append_follows_strides(cuda_device):
    """A pool laid out (pages, page_size, G, D), rows of one projection, a table of wider rows, broadcast keys."""
    rows = _rand((2, 5, 4, 16), BF16, 1)                       # (B, n, 2 G, D): keys and values of two heads
    table, pages = _table(2, 6, 0, 2)
    pool = torch.zeros(2, pages, 3, 2, 16, dtype=BF16, device=cuda_device)
    cache = PagedCache(pool[0].transpose(1, 2), pool[1].transpose(1, 2))
    on = rows.to(cuda_device)
    wide = torch.full((2, 9), -1, dtype=torch.int32, device=cuda_device)
    wide[:, 2:8] = table.to(cuda_device)
    start = torch.tensor([4, 0], device=cuda_device)
    cache.append(on[:, :, :2].transpose(1, 2), on[:, :, 2:].transpose(1, 2), page_table=wide[:, 2:8], start=start)
    keys, values = torch.zeros(pages, 2, 3, 16).bfloat16(), torch.zeros(pages, 2, 3, 16).bfloat16()
    oracle.append(keys, values, rows[:, :, :2].transpose(1, 2), rows[:, :, 2:].transpose(1, 2), page_table=table, start=[4, 0])
    assert torch.equal(cache.keys.cpu(), keys) and torch.equal(cache.values.cpu(), values)
    one = on[:1, :, :1].transpose(1, 2).expand(2, 2, 5, 16)
    cache.append(one, one, page_table=wide[:, 2:8], start=start)
    oracle.append(keys, values, one.cpu(), one.cpu(), page_table=table, start=[4, 0])
    assert torch.equal(cache.keys.cpu(), keys) and torch.equal(cache.values.cpu(), values)


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,groups,dim", [(1, 1, 8), (3, 3, 64), (8, 2, 64), (8, 1, 128), (9, 1, 40), (32, 2, 72), (6, 2, 128),
                                              (4, 2, 24), (16, 4, 32), (6, 3, 96), (12, 1, 104)])
@pytest.mark.parametrize("states,page_size", [(1, 1), (15, 16), (16, 3), (17, 16), (100, 5), (333, 32)])
@pytest.mark.parametrize("kernel", KERNELS)
def test_token_matches_oracle(cuda_device, dtype, heads, groups, dim, states, page_size, kernel):
    keys, values, table = _filled(2, groups, states, dim, page_size, dtype, 10)
    q = _rand((2, heads, 1, dim), dtype, 20)
    _check(cuda_device, q, keys, values, table, [states - 1, states // 2], kernel=kernel, scale=dim ** -0.5)


@pytest.mark.parametrize("batch,groups,states", [(1, 1, 5000), (1, 3, 1201), (5, 2, 700), (40, 1, 257), (75, 2, 64), (150, 1, 130)])
@pytest.mark.parametrize("kernel", KERNELS)
def test_sequences_of_every_split(cuda_device, batch, groups, states, kernel):
    """From one sequence that many CTAs share to more sequences than the GPU holds CTAs; ragged lengths, some of none."""
    keys, values, table = _filled(batch, groups, states, 64, 16, BF16, 30)
    g = torch.Generator().manual_seed(31)
    start = torch.randint(0, states, (batch,), generator=g).tolist()
    start[0] = states - 1
    if batch > 2:
        start[1], start[2] = -1, 0
    _check(cuda_device, _rand((batch, 2 * groups, 1, 64), BF16, 32), keys, values, table, start, kernel=kernel, scale=0.125)


@pytest.mark.parametrize("batch,groups,states,queries", [(43, 3, 150, 1), (130, 1, 70, 3), (300, 1, 20, 1)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_parts_of_many_sequences(cuda_device, batch, groups, states, queries, dtype):
    """Heads of 128 and 128 sequences and key heads or more: three CTAs an SM."""
    keys, values, table = _filled(batch, groups, states, 128, 8, dtype, 35)
    start = torch.randint(-queries, states - queries + 1, (batch,), generator=torch.Generator().manual_seed(36)).tolist()
    q = _rand((batch, 2 * groups, queries, 128), dtype, 37)
    _check(cuda_device, q, keys, values, table, start, kernel="parts", scale=128 ** -0.5)
    _check(cuda_device, q, keys, values, table, start, kernel="parts", scale=128 ** -0.5, window=33, sinks=2)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,groups,queries", [(4, 4, 2), (4, 2, 5), (8, 1, 3), (1, 1, 40), (12, 4, 17)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (5, 0), (7, 3), (40, 20), (1000, 4), (16, 100)])
@pytest.mark.parametrize("kernel", KERNELS)
def test_tokens_see_what_is_before_them(cuda_device, dtype, heads, groups, queries, window, sinks, kernel):
    if kernel == "parts" and queries * heads // groups > 16:
        kernel = "auto"  # rows that the parts do not take
    states, page_size = 90, 7
    keys, values, table = _filled(3, groups, states, 32, page_size, dtype, 40)
    q = _rand((3, heads, queries, 32), dtype, 41)
    _check(cuda_device, q, keys, values, table, [states - queries, 0, -2], kernel=kernel, scale=0.2, window=window,
           sinks=sinks)


@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (64, 4), (100, 17), (333, 0), (1024, 1), (2000, 0)])
@pytest.mark.parametrize("batch,groups", [(1, 1), (30, 2)])
@pytest.mark.parametrize("kernel", KERNELS)
def test_windows_over_long_sequences(cuda_device, window, sinks, batch, groups, kernel):
    states = 1500
    keys, values, table = _filled(batch, groups, states, 64, 24, BF16, 50)
    start = [(states - 1) * (i + 1) // batch for i in range(batch)]
    _check(cuda_device, _rand((batch, 4 * groups, 1, 64), BF16, 51), keys, values, table, start, kernel=kernel, scale=0.125,
           window=window, sinks=sinks)


@pytest.mark.parametrize("kernel", KERNELS)
def test_rows_past_their_count_are_zero(cuda_device, kernel):
    keys, values, table = _filled(4, 2, 50, 64, 16, BF16, 60)
    q = _rand((4, 4, 6, 64), BF16, 61)
    got = _check(cuda_device, q, keys, values, table, [40, 40, 40, 40], kernel=kernel, scale=0.125, counts=[0, 3, 6, -5])
    assert bool((got[0] == 0).all()) and bool((got[1, :, 3:] == 0).all()) and bool((got[3] == 0).all())
    assert bool((got[2] != 0).all())


@pytest.mark.parametrize("kernel", KERNELS)
def test_start_outside_the_table(cuda_device, kernel):
    """Positions past the table see all of it, far ones too; positions before the sequence see nothing."""
    keys, values, table = _filled(6, 1, 32, 16, 8, F16, 70)
    start = [31, 32, 100, 2**31 - 1, -1, -2**31]
    got = _attend(cuda_device, _rand((1, 2, 1, 16), F16, 71).expand(6, -1, -1, -1), keys, values, table, start, scale=0.25,
                  kernel=kernel)
    q = _rand((1, 2, 1, 16), F16, 71).expand(6, -1, -1, -1)
    want, bound = oracle.attend(q, keys, values, page_table=table, start=[31, 31, 31, 31, -1, -1], scale=0.25)
    assert ((got.cpu().double() - want).abs() <= bound).all()
    assert bool((got[4:] == 0).all())
    got = _attend(cuda_device, q, keys, values, table, start, scale=0.25, window=4, sinks=2, kernel=kernel)
    want, bound = oracle.attend(q, keys, values, page_table=table, start=[31, 32, 100, 10**6, -1, -1], scale=0.25, window=4,
                                sinks=2)
    assert ((got.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("kernel", KERNELS)
def test_pages_that_are_none_take_no_part(cuda_device, kernel):
    keys, values, table = _filled(4, 2, 60, 32, 5, BF16, 80)
    pages = keys.shape[0]
    table[0, 3], table[1, 0], table[2, 11], table[3, :] = -1, pages, 2**31 - 1, -2**31
    q = _rand((4, 4, 3, 32), BF16, 81)
    got = _check(cuda_device, q, keys, values, table, [57] * 4, kernel=kernel, scale=0.2)
    assert bool((got[3] == 0).all())
    _check(cuda_device, q[:, :, :1], keys, values, table, [59] * 4, kernel=kernel, scale=0.2, window=30, sinks=6)


def test_shared_pages_and_a_broadcast_table(cuda_device):
    """Sequences that read the same pages, and a page twice in one table."""
    keys, values, table = _filled(1, 2, 48, 64, 16, BF16, 90)
    table = table.expand(3, 3)
    _check(cuda_device, _rand((3, 2, 1, 64), BF16, 91), keys, values, table, [47, 20, 33], scale=0.125)
    twice = table[:1, [0, 1, 0]].contiguous()
    _check(cuda_device, _rand((1, 2, 1, 64), BF16, 92), keys, values, twice, [47], scale=0.125)


# ------------------------------------------------------------------ what is not finite
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
@pytest.mark.parametrize("queries,window", [(4, None), (4, 6), (17, None), (17, 3)])
@pytest.mark.parametrize("heads", [1, 3])
@pytest.mark.parametrize("kernel", KERNELS)
def test_states_that_a_row_does_not_see_never_show(cuda_device, bad, queries, window, heads, kernel):
    """A state that later rows of the same tile see, or that left the window of some, holds what is not finite."""
    states = 50
    if kernel == "parts" and queries * heads > 16:
        kernel = "auto"
    for at in (states - 1, states - 2, states - queries + 1, states - queries - 2):
        for which in (0, 1):
            keys, values, table = _filled(1, 1, states, 32, 16, BF16, 100)
            clean = (keys.clone(), values.clone())
            page, row = oracle.place(table, 16, keys.shape[0], 0, at)
            (keys, values)[which][page, 0, row, 5] = bad
            q = _rand((1, heads, queries, 32), BF16, 101)
            start = [states - queries]
            got = _attend(cuda_device, q, keys, values, table, start, scale=0.2, window=window, kernel=kernel).cpu()
            base = _attend(cuda_device, q, *clean, table, start, scale=0.2, window=window, kernel=kernel).cpu()
            for m in range(queries):
                position = start[0] + m
                sees = at <= position and (window is None or at > position - window)
                if not sees:
                    assert torch.equal(got[:, :, m], base[:, :, m])
                elif which == 1:
                    column = got[:, :, m, 5]
                    assert bool((torch.isnan(column) if bad != bad else column == bad).all())
                    other = torch.arange(32) != 5
                    assert torch.equal(got[:, :, m][..., other], base[:, :, m][..., other])


@pytest.mark.parametrize("kernel", KERNELS)
def test_minus_infinite_scores(cuda_device, kernel):
    """A row whose every score is -inf gives zeros; a single one takes no weight."""
    keys, values, table = _filled(2, 1, 20, 16, 4, BF16, 110)
    q = torch.ones(2, 1, 1, 16).bfloat16()
    for j in range(20):
        page, row = oracle.place(table, 4, keys.shape[0], 0, j)
        keys[page, 0, row] = -INF
    page, row = oracle.place(table, 4, keys.shape[0], 1, 3)
    keys[page, 0, row] = -INF
    got = _check(cuda_device, q, keys, values, table, [19, 19], kernel=kernel, scale=0.25)
    assert bool((got[0] == 0).all())


@pytest.mark.parametrize("kernel", KERNELS)
def test_plus_infinite_scores_and_nan_spread(cuda_device, kernel):
    keys, values, table = _filled(2, 1, 200, 16, 16, BF16, 120)
    q = torch.ones(2, 1, 1, 16).bfloat16()
    page, row = oracle.place(table, 16, keys.shape[0], 0, 100)
    keys[page, 0, row] = INF
    got = _attend(cuda_device, q, keys, values, table, [199, 199], scale=0.25, kernel=kernel)
    assert bool(torch.isnan(got[0]).all()) and bool(torch.isfinite(got[1]).all())
    q[1, 0, 0, 3] = NAN
    got = _attend(cuda_device, q, keys, values, table, [99, 199], scale=0.25, kernel=kernel)
    assert bool(torch.isnan(got[1]).all()) and bool(torch.isfinite(got[0]).all())


@pytest.mark.parametrize("kernel", KERNELS)
def test_scores_of_any_size(cuda_device, kernel):
    keys, values, table = _filled(1, 1, 300, 64, 16, BF16, 130)
    _check(cuda_device, _rand((1, 1, 1, 64), BF16, 131, 30.0), keys, values, table, [299], kernel=kernel, scale=1.0)
    _check(cuda_device, _rand((1, 1, 1, 64), BF16, 132, 1e-20), keys, values, table, [299], kernel=kernel, scale=1.0)


# ------------------------------------------------------------------ as it is used
def _pool(device, batch, groups, states, dim, page_size, dtype=BF16):
    table, pages = _table(batch, -(-states // page_size), 2, 140)
    return PagedCache.empty(pages, groups, page_size, dim, dtype=dtype, device=device), table.to(device)


def test_a_prompt_and_steps_behind_it(cuda_device):
    """Prompt, then tokens one at a time, all through append and paged_attention: each row is cross
    attention to the states before it, turned by their positions."""
    batch, heads, groups, dim, rows, steps = 3, 8, 2, 64, 37, 6
    cache, table = _pool(cuda_device, batch, groups, 64, dim, 16)
    rotary = RotaryAxes.sections([32], device=cuda_device)
    q, k, v = (_rand((batch, h, rows + steps, dim), BF16, 150 + h).to(cuda_device) for h in (heads, groups, groups + 1))
    v = v[:, :groups]
    counts = torch.tensor([37, 20, 1], dtype=torch.int32, device=cuda_device)
    start = torch.zeros(batch, dtype=torch.int32, device=cuda_device)

    def run(lo, hi, start, counts):
        turned = cache.append(k[:, :, lo:hi], v[:, :, lo:hi], page_table=table, start=start, counts=counts, rotary=rotary,
                              q=q[:, :, lo:hi])
        return paged_attention(turned, cache, page_table=table, start=start, counts=counts, scale=dim ** -0.5)

    outs = [run(0, rows, start, counts)]
    start = start + counts
    for i in range(steps):
        outs.append(run(rows + i, rows + i + 1, start, None))
        start = start + 1
    for b, count in enumerate(counts.tolist()):
        index = [*range(count), *range(rows, rows + steps)]
        at = torch.arange(len(index), device=cuda_device)[:, None]
        tq, tk = rotate_positions(q[b:b + 1, :, index], k[b:b + 1, :, index], rotary=rotary, positions=at)
        got = torch.cat((outs[0][b:b + 1, :, :count], *(o[b:b + 1] for o in outs[1:])), dim=2)
        assert bool((outs[0][b, :, count:] == 0).all())
        for m in range(len(index)):
            want = cross_attention(tq[:, :, m:m + 1], tk[:, :, :m + 1], v[b:b + 1][:, :, index][:, :, :m + 1], scale=dim ** -0.5)
            # both round the same 64-bit result once: a unit in the last place apart, and what fp32 adds
            gap = (got[:, :, m:m + 1].float() - want.float()).abs()
            assert bool((gap <= 2.0 ** -7 * want.float().abs() + 1e-5).all())


def test_captured_decode_step(cuda_device):
    """A step captured once, replayed with lengths, pages and tokens that change in place."""
    batch, heads, groups, dim = 4, 8, 4, 64
    cache, table = _pool(cuda_device, batch, groups, 96, dim, 8)
    eager, _ = _pool(cuda_device, batch, groups, 96, dim, 8)
    rotary = RotaryAxes.sections([16, 8, 8], device=cuda_device)
    q, k, v = (torch.zeros(batch, h, 1, dim, dtype=BF16, device=cuda_device) for h in (heads, groups, groups))
    start = torch.zeros(batch, dtype=torch.int32, device=cuda_device)

    def step(pool):
        turned = pool.append(k, v, page_table=table, start=start, rotary=rotary, q=q)
        return paged_attention(turned, pool, page_table=table, start=start, scale=0.125, window=30, sinks=2)

    step(PagedCache.empty(*cache.shape, device=cuda_device))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cache)
    cache.keys.zero_()
    cache.values.zero_()
    for i in range(90):
        for t, seed in ((q, 3 * i), (k, 3 * i + 1), (v, 3 * i + 2)):
            t.copy_(_rand(t.shape, BF16, seed))
        graph.replay()
        assert torch.equal(out, step(eager))
        start += 1
    assert torch.equal(cache.keys, eager.keys)


def test_other_streams_strides_and_repeats(cuda_device):
    keys, values, table = _filled(2, 2, 400, 64, 16, BF16, 160)
    table = table.to(cuda_device)
    cache = PagedCache(keys.to(cuda_device), values.to(cuda_device))
    q = _rand((2, 1, 4, 64), BF16, 161).to(cuda_device).transpose(1, 2)           # token-major rows
    start = torch.tensor([399, 123], device=cuda_device)
    first = paged_attention(q, cache, page_table=table, start=start, scale=0.125)
    for kernel in KERNELS * 2:
        again = [paged_attention(q, cache, page_table=table, start=start, scale=0.125, kernel=kernel) for _ in range(3)]
        assert torch.equal(again[0], again[1]) and torch.equal(again[0], again[2])
    for _ in range(3):
        assert torch.equal(first, paged_attention(q, cache, page_table=table, start=start, scale=0.125))
    stream = torch.cuda.Stream(cuda_device)
    stream.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(stream):
        other = paged_attention(q, cache, page_table=table, start=start, scale=0.125)
    torch.cuda.current_stream(cuda_device).wait_stream(stream)
    assert torch.equal(first, other)
    # a pool laid out (pages, page_size, G, D), rows that are not aligned, a wider output
    pool = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (cache.keys, cache.values)]
    odd = torch.zeros(2, 4, 1, 65, dtype=BF16, device=cuda_device)[..., 1:]
    odd.copy_(q)
    wide = torch.full((2, 4, 3, 64), 7.0, dtype=BF16, device=cuda_device)
    got = paged_attention(odd, PagedCache(*pool), page_table=table, start=start, scale=0.125, out=wide[:, :, 1:2])
    assert got.data_ptr() == wide[:, :, 1:2].data_ptr() and torch.equal(got, first)
    assert bool((wide[:, :, 0] == 7).all()) and bool((wide[:, :, 2] == 7).all())


def test_a_first_call_may_be_captured(cuda_device):
    """In a process of its own: nothing of a call has to have run before it is captured."""
    import subprocess
    import sys
    from pathlib import Path

    code = """
import torch
from intp_preliminary_b200 import PagedCache, RotaryAxes, paged_attention
cache = PagedCache.empty(9, 2, 8, 64, device="cuda")
rotary = RotaryAxes.sections([32], device="cuda")
table = torch.arange(8, dtype=torch.int32, device="cuda").reshape(2, 4)
start = torch.zeros(2, dtype=torch.int32, device="cuda")
q, k = torch.randn(2, 4, 3, 64, device="cuda").bfloat16(), torch.randn(2, 2, 3, 64, device="cuda").bfloat16()
def step(kernel):
    turned = cache.append(k, k, page_table=table, start=start, rotary=rotary, q=q)
    return paged_attention(turned, cache, page_table=table, start=start, scale=0.125, kernel=kernel)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    outs = [step("joined"), step("parts")]
graph.replay()
wants = [step("joined"), step("parts")]
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(outs, wants)) and bool((outs[0] != 0).any())
"""
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300, cwd=Path(__file__).resolve().parent.parent)


def test_two_graphs_at_once(cuda_device):
    """Graphs of the two kernels replayed together on two streams: each has its own scratch."""
    keys, values, table = _filled(3, 2, 700, 64, 16, BF16, 180)
    cache, table = PagedCache(keys.to(cuda_device), values.to(cuda_device)), table.to(cuda_device)
    start = torch.tensor([699, 200, 3], dtype=torch.int32, device=cuda_device)
    work = []
    for seed in range(4):
        q = _rand((3, 4, 1, 64), BF16, 181 + seed).to(cuda_device)
        more = dict(page_table=table, start=start, scale=0.125, kernel=KERNELS[seed % 2])
        want = paged_attention(q, cache, **more)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = paged_attention(q, cache, **more)
        work.append((q, graph, out, want, torch.cuda.Stream(cuda_device)))  # a graph does not keep its inputs
    for _ in range(20):
        for _, graph, out, _, stream in work:
            stream.wait_stream(torch.cuda.current_stream(cuda_device))
            with torch.cuda.stream(stream):
                out.zero_()
                graph.replay()
        for *_, stream in work:
            torch.cuda.current_stream(cuda_device).wait_stream(stream)
        assert all(torch.equal(out, want) for *_, out, want, _ in work)


def test_calls_from_two_threads(cuda_device):
    import threading

    keys, values, table = _filled(2, 2, 300, 64, 16, BF16, 190)
    cache, table = PagedCache(keys.to(cuda_device), values.to(cuda_device)), table.to(cuda_device)
    rotary = RotaryAxes.sections([32], device=cuda_device)
    start = torch.tensor([299, 100], dtype=torch.int32, device=cuda_device)
    results, wants = [[], []], []
    for which in range(2):
        q = _rand((2, 4, 1, 64), BF16, 191 + which).to(cuda_device)
        turned, _ = rotate_positions(q, rotary=rotary, positions=start[:, None, None])
        wants.append((q, paged_attention(turned, cache, page_table=table, start=start, scale=0.125, kernel=KERNELS[which])))
    torch.cuda.synchronize(cuda_device)

    def call(which):
        stream = torch.cuda.Stream(cuda_device)
        with torch.cuda.stream(stream):
            for _ in range(50):
                turned, _ = rotate_positions(wants[which][0], rotary=rotary, positions=start[:, None, None])
                results[which].append(paged_attention(turned, cache, page_table=table, start=start, scale=0.125,
                                                      kernel=KERNELS[which]))
        stream.synchronize()

    threads = [threading.Thread(target=call, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for got, (_, want) in zip(results, wants):
        assert len(got) == 50 and all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("kernel", KERNELS)
def test_the_result_may_take_the_queries_place(cuda_device, kernel):
    keys, values, table = _filled(2, 2, 900, 64, 16, BF16, 200)
    q = _rand((2, 8, 3, 64), BF16, 201).to(cuda_device)
    cache, table = PagedCache(keys.to(cuda_device), values.to(cuda_device)), table.to(cuda_device)
    start = torch.tensor([897, 40], dtype=torch.int32, device=cuda_device)
    more = dict(page_table=table, start=start, scale=0.125, kernel=kernel)
    want = paged_attention(q, cache, **more)
    assert paged_attention(q, cache, out=q, **more) is q
    assert torch.equal(q, want)


def test_a_long_row_of_new_tokens(cuda_device):
    """More rows than a tile holds: a prompt of 300 tokens behind 50 states, every query head group size."""
    for heads, groups in ((2, 2), (6, 2), (16, 1)):
        keys, values, table = _filled(2, groups, 350, 32, 16, BF16, 210 + heads)
        q = _rand((2, heads, 300, 32), BF16, 211 + heads)
        got = _attend(cuda_device, q, keys, values, table, [50, 0], scale=0.2, counts=[300, 290]).cpu()
        for rows in (slice(0, 3), slice(150, 153), slice(287, 290), slice(297, 300)):
            at = rows.start
            want, bound = oracle.attend(q[:, :, rows], keys, values, page_table=table, start=[50 + at, at], scale=0.2,
                                        counts=[min(max(c - at, 0), 3) for c in (300, 290)])
            assert ((got[:, :, rows].double() - want).abs() <= bound).all()


def test_long_cache_past_32_bit_offsets(cuda_device):
    """Pages whose elements lie past 2^31, written and read."""
    page_size, dim, groups = 256, 128, 8
    pages = (1 << 31) // (page_size * dim * groups) + 20
    keys = torch.zeros(pages, groups, page_size, dim, dtype=BF16, device=cuda_device)
    cache = PagedCache(keys, torch.zeros_like(keys))
    far = torch.tensor([[pages - 1, 0, pages - 3]], dtype=torch.int32, device=cuda_device)
    near = torch.tensor([[1, 2, 3]], dtype=torch.int32, device=cuda_device)
    k, v = (_rand((1, groups, 700, dim), BF16, s).to(cuda_device) for s in (170, 171))
    q = _rand((1, 32, 1, dim), BF16, 172).to(cuda_device)
    start = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    outs = []
    for table in (far, near):
        cache.append(k, v, page_table=table, start=start)
        outs += [paged_attention(q, cache, page_table=table, start=start + 699, scale=dim ** -0.5, kernel=kernel)
                 for kernel in KERNELS]
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3]) and torch.equal(cache.keys[pages - 1, :, 3], k[0, :, 3])
    want = cross_attention(q, k, v, scale=dim ** -0.5)
    for got in outs[:2]:
        assert bool(((got.float() - want.float()).abs() <= 2.0 ** -7 * want.float().abs() + 1e-5).all())


def test_refusals(cuda_device):
    cache, table = _pool(cuda_device, 2, 2, 32, 16, 8)
    q = torch.zeros(2, 4, 1, 16, dtype=BF16, device=cuda_device)
    k = torch.zeros(2, 2, 1, 16, dtype=BF16, device=cuda_device)
    start = torch.zeros(2, dtype=torch.int32, device=cuda_device)
    rotary = RotaryAxes.sections([8], device=cuda_device)
    good = dict(page_table=table, start=start, scale=0.25)
    for args, over, message in (
            ((q.float(), cache), {}, "must be bfloat16"), ((q.half(), cache), {}, "cache's dtype"), ((q[:, :3], cache), {}, "multiple"),
            ((q[..., :8], cache), {}, "head_dim"), ((q[:1], cache), {}, "row for each sequence"), ((q[0], cache), {}, "shape"),
            ((q, cache), {"page_table": table.float()}, "page_table"), ((q, cache), {"page_table": table[0]}, "page_table"),
            ((q, cache), {"page_table": table.cpu()}, "same CUDA device"), ((q, cache), {"page_table": table[:, :0]}, "at least one page"),
            ((q, cache), {"start": None}, "start"), ((q, cache), {"start": start[:1]}, "start"), ((q, cache), {"start": start.float()}, "start"),
            ((q, cache), {"page_table": [[0]]}, "page_table"), ((3, cache), {}, "CUDA"), ((q, cache), {"counts": [1, 1]}, "counts"),
            ((q, cache), {"out": 3}, "out"), ((q, q), {}, "PagedCache"),
            ((q, cache), {"counts": start[:1]}, "counts"), ((q, cache), {"scale": 0.0}, "scale"), ((q, cache), {"window": 0}, "window"),
            ((q, cache), {"sinks": -1, "window": 4}, "sinks"), ((q, cache), {"sinks": 2}, "window"),
            ((q, cache), {"out": q[..., :8]}, "out"), ((q, cache), {"kernel": "tiles"}, "kernel"),
            ((torch.zeros(2, 20, 2, 16, dtype=BF16, device=cuda_device), cache), {"kernel": "parts"}, "does not take"), ((q.clone().requires_grad_(), cache), {}, "no backward")):
        with pytest.raises(ValueError, match=message):
            paged_attention(*args, **{**good, **over})
    good = dict(page_table=table, start=start)
    for args, over, message in (
            ((k, k.float()), {}, "must be bfloat16"), ((k.half(), k.half()), {}, "cache's dtype"), ((k[:, :1], k[:, :1]), {}, "shape"),
            ((k, k[:1]), {}, "shape"), ((k[..., :8], k[..., :8]), {}, "shape"), ((k, None), {}, "CUDA"), ((k, k), {"start": None}, "start"),
            ((k, k), {"q": q}, "rotary"), ((k, k), {"positions": start[:1, None]}, "rotary"), ((k, k), {"rotary": 3}, "RotaryAxes"),
            ((k, k), {"rotary": rotary, "q": q[:1]}, "shape"), ((k, k), {"rotary": rotary, "positions": start[:, None]}, "positions"),
            ((k, k), {"rotary": RotaryAxes.sections([12], device=cuda_device)}, "more columns"),
            ((k, k.clone().requires_grad_()), {}, "no backward"), ((k, k), {"start": [0, 0]}, "start"),
            ((k, k), {"rotary": rotary, "positions": torch.zeros(1, 1, device=cuda_device, requires_grad=True)}, "no backward"),
            ((k, k), {"rotary": rotary, "q": q.clone().requires_grad_()}, "no backward"), ((k, 3), {}, "CUDA"),
            ((k, k), {"rotary": rotary, "positions": [0]}, "positions"), ((k, k), {"page_table": table[:1]}, "row for each sequence")):
        with pytest.raises(ValueError, match=message):
            cache.append(*args, **{**good, **over})
    for keys, values, message in ((k, k.half(), "dtype"), (k.float(), k.float(), "bfloat16"), (k[0], k[0], "shape"),
                                  (k[:0], k[:0], "needs a page"), (k[..., :4], k[..., :4], "multiple of 8"),
                                  (k[..., :8].transpose(1, 3), k[..., :8].transpose(1, 3), "multiple of 8"),
                                  (k.expand(2, 2, 5, 16), k.expand(2, 2, 5, 16), "unit stride"),
                                  (table.new_zeros(2, 2, 3, 16, dtype=BF16), table.new_zeros(2, 3, 2, 16, dtype=BF16).transpose(1, 2), "share their strides")):
        with pytest.raises(ValueError, match=message):
            PagedCache(keys, values)
    with pytest.raises(ValueError, match="no part in autograd"):
        PagedCache(k.clone().requires_grad_(), k)
    for name in ("keys", "values", "layout"):
        with pytest.raises(AttributeError):
            setattr(cache, name, None)


def test_tangents_and_traces_are_refused(cuda_device):
    cache, table = _pool(cuda_device, 2, 2, 32, 16, 8)
    q = torch.zeros(2, 4, 1, 16, dtype=BF16, device=cuda_device)
    k = torch.zeros(2, 2, 1, 16, dtype=BF16, device=cuda_device)
    more = dict(page_table=table, start=torch.zeros(2, dtype=torch.int32, device=cuda_device))
    paged_attention(q, cache, scale=0.25, **more)                 # a call that is known by its layout is refused too
    cache.append(k, k, **more)
    forward_ad = torch.autograd.forward_ad
    with forward_ad.dual_level():
        dual_q, dual_k = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (q, k))
        for call in (lambda: paged_attention(dual_q, cache, scale=0.25, **more), lambda: cache.append(dual_k, k, **more),
                     lambda: cache.append(k, dual_k, **more)):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
        paged_attention(q, cache, scale=0.25, **more)             # the primal alone is none of that
    for call in (lambda: paged_attention(q, cache, scale=0.25, **more), lambda: cache.append(k, k, **more)):
        with pytest.raises(ValueError, match="traced"):
            torch.jit.trace(lambda t: (call(), t)[1], torch.zeros(1, device=cuda_device), check_trace=False)


def test_empty_batches_and_rows(cuda_device):
    cache, table = _pool(cuda_device, 2, 2, 32, 16, 8)
    start = torch.zeros(2, dtype=torch.int32, device=cuda_device)
    q = torch.zeros(2, 4, 0, 16, dtype=BF16, device=cuda_device)
    assert paged_attention(q, cache, page_table=table, start=start, scale=0.25).shape == q.shape
    cache.append(q[:, :2], q[:, :2], page_table=table, start=start)
    q = torch.zeros(0, 4, 1, 16, dtype=BF16, device=cuda_device)
    assert paged_attention(q, cache, page_table=table[:0], start=start[:0], scale=0.25).shape == q.shape
    cache.append(q[:, :2], q[:, :2], page_table=table[:0], start=start[:0])
    assert bool((cache.keys == 0).all())


def test_copied_caches_hold_states_of_their_own(cuda_device):
    import copy
    import io
    import pickle

    from intp_preliminary_b200 import StateCache

    keys, values, table = _filled(2, 2, 40, 32, 8, BF16, 220, hole=0.0)
    pool = torch.stack((keys, values)).transpose(2, 3).contiguous().to(cuda_device).transpose(2, 3)
    cache = PagedCache(pool[0], pool[1])
    state = StateCache.empty(2, 2, 16, 32, device=cuda_device)
    state.write(*(_rand((2, 2, 16, 32), BF16, 221 + i).to(cuda_device) for i in range(2)))
    q, table = _rand((2, 4, 1, 32), BF16, 223).to(cuda_device), table.to(cuda_device)
    start = torch.tensor([39, 20], device=cuda_device)
    want, states = paged_attention(q, cache, page_table=table, start=start, scale=0.2), state.read()
    file = io.BytesIO()
    torch.save([cache, state], file)
    file.seek(0)
    loaded = torch.load(file, weights_only=False)
    copies = [copy.deepcopy((cache, state)), (pickle.loads(pickle.dumps(cache)), loaded[1]), loaded]
    pool.zero_()
    state.keys.zero_()
    for paged, other in copies:
        assert paged.keys.stride() == cache.keys.stride()
        assert torch.equal(paged_attention(q, paged, page_table=table, start=start, scale=0.2), want)
        assert all(torch.equal(a, b) for a, b in zip(other.read(), states))
    file.seek(0)
    with pytest.raises(ValueError, match="CUDA"):
        torch.load(file, weights_only=False, map_location="cpu")


@pytest.mark.parametrize("start", [2**30 + 1000, 2**30 - 3, 2**31 - 1, 2**30 + 2100])
@pytest.mark.parametrize("queries", [1, 4, 20])
@pytest.mark.parametrize("sinks", [0, 3])
@pytest.mark.parametrize("kernel", KERNELS)
def test_a_long_window_of_far_rows(cuda_device, start, queries, sinks, kernel):
    """The window of a row far behind the table ends inside it, at the row's own place: 2^30 states back."""
    if kernel == "parts" and queries > 16:
        kernel = "auto"
    keys, values, table = _filled(2, 1, 2000, 16, 64, BF16, 230)
    q = _rand((2, 1, queries, 16), BF16, 231)
    got = _check(cuda_device, q, keys, values, table, [start, 1990], kernel=kernel, scale=0.25, window=2**30, sinks=sinks)
    if start > 2**30 + 2000 and sinks == 0:
        assert bool((got[0] == 0).all())


# ------------------------------------------------------------------ small probabilities
def _steps(dtype, dim, states, scores, seed):
    """One sequence whose state j has the score scores.get(j, 0) for every query, and its queries."""
    keys, values, table = _filled(1, 1, states, dim, 16, dtype, seed)
    for j in range(states):
        page, row = oracle.place(table, 16, keys.shape[0], 0, j)
        keys[page, 0, row] = 0
        keys[page, 0, row, 0] = scores.get(j, 0.0)
    return keys, values, table


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [8, 32, 64, 72, 128])
@pytest.mark.parametrize("heads,queries", [(1, 1), (2, 3), (5, 3)])
@pytest.mark.parametrize("gap", [5.0, 18.0, 25.0, 40.0, 60.0, 86.0])
@pytest.mark.parametrize("kernel", KERNELS)
def test_an_infinite_state_shows_however_small_its_probability(cuda_device, dtype, dim, heads, queries, gap, kernel):
    """Before and behind the state of the largest score; 86 below it is 2^-124, which 32 bits hold."""
    states, column = 300, dim - 3
    q = torch.zeros(1, heads, queries, dim).to(dtype)
    q[..., 0] = 1
    for top, at, bad in ((150, 7, INF), (150, 290, -INF), (40, 44, INF), (150, 288, NAN)):
        keys, values, table = _steps(dtype, dim, states, {top: gap}, 240)
        page, row = oracle.place(table, 16, keys.shape[0], 0, at)
        values[page, 0, row, column] = bad
        got = _check(cuda_device, q, keys, values, table, [states - queries], kernel=kernel, scale=1.0)
        shown = got[..., column]
        assert bool((torch.isnan(shown) if bad != bad else shown == bad).all())
        assert bool(torch.isfinite(got[..., torch.arange(dim) != column]).all())


@pytest.mark.parametrize("dtype,gap,size", [(BF16, 30.0, 1.0), (BF16, 45.0, 2.0**60), (BF16, 60.0, 2.0**90), (BF16, 75.0, 2.0**100),
                                            (F16, 10.0, 1.0), (F16, 14.0, 1000.0), (F16, 15.0, 20000.0), (F16, 16.0, 20000.0),
                                            (F16, 17.0, 20000.0), (F16, 20.0, 30000.0)])
@pytest.mark.parametrize("dim", [32, 64, 80, 128])
@pytest.mark.parametrize("heads,queries", [(1, 1), (3, 4)])
@pytest.mark.parametrize("kernel", KERNELS)
def test_small_probabilities_count_once(cuda_device, dtype, gap, size, dim, heads, queries, kernel):
    """One state takes nearly all of the weight and holds zeros: the result is what the others add to it."""
    states, top = 300, 150
    q = torch.zeros(1, heads, queries, dim).to(dtype)
    q[..., 0] = 1
    keys, values, table = _steps(dtype, dim, states, {top: gap}, 250)
    values = ((values.float().abs() + 0.5).clamp(max=1.9) * size).to(dtype)  # of one sign: errors of one sign add up
    page, row = oracle.place(table, 16, keys.shape[0], 0, top)
    values[page, 0, row] = 0
    got = _check(cuda_device, q, keys, values, table, [states - queries], kernel=kernel, scale=1.0)
    assert bool((got > 0).all())


class NamedPool(PagedCache):
    def __init__(self, name, pages):
        super().__init__(*(torch.zeros(pages, 1, 8, 16, dtype=BF16, device="cuda") for _ in range(2)))
        self.name = name


def test_copies_of_a_subclass_keep_what_it_holds(cuda_device):
    import copy
    import pickle

    pool = NamedPool("first", 3)
    for other in (copy.copy(pool), copy.deepcopy(pool), pickle.loads(pickle.dumps(pool))):
        assert type(other) is NamedPool and other.name == "first" and other.layout == pool.layout
    assert copy.copy(pool).keys is pool.keys and copy.deepcopy(pool).keys is not pool.keys
