"""Attention over pages at the lengths it is made for: rings that come round several times, shares of many
slices, joins of many parts, both sides of the choice between the kernels; several tokens at every kind
of head dim.  Against the float64 oracle."""

import pytest
import torch

from intp_preliminary_b200 import PagedCache, check_device_status, paged_attention
from intp_preliminary_b200.paged_cache import _attention_plan
from oracle import paged as oracle

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
KERNELS = ["joined", "parts"]
NAN, INF = float("nan"), float("inf")
MOST_WARPS = 148 * 12        # that share a batch: three CTAs of four an SM


@pytest.fixture(autouse=True)
def _device_status(cuda_device):
    yield
    check_device_status(cuda_device)


def _rand(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _dealt(lengths, groups, dim, page_size, dtype, seed):
    """Pools in which sequence b holds lengths[b] states, and its table; NaN wherever no state is."""
    batch, width = len(lengths), -(-max(lengths) // page_size)
    pages = batch * width + 3
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[:batch * width]
    pools = []
    for i in (1, 2):
        states = _rand((batch, groups, width * page_size, dim), dtype, seed + i)
        for b, n in enumerate(lengths):
            states[b, :, n:] = NAN
        pool = torch.full((pages, groups, page_size, dim), NAN, dtype=dtype)
        pool[order] = states.unflatten(2, (width, page_size)).transpose(1, 2).flatten(0, 1)
        pools.append(pool)
    return *pools, order.reshape(batch, width).to(torch.int32)


def _check(device, q, keys, values, table, start, kernels=KERNELS, **more):
    cache = PagedCache(keys.to(device), values.to(device))
    on = dict(page_table=table.to(device), start=torch.tensor(start, device=device),
              **{n: torch.tensor(x, device=device) if isinstance(x, list) else x for n, x in more.items()})
    want, bound = oracle.attend(q, keys, values, page_table=table, start=start, **more)
    for kernel in kernels:
        got = paged_attention(q.to(device), cache, kernel=kernel, **on).cpu().double()
        error = (got - want).abs()
        assert bool((error <= bound).all()), f"{kernel}: {float((error / bound).nan_to_num(INF).max())} times the bound"


def _slices(lengths, groups, dim):
    return groups * sum(-(-n // (32 if dim <= 64 else 16)) for n in lengths)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("batch,groups,per_group,queries,dim,longest", [
    (32, 4, 2, 1, 128, 2500),      # many items of 8 rows at most at head_dim 128
    (43, 3, 2, 3, 128, 1900),
    (8, 4, 4, 2, 128, 5800),
    (4, 4, 4, 2, 128, 15000),      # few of them
    (8, 4, 4, 4, 128, 5800),       # 16 rows
    (8, 4, 4, 2, 80, 5800),
    (8, 4, 3, 5, 80, 5800),
    (8, 4, 1, 7, 72, 5800),
    (8, 4, 4, 2, 64, 11600),
    (15, 4, 4, 4, 64, 7000),       # parts of a row joined by four warps
    (8, 4, 2, 3, 32, 19000),
    (8, 4, 8, 2, 24, 19000),
])
def test_shares_of_many_slices(cuda_device, dtype, batch, groups, per_group, queries, dim, longest):
    """Every warp has more slices than its ring holds, and the parts' slices run across items."""
    g = torch.Generator().manual_seed(300)
    lengths = (longest - torch.randint(0, longest // 8, (batch,), generator=g)).tolist()
    lengths[1] = 0
    depth = 6 if dim <= 32 else 3
    assert _slices(lengths, groups, dim) >= (depth + 2) * MOST_WARPS
    warps = min(64, 2 * MOST_WARPS // (batch * groups))            # that an item may get of the other kernel
    assert min(n for n in lengths if n) // (32 if dim <= 64 else 16) > depth * warps
    keys, values, table = _dealt(lengths, groups, dim, 24, dtype, 301)
    q = _rand((batch, groups * per_group, queries, dim), dtype, 304)
    start = [n - queries for n in lengths]
    counts = [queries] * batch
    counts[2] -= 1
    _check(cuda_device, q, keys, values, table, start, scale=dim ** -0.5, counts=counts)
    _check(cuda_device, q, keys, values, table, start, scale=dim ** -0.5, window=longest // 2, sinks=5)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim,states", [(128, 20000), (64, 40000)])
def test_a_row_of_more_parts_than_one_pass_joins(cuda_device, dtype, dim, states):
    assert _slices([states], 1, dim) > 1024                       # two slices a warp: more than 512 parts
    keys, values, table = _dealt([states], 1, dim, 64, dtype, 310)
    _check(cuda_device, _rand((1, 4, 1, dim), dtype, 313), keys, values, table, [states - 1], scale=dim ** -0.5)


@pytest.mark.parametrize("batch,groups,dim,states,parts", [
    (1, 1, 128, 20000, False), (1, 1, 128, 30000, True),          # a warp's slices while most warps are idle
    (100, 6, 72, 1900, False), (100, 6, 72, 2100, True),          # and while all are at work
])
def test_the_choice_between_the_kernels(cuda_device, batch, groups, dim, states, parts):
    g = torch.Generator(device=cuda_device).manual_seed(320)
    width = -(-states // 16)
    pages = batch * width
    table = torch.randperm(pages, generator=g, device=cuda_device).reshape(batch, width).to(torch.int32)
    cache = PagedCache(*(torch.randn(pages, groups, 16, dim, generator=g, device=cuda_device, dtype=BF16) for _ in range(2)))
    q = torch.randn(batch, 2 * groups, 1, dim, generator=g, device=cuda_device, dtype=BF16)
    start = torch.randint(0, states, (batch,), generator=g, device=cuda_device, dtype=torch.int32)
    assert (_attention_plan(q, cache, table, 0.1, None, 0, "auto", None)[1] > 0) == parts
    more = dict(page_table=table, start=start, scale=dim ** -0.5)
    auto, forced = (paged_attention(q, cache, kernel=k, **more) for k in ("auto", KERNELS[parts]))
    assert torch.equal(auto, forced)
    other = paged_attention(q, cache, kernel=KERNELS[not parts], **more)
    # the same 64-bit result, rounded once by each
    assert bool(((auto.float() - other.float()).abs() <= 2.0 ** -7 * auto.float().abs() + 1e-4).all())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [56, 64, 80, 104, 128])
@pytest.mark.parametrize("heads,groups,queries", [(4, 4, 2), (4, 2, 4), (6, 2, 5), (8, 1, 2), (12, 4, 17)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (7, 3), (40, 20), (16, 100)])
def test_tokens_see_what_is_before_them(cuda_device, dtype, dim, heads, groups, queries, window, sinks):
    keys, values, table = _dealt([90, queries, 61], groups, dim, 7, dtype, 330)
    q = _rand((3, heads, queries, dim), dtype, 333)
    _check(cuda_device, q, keys, values, table, [90 - queries, 0, 61 - queries - 2], scale=dim ** -0.5, window=window,
           sinks=sinks, kernels=KERNELS if queries * heads // groups <= 16 else ["joined"])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [24, 64, 72, 80, 128])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
@pytest.mark.parametrize("heads,queries,window,sinks", [(1, 4, None, 0), (3, 4, 6, 2), (4, 4, None, 0), (1, 17, 3, 1)])
def test_states_that_a_row_does_not_see_never_show(cuda_device, dtype, dim, bad, heads, queries, window, sinks):
    """A key or value that later rows of the tile see, or that left the window of some, is not finite; column 5 alone
    of the rows that see it shows it."""
    states = 50
    q = _rand((1, heads, queries, dim), dtype, 340).to(cuda_device)
    for at in (states - 1, states - queries + 1, states - queries - 2, 1):
        for which in (0, 1):
            pools = _dealt([states], 1, dim, 16, dtype, 341)
            clean = PagedCache(*(t.to(cuda_device) for t in pools[:2]))
            page, row = oracle.place(pools[2], 16, pools[0].shape[0], 0, at)
            pools[which][page, 0, row, 5] = bad
            cache = PagedCache(*(t.to(cuda_device) for t in pools[:2]))
            more = dict(page_table=pools[2].to(cuda_device), start=torch.tensor([states - queries], device=cuda_device),
                        scale=dim ** -0.5, window=window, sinks=sinks)
            for kernel in KERNELS if heads * queries <= 16 else ["joined"]:
                got, base = (paged_attention(q, c, kernel=kernel, **more).cpu() for c in (cache, clean))
                for m in range(queries):
                    position = states - queries + m
                    sees = at <= position and (window is None or at > position - window or at < sinks)
                    if not sees:
                        assert torch.equal(got[:, :, m], base[:, :, m])
                    elif which == 1:
                        column = got[:, :, m, 5]
                        assert bool((torch.isnan(column) if bad != bad else column == bad).all())
                        other = torch.arange(dim) != 5
                        assert torch.equal(got[:, :, m][..., other], base[:, :, m][..., other])


@pytest.mark.parametrize("dim,kernel", [(64, "parts"), (128, "parts"), (64, "joined"), (128, "joined")])
def test_values_that_are_not_finite_in_one_item_of_many(cuda_device, dim, kernel):
    """A warp whose share holds several items: those beside the one that is done again keep their bits."""
    lengths = [1500] * 9 + [40] * 60
    keys, values, table = _dealt(lengths, 2, dim, 16, BF16, 350)
    q = _rand((len(lengths), 4, 2, dim), BF16, 353).to(cuda_device)
    more = dict(page_table=table.to(cuda_device), start=torch.tensor([n - 2 for n in lengths], device=cuda_device),
                scale=dim ** -0.5, kernel=kernel)
    clean = paged_attention(q, PagedCache(keys.to(cuda_device), values.to(cuda_device)), **more).cpu()
    for b, at, bad in ((3, 700, INF), (20, 39, NAN), (40, 0, -INF)):
        page, row = oracle.place(table, 16, keys.shape[0], b, at)
        values[page, 1, row, 7] = bad
    got = paged_attention(q, PagedCache(keys.to(cuda_device), values.to(cuda_device)), **more).cpu()
    shows = torch.zeros(clean.shape, dtype=torch.bool)
    shows[[3, 40], 2:, :, 7] = True
    shows[20, 2:, 1, 7] = True                                    # state 39 is the second token's own
    assert torch.equal(~torch.isfinite(got), shows)
    assert torch.equal(got[~shows], clean[~shows])
    assert bool((got[3, 2:, :, 7] == INF).all()) and bool((got[40, 2:, :, 7] == -INF).all())
