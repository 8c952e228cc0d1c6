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
