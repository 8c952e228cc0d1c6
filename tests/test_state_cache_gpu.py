"""The 8-bit state cache on the GPU: what is written is exactly what the rounding rule
says, what is not written stays, and attention over it matches the float64 oracle on
the values the codes stand for."""

import pytest
import torch

from intp_preliminary_b200 import (StateCache, cached_cross_attention, check_device_status, cross_attention,
                                   shared_prefix_attention)
from oracle import cross_attention as oracle

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _device_status(cuda_device):
    yield
    check_device_status(cuda_device)


def _normal(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    rows = torch.randn(shape, generator=g)
    spread = torch.exp2(torch.randint(-6, 7, shape[:-1], generator=g).float())
    return (rows * spread[..., None]).to(dtype)


def _values(codes, exponents):
    return codes.cpu().double() * torch.exp2(exponents.cpu().double() - 127)[..., None]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 128])
@pytest.mark.parametrize("count", [1, 7, 100])
def test_write_follows_the_rounding_rule(cuda_device, dtype, dim, count):
    k, v = _normal((2, 3, count, dim), dtype, 1), _normal((2, 3, count, dim), dtype, 2)
    k[0, 0, 0] = 0
    cache = StateCache.empty(2, 3, count + 5, dim, device=cuda_device)
    start = torch.tensor([0, 5], dtype=torch.int32, device=cuda_device)
    cache.write(k.to(cuda_device), v.to(cuda_device), start=start)
    read = cache.read(count, start=start, dtype=dtype)
    for x, codes, exponents, got in ((k, cache.keys, cache.key_exponents, read[0]),
                                     (v, cache.values, cache.value_exponents, read[1])):
        want, e = oracle.quantise_rows(x)
        for b, s in enumerate((0, 5)):
            assert torch.equal(exponents[b, :, s:s + count].cpu().long() - 127, e[b])
            assert torch.equal(_values(codes, exponents)[b, :, s:s + count], want[b])
        assert torch.equal(got.cpu().double(), want)  # exact in 16 bits
        assert (exponents[0, :, count:] == 127).all() and codes[0, :, count:].float().abs().max() == 0


def test_extreme_rows(cuda_device):
    """Largest and smallest finite values, borders of the power of two, infinities and NaN."""
    rows = torch.zeros(1, 1, 12, 32, dtype=BF16)
    big, small = torch.finfo(BF16).max, 2.0 ** -133
    rows[0, 0, 0, 3], rows[0, 0, 1, :] = big, -big
    rows[0, 0, 2, 0], rows[0, 0, 3, 5] = small, torch.finfo(BF16).tiny
    rows[0, 0, 4, 1], rows[0, 0, 5, 1] = 448.0, 450.0
    rows[0, 0, 6, :] = torch.linspace(-1.75, 1.75, 32)
    rows[0, 0, 7, 0], rows[0, 0, 7, 1] = float("inf"), 3.0
    rows[0, 0, 8, 2], rows[0, 0, 8, 3] = float("nan"), -5.0
    rows[0, 0, 9, 2] = -float("inf")
    rows[0, 0, 10, :2] = torch.tensor([1.0, 2.0 ** -9])
    cache = StateCache.empty(1, 1, 12, 32, device=cuda_device)
    cache.write(rows.to(cuda_device), rows.to(cuda_device))
    want, e = oracle.quantise_rows(rows)
    assert torch.equal(cache.key_exponents.cpu().long() - 127, e)
    got = cache.read(dtype=BF16)[0].cpu().double()
    want = want.clamp(-big, big)  # the largest bf16 rounds up to 2^128: read back as the largest again
    torch.testing.assert_close(got, want, rtol=0, atol=2.0 ** -134, equal_nan=True)  # bf16's own smallest step is 2^-133
    top = torch.full((1, 1, 1, 32), 65504.0, dtype=F16, device=cuda_device)
    cache.write(top, top)
    assert torch.equal(cache.read(1, dtype=F16)[0], top)  # 65536 is past f16: its largest instead


def test_states_that_are_not_written_stay(cuda_device):
    cache = StateCache.empty(3, 2, 10, 64, device=cuda_device)
    base_k, base_v = _normal((3, 2, 10, 64), BF16, 5).to(cuda_device), _normal((3, 2, 10, 64), BF16, 6).to(cuda_device)
    cache.write(base_k, base_v)
    before = [t.clone() for t in (cache.keys.view(torch.uint8), cache.key_exponents, cache.values.view(torch.uint8),
                                  cache.value_exponents)]
    k, v = _normal((3, 2, 6, 64), BF16, 7).to(cuda_device), _normal((3, 2, 6, 64), BF16, 8).to(cuda_device)
    start = torch.tensor([-2, 7, 2], device=cuda_device)          # before, past and inside the cache
    counts = torch.tensor([6, 6, 4], dtype=torch.int32, device=cuda_device)
    cache.write(k, v, start=start, counts=counts)
    after = [cache.keys.view(torch.uint8), cache.key_exponents, cache.values.view(torch.uint8), cache.value_exponents]
    fresh = StateCache.empty(3, 2, 6, 64, device=cuda_device)
    fresh.write(k, v)
    new = [fresh.keys.view(torch.uint8), fresh.key_exponents, fresh.values.view(torch.uint8), fresh.value_exponents]
    for was, now, put in zip(before, after, new):
        want = was.clone()
        want[0, :, :4] = put[0, :, 2:]
        want[1, :, 7:] = put[1, :, :3]
        want[2, :, 2:6] = put[2, :, :4]
        assert torch.equal(now, want)
    rk, rv = cache.read(6, start=start, counts=counts)
    assert rk[0, :, :2].abs().sum() == 0 and rk[1, :, 3:].abs().sum() == 0 and rv[2, :, 4:].abs().sum() == 0
    fk, fv = fresh.read()
    assert torch.equal(rk[0, :, 2:], fk[0, :, 2:]) and torch.equal(rv[2, :, :4], fv[2, :, :4])


def _filled(batch, groups, capacity, dim, device, seed=10):
    cache = StateCache.empty(batch, groups, capacity, dim, device=device)
    cache.write(_normal((batch, groups, capacity, dim), BF16, seed).to(device) * 0.05,
                _normal((batch, groups, capacity, dim), BF16, seed + 1).to(device))
    return cache, _values(cache.keys, cache.key_exponents), _values(cache.values, cache.value_exponents)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1, 16, None), (2, 3, 3, 1, 196, 64, [196, 70]),
                                   (3, 8, 2, 2, 777, 128, [0, 777, 500]), (2, 4, 1, 9, 300, 80, [299, 17]),
                                   (1, 16, 4, 1, 5000, 128, None), (2, 2, 2, 1, 2600, 32, [2049, 2600])])
def test_cached_attention_matches_oracle(cuda_device, shape, dtype):
    batch, heads, groups, queries, states, dim, lengths = shape
    cache, k, v = _filled(batch, groups, states, dim, cuda_device)
    q = _normal((batch, heads, queries, dim), dtype, 3)
    weight = torch.exp2(cache.value_exponents.double() - 127)
    scale = 0.05
    want, _, bound = oracle.cross_attention(q, k, v, scale=scale, lengths=lengths, out_dtype=dtype, p_dtype=F16,
                                            key_weight=weight)
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=cuda_device)
    got = cached_cross_attention(q.to(cuda_device), cache, scale=scale, lengths=lens)
    off = (got.cpu().double() - want).abs()
    assert (off <= bound).all(), f"error {float((off / bound).max()):.2f} times the bound"


def test_cached_attention_with_exponents_far_apart(cuda_device):
    """Value rows from 2^-100 to 2^100 and queries past f16's range."""
    groups, states, dim = 1, 64, 32
    cache = StateCache.empty(1, groups, states, dim, device=cuda_device)
    k = torch.randn(1, 1, states, dim, generator=torch.Generator().manual_seed(1)) * 2.0 ** -30
    v = torch.randn(1, 1, states, dim, generator=torch.Generator().manual_seed(2))
    v *= torch.exp2(torch.linspace(-100, 100, states).round())[None, None, :, None]
    cache.write(k.to(BF16).to(cuda_device), v.to(BF16).to(cuda_device))
    q = (torch.randn(1, 2, 3, dim, generator=torch.Generator().manual_seed(3)) * 2.0 ** 30).to(BF16)
    kd, vd = _values(cache.keys, cache.key_exponents), _values(cache.values, cache.value_exponents)
    want, _, bound = oracle.cross_attention(q, kd, vd, scale=0.2, p_dtype=F16, out_dtype=BF16,
                                            key_weight=torch.exp2(cache.value_exponents.double() - 127))
    got = cached_cross_attention(q.to(cuda_device), cache, scale=0.2).cpu().double()
    assert ((got - want).abs() <= bound).all()


def test_padded_codes_never_show(cuda_device):
    cache, _, _ = _filled(2, 2, 300, 64, cuda_device)
    q = _normal((2, 4, 1, 64), BF16, 3).to(cuda_device)
    lengths = torch.tensor([0, 130], dtype=torch.int32, device=cuda_device)
    want = cached_cross_attention(q, cache, scale=0.1, lengths=lengths)
    for codes, exponents in ((cache.keys, cache.key_exponents), (cache.values, cache.value_exponents)):
        codes.view(torch.uint8)[0], codes.view(torch.uint8)[1, :, 130:] = 0x7f, 0xff  # NaN
        exponents[0], exponents[1, :, 130:] = 255, 0
    assert torch.equal(cached_cross_attention(q, cache, scale=0.1, lengths=lengths), want)
    assert want[0].abs().max() == 0


def test_prefix_with_cached_own_states(cuda_device):
    cache, k, v = _filled(3, 2, 90, 64, cuda_device)
    q = _normal((3, 4, 1, 64), BF16, 3)
    pk, pv = (torch.randn(2, 333, 64, generator=torch.Generator().manual_seed(s)).to(BF16) for s in (1, 2))
    lengths = [90, 0, 31]
    # the prefix's probabilities are rounded to bf16, the cache's to f16: the larger bound holds for both
    want, _, bound = oracle.cross_attention(q, k, v, scale=0.1, lengths=lengths, prefix=(pk, pv), p_dtype=BF16)
    got = shared_prefix_attention(q.to(cuda_device), pk.to(cuda_device), pv.to(cuda_device), cache, scale=0.1,
                                  lengths=torch.tensor(lengths, device=cuda_device))
    assert ((got.cpu().double() - want).abs() <= bound).all()


def test_training_then_serving(cuda_device):
    """The operators as they are used together: a step of training over an encoder's states,
    then the states go to the cache, tokens attend to it, one at a time and behind a prefix."""
    batch, heads, groups, states, dim = 2, 4, 2, 196, 64
    g = torch.Generator().manual_seed(0)
    encoded = torch.randn(batch, states, 96, generator=g).to(BF16).to(cuda_device)
    weights = [(torch.randn(96, groups * dim, generator=g) / 10).to(BF16).to(cuda_device).requires_grad_() for _ in range(2)]
    target = torch.randn(batch, heads, 12, dim, generator=g).to(BF16).to(cuda_device)

    def project():
        return [(encoded @ w).view(batch, states, groups, dim).transpose(1, 2) for w in weights]

    out = cross_attention(target, *project(), scale=dim ** -0.5)
    grads = torch.autograd.grad(out.float().square().mean(), weights)
    assert all(torch.isfinite(x).all() and x.abs().max() > 0 for x in grads)
    with torch.no_grad():
        k, v = project()
        cache = StateCache.empty(batch, groups, 256, dim, device=cuda_device)
        cache.write(k, v)
        extra = [torch.randn(batch, groups, 1, dim, generator=g).to(BF16).to(cuda_device) for _ in range(2)]
        length = torch.full((batch,), states, dtype=torch.int32, device=cuda_device)
        cache.write(*extra, start=length)
        length = length + 1
        q = target[:, :, :1]
        kd, vd = _values(cache.keys, cache.key_exponents), _values(cache.values, cache.value_exponents)
        want, _, bound = oracle.cross_attention(q, kd, vd, scale=dim ** -0.5, lengths=length.tolist(), p_dtype=F16,
                                                out_dtype=BF16,
                                                key_weight=torch.exp2(cache.value_exponents.double() - 127))
        got = cached_cross_attention(q, cache, scale=dim ** -0.5, lengths=length)
        assert ((got.cpu().double() - want).abs() <= bound).all()
        rk, rv = cache.read(dtype=BF16)
        same = cross_attention(q, rk, rv, scale=dim ** -0.5, lengths=length)
        wide, _, wide_bound = oracle.cross_attention(q, rk, rv, scale=dim ** -0.5, lengths=length.tolist())
        assert ((same.cpu().double() - wide).abs() <= wide_bound).all()
        behind = shared_prefix_attention(q, rk[0], rv[0], cache, scale=dim ** -0.5, lengths=length)
        want, _, bound = oracle.cross_attention(q, kd, vd, scale=dim ** -0.5, lengths=length.tolist(),
                                                prefix=(rk[0], rv[0]), p_dtype=BF16)
        assert ((behind.cpu().double() - want).abs() <= bound).all()


def test_captured_decode_step(cuda_device):
    """Write, then attend, in one graph: replayed with moving positions."""
    cache = StateCache.empty(2, 2, 64, 64, device=cuda_device)
    k, v = (torch.zeros(2, 2, 1, 64, dtype=BF16, device=cuda_device) for _ in range(2))
    q = torch.zeros(2, 4, 1, 64, dtype=BF16, device=cuda_device)
    start = torch.zeros(2, dtype=torch.int32, device=cuda_device)
    lengths = torch.ones(2, dtype=torch.int32, device=cuda_device)
    cached_cross_attention(q, cache, scale=0.125, lengths=lengths)
    cache.write(k, v, start=start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.write(k, v, start=start)
        out = cached_cross_attention(q, cache, scale=0.125, lengths=lengths)
    other = StateCache.empty(2, 2, 64, 64, device=cuda_device)
    for t in range(5):
        for i, x in enumerate((k, v, q)):
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(10 * t + i)))
        start.fill_(t)
        lengths.fill_(t + 1)
        graph.replay()
        other.write(k, v, start=start)
        assert torch.equal(out, cached_cross_attention(q, other, scale=0.125, lengths=lengths))


def test_refusals(cuda_device):
    cache = StateCache.empty(2, 2, 16, 64, device=cuda_device)
    x = torch.zeros(2, 2, 3, 64, dtype=BF16, device=cuda_device)
    for bad, text in [((x.float(), x.float()), "bfloat16 or float16"), ((x, x[:, :, :2]), "share shape"),
                      ((x[:, :1], x[:, :1]), "cache's"), ((x.cpu(), x.cpu()), "CUDA"), ((x, x.half()), "share a dtype")]:
        with pytest.raises(ValueError, match=text):
            cache.write(*bad)
    with pytest.raises(ValueError, match="start"):
        cache.write(x, x, start=torch.zeros(3, device=cuda_device))
    with pytest.raises(ValueError, match="no backward"):
        cache.write(x.clone().requires_grad_(), x)
    with pytest.raises(ValueError, match="dtype"):
        cache.read(dtype=torch.float32)
    with pytest.raises(ValueError, match="count"):
        cache.read(-1)
    with pytest.raises(ValueError, match="multiple of 16"):
        StateCache.empty(1, 1, 4, 40, device=cuda_device)
    with pytest.raises(ValueError, match="contiguous"):
        StateCache(cache.keys[:, :, ::2], cache.key_exponents[:, :, ::2], cache.values[:, :, ::2],
                   cache.value_exponents[:, :, ::2])
    with pytest.raises(ValueError, match="float8"):
        StateCache(x, cache.key_exponents[:, :, :3].contiguous(), x, cache.value_exponents[:, :, :3].contiguous())
    q = torch.zeros(2, 4, 1, 64, dtype=BF16, device=cuda_device)
    for bad, text in [((q[:1], cache), "batch"), ((q[:, :3], cache), "multiple of the key heads"),
                      ((q[..., :32], cache), "head_dim"), ((q.float(), cache), "bfloat16"),
                      ((q, (x, x)), "StateCache")]:
        with pytest.raises(ValueError, match=text):
            cached_cross_attention(*bad, scale=0.125)
    with pytest.raises(ValueError, match="leave v out"):
        shared_prefix_attention(q, x[0], x[0], cache, x, scale=0.125)


def test_long_cache_past_32_bit_offsets(cuda_device):
    """The last sequence's codes start past 2^31 bytes: written, read and attended to there."""
    batch, capacity, dim = 9, 2_000_000, 128
    cache = StateCache.empty(batch, 1, capacity, dim, device=cuda_device)
    k, v = _normal((batch, 1, 50, dim), BF16, 1), _normal((batch, 1, 50, dim), BF16, 2)
    start = torch.full((batch,), capacity - 50, dtype=torch.int32, device=cuda_device)
    cache.write(k.to(cuda_device) * 0.05, v.to(cuda_device), start=start)
    rk, rv = cache.read(50, start=start)
    want_k, _ = oracle.quantise_rows((k.to(cuda_device) * 0.05)[-1:])
    assert torch.equal(rk[-1:].cpu().double(), want_k)
    q = _normal((batch, 2, 1, dim), BF16, 3).to(cuda_device)
    tail = StateCache(cache.keys[:, :, -50:].contiguous(), cache.key_exponents[:, :, -50:].contiguous(),
                      cache.values[:, :, -50:].contiguous(), cache.value_exponents[:, :, -50:].contiguous())
    # zero keys score 0 and zero values add nothing: the sums over the tail and over all states
    # differ by the number of zero states alone
    part, full = (cached_cross_attention(q, c, scale=0.05).cpu().double() for c in (tail, cache))
    kd, vd = _values(tail.keys, tail.key_exponents), _values(tail.values, tail.value_exponents)
    want, lse, bound = oracle.cross_attention(q, kd, vd, scale=0.05, p_dtype=F16, out_dtype=BF16,
                                              key_weight=torch.exp2(tail.value_exponents.double() - 127))
    assert ((part - want).abs() <= bound).all()
    share = torch.sigmoid(lse - torch.log(torch.tensor(float(capacity - 50))))[..., None]
    # fp32 sums of two million equal terms over parts of 2048 keys or fewer: within 1e-4 of the count
    assert ((full - want * share).abs() <= share * bound + 2e-4 * (want * share).abs() + 1e-7).all()


def test_write_follows_strides(cuda_device):
    """(B, n, G, 2, D) projections seen as keys and values."""
    kv = _normal((2, 37, 3, 2, 64), BF16, 1).to(cuda_device)
    k, v = kv[:, :, :, 0].transpose(1, 2), kv[:, :, :, 1].transpose(1, 2)
    a, b = (StateCache.empty(2, 3, 40, 64, device=cuda_device) for _ in range(2))
    a.write(k, v)
    b.write(k.contiguous(), v.contiguous())
    assert torch.equal(a.keys.view(torch.uint8), b.keys.view(torch.uint8))
    assert torch.equal(a.values.view(torch.uint8), b.values.view(torch.uint8))
    odd = torch.empty(2, 3, 37, 65, dtype=BF16, device=cuda_device)[..., 1:].copy_(k)  # not 16-byte aligned
    a.write(odd, v)
    assert torch.equal(a.keys.view(torch.uint8), b.keys.view(torch.uint8))


def test_a_cache_without_room(cuda_device):
    """Capacity 0: writes are skipped, reads give zeros, a prefix alone is attended to."""
    cache = StateCache.empty(2, 2, 0, 64, device=cuda_device)
    k, v = (_normal((2, 2, 3, 64), BF16, s).to(cuda_device) for s in (1, 2))
    cache.write(k, v)
    cache.write(k, v, start=torch.tensor([0, 5], device=cuda_device))
    rk, rv = cache.read(3)
    assert rk.shape == rv.shape == (2, 2, 3, 64) and rk.abs().sum() == 0 and rv.abs().sum() == 0
    assert cache.read()[0].shape == (2, 2, 0, 64)
    q = _normal((2, 4, 1, 64), BF16, 3)
    pk, pv = k[0, :, :3].contiguous(), v[0, :, :3].contiguous()
    none = torch.zeros(2, 2, 0, 64)
    want, _, bound = oracle.cross_attention(q, none, none, scale=0.125, prefix=(pk, pv))
    got = shared_prefix_attention(q.to(cuda_device), pk, pv, cache, scale=0.125)
    assert ((got.cpu().double() - want).abs() <= bound).all()
    with pytest.raises(ValueError, match="at least one state"):
        cached_cross_attention(q.to(cuda_device), cache, scale=0.125)


def test_tangents_and_traces_are_refused(cuda_device):
    forward_ad = torch.autograd.forward_ad
    cache = StateCache.empty(2, 2, 16, 64, device=cuda_device)
    x = torch.zeros(2, 2, 3, 64, dtype=BF16, device=cuda_device)
    q = torch.zeros(2, 4, 1, 64, dtype=BF16, device=cuda_device)
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="forward-mode"):
            cache.write(x, forward_ad.make_dual(x, torch.ones_like(x)))
        with pytest.raises(ValueError, match="forward-mode"):
            cached_cross_attention(forward_ad.make_dual(q, torch.ones_like(q)), cache, scale=0.125)
    for fn in (lambda t: cached_cross_attention(t, cache, scale=0.125), lambda t: (cache.read(), t)[1],
               lambda t: (cache.write(x, x), t)[1]):
        with pytest.raises(ValueError, match="traced"):
            torch.jit.trace(fn, q, check_trace=False)


def test_from_the_encoder_to_a_decoder(cuda_device):
    """As a program uses them: the encoder's features, a step of training over their keys and values,
    then the cache, a new state, and tokens over it and behind a prefix."""
    from intp_preliminary_b200.share_vit import ShareViTHalf6d3r

    batch, heads, groups, dim, capacity = 2, 4, 2, 64, 200
    g = torch.Generator().manual_seed(7)
    encoder = ShareViTHalf6d3r(precision="bf16").init_weights(seed=1, look_grid_std=0.02).to(cuda_device)
    images = torch.randn(batch, 3, 224, 224, generator=g).to(cuda_device)
    to_k, to_v = (torch.nn.Linear(192, groups * dim, bias=False).to(cuda_device, BF16) for _ in range(2))
    with torch.no_grad():
        states = encoder.forward_features(images).bfloat16()

    def keys_and_values(states):
        return [w(states).view(batch, -1, groups, dim).transpose(1, 2) for w in (to_k, to_v)]

    k, v = keys_and_values(states)
    q = torch.randn(batch, heads, 9, dim, generator=g).to(BF16).to(cuda_device).requires_grad_()
    grad = torch.randn(batch, heads, 9, dim, generator=g).to(BF16).to(cuda_device)
    scale = dim ** -0.5
    out = cross_attention(q, k, v, scale=scale)
    want, _, bound = oracle.cross_attention(q, k, v, scale=scale)
    assert ((out.detach().cpu().double() - want).abs() <= bound).all()
    wants, bounds = oracle.cross_attention_gradients(q, k, v, grad, scale=scale)
    for got, want, bound in zip(torch.autograd.grad(out, (q, k, v), grad, retain_graph=True), wants, bounds):
        assert ((got.cpu().double() - want).abs() <= bound).all()
    out.backward(grad)
    assert all(torch.isfinite(w.weight.grad).all() and w.weight.grad.abs().max() > 0 for w in (to_k, to_v))

    cache = StateCache.empty(batch, groups, capacity, dim, device=cuda_device)
    with pytest.raises(ValueError, match="no backward"):
        cache.write(k, v)
    filled = torch.full((batch,), k.shape[2], dtype=torch.int32, device=cuda_device)
    with torch.no_grad():
        k, v = keys_and_values(states)
        cache.write(k, v)
        cache.write(k[:, :, :1], v[:, :, 1:2], start=filled)
        token = q[:, :, :1]
        lengths = filled + 1
        kd, vd = _values(cache.keys, cache.key_exponents), _values(cache.values, cache.value_exponents)
        got = cached_cross_attention(token, cache, scale=scale, lengths=lengths)
        want, _, bound = oracle.cross_attention(token, kd, vd, scale=scale, lengths=lengths.tolist(), p_dtype=F16,
                                                out_dtype=BF16,
                                                key_weight=torch.exp2(cache.value_exponents.double() - 127))
        assert ((got.cpu().double() - want).abs() <= bound).all()
        got = shared_prefix_attention(token, k[0], v[0], cache, scale=scale, lengths=lengths)
        want, _, bound = oracle.cross_attention(token, kd, vd, scale=scale, lengths=lengths.tolist(),
                                                prefix=(k[0], v[0]), p_dtype=BF16)
        assert ((got.cpu().double() - want).abs() <= bound).all()
