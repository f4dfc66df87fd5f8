"""GPU parity of the keys' attention weights with the formula in 64 bits, and of eviction
with a statement of its rule, bit for bit.

A weight's tolerance: the fp32 score (D + 2 additions and products, 2^-23 of scale * sum
|q k| each), the rounding of scale * log2(e), of the exponent and of lse * log2(e) (2^-23 of |s| +
|lse| in all, twice that is allowed) and the exponential (2^-22) move each row's share by a
factor; the rows are added in fp32 (2^-24 per row), as is the weight before (2^-24).
"""
import pytest
import torch

from lynnreal_omni_amd import cache
from lynnreal_omni_amd.attention import attention_shared_prefix
from test_gpu_attention import mask

pytestmark = pytest.mark.gpu


def make(batch, new, size, heads, kv_heads, dim, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(batch, new, heads, dim, generator=g) * 1.5).to(dtype).cuda()
    k = torch.randn(batch, size, kv_heads, dim, generator=g).to(dtype).cuda()
    w = torch.rand(batch, kv_heads, size, generator=g).cuda()
    return w, q, k


def check(got, w, q, k, lse, lengths, causal, scale):
    batch, new, heads, _ = q.shape
    kv_heads, size = w.shape[1:]
    got, w, q, k, lse = (t.double().cpu() for t in (got, w, q, k, lse))
    for i in range(batch):
        n = size if lengths is None else min(max(lengths[i], 0), size)
        seen = mask(new, n, causal)
        keys = k[i, :n].transpose(0, 1).repeat_interleave(heads // kv_heads, 0)
        s = q[i].transpose(0, 1) @ keys.transpose(1, 2) * scale
        sums = lse[i].t()[..., None]
        p = torch.where(seen, torch.exp(s - sums), 0.0)
        absolute = q[i].abs().transpose(0, 1) @ keys.abs().transpose(1, 2) * scale
        off = p * ((q.shape[-1] + 2) * 2.0 ** -23 * absolute + 2.0 ** -22 * (s.abs() + sums.abs()) + 2.0 ** -22)
        # p is 0 where a row sees nothing, whose lse is -inf.
        off = torch.where(p == 0, 0.0, off)
        add = lambda t: t.reshape(kv_heads, heads // kv_heads * new, n).sum(1)  # noqa: E731
        want = w[i, :, :n] + add(p)
        bound = 1.01 * (add(off) + new * heads // kv_heads * 2.0 ** -24 * add(p) + 2.0 ** -23 * want)
        assert ((got[i, :, :n] - want).abs() <= bound).all()
        assert torch.equal(got[i, :, n:], w[i, :, n:])


def sums_of(q, k, lengths, causal, scale=None):
    """lse as the attention leaves it."""
    none = k.new_empty((0, *k.shape[2:]))
    given = None if lengths is None else torch.tensor(lengths, device="cuda")
    return attention_shared_prefix(q, none, none, k, k, causal=causal, scale=scale, key_lengths=given, return_lse=True)[1]


CASES = [
    # batch, new, size, heads, kv_heads, dim, lengths
    (1, 1, 1, 1, 1, 32, None), (2, 1, 5, 2, 1, 64, [5, 0]), (8, 1, 1200, 40, 8, 128, [1200, 317, 1, 1024, 878, 0, 129, 128]),
    (3, 4, 300, 16, 2, 64, [4, 300, 1]), (1, 70, 70, 3, 3, 128, None), (2, 130, 513, 4, 2, 32, [513, 130]),
    (1, 700, 900, 10, 2, 128, [801]), (2, 257, 257, 7, 1, 64, [257, 100]), (70, 1, 64, 5, 5, 32, [i for i in range(70)]),
    (1, 2000, 128, 2, 2, 64, None), (1, 64, 129, 1, 1, 128, None), (1, 1500, 1500, 56, 8, 128, None),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("batch,new,size,heads,kv_heads,dim,lengths", CASES)
def test_weights(batch, new, size, heads, kv_heads, dim, lengths, causal, dtype):
    w, q, k = make(batch, new, size, heads, kv_heads, dim, dtype, new + size)
    lse = sums_of(q, k, lengths, causal)
    given = None if lengths is None else torch.tensor(lengths, device="cuda")
    got = cache.accumulate_weights(w, q, k, lse, causal=causal, key_lengths=given)
    check(got, w, q, k, lse, lengths, causal, dim ** -0.5)
    again = w.clone()
    assert cache.accumulate_weights(again, q, k, lse, causal=causal, key_lengths=given, out=again) is again
    assert torch.equal(again, got)
    # Every row's shares add up to one where it sees a key.
    if not causal:
        total = (got.double() - w.double()).sum((1, 2))
        alive = torch.tensor([1.0 if n else 0.0 for n in (lengths or [size] * batch)], device="cuda").double()
        assert ((total - alive * new * heads).abs() <= 1e-4 * new * heads).all()


@pytest.mark.parametrize("new", [1, 200])
def test_behind_a_prefix(new):
    """The sums of a shared prefix and the own keys: the own keys get the rest of it."""
    w, q, k = make(2, new, 260, 4, 2, 64, torch.bfloat16, new)
    prefix = k[0, :100].flip(0).contiguous()
    lengths = torch.tensor([260, new], device="cuda")
    _, lse = attention_shared_prefix(q, prefix, prefix, k, k, causal=True, key_lengths=lengths, return_lse=True)
    got = cache.accumulate_weights(w, q, k, lse, causal=True, key_lengths=lengths)
    check(got, w, q, k, lse, [260, new], True, 64 ** -0.5)


@pytest.mark.parametrize("new", [1, 150])
def test_hidden_keys_get_nothing(new):
    """NaN and infinities in keys that no token sees, and rows that see none (lse -inf)."""
    w, q, k = make(3, new, 400, 4, 2, 64, torch.float16, new)
    lengths = [new + 30, new // 2, 0]
    lse = sums_of(q, k, lengths, True)
    want = cache.accumulate_weights(w, q, k, lse, causal=True, key_lengths=torch.tensor(lengths, device="cuda"))
    check(want, w, q, k, lse, lengths, True, 64 ** -0.5)
    for i, n in enumerate(lengths):
        k[i, n:] = float("nan") if i else float("inf")
    got = cache.accumulate_weights(w, q, k, lse, causal=True, key_lengths=torch.tensor(lengths, device="cuda"))
    assert torch.equal(got, want)


@pytest.mark.parametrize("new", [1, 150])
@pytest.mark.parametrize("scale", [1e-3, 2.0])
def test_scales(scale, new):
    w, q, k = make(2, new, 300, 4, 2, 64, torch.bfloat16, new)
    lse = sums_of(q, k, None, False, scale)
    check(cache.accumulate_weights(w, q, k, lse, scale=scale), w, q, k, lse, None, False, scale)


@pytest.mark.parametrize("new", [1, 90])
def test_weights_of_views(new):
    g = torch.Generator().manual_seed(new)
    dim = 64
    q = torch.randn(2, new, 8 * dim, generator=g).bfloat16().cuda()[..., 2 * dim:6 * dim].unflatten(-1, (4, dim))
    outside = torch.randn(2, 2, 200, dim, generator=g).bfloat16().cuda().transpose(1, 2)
    w = torch.rand(2, 200, 2, generator=g).cuda().transpose(1, 2)
    lse = sums_of(q, outside, None, False)
    want = cache.accumulate_weights(w.contiguous(), q.contiguous(), outside.contiguous(), lse)
    assert torch.equal(cache.accumulate_weights(w, q, outside, lse), want)
    far = lse.transpose(1, 2).contiguous().transpose(1, 2)
    heads_first = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(cache.accumulate_weights(w, heads_first, outside, far), want)
    odd = [torch.zeros(*t.shape[:-1], dim + 1, dtype=t.dtype, device="cuda")[..., 1:].copy_(t) for t in (q, outside)]
    assert torch.equal(cache.accumulate_weights(w, *odd, lse), want)


@pytest.mark.parametrize("batch", [512, 513])
@pytest.mark.parametrize("new", [1, 4])
def test_weights_of_many_caches(batch, new):
    w, q, k = make(batch, new, 150, 4, 2, 32, torch.bfloat16, batch)
    lengths = [(37 * i) % 152 for i in range(batch)]
    lse = sums_of(q, k, lengths, True)
    got = cache.accumulate_weights(w, q, k, lse, causal=True, key_lengths=torch.tensor(lengths, device="cuda"))
    check(got, w, q, k, lse, lengths, True, 32 ** -0.5)


@pytest.mark.parametrize("new,heads", [(1, 32), (1, 33), (16, 2), (32, 1), (33, 1)])
def test_weights_around_32_rows(new, heads):
    w, q, k = make(2, new, 1500, heads, 1, 64, torch.float16, new + heads)
    lengths = [1500, 700]
    lse = sums_of(q, k, lengths, True)
    got = cache.accumulate_weights(w, q, k, lse, causal=True, key_lengths=torch.tensor(lengths, device="cuda"))
    check(got, w, q, k, lse, lengths, True, 64 ** -0.5)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("batch,new,size,heads,kv_heads,dim", [
    (64, 400, 300, 4, 1, 32), (65, 400, 300, 4, 1, 32), (7, 310, 1100, 5, 1, 64), (3, 1600, 700, 2, 2, 128),
    (2, 1473, 256, 1, 1, 64)])
def test_weights_dealt_out(batch, new, size, heads, kv_heads, dim, causal):
    """Many rows over few keys, whose work is dealt out over the GPU: empty and short caches between
    long ones, and more tokens than keys."""
    w, q, k = make(batch, new, size, heads, kv_heads, dim, torch.bfloat16, batch)
    lengths = [(0, size, 1, 257, size - 1, 128, 0, 77)[i % 8] for i in range(batch)]
    lengths = [min(n, size) for n in lengths]
    lse = sums_of(q, k, lengths, causal)
    given = torch.tensor(lengths, device="cuda")
    got = cache.accumulate_weights(w, q, k, lse, causal=causal, key_lengths=given)
    check(got, w, q, k, lse, lengths, causal, dim ** -0.5)
    assert torch.equal(cache.accumulate_weights(w, q, k, lse, causal=causal, key_lengths=given, out=w), got)


@pytest.mark.parametrize("new", [20, 40, 2000])
def test_weights_of_infinite_sums(new):
    """A token whose lse is -infinity, as where all of its scores are: infinity for the keys that it
    sees, as the formula's exp(s + inf), and nothing for the others."""
    size = new + 200
    w, q, k = make(1, new, size, 1, 1, 64, torch.float16, new)
    lse = sums_of(q, k, None, True)
    lse[:, 5] = float("inf")   # exp(s - inf) = 0
    want = cache.accumulate_weights(w, q, k, lse, causal=True)
    lse[:, 5] = -float("inf")
    got = cache.accumulate_weights(w, q, k, lse, causal=True)
    assert (got[..., :206] == float("inf")).all()
    assert torch.equal(got[..., 206:], want[..., 206:]) and want.isfinite().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("at", [0, 5, -1])
@pytest.mark.parametrize("new,size,heads", [(20, 220, 1), (40, 240, 1), (40, 240, 3), (2000, 2200, 1), (700, 700, 3)])
def test_weights_of_nan_sums(new, size, heads, at, dtype):
    """A token whose lse is NaN, as the attention leaves it for a query of NaN: NaN for the keys
    that it sees, and nothing for the others, which keep the bits of a run where it counts for nothing."""
    w, q, k = make(1, new, size, heads, 1, 64, dtype, new + heads)
    at %= new
    lse = sums_of(q, k, None, True)
    lse[:, at] = float("inf")   # exp(s - inf) = 0
    want = cache.accumulate_weights(w, q, k, lse, causal=True)
    assert want.isfinite().all()
    seen = size - new + at + 1
    lse[:, at, heads // 2] = float("nan")
    got = cache.accumulate_weights(w, q, k, lse, causal=True)
    assert got[..., :seen].isnan().all() and torch.equal(got[..., seen:], want[..., seen:])
    q[:, at] = float("nan")
    lse = sums_of(q, k, None, True)
    assert lse[:, at].isnan().all()
    got = cache.accumulate_weights(w, q, k, lse, causal=True)
    assert got[..., :seen].isnan().all() and torch.equal(got[..., seen:], want[..., seen:])


@pytest.mark.parametrize("new", [1, 100])
def test_weights_of_far_keys(new):
    """Keys past 2^31 elements of the first."""
    size, step = 300, 2 ** 23 - 64
    k = torch.empty(size * step, dtype=torch.bfloat16, device="cuda").as_strided((1, size, 1, 64), (size * step, step, 64, 1))
    assert (size - 1) * step > 2 ** 31
    w, q, near = make(1, new, size, 3, 1, 64, torch.bfloat16, new)
    k.copy_(near)
    lse = sums_of(q, near, None, False)
    assert torch.equal(cache.accumulate_weights(w, q, k, lse), cache.accumulate_weights(w, q, near, lse))


def kept_of(weights, length, budget, recent):
    """The rule, for one head: the places that stay."""
    if length <= budget:
        return list(range(length))
    old = length - min(recent, length)
    values = weights[:old].tolist()
    rank = lambda i: (values[i] != values[i], -values[i] if values[i] == values[i] else 0.0, i)  # noqa: E731
    return sorted(sorted(range(old), key=rank)[:budget - (length - old)]) + list(range(old, length))


def check_evicted(result, key, value, weights, lengths, budget, recent, clear=True):
    keys, values, new_weights, new_lengths, kept = (t.cpu() for t in result)
    key, value, weights = key.cpu(), value.cpu(), weights.cpu()
    for i in range(key.shape[0]):
        n = key.shape[1] if lengths is None else min(max(lengths[i], 0), key.shape[1])
        end = min(n, budget)
        assert new_lengths[i] == end
        for h in range(key.shape[2]):
            want = kept_of(weights[i, h], n, budget, recent)
            assert kept[i, h].tolist() == want + [-1] * (budget - end)
            assert torch.equal(keys[i, :end, h].view(torch.int16), key[i, want, h].view(torch.int16))
            assert torch.equal(values[i, :end, h].view(torch.int16), value[i, want, h].view(torch.int16))
            assert torch.equal(new_weights[i, h, :end].view(torch.int32), weights[i, h, want].view(torch.int32))
            assert (new_weights[i, h, end:] == 0).all()
            if clear:
                assert (keys[i, end:, h] == 0).all() and (values[i, end:, h] == 0).all()


def caches(batch, size, heads, dim, dtype=torch.bfloat16, seed=0, levels=None):
    g = torch.Generator().manual_seed(seed + size)
    key, value = (torch.randn(batch, size, heads, dim, generator=g).to(dtype).cuda() for _ in range(2))
    weights = torch.exp(3 * torch.randn(batch, heads, size, generator=g))
    if levels:
        weights = torch.randint(levels, (batch, heads, size), generator=g) / 8.0
    return key, value, weights.cuda()


@pytest.mark.parametrize("batch,size,heads,dim,lengths,budget,recent", [
    (1, 1, 1, 8, None, 1, 0), (2, 5, 2, 32, [5, 3], 4, 0), (1, 5, 1, 64, None, 9, 3), (3, 100, 3, 128, [100, 0, 64], 64, 16),
    (2, 1100, 8, 128, [1100, 1030], 1024, 128), (1, 3000, 2, 64, [2999], 1, 0), (1, 3000, 2, 64, [2999], 1, 1),
    (2, 2049, 1, 40, None, 2048, 2048), (1, 20000, 2, 8, [19999], 777, 100), (70, 65, 1, 16, list(range(70)), 30, 30),
    (1, 100000, 1, 8, None, 50000, 10), (2, 17000, 2, 16, [17000, 16385], 16384, 1)])
@pytest.mark.parametrize("levels", [None, 4, 1])
def test_evict(batch, size, heads, dim, lengths, budget, recent, levels):
    """levels: few different weights, so that the border falls among equal ones."""
    key, value, weights = caches(batch, size, heads, dim, levels=levels)
    given = None if lengths is None else torch.tensor(lengths, device="cuda")
    result = cache.evict(key, value, weights, given, budget, recent=recent)
    assert result[0].shape == (batch, budget, heads, dim) and result[2].shape == (batch, heads, budget)
    check_evicted(result, key, value, weights, lengths, budget, recent)


def test_unusual_weights():
    """Negative ones, zeros of both signs, infinities, subnormal numbers and NaN."""
    inf, nan = float("inf"), float("nan")
    row = [0.0, -0.0, 1e-42, -1e-42, inf, -inf, nan, -nan, 1.0, -1.0, 3e38, -3e38, nan, 0.0, -0.0, 2.0]
    key, value, _ = caches(1, 16, 2, 16, torch.float16)
    weights = torch.tensor([[row, row[::-1]]], device="cuda")
    for budget in range(1, 17):
        for recent in (0, min(2, budget)):
            result = cache.evict(key, value, weights, None, budget, recent=recent)
            check_evicted(result, key, value, weights, None, budget, recent)


def test_lengths_and_unused_places():
    key, value, weights = caches(3, 50, 2, 16)
    weights[:, :, 40:] = float("inf")
    for dtype in (torch.int32, torch.int64):
        result = cache.evict(key, value, weights, torch.tensor([40, -7, 2 ** 31 - 1], device="cuda").to(dtype), 20, recent=3)
        check_evicted(result, key, value, weights, [40, 0, 50], 20, 3)


def test_into_given_caches():
    """Larger caches with their heads outside and keys and values in one buffer: rows behind the
    last stay as they were."""
    key, value, weights = caches(3, 90, 2, 32)
    lengths = [90, 10, 0]
    both = torch.full((3, 2, 60, 2, 32), 7.0, dtype=torch.bfloat16, device="cuda")
    out = (both[:, :, :, 0].transpose(1, 2), both[:, :, :, 1].transpose(1, 2), torch.full((3, 2, 60), 7.0, device="cuda"))
    result = cache.evict(key, value, weights, torch.tensor(lengths, device="cuda"), 40, recent=5, out=out)
    assert all(a is b for a, b in zip(result, out))
    check_evicted(result, key, value, weights, lengths, 40, 5, clear=False)
    for t in result[:2]:
        for i, n in enumerate((40, 10, 0)):
            assert (t[i, n:] == 7).all()


def test_views_are_evicted():
    key, value, weights = caches(2, 70, 2, 32)
    views = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (key, value)]
    odd = [torch.zeros(*t.shape[:-1], 33, dtype=t.dtype, device="cuda")[..., 1:].copy_(t) for t in (key, value)]
    expanded = weights[:1].expand(2, -1, -1)
    for k, v in ((key, value), views, odd):
        check_evicted(cache.evict(k, v, expanded, None, 33, recent=2), key, value, expanded, None, 33, 2)


def test_far_caches():
    """Rows past 2^31 elements of a cache."""
    size = 2 ** 31 // 2048 + 100
    key = torch.zeros(1, size, 2, 1024, dtype=torch.bfloat16, device="cuda")
    key[0, -1] = 1.0
    key[0, 5] = 2.0
    weights = torch.zeros(1, 2, size, device="cuda")
    weights[..., 5] = weights[..., size - 1] = 1.0
    keys, values, _, _, kept = cache.evict(key, key, weights, None, 2)
    assert kept.tolist() == [[[5, size - 1]] * 2]
    assert (keys[0, 0] == 2).all() and (keys[0, 1] == 1).all() and torch.equal(keys, values)


@pytest.mark.parametrize("new", [1, 500])
def test_graph(new):
    """The attention, the weights and an eviction in one graph, replayed as the caches change."""
    w, q, k = make(3, new, 300, 8, 2, 64, torch.bfloat16, 3)
    v = k.flip(1).contiguous()
    prefix = k[0, :100].contiguous()
    lengths = torch.full((3,), 300, device="cuda", dtype=torch.int32)

    def step():
        out, lse = attention_shared_prefix(q, prefix, prefix, k, v, causal=True, key_lengths=lengths, return_lse=True)
        weights = cache.accumulate_weights(w, q, k, lse, causal=True, key_lengths=lengths)
        return out, lse, weights, *cache.evict(k, v, weights, lengths, 100, recent=10)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        lengths.copy_(torch.tensor([300 - i, 101 + i, 7 * i], dtype=torch.int32))
        q.mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        check_evicted(got[3:], k, v, got[2], lengths.tolist(), 100, 10)
