"""GPU parity of low-rank adapters with their formula in 64 bits.

Tolerance, eps being the half step of the type: the inner products are fp32 sums of k
products (2^-23 of the sum of magnitudes each); each then becomes two numbers of the type, off by
eps^2 of it, or, below the type's normal numbers, by 2^-25 of the row's largest; the outer
products sum 2 * rank of those, in fp32 too; base is added in fp32 (2^-23) and the output
is rounded once, by eps of it.
"""
import pytest
import torch
from torch import nn

from lynnreal_omni_amd import adapters as L
from lynnreal_omni_amd.int8 import Int8Linear
from lynnreal_omni_amd.mxfp4 import Mxfp4Linear

pytestmark = pytest.mark.gpu


def make(count, rank, n, k, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    down = (torch.randn(count, rank, k, generator=g) * k ** -0.5).to(dtype).cuda()
    up = (torch.randn(count, n, rank, generator=g) * rank ** -0.5).to(dtype).cuda()
    return down, up, (torch.rand(count, generator=g) + 0.5).cuda()


def rows(tokens, n, k, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(tokens, k, generator=g).to(dtype).cuda(), torch.randn(tokens, n, generator=g).to(dtype).cuda()


def check(got, x, base, indices, down, up, scale):
    dtype = x.dtype
    eps, rank, k = torch.finfo(dtype).eps / 2, down.shape[1], x.shape[1]
    got, x, base, down, up, scale = (t.double().cpu() for t in (got, x, base, down, up, scale))
    indices = indices.cpu()
    for a in range(-1, down.shape[0]):
        at = (indices == a).nonzero()[:, 0] if a >= 0 else ((indices < 0) | (indices >= down.shape[0])).nonzero()[:, 0]
        if a < 0:
            assert torch.equal(got[at], base[at])
            continue
        if not len(at):
            continue
        inner = scale[a] * (x[at] @ down[a].t())
        size = scale[a] * (x[at].abs() @ down[a].abs().t())
        want = base[at] + inner @ up[a].t()
        outer = inner.abs() @ up[a].abs().t()
        top = inner.abs().amax(1, keepdim=True) * up[a].abs().sum(1)
        bound = ((k + 4) * 2.0 ** -23 * size @ up[a].abs().t() + (eps ** 2 + (2 * rank + 4) * 2.0 ** -23) * outer
                 + 2.0 ** -25 * top + 2.0 ** -23 * (base[at].abs() + outer))
        bound = bound + eps * (want.abs() + bound) + torch.finfo(dtype).smallest_normal * eps
        assert ((got[at] - want).abs() <= bound).all()


def run(indices, count, rank, n, k, dtype, seed=0):
    weights = make(count, rank, n, k, dtype, seed)
    x, base = rows(len(indices), n, k, dtype, seed + 1)
    indices = torch.tensor(indices, dtype=torch.int32).cuda()
    plan = L.AdapterPlan(indices, count)
    layer = L.LowRankAdapters(*weights)
    got = layer(x, base, plan)
    check(got, x, base, indices, *weights)
    again = base.clone()
    assert layer(x, again, plan, out=again) is again and torch.equal(again, got)
    return got


def spread(tokens, count, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(-1, count, (tokens,), generator=g)).tolist()


CASES = [
    # indices, adapters, rank, n, k
    ([0], 1, 1, 1, 1), ([2], 5, 16, 5376, 640), ([-1], 3, 8, 40, 24), ([0, 1, 2, 1, -1, 7, 0], 3, 4, 17, 33),
    (spread(64, 33), 33, 32, 1000, 520), ([1] * 64, 2, 8, 256, 64), ([0] * 65, 1, 16, 128, 128), ([0] * 31 + [1] * 33, 2, 64, 384, 2000),
    (spread(300, 2), 2, 128, 1416, 1000), ([3] * 200 + [-1] * 50 + [0] * 130, 4, 33, 520, 712), (spread(1000, 300), 300, 8, 72, 48),
    (spread(130, 1000), 1000, 1, 8, 8), ([4] * 700, 7, 100, 2056, 5000), (spread(40, 9), 9, 128, 129, 127),
    ([-1] * 300, 2, 16, 256, 128), ([0] * 1300 + [1] * 700, 2, 64, 1024, 4096),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("indices,count,rank,n,k", CASES)
def test_cases(indices, count, rank, n, k, dtype):
    run(indices, count, rank, n, k, dtype, rank + n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes,rank,k", [
    ((6000, -100, 6100), 128, 8008), ((9000, 1, 65), 100, 12000), ((-1000, 4000, 64, 4036), 128, 12120)])
def test_pairs_of_tiles(sizes, rank, k, dtype):
    """Many tokens of few adapters at a high rank: pairs of tiles, odd numbers of them, adapters of a
    tile or less, and tokens of none (negative sizes)."""
    indices, at = [], 0
    for n in sizes:
        indices += [at if n > 0 else -1] * abs(n)
        at += n > 0
    order = torch.randperm(len(indices), generator=torch.Generator().manual_seed(rank)).tolist()
    run([indices[i] for i in order], at, rank, 40, k, dtype, rank)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes,rank,k", [
    ((3000, 1090), 128, 8008), ((64, 1, 1500, 63, 65, 128, 129, -7, 1900), 70, 12000), ((2049, -2051), 127, 8000),
    ((900,), 128, 33000)])
def test_pairs_of_fewer_tiles(sizes, rank, k, dtype):
    """Around the fewest tokens and steps that are taken in pairs of tiles: shares of k, and adapters of one
    tile, of a tile and a token, and of none."""
    indices, at = [], 0
    for n in sizes:
        indices += [at if n > 0 else -1] * abs(n)
        at += n > 0
    order = torch.randperm(len(indices), generator=torch.Generator().manual_seed(rank)).tolist()
    run([indices[i] for i in order], at, rank, 40, k, dtype, rank)


@pytest.mark.parametrize("seed", range(6))
def test_plans(seed):
    """A plan lists every token once, in tiles of one adapter, in order."""
    g = torch.Generator().manual_seed(seed)
    tokens = [1, 63, 1000, 5000, 12605, 257][seed]
    count = [1, 1000, 7, 40, 3, 1000][seed]
    for dtype in (torch.int32, torch.int64):
        indices = torch.randint(-2, count + 2, (tokens,), generator=g).to(dtype)
        if dtype == torch.int64:
            indices[0] = 2 ** 33     # 0 if it wrapped
        plan = L.AdapterPlan(indices.cuda(), count)
        for _ in range(2):
            order, tiles = plan.order.cpu().long(), plan.tiles.cpu()
            kinds = torch.where((indices < 0) | (indices >= count), count, indices)
            assert torch.equal(order, torch.sort(kinds, stable=True).indices)
            at = 0
            for a, first, n, _ in tiles.tolist():
                if n:
                    assert first == at and 0 < n <= 64
                    assert (kinds[order[first:first + n]] == (a if a >= 0 else count)).all()
                    at += n
            assert at == tokens
            indices = indices.flip(0)
            plan.update(indices.cuda())


def test_views():
    """Slices of wider rows, an expanded base, inputs of more dimensions, odd ones that are copied."""
    weights = make(3, 8, 72, 40, torch.bfloat16, 1)
    layer = L.LowRankAdapters(*weights)
    x, base = rows(12, 72, 40, torch.bfloat16, 2)
    indices = torch.tensor(spread(12, 3)).cuda()
    plan = L.AdapterPlan(indices.view(3, 4), 3)
    want = layer(x, base, plan)
    check(want, x, base, indices, *weights)
    wide = torch.zeros(12, 200, dtype=torch.bfloat16, device="cuda")
    for first in (0, 8, 3):
        a, b = wide[:, first:first + 40].copy_(x), wide[:, 96 + first:168 + first].copy_(base)
        assert torch.equal(layer(a, b, plan), want)
    assert torch.equal(layer(x.view(3, 4, 40), base.view(3, 4, 72), plan), want.view(3, 4, 72))
    columns = x.t().contiguous().t(), base.t().contiguous().t()
    assert torch.equal(layer(*columns, plan), want)
    one = base[:1].expand(12, -1)
    assert torch.equal(layer(x, one, plan), layer(x, one.contiguous(), plan))
    same = x[:1].expand(12, -1)
    assert torch.equal(layer(same, base, plan), layer(same.contiguous(), base, plan))


@pytest.mark.parametrize("k", [1, 40, 33, 4969])
@pytest.mark.parametrize("tokens", [1, 70, 300])
def test_copied_rows(tokens, k):
    """Rows of x at any place, and ones that overlap."""
    n = 24
    weights = make(3, 20, n, k, torch.float16, 1)
    layer = L.LowRankAdapters(*weights)
    g = torch.Generator().manual_seed(k)
    flat = torch.randn(tokens * (k + 8) + 16, generator=g).half().cuda()
    base = torch.randn(tokens, n, generator=g).half().cuda()
    indices = torch.tensor(spread(tokens, 3)).cuda()
    plan = L.AdapterPlan(indices, 3)
    for first, step in ((0, k), (3, k), (8, k + 5), (1, 1), (0, 8), (5, 0)):
        x = flat[first:].as_strided((tokens, k), (step, 1), first)
        got = layer(x, base, plan)
        check(got, x, base, indices, *weights)
        assert torch.equal(layer(x.clone(memory_format=torch.contiguous_format), base, plan), got)


def test_rows_do_not_depend_on_the_batch():
    """A token gives the same bits in whatever tile it lies, and an infinity or NaN of another
    token stays there."""
    weights = make(4, 16, 264, 512, torch.bfloat16, 3)
    layer = L.LowRankAdapters(*weights)
    x, base = rows(200, 264, 512, torch.bfloat16, 4)
    indices = torch.tensor(spread(200, 4)).cuda()
    want = layer(x, base, L.AdapterPlan(indices, 4))
    turn = torch.randperm(200).cuda()
    got = layer(x[turn], base[turn], L.AdapterPlan(indices[turn], 4))
    assert torch.equal(got, want[turn])
    x[7, 3], x[100] = float("inf"), float("nan")
    got = layer(x, base, L.AdapterPlan(indices, 4))
    clean = torch.ones(200, dtype=torch.bool, device="cuda")
    clean[7] = clean[100] = False
    assert torch.equal(got[clean], want[clean])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_ranges(dtype):
    """Inner products far outside the type's range, whose products with up are not."""
    tokens, rank, n, k = 40, 16, 64, 256
    g = torch.Generator().manual_seed(1)
    for power in (-12, 10):
        x = (torch.randn(tokens, k, generator=g) * 2.0 ** power).to(dtype).cuda()
        down = (torch.randn(1, rank, k, generator=g) * 2.0 ** (power / 2)).to(dtype).cuda()
        up = (torch.randn(1, n, rank, generator=g) * 2.0 ** -power).to(dtype).cuda()
        scale = torch.tensor([2.0 ** (-power / 2)], device="cuda")
        base = torch.randn(tokens, n, generator=g).to(dtype).cuda()
        indices = torch.zeros(tokens, dtype=torch.int32, device="cuda")
        got = L.LowRankAdapters(down, up, scale)(x, base, L.AdapterPlan(indices, 1))
        assert torch.isfinite(got).all()
        check(got, x, base, indices, down, up, scale)


def test_infinite_inner_products():
    """x of infinity gives what its products give: infinities by up's sign, NaN where up is 0."""
    x = torch.zeros(1, 8, dtype=torch.bfloat16, device="cuda")
    x[0, 0] = float("inf")
    down = torch.ones(1, 1, 8, dtype=torch.bfloat16, device="cuda")
    up = torch.tensor([[[1.0], [-2.0], [0.0]]], dtype=torch.bfloat16, device="cuda")
    got = L.LowRankAdapters(down, up)(x, torch.zeros(1, 3, dtype=torch.bfloat16, device="cuda"),
                                      L.AdapterPlan(torch.zeros(1, dtype=torch.int32, device="cuda"), 1))
    assert got[0, 0] == float("inf") and got[0, 1] == float("-inf") and got[0, 2].isnan()


def test_inputs_past_32_bits():
    """Rows of x past 2^32 bytes, in an order that mixes both ends in a tile."""
    k, n, tokens = 8, 16, 70
    step = 2 ** 26 + 8
    big = torch.zeros((tokens - 1) * step + k, dtype=torch.bfloat16, device="cuda")
    x = big.as_strided((tokens, k), (step, 1))
    small, base = rows(tokens, n, k, torch.bfloat16, 5)
    x.copy_(small)
    weights = make(2, 4, n, k, torch.bfloat16, 6)
    indices = torch.tensor(spread(tokens, 2)).cuda()
    layer, plan = L.LowRankAdapters(*weights), L.AdapterPlan(indices, 2)
    got = layer(x, base, plan)
    assert torch.equal(got, layer(small, base, plan))


def test_pairs_of_tiles_past_32_bits():
    k, n, tokens, step = 8064, 16, 12605, 180000
    big = torch.empty((tokens - 1) * step + k, dtype=torch.bfloat16, device="cuda")
    x = big.as_strided((tokens, k), (step, 1))
    small, base = rows(tokens, n, k, torch.bfloat16, 5)
    x.copy_(small)
    weights = make(2, 128, n, k, torch.bfloat16, 6)
    indices = torch.tensor(spread(tokens, 2)).cuda()
    layer, plan = L.LowRankAdapters(*weights), L.AdapterPlan(indices, 2)
    assert torch.equal(layer(x, base, plan), layer(small, base, plan))


@pytest.mark.parametrize("kind", ["int8", "mxfp4", "linear"])
def test_adapted_layers(kind):
    g = torch.Generator().manual_seed(2)
    source = nn.Linear(256, 392)
    with torch.no_grad():
        source.weight.copy_(torch.randn(392, 256, generator=g) / 16)
    source = source.bfloat16().cuda()
    layer = {"int8": lambda: Int8Linear(source, "hip"), "mxfp4": lambda: Mxfp4Linear(source), "linear": lambda: source}[kind]()
    if kind == "int8":
        layer.fused_ops = True
    weights = make(3, 16, 392, 256, torch.bfloat16, 7)
    x, _ = rows(90, 392, 256, torch.bfloat16, 8)
    indices = torch.tensor(spread(90, 3)).cuda()
    with torch.no_grad():
        base = layer(x)
        requests = L.Requests()
        adapted = L.AdaptedLinear(layer, L.LowRankAdapters(*weights), requests)
        assert torch.equal(adapted(x.view(2, 45, 256)), base.view(2, 45, 392))
        requests.plan = L.AdapterPlan(indices.view(2, 45), 3)
        got = adapted(x.view(2, 45, 256))
    check(got.view(90, 392), x, base, indices, *weights)


def test_graph_whose_requests_change():
    weights = make(5, 16, 520, 512, torch.bfloat16, 9)
    layer = L.LowRankAdapters(*weights)
    x, base = rows(100, 520, 512, torch.bfloat16, 10)
    indices = torch.tensor(spread(100, 5), dtype=torch.int32).cuda()
    plan = L.AdapterPlan(indices, 5)
    layer(x, base, plan)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.update(indices)
        got = layer(x, base, plan)
    for step in range(4):
        indices.copy_(torch.tensor(spread(100, 5, step + 1), dtype=torch.int32))
        x.mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, layer(x, base, L.AdapterPlan(indices, 5)))
        check(got, x, base, indices, *weights)


def test_other_stream():
    weights = make(5, 16, 520, 512, torch.bfloat16, 9)
    layer = L.LowRankAdapters(*weights)
    x, base = rows(100, 520, 512, torch.bfloat16, 10)
    indices = torch.tensor(spread(100, 5), dtype=torch.int32).cuda()
    want = layer(x, base, L.AdapterPlan(indices, 5))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer(x, base, L.AdapterPlan(indices, 5))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_no_tokens():
    weights = make(2, 4, 16, 8, torch.bfloat16, 0)
    empty = torch.zeros(0, dtype=torch.int32, device="cuda")
    got = L.LowRankAdapters(*weights)(torch.zeros(0, 8, dtype=torch.bfloat16, device="cuda"),
                                      torch.zeros(0, 16, dtype=torch.bfloat16, device="cuda"), L.AdapterPlan(empty, 2))
    assert got.shape == (0, 16)


@pytest.mark.parametrize("name", ["down", "up", "scale", "order", "tiles"])
def test_out_is_apart_from_adapters_and_plan(name):
    layer = L.LowRankAdapters(*make(2, 4, 16, 8, torch.bfloat16, 0))
    x, base = rows(60, 16, 8, torch.bfloat16, 1)
    plan = L.AdapterPlan(torch.zeros(60, dtype=torch.int32, device="cuda"), 2)
    owner = plan if hasattr(plan, name) else layer
    want, read = layer(x, base, plan), getattr(owner, name)
    memory = torch.zeros(8192, dtype=torch.uint8, device="cuda")
    setattr(owner, name, memory[:read.nbytes].view(read.dtype).view(read.shape).copy_(read))
    with pytest.raises(ValueError, match="out must"):
        layer(x, base, plan, out=memory[:base.nbytes].view(torch.bfloat16).view(60, 16))
    out = memory[-base.nbytes:].view(torch.bfloat16).view(60, 16)
    assert torch.equal(layer(x, base, plan, out=out), want)
