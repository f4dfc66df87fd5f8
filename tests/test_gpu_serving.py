"""Adapters, a shared prefix, the keys' weights and eviction as requests are served with
them: blocks of a transformer with adapters beside their projections, and a batch of
requests, token by token, over a prefix that they share and caches of their own with a
budget."""
import pytest
import torch
from torch import nn

import blocks as toy
from lynnreal_omni_amd import adapters as L
from lynnreal_omni_amd import cache, fusion, kernels as k
from lynnreal_omni_amd.attention import attention, attention_shared_prefix, block_attention
from lynnreal_omni_amd.int8 import Int8Linear
from lynnreal_omni_amd.mxfp4 import Mxfp4Linear
from test_gpu_attention import check as check_attention, formula, mask
from test_gpu_adapters import check as check_adapters, make as some_adapters, spread
from test_gpu_cache import check as check_weights, check_evicted
from test_gpu_fused_block import DIM, HEADS, _block, _inputs
from test_gpu_mxfp4_block import _mxfp4_block

pytestmark = pytest.mark.gpu

NAMES = ("attn.to_qkv", "attn.to_out.0", "ff.net.0.proj", "ff.net.2")


@torch.inference_mode()
@pytest.mark.parametrize("fused_quant", [False, True])
@pytest.mark.parametrize("kind", ["int8", "mxfp4"])
def test_blocks_with_adapters(kind, fused_quant):
    """A fused block whose four projections have adapters gives the bits of its steps one by
    one, and those of the block alone without a plan."""
    make = _block if kind == "int8" else _mxfp4_block
    plain, block = make(4), make(4)
    tokens, count = 130, 5
    x, temb, idx, rotary = _inputs(tokens)
    transformer = toy.Transformer([block])
    beside = {}
    for i, name in enumerate(NAMES):
        layer = block.get_submodule(name)
        down, up, scale = some_adapters(count, 8 + 4 * i, layer.out_features, layer.in_features, torch.bfloat16, i)
        beside["transformer_blocks.0." + name] = L.LowRankAdapters(down, up, scale)
    requests = L.adapt_transformer(transformer, beside)
    fusion.enable_fusion(transformer, fused_quant=fused_quant, attention=block_attention)
    fusion.enable_fusion(toy.Transformer([plain]), attention=block_attention)
    none = block(x, temb, idx, rotary)
    # The layers quantize their inputs themselves, as those of a block without fused_quant do.
    if not fused_quant:
        assert torch.equal(none, plain(x, temb, idx, rotary))
    requests.plan = L.AdapterPlan(torch.tensor(spread(tokens, count)).cuda(), count)
    got = block(x, temb, idx, rotary)

    def project(name, value):
        layer = block.get_submodule(name)
        return beside["transformer_blocks.0." + name](value, layer.layer(value), requests.plan)

    lin = block.adaln_proj.linear
    table = k.adaln_table(temb, lin.weight, lin.bias).view(-1, 6 * DIM)
    qkv = project(NAMES[0], k._rms_adaln(x, block.norm1, table, idx, 0, 1))
    query, key, value = (t.unflatten(-1, (HEADS, -1)) for t in qkv.chunk(3, dim=-1))
    qo, ko = k.qk_norm_rope(query, key, block.attn.norm_q.weight, block.attn.norm_k.weight, rotary,
                            block.attn.norm_q.eps)
    x1 = k._gated_residual(x, project(NAMES[1], attention(qo, ko, value).flatten(2, 3)), table, idx, 2)
    h = project(NAMES[2], k._rms_adaln(x1, block.norm2, table, idx, 3, 4))
    want = k._gated_residual(x1, project(NAMES[3], k._swiglu(h)), table, idx, 5)
    assert got.isfinite().all() and torch.equal(got, want) and not torch.equal(got, none)
    requests.plan = None
    assert torch.equal(block(x, temb, idx, rotary), none)


class Layer(nn.Module):
    """One layer of a model that is served: Q/K/V, attention, output projection, with adapters."""

    def __init__(self, hidden, heads, kv_heads, dim, count, requests, seed):
        super().__init__()
        g = torch.Generator().manual_seed(seed)
        qkv, out = nn.Linear(hidden, (heads + 2 * kv_heads) * dim), nn.Linear(heads * dim, hidden)
        with torch.no_grad():
            for linear in (qkv, out):
                linear.weight.copy_(torch.randn(linear.weight.shape, generator=g) * linear.in_features ** -0.5)
                linear.bias.copy_(0.02 * torch.randn(linear.bias.shape, generator=g))
        qkv, out = Int8Linear(qkv.bfloat16().cuda(), "hip"), Mxfp4Linear(out.bfloat16().cuda())
        qkv.fused_ops = True
        self.weights = [some_adapters(count, 16, n.out_features, n.in_features, torch.bfloat16, seed + i)
                        for i, n in enumerate((qkv, out))]
        self.qkv, self.out = (L.AdaptedLinear(n, L.LowRankAdapters(*w), requests)
                              for n, w in zip((qkv, out), self.weights))


@torch.inference_mode()
def test_requests_over_a_shared_prefix():
    hidden, heads, kv_heads, dim, batch, count = 256, 8, 2, 64, 4, 3
    shared, prompt, size, budget, recent, steps = 333, 20, 40, 24, 6, 45
    picks = torch.tensor([2, -1, 0, 2]).cuda()
    requests = L.Requests()
    layer = Layer(hidden, heads, kv_heads, dim, count, requests, 1)
    g = torch.Generator().manual_seed(2)
    prefix_k, prefix_v = (torch.randn(shared, kv_heads, dim, generator=g).bfloat16().cuda() for _ in range(2))
    keys, values, spare_keys, spare_values = (
        torch.full((batch, size, kv_heads, dim), float("nan"), device="cuda", dtype=torch.bfloat16) for _ in range(4))
    weights, spare_weights = (torch.zeros(batch, kv_heads, size, device="cuda") for _ in range(2))
    lengths = torch.zeros(batch, dtype=torch.int32, device="cuda")
    rows = torch.arange(batch, device="cuda")[:, None]
    filled, evictions = 0, 0
    for step in range(steps):
        new = prompt if step == 0 else 1
        if filled + new > size:
            # Full caches go down to the budget, into the spare ones, which they change places with.
            result = cache.evict(keys, values, weights, lengths, budget, recent=recent,
                                 out=(spare_keys, spare_values, spare_weights))
            check_evicted(result, keys, values, weights, [filled] * batch, budget, recent, clear=False)
            (spare_keys, spare_values, spare_weights), (keys, values, weights, lengths, _) = (keys, values, weights), result
            filled, evictions = budget, evictions + 1
        x = torch.randn(batch, new, hidden, generator=g).bfloat16().cuda()
        requests.plan = L.AdapterPlan(picks[:, None].expand(batch, new), count)
        fused = layer.qkv(x)
        check_adapters(fused.view(batch * new, -1), x.view(batch * new, -1), layer.qkv.layer(x).view(batch * new, -1),
                       picks.repeat_interleave(new), *layer.weights[0])
        query, key, value = (t.unflatten(-1, (-1, dim)) for t in
                             fused.split([heads * dim, kv_heads * dim, kv_heads * dim], -1))
        places = lengths[:, None] + torch.arange(new, device="cuda")
        keys[rows, places], values[rows, places] = key, value
        lengths = lengths + new
        filled += new
        attended, lse = attention_shared_prefix(query, prefix_k, prefix_v, keys, values, causal=True,
                                                key_lengths=lengths, return_lse=True)
        seen = torch.cat([torch.ones(new, shared, dtype=torch.bool), mask(new, filled, True)], 1)
        for i in range(batch):
            both = (torch.cat([a, b[i, :filled]]) for a, b in ((prefix_k, keys), (prefix_v, values)))
            check_attention(attended[i], *formula(query[i], *both, dim ** -0.5, seen))
        before = weights.clone()
        weights = cache.accumulate_weights(weights, query, keys, lse, causal=True, key_lengths=lengths, out=weights)
        check_weights(weights, before, query, keys, lse, [filled] * batch, True, dim ** -0.5)
        x = attended.flatten(2)
        out = layer.out(x)
        check_adapters(out.view(batch * new, -1), x.view(batch * new, -1), layer.out.layer(x).view(batch * new, -1),
                       picks.repeat_interleave(new), *layer.weights[1])
    assert evictions == 2


@torch.inference_mode()
def test_two_streams_at_once():
    """Two batches on streams of their own, whose calls run beside each other: each has what it has alone."""
    heads, kv_heads, dim, batch = 8, 2, 64, 3

    def make(seed):
        g = torch.Generator().manual_seed(seed)
        q, k, v = (torch.randn(batch, n, h, dim, generator=g).bfloat16().cuda()
                   for n, h in ((1, heads), (40000, kv_heads), (40000, kv_heads)))
        prefix = torch.randn(5000, kv_heads, dim, generator=g).bfloat16().cuda()
        weights = torch.rand(batch, kv_heads, 40000, generator=g).cuda()
        x = torch.randn(700, 512, generator=g).bfloat16().cuda()
        base = torch.randn(700, 1024, generator=g).bfloat16().cuda()
        adapters = L.LowRankAdapters(*some_adapters(5, 32, 1024, 512, torch.bfloat16, seed))
        return q, k, v, prefix, weights, x, base, adapters, torch.randint(-1, 5, (700,), generator=g).cuda()

    def run(q, k, v, prefix, weights, x, base, adapters, picks):
        out, lse = attention_shared_prefix(q, prefix, prefix, k, v, return_lse=True)
        weights = cache.accumulate_weights(weights, q, k, lse)
        return out, lse, weights, *cache.evict(k, v, weights, None, 9000, recent=9), adapters(x, base, L.AdapterPlan(picks, 5))

    given = [make(seed) for seed in (1, 2)]
    want = [run(*args) for args in given]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in given]
    got = [[] for _ in given]
    for _ in range(6):
        for stream, args, results in zip(streams, given, got):
            with torch.cuda.stream(stream):
                results.append(run(*args))
    torch.cuda.synchronize()
    for results, alone in zip(got, want):
        for result in results:
            assert all(torch.equal(a, b) for a, b in zip(result, alone))
