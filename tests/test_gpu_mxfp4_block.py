"""The 4-bit projections and the attention as a block uses them: the fused block
with Mxfp4Linear layers and block_attention, and the projection chain, against the
same steps one by one."""
import pytest
import torch

import blocks as toy
from lynnreal_omni_amd import fusion, kernels as k
from lynnreal_omni_amd.attention import attention, attention_packed, block_attention
from lynnreal_omni_amd.mxfp4 import Mxfp4Linear, quantize_weight
from test_gpu_fused_block import DIM, HEADS, _block, _inputs

pytestmark = pytest.mark.gpu


def _mxfp4(layer):
    """An Int8Linear's weight as MXFP4."""
    w = layer.weight_int8.t().float() * layer.weight_scale.reshape(-1, 1)
    return Mxfp4Linear.from_packed(*quantize_weight(w), layer.bias)


def _mxfp4_block(seed=1):
    block = _block(seed)
    block.attn.to_qkv, block.attn.to_out[0] = _mxfp4(block.attn.to_qkv), _mxfp4(block.attn.to_out[0])
    block.ff.net[0].proj, block.ff.net[2] = _mxfp4(block.ff.net[0].proj), _mxfp4(block.ff.net[2])
    return block


def _steps(block, x, temb, idx, rotary):
    lin = block.adaln_proj.linear
    table = k.adaln_table(temb, lin.weight, lin.bias).view(-1, 6 * DIM)

    def project(layer, value):
        return layer.forward_codes(*k.quantize_rows_mxfp4(value.reshape(-1, value.shape[-1])), value.shape[:-1])

    qkv = project(block.attn.to_qkv, k._rms_adaln(x, block.norm1, table, idx, 0, 1))
    query, key, value = (t.unflatten(-1, (HEADS, -1)) for t in qkv.chunk(3, dim=-1))
    qo, ko = k.qk_norm_rope(query, key, block.attn.norm_q.weight, block.attn.norm_k.weight, rotary,
                            block.attn.norm_q.eps)
    out = project(block.attn.to_out[0], attention(qo, ko, value).flatten(2, 3))
    x1 = k._gated_residual(x, out, table, idx, 2)
    h = project(block.ff.net[0].proj, k._rms_adaln(x1, block.norm2, table, idx, 3, 4))
    return k._gated_residual(x1, project(block.ff.net[2], k._swiglu(h)), table, idx, 5)


@torch.inference_mode()
@pytest.mark.parametrize("fused_quant", [False, True])
@pytest.mark.parametrize("tokens", [1, 96, 300])
def test_fused_block_equals_its_steps(tokens, fused_quant):
    block = _mxfp4_block()
    x, temb, idx, rotary = _inputs(tokens)
    want = _steps(block, x, temb, idx, rotary)
    fusion.enable_fusion(toy.Transformer([block]), fused_quant=fused_quant, attention=block_attention)
    got = block(x, temb, idx, rotary)
    assert got.dtype == torch.bfloat16 and got.isfinite().all() and torch.equal(got, want)


@torch.inference_mode()
def test_fused_block_in_a_graph():
    block = _mxfp4_block(3)
    x, temb, idx, rotary = _inputs(96, 2)
    fusion.enable_fusion(toy.Transformer([block]), attention=block_attention)
    others = [x, x.flip(1).contiguous(), x * 0.5]
    want = [block(v, temb, idx, rotary) for v in others]
    live, graph = x.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block(live, temb, idx, rotary)
    for v, w in zip(others, want):
        live.copy_(v)
        graph.replay()
        block(x, temb, idx, rotary)
        torch.cuda.synchronize()
        assert torch.equal(out, w)


@torch.inference_mode()
@pytest.mark.parametrize("ffn", ["gelu_tanh", "swiglu"])
def test_projection_chain(ffn):
    block = _mxfp4_block(5)
    x, temb, idx, _ = _inputs(130)
    lin = block.adaln_proj.linear
    table = k.adaln_table(temb, lin.weight, lin.bias).view(-1, 6 * DIM)
    up = block.ff.net[0].proj
    if ffn == "gelu_tanh":   # the FFN's inner width is up's
        up = Mxfp4Linear.from_packed(up.weight_codes[:512].contiguous(),
                                     _natural(up)[:512], up.bias[:512].contiguous())
    layers = fusion.ChainLayers(block.attn.to_qkv, block.attn.to_out[0], up, block.ff.net[2])
    attended = torch.randn(x.shape, generator=torch.Generator().manual_seed(7)).bfloat16().cuda()
    qkv, x1, x2 = fusion.projection_chain(x, layers, block.norm1, block.norm2, table, idx, attended, ffn=ffn)
    assert torch.equal(qkv, layers.to_qkv(k._rms_adaln(x, block.norm1, table, idx, 0, 1)))
    assert torch.equal(x1, k._gated_residual(x, layers.to_out(attended), table, idx, 2))
    h = layers.up(k._rms_adaln(x1, block.norm2, table, idx, 3, 4))
    h = k.gelu_tanh(h) if ffn == "gelu_tanh" else k._swiglu(h)
    assert torch.equal(x2, k._gated_residual(x1, layers.down(h), table, idx, 5))


def _natural(layer):
    from lynnreal_omni_amd.mxfp4_gemm import untile_scales
    return untile_scales(layer.weight_scale, layer.out_features, layer.weight_codes.shape[1] // 16)


@torch.inference_mode()
def test_prompt_then_tokens():
    """Two prompts through packed attention, then tokens one by one over the cache
    that the prompts left: the numbers of the whole sequences at once. Either side is
    off by the rounding of its weights and of its output, each at most a half step
    (2^-8) of the largest value: four half steps between them."""
    heads, kv_heads, dim, lengths, size = 8, 2, 64, [70, 133], 160
    g = torch.Generator().manual_seed(3)
    total = [n + 3 for n in lengths]
    q, kk, v = (torch.randn(sum(total), h, dim, generator=g).bfloat16().cuda() for h in (heads, kv_heads, kv_heads))
    cu = torch.tensor([0] + total, device="cuda").cumsum(0)
    whole = attention_packed(q, kk, v, cu, causal=True)
    keys, values = (torch.full((2, size, kv_heads, dim), float("nan"), device="cuda", dtype=torch.bfloat16)
                    for _ in range(2))
    first = []
    for i, n in enumerate(lengths):
        a = cu[i].item()
        keys[i, :n], values[i, :n] = kk[a:a + n], v[a:a + n]
        first.append(torch.arange(a, a + n))
    prompt = torch.cat(first).cuda()
    cu_prompt = torch.tensor([0] + lengths, device="cuda").cumsum(0)
    out = attention_packed(q[prompt], kk[prompt], v[prompt], cu_prompt, causal=True)
    bound = 2.0 ** -8 * 4 * v.abs().max().item()
    assert (out.float() - whole[prompt].float()).abs().max() <= bound
    for step in range(3):
        at = torch.tensor([cu[i].item() + n + step for i, n in enumerate(lengths)], device="cuda")
        for i, n in enumerate(lengths):
            keys[i, n + step], values[i, n + step] = kk[at[i]], v[at[i]]
        valid = torch.tensor([n + step + 1 for n in lengths], device="cuda")
        new = attention(q[at][:, None], keys, values, causal=True, key_lengths=valid)
        assert (new[:, 0].float() - whole[at].float()).abs().max() <= bound
