"""MXFP4 on the CPU: the weight quantizer, the scale order and what the entry points refuse."""
import numpy as np
import pytest
import torch

import mxfp4_ref as ref
from lynnreal_omni_amd import _lib, kernels, mxfp4, mxfp4_gemm


def rows(n, k, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(n, k, generator=g) * torch.exp2(torch.randint(-20, 20, (n, 1), generator=g).float())


def hard_rows():
    """Ties, borders, zeros, tiny and huge blocks."""
    x = np.zeros((8, 96), np.float32)
    x[0, :] = np.linspace(-7.9, 7.9, 96)
    x[1, :32] = np.arange(-16, 16) * 0.25          # every tie of a block whose scale is 1
    x[1, 32] = 4.0
    x[2, :] = -0.0
    x[3, :32] = 2.0 ** -126 * np.arange(32) / 4    # scale clamped at 2^-127
    x[4, :32] = 2.0 ** -140
    x[5, :] = 3.0e38
    x[6, 40] = np.nan
    x[6, 70] = -np.inf
    x[7, :] = 2.0 ** -120 * np.linspace(-1, 1, 96)
    return torch.from_numpy(x)


@pytest.mark.parametrize("w", [rows(5, 64), rows(3, 31), rows(70, 33), rows(2, 300), hard_rows()])
def test_quantize_weight_is_the_definition(w):
    codes, scale = mxfp4.quantize_weight(w)
    code, byte, _ = ref.quantize(w.numpy())
    assert np.array_equal(scale.numpy(), byte)
    assert np.array_equal(codes.numpy(), ref.pack(code))


@pytest.mark.parametrize("n,blocks", [(1, 1), (64, 8), (65, 9), (130, 3), (17, 21)])
def test_scale_tiles(n, blocks):
    g = torch.Generator().manual_seed(n)
    scale = torch.randint(0, 256, (n, blocks), dtype=torch.uint8, generator=g)
    tiles = mxfp4_gemm.tile_scales(scale)
    assert tuple(tiles.shape) == mxfp4_gemm.scale_shape(n, blocks * 32)
    assert torch.equal(mxfp4_gemm.untile_scales(tiles, n, blocks), scale)
    for r in range(0, n, 13):
        for b in range(blocks):
            at = (16 * (b % 4) + r % 16) * 8 + 2 * (r // 16 % 4) + b // 4 % 2
            assert tiles[r // 64, b // 8, at] == scale[r, b]


def test_layer_from_packed_checks():
    codes, scale = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    layer = mxfp4.Mxfp4Linear.from_packed(codes, scale, in_features=40)
    assert (layer.in_features, layer.out_features) == (40, 4)
    for bad in [lambda: mxfp4.Mxfp4Linear.from_packed(codes.to(torch.int8), scale),
                lambda: mxfp4.Mxfp4Linear.from_packed(codes, scale[:, :1]),
                lambda: mxfp4.Mxfp4Linear.from_packed(codes[:, :20], scale),
                lambda: mxfp4.Mxfp4Linear.from_packed(codes, scale, in_features=32),
                lambda: mxfp4.Mxfp4Linear.from_packed(codes, scale, torch.zeros(4)),
                lambda: layer(torch.zeros(2, 64, dtype=torch.bfloat16))]:
        with pytest.raises(ValueError):
            bad()


def test_refusals():
    with pytest.raises(RuntimeError, match="not supported"):
        kernels.quantize_rows_mxfp4(torch.zeros(2, 8, dtype=torch.float64))
    with pytest.raises(ValueError):
        kernels.quantize_rows_mxfp4(torch.zeros(8, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        kernels.quantize_rows_mxfp4(torch.zeros(2, 8, dtype=torch.bfloat16))       # no GPU tensor
    codes, scales = torch.zeros(3, 32, dtype=torch.uint8), torch.zeros(1, 1, 512, dtype=torch.uint8)
    with pytest.raises(ValueError):
        kernels.dequantize_rows_mxfp4(codes, scales, 32)                           # one block, codes of two
    with pytest.raises(ValueError):
        kernels.dequantize_rows_mxfp4(codes, scales[..., :256], 64)
    for bad in [dict(activation="relu"), dict(gate_slot=1), dict(activation="gelu_tanh", residual=torch.zeros(3, 3))]:
        with pytest.raises(ValueError):
            mxfp4_gemm._epilogue(3, 3, **{**dict(activation=None, residual=None, table=None, indices=None,
                                                 gate_slot=None), **bad})
    for args in [(codes[:, :20], codes, scales, scales), (codes, codes, scales[0], scales),
                 (codes.to(torch.int8), codes, scales, scales), (codes, codes[:, :16].contiguous(), scales, scales),
                 (codes.t().contiguous().t(), codes, scales, scales), (codes, codes, scales, scales)]:
        with pytest.raises(ValueError):
            mxfp4_gemm.mxfp4_matmul(*args)


def test_entry_points_refuse_without_a_gpu():
    lib = _lib.load()
    p = 4096
    gemm = lambda **kw: lib.lr_mxfp4_gemm(*{**dict(a=p, sa=p, b=p, sb=p, m=4, n=8, k=64, bias=None, out=p, epi=0,  # noqa: E731
                                                   res=None, table=None, rows=0, width=0, idx=None, seq=0, slot=0,
                                                   stream=None), **kw}.values())
    for bad in [dict(a=None), dict(a=p + 8), dict(sb=p + 4), dict(epi=3), dict(epi=2), dict(m=-1), dict(k=0),
                dict(k=(1 << 23) + 1), dict(epi=2, res=p, table=p, idx=p, rows=1, width=16, seq=4, slot=2)]:
        assert gemm(**bad) == _lib.LR_EINVAL, bad
    assert gemm(m=0) == _lib.LR_OK
    for bad in [(p, 7, 2, 32, p, p, None), (p, 0, -1, 32, p, p, None), (None, 0, 2, 32, p, p, None),
                (p, 0, 2, 32, p + 4, p, None), (p + 1, 0, 2, 32, p, p, None)]:
        assert lib.lr_quantize_rows_mxfp4(*bad) == _lib.LR_EINVAL, bad
    assert lib.lr_quantize_rows_mxfp4(None, 0, 0, 32, None, None, None) == _lib.LR_OK
    assert lib.lr_dequantize_rows_mxfp4(p, p, 0, 2, 32, p + 2, None) == _lib.LR_EINVAL
    # codes of 3 rows of 64 columns: 96 bytes, kept as 256, and one tile of scales
    linear = lambda **kw: lib.lr_mxfp4_linear(*{**dict(x=p, dtype=0, m=3, n=8, k=64, s=p, sb=768, b=p, bs=p, bias=None,  # noqa: E731
                                                       out=p, epi=0, res=None, table=None, rows=0, width=0, idx=None,
                                                       seq=0, slot=0, stream=None), **kw}.values())
    for bad in [dict(sb=767), dict(s=None), dict(s=p + 8), dict(k=0), dict(dtype=9), dict(x=None)]:
        assert linear(**bad) == _lib.LR_EINVAL, bad
    assert linear(m=0, s=None, sb=0) == _lib.LR_OK
    assert mxfp4_gemm._scratch(3, 64) == 768


def test_quantize_transformer():
    from test_host import _fake_transformer
    t = _fake_transformer()
    b1 = t.transformer_blocks[1]
    q, k, v = b1.attn.to_q, b1.attn.to_k, b1.attn.to_v
    report = mxfp4.quantize_transformer(t, protected_edges=1)
    assert report["quantized_blocks"] == [1, 2] and report["quantized_linears"] == 8
    for i, b in enumerate(t.transformer_blocks):
        assert b.attn.to_q is None and b.attn.fused_projections
        for layer in (b.attn.to_qkv, b.attn.to_out[0], b.ff.net[0].proj, b.ff.net[2]):
            assert isinstance(layer, mxfp4.Mxfp4Linear) == (i in (1, 2))
    codes, scale = mxfp4.quantize_weight(torch.cat([q.weight, k.weight, v.weight]))
    assert torch.equal(b1.attn.to_qkv.weight_codes, codes)
    assert torch.equal(b1.attn.to_qkv.weight_scale, mxfp4_gemm.tile_scales(scale))
    with pytest.raises(ValueError, match="unconverted"):
        mxfp4.quantize_transformer(t)
    with pytest.raises(ValueError, match="protected"):
        mxfp4.quantize_transformer(_fake_transformer(blocks=2), protected_edges=1)
    again = mxfp4.Mxfp4Linear.from_packed(codes, scale, b1.attn.to_qkv.bias, in_features=q.in_features)
    again.load_state_dict(b1.attn.to_qkv.state_dict())
