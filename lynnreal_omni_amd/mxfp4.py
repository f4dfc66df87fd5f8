"""4-bit projections: Mxfp4Linear, the MXFP4 counterpart of int8.Int8Linear.

Weights and activations are E2M1 codes with an E8M0 scale for each 32 values
along K (the OCP microscaling format MXFP4, scale exponent floor(log2(absmax))
- 2). Against W8A8 a weight takes 0.53 bytes instead of one and a large product
1.5 times less time (12605 x 28672 x 5376: 0.90 ms for 1.37); the price is 4-bit
precision in weights and activations.
Inference only, as the rest of the package: inputs that require a gradient are
refused.
"""
from __future__ import annotations

import torch
from torch import nn

from . import mxfp4_gemm
from .int8 import _concat_qkv
from .mxfp4_gemm import BLOCK

# Where |x| / 2^e passes from a code's magnitude to the next one's; at an odd
# border (index 0, 2, ..) a tie stays below, at an even one it goes up, so that
# ties end at the even code.
_BORDERS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)


def quantize_weight(weight: torch.Tensor):
    """MXFP4 of a float [N, K] weight in torch ops, on any device: codes uint8
    [N, 16 * ceil(K / 32)] (the even column in a byte's low half) and scale bytes
    uint8 [N, ceil(K / 32)], the values that kernels.quantize_rows_mxfp4 gives."""
    rows, width = weight.shape
    w = nn.functional.pad(weight.detach().float(), (0, -width % BLOCK)).view(rows, -1, BLOCK)
    bits = w.abs().amax(-1).view(torch.int32)
    finite = torch.isfinite(w).all(-1)
    byte = torch.where(finite, ((bits >> 23) - 2).clamp_min(0), torch.full_like(bits, 255))
    # x / 2^e in two exact steps, since 2^-e may lie outside fp32.
    half = (127 - byte.clamp_max(254)) // 2
    scaled = torch.ldexp(torch.ldexp(w, half[..., None]), (127 - byte.clamp_max(254) - half)[..., None])
    a = scaled.abs()
    code = sum(((a > t) if i % 2 == 0 else (a >= t)).to(torch.uint8) for i, t in enumerate(_BORDERS))
    code = torch.where(finite[..., None], code | (torch.signbit(w).to(torch.uint8) << 3), torch.zeros_like(code))
    pairs = code.view(rows, -1, 2)
    return pairs[..., 0] | (pairs[..., 1] << 4), byte.to(torch.uint8)


class Mxfp4Linear(nn.Module):
    """Linear layer on 4-bit weights and activations (W4A4, MXFP4).

    Buffers: `weight_codes` uint8 [N, 16 * ceil(K / 32)], `weight_scale` uint8 in
    the kernels' tile order, `bias` bf16 [N] or None; `weight` is an empty tensor
    whose dtype stands for the layer's compute dtype, as in Int8Linear.
    """

    def __init__(self, source):
        super().__init__()
        codes, scale = quantize_weight(source.weight)
        bias = None if source.bias is None else source.bias.detach().to(torch.bfloat16)
        self._install(codes, scale, bias, source.in_features, token=source.weight.new_empty(0))

    def _install(self, codes, scale, bias, in_features, token):
        self.in_features, self.out_features = in_features, codes.shape[0]
        self.register_buffer("weight_codes", codes.contiguous())
        self.register_buffer("weight_scale", mxfp4_gemm.tile_scales(scale))
        self.register_buffer("bias", bias)
        self.register_buffer("_dtype_token", token, persistent=False)

    @property
    def weight(self):
        return self._dtype_token

    @classmethod
    def from_packed(cls, weight, scale, bias=None, in_features=None):
        """Wrap MXFP4 weights as they are: codes uint8 [N, 16 * blocks], the even
        column in a byte's low half, and E8M0 bytes uint8 [N, blocks]. in_features
        defaults to 32 * blocks; codes past it must be 0."""
        if (weight.dtype != torch.uint8 or scale.dtype != torch.uint8 or weight.dim() != 2
                or scale.shape != (weight.shape[0], weight.shape[1] // 16) or weight.shape[1] % 16):
            raise ValueError("expected uint8 [out, 16 * blocks] codes and uint8 [out, blocks] scales")
        in_features = 2 * weight.shape[1] if in_features is None else int(in_features)
        if mxfp4_gemm.code_bytes(in_features) != weight.shape[1]:
            raise ValueError(f"{in_features} inputs do not make {weight.shape[1] // 16} blocks")
        if bias is not None and (bias.dtype != torch.bfloat16 or bias.shape != (weight.shape[0],)):
            raise ValueError("bias must be bfloat16 [out]")
        layer = cls.__new__(cls)
        nn.Module.__init__(layer)
        layer._install(weight, scale, bias, in_features,
                       token=torch.empty(0, device=weight.device, dtype=torch.bfloat16))
        return layer

    def forward_codes(self, codes, scales, output_shape, **epilogue):
        """Project rows that kernels.quantize_rows_mxfp4 quantized, to bf16
        [*output_shape, out_features]. `epilogue`: mxfp4_matmul's keywords."""
        y = mxfp4_gemm.mxfp4_matmul(codes, self.weight_codes, scales, self.weight_scale, self.bias, **epilogue)
        return y.view(*output_shape, self.out_features)

    def forward(self, value, **epilogue):
        """Quantize the rows of value (bf16, fp16 or fp32) and project them to bf16
        [.., out_features]. `epilogue`: mxfp4_matmul's keywords."""
        if value.shape[-1] != self.in_features:
            raise ValueError(f"the layer takes {self.in_features} features, got {value.shape[-1]}")
        buffers = self._buffers
        rows = value if value.dim() == 2 else value.reshape(-1, self.in_features)
        y = mxfp4_gemm.linear_rows(rows, buffers["weight_codes"], buffers["weight_scale"], buffers["bias"],
                                   **epilogue)
        return y if rows is value else y.view(*value.shape[:-1], self.out_features)


@torch.no_grad()
def quantize_transformer(transformer, protected_edges=1):
    """Convert the block projections of a DiT to MXFP4, the blocks and layers that
    int8.quantize_transformer converts (model/int8.py:71-104)."""
    blocks = list(transformer.transformer_blocks)
    if protected_edges < 0 or 2 * protected_edges >= len(blocks):
        raise ValueError("invalid number of protected edge blocks")
    converted = []
    for index, block in enumerate(blocks):
        attn = block.attn
        fused = _concat_qkv(attn)
        attn.to_q = attn.to_k = attn.to_v = None
        attn.fused_projections = True
        if not protected_edges <= index < len(blocks) - protected_edges:
            attn.to_qkv = fused
            continue
        attn.to_qkv = Mxfp4Linear(fused)
        attn.to_out[0] = Mxfp4Linear(attn.to_out[0])
        block.ff.net[0].proj = Mxfp4Linear(block.ff.net[0].proj)
        block.ff.net[2] = Mxfp4Linear(block.ff.net[2])
        converted.append(index)
    return {"format": "MXFP4 (W4A4)", "gemm": "gfx950 HIP scaled MFMA with fused BF16 epilogue",
            "accumulator": "FP32", "activation_scale": "E8M0 per 32 of a token",
            "weight_scale": "E8M0 per 32 of an output channel", "rounding": "nearest-even",
            "protected_edge_blocks": protected_edges, "quantized_blocks": converted,
            "quantized_linears": 4 * len(converted), "qkv_fused": True,
            "adaln_and_refiner_and_io_quantized": False}
