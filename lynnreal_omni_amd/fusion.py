"""Fused DiT blocks on gfx950: drop-in for the reference's model/fusion.py.

Two layers:

* The block surface the reference installs on a transformer:
  FusedAttention (the attention processor, model/fusion.py:12-58),
  fused_block / guarded_block (:61-116), enable_fusion (:119-142) and
  cache_time_modulation (:145-162). Same names, arguments, hook state
  (_lynnreal_*) and errors; every dense op runs on this package's kernels:
  the adaLN table (kernels.adaln_table), the fused norm/modulate(/quant)
  prologues, the W8A8 GEMMs, Q/K RMSNorm + RoPE, SwiGLU(+quant) and the
  gated residuals, with the FFN-down residual fused into the GEMM epilogue
  (bit-identical to the separate _gated_residual).
* projection_chain: the block's projections alone, as the benchmark runs
  them. It follows the op order of the fused block for everything except
  attention, which the caller supplies:

  q, s   = _rms_adaln_quant_int8(x, norm1, table, idx, 0, 1)     prologue
  qkv    = to_qkv(q, s)                                           W8A8 GEMM
  (attention, outside this chain)
  x1     = x + gate2 * to_out(quantize_rows(attn))                GEMM + gated-residual epilogue
  q2, s2 = _rms_adaln_quant_int8(x1, norm2, table, idx, 3, 4)
  FFN, either
    "gelu_tanh": q3, s3 = _gelu_quant_int8(up(q2, s2))            GEMM, then GELU + quant in one kernel
    "swiglu":    q3, s3 = _swiglu_quant_int8(up(q2, s2))          (the reference FFN)
  x2     = x1 + gate5 * down(q3, s3)                              GEMM + gated-residual epilogue

Against the reference's unfused sequence (_gated_residual after a bf16 GEMM)
the fused epilogues are bit-identical: the GEMM's bf16 value is rounded
first, then gate * y is rounded, then x + (.) is rounded, as in
model/kernels.py:152-153.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import kernels as k
from .int8 import Int8Linear
from .mxfp4 import Mxfp4Linear


@dataclass
class ChainLayers:
    """The four projections of a block, all W8A8 or all MXFP4."""
    to_qkv: Int8Linear | Mxfp4Linear
    to_out: Int8Linear | Mxfp4Linear
    up: Int8Linear | Mxfp4Linear
    down: Int8Linear | Mxfp4Linear


@torch.inference_mode()
def attention_input(hidden_states, norm1, table, indices):
    """Quantized input of the QKV projection (model/fusion.py:76)."""
    return k._rms_adaln_quant_int8(hidden_states, norm1, table, indices, 0, 1)


@torch.inference_mode()
def projection_chain(hidden_states, layers: ChainLayers, norm1, norm2, table, indices,
                     attention_output, *, ffn="gelu_tanh", attention_quantized=None):
    """Run the block's projections; returns (qkv, hidden_after_attention, hidden_out).

    hidden_states bf16 [B, T, D]; attention_output bf16 [B, T, D] (stand-in for
    the attention result); table bf16 [R, 6D]; indices int64 [T].
    attention_quantized: optional precomputed (q, s) of the QKV input (W8A8).
    """
    if isinstance(layers.to_qkv, Mxfp4Linear):
        if attention_quantized is not None:
            raise ValueError("attention_quantized belongs to W8A8 layers")
        return _mxfp4_chain(hidden_states, layers, norm1, norm2, table, indices, attention_output, ffn)
    shape = hidden_states.shape[:-1]
    q, s = attention_quantized or attention_input(hidden_states, norm1, table, indices)
    qkv = layers.to_qkv.forward_quantized(q, s, shape)
    qa, sa = k.quantize_rows(attention_output.reshape(-1, attention_output.shape[-1]))
    x1 = layers.to_out.forward_quantized(qa, sa, shape, residual=hidden_states, table=table,
                                         indices=indices, gate_slot=2)
    q2, s2 = k._rms_adaln_quant_int8(x1, norm2, table, indices, 3, 4)
    if ffn == "gelu_tanh":
        # The GELU runs in the re-quantizer (as _swiglu_quant_int8 does for
        # SwiGLU): the same bits as the GEMM's GELU epilogue followed by
        # quantize_rows, 40-60 us less per FFN at the C3 shape.
        q3, s3 = k._gelu_quant_int8(layers.up.forward_quantized(q2, s2, shape))
    elif ffn == "swiglu":
        q3, s3 = k._swiglu_quant_int8(layers.up.forward_quantized(q2, s2, shape))
    else:
        raise ValueError(f"unknown FFN activation {ffn!r}")
    x2 = layers.down.forward_quantized(q3, s3, shape, residual=x1, table=table, indices=indices,
                                       gate_slot=5)
    return qkv, x1, x2


def _mxfp4_chain(x, layers, norm1, norm2, table, indices, attention_output, ffn):
    """projection_chain of MXFP4 layers: the norms write bf16, the layers quantize
    their own inputs, GELU and the gated residuals run in the products' epilogues."""
    qkv = layers.to_qkv(k._rms_adaln(x, norm1, table, indices, 0, 1))
    x1 = layers.to_out(attention_output, residual=x, table=table, indices=indices, gate_slot=2)
    h = k._rms_adaln(x1, norm2, table, indices, 3, 4)
    if ffn == "gelu_tanh":
        h = layers.up(h, activation="gelu_tanh")
    elif ffn == "swiglu":
        h = k._swiglu(layers.up(h))
    else:
        raise ValueError(f"unknown FFN activation {ffn!r}")
    return qkv, x1, layers.down(h, residual=x1, table=table, indices=indices, gate_slot=5)


# ----------------------------------------------------------------------------
# The reference's block surface (model/fusion.py:12-162).
# ----------------------------------------------------------------------------
import os
import warnings
from types import MethodType

import torch.nn.functional as F

_TABLE_CACHE_ENTRIES = 16


def modulation_table(block, temb):
    """The block's adaLN table linear(F.silu(temb).to(bf16)).view(-1, 6 * hidden)
    (model/fusion.py:68-69) through kernels.adaln_table."""
    linear = block.adaln_proj.linear
    width = block.adaln_proj.hidden_size
    return k.adaln_table(temb, linear.weight, linear.bias).view(-1, 6 * width)


def _diffusers_attention():
    try:
        from diffusers.models.attention_dispatch import dispatch_attention_fn
    except ImportError:
        return None
    return dispatch_attention_fn


def _fp32_attention(query, key, value, attention_mask, processor):
    """Stand-in when diffusers is absent and enable_fusion was given no attention:
    scaled dot-product attention over [batch, sequence, heads, head_dim]
    computed in fp32 and returned in the query's dtype."""
    q, kk, v = (t.transpose(1, 2).float().contiguous() for t in (query, key, value))
    mask = attention_mask
    if mask is not None and mask.dtype == torch.bool and mask.dim() == 2:
        mask = mask[:, None, None, :]
    out = F.scaled_dot_product_attention(q, kk, v, attn_mask=mask)
    return out.transpose(1, 2).to(query.dtype)


class FusedAttention:
    """Attention processor with the fused Q/K RMSNorm + RoPE (model/fusion.py:12-58).

    hidden_states is either bf16 [B, S, D] or the pre-quantized tuple
    (int8 rows, row scales, shape) that fused_block hands over. Q/K/V come
    from attn.to_qkv (or to_q/to_k/to_v); Q and K go through one
    kernels.qk_norm_rope launch on their strided views. `attention` (a
    callable (query, key, value, mask, processor) -> [B, S, H, Dh]) defaults
    to diffusers' dispatch_attention_fn with the original processor's backend;
    attention.block_attention is this package's own kernel.
    """

    def __init__(self, original, ordered_qk=False, attention=None):
        self.ordered_qk = ordered_qk    # the kernel always uses the ordered reduction
        self._attention_backend = getattr(original, "_attention_backend", None)
        self._parallel_config = getattr(original, "_parallel_config", None)
        self._attention = attention

    def _attend(self, query, key, value, attention_mask):
        if self._attention is not None:
            return self._attention(query, key, value, attention_mask, self)
        dispatch = _diffusers_attention()
        if dispatch is None:
            return _fp32_attention(query, key, value, attention_mask, self)
        return dispatch(query, key, value, attn_mask=attention_mask, dropout_p=0.0, is_causal=False,
                        backend=self._attention_backend, parallel_config=self._parallel_config)

    def __call__(self, attn, hidden_states, rotary_emb=None, attention_mask=None):
        if rotary_emb is None or rotary_emb[0].ndim != 2:
            raise ValueError("fused attention requires a padless rotary layout")
        if isinstance(hidden_states, tuple):
            rows, scales, shape = hidden_states
            qkv = attn.to_qkv.forward_quantized(rows, scales, shape[:-1])
            parts = qkv.chunk(3, dim=-1)
        elif attn.fused_projections:
            parts = attn.to_qkv(hidden_states).chunk(3, dim=-1)
        else:
            parts = (attn.to_q(hidden_states), attn.to_k(hidden_states), attn.to_v(hidden_states))
        query, key, value = (t.unflatten(-1, (attn.heads, -1)) for t in parts)
        q_out, k_out = k.qk_norm_rope(query, key, attn.norm_q.weight, attn.norm_k.weight, rotary_emb,
                                      float(attn.norm_q.eps))
        output = self._attend(q_out, k_out, value, attention_mask)
        return attn.to_out[1](attn.to_out[0](output.flatten(2, 3).type_as(q_out)))


def _block_table(block, temb, adaln_table):
    """The given table, else the cached one for the current time key, else a
    new one (cached under the key, at most 16 per block, oldest out first)."""
    if adaln_table is not None:
        return adaln_table
    cache = getattr(block, "_lynnreal_adaln_cache", None)
    key = block._lynnreal_cache_key.value if cache is not None else None
    if key is not None and key in cache:
        return cache[key]
    table = modulation_table(block, temb)
    if key is not None:
        while len(cache) >= _TABLE_CACHE_ENTRIES:
            cache.pop(next(iter(cache)))
        cache[key] = table
    return table


def fused_block(self, hidden_states, temb, adaln_indices, rotary_emb, attention_mask=None,
                adaln_table=None):
    """One DiT block on the fused kernels, in the reference's op order
    (model/fusion.py:61-98):

      table -> norm1+modulate(0,1)(+quant) -> attention -> x + gate2 * attn
      [-> residual_rms_quant] -> norm2+modulate(3,4)(+quant) -> FFN up ->
      SwiGLU(+quant) -> FFN down -> x + gate5 * down
    """
    table = _block_table(self, temb, adaln_table)
    quant = self._lynnreal_fused_quant
    up, down = self.ff.net[0].proj, self.ff.net[2]
    if quant and hasattr(self.attn.to_qkv, "forward_quantized"):
        rows, scales = k._rms_adaln_quant_int8(hidden_states, self.norm1, table, adaln_indices, 0, 1)
        attention_in = (rows, scales, hidden_states.shape)
    else:
        attention_in = k._rms_adaln(hidden_states, self.norm1, table, adaln_indices, 0, 1)
    update = self.attn(attention_in, rotary_emb, attention_mask)
    if quant and hasattr(up, "forward_quantized"):
        if self._lynnreal_residual_quant:
            hidden_states, rows, scales = k.residual_rms_quant(hidden_states, update, self.norm2, table,
                                                               adaln_indices)
        else:
            hidden_states = k._gated_residual(hidden_states, update, table, adaln_indices, 2)
            rows, scales = k._rms_adaln_quant_int8(hidden_states, self.norm2, table, adaln_indices, 3, 4)
        projected = up.forward_quantized(rows, scales, hidden_states.shape[:-1])
    else:
        hidden_states = k._gated_residual(hidden_states, update, table, adaln_indices, 2)
        projected = up(k._rms_adaln(hidden_states, self.norm2, table, adaln_indices, 3, 4))
    if quant and hasattr(down, "forward_quantized") and down.gemm != "torch":
        rows, scales = k._swiglu_quant_int8(projected)
        out = down.forward_quantized(rows, scales, projected.shape[:-1], residual=hidden_states,
                                     table=table, indices=adaln_indices, gate_slot=5)
        return out
    if isinstance(down, Mxfp4Linear):
        return down(k._swiglu(projected), residual=hidden_states, table=table, indices=adaln_indices, gate_slot=5)
    if quant and hasattr(down, "forward_quantized"):
        rows, scales = k._swiglu_quant_int8(projected)
        output = down.forward_quantized(rows, scales, projected.shape[:-1])
    else:
        output = down(k._swiglu(projected))
    return k._gated_residual(hidden_states, output, table, adaln_indices, 5)


def _int8_layers(module):
    return [layer for layer in module.modules() if isinstance(layer, Int8Linear)]


def _run_native(block):
    """Give the block back its own forward and attention processor, with its
    W8A8 layers unfused."""
    block.forward = block._lynnreal_native_forward
    block.attn.set_processor(block._lynnreal_native_processor)
    for layer in _int8_layers(block):
        layer.fused_ops = False


def guarded_block(self, *args, **kwargs):
    """fused_block, or on a recoverable kernel failure (acceleration.
    optional_kernel_failure) the block's native forward and processor from
    then on, with a RuntimeWarning (model/fusion.py:101-116)."""
    from .acceleration import optional_kernel_failure
    try:
        return fused_block(self, *args, **kwargs)
    except Exception as error:
        if not optional_kernel_failure(error):
            raise
        warnings.warn(f"Optional block fusion unavailable; using native block: {error}", RuntimeWarning)
    _run_native(self)
    return self.forward(*args, **kwargs)


# Block attributes that, when not 1, mean the block strides over tokens or
# depth inside its attention/FFN math, which the fused block does not do.
_DENSE_MATH = ("h3_attention_token_stride", "h3_ffn_token_stride", "h3_depth_span")


def enable_fusion(transformer, fused_quant=False, attention=None):
    """Install fused blocks and processors on every block (model/fusion.py:119-142).

    Every block is checked before any is changed. fused_quant=True also fuses
    activation quantization into the norms and SwiGLU and marks every
    Int8Linear fused_ops; the residual + norm2 + quant kernel
    (residual_rms_quant) then runs as well (the reference limits it to Hopper;
    here it is a gfx950 kernel). Mxfp4Linear layers quantize their own inputs,
    fused_quant or not. `attention` optionally replaces the attention call of
    FusedAttention (attention.block_attention: the HIP kernel). Enabling again
    keeps the original native forward.
    """
    blocks = list(transformer.transformer_blocks)
    if any(getattr(block, name, 1) != 1 for block in blocks for name in _DENSE_MATH):
        raise ValueError("fusion requires dense attention and FFN math within each block")
    fused_quant = bool(fused_quant)
    ordered_qk = os.environ.get("LYNNREAL_LONG_KERNELS", "1") != "0"
    if fused_quant:
        owners = [transformer] if hasattr(transformer, "modules") else blocks
        for layer in (layer for owner in owners for layer in _int8_layers(owner)):
            layer.fused_ops = True
    for block in blocks:
        if not hasattr(block, "_lynnreal_native_forward"):
            block._lynnreal_native_forward = block.forward
            block._lynnreal_native_processor = block.attn.processor
        block._lynnreal_fused_quant = fused_quant
        block._lynnreal_residual_quant = fused_quant
        block.forward = MethodType(guarded_block, block)
        block.attn.set_processor(FusedAttention(block.attn.processor, ordered_qk, attention))
    return {"rmsnorm_adaln": True, "qk_norm_rope": True, "swiglu": True,
            "qk_output_allocation": "contiguous_without_copy", "residual_block": 1024,
            "gated_residual": True, "activation_quantization_fused": fused_quant,
            "residual_ffn_norm_fused": fused_quant, "qk_ordered_reduction": True,
            "int8_epilogue_fused": fused_quant, "blocks": len(blocks), "token_dropping": False}


class _TimeKey:
    """Key of the current forward's adaLN tables: the complete timestep tensor
    (shape, dtype and the bytes of its values), shared by all blocks."""

    def __init__(self):
        self.value = None

    def select(self, module, args, kwargs):
        if module.training or torch.is_grad_enabled():
            raise ValueError("cached time modulation requires frozen inference")
        times = kwargs["timestep"].detach()
        raw = times.cpu().contiguous().reshape(-1).view(torch.uint8)
        self.value = (tuple(times.shape), str(times.dtype), bytes(raw.numpy()))


def cache_time_modulation(transformer):
    """Cache each block's adaLN table per complete timestep tensor (model/fusion.py:145-162).

    A transformer pre-hook keys the current forward by the timestep tensor;
    fused_block reuses a block's table for a key it has seen (at most 16 per
    block, the oldest dropped first). Weights must not change while cached.
    """
    blocks = list(transformer.transformer_blocks)
    if not all(hasattr(block, "_lynnreal_fused_quant") for block in blocks):
        raise ValueError("time modulation caching requires fused blocks")
    key = _TimeKey()
    for block in blocks:
        block._lynnreal_adaln_cache = {}
        block._lynnreal_cache_key = key
    transformer.register_forward_pre_hook(key.select, with_kwargs=True)
    return {"kind": "exact AdaLN tables", "key": "complete input noise-time tensor",
            "maximum_entries_per_block": _TABLE_CACHE_ENTRIES, "requires_immutable_weights": True}
