"""Softmax attention on gfx950 MFMA: the step of a block between the Q/K norm +
RoPE (kernels.qk_norm_rope) and the output projection.

  attention         a batch of sequences of one length, or a few new tokens over
                    padded caches with their own numbers of valid keys
  attention_packed  sequences of different lengths behind each other
  attention_shared_prefix  a batch whose sequences all see a common prefix of keys
                    before their own caches, which is read for all of them at once
  block_attention   the same as fusion.FusedAttention calls it, for
                    fusion.enable_fusion(..., attention=block_attention)

bf16 or fp16; head_dim 32, 64 or 128; query heads may share key heads. Scores,
maxima, sums and accumulators are fp32. The softmax weights are rounded to the
inputs' type for the product with v; where `attention` has at most 32 rows (tokens
x query heads of a key head) they keep the rest of that rounding as a second number,
so that the output's own rounding is all that remains. attention_packed rounds them
once whatever its number of tokens, so that a sequence gives the same bits whatever
lies around it: the same token may differ by the weights' rounding between the two.
In attention_shared_prefix a sequence's rows over its own keys keep the rest where they are
at most 32, and the rows of all sequences together over the prefix where they are at most 32, or where
the keys are so few that a sequence's rows take them all in one kernel. With more rows the weights
are rounded once: a token's last bits depend on how many others share its prefix (bf16
outputs are off by 2.3e-3 of their size then, 1.66e-3 else).

Tensors whose last dimension is dense, whose other strides are multiples of 8 elements
(those between tokens below 2^23) and whose memory is 16-byte aligned are read as
they are: slices of a fused projection, caches with the heads outside, expanded
batches. Any other is copied as a whole in every call: lay a cache out so. Keys that a token may not see are left
out whatever their scores; the values of a sequence have to be finite (a weight
of zero times an infinity is NaN, as in the formula). Inference only: inputs that
require a gradient are refused.
"""
from __future__ import annotations

import functools
import struct
from array import array

import torch

from . import _lib

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_HEAD_DIMS = (32, 64, 128)
_MAX_SCALE = torch.finfo(torch.float32).max
_DENSE, _PACKED, _LENGTHS = range(3)


def _dense(stride, shape):
    """Whether the kernel reads a tensor of these strides: a dense head dimension, rows
    a multiple of 16 bytes apart."""
    return stride[-1] == 1 and stride[-3] < 1 << 23 and all(not st % 8 or n == 1 for st, n in zip(stride[:-1], shape))


def _rows(t):
    """t where the kernel can read it, or a copy."""
    if not t.data_ptr() % 16 and _dense(t.stride(), t.shape):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


@functools.lru_cache(maxsize=4096)
def _strides(q, k, v, q_shape, k_shape, copied):
    """The nine strides that lr_attention takes, of tensors with the strides q, k, v;
    None where one has to be copied first."""
    nine = array("q")
    for stride, shape in ((q, q_shape), (k, k_shape), (v, k_shape)):
        if not copied and not _dense(stride, shape):
            return None
        # A dimension of one element may have any stride; it is not used.
        s = [st if n > 1 else 0 for st, n in zip(stride, shape)]
        nine.extend((s[-3], s[-2], s[0] if len(s) == 4 else 0))
    return nine


@functools.lru_cache(maxsize=4096)
def _splits(sequences, q_rows, k_rows, kind, heads, kv_heads):
    return int(_lib.load().lr_attention_splits(sequences, q_rows, k_rows, kind, heads, kv_heads))


@functools.lru_cache(maxsize=64)
def _scale_bits(scale):
    if not 0 < scale <= _MAX_SCALE:
        raise ValueError(f"scale must be positive and finite in fp32, got {scale}")
    return struct.unpack("i", struct.pack("f", scale))[0]


def _check_tensors(query, key, value, dims):
    names = "[batch, tokens, heads, head_dim]" if dims == 4 else "[tokens, heads, head_dim]"
    if query.dim() != dims or key.dim() != dims or value.shape != key.shape:
        raise ValueError(f"query, key and value must be {names}, key and value of one shape")
    if query.dtype != key.dtype or query.dtype != value.dtype:
        raise ValueError(f"query, key and value must have one dtype, got {query.dtype}, {key.dtype}, {value.dtype}")
    if query.dtype not in _DTYPES:
        raise RuntimeError(f"dtype {query.dtype} is not supported by the HIP attention (bfloat16 or float16)")
    heads, dim = query.shape[-2:]
    if key.shape[-1] != dim or key.shape[-2] == 0 or heads % key.shape[-2]:
        raise ValueError(f"{heads} query heads of {dim} do not share {key.shape[-2]} key heads of {key.shape[-1]}")
    if dim not in _HEAD_DIMS:
        raise RuntimeError(f"head_dim {dim} is not supported by the HIP attention (32, 64 or 128)")
    if torch.is_grad_enabled() and (query.requires_grad or key.requires_grad or value.requires_grad):
        raise RuntimeError("gradients are not supported by the HIP attention: call it under torch.no_grad()")


def _check(query, key, value, dims):
    _check_tensors(query, key, value, dims)
    _lib.check_device(query)


def _launch(query, key, value, cu_q, cu_k, lengths, causal, scale, sequences, q_rows, k_rows, out=None):
    strides = None
    if not (query.data_ptr() | key.data_ptr() | value.data_ptr()) & 15:
        strides = _strides(query.stride(), key.stride(), value.stride(), query.shape, key.shape, False)
    if strides is None:
        query, key, value = _rows(query), _rows(key), _rows(value)
        strides = _strides(query.stride(), key.stride(), value.stride(), query.shape, key.shape, True)
    if out is None:
        out = query.new_empty(query.shape)
    heads, dim = query.shape[-2:]
    kv_heads = key.shape[-2]
    packed = cu_q is not None
    kind = _PACKED if packed else (_DENSE if lengths is None else _LENGTHS)
    splits = _splits(sequences, q_rows, k_rows, kind, heads, kv_heads)
    ws, nbytes = None, 0
    if splits > 1:
        nbytes = splits * (sequences if kind == _DENSE else 1) * q_rows * heads * (dim + 2) * 4
        ws = _lib.workspace(query, nbytes)   # held until the launch
    _lib.launch(query, "lr_attention", query.data_ptr(), key.data_ptr(), value.data_ptr(), out.data_ptr(),
                _DTYPES[query.dtype], sequences, q_rows, k_rows, heads, kv_heads, dim, strides.buffer_info()[0],
                _lib.ptr(cu_q), _lib.ptr(cu_k), _lib.ptr(lengths), int(bool(causal)),
                _scale_bits(float(dim ** -0.5 if scale is None else scale)), _lib.ptr(ws), nbytes, splits)
    return out


def _lengths(key_lengths, batch, keys):
    """key_lengths as the kernels read them."""
    if key_lengths.shape != (batch,) or key_lengths.dtype not in (torch.int32, torch.int64):
        raise ValueError("key_lengths must be int32 or int64 [batch]")
    # Clamped before the conversion, which would wrap what lies past 32 bits.
    if key_lengths.dtype == torch.int64:
        key_lengths = key_lengths.clamp(0, keys).to(torch.int32)
    return key_lengths.contiguous()


def attention(query, key, value, *, causal=False, scale=None, key_lengths=None):
    """softmax(scale * q k^T) v for query [batch, tokens, heads, head_dim] and key,
    value [batch, keys, kv_heads, head_dim]; returns a contiguous tensor like query.

    heads / kv_heads query heads in a row share a key head. causal: the last
    token sees all keys, each one before it one key fewer. scale defaults to
    head_dim ** -0.5. key_lengths (int32 or int64 [batch], on the GPU): sequence i
    has its first key_lengths[i] keys; what lies behind them, the unused part of a
    cache, is not read. A token that sees no key gives zeros, one whose keys all
    score -inf NaN (the formula's 0 / 0).
    """
    _check(query, key, value, 4)
    if key.shape[0] != query.shape[0]:
        raise ValueError(f"query has a batch of {query.shape[0]}, key of {key.shape[0]}")
    batch, tokens, keys = query.shape[0], query.shape[1], key.shape[1]
    if key_lengths is not None:
        key_lengths = _lengths(key_lengths, batch, keys)
    _lib.same_device(query, key=key, value=value, key_lengths=key_lengths)
    return _launch(query, key, value, None, None, key_lengths, causal, scale, batch, tokens, keys)


def _first_rows(t, name):
    if t.dim() != 1 or t.numel() < 1 or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be int32 or int64 [sequences + 1]")
    # Clamped before the conversion, which would wrap what lies past 32 bits.
    return (t.clamp(0, 2 ** 31 - 1).to(torch.int32) if t.dtype == torch.int64 else t).contiguous()


def attention_packed(query, key, value, cu_query, cu_key=None, *, causal=False, scale=None):
    """attention of sequences that lie behind each other: query [tokens, heads,
    head_dim], key and value [keys, kv_heads, head_dim].

    cu_query, cu_key (int32 or int64 [sequences + 1], nondecreasing, on the GPU;
    they are not copied to the host): sequence i has tokens cu_query[i] ..
    cu_query[i + 1] - 1 and keys cu_key[i] ..; cu_key defaults to cu_query. Empty
    sequences are allowed. Tokens of no sequence (before the first, behind the
    last) and tokens that see no key give zeros.
    """
    _check(query, key, value, 3)
    if cu_key is None:
        if key.shape[0] != query.shape[0]:
            raise ValueError("cu_key is needed where query and key differ in length")
        cu_key = cu_query
    if cu_key.numel() != cu_query.numel():
        raise ValueError("cu_query and cu_key must describe one number of sequences")
    _lib.same_device(query, key=key, value=value, cu_query=cu_query, cu_key=cu_key)
    same = cu_key is cu_query
    cu_query = _first_rows(cu_query, "cu_query")
    cu_key = cu_query if same else _first_rows(cu_key, "cu_key")
    return _launch(query, key, value, cu_query, cu_key, None, causal, scale, cu_query.numel() - 1, query.shape[0],
                   key.shape[0])


@functools.lru_cache(maxsize=4096)
def _prefix_strides(query, prefix_key, prefix_value, key, value, copied, q_shape, p_shape, k_shape):
    """The thirteen strides that lr_attention_prefix takes, of tensors with these strides:
    token, head and, of batches, sequence; None where one has to be copied first."""
    thirteen = array("q")
    for stride, shape in ((query, q_shape), (prefix_key, p_shape), (prefix_value, p_shape), (key, k_shape),
                          (value, k_shape)):
        if not copied and not _dense(stride, shape):
            return None
        s = [st if n > 1 else 0 for st, n in zip(stride, shape)]
        thirteen.extend((s[-3], s[-2]) if len(s) == 3 else (s[1], s[2], s[0]))
    return thirteen


@functools.lru_cache(maxsize=4096)
def _prefix_workspace(device, q_shape, p_shape, k_shape):
    """The bytes of its workspace, for shapes that fit together (checked here, once for each)."""
    batch, tokens, heads, dim = q_shape
    if p_shape[1:] != k_shape[2:]:
        raise ValueError("prefix_key and prefix_value must be [prefix, kv_heads, head_dim], with key's heads")
    if k_shape[0] != batch:
        raise ValueError(f"query has a batch of {batch}, key of {k_shape[0]}")
    if device < 0:
        return 0
    nbytes = array("q", [0])
    with torch.cuda.device(device):
        _lib.call("lr_attention_prefix_workspace", batch, tokens, k_shape[1], p_shape[0], heads, k_shape[2], dim,
                  nbytes.buffer_info()[0])
    return nbytes[0]


def attention_shared_prefix(query, prefix_key, prefix_value, key, value, *, causal=False, scale=None, key_lengths=None,
                            return_lse=False):
    """attention of a batch whose sequences share their first keys: query [batch, tokens,
    heads, head_dim], prefix_key and prefix_value [prefix, kv_heads, head_dim], key and
    value [batch, keys, kv_heads, head_dim]; returns a contiguous tensor like query.

    A token sees the whole prefix and the keys of its own sequence that it sees in
    attention(query, key, value, causal=.., key_lengths=..): causal counts the own
    keys alone. The prefix is read once for all sequences where they have few tokens
    each. Prefix, keys or both may be empty. return_lse: returns (output, lse), lse
    fp32 [batch, tokens, heads] the logarithm of the sum of exp(scale * q k) over the
    keys that a token sees, -inf where it sees none or all score -inf.
    """
    _check_tensors(query, key, value, 4)
    q_shape, p_shape, k_shape = query.shape, prefix_key.shape, key.shape
    if len(p_shape) != 3 or prefix_value.shape != p_shape:
        raise ValueError("prefix_key and prefix_value must be [prefix, kv_heads, head_dim], with key's heads")
    dtype = query.dtype
    if prefix_key.dtype != dtype or prefix_value.dtype != dtype:
        raise ValueError(f"the prefix must have the query's dtype, got {prefix_key.dtype}, {prefix_value.dtype}")
    if torch.is_grad_enabled() and (prefix_key.requires_grad or prefix_value.requires_grad):
        raise RuntimeError("gradients are not supported by the HIP attention: call it under torch.no_grad()")
    batch, tokens, heads, dim = q_shape
    keys, kv_heads = k_shape[1:3]
    nbytes = _prefix_workspace(query.get_device(), q_shape, p_shape, k_shape)
    if key_lengths is not None:
        key_lengths = _lengths(key_lengths, batch, keys)
    _lib.check_device(query)
    _lib.same_device(query, prefix_key=prefix_key, prefix_value=prefix_value, key=key, value=value,
                     key_lengths=key_lengths)
    scale = _scale_bits(float(dim ** -0.5 if scale is None else scale))
    given = (query, prefix_key, prefix_value, key, value)
    pointers = [t.data_ptr() for t in given]
    strides = None
    if not (pointers[0] | pointers[1] | pointers[2] | pointers[3] | pointers[4]) & 15:
        strides = _prefix_strides(*[t.stride() for t in given], False, q_shape, p_shape, k_shape)
    if strides is None:
        given = [_rows(t) for t in given]
        pointers = [t.data_ptr() for t in given]
        strides = _prefix_strides(*[t.stride() for t in given], True, q_shape, p_shape, k_shape)
    out = query.new_empty(q_shape)
    lse = torch.empty((batch, tokens, heads), dtype=torch.float32, device=query.device) if return_lse else None
    ws = _lib.workspace(query, nbytes) if nbytes else None   # held until the launch
    _lib.launch(query, "lr_attention_prefix", *pointers, out.data_ptr(), _lib.ptr(lse), _DTYPES[dtype], batch, tokens,
                keys, p_shape[0], heads, kv_heads, dim, strides.buffer_info()[0], _lib.ptr(key_lengths),
                int(bool(causal)), scale, _lib.ptr(ws), nbytes)
    return (out, lse) if return_lse else out


def block_attention(query, key, value, attention_mask, processor=None):
    """The attention of fusion.FusedAttention on this kernel: all tokens of
    [batch, tokens, heads, head_dim] see all keys. Masks are not supported, nor
    tokens that a processor's _parallel_config spreads over ranks (each would see its
    own alone); those errors are ones a guarded block falls back from."""
    if attention_mask is not None:
        raise RuntimeError("an attention mask is not supported by the HIP attention")
    if getattr(processor, "_parallel_config", None) is not None:
        raise RuntimeError("a parallel configuration is not supported by the HIP attention")
    return attention(query, key, value)
