"""Padded key/value caches of bounded size, on gfx950: which keys the attention needs,
and caches cut down to those.

  accumulate_weights  adds to each key's weight what new tokens' softmax gives it
  evict               the latest keys and those of most weight, moved to a smaller cache

A step of a request whose cache has a budget:

  out, lse = attention_shared_prefix(q, prefix_k, prefix_v, k, v, causal=True,
                                     key_lengths=lengths, return_lse=True)
  weights = accumulate_weights(weights, q, k, lse, causal=True, key_lengths=lengths, out=weights)
  ..      # and when the caches have outgrown the budget
  k, v, weights, lengths, kept = evict(k, v, weights, lengths, budget, recent=64)

(without a shared prefix: attention_shared_prefix with an empty one). Keys are
[batch, keys, kv_heads, head_dim], bf16 or fp16, read as attention reads them;
each head keeps its own keys, so that after an eviction a place holds other keys in
other heads, with the same number of them in all. Weights are fp32 [batch, kv_heads,
keys]. Lengths are never copied to the host. Inference only: inputs that require a
gradient are refused.
"""
from __future__ import annotations

import functools
from array import array

import torch

from . import _lib
from . import attention as _attention


def _check_weights(weights, key, name="weights"):
    batch, keys, kv_heads = key.shape[:3]
    if weights.shape != (batch, kv_heads, keys) or weights.dtype != torch.float32:
        raise ValueError(f"{name} must be float32 [batch, kv_heads, keys] = {(batch, kv_heads, keys)}, "
                         f"got {weights.dtype} {tuple(weights.shape)}")


def _no_gradients(*tensors):
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError("gradients are not supported by the HIP caches: call it under torch.no_grad()")


@functools.lru_cache(maxsize=4096)
def _weights_workspace(device, batch, tokens, keys, heads, kv_heads, dim):
    nbytes = array("q", [0])
    with torch.cuda.device(device):
        _lib.call("lr_attention_weights_workspace", batch, tokens, keys, heads, kv_heads, dim, nbytes.buffer_info()[0])
    return nbytes[0]


@functools.lru_cache(maxsize=4096)
def _six_strides(query, key, copied, q_shape, k_shape):
    """The six strides that lr_attention_weights takes, of batches with these strides: token,
    head and sequence; None where one has to be copied first."""
    six = array("q")
    for stride, shape in ((query, q_shape), (key, k_shape)):
        if not copied and not _attention._dense(stride, shape):
            return None
        s = [st if n > 1 else 0 for st, n in zip(stride, shape)]
        six.extend((s[1], s[2], s[0]))
    # The kernel's 32-bit offsets have to reach the heads of a key head and 64 tokens.
    return six if copied or q_shape[2] * six[1] < 1 << 30 else None


def accumulate_weights(weights, query, key, lse, *, causal=False, scale=None, key_lengths=None, out=None):
    """weights plus the attention weight that each key gets from query's tokens: exp(scale *
    q . k - lse), summed over the tokens and query heads that see the key, for query
    [batch, tokens, heads, head_dim], key [batch, keys, kv_heads, head_dim] and lse
    float32 [batch, tokens, heads], the logarithm of each softmax's sum.

    weights: float32 [batch, kv_heads, keys]; returned as a new tensor, or in `out`,
    which may be weights itself. causal, scale and key_lengths as in attention: what a
    token does not see gets nothing from it, and places behind key_lengths keep their
    weight. Sums are fp32 in a fixed order.
    """
    _attention._check_tensors(query, key, key, 4)
    if key.shape[0] != query.shape[0]:
        raise ValueError(f"query has a batch of {query.shape[0]}, key of {key.shape[0]}")
    _check_weights(weights, key)
    if lse.shape != query.shape[:3] or lse.dtype != torch.float32:
        raise ValueError(f"lse must be float32 [batch, tokens, heads] = {tuple(query.shape[:3])}")
    _no_gradients(weights, lse)
    batch, tokens, heads, dim = query.shape
    keys, kv_heads = key.shape[1:3]
    if key_lengths is not None:
        key_lengths = _attention._lengths(key_lengths, batch, keys)
    if out is not None:
        _check_weights(out, key, "out")
        _no_gradients(out)
        same = out.data_ptr() == weights.data_ptr() and weights.is_contiguous()
        if not out.is_contiguous() or _clash((out,), (None if same else weights, query, key, lse, key_lengths)):
            raise ValueError("out must be contiguous, and weights themselves or memory of its own")
    scale = _attention._scale_bits(float(dim ** -0.5 if scale is None else scale))
    _lib.check_device(query)
    _lib.same_device(query, key=key, weights=weights, lse=lse, key_lengths=key_lengths, out=out)
    if out is None:
        out = torch.empty_like(weights, memory_format=torch.contiguous_format)
    weights, lse = weights.contiguous(), lse.contiguous()
    strides = None
    if not (query.data_ptr() | key.data_ptr()) & 15:
        strides = _six_strides(query.stride(), key.stride(), False, query.shape, key.shape)
    if strides is None:
        query, key = query.clone(memory_format=torch.contiguous_format), _attention._rows(key)
        strides = _six_strides(query.stride(), key.stride(), True, query.shape, key.shape)
    nbytes = _weights_workspace(query.get_device(), batch, tokens, keys, heads, kv_heads, dim)
    ws = _lib.workspace(query, nbytes) if nbytes else None   # held until the launch
    _lib.launch(query, "lr_attention_weights", query.data_ptr(), key.data_ptr(), lse.data_ptr(), weights.data_ptr(),
                out.data_ptr(), _attention._DTYPES[query.dtype], batch, tokens, keys, heads, kv_heads, dim,
                strides.buffer_info()[0], _lib.ptr(key_lengths), int(bool(causal)), scale, _lib.ptr(ws), nbytes)
    return out


def _span(t):
    """First and last byte (exclusive) of what a tensor's elements lie in; nothing where it has none."""
    first, size = t.data_ptr(), t.element_size()
    if t.is_contiguous():
        return first, first + t.numel() * size
    shape = t.shape
    return first, first if 0 in shape else first + (sum([(n - 1) * st for n, st in zip(shape, t.stride())]) + 1) * size


def _clash(written, read):
    """Whether one of the tensors in `written` has memory in common with another of them or with one
    in `read` (None is skipped). Rows between each other's are apart."""
    spans = [(t, *_span(t)) for t in written]
    for i, (a, a0, a1) in enumerate(spans):
        for b, b0, b1 in spans[:i]:
            if a0 < b1 and b0 < a1 and _share(_layout(a), _layout(b), b0 - a0):
                return True
    last = max([a1 for _, _, a1 in spans])
    for b in read:
        if b is None or b.data_ptr() >= last:   # behind them all, as half of what is looked at
            continue
        b0, b1 = _span(b)
        for a, a0, a1 in spans:
            if a0 < b1 and b0 < a1 and _share(_layout(a), _layout(b), b0 - a0):
                return True
    return False


def _layout(t):
    return t.shape, t.stride(), t.element_size()


@functools.lru_cache(maxsize=4096)
def _share(a, b, apart):
    return _meet(_runs(*a), _runs(*b), apart, [10000])


def _runs(shape, stride, size):
    """A tensor's memory as (bytes between, number of) runs from the outermost on, the last one
    of single bytes."""
    runs = [(1, size)]
    for st, n in sorted((st * size, n) for st, n in zip(stride, shape) if n > 1 and st > 0):
        step, count = runs[-1]
        if st == step * count:
            runs[-1] = (step, count * n)   # behind each other
        else:
            runs.append((st, n))
    return tuple(reversed(runs))


def _meet(a, b, apart, budget):
    """Whether runs a and b, which begin `apart` bytes behind a's, have a byte in common. Exact,
    but for strides so unlike each other that the budget of steps ends: those are taken to have."""
    reach_a, reach_b = (sum((n - 1) * st for st, n in runs) + 1 for runs in (a, b))
    if apart >= reach_a or -apart >= reach_b:
        return False
    if len(a) == 1 and len(b) == 1:
        return True
    budget[0] -= 1
    if budget[0] < 0:
        return True
    if a[0][0] < b[0][0]:
        a, b, reach_a, reach_b, apart = b, a, reach_b, reach_a, -apart
    (step, n), inner = a[0], a[1:]
    reach = reach_a - (n - 1) * step
    if b[0][0] == step:
        # Only how many steps a's run lies before b's matters.
        others, reach_b, low = b[1:], reach_b - (b[0][1] - 1) * step, 1 - b[0][1]
    else:
        others, low = b, 0
    # The run i of a begins i steps behind its first and has to reach others, from `apart` to there + reach_b.
    first, last = max(low, -((reach - apart - 1) // step)), min(n - 1, (apart + reach_b - 1) // step)
    return any(_meet(inner, others, apart - i * step, budget) for i in range(first, last + 1))


def _distinct(t):
    """Whether no two elements of t are the same memory, for strides that nest (as those
    of slices and transposes do)."""
    at = 1
    for st, n in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1):
        if st < at:
            return False
        at = st * (n - 1) + at
    return True


@functools.lru_cache(maxsize=4096)
def _byte_strides(copied, *tensors):
    """The twelve strides in bytes that lr_cache_evict takes, of 16-bit tensors given as
    (stride, shape); None where one of the first two has to be copied first."""
    twelve = array("q")
    for i, (stride, shape) in enumerate(tensors):
        if i < 2 and not copied and not _attention._dense(stride, shape):
            return None
        s = [2 * st if n > 1 else 0 for st, n in zip(stride, shape)]
        twelve.extend((s[1], s[2], s[0]))
    return twelve


def evict(key, value, weights, key_lengths, budget, *, recent=0, out=None):
    """Caches cut down to `budget` keys per head: of each cache's first key_lengths[i] keys
    (all where None) the last `recent` and, of those before them, the ones of most weight; of
    equal weights the first ones, NaN counting least; all of them where there are no more than
    the budget. They keep their order.

    key, value [batch, keys, kv_heads, head_dim], weights float32 [batch, kv_heads, keys],
    budget >= 1, 0 <= recent <= budget. Returns (key, value, weights, lengths, kept):
    new caches [batch, budget, kv_heads, head_dim], zeros behind their last keys; their
    weights [batch, kv_heads, budget], 0 behind; lengths int32 [batch]; and kept int32
    [batch, kv_heads, budget], the places that the keys had, -1 behind the last.

    out = (key, value, weights): caches of any number of places from `budget` on, of
    memory that neither the inputs nor another of them have (rows between each other's are
    fine), written instead of new ones; rows of theirs behind the last key stay as they
    were, weights there become 0.
    """
    if key.dim() != 4 or value.shape != key.shape or value.dtype != key.dtype:
        raise ValueError("key and value must be [batch, keys, kv_heads, head_dim], of one shape and dtype")
    if key.dtype not in _attention._DTYPES:
        raise RuntimeError(f"dtype {key.dtype} is not supported by the HIP caches (bfloat16 or float16)")
    batch, keys, kv_heads, dim = key.shape
    if kv_heads == 0 or dim == 0:
        raise ValueError("key and value have no heads or no columns")
    if dim % 8:
        raise RuntimeError(f"head_dim {dim} is not supported by the HIP caches (a multiple of 8)")
    _check_weights(weights, key)
    budget, recent = int(budget), int(recent)
    if budget < 1 or not 0 <= recent <= budget:
        raise ValueError(f"budget must be at least 1 and recent from 0 to budget, got {budget} and {recent}")
    _no_gradients(key, value, weights)
    if key_lengths is not None:
        key_lengths = _attention._lengths(key_lengths, batch, keys)
    if out is not None:
        key_out, value_out, weights_out = out
        _check_out(key, value, weights, key_lengths, key_out, value_out, weights_out, budget)
    _lib.check_device(key)
    _lib.same_device(key, value=value, weights=weights, key_lengths=key_lengths)
    if out is None:
        shape = (batch, budget, kv_heads, dim)
        key_out, value_out = key.new_empty(shape), key.new_empty(shape)
        weights_out = weights.new_empty((batch, kv_heads, budget))
    lengths = torch.empty(batch, dtype=torch.int32, device=key.device)
    kept = torch.empty((batch, kv_heads, budget), dtype=torch.int32, device=key.device)
    if not weights.is_contiguous():
        weights = weights.contiguous()
    shape, new = key.shape, key_out.shape
    outs = (key_out.stride(), new), (value_out.stride(), new)
    strides = None
    if not (key.data_ptr() | value.data_ptr()) & 15:
        strides = _byte_strides(False, (key.stride(), shape), (value.stride(), shape), *outs)
    if strides is None:
        key, value = _attention._rows(key), _attention._rows(value)
        strides = _byte_strides(True, (key.stride(), shape), (value.stride(), shape), *outs)
    nbytes = _evict_workspace(batch, keys, kv_heads)
    ws = _lib.workspace(key, nbytes) if nbytes else None   # held until the launch
    _lib.launch(key, "lr_cache_evict", key.data_ptr(), value.data_ptr(), weights.data_ptr(), _lib.ptr(key_lengths),
                key_out.data_ptr(), value_out.data_ptr(), weights_out.data_ptr(), lengths.data_ptr(), kept.data_ptr(),
                batch, keys, kv_heads, 2 * dim, budget, recent, new[1], strides.buffer_info()[0],
                int(out is None), _lib.ptr(ws), nbytes)
    return key_out, value_out, weights_out, lengths, kept


@functools.lru_cache(maxsize=4096)
def _evict_workspace(batch, keys, kv_heads):
    nbytes = array("q", [0])
    _lib.call("lr_cache_evict_workspace", batch, keys, kv_heads, nbytes.buffer_info()[0])
    return nbytes[0]


def _check_out(key, value, weights, key_lengths, key_out, value_out, weights_out, budget):
    batch, _, kv_heads, dim = key.shape
    if (key_out.dim() != 4 or key_out.shape[1] < budget or key_out.shape != (batch, key_out.shape[1], kv_heads, dim)
            or value_out.shape != key_out.shape or key_out.dtype != key.dtype or value_out.dtype != key.dtype):
        raise ValueError(f"out must hold {key.dtype} caches [{batch}, at least {budget}, {kv_heads}, {dim}]")
    _check_weights(weights_out, key_out, "out's weights")
    _lib.same_device(key, key_out=key_out, value_out=value_out, weights_out=weights_out)
    _no_gradients(key_out, value_out, weights_out)
    if not weights_out.is_contiguous() or any(
            t.data_ptr() & 15 or not _attention._dense(t.stride(), t.shape) or not _distinct(t)
            for t in (key_out, value_out)):
        raise ValueError("out must be caches whose rows are dense, 16-byte aligned and distinct, and contiguous weights")
    if _clash((key_out, value_out, weights_out), (key, value, weights, key_lengths)):
        raise ValueError("out's keys, values and weights must not overlap each other, nor the caches that are cut down")
