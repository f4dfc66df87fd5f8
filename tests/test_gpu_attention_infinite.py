"""Rows of the attention whose visible scores are all -inf: NaN, as the formula
(exp(-inf + inf) / 0), in every path; a row that sees no key gives zeros, and -inf
scores beside finite ones have the weight zero."""
import math

import pytest
import torch

from lynnreal_omni_amd import _lib
from lynnreal_omni_amd import attention as A
from test_gpu_attention import check, formula, mask, tensors

pytestmark = pytest.mark.gpu

INF = -math.inf


def positive(q, k):
    """Queries of positive numbers, so that a key of -inf has the score -inf."""
    return q.abs() + 0.01, k


def split(kind, *shape):
    """Whether a call of this shape cuts its keys."""
    return _lib.load().lr_attention_splits(*shape[:3], kind, *shape[3:]) > 1


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,dim", [(20, 64), (70, 128), (300, 32)])
def test_causal_first_tokens(rows, dim, dtype):
    """The first two keys are -inf: the first two tokens see nothing else."""
    q, k, v = tensors(rows, rows, 2, 2, dim, dtype, rows)
    q, k = positive(q, k)
    k[:2] = INF
    got = A.attention(q[None], k[None], v[None], causal=True)[0]
    assert got[:2].isnan().all()
    # A token i from the third on: keys 2 .. i.
    check(got[2:], *formula(q[2:], k[2:], v[2:], dim ** -0.5, mask(rows - 2, rows - 2, True)))
    packed = A.attention_packed(q, k, v, torch.tensor([0, 0, 2, rows], device="cuda"), causal=True)
    assert packed[:2].isnan().all()
    check(packed[2:], *formula(q[2:], k[2:], v[2:], dim ** -0.5, mask(rows - 2, rows - 2, True)))


@pytest.mark.parametrize("rows", [1, 40])
def test_split_keys(rows):
    """One sequence over many workgroups: all keys, all but one of the last, none."""
    keys, heads, dim = 4096, 2, 64
    assert split(0, 1, rows, keys, heads, heads)
    q, k, v = tensors(rows, keys, heads, heads, dim, torch.bfloat16, rows)
    q, k = positive(q, k)
    none = torch.full_like(k, INF)
    assert A.attention(q[None], none[None], v[None]).isnan().all()
    for at in (0, 63, 2000, keys - 1):
        one = none.clone()
        one[at] = k[at]
        assert torch.equal(A.attention(q[None], one[None], v[None])[0], v[at].expand(rows, heads, dim))
    # The first half alone, and causal: tokens that see the first half only.
    half = k.clone()
    half[:keys // 2] = INF
    check(A.attention(q[None], half[None], v[None])[0],
          *formula(q, k[keys // 2:], v[keys // 2:], dim ** -0.5, mask(rows, keys // 2, False)))
    tail = k.clone()
    tail[:keys - rows + 1] = INF       # token i sees i keys that are not -inf
    got = A.attention(q[None], tail[None], v[None], causal=True)[0]
    assert got[0].isnan().all()
    if rows > 1:
        check(got[1:], *formula(q[1:], k[keys - rows + 1:], v[keys - rows + 1:], dim ** -0.5,
                                mask(rows - 1, rows - 1, True)))


@pytest.mark.parametrize("new,heads,kv_heads", [(1, 4, 2), (40, 4, 4)])
@pytest.mark.parametrize("size", [50, 2000])
def test_padded_caches(size, new, heads, kv_heads):
    """A cache of -inf keys gives NaN, an empty one beside it zeros, and keys behind the
    valid ones do not count."""
    lengths, dim = [size, 0, 30, size - 3, 1], 64
    g = torch.Generator().manual_seed(size)
    q = torch.rand(5, new, heads, dim, generator=g).add(0.01).half().cuda()
    k, v = (torch.randn(5, size, kv_heads, dim, generator=g).half().cuda() for _ in range(2))
    k[0], k[2, :30], k[3, :29], k[4, 0] = INF, INF, INF, INF
    given = torch.tensor(lengths, device="cuda", dtype=torch.int32)
    got = A.attention(q, k, v, key_lengths=given)
    assert got[[0, 2, 4]].isnan().all() and (got[1] == 0).all()
    check(got[3], *formula(q[3], k[3, 29:size - 3], v[3, 29:size - 3], dim ** -0.5, mask(new, size - 32, False)))
    # Causal: the tokens before the last `lengths` see no key and stay zero.
    got = A.attention(q, k, v, key_lengths=given, causal=True)
    for i, n in enumerate(lengths):
        assert (got[i, :max(0, new - n)] == 0).all()
    assert got[0, max(0, new - size):].isnan().all() and got[2, max(0, new - 30):].isnan().all()
    assert got[4, -1].isnan().all()
