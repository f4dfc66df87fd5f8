"""Calls that the attention has to refuse instead of answering wrongly, on the CPU."""
import types

import pytest
import torch

from lynnreal_omni_amd import acceleration, fusion
from lynnreal_omni_amd import attention as A


def qkv():
    return tuple(torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16) for _ in range(3))


def test_sharded_tokens_are_refused():
    """With its tokens over several ranks a block's attention has to see the other ranks'
    keys: block_attention refuses, with an error that a guarded block falls back from."""
    native = types.SimpleNamespace(_attention_backend=None, _parallel_config=object())
    processor = fusion.FusedAttention(native, attention=A.block_attention)
    with pytest.raises(RuntimeError, match="not supported") as refused:
        processor._attend(*qkv(), None)
    assert acceleration.optional_kernel_failure(refused.value)
    # Without one it gets as far as the device check.
    for config in ({}, {"_parallel_config": None}):
        processor = fusion.FusedAttention(types.SimpleNamespace(**config), attention=A.block_attention)
        with pytest.raises(ValueError, match="GPU"):
            processor._attend(*qkv(), None)
    with pytest.raises(ValueError, match="GPU"):
        A.block_attention(*qkv(), None)
