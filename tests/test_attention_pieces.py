"""The places of a list of pieces over padded caches: the kernel counts on two for each
sequence at least, on the CPU."""
import random

import pytest

from lynnreal_omni_amd import _lib

LENGTHS = 2     # lr_attention_splits' kind of a batch with key lengths


@pytest.mark.parametrize("seed", range(4))
def test_lists_have_two_places_for_each_sequence(seed):
    lib, rng = _lib.load(), random.Random(seed)

    def log_int(lo, hi):
        return round(lo * (hi / lo) ** rng.random())

    lists = 0
    for _ in range(5000):
        kv_heads = log_int(1, 64)
        n, rows, keys = log_int(1, 600), log_int(1, 600), log_int(1, 1 << 20)
        splits = lib.lr_attention_splits(n, rows, keys, LENGTHS, kv_heads * log_int(1, 16), kv_heads)
        assert splits == 1 or splits >= 2 * n
        lists += splits > 1
    assert lists > 500
