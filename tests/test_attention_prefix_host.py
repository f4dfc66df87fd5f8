"""What attention over a shared prefix refuses, and how it plans, on the CPU."""
import random
import struct
from array import array

import pytest
import torch

from lynnreal_omni_amd import _lib, attention as A


def five(q=(2, 3, 4, 64), p=(7, 2, 64), k=(2, 5, 2, 64), dtype=torch.bfloat16):
    return [torch.zeros(shape, dtype=dtype) for shape in (q, p, p, k, k)]


def changed(at, t):
    args = five()
    args[at] = t
    return args


@pytest.mark.parametrize("args", [
    five(q=(3, 4, 64)), five(q=(2, 3, 3, 64)), five(p=(7, 4, 64)), five(p=(7, 2, 32)), five(p=(1, 7, 2, 64)),
    five(k=(3, 5, 2, 64)), five(k=(2, 5, 0, 64), p=(7, 0, 64)), changed(2, torch.zeros(8, 2, 64, dtype=torch.bfloat16)),
    changed(1, torch.zeros(7, 2, 64)), changed(2, torch.zeros(7, 2, 64, dtype=torch.float16)),
    changed(4, torch.zeros(2, 6, 2, 64, dtype=torch.bfloat16)), five()])
def test_wrong_tensors(args):
    with pytest.raises(ValueError):     # the last: right, but not on a GPU
        A.attention_shared_prefix(*args)


@pytest.mark.parametrize("args", [five(dtype=torch.float32), five(q=(2, 3, 4, 96), p=(7, 2, 96), k=(2, 5, 2, 96))])
def test_not_supported_is_recoverable(args):
    with pytest.raises(RuntimeError, match="not supported"):
        A.attention_shared_prefix(*args)


@pytest.mark.parametrize("at", range(5))
def test_gradients_are_refused(at):
    args = five()
    args[at].requires_grad_()
    # (The prefix is looked at behind the device, which is none here.)
    with pytest.raises((RuntimeError, ValueError), match="gradients are not supported|GPU"):
        A.attention_shared_prefix(*args)


def test_entry_point_refusals_without_a_gpu():
    lib, p = _lib.load(), 4096
    one = struct.unpack("i", struct.pack("f", 1.0))[0]
    kept = []

    def strides(at=0, value=256):
        s = array("q", [256, 64, 1024, 128, 64, 128, 64, 128, 64, 640, 128, 64, 640])
        s[at] = value
        kept.append(s)
        return s.buffer_info()[0]

    good = dict(q=p, pk=p, pv=p, k=p, v=p, out=p, lse=p, dtype=0, n=1, qr=4, kr=4, pr=4, heads=4, kv=2, dim=64,
                st=strides(), lens=None, causal=0, scale=one, ws=None, wsb=0, stream=None)
    call = lambda **kw: lib.lr_attention_prefix(*{**good, **kw}.values())  # noqa: E731
    assert call(qr=0) == _lib.LR_OK and call(n=0) == _lib.LR_OK
    assert call(dim=96) == _lib.LR_EUNSUPPORTED
    infinite = struct.unpack("i", struct.pack("f", float("inf")))[0]
    for bad in [dict(dtype=2), dict(heads=3), dict(kv=0), dict(q=None), dict(k=None), dict(pk=None), dict(pv=None),
                dict(out=None), dict(q=p + 2), dict(pk=p + 8), dict(lse=p + 2), dict(st=None), dict(st=strides(0, 252)),
                dict(st=strides(3, 1 << 23)), dict(st=strides(5, 1 << 23)), dict(st=strides(7, 1 << 23)),
                dict(st=strides(10, 1 << 23)), dict(st=strides(12, -640)), dict(n=-1), dict(pr=-1), dict(pr=1 << 30),
                dict(n=1 << 24), dict(n=1 << 20, qr=1 << 20), dict(scale=0), dict(scale=infinite),
                # Two short sequences behind a long prefix need a workspace.
                dict(n=2, qr=1, pr=100000), dict(n=2, qr=1, pr=100000, ws=p, wsb=1024)]:
        assert call(**bad) == _lib.LR_EINVAL, bad


def test_workspace():
    lib, out = _lib.load(), array("q", [0])
    size = lambda *shape: lib.lr_attention_prefix_workspace(*shape, out.buffer_info()[0])  # noqa: E731
    assert size(0, 1, 1, 1, 4, 2, 64) == _lib.LR_OK and out[0] == 0
    assert size(32, 1, 1024, 12605, 40, 8, 128) == _lib.LR_OK and out[0] > 0
    # Whole prompts are walked in one pass: none where that makes full rounds of workgroups (four
    # of them on 256 CUs), a few rows for what is left behind them where not.
    assert size(4, 1024, 1024, 12605, 64, 64, 128) == _lib.LR_OK and out[0] == 0
    assert size(4, 878, 878, 12605, 56, 56, 128) == _lib.LR_OK and 0 < out[0] < 1 << 25
    assert size(1, 1, 1, 1, 3, 2, 64) == _lib.LR_EINVAL
    assert size(1, 1, 1, 1, 4, 2, 96) == _lib.LR_EUNSUPPORTED
    rng = random.Random(1)

    def log_int(lo, hi):
        return round(lo * (hi / lo) ** rng.random())

    for _ in range(5000):
        kv = log_int(1, 64)
        rc = size(log_int(1, 5000), log_int(1, 4000), log_int(1, 1 << 20), log_int(1, 1 << 20), kv * log_int(1, 16), kv,
                  128)
        assert rc in (_lib.LR_OK, _lib.LR_EINVAL) and out[0] >= 0
