"""What the attention entry points refuse, on the CPU."""
import struct
from array import array

import pytest
import torch

from lynnreal_omni_amd import _lib, attention as A


def qkv(q=(2, 3, 4, 64), k=(2, 5, 2, 64), dtype=torch.bfloat16):
    return torch.zeros(q, dtype=dtype), torch.zeros(k, dtype=dtype), torch.zeros(k, dtype=dtype)


@pytest.mark.parametrize("args", [
    qkv(q=(3, 4, 64)), qkv(q=(2, 3, 3, 64)), qkv(q=(2, 3, 4, 32)), qkv(k=(2, 5, 0, 64)), qkv(),
    qkv()[:2] + (torch.zeros(2, 6, 2, 64, dtype=torch.bfloat16),),
    qkv()[:2] + (torch.zeros(2, 5, 2, 64),)])
def test_wrong_tensors(args):
    with pytest.raises(ValueError):
        A.attention(*args)


@pytest.mark.parametrize("args", [qkv(dtype=torch.float32), qkv(q=(2, 3, 4, 96), k=(2, 5, 2, 96))])
def test_not_supported_is_recoverable(args):
    with pytest.raises(RuntimeError, match="not supported"):
        A.attention(*args)


def test_gradients_are_refused():
    q, k, v = qkv()
    with pytest.raises(RuntimeError, match="gradients are not supported"):
        A.attention(q.requires_grad_(), k, v)
    with pytest.raises(ValueError, match="GPU"):       # without gradients it gets as far as the device check
        with torch.no_grad():
            A.attention(q, k, v)


def test_masks_are_refused():
    with pytest.raises(RuntimeError, match="not supported"):
        A.block_attention(*qkv(), torch.ones(2, 5, dtype=torch.bool))


def test_lists():
    q, k, v = (t[0] for t in qkv(q=(1, 5, 4, 64), k=(1, 5, 2, 64)))
    with pytest.raises(ValueError):
        A.attention_packed(q, k, v, torch.zeros(2, 2, dtype=torch.int32))
    with pytest.raises(ValueError):
        A._first_rows(torch.zeros(3), "cu_query")
    # What lies past 32 bits stays behind the last row instead of wrapping.
    assert A._first_rows(torch.tensor([-2 ** 40, 5, 2 ** 40]), "cu_query").tolist() == [0, 5, 2 ** 31 - 1]
    with pytest.raises(ValueError):
        A._scale_bits(0.0)
    with pytest.raises(ValueError):
        A._scale_bits(float("nan"))


def test_rows_are_copied_only_where_needed():
    fused = torch.zeros(2, 5, 3, 4, 64, dtype=torch.bfloat16)
    assert A._rows(fused[:, :, 1]).data_ptr() == fused[:, :, 1].data_ptr()
    odd = torch.zeros(2, 5, 4, 65, dtype=torch.bfloat16)[..., :64]
    assert A._rows(odd).is_contiguous()
    assert A._rows(torch.zeros(2, 64, 4, 5, dtype=torch.bfloat16).permute(0, 3, 2, 1)).is_contiguous()
    shifted = torch.zeros(2 * 5 * 4 * 64 + 1, dtype=torch.bfloat16)[1:].view(2, 5, 4, 64)
    assert A._rows(shifted).data_ptr() % 16 == 0


def test_entry_point_refusals_without_a_gpu():
    lib, p = _lib.load(), 4096
    one = struct.unpack("i", struct.pack("f", 1.0))[0]
    kept = []

    def strides(**kw):
        s = array("q", {**dict(qt=256, qh=64, qs=0, kt=128, kh=64, ks=0, vt=128, vh=64, vs=0), **kw}.values())
        kept.append(s)
        return s.buffer_info()[0]

    good = dict(q=p, k=p, v=p, out=p, dtype=0, n=1, qr=4, kr=4, heads=4, kv=2, dim=64, st=strides(), cuq=None, cuk=None, lens=None, causal=0, scale=one, ws=None, wsb=0,
                splits=1, stream=None)
    call = lambda **kw: lib.lr_attention(*{**good, **kw}.values())  # noqa: E731
    assert call(qr=0) == _lib.LR_OK and call(n=0) == _lib.LR_OK
    assert call(dim=96) == _lib.LR_EUNSUPPORTED
    for bad in [dict(dtype=2), dict(heads=3), dict(kv=0), dict(q=None), dict(k=None), dict(q=p + 2), dict(st=strides(qt=252)),
                dict(st=strides(kt=1 << 23)), dict(st=strides(vh=-64)), dict(st=None), dict(cuq=p), dict(cuq=p, cuk=p, lens=p), dict(scale=0), dict(n=-1),
                dict(splits=0), dict(splits=2), dict(splits=2, ws=p, wsb=8), dict(qr=1 << 30),
                dict(scale=struct.unpack("i", struct.pack("f", float("inf")))[0])]:
        assert call(**bad) == _lib.LR_EINVAL, bad
    assert lib.lr_attention_splits(0, 1, 1, 0, 4, 2) == 1
    assert lib.lr_attention_splits(1, 1, 131072, 0, 56, 8) > 1
    # Padded caches: pieces of all sequences, none where there is a single tile of keys.
    assert lib.lr_attention_splits(8, 1, 8192, 2, 40, 8) > 8
    assert lib.lr_attention_splits(2, 32, 64, 2, 8, 8) == 1
    assert lib.lr_attention_splits(1, 12605, 12605, 0, 56, 56) == 1
