"""What the operators of bounded caches refuse, on the CPU."""
import itertools
import random
import struct
from array import array

import pytest
import torch

from lynnreal_omni_amd import _lib, cache

BF16 = torch.bfloat16


def weigh(q=(2, 3, 4, 64), k=(2, 5, 2, 64), w=(2, 2, 5), lse=(2, 3, 4), dtype=BF16):
    return torch.zeros(w), torch.zeros(q, dtype=dtype), torch.zeros(k, dtype=dtype), torch.zeros(lse)


@pytest.mark.parametrize("args,kwargs,match", [
    (weigh(q=(3, 4, 64)), {}, "query, key"), (weigh(q=(2, 3, 3, 64), lse=(2, 3, 3)), {}, "share"),
    (weigh(q=(3, 3, 4, 64), lse=(3, 3, 4)), {}, "batch"), (weigh(w=(2, 5, 2)), {}, "weights must be"),
    (weigh(lse=(2, 4, 3)), {}, "lse must be"), (weigh(), dict(scale=0.0), "scale"),
    (weigh(), dict(key_lengths=torch.zeros(3, dtype=torch.int32)), "key_lengths"),
    (weigh(), dict(key_lengths=torch.zeros(2)), "key_lengths"), (weigh(), dict(out=torch.zeros(2, 2, 6)), "out must be"),
    (weigh(), dict(out=torch.zeros(2, 5, 2).transpose(1, 2)), "out must be contiguous"), (weigh(), {}, "GPU")])
def test_wrong_weights(args, kwargs, match):
    with pytest.raises(ValueError, match=match):
        cache.accumulate_weights(*args, **kwargs)


def test_weights_out_is_weights_or_other_memory():
    memory = torch.zeros(30)
    weights, q, k, lse = weigh()
    w = memory[:20].view(2, 2, 5)
    for out, match in ((memory[5:25].view(2, 2, 5), "out must"), (w, "GPU"), (torch.zeros(2, 2, 5), "GPU")):
        with pytest.raises(ValueError, match=match):
            cache.accumulate_weights(w, q, k, lse, out=out)
    shared = torch.zeros(64)
    with pytest.raises(ValueError, match="out must"):
        cache.accumulate_weights(weights, q, k, shared[:24].view(2, 3, 4), out=shared[20:40].view(2, 2, 5))
    # Weights read through other strides than out's, from the same first element.
    with pytest.raises(ValueError, match="out must"):
        cache.accumulate_weights(memory[:20].view(2, 5, 2).transpose(1, 2), q, k, lse, out=w)


@pytest.mark.parametrize("args", [weigh(dtype=torch.float32), weigh(q=(2, 3, 4, 96), k=(2, 5, 2, 96))])
def test_weights_not_supported(args):
    with pytest.raises(RuntimeError, match="not supported"):
        cache.accumulate_weights(*args)


def test_gradients_are_refused():
    for at in range(4):
        args = weigh()
        args[at].requires_grad_()
        with pytest.raises(RuntimeError, match="gradients are not supported"):
            cache.accumulate_weights(*args)
    for at in range(3):
        args = caches()[:3]
        args[at].requires_grad_()
        with pytest.raises(RuntimeError, match="gradients are not supported"):
            cache.evict(*args, None, 3)


def caches(k=(2, 5, 2, 64), w=(2, 2, 5), dtype=BF16):
    return torch.zeros(k, dtype=dtype), torch.zeros(k, dtype=dtype), torch.zeros(w), None


@pytest.mark.parametrize("args,kwargs,match", [
    ((*caches(k=(5, 2, 64)), 3), {}, "key and value"), ((*caches(w=(2, 5, 2)), 3), {}, "weights must be"),
    ((*caches(), 0), {}, "budget"), ((*caches(), 3), dict(recent=4), "recent"), ((*caches(), 3), dict(recent=-1), "recent"),
    ((*caches(k=(2, 5, 0, 64), w=(2, 0, 5)), 3), {}, "no heads"),
    ((*caches()[:3], torch.zeros(3, dtype=torch.int32), 3), {}, "key_lengths"), ((*caches(), 3), {}, "GPU")])
def test_wrong_evictions(args, kwargs, match):
    with pytest.raises(ValueError, match=match):
        cache.evict(*args, **kwargs)


@pytest.mark.parametrize("args", [caches(dtype=torch.float32), caches(k=(2, 5, 2, 60))])
def test_evictions_not_supported(args):
    with pytest.raises(RuntimeError, match="not supported"):
        cache.evict(*args, 3)


def test_eviction_into_given_caches():
    key, value, weights, _ = caches()

    def new(places=4, dtype=BF16):
        return [torch.zeros(2, places, 2, 64, dtype=dtype), torch.zeros(2, places, 2, 64, dtype=dtype),
                torch.zeros(2, 2, places)]

    def out(at, t):
        tensors = new()
        tensors[at] = t
        return tensors

    twice = torch.zeros(2, 4, 2, 64, dtype=BF16)
    one = torch.zeros(1, 4, 2, 64, dtype=BF16).expand(2, -1, -1, -1)
    for bad in (new(2), new(dtype=torch.float16), out(0, torch.zeros(2, 5, 2, 64, dtype=BF16)), out(2, torch.zeros(2, 2, 5)),
                out(0, key[:, :4]), out(1, value[:, 1:]), out(2, weights[..., :4]), [twice, twice, torch.zeros(2, 2, 4)],
                out(0, one), out(0, torch.zeros(2, 4, 2, 65, dtype=BF16)[..., :64]),
                out(2, torch.zeros(2, 4, 2).transpose(1, 2))):
        with pytest.raises(ValueError, match="out"):
            cache.evict(key, value, weights, None, 3, out=bad)
    # Right ones, keys and values in one buffer among them, get as far as the device check.
    both = torch.zeros(2, 4, 2, 2, 64, dtype=BF16)
    for good in (new(), [both[:, :, 0], both[:, :, 1], torch.zeros(2, 2, 4)]):
        with pytest.raises(ValueError, match="GPU"):
            cache.evict(key, value, weights, None, 3, out=good)


def test_weights_out_is_apart_from_all_that_is_read():
    memory = torch.zeros(4096, dtype=torch.int32)
    out = memory[8:28].view(torch.float32).view(2, 2, 5)
    _, q, k, lse = weigh()
    w = torch.zeros(2, 2, 5)
    halves = memory.view(BF16)
    for bad in (dict(query=halves[:q.numel()].view(q.shape)), dict(key=halves[48:48 + k.numel()].view(k.shape)),
                dict(lse=memory[:24].view(torch.float32).view(2, 3, 4)), dict(key_lengths=memory[27:29])):
        with pytest.raises(ValueError, match="out must"):
            cache.accumulate_weights(**{**dict(weights=w, query=q, key=k, lse=lse, out=out), **bad})
    # Behind and before them; lengths of 64 bits, which are copied first.
    for lengths in (memory[6:8], memory[26:30].view(torch.int64)):
        with pytest.raises(ValueError, match="GPU"):
            cache.accumulate_weights(w, halves[56:56 + q.numel()].view(q.shape), k, lse, out=out, key_lengths=lengths)


def test_outputs_of_an_eviction_are_memory_of_their_own():
    """Of each other's, of the inputs', and of nothing that only lies between their rows."""
    key, value, weights, _ = caches()
    buffer = torch.zeros(2 * 40 * 2 * 64, dtype=BF16)
    rows = buffer.view(2, 40, 2, 64)
    other = lambda: torch.zeros(2, 4, 2, 64, dtype=BF16)  # noqa: E731
    sums = lambda: torch.zeros(2, 2, 4)  # noqa: E731
    shared = torch.zeros(4096, dtype=torch.int32)
    as_floats, as_rows = shared[:16].view(torch.float32).view(2, 2, 4), shared[:512].view(BF16).view(2, 4, 2, 64)
    for bad in ([rows[:, :4], rows[:, 3:7], sums()], [rows[:, 3:7], rows[:, :4], sums()], [rows[:, :4], rows[:, 1:5], sums()],
                [rows[:, 0:8:2], rows[:, 2:10:2], sums()], [rows[:, 0:8:2], rows[:, 0:4], sums()],
                # Keys and values with their tokens and heads the other way round, in one place.
                [buffer[:1024].view(2, 4, 2, 64), buffer[:1024].view(2, 2, 4, 64).transpose(1, 2), sums()],
                [as_rows, other(), as_floats], [other(), as_rows, as_floats]):
        with pytest.raises(ValueError, match="out"):
            cache.evict(key, value, weights, None, 3, out=bad)
    lengths = torch.zeros(18, dtype=torch.int32)
    with pytest.raises(ValueError, match="out"):
        cache.evict(key, value, weights, lengths[15:17], 3, out=[other(), other(), lengths[:16].view(torch.float32).view(2, 2, 4)])
    inside = rows[:, 5:10], rows[:, 20:25]
    for bad in ([rows[:, 9:13], other(), sums()], [other(), rows[:, 17:21], sums()]):
        with pytest.raises(ValueError, match="out"):
            cache.evict(*inside, weights, None, 3, out=bad)
    # Rows between each other's, and between those of the inputs.
    halves = torch.zeros(2, 16 * 64, dtype=BF16)
    heads_outside = halves[:, 8 * 64:].view(2, 2, 4, 64).transpose(1, 2)
    for good in ([rows[:, 10:18:2], rows[:, 11:19:2], sums()], [rows[:, 10:14], rows[:, 25:29], sums()], [rows[:, 30:34], rows[:, 34:38], sums()],
                 [halves[:, :8 * 64].view(2, 4, 2, 64), heads_outside, sums()]):
        with pytest.raises(ValueError, match="GPU"):
            cache.evict(*inside, weights, None, 3, out=good)


@pytest.mark.parametrize("seed", range(40))
def test_overlap(seed):
    """Whether two strided tensors share memory, against the sets of their bytes."""
    g = random.Random(seed)
    memory = torch.zeros(600, dtype=torch.int16)

    def some():
        dtype = g.choice([torch.int16, torch.float32])
        base = memory.view(dtype)
        if g.random() < 0.5:   # a slice with its dimensions in any order
            shape = [g.randint(1, 5) for _ in range(3)]
            at = g.randint(0, 20)
            t = base[at:at + shape[0] * shape[1] * shape[2]].view(shape).permute(*g.sample(range(3), 3))
            return t[::g.randint(1, 3), g.randint(0, t.shape[1] - 1):]
        shape, stride = [g.randint(0, 4) for _ in range(3)], [g.randint(0, 30) for _ in range(3)]
        return base.as_strided(shape, stride, g.randint(0, 20))

    def places(t):
        first, size = (t.data_ptr() - memory.data_ptr()), t.element_size()
        return {first + size * sum(i * st for i, st in zip(at, t.stride())) + b
                for at in itertools.product(*(range(n) for n in t.shape)) for b in range(size)}

    for _ in range(20):
        a, b = some(), some()
        assert cache._clash((a,), (b,)) == bool(places(a) & places(b)), (a.shape, a.stride(), b.shape, b.stride())


def test_entry_point_refusals_without_a_gpu():
    lib, p, kept = _lib.load(), 4096, []
    one = struct.unpack("i", struct.pack("f", 1.0))[0]

    def numbers(values, at=0, value=None):
        s = array("q", values)
        if value is not None:
            s[at] = value
        kept.append(s)
        return s.buffer_info()[0]

    six = (256, 64, 1024, 128, 64, 640)
    good = dict(q=p, k=p, lse=p, w=p, out=p, dtype=0, n=1, qr=4, kr=4, heads=4, kv=2, dim=64, st=numbers(six), lens=None,
                causal=0, scale=one, ws=None, wsb=0, stream=None)
    call = lambda **kw: lib.lr_attention_weights(*{**good, **kw}.values())  # noqa: E731
    assert call(n=0) == _lib.LR_OK and call(kr=0) == _lib.LR_OK
    assert call(dim=96) == _lib.LR_EUNSUPPORTED
    for bad in [dict(dtype=2), dict(heads=3), dict(kv=0), dict(q=None), dict(k=None), dict(lse=None), dict(w=None),
                dict(out=None), dict(q=p + 8), dict(k=p + 2), dict(lse=p + 2), dict(out=p + 1), dict(st=None),
                dict(st=numbers(six, 0, 252)), dict(st=numbers(six, 0, 1 << 23)), dict(st=numbers(six, 1, 1 << 29)),
                dict(st=numbers(six, 3, 1 << 23)), dict(st=numbers(six, 5, -640)), dict(n=-1), dict(kr=1 << 30),
                dict(n=1 << 24), dict(qr=1 << 29), dict(scale=0), dict(qr=4096, ws=None), dict(qr=4096, ws=p, wsb=8)]:
        assert call(**bad) == _lib.LR_EINVAL, bad
    out = array("q", [0])
    size = lambda *shape: lib.lr_attention_weights_workspace(*shape, out.buffer_info()[0])  # noqa: E731
    assert size(1, 4096, 64, 8, 8, 128) == _lib.LR_OK and out[0] > 0
    assert size(64, 1, 8192, 40, 8, 128) == _lib.LR_OK and out[0] == 0
    assert size(1, 1, 1, 3, 2, 64) == _lib.LR_EINVAL

    size = lambda *shape: lib.lr_cache_evict_workspace(*shape, out.buffer_info()[0])  # noqa: E731
    assert size(4, 16384, 8) == _lib.LR_OK and out[0] == 0
    assert size(4, 16385, 8) == _lib.LR_OK and out[0] == 4 * 8 * 2 * (3 * 2048 * 4 + 16)
    assert size(1 << 24, 1, 8) == _lib.LR_EINVAL and size(1, 1, 0) == _lib.LR_EINVAL

    twelve = (256, 128, 1280) * 4
    good = dict(k=p, v=p, w=p, lens=None, ko=p, vo=p, wo=p, lo=p, kept=p, n=1, size=5, heads=2, row=128, budget=3, recent=1,
                capacity=3, st=numbers(twelve), clear=1, ws=None, wsb=0, stream=None)
    call = lambda **kw: lib.lr_cache_evict(*{**good, **kw}.values())  # noqa: E731
    assert call(n=0) == _lib.LR_OK
    for bad in [dict(k=None), dict(w=None), dict(ko=None), dict(kept=None), dict(lo=None), dict(k=p + 8), dict(vo=p + 2),
                dict(w=p + 1), dict(row=120), dict(row=0), dict(heads=0), dict(budget=0), dict(recent=4), dict(recent=-1),
                dict(capacity=2), dict(n=-1), dict(n=1 << 24), dict(size=1 << 30), dict(budget=1 << 29, capacity=1 << 29),
                dict(st=None), dict(st=numbers(twelve, 3, 136)), dict(st=numbers(twelve, 11, -16)), dict(size=16385),
                dict(size=16385, ws=p, wsb=8)]:
        assert call(**bad) == _lib.LR_EINVAL, bad
