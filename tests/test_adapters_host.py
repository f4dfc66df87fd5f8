"""What the adapters of many requests refuse, and how they hold their weights, on the CPU."""
from array import array

import pytest
import torch
from torch import nn

from lynnreal_omni_amd import _lib, adapters as L, int8

BF16 = torch.bfloat16


def some(count=3, rank=4, k=24, n=40, dtype=BF16, scale=1.0):
    return L.LowRankAdapters(torch.ones(count, rank, k, dtype=dtype), torch.ones(count, n, rank, dtype=dtype), scale)


class Plan:
    def __init__(self, tokens=5, adapters=3):
        self.tokens, self.adapters, self.order = tokens, adapters, torch.zeros(tokens, dtype=torch.int32)


def test_weights_are_filled_up_with_zeros():
    a = some(rank=5, k=13, n=7, scale=torch.tensor([1.0, 2.0, 3.0], dtype=torch.float64))
    assert a.down.shape == (3, 5, 16) and a.up.shape == (3, 7, 8) and len(a) == 3
    assert (a.down[..., :13] == 1).all() and (a.down[..., 13:] == 0).all() and (a.up[..., 5:] == 0).all()
    assert a.scale.tolist() == [1.0, 2.0, 3.0] and a.scale.dtype == torch.float32
    assert some(scale=0.5).scale.tolist() == [0.5] * 3
    assert set(dict(a.named_buffers())) == {"down", "up", "scale"}


@pytest.mark.parametrize("down,up", [
    (torch.zeros(2, 4, 8), torch.zeros(3, 8, 4)), (torch.zeros(2, 4, 8), torch.zeros(2, 4, 8)),
    (torch.zeros(4, 8), torch.zeros(8, 4)), (torch.zeros(2, 4, 8), torch.zeros(2, 8, 4, dtype=BF16)),
    (torch.zeros(2, 4, 0, dtype=BF16), torch.zeros(2, 8, 4, dtype=BF16)),
    (torch.zeros(0, 4, 8, dtype=BF16), torch.zeros(0, 8, 4, dtype=BF16))])
def test_wrong_adapters(down, up):
    with pytest.raises(ValueError):
        L.LowRankAdapters(down, up)


def test_wrong_scales():
    for scale in (torch.ones(2), torch.ones(1, 3)):
        with pytest.raises(ValueError, match="scale"):
            some(scale=scale)


def test_not_supported():
    for kwargs in (dict(dtype=torch.float32), dict(rank=129), dict(count=1001, rank=1, k=8, n=8)):
        with pytest.raises(RuntimeError, match="not supported"):
            some(**kwargs)


@pytest.mark.parametrize("indices,count", [(torch.zeros(5), 3), (torch.zeros(5, dtype=torch.int32), 0),
                                           (torch.zeros(5, dtype=torch.int32), 1001), (torch.zeros(5, dtype=torch.int16), 3),
                                           (torch.zeros(5, dtype=torch.int32), 3)])
def test_plans(indices, count):
    with pytest.raises(ValueError):     # the last: right, but not on a GPU
        L.AdapterPlan(indices, count)


@pytest.mark.parametrize("x,base,plan,match", [
    ((5, 23), (5, 40), Plan(), "expected x"), ((5, 24), (5, 41), Plan(), "expected x"), ((5, 24), (1, 5, 40), Plan(), "expected"),
    ((5, 24), (5, 40), Plan(6), "plan"), ((5, 24), (5, 40), Plan(5, 2), "plan"), ((5, 24), (5, 40), Plan(), "GPU"),
    ((5, 1, 24), (5, 1, 40), Plan(), "GPU")])
def test_wrong_calls(x, base, plan, match):
    with pytest.raises(ValueError, match=match):
        some()(torch.zeros(x, dtype=BF16), torch.zeros(base, dtype=BF16), plan)


def test_dtypes_and_gradients():
    x, base = torch.zeros(5, 24, dtype=BF16), torch.zeros(5, 40, dtype=BF16)
    for bad in ((x.float(), base), (x, base.half())):
        with pytest.raises(ValueError, match="dtype"):
            some()(*bad, Plan())
    for bad in ((x.clone().requires_grad_(), base), (x, base.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="gradients are not supported"):
            some()(*bad, Plan())
    # A module moved to other types.
    with pytest.raises(RuntimeError, match="not supported"):
        some().float()(x.float(), base.float(), Plan())
    with pytest.raises(ValueError, match="scale float32"):
        some().bfloat16()(x, base, Plan())


def test_out_is_base_or_other_memory():
    memory = torch.zeros(400, dtype=BF16)
    x, base = torch.zeros(5, 24, dtype=BF16), memory[:200].view(5, 40)
    for out in (memory[8:208].view(5, 40), torch.zeros(5, 41, dtype=BF16)[:, :40], torch.zeros(5, 40), memory[:160].view(4, 40)):
        with pytest.raises(ValueError, match="out must"):
            some()(x, base, Plan(), out=out)
    with pytest.raises(ValueError, match="out must"):
        some()(memory[100:220].view(5, 24), torch.zeros(5, 40, dtype=BF16), Plan(), out=base)
    for out in (base, memory[200:].view(5, 40)):
        with pytest.raises(ValueError, match="GPU"):
            some()(x, base, Plan(), out=out)


def test_rows_are_read_as_they_are_where_they_can():
    wide = torch.zeros(9, 64, dtype=BF16)
    copies = lambda t: L._copies(t.shape[1], t.stride(0), t.data_ptr() & 15)  # noqa: E731
    assert not copies(wide) and not copies(wide[:, 8:32]) and not copies(wide[::2]) and not copies(wide[3:4, :24])
    assert not copies(wide[:1].expand(9, -1))
    assert copies(wide[:, 4:36]) and copies(wide[:, :60]) and copies(torch.zeros(9, 65, dtype=BF16)[:, :64])
    assert copies(torch.zeros(100, dtype=BF16).as_strided((5, 64), (8, 1)))
    assert L._copies(64, 1 << 30, 0) and not L._copies(64, (1 << 30) - 8, 0)


def test_adapted_transformer():
    """Names are checked before any layer is changed; without a plan a layer is the layer."""
    model = nn.Sequential(nn.Linear(24, 40, dtype=BF16), nn.ModuleDict({"out": nn.Linear(40, 24, dtype=BF16)}))
    x = torch.randn(5, 24, dtype=BF16)
    want = model[0](x)
    with pytest.raises(ValueError, match="maps"):
        L.adapt_transformer(model, {"0": some(), "1.out": some()})
    with pytest.raises(AttributeError):
        L.adapt_transformer(model, {"0": some(), "2": some()})
    assert type(model[0]) is nn.Linear
    requests = L.adapt_transformer(model, {"0": some(), "1.out": some(k=40, n=24)})
    assert isinstance(model[0], L.AdaptedLinear) and isinstance(model[1]["out"], L.AdaptedLinear)
    assert model[0].requests is requests and model[1]["out"].requests is requests
    assert torch.equal(model[0](x), want)
    assert model[0].weight is model[0].layer.weight and model[0].bias is model[0].layer.bias
    requests.plan = Plan()
    with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
        model[0](x)
    with pytest.raises(ValueError, match="already"):
        L.adapt_transformer(model, {"0": some()})


class Beside:
    """Stands for the adapters of a layer: adds one, where it is told to, and remembers where that was."""
    in_features, out_features = 24, 40

    def __call__(self, x, base, plan, out=None):
        self.out = out
        return out.copy_(base + 1) if out is not None else base + 1


def adapted(layer):
    beside, requests = Beside(), L.Requests(Plan())
    return L.AdaptedLinear(layer, beside, requests), beside


@torch.no_grad()
def test_products_go_into_memory_of_the_layer_alone():
    """What a hook keeps of the layer's result stays as it was, and so does a buffer that it puts in its place."""
    x = torch.randn(5, 24, dtype=BF16)
    layer = nn.Linear(24, 40, dtype=BF16)
    want = layer(x)
    model, beside = adapted(layer)
    assert torch.equal(model(x), want + 1) and beside.out is not None
    seen = []
    handle = layer.register_forward_hook(lambda m, args, y: seen.append(y))
    assert torch.equal(model(x), want + 1) and torch.equal(seen[0], want)
    handle.remove()
    buffer = torch.zeros(5, 40, dtype=BF16)
    handle = layer.register_forward_hook(lambda m, args, y: buffer)
    assert torch.equal(model(x), torch.ones(5, 40, dtype=BF16)) and not buffer.any()
    handle.remove()
    seen.clear()
    handle = nn.modules.module.register_module_forward_hook(lambda m, args, y: seen.append((m, y)))
    try:
        got = model(x)
    finally:
        handle.remove()
    assert torch.equal(got, want + 1) and torch.equal(next(y for m, y in seen if m is layer), want)
    assert torch.equal(model(x), want + 1) and beside.out is not None   # no hook is left


@torch.no_grad()
def test_layers_that_keep_their_result():
    x = torch.randn(5, 24, dtype=BF16)

    class Keeps(nn.Linear):
        def forward(self, value):
            self.kept = super().forward(value)
            return self.kept

    layer = Keeps(24, 40, dtype=BF16)
    got = adapted(layer)[0](x)
    assert torch.equal(got, layer.kept + 1)
    # One whose rows are not next to each other.
    class Columns(nn.Linear):
        def forward(self, value):
            return super().forward(value).t().contiguous().t()

    layer = Columns(24, 40, dtype=BF16)
    assert torch.equal(adapted(layer)[0](x), layer(x) + 1)
    # A forward put in the place of the layer's own.
    layer, kept = nn.Linear(24, 40, dtype=BF16), torch.zeros(5, 40, dtype=BF16)
    layer.forward = lambda value: kept
    assert torch.equal(adapted(layer)[0](x), torch.ones(5, 40, dtype=BF16)) and not kept.any()


@torch.no_grad()
@pytest.mark.parametrize("wrapped", ["int8_matmul", "forward_quantized", "class"])
def test_products_of_replaced_functions_stay(wrapped, monkeypatch):
    """What a caller's own int8_matmul or forward_quantized has returned may be the caller's to keep."""
    x, kept = torch.randn(5, 24, dtype=BF16), torch.zeros(5, 40, dtype=BF16)
    layer = int8.Int8Linear(nn.Linear(24, 40, dtype=BF16), "hip")
    if wrapped == "int8_matmul":
        monkeypatch.setattr(int8.int8_gemm, "int8_matmul", lambda *args, **kwargs: kept)
    elif wrapped == "class":
        monkeypatch.setattr(int8.Int8Linear, "forward_quantized", lambda self, *args: kept)
    else:
        layer.forward_quantized = lambda *args: kept
    model, beside = adapted(layer)
    assert torch.equal(model(x), torch.ones(5, 40, dtype=BF16)) and not kept.any() and beside.out is None


def test_entry_point_refusals_without_a_gpu():
    lib, p = _lib.load(), 4096
    assert lib.lr_adapter_tiles(0, 3) == 0 and lib.lr_adapter_tiles(5, 1001) == 0 and lib.lr_adapter_tiles(-1, 3) == 0
    assert lib.lr_adapter_tiles(1, 8) == 1 and lib.lr_adapter_tiles(64, 8) == 10 and lib.lr_adapter_tiles(5, 8) == 5
    good = dict(index=p, tokens=5, adapters=3, order=p, tiles=p, stream=None)
    call = lambda **kw: lib.lr_adapter_plan(*{**good, **kw}.values())  # noqa: E731
    assert call(tokens=0) == _lib.LR_OK and call(adapters=1001) == _lib.LR_EUNSUPPORTED
    for bad in [dict(index=None), dict(order=None), dict(tiles=None), dict(tiles=p + 4), dict(index=p + 2), dict(tokens=-1),
                dict(tokens=1 << 24), dict(adapters=0)]:
        assert call(**bad) == _lib.LR_EINVAL, bad
    out = array("q", [0])
    size = lambda *shape: lib.lr_adapter_workspace(*shape, out.buffer_info()[0])  # noqa: E731
    assert size(0, 40, 24, 4, 3, 1) == _lib.LR_OK and out[0] == 0
    assert size(5, 40, 24, 129, 3, 0) == _lib.LR_EUNSUPPORTED and size(5, 0, 24, 4, 3, 0) == _lib.LR_EINVAL
    assert size(5, 40, 23, 4, 3, 0) == _lib.LR_OK and out[0] > 0
    plain = out[0]
    assert size(5, 40, 23, 4, 3, 1) == _lib.LR_OK and out[0] == plain + 5 * 24 * 2
    good = dict(x=p, xs=24, down=p, up=p, scale=p, base=p, bs=40, out=p, os=40, dtype=0, tokens=5, n=40, k=24, rank=4,
                adapters=3, order=p, tiles=p, ws=p, wsb=1 << 30, stream=None)
    call = lambda **kw: lib.lr_adapter_add(*{**good, **kw}.values())  # noqa: E731
    assert call(tokens=0) == _lib.LR_OK
    assert call(rank=129) == _lib.LR_EUNSUPPORTED and call(adapters=1001) == _lib.LR_EUNSUPPORTED
    for bad in [dict(x=None), dict(down=None), dict(up=None), dict(scale=None), dict(base=None), dict(out=None), dict(order=None),
                dict(tiles=None), dict(ws=None), dict(wsb=8), dict(x=p + 1), dict(up=p + 2), dict(base=p + 1), dict(tiles=p + 4),
                dict(xs=-8), dict(xs=25, wsb=plain), dict(xs=16, wsb=plain), dict(xs=1 << 30, wsb=plain),
                dict(x=p + 8, wsb=plain), dict(k=23, wsb=plain), dict(os=39), dict(bs=-8), dict(dtype=2), dict(tokens=-1),
                dict(tokens=1 << 24), dict(n=0), dict(n=1 << 24), dict(k=(1 << 23) + 8), dict(rank=0)]:
        assert call(**bad) == _lib.LR_EINVAL, bad


def test_entry_point_refuses_outputs_over_its_inputs():
    lib = _lib.load()
    at = lambda i, by=0: (i + 1 << 20) + by  # noqa: E731
    sizes = dict(down=3 * 4 * 24 * 2, up=3 * 40 * 8 * 2, scale=3 * 4, order=5 * 4, tiles=lib.lr_adapter_tiles(5, 3) * 16)
    good = dict(x=at(0), xs=24, down=at(1), up=at(2), scale=at(3), base=at(6), bs=40, out=at(7), os=40, dtype=0, tokens=5, n=40,
                k=24, rank=4, adapters=3, order=at(4), tiles=at(5), ws=None, wsb=0, stream=None)
    call = lambda **kw: lib.lr_adapter_add(*{**good, **kw}.values())  # noqa: E731
    error = lambda: lib.lr_last_error().decode()  # noqa: E731
    for name, size in sizes.items():
        first = good[name]
        for out in (first, first - 5 * 40 * 2 + 2, first + size - 2):
            assert call(out=out) == _lib.LR_EINVAL and "overlap" in error(), (name, out)
        # Behind and before it the call gets as far as the workspace, which is missing.
        for out in (first - 5 * 40 * 2, first + size):
            assert call(out=out) == _lib.LR_EINVAL and "workspace" in error(), (name, out)
