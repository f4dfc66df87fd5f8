"""GPU parity of the MXFP4 quantizer (exact) and of the product of MXFP4 rows.

Product: the terms are exact in fp32, so a sum of K of them is off by at most
K * 2^-24 * sum |a w| for correctly rounded additions; the matrix unit aligns
and truncates inside a step, at most one more unit in the last place per
addition: 2 * K * 2^-24 in all. The result is rounded to bf16 once (2^-8).
"""

import numpy as np
import pytest
import torch

import mxfp4_ref as ref
from lynnreal_omni_amd import _lib, kernels, mxfp4, mxfp4_gemm
from test_mxfp4_host import hard_rows, rows

pytestmark = pytest.mark.gpu


def check_rows(x):
    """x: a float tensor on the GPU; codes, scales and values against the definition."""
    code, byte, value = ref.quantize(x.float().cpu().numpy())
    codes, scales = kernels.quantize_rows_mxfp4(x)
    assert np.array_equal(codes.cpu().numpy(), ref.pack(code))
    assert np.array_equal(mxfp4_gemm.untile_scales(scales, *byte.shape).cpu().numpy(), byte)
    for dtype in (torch.float32, torch.bfloat16):
        back = kernels.dequantize_rows_mxfp4(codes, scales, x.shape[1], dtype)
        assert back.dtype == dtype and np.array_equal(back.double().cpu().numpy(), value, equal_nan=True)
    back = kernels.dequantize_rows_mxfp4(codes, scales, x.shape[1], torch.float16)
    with np.errstate(over="ignore"):
        want = value.astype(np.float16)
    assert np.array_equal(back.cpu().numpy(), want, equal_nan=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,k", [(1, 1), (1, 32), (3, 31), (17, 33), (64, 256), (65, 257), (130, 520), (1, 5376),
                                 (33, 1000), (5, 8), (200, 264)])
def test_quantizer(n, k, dtype):
    check_rows((rows(n, k, n + k) * 2.0 ** -4).to(dtype).cuda())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantizer_hard_rows(dtype):
    check_rows(hard_rows().to(dtype).cuda())


def test_quantizer_many_rows():
    """The 64-row form (many tiles) with rows and columns past the last tile, and a strided input."""
    x = rows(4097, 5376 + 8, 3).bfloat16().cuda()
    check_rows(x)
    check_rows(x[:, 3:1003])


def test_quantizer_leaves_the_rest_alone():
    x = rows(17, 96, 5).bfloat16().cuda()
    codes = torch.full((17 * 48 + 64,), 7, dtype=torch.uint8, device="cuda")
    scales = torch.full((512 + 64,), 7, dtype=torch.uint8, device="cuda")
    _lib.launch(x, "lr_quantize_rows_mxfp4", x.data_ptr(), _lib.DTYPE_BF16, 17, 96, codes.data_ptr(), scales.data_ptr())
    assert (codes[17 * 48:] == 7).all() and (scales[512:] == 7).all()


def operands(m, n, k, seed, bias=True):
    x = rows(m, k, seed).bfloat16()
    x = (x / x.float().abs().amax(-1, keepdim=True)).bfloat16()
    w = rows(n, k, seed + 1)
    w = w / w.abs().amax(-1, keepdim=True)
    b = torch.randn(n, generator=torch.Generator().manual_seed(seed)).bfloat16() if bias else None
    return x, w, b


def product(x, w, b):
    xv, wv = ref.quantize(x.float().numpy())[2], ref.quantize(w.numpy())[2]
    y, size = xv @ wv.T, np.abs(xv) @ np.abs(wv).T
    if b is not None:
        y = y + b.double().numpy()
    return y, size


def check_product(got, y, size, k):
    bound = 2.0 ** -8 * np.abs(y) + (1 + 2.0 ** -8) * 2 * k * 2.0 ** -24 * size + 2.0 ** -24 * np.abs(y)
    off = np.abs(got.double().cpu().numpy() - y) - bound
    assert off.max(initial=-1) <= 0, f"off by {off.max()} past the bound"


SHAPES = [(1, 1, 1), (1, 8, 32), (1, 5376, 5376), (3, 17, 33), (15, 72, 96), (16, 64, 256), (17, 130, 257),
          (33, 264, 1000), (64, 256, 512), (65, 512, 513), (100, 7, 2048), (128, 128, 4096), (130, 272, 544),
          (257, 520, 768), (300, 1032, 1312), (520, 1288, 7168), (1000, 2056, 640)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("bias", [True, False])
def test_product(m, n, k, bias):
    x, w, b = operands(m, n, k, m + n + k, bias)
    y, size = product(x, w, b)
    codes, scale = mxfp4.quantize_weight(w)
    layer = mxfp4.Mxfp4Linear.from_packed(codes, scale, b, in_features=k).cuda()
    check_product(layer(x.cuda()), y, size, k)


# On 256 CUs: one round of 64 x 128 tiles (the last of an odd N), more than a round of
# ragged ones, and the ping-pong kernel's tiles from 64 x 128 to 256 x 256, with odd and
# even numbers of k-steps.
TILES = [(100, 8200, 768), (200, 5128, 300), (65, 16001, 96), (256, 5120, 1280), (1000, 4104, 800), (700, 6001, 64),
         (38, 37800, 256), (402, 22672, 768), (500, 4104, 768), (1000, 4104, 512), (2000, 4104, 768),
         (2000, 5128, 256), (2000, 6152, 768)]


@pytest.mark.parametrize("m,n,k", TILES)
def test_product_of_every_tile(m, n, k):
    test_product(m, n, k, True)


def _table(n, rows_, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(rows_, 6 * n, generator=g).bfloat16().cuda()


@pytest.mark.parametrize("m,n,k", [(1, 64, 64), (5, 33, 96), (64, 264, 256), (130, 136, 512), (300, 520, 1024),
                                   (1000, 1032, 512)])
def test_epilogues_are_the_separate_kernels(m, n, k):
    x, w, b = operands(m, n, k, m + n, True)
    layer = mxfp4.Mxfp4Linear.from_packed(*mxfp4.quantize_weight(w), b, in_features=k).cuda()
    x = x.cuda()[None]
    y = layer(x)
    assert torch.equal(layer(x, activation="gelu_tanh"), kernels.gelu_tanh(y))
    residual = rows(m, n, 9).bfloat16().cuda()[None]
    table, indices = _table(n, 3, m), torch.randint(-1, 4, (m,), generator=torch.Generator().manual_seed(m)).cuda()
    got = layer(x, residual=residual, table=table, indices=indices, gate_slot=5)
    assert torch.equal(got, kernels._gated_residual(residual, y, table, indices, 5))
    # a batch of two sequences shares the indices
    two, again = torch.cat([x, x.flip(1)]), torch.cat([residual, residual])
    got = layer(two, residual=again, table=table, indices=indices, gate_slot=0)
    assert torch.equal(got, kernels._gated_residual(again, layer(two), table, indices, 0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,k", [(64, 64), (33, 96), (520, 8), (5120, 264), (264, 5376), (17000, 2056), (48, 12288),
                                 (40, 12296), (17000, 6144), (17000, 6152), (35000, 256), (100, 36)])
def test_one_row_is_the_two_kernels(n, k, dtype):
    """A layer's single row is quantized inside the product: the bits of the quantizer
    and the product one after the other, for every epilogue."""
    g = torch.Generator(device="cuda").manual_seed(n + k)
    x = (torch.randn(1, k, device="cuda", generator=g) * 10 ** torch.linspace(-6, 4, k, device="cuda")).to(dtype)
    w = torch.randn(n, k, device="cuda", generator=g)
    layer = mxfp4.Mxfp4Linear.from_packed(*mxfp4.quantize_weight(w), torch.randn(n, device="cuda", generator=g).bfloat16(), k)
    table = torch.randn(3, 2 * n, device="cuda", generator=g).bfloat16()
    gated = dict(residual=torch.randn(1, 1, n, device="cuda", generator=g).bfloat16(), table=table,
                 indices=torch.tensor([2], device="cuda"), gate_slot=1)
    for epilogue in ({}, {"activation": "gelu_tanh"}, gated):
        want = layer.forward_codes(*kernels.quantize_rows_mxfp4(x), (1,), **epilogue)
        assert torch.equal(layer(x, **epilogue), want)
    x[0, k // 2] = float("nan")
    assert layer(x).isnan().all()
    x[0, k // 2] = 0
    x[0, :min(k, 40)] = 0
    want = layer.forward_codes(*kernels.quantize_rows_mxfp4(x), (1,))
    assert torch.equal(layer(x), want)
    # A row of a wider tensor, and one that is not 16-byte aligned.
    wide = torch.zeros(1, k + 1, device="cuda", dtype=dtype)
    wide[:, 1:] = x
    assert torch.equal(layer(wide[:, 1:]), want)


def test_nan_blocks_reach_their_row_alone():
    x, w, b = operands(70, 136, 256, 4)
    layer = mxfp4.Mxfp4Linear.from_packed(*mxfp4.quantize_weight(w), b).cuda()
    clean = layer(x.cuda())
    x[3, 40], x[69, 255] = float("nan"), float("inf")
    got = layer(x.cuda())
    bad = torch.zeros(70, dtype=torch.bool)
    bad[[3, 69]] = True
    assert got[bad].isnan().all() and torch.equal(got[~bad], clean[~bad])


def test_layer_from_linear_and_transformer_rules():
    source = torch.nn.Linear(96, 40).bfloat16().cuda()
    x, _, _ = operands(9, 1, 96, 2)
    layer = mxfp4.Mxfp4Linear(source)
    y, size = product(x, source.weight.detach().float().cpu(), source.bias.detach().cpu())
    check_product(layer(x.cuda()), y, size, 96)
    assert layer.weight.dtype == torch.bfloat16


def test_streams_and_graphs():
    """Work on another stream; two captured calls replayed between eager ones."""
    x, w, b = operands(40, 264, 1024, 1)
    layer = mxfp4.Mxfp4Linear.from_packed(*mxfp4.quantize_weight(w), b).cuda()
    xs = [x.cuda(), x.flip(0).contiguous().cuda()]
    want = [layer(v) for v in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer(xs[0])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want[0])
    graphs, outs, ins = [], [], [v.clone() for v in xs]
    for v in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer(v))
        graphs.append(g)
    for turn in range(3):
        ins[0].copy_(xs[turn % 2])
        ins[1].copy_(xs[1 - turn % 2])
        for g in graphs:
            g.replay()
        layer(xs[0])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[turn % 2]) and torch.equal(outs[1], want[1 - turn % 2])


def test_offsets_past_32_bits():
    """Output and code offsets past 2^31: the last rows are right."""
    m, n, k = 70000, 32768, 64
    g = torch.Generator().manual_seed(0)
    w = torch.randn(n, k, generator=g)
    layer = mxfp4.Mxfp4Linear.from_packed(*mxfp4.quantize_weight(w)).cuda()
    x = torch.randn(m, k, generator=g).bfloat16().cuda()
    y = layer(x)
    assert torch.equal(y[-130:], layer(x[-130:].contiguous()))


def test_indices_past_the_table_are_clamped():
    """As in every epilogue that reads the table."""
    x, w, _ = operands(8, 64, 64, 3, False)
    layer = mxfp4.Mxfp4Linear.from_packed(*mxfp4.quantize_weight(w)).cuda()
    residual, table = rows(8, 64, 1).bfloat16().cuda(), _table(64, 1, 2)
    a = layer(x.cuda(), residual=residual, table=table, indices=torch.full((8,), 99, device="cuda"), gate_slot=1)
    b = layer(x.cuda(), residual=residual, table=table, indices=torch.zeros(8, dtype=torch.int64, device="cuda"),
              gate_slot=1)
    assert torch.equal(a, b)
