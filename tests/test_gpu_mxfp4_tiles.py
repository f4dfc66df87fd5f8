"""Every kernel of the MXFP4 product, named by its grid: the fused epilogues are the
separate kernels bit for bit, NaN blocks reach their row or column alone, and offsets
past 32 bits are right."""
import pytest
import torch

from graph_nodes import kernels as launched
from lynnreal_omni_amd import kernels, mxfp4
from lynnreal_omni_amd.mxfp4_gemm import tile_scales, untile_scales

pytestmark = pytest.mark.gpu

CUS = 256       # the compute units that the shapes below are chosen for

# (m, n, k): rows and columns of the workgroup's outputs, and its threads. Ragged in m and
# n, odd and even numbers of k-steps; the last ones are not whole k-steps or whole chunks.
# 512 threads: the ping-pong kernel, or with 64 x 128 tiles of one round the ring of five.
TILES = [
    ((12, 4104, 768), (16, 32), 128), ((12, 20488, 512), (16, 32), 64),
    ((130, 1032, 768), (32, 32), 128), ((90, 8200, 512), (32, 32), 64),
    ((100, 8200, 768), (64, 128), 512), ((1000, 1096, 512), (64, 128), 512),
    ((38, 37800, 256), (64, 128), 512), ((38, 37800, 768), (64, 128), 512),
    ((500, 4104, 768), (128, 128), 512), ((1000, 4104, 512), (128, 256), 512),
    ((2000, 4104, 768), (160, 256), 512), ((2000, 5128, 256), (192, 256), 512),
    ((402, 22672, 768), (256, 256), 512), ((2000, 6152, 1280), (256, 256), 512),
    ((1000, 4104, 800), (128, 128), 256), ((1002, 4099, 512), (128, 128), 256),
    ((700, 6001, 64), (128, 128), 256), ((200, 5125, 300), (64, 128), 512),
]


def _layer(n, k, seed):
    """A layer of random codes and scales near one, and rows of the same kind."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    blocks = -(-k // 32)
    codes = torch.randint(0, 256, (n, blocks * 16), device="cuda", dtype=torch.uint8, generator=g)
    scale = torch.randint(118, 123, (n, blocks), device="cuda", dtype=torch.uint8, generator=g)
    bias = torch.randn(n, device="cuda", generator=g).bfloat16()
    return g, mxfp4.Mxfp4Linear.from_packed(codes, scale, bias, in_features=k)


def _check_kernel(call, m, n, tile, threads):
    blocks = -(-m // tile[0]) * -(-n // tile[1])
    assert launched(call)[-1] == (blocks, threads)


@pytest.fixture(autouse=True, scope="module")
def _device():
    if torch.cuda.get_device_properties(0).multi_processor_count != CUS:
        pytest.skip("the shapes are chosen for 256 compute units")


@pytest.mark.parametrize("shape,tile,threads", TILES)
def test_fused_epilogues(shape, tile, threads):
    m, n, k = shape
    g, layer = _layer(n, k, m + n + k)
    x = torch.randn(m, k, device="cuda", generator=g).bfloat16()
    y = layer(x)
    _check_kernel(lambda: layer(x), m, n, tile, threads)
    assert y.isfinite().all()
    gelu = layer(x, activation="gelu_tanh")
    _check_kernel(lambda: layer(x, activation="gelu_tanh"), m, n, tile, threads)
    assert torch.equal(gelu, kernels.gelu_tanh(y))
    table = torch.randn(3, 6 * n, device="cuda", generator=g).bfloat16()
    # One sequence, and two that share the indices (some of which are clamped to the table).
    for batch in (1, 2):
        rows = m // batch
        residual = torch.randn(batch, rows, n, device="cuda", generator=g).bfloat16()
        indices = torch.randint(-1, 4, (rows,), device="cuda", generator=g)
        given = dict(residual=residual, table=table, indices=indices, gate_slot=3 + batch)
        value = x.view(batch, rows, k)
        got = layer(value, **given)
        _check_kernel(lambda: layer(value, **given), m, n, tile, threads)
        assert torch.equal(got, kernels._gated_residual(residual, y.view(batch, rows, n), table, indices, 3 + batch))


@pytest.mark.parametrize("shape,tile,threads", TILES)
def test_nan_blocks(shape, tile, threads):
    """A NaN in a block of a row, or the byte 255 of a weight's block: that row, that column."""
    m, n, k = shape
    g, layer = _layer(n, k, m + n)
    x = torch.randn(m, k, device="cuda", generator=g).bfloat16()
    clean = layer(x)
    rows, columns = torch.zeros(m, dtype=torch.bool, device="cuda"), torch.zeros(n, dtype=torch.bool, device="cuda")
    rows[[0, m // 2, m - 1]] = True
    columns[[1, n // 2, n - 1]] = True
    x[0, 0], x[m // 2, k // 2], x[m - 1, k - 1] = float("nan"), float("inf"), -float("inf")
    scale = untile_scales(layer.weight_scale, n, -(-k // 32))
    scale[1, 0], scale[n // 2, scale.shape[1] // 2], scale[n - 1, -1] = 255, 255, 255
    layer.weight_scale.copy_(tile_scales(scale))
    got = layer(x)
    bad = rows[:, None] | columns[None]
    assert got[bad].isnan().all() and torch.equal(got[~bad], clean[~bad])
    gelu = layer(x, activation="gelu_tanh")
    assert gelu[bad].isnan().all() and gelu[~bad].isfinite().all()


def _exact(rows, k, seed):
    """Codes of whole and half numbers with the scale one: a sum of k products of two is a
    whole number of quarters below 2^24, exact in fp32 in whatever order."""
    assert 36 * 4 * k < 1 << 24
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (rows, k // 2), device="cuda", dtype=torch.uint8, generator=g)
    return codes, torch.full((rows, k // 32), 127, device="cuda", dtype=torch.uint8)


@pytest.mark.parametrize("m,tile", [(40, (64, 128)), (300, (160, 256))])
def test_weights_past_2_31_bytes(m, tile):
    """Weights whose last rows lie past 2^31 bytes of codes."""
    n, k = 70000, 65536
    layer = mxfp4.Mxfp4Linear.from_packed(*_exact(n, k, 1))
    assert layer.weight_codes.numel() > 1 << 31
    x = mxfp4.Mxfp4Linear.from_packed(*_exact(m, k, 2))     # codes and scales of the rows
    got = layer.forward_codes(x.weight_codes, x.weight_scale, (m,))
    _check_kernel(lambda: layer.forward_codes(x.weight_codes, x.weight_scale, (m,)), m, n, tile, 512)
    for first in (0, 65472, 69952):      # multiples of 64: whole scale tiles
        last = min(first + 64, n)
        part = mxfp4.Mxfp4Linear.from_packed(layer.weight_codes[first:last].clone(),
                                             torch.full((last - first, k // 32), 127, device="cuda", dtype=torch.uint8))
        assert torch.equal(got[:, first:last], part.forward_codes(x.weight_codes, x.weight_scale, (m,)))


def test_rows_past_2_31_bytes():
    """The same of the rows: a layer's quantizer and product with codes past 2^31 bytes."""
    m, n, k = 70000, 264, 65536
    layer = mxfp4.Mxfp4Linear.from_packed(*_exact(n, k, 3))
    x = torch.zeros(m, k, device="cuda", dtype=torch.bfloat16)
    g = torch.Generator(device="cuda").manual_seed(4)
    for at in (0, 65530, 69990):         # whole numbers of four bits, 4 in every block
        x[at:at + 10] = torch.randint(-4, 5, (10, k), device="cuda", generator=g).bfloat16()
        x[at:at + 10, ::32] = 4
    got = layer(x)
    for at in (0, 65530, 69990):
        part = layer(x[at:at + 10].clone())
        assert part.any() and torch.equal(got[at:at + 10], part)
    assert not got[10:65530].any() and not got[65540:69990].any()


@pytest.mark.parametrize("epilogue", ["none", "gelu", "gated"])
def test_outputs_past_2_31_elements(epilogue):
    """Outputs and residual past 2^31 elements in the ping-pong kernel."""
    m, n, k = 66000, 32776, 256
    assert m * n > 1 << 31
    layer = mxfp4.Mxfp4Linear.from_packed(*_exact(n, k, 5))
    x = torch.randint(-4, 5, (m, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(6)).bfloat16()
    x[:, ::32] = 4
    given = {}
    if epilogue == "gelu":
        given = dict(activation="gelu_tanh")
    elif epilogue == "gated":
        residual = torch.randn(m, 1, device="cuda", generator=torch.Generator(device="cuda").manual_seed(7))
        given = dict(residual=residual.bfloat16().expand(m, n).contiguous(), gate_slot=0,
                     table=torch.ones(1, n, device="cuda", dtype=torch.bfloat16),
                     indices=torch.zeros(m, device="cuda", dtype=torch.int64))
    got = layer(x, **given)
    _check_kernel(lambda: layer(x, **given), m, n, (256, 256), 512)
    for at in (0, 65500, m - 130):
        if epilogue == "gated":
            given["residual"], given["indices"] = residual[at:at + 130].bfloat16().expand(130, n), torch.zeros(
                130, device="cuda", dtype=torch.int64)
        assert torch.equal(got[at:at + 130], layer(x[at:at + 130].clone(), **given))
