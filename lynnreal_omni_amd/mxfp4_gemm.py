"""Products of MXFP4 rows (4-bit codes with a power-of-two scale for each 32) on
gfx950's scaled MFMA: the 4-bit counterpart of int8_gemm.

Operands are what kernels.quantize_rows_mxfp4 returns for [rows, K] values:
codes uint8 [rows, 16 * ceil(K / 32)] and scales uint8 in tile order. The
weight is [N, K] like nn.Linear's, so mxfp4_matmul(a, w, ...) is a @ w.T.
Inference only: the outputs carry no gradient, and inputs that require one are
refused.
"""
from __future__ import annotations

import functools

import torch

from . import _lib
from .int8_gemm import _ROW_DTYPES

BLOCK = 32          # values that share a scale
_TILE_ROWS, _TILE_BLOCKS = 64, 8


def code_bytes(width: int) -> int:
    """Bytes of a row's codes."""
    return -(-width // BLOCK) * (BLOCK // 2)


@functools.lru_cache(maxsize=4096)
def scale_shape(rows: int, width: int) -> tuple[int, int, int]:
    """Shape of the tile-ordered scales of [rows, width] values."""
    return -(-rows // _TILE_ROWS), -(-width // (BLOCK * _TILE_BLOCKS)), _TILE_ROWS * _TILE_BLOCKS


def tile_scales(scales: torch.Tensor) -> torch.Tensor:
    """E8M0 bytes [rows, blocks] in the order of the kernels: tiles of 64 rows x 8
    blocks, in which the matrix instruction's lane 16 * (b % 4) + r % 16 finds the
    bytes of rows r, r + 16, .. and blocks b, b + 4 behind each other. Bytes of
    rows and blocks past the end are 0."""
    if scales.dim() != 2 or scales.dtype != torch.uint8:
        raise ValueError("scales must be uint8 [rows, blocks]")
    rows, blocks = scales.shape
    tiles_r, tiles_b = -(-rows // _TILE_ROWS), -(-blocks // _TILE_BLOCKS)
    full = scales.new_zeros(tiles_r * _TILE_ROWS, tiles_b * _TILE_BLOCKS)
    full[:rows, :blocks] = scales
    # row = 64 t + 16 f + r, block = 8 u + 4 h + g  ->  [t, u, g, r, f, h]
    full = full.view(tiles_r, 4, 16, tiles_b, 2, 4).permute(0, 3, 5, 2, 1, 4)
    return full.reshape(tiles_r, tiles_b, _TILE_ROWS * _TILE_BLOCKS)


def untile_scales(tiles: torch.Tensor, rows: int, blocks: int) -> torch.Tensor:
    """The inverse of tile_scales: E8M0 bytes [rows, blocks]."""
    if tiles.dtype != torch.uint8 or tuple(tiles.shape) != scale_shape(rows, blocks * BLOCK):
        raise ValueError(f"tiles must be uint8 {scale_shape(rows, blocks * BLOCK)}")
    full = tiles.view(*tiles.shape[:2], 4, 16, 4, 2).permute(0, 4, 3, 1, 5, 2)
    return full.reshape(tiles.shape[0] * _TILE_ROWS, tiles.shape[1] * _TILE_BLOCKS)[:rows, :blocks].contiguous()


def _operand(codes, scales, name):
    shape = codes.shape
    if (len(shape) == 2 and codes.dtype is torch.uint8 and scales.dtype is torch.uint8 and not shape[1] % 16
            and scales.shape == scale_shape(shape[0], 2 * shape[1]) and codes.is_contiguous()
            and scales.is_contiguous()):
        return
    if codes.dim() != 2 or codes.dtype != torch.uint8 or not codes.is_contiguous() or codes.shape[1] % 16:
        raise ValueError(f"{name} must be contiguous uint8 codes [rows, 16 * blocks]")
    if scales.dtype != torch.uint8 or tuple(scales.shape) != scale_shape(codes.shape[0], 2 * codes.shape[1]):
        raise ValueError(f"{name}_scale must be uint8 {scale_shape(codes.shape[0], 2 * codes.shape[1])}, "
                         f"got {scales.dtype} {tuple(scales.shape)}")
    raise ValueError(f"{name}_scale must be contiguous")


def _gated(m, n, residual, table, indices, gate_slot):
    """The gated residual's tensors as the kernel reads them (int8_matmul's rules)."""
    if table is None or indices is None or gate_slot is None:
        raise ValueError("a gated-residual epilogue needs table, indices and gate_slot")
    if residual.dtype != torch.bfloat16 or table.dtype != torch.bfloat16:
        raise ValueError("residual and table must be bfloat16")
    if residual.numel() != m * n:
        raise ValueError("residual must have M*N elements")
    sequence = residual.shape[-2] if residual.dim() >= 2 else 1
    indices = indices.reshape(-1).contiguous().to(torch.int64)
    if indices.numel() < sequence:
        raise ValueError("indices shorter than the sequence")
    return residual.reshape(m, n).contiguous(), table.contiguous(), indices, sequence


def _epilogue(m, n, activation, residual, table, indices, gate_slot):
    """(epilogue, residual, table, table rows, table width, indices, sequence, slot) of a call's keywords."""
    if residual is not None:
        if activation is not None:
            raise ValueError("activation and gated residual epilogues are exclusive")
        residual, table, indices, sequence = _gated(m, n, residual, table, indices, gate_slot)
        width = table.shape[-1]
        rows = table.numel() // width if width else 0
        return _lib.EPI_GATED_RESIDUAL, residual, table, rows, width, indices, sequence, int(gate_slot)
    if table is not None or indices is not None or gate_slot is not None:
        raise ValueError("table, indices and gate_slot belong to a gated residual: residual is missing")
    if activation is None:
        return _PLAIN
    if activation == "gelu_tanh":
        return _GELU
    raise ValueError(f"unsupported activation {activation!r}")


_PLAIN = (_lib.EPI_BF16, None, None, 0, 0, None, 0, 0)
_GELU = (_lib.EPI_GELU_TANH, None, None, 0, 0, None, 0, 0)


def _no_gradient(*tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("gradients are not supported by the MXFP4 product: call it under torch.no_grad()")


def _bias(bias, n):
    if bias is None:
        return None
    if bias.dtype != torch.bfloat16 or bias.numel() != n:
        raise ValueError("bias must be bfloat16 with N entries")
    return bias.contiguous()


def mxfp4_matmul(a, b, a_scale, b_scale, bias=None, *, activation=None, residual=None, table=None, indices=None,
                 gate_slot=None):
    """bf16(A @ W.T + bias) of MXFP4 rows A [M, K] and W [N, K].

    a, b: their codes; a_scale, b_scale: their scales in tile order; bias bf16
    [N] or None. activation="gelu_tanh" or residual/table/indices/gate_slot apply
    the epilogues of int8_matmul to the bf16 product, with the same bits as
    kernels.gelu_tanh and kernels._gated_residual. A block whose scale byte is
    255 (it held a NaN or an infinity) makes the outputs of its row NaN.
    """
    _operand(a, a_scale, "a")
    _operand(b, b_scale, "b")
    if a.shape[1] != b.shape[1]:
        raise ValueError(f"a has {a.shape[1]} bytes of codes per row, b {b.shape[1]}")
    if a.shape[1] == 0:
        raise ValueError("a and b have no columns")
    _no_gradient(bias, residual, table)
    _lib.check_device(a)
    _lib.same_device(a, b=b, a_scale=a_scale, b_scale=b_scale, bias=bias, residual=residual, table=table,
                     indices=indices)
    m, n = a.shape[0], b.shape[0]
    bias = _bias(bias, n)
    epilogue, residual, table, rows, width, indices, sequence, slot = _epilogue(m, n, activation, residual, table,
                                                                                indices, gate_slot)
    output = torch.empty((m, n), device=a.device, dtype=torch.bfloat16)
    _lib.launch(a, "lr_mxfp4_gemm", a.data_ptr(), a_scale.data_ptr(), b.data_ptr(), b_scale.data_ptr(), m, n,
                2 * a.shape[1], _lib.ptr(bias), output.data_ptr(), epilogue, _lib.ptr(residual), _lib.ptr(table), rows,
                width, _lib.ptr(indices), sequence, slot)
    return output


@functools.lru_cache(maxsize=4096)
def _scratch(m, k):
    """Bytes of lr_mxfp4_linear's scratch."""
    codes = -(-m * code_bytes(k) // 256) * 256
    tiles, blocks, size = scale_shape(m, k)
    return codes + tiles * blocks * size


def linear_rows(rows, b, b_scale, bias=None, *, activation=None, residual=None, table=None, indices=None,
                gate_slot=None):
    """mxfp4_matmul of kernels.quantize_rows_mxfp4(rows) and the weight, with one
    allocation for codes and scales and one call for both kernels. At a few rows the
    host bounds a layer: 13 us (10 at one row, which one kernel quantizes and
    multiplies), 20 for the two functions one after the other."""
    m, k = rows.shape
    n = b.shape[0]
    dtype = _ROW_DTYPES.get(rows.dtype)
    if dtype is None:
        raise RuntimeError(f"value: dtype {rows.dtype} is not supported by the HIP quantizer")
    _operand(b, b_scale, "b")
    if b.shape[1] != code_bytes(k) or k == 0:
        raise ValueError(f"rows of {k} columns do not fit a weight of {2 * b.shape[1]}")
    _no_gradient(rows, bias, residual, table)
    _lib.check_device(rows)
    epilogue = _PLAIN
    if activation is None and residual is None and table is None and indices is None and gate_slot is None:
        _lib.same_device(rows, b=b, b_scale=b_scale, bias=bias)
    else:
        _lib.same_device(rows, b=b, b_scale=b_scale, bias=bias, residual=residual, table=table, indices=indices)
        epilogue = _epilogue(m, n, activation, residual, table, indices, gate_slot)
    if not rows.is_contiguous():
        rows = rows.contiguous()
    bias = _bias(bias, n)
    nbytes = _scratch(m, k)
    scratch = rows.new_empty(nbytes, dtype=torch.uint8)
    output = rows.new_empty((m, n), dtype=torch.bfloat16)
    kind, residual, table, table_rows, width, indices, sequence, slot = epilogue
    _lib.launch(rows, "lr_mxfp4_linear", rows.data_ptr(), dtype, m, n, k, scratch.data_ptr(), nbytes, b.data_ptr(),
                b_scale.data_ptr(), _lib.ptr(bias), output.data_ptr(), kind, _lib.ptr(residual), _lib.ptr(table),
                table_rows, width, _lib.ptr(indices), sequence, slot)
    return output
