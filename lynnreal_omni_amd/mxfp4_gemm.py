"""Products of MXFP4 rows (4-bit codes with a power-of-two scale for each 32) on
gfx950's scaled MFMA: the 4-bit counterpart of int8_gemm.

Operands are what kernels.quantize_rows_mxfp4 returns for [rows, K] values:
codes uint8 [rows, 16 * ceil(K / 32)] and scales uint8 in tile order. The
weight is [N, K] like nn.Linear's, so mxfp4_matmul(a, w, ...) is a @ w.T.
Inference only: the outputs carry no gradient.
"""
from __future__ import annotations

import torch

from . import _lib

BLOCK = 32          # values that share a scale
_TILE_ROWS, _TILE_BLOCKS = 64, 8


def code_bytes(width: int) -> int:
    """Bytes of a row's codes."""
    return -(-width // BLOCK) * (BLOCK // 2)


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
    if codes.dim() != 2 or codes.dtype != torch.uint8 or not codes.is_contiguous() or codes.shape[1] % 16:
        raise ValueError(f"{name} must be contiguous uint8 codes [rows, 16 * blocks]")
    if scales.dtype != torch.uint8 or tuple(scales.shape) != scale_shape(codes.shape[0], 2 * codes.shape[1]):
        raise ValueError(f"{name}_scale must be uint8 {scale_shape(codes.shape[0], 2 * codes.shape[1])}, "
                         f"got {scales.dtype} {tuple(scales.shape)}")
    if not scales.is_contiguous():
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
    _lib.check_device(a)
    _lib.same_device(a, b=b, a_scale=a_scale, b_scale=b_scale, bias=bias, residual=residual, table=table,
                     indices=indices)
    m, n = a.shape[0], b.shape[0]
    if bias is not None:
        if bias.dtype != torch.bfloat16 or bias.numel() != n:
            raise ValueError("bias must be bfloat16 with N entries")
        bias = bias.contiguous()
    epilogue, sequence, slot, rows, width = _lib.EPI_BF16, 0, 0, 0, 0
    if residual is not None:
        if activation is not None:
            raise ValueError("activation and gated residual epilogues are exclusive")
        residual, table, indices, sequence = _gated(m, n, residual, table, indices, gate_slot)
        epilogue, slot, width = _lib.EPI_GATED_RESIDUAL, int(gate_slot), table.shape[-1]
        rows = table.numel() // width if width else 0
    elif table is not None or indices is not None or gate_slot is not None:
        raise ValueError("table, indices and gate_slot belong to a gated residual: residual is missing")
    elif activation == "gelu_tanh":
        epilogue = _lib.EPI_GELU_TANH
    elif activation is not None:
        raise ValueError(f"unsupported activation {activation!r}")
    output = torch.empty((m, n), device=a.device, dtype=torch.bfloat16)
    if a.shape[1] == 0:
        raise ValueError("a and b have no columns")
    _lib.launch(a, "lr_mxfp4_gemm", a.data_ptr(), a_scale.data_ptr(), b.data_ptr(), b_scale.data_ptr(), m, n,
                2 * a.shape[1], _lib.ptr(bias), output.data_ptr(), epilogue, _lib.ptr(residual), _lib.ptr(table), rows,
                width, _lib.ptr(indices), sequence, slot)
    return output
