"""MXFP4 in numpy float64: the definition, written apart from the package."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x):
    """(codes [rows, blocks * 32] 0..15, scale bytes [rows, blocks], values [rows, width])."""
    x = np.asarray(x, np.float64)
    rows, width = x.shape
    blocks = -(-width // 32)
    full = np.zeros((rows, blocks * 32))
    full[:, :width] = x
    sign = np.signbit(full)
    b = full.reshape(rows, blocks, 32)
    bad = ~np.isfinite(b).all(-1)
    amax = np.abs(np.where(np.isfinite(b), b, 0)).max(-1)
    with np.errstate(divide="ignore"):
        e = np.where(amax > 0, np.frexp(amax)[1] - 1 - 2, -127)
    e = np.maximum(e, -127)
    a = np.abs(np.where(bad[..., None], 0, b)) / (2.0 ** e)[..., None]
    # nearest grid value; among two equally near ones the even code
    d = np.abs(a[..., None] - GRID)
    near = d == d.min(-1, keepdims=True)
    even = near & (np.arange(8) % 2 == 0)
    code = np.where(even.any(-1), even.argmax(-1), near.argmax(-1)).reshape(rows, -1)
    code = np.where(np.repeat(bad, 32, 1), 0, code | (sign.astype(int) << 3))
    return code.astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8), decode(code, e, bad)[:, :width]


def decode(code, e, bad=None):
    v = GRID[code & 7] * np.where(code & 8, -1.0, 1.0)
    v = v.reshape(code.shape[0], -1, 32) * (2.0 ** e)[..., None]
    if bad is not None:
        v = np.where(bad[..., None], np.nan, v)
    return v.reshape(code.shape)


def pack(code):
    """Two codes per byte, the even column in the low half."""
    return (code[:, 0::2] | (code[:, 1::2] << 4)).astype(np.uint8)
