"""CPU oracle of the microscaled 4-bit formats, in float64 (test infrastructure).

A matrix is quantised by comparing with the borders between representable values; nothing is
shared with the kernels' arithmetic.  Values are float64 arrays; codes are 0..15 (sign in bit 3).
"""
import numpy as np

POINTS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BLOCK = {"mxfp4": 32, "nvfp4": 16}
_BORDERS = (POINTS[1:] + POINTS[:-1]) / 2


def _e2m1(a):
    """|value| -> magnitude code, to nearest, ties to the even code, saturating."""
    code = np.zeros(a.shape, np.int64)
    for i, b in enumerate(_BORDERS):
        code += (a > b) if i % 2 == 0 else (a >= b)
    return code


def _blocks(v, kind):
    b = BLOCK[kind]
    pad = -v.shape[1] % b
    return np.pad(v, ((0, 0), (0, pad))).reshape(v.shape[0], (v.shape[1] + pad) // b, b)


def e4m3_value(byte):
    byte = np.asarray(byte, np.int64)
    e, f = byte >> 3, byte & 7
    v = np.where(e > 0, (1 + f / 8) * np.exp2(e - 7.0), f * 2.0 ** -9)
    return np.where(byte == 0x7F, np.nan, v)


def e8m0_value(byte):
    byte = np.asarray(byte, np.int64)
    return np.where(byte == 255, np.nan, np.exp2(byte - 127.0))


_E4M3 = e4m3_value(np.arange(127))   # 0 .. 448, increasing


def _e4m3(v):
    """Nearest e4m3 byte of values in [0, 448], ties to the even byte."""
    hi = np.clip(np.searchsorted(_E4M3, v), 1, 126)
    lo = hi - 1
    mid = (_E4M3[lo] + _E4M3[hi]) / 2
    up = (v > mid) | ((v == mid) & (hi % 2 == 0))
    return np.where(up, hi, lo)


def quant(v, kind):
    """bf16 values as float64 [S, D] -> (magnitude codes with sign [S, D], scale bytes [S, blocks], row
    scale [S] or None).  Codes of a block (mxfp4) or row (nvfp4) with a NaN or infinity are 0."""
    with np.errstate(all="ignore"):
        x = _blocks(np.asarray(v, np.float64), kind)
        bad = ~np.isfinite(x).all(2)
        x = np.where(np.isfinite(x), x, 0)
        top = np.abs(x).max(2)
        if kind == "mxfp4":
            e = np.frexp(np.where(top > 0, top, 1))[1] - 1
            byte = np.where(top > 0, np.clip(e - 2 + 127, 0, 254), 0)
            scale, rs = np.exp2(byte - 127.0), None
            byte = np.where(bad, 255, byte)
            dead = bad
        else:
            amax = top.max(1)
            r = np.frexp(np.where(amax > 0, amax, 1) / 2688)[1] - 1
            r = np.where(amax > 2688 * np.exp2(r * 1.0), r + 1, r)
            rs = np.exp2(np.where(amax > 0, np.maximum(r, -100), -100) * 1.0)
            row_bad = bad.any(1)
            byte = _e4m3(np.minimum(top / (6 * rs[:, None]), 448))
            scale = e4m3_value(byte) * rs[:, None]
            rs = np.where(row_bad, np.nan, rs)
            dead = np.broadcast_to(row_bad[:, None], bad.shape)
        a = np.abs(x) / np.where(scale > 0, scale, np.inf)[:, :, None]
        code = np.where(dead[:, :, None], 0, _e2m1(a) | (np.signbit(x).astype(np.int64) << 3))
    return code.reshape(v.shape[0], -1)[:, :v.shape[1]], byte, rs


def value(code, byte, rs, kind):
    """Codes, scale bytes and row scale -> the float64 values they stand for."""
    v = POINTS[code & 7] * np.where(code & 8, -1.0, 1.0)
    scale = e8m0_value(byte) if kind == "mxfp4" else e4m3_value(byte)
    v = (_blocks(v, kind) * scale[:, :, None]).reshape(code.shape[0], -1)[:, :code.shape[1]]
    return v if rs is None else v * np.asarray(rs, np.float64)[:, None]


def tile_scales(byte):
    """[S, blocks] scale bytes -> the tiled buffer (rows and blocks filled up with zeros)."""
    s, b = byte.shape
    p = np.pad(byte.astype(np.uint8), ((0, -s % 128), (0, -b % 4)))
    return p.reshape(p.shape[0] // 128, 4, 32, p.shape[1] // 4, 4).transpose(0, 3, 2, 1, 4).reshape(-1)


def pack(code):
    return (code[:, 0::2] | (code[:, 1::2] << 4)).astype(np.uint8)
