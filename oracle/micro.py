"""Microscaled formats in 64 bits (numpy): what the operators of cs464_b200.micro are tested against.

Written from the definitions in include/b2g_micro.h: the largest magnitude of a block sets its scale, codes round to
nearest with ties to even, a block with an infinity or a NaN has a NaN scale. Values are computed from codes by their
bit fields, and codes by search among all values of the element type, so nothing here shares a shortcut with the
kernels' bit arithmetic.
"""
from __future__ import annotations

import numpy as np

BLOCK = {"mxfp8": 32, "mxfp4": 32, "nvfp4": 16}


def _table(exp_bits: int, man_bits: int, bias: int, codes: int) -> np.ndarray:
    """The magnitudes of codes 0 .. codes-1 (sign bit left out)."""
    c = np.arange(codes)
    e, m = c >> man_bits, (c & ((1 << man_bits) - 1)) / float(1 << man_bits)
    return np.where(e > 0, (1.0 + m) * 2.0 ** (e - bias), m * 2.0 ** (1 - bias))


E4M3 = _table(4, 3, 7, 127)   # 0 .. 448 (code 127 is NaN)
E2M1 = _table(2, 1, 1, 8)     # 0 .. 6


def _nearest(v: np.ndarray, table: np.ndarray) -> np.ndarray:
    """Code of the table value nearest to v >= 0, ties to the even code, values past the last to the last."""
    hi = np.clip(np.searchsorted(table, v), 1, len(table) - 1)
    lo = hi - 1
    below, above = v - table[lo], table[hi] - v
    up = (above < below) | ((above == below) & (hi % 2 == 0))
    return np.where(v >= table[-1], len(table) - 1, np.where(up, hi, lo))


def tensor_scale(x: np.ndarray) -> float:
    """nvfp4's default scale: the smallest power of two >= 2^-100 at which the largest finite magnitude is <= 2688."""
    f = np.abs(x[np.isfinite(x)])
    g = 2.0 ** -100
    while f.size and f.max() > 2688.0 * g:
        g *= 2.0
    return g


def quantize(x: np.ndarray, fmt: str, scale: float | None = None):
    """(codes [R, C] uint8 with the sign in the top bit of the format, scale bytes [R, B] uint8) of x in 64 bits."""
    r, c = x.shape
    size = BLOCK[fmt]
    n = -(-c // size)
    p = np.zeros((r, n * size))
    p[:, :c] = x
    p = p.reshape(r, n, size)
    bad = ~np.isfinite(p).all(2)
    amax = np.where(bad, 0.0, np.abs(np.where(np.isfinite(p), p, 0.0)).max(2))
    if fmt == "nvfp4":
        sb = _nearest(np.minimum(amax / (6.0 * scale), 448.0), E4M3)
        unit = E4M3[sb] * scale
        sb = np.where(bad, 0x7F, sb)
    else:
        top = 448.0 if fmt == "mxfp8" else 6.0
        e = np.full(amax.shape, -127)
        with np.errstate(divide="ignore"):
            k = np.ceil(np.log2(np.where(amax > 0, amax / top, 2.0 ** -200))).astype(int)
        for d in (-1, 0, 1):  # the logarithm may be off by an ulp at a power of two: the definition decides
            ok = amax <= top * 2.0 ** (k + d).astype(float)
            e = np.where(ok & (e == -127) & (k + d > -127), k + d, e)
        sb = np.where(bad, 255, e + 127)
        unit = 2.0 ** e.astype(float)
    with np.errstate(divide="ignore", invalid="ignore"):
        v = np.where(bad[..., None] | (unit[..., None] == 0), 0.0, p / unit[..., None])
    v = np.nan_to_num(v)
    code = _nearest(np.abs(v), E4M3 if fmt == "mxfp8" else E2M1)
    sign = np.signbit(np.where(np.isfinite(p), p, 0.0)) & ~bad[..., None]
    code = code | (sign.astype(int) << (7 if fmt == "mxfp8" else 3))
    return code.reshape(r, -1)[:, :c].astype(np.uint8), sb.astype(np.uint8)


def values(codes: np.ndarray, scale_bytes: np.ndarray, fmt: str, scale: float | None = None) -> np.ndarray:
    """The values [R, C] of codes and block scale bytes."""
    if fmt == "mxfp8":
        q = np.append(E4M3, np.nan)[codes & 127] * np.where(codes >> 7, -1.0, 1.0)
    else:
        q = E2M1[codes & 7] * np.where(codes >> 3, -1.0, 1.0)
    b = scale_bytes.astype(int)
    s = np.append(E4M3, np.nan)[b] * scale if fmt == "nvfp4" else np.where(b == 255, np.nan, 2.0 ** (b - 127.0))
    return q * np.repeat(s, BLOCK[fmt], 1)[:, :codes.shape[1]]


def unpack(codes: np.ndarray, scales: np.ndarray, rows: int, cols: int, fmt: str):
    """(codes [R, C], scale bytes [R, B], True if everything outside them is zero) of a stored tensor: its code bytes
    [R, pitch] and its scale bytes in tile order."""
    if fmt == "mxfp8":
        c = codes
    else:
        c = np.stack([codes & 15, codes >> 4], 2).reshape(codes.shape[0], -1)
    n = -(-cols // BLOCK[fmt])
    kt = -(-n // 4)
    rt = -(-rows // 128)
    full = scales.reshape(rt, kt, 32, 4, 4).transpose(0, 3, 2, 1, 4).reshape(rt * 128, kt * 4)
    rest = full.copy()
    rest[:rows, :n] = 0
    return c[:, :cols], full[:rows, :n], not rest.any() and not c[:, cols:].any()
