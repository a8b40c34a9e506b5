"""MXFP4 in 64 bits, from the format's definition (numpy; test reference only)."""
from __future__ import annotations

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
MIDS = (GRID[1:] + GRID[:-1]) / 2  # decision points between neighbours


def blocks(x: np.ndarray) -> np.ndarray:
    """float64 [..., K] -> [..., ceil(K / 32), 32], filled up with zeros."""
    x = np.asarray(x, np.float64)
    pad = -x.shape[-1] % 32
    x = np.concatenate([x, np.zeros((*x.shape[:-1], pad))], axis=-1)
    return x.reshape(*x.shape[:-1], -1, 32)


def scale_bytes(amax: np.ndarray) -> np.ndarray:
    """e8m0 byte of blocks with the given largest magnitude."""
    finite = np.isfinite(amax)
    _, e = np.frexp(np.where(finite, amax, 1.0))  # mantissa in [0.5, 1)
    byte = np.where(amax == 0, 0, np.clip(e - 3, -127, None) + 127)
    return np.where(finite, byte, 255).astype(np.int64)


def quantize(x: np.ndarray):
    """(codes [..., K'] one per byte, scale bytes [..., K'/32])."""
    b = blocks(x)
    s = scale_bytes(np.abs(b).max(-1))
    with np.errstate(invalid="ignore"):
        y = np.abs(b) * 2.0 ** (127.0 - s[..., None])
    below = np.searchsorted(MIDS, y, side="left")   # codes whose upper midpoint is < y
    above = np.searchsorted(MIDS, y, side="right")
    code = np.where(below == above, below, np.where(below % 2 == 0, below, above))  # tie: even
    code = code + 8 * np.signbit(b)
    code = np.where(s[..., None] == 255, 0, code)
    return code.reshape(*code.shape[:-2], -1).astype(np.uint8), s


def values(codes: np.ndarray, s: np.ndarray) -> np.ndarray:
    """float64 values of codes (one per byte) and scale bytes."""
    v = np.where(codes >= 8, -GRID[codes & 7], GRID[codes & 7]).reshape(*s.shape, 32)
    scale = np.where(s == 255, np.nan, 2.0 ** (s.astype(np.float64) - 127))
    return (v * scale[..., None]).reshape(codes.shape)


def rounded(x: np.ndarray) -> np.ndarray:
    """The MXFP4 values nearest to x [..., K]."""
    return values(*quantize(x))[..., :x.shape[-1]]


def unpack_codes(packed: np.ndarray) -> np.ndarray:
    return np.stack([packed & 15, packed >> 4], axis=-1).reshape(*packed.shape[:-1], -1)


def flip_room(h: np.ndarray, tol: np.ndarray) -> np.ndarray:
    """How far MXFP4(h + e) may be from MXFP4(h), element by element, for any |e| <= tol:
    nothing where neither the scale nor the element is within tol of a decision point, else
    one step of the (possibly doubled) scale."""
    hb, tb = blocks(np.abs(h)), blocks(tol)
    amax, t = hb.max(-1), tb.max(-1)
    s_lo, s_hi = scale_bytes(np.maximum(amax - t, 0)), scale_bytes(amax + t)
    scale = 2.0 ** (s_hi - 127.0)[..., None]
    near = np.zeros(hb.shape, bool)
    for m in MIDS:
        near |= np.abs(hb - m * scale) <= tb
    step = np.where(hb < 1.75 * scale, 0.5, np.where(hb < 3.5 * scale, 1.0, 2.0)) * scale
    room = np.where(near, step, 0.0)
    # another scale: both grids are within one step of h (two of its own past 6 scales)
    room = np.where((s_lo != s_hi)[..., None], 2 * step, room)
    return room.reshape(*h.shape[:-1], -1)[..., :h.shape[-1]]
