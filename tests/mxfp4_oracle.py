"""MXFP4 from its definition (OCP Microscaling: e2m1 elements, an e8m0 power of two per 32), in numpy and 64 bits; shares no code with
the product."""

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x):
    """(nibbles uint8 [rows, k], exponents uint8 [rows, k / 32]) of x, any floating type."""
    x = np.asarray(x, np.float64)
    rows, k = x.shape
    blocks = x.reshape(rows, k // 32, 32)
    finite = np.isfinite(blocks).all(-1)
    safe = np.where(finite[..., None], blocks, 0.0)
    most = np.abs(safe).max(-1)
    _, exponent = np.frexp(most)  # most = fraction * 2^exponent, fraction in [0.5, 1)
    power = np.where(most > 0, np.clip(exponent - 3, -127, 127), -127)
    size = np.abs(safe) * np.exp2(-power.astype(np.float64))[..., None]
    middle = (GRID[1:] + GRID[:-1]) / 2
    code = np.zeros(size.shape, np.int64)
    for i, m in enumerate(middle):  # above a middle the next element, at it the one with the even code
        code += (size > m) | ((size == m) & (i % 2 == 1))
    code |= np.signbit(safe).astype(np.int64) << 3
    code[~finite] = 0
    return code.reshape(rows, k).astype(np.uint8), np.where(finite, power + 127, 255).astype(np.uint8)


def values(nibbles, exponents):
    """float64 [rows, k]; blocks with exponent 255 are NaN."""
    rows, k = nibbles.shape
    signed = np.where(nibbles & 8, -1.0, 1.0) * GRID[nibbles & 7]
    scale = np.where(exponents == 255, np.nan, np.exp2(exponents.astype(np.float64) - 127.0))
    return (signed.reshape(rows, k // 32, 32) * scale[..., None]).reshape(rows, k)


def pack(nibbles):
    return (nibbles[:, 0::2] | (nibbles[:, 1::2] << 4)).astype(np.uint8)


def unpack(codes):
    return np.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[0], -1)


def words(exponents, fill=0):
    """u32 [ceil(k / 128), rows]; bytes behind k are `fill`."""
    rows, blocks = exponents.shape
    padded = np.full((rows, (blocks + 3) // 4 * 4), fill, np.uint8)
    padded[:, :blocks] = exponents
    return np.ascontiguousarray(np.ascontiguousarray(padded).view("<u4").T)


def exponents(scale_words, k):
    return np.ascontiguousarray(scale_words.T).view(np.uint8).reshape(scale_words.shape[1], -1)[:, :k // 32]


def plan_of(expert_of_slot, experts, most=None):
    """The plan of slots that are sorted by expert: u32 [1 + tiles, 4]."""
    tiles = []
    for e in range(experts):
        at = np.flatnonzero(expert_of_slot == e)
        tiles += [(e, first, min(first + 128, at[-1] + 1), 0) for first in range(at[0], at[-1] + 1, 128)] if len(at) else []
    slots = len(expert_of_slot)
    out = np.zeros((1 + (slots // 128 + min(experts, slots) if most is None else most), 4), np.uint32)
    out[0, 0] = len(tiles)
    if tiles:
        out[1:1 + len(tiles)] = tiles
    return out
