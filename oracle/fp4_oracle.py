"""CPU restatement of the 4-bit block formats and their product, in 64 bits.

Test infrastructure only; the product package never imports it.  Codes, block
scales and row scales are decided by comparing exact values with the borders
between neighbouring representable numbers, so the kernels are held to every
bit; products are float64 sums of the stored values.
"""
from __future__ import annotations

import math

import numpy as np
import torch

BLOCK = {"nvfp4": 16, "mxfp4": 32}
E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def e4m3_values() -> np.ndarray:
    """The 127 finite non-negative e4m3 numbers, by code."""
    out = []
    for code in range(127):
        exponent, mantissa = code >> 3, code & 7
        out.append(mantissa * 2.0 ** -9 if exponent == 0 else (8 + mantissa) * 2.0 ** (exponent - 10))
    return np.array(out)


E4M3 = e4m3_values()


def nearest_code(num: np.ndarray, unit: np.ndarray, values: np.ndarray) -> np.ndarray:
    """Code of the value nearest to num / unit (both >= 0, unit > 0), ties to
    the even code.  ``border * unit`` is exact in float64: a border has at
    most 5 significant bits, a unit at most 31."""
    borders = (values[1:] + values[:-1]) / 2
    code = np.zeros(np.broadcast(num, unit).shape, dtype=np.int64)
    for i, border in enumerate(borders):
        edge = border * unit
        code += (num > edge) | ((num == edge) & (i % 2 == 1))
    return code


def scale_tiles(rows: int, cols: int, fmt: str) -> tuple[int, int]:
    return -(-rows // 128) * 128, -(-(cols // BLOCK[fmt]) // 4) * 4


def tile_offsets(rows: int, blocks: int) -> np.ndarray:
    """Byte of each (row, block) scale in the stored order."""
    tiles = -(-blocks // 4)
    r, c = np.arange(rows)[:, None], np.arange(blocks)[None, :]
    return (r // 128 * tiles + c // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + c % 4


def quantise(x: torch.Tensor, fmt: str, given: float | None = None):
    """``(codes uint8 [rows, K/2], scale bytes uint8 [padded], row scales fp32 or None)``."""
    rows, cols = x.shape
    xv = x.to(torch.float64).numpy()
    blocks = xv.reshape(rows, -1, BLOCK[fmt])
    finite = np.isfinite(blocks)
    mag = np.where(finite, np.abs(blocks), 0.0)
    bad_block = ~finite.all(-1)
    m = mag.max(-1)
    if fmt == "mxfp4":
        power = np.where(m > 0, np.frexp(m)[1] - 3, -127).clip(min=-127)
        byte = (power + 127).astype(np.uint8)
        unit, row = np.ldexp(1.0, power), None
        byte = np.where(bad_block, 255, byte)
    else:
        if given is None:
            row = (np.maximum(m.max(-1), 2.0 ** -100).astype(np.float32) / np.float32(2688.0))
            bad_row = bad_block.any(-1)
            row = np.where(bad_row, np.float32("nan"), row).astype(np.float32)
            o = np.where(bad_row, 1.0, row.astype(np.float64))[:, None]
        else:
            row, o = None, np.full((rows, 1), np.float64(np.float32(given)))
        byte = nearest_code(m, 6.0 * o, E4M3)
        unit = E4M3[byte] * o
        if given is None:
            byte = np.where(bad_row[:, None], 0, byte)
            unit = np.where(bad_row[:, None], 0.0, unit)
        else:
            byte = np.where(bad_block, 0x7F, byte)
    usable = (unit > 0) & ~bad_block
    code = nearest_code(mag, np.where(usable, unit, 1.0)[..., None], E2M1)
    sign = np.signbit(blocks) * 8
    code = np.where(usable[..., None], code + sign, 0).reshape(rows, cols).astype(np.uint8)
    packed = code[:, 0::2] | (code[:, 1::2] << 4)
    r, c = scale_tiles(rows, cols, fmt)
    tiles = np.zeros(r * c, dtype=np.uint8)
    tiles[tile_offsets(rows, cols // BLOCK[fmt])] = byte
    return packed, tiles.reshape(r, c), row


def stored_values(packed: np.ndarray, tiles: np.ndarray, fmt: str) -> np.ndarray:
    """code * block scale in float64 (NaN where the scale is)."""
    rows, blocks = packed.shape[0], packed.shape[1] * 2 // BLOCK[fmt]
    code = np.stack((packed & 15, packed >> 4), -1).reshape(rows, blocks, -1)
    value = E2M1[code & 7] * np.where(code & 8, -1.0, 1.0)
    byte = tiles.reshape(-1)[tile_offsets(rows, blocks)].astype(np.int64)
    if fmt == "mxfp4":
        scale = np.where(byte == 255, np.nan, np.ldexp(1.0, np.minimum(byte, 254) - 127))
    else:
        scale = np.where(byte == 0x7F, np.nan, E4M3[np.minimum(byte, 126)])
    return (value * scale[..., None]).reshape(rows, -1)


def gelu_tanh(y: np.ndarray) -> np.ndarray:
    return 0.5 * y * (1.0 + np.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3)))


def swiglu(y: np.ndarray) -> np.ndarray:
    """16 gate columns, then the 16 matching up columns."""
    pairs = y.reshape(y.shape[0], -1, 2, 16)
    g, u = pairs[:, :, 0], pairs[:, :, 1]
    return (g / (1.0 + np.exp(-g)) * u).reshape(y.shape[0], -1)
