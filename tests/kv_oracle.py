"""The paged KV cache in plain numpy, 64 bits: the page layout, the 8-bit
formats and attention, written from their definitions (include/hsb.h)."""
from __future__ import annotations

import numpy as np

PAGE = 64
FORMATS = ("f16", "int8", "e4m3")
PAGE_BYTES = {"f16": 32768, "int8": 16896, "e4m3": 16896}
TOP = {"int8": np.float32(127.0), "e4m3": np.float32(448.0)}


def e4m3_values() -> np.ndarray:
    """The 256 values of e4m3 (bias 7, no infinity, 0x7f and 0xff NaN)."""
    v = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = m * 2.0**-9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        v[c] = np.nan if (c & 127) == 127 else -x if c & 128 else x
    return v


E4M3 = e4m3_values()


def e4m3_round(y: np.ndarray) -> np.ndarray:
    """Nearest e4m3 codes of |y| <= 448, ties to the even mantissa."""
    mag = np.abs(y.astype(np.float64))
    codes = np.arange(127)
    vals = E4M3[:127]
    hi = np.clip(np.searchsorted(vals, mag), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = mag - vals[lo], vals[hi] - mag
    pick = np.where((dl < dh) | ((dl == dh) & (codes[lo] % 2 == 0)), lo, hi)
    return (pick | np.where(np.signbit(y), 128, 0)).astype(np.uint8)


def quantise(x: np.ndarray, fmt: str):
    """F16 vectors [..., 128] -> (codes uint8 [..., 128], scales F32 [...])."""
    x = x.astype(np.float32)
    amax = np.max(np.where(np.isfinite(x), np.abs(x), np.float32(0)), axis=-1)
    with np.errstate(divide="ignore", invalid="ignore"):
        inv = np.where(amax > 0, TOP[fmt] / amax, np.float32(0)).astype(np.float32)
        y = (x * inv[..., None]).astype(np.float32)
    y = np.clip(np.where(np.isnan(y), np.float32(0), y), -TOP[fmt], TOP[fmt])
    codes = np.rint(y).astype(np.int8).view(np.uint8) if fmt == "int8" else e4m3_round(y)
    return codes, (amax / TOP[fmt]).astype(np.float32)


def code_values(codes: np.ndarray, fmt: str) -> np.ndarray:
    return codes.view(np.int8).astype(np.float64) if fmt == "int8" else E4M3[codes]


def stored(x: np.ndarray, fmt: str) -> np.ndarray:
    """What written F16 vectors stand for, in 64 bits."""
    if fmt == "f16":
        return x.astype(np.float64)
    codes, scales = quantise(x, fmt)
    return code_values(codes, fmt) * scales[..., None].astype(np.float64)


def read_back(values: np.ndarray) -> np.ndarray:
    """F16 rows of stored values: the product code * scale is rounded to F32, then to
    F16 (hsb_kv_read's rule; 28 bits of product, so one rounding may differ at a tie)."""
    return values.astype(np.float32).astype(np.float16)


def write_rows(pool: np.ndarray, fmt: str, page: int, row: int, kv: np.ndarray) -> None:
    """Stores one token's K/V [2, heads, 128] (F16) byte by byte in a uint8 pool."""
    panels = 2 if fmt == "f16" else 1
    for part in range(2):
        for h in range(kv.shape[1]):
            block = pool[page, h]
            if fmt == "f16":
                data = np.ascontiguousarray(kv[part, h]).view(np.uint8)
            else:
                data, scale = quantise(kv[part, h], fmt)
                at = 2 * 8192 + part * 256 + row * 4
                block[at:at + 4] = np.array([scale], dtype=np.float32).view(np.uint8)
            for p in range(panels):
                for c in range(8):
                    at = (part * panels + p) * 8192 + row * 128 + (c ^ (row & 7)) * 16
                    block[at:at + 16] = data[p * 128 + c * 16:p * 128 + c * 16 + 16]


def attention(q: np.ndarray, k: np.ndarray, v: np.ndarray) -> np.ndarray:
    """q [4 heads, 128], k / v [n, heads, 128] -> [4 heads, 128], zeros for n = 0."""
    out = np.zeros(q.shape)
    if not len(k):
        return out
    for h in range(q.shape[0]):
        x = k[:, h // 4] @ q[h].astype(np.float64) / np.sqrt(128.0)
        p = np.exp(x - x.max())
        out[h] = (p / p.sum()) @ v[:, h // 4]
    return out


def tables(rng, lengths, spare: int = 3, gap: int = -1):
    """Page tables of the lengths (unused entries `gap`), pages in no order, and the pool's size."""
    need = [-(-int(n) // PAGE) for n in lengths]
    pages = sum(need) + spare
    order = rng.permutation(pages).astype(np.int32)
    table = np.full((len(lengths), max(1, max(need))), gap, dtype=np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, pages


def rows(rng, n: int, heads: int, scale: float = 1.0) -> np.ndarray:
    """K/V rows F16 [n, 2, heads, 128], every 32nd channel of K louder."""
    x = rng.standard_normal((n, 2, heads, 128)) * scale
    x[:, 0, :, 5::32] *= 6.0
    return x.astype(np.float16)
