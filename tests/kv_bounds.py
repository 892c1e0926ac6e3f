"""How far the paged attention may be from 64 bits, channel by channel, by
counting its roundings.

A logit x = (k . q) / sqrt(128), with S = sum |k q| / sqrt(128), is off by
  2^-22 S       q as two F16 halves (F32 queries; F16 ones are exact),
  16 2^-23 S    eight products of 16 channels, each cut when it is summed and
                again when it is added to the accumulator,
  6 2^-24 |x|   the scales' products, the subtraction of the reference,
  2^-21         the power of two (also by polynomial 2.7e-6, in `power`),
relative to the weight p.  A weight enters the second product rounded:
  paged         2^-21 p, or 2^-31 of the largest (in 8 bits of p x scale);
  prefix        2^-11 p, or 2^-32 of the largest.
An output is cut (8 + 2 a tile) times by 2^-23, rounded 2^-24 once a unit and
partial, and where it is F16 by 2^-11 of itself and 2^-25.  A weighted mean
moves by sum p e |v| + |mean| sum p e."""
from __future__ import annotations

import numpy as np


def paged(q, k, v, top=None, units=64, halves=True):
    """(result, bound) of one query row q [128] over k, v [n, 128]; `top`: the largest code of the 8-bit formats."""
    x = k @ q.astype(np.float64) / np.sqrt(128.0)
    size = np.abs(k) @ np.abs(q.astype(np.float64)) / np.sqrt(128.0)
    p = np.exp(x - x.max())
    p /= p.sum()
    out = p @ v
    s = np.max(np.abs(v), axis=1) / top if top else np.ones(len(v))
    e = (2.0**-22 + 16 * 2.0**-23) * size + 6 * 2.0**-24 * np.abs(x) + 2.0**-21
    w = 2.0**-21 * p + np.minimum(p, 2.0**-31 * np.max(p * s) / np.maximum(s, 1e-30))
    a = p @ np.abs(v)
    bound = (p * e + w) @ np.abs(v) + np.abs(out) * (p @ e) + (16 * 2.0**-23 + units * 2.0**-24) * a
    return out, bound + 1e-30


def shared(q, kp, vp, ko, vo, tiles):
    """The same of an F16 row over a prefix's and its own tokens; `tiles`: of a CTA's stretch, at most."""
    k, v, n = np.concatenate([kp, ko]), np.concatenate([vp, vo]), len(kp)
    x = k @ q.astype(np.float64) / np.sqrt(128.0)
    size = np.abs(k) @ np.abs(q.astype(np.float64)) / np.sqrt(128.0)
    p = np.exp(x - x.max())
    p /= p.sum()
    out = p @ v
    e = 16 * 2.0**-23 * size + 6 * 2.0**-24 * np.abs(x) + 2.0**-21
    e[:n] += 3e-6  # the polynomial
    w = 2.0**-21 * p + 2.0**-31 * p.max()
    w[:n] = np.maximum(2.0**-11 * p[:n], 2.0**-32 * p.max())
    a = p @ np.abs(v)
    bound = (p * e + w) @ np.abs(v) + np.abs(out) * (p @ e) + min(tiles, 256) * 10 * 2.0**-23 * a
    return out, bound + 2.0**-11 * np.abs(out) + 2.0**-25


def level_rows(rng, n, heads, batch=1):
    """Tokens of equal weight, 0.37 below the one at n // 3, with V of one sign; and their queries F16."""
    rows = np.zeros((n, 2, heads, 128))
    rows[:, 0, :, 0], rows[n // 3, 0, :, 0] = -0.37, 0.0
    rows[:, 1] = 1.0 + 0.1 * rng.standard_normal((n, heads, 128))
    rows[:, 1, :, 7] = 2.0  # (a common V scale, so that equal weights stay equal)
    q = np.zeros((batch, 4 * heads, 128), np.float16)
    q[:, :, 0] = np.sqrt(128.0)
    return rows.astype(np.float16), q
