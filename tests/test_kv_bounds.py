"""The bounds of kv_bounds.py on the CPU: a model of the paged attention's arithmetic keeps them, and the same with
one of its parts left out does not."""
from __future__ import annotations

import numpy as np
import pytest

import kv_bounds as kb
import kv_oracle as ko


def model(q, k, v, scale, weights=True, queries=True):
    """F32 softmax with q and p x scale as F16 halves; `weights` or `queries` False: without the second half."""
    def halves(x, both):
        hi = x.astype(np.float16).astype(np.float64)
        return hi + (x - hi).astype(np.float16).astype(np.float64) if both else hi

    up = 2.0 ** np.floor(15 - np.log2(np.abs(q).max() + 1e-30))
    x = (k @ halves(q.astype(np.float64) * up, queries) / up / np.sqrt(128.0)).astype(np.float32)
    p = np.exp((x - x.max()).astype(np.float64)).astype(np.float32)
    w = p.astype(np.float64) * scale
    unit = 128.0 / 2.0 ** np.ceil(np.log2(w.max()))
    return halves(w * unit, weights) / unit @ (v / scale[:, None]) / p.astype(np.float64).sum()


def worst(fmt, kv, q, **kw):
    top = {"f16": None, "int8": 127.0, "e4m3": 448.0}[fmt]
    k, v = kv[:, 0, 0], kv[:, 1, 0]
    scale = np.max(np.abs(v), axis=1) / top if top else np.ones(len(v))
    want, bound = kb.paged(q, k, v, top)
    return np.max(np.abs(model(q, k, v, scale, **kw) - want) / bound)


@pytest.mark.parametrize("fmt", ko.FORMATS)
@pytest.mark.parametrize("n", [77, 500])
def test_the_bound_tells_a_lost_half(fmt, n):
    rng = np.random.default_rng(n)
    kv = ko.stored(ko.rows(rng, n, 1), fmt)
    q = (0.7 * rng.standard_normal(128)).astype(np.float32)
    assert worst(fmt, kv, q) < 0.5
    assert worst(fmt, kv, q, weights=False) > 1 and worst(fmt, kv, q, queries=False) > 1


@pytest.mark.parametrize("fmt", ko.FORMATS)
@pytest.mark.parametrize("n", [4096, 20011])
def test_the_bound_tells_lost_halves_of_equal_weights(fmt, n):
    """Many tokens of random weights average a lost half away; equal ones, with V of one sign, do not."""
    rows, q = kb.level_rows(np.random.default_rng(n), n, 1)
    kv = ko.stored(rows, fmt)
    assert worst(fmt, kv, q[0, 0].astype(np.float32)) < 0.5
    assert worst(fmt, kv, q[0, 0].astype(np.float32), weights=False) > 1
