"""How exact the paged attention is where its arithmetic is under strain, against
64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import kv_oracle as ko
from test_gpu_kv_long import pool_of
from test_gpu_kv_pages import TOL16, dev, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch", [3, 40])
@pytest.mark.parametrize("size", [3000.0, 10000.0, 20000.0])
def test_shared_huge_finite_logits(cuda, batch, size):
    """Queries and keys near F16's largest values: logits up to 2^36, whose products are rounded by thousands.
    Every row's largest logit is well above the rest (by more than the 2^-20 that the products' sum is off by),
    so the exact result is that token's V."""
    rng = np.random.default_rng(41)
    heads, prefix = 2, 20 * 64
    kv = ko.rows(rng, prefix, heads)
    kv[:, 0] = np.clip(rng.standard_normal((prefix, heads, 128)) * size, -65504, 65504).astype(np.float16)
    pre, pkv = pool_of(cuda, rng, "f16", heads, 20, kv)
    own, okv = pool_of(cuda, rng, "int8", heads, 1)
    q = np.clip(rng.standard_normal((batch, 4 * heads, 128)) * size, -65504, 65504).astype(np.float16)
    want = np.empty(q.shape)
    for b in range(batch):
        for h in range(4 * heads):
            x = pkv[:, 0, h // 4] @ q[b, h].astype(np.float64)
            first = np.sort(x)[-2:]
            want[b, h] = pkv[np.argmax(x), 1, h // 4] if first[1] - first[0] > 2.0**-20 * np.abs(
                pkv[:, 0, h // 4] * q[b, h].astype(np.float64)).sum(1).max() else np.nan
    sure = ~np.isnan(want)
    assert sure.mean() > 0.99
    got = own.attention_shared(dev(q), i32(np.zeros((batch, 1))), i32([0] * batch), pre, i32(np.arange(20)), prefix)
    own.check()
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all()
    assert np.max(np.abs(got - want)[sure]) < TOL16 * np.max(np.abs(pkv[:, 1]))
