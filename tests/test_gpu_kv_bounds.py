"""The paged attention against 64 bits, every channel within the bound that its roundings give (kv_bounds.py)."""
from __future__ import annotations

import numpy as np
import pytest

import kv_bounds as kb
import kv_oracle as ko
from test_gpu_kv_pages import dev, i32, quick_fill

pytestmark = pytest.mark.gpu
TOPS = {"f16": None, "int8": 127.0, "e4m3": 448.0}


def written(cuda, rng, fmt, heads, rows):
    table, pages = ko.tables(rng, [len(rows)])
    cache = cuda.KVPages(pages=pages, kv_heads=heads, format=fmt)
    cache.append(dev(rows), i32(table), i32([0]), offsets=i32([0, len(rows)]))
    cache.check()
    return cache, i32(table), ko.stored(rows, fmt)


def worst(got, pairs):
    return max(np.max(np.abs(g - want) / bound) for g, (want, bound) in zip(got, pairs))


@pytest.mark.parametrize("fmt", ko.FORMATS)
@pytest.mark.parametrize("lengths", [[77], [500], [1, 2, 63, 64, 65, 0, 129], [20011], [500, 1, 2048, 0, 777, 4096]])
def test_paged(cuda, fmt, lengths):
    rng = np.random.default_rng(51)
    cache, table, kvs = quick_fill(cuda, rng, fmt, 2, lengths)
    q = (0.7 * rng.standard_normal((len(lengths), 8, 128))).astype(np.float32)
    got = cache.attention(dev(q), i32(table), i32(lengths)).double().cpu().numpy()
    cache.check()
    for b, kv in enumerate(kvs):
        if len(kv):
            assert worst(got[b], [kb.paged(q[b, h], kv[:, 0, h // 4], kv[:, 1, h // 4], TOPS[fmt])
                                  for h in range(8)]) < 1, b


@pytest.mark.parametrize("fmt", ko.FORMATS)
@pytest.mark.parametrize("n", [300, 4096, 20011, 120000])
def test_paged_equal_weights(cuda, fmt, n):
    rng = np.random.default_rng(52)
    rows, q = kb.level_rows(rng, n, 1)
    cache, table, kv = written(cuda, rng, fmt, 1, rows)
    got = cache.attention(dev(q.astype(np.float32)), table, i32([n])).double().cpu().numpy()
    cache.check()
    assert worst(got[0], [kb.paged(q[0, h], kv[:, 0, 0], kv[:, 1, 0], TOPS[fmt]) for h in range(4)]) < 1


@pytest.mark.parametrize("fmt", ko.FORMATS)
@pytest.mark.parametrize("heads,batch,prefix,own", [(2, 3, 130, 70), (1, 40, 5000, 300), (2, 70, 3001, 1),
                                                    (8, 64, 8000, 5), (2, 5, 20000, 64)])
def test_shared(cuda, fmt, heads, batch, prefix, own):
    rng = np.random.default_rng(53)
    cache, table, kvs = quick_fill(cuda, rng, fmt, heads, [own] * batch)
    pre, ptable, pkv = written(cuda, rng, "f16", heads, ko.rows(rng, prefix, heads))
    q = (0.7 * rng.standard_normal((batch, 4 * heads, 128))).astype(np.float16)
    got = cache.attention_shared(dev(q), i32(table), i32([own] * batch), pre, ptable[0].contiguous(), prefix)
    cache.check()
    got = got.double().cpu().numpy()
    for b in sorted({0, 1, batch // 2, batch - 1}):
        assert worst(got[b], [kb.shared(q[b, h], pkv[:, 0, h // 4], pkv[:, 1, h // 4], kvs[b][:, 0, h // 4],
                                        kvs[b][:, 1, h // 4], -(-prefix // 128)) for h in range(4 * heads)]) < 1, b
