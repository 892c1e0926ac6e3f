"""The paged attention's loops at the lengths they are for: many units a warp,
many tiles a CTA, page look-ups behind the first, idle places before a run, a
maximum that rises inside a stretch, bad pages deep in one.

Tables name a few pages again and again, so that pools stay small and the
definition in 64 bits needs each distinct token once, with its count.  The work
of a warp or CTA, on 148 SMs, stands beside each case.

Tolerances relative to the largest |v|, as in test_gpu_kv_pages.py; long sums
add what the tensor cores' truncation loses: 2^-23 for each addition to an
accumulator, 8 a tile of 128 tokens (fewer in the paged kernel, whose units
start from zero)."""
from __future__ import annotations

import numpy as np
import pytest

import kv_oracle as ko
from test_gpu_kv_pages import TOL16, TOL32, close, dev, i32

pytestmark = pytest.mark.gpu


def pool_of(cuda, rng, fmt, heads, pages, kv=None):
    """A pool of that many written pages, and their tokens' K/V in 64 bits."""
    kv = ko.rows(rng, pages * 64, heads) if kv is None else kv
    cache = cuda.KVPages(pages=pages, kv_heads=heads, format=fmt)
    cache.append(dev(kv), i32(np.arange(pages)[None]), i32([0]), offsets=i32([0, pages * 64]))
    cache.check()
    return cache, ko.stored(kv, fmt)


def counts_of(table, n, pages):
    """How often each token of the pool is among the first n positions of a table row."""
    got = np.zeros((pages, 64))
    full, rest = divmod(n, 64)
    good = [e for e in table[:full] if 0 <= e < pages]
    np.add.at(got, good, 1.0)
    if rest and 0 <= table[full] < pages:
        got[table[full], :rest] += 1
    return got.reshape(-1)


def attention(q, kv, counts):
    """q [4 heads, 128] over the tokens kv with these counts."""
    out = np.zeros(q.shape)
    kv, counts = kv[counts > 0], counts[counts > 0]
    if len(kv):
        for h in range(len(q)):
            x = kv[:, 0, h // 4] @ q[h].astype(np.float64) / np.sqrt(128.0) + np.log(counts)
            p = np.exp(x - x.max())
            out[h] = (p / p.sum()) @ kv[:, 1, h // 4]
    return out


# ------------------------------------------------------------ paged attention
@pytest.mark.parametrize("fmt", ko.FORMATS)
@pytest.mark.parametrize("heads,lengths", [
    (1, [148 * 8 * 40 * 64 - 17]),  # one run, 40 pages a warp
    (8, [150001, 0, 64 * 3000, 5, 120000]),  # runs of 2000 to 3000 pages, 50 pages a warp, run ends inside
])
def test_many_pages_a_warp(cuda, fmt, heads, lengths):
    rng = np.random.default_rng(len(lengths))
    pages = 24
    cache, kv = pool_of(cuda, rng, fmt, heads, pages)
    width = -(-max(lengths) // 64)
    table = rng.integers(0, pages, (len(lengths), width)).astype(np.int32)
    q = rng.standard_normal((len(lengths), 4 * heads, 128)).astype(np.float32)
    want = np.stack([attention(q[b], kv, counts_of(table[b], n, pages)) for b, n in enumerate(lengths)])
    got = cache.attention(dev(q), i32(table), i32(lengths))
    cache.check()
    close(got, want, [kv], TOL32)
    again = cache.attention(dev(q), i32(table), i32(lengths))
    assert bool((got == again).all())
    # bad entries everywhere, two of three in places, are left out
    table[rng.random(table.shape) < 0.05] = -3
    table[:, 33:1000:3], table[:, 34:1000:3] = pages, 2**31 - 1
    want = np.stack([attention(q[b], kv, counts_of(table[b], n, pages)) for b, n in enumerate(lengths)])
    close(cache.attention(dev(q), i32(table), i32(lengths)), want, [kv], TOL32)
    with pytest.raises(cuda.InvalidArgument) as e:
        cache.check()
    assert e.value.status == 121


@pytest.mark.parametrize("fmt", ko.FORMATS)
def test_served_batch(cuda, fmt):
    """64 sequences of up to 32768 tokens, 8 heads, wide tables: some 110 pages a warp."""
    rng = np.random.default_rng(64)
    pages, batch = 16, 64
    cache, kv = pool_of(cuda, rng, fmt, 8, pages)
    lengths = rng.integers(16384, 32769, batch)
    lengths[[0, 5, 63]] = 32768, 0, 1
    table = rng.integers(0, pages, (batch, 600)).astype(np.int32)
    q = rng.standard_normal((batch, 32, 128)).astype(np.float32)
    want = np.stack([attention(q[b], kv, counts_of(table[b], int(n), pages)) for b, n in enumerate(lengths)])
    got = cache.attention(dev(q), i32(table), i32(lengths))
    cache.check()
    close(got, want, [kv], TOL32)


# -------------------------------------------------------------- shared prefix
# (heads, batch, prefix tokens): tiles a CTA, plan
LONG = [(2, 4, 170003),    # 17.9, one M tile: six stages go round, a second page look-up, idle places
        (8, 32, 45000),    # 19.0, one M tile
        (2, 64, 170003),   # 17.9, two M tiles
        (1, 100, 200065),  # 21.1, two groups of M tiles, the last half empty
        (8, 256, 16461)]   # 27.9, four groups


def shared(cuda, rng, heads, batch, prefix, kv=None, q=None, bad=None):
    pages = 24 if kv is None else len(kv) // 64
    pre, pkv = pool_of(cuda, rng, "f16", heads, pages, kv)
    table = rng.integers(0, pages, -(-prefix // 64)).astype(np.int32) if bad != "rising" else \
        (np.arange(-(-prefix // 64)) % pages).astype(np.int32)
    if isinstance(bad, (int, float)):
        table[rng.random(len(table)) < bad] = -1
        table[40:48] = pages  # (whole tiles too)
    counts = counts_of(table, prefix, pages)
    own, okv = pool_of(cuda, rng, "int8", heads, 2)
    lengths = rng.integers(0, 129, batch)
    lengths[batch // 2] = 0
    q = rng.standard_normal((batch, 4 * heads, 128)).astype(np.float16) if q is None else q
    got = own.attention_shared(dev(q), i32(np.tile([[0, 1]], (batch, 1))), i32(lengths), pre, i32(table), prefix)
    both = np.concatenate([pkv, okv])
    want = np.stack([attention(q[b], both, np.concatenate([counts, np.arange(128) < lengths[b]]))
                     for b in range(batch)])
    return own, got, want, both


@pytest.mark.parametrize("heads,batch,prefix", LONG)
def test_many_tiles_a_cta(cuda, heads, batch, prefix):
    own, got, want, kv = shared(cuda, np.random.default_rng(prefix), heads, batch, prefix)
    own.check()
    close(got, want, [kv], TOL16 + 30 * 8 * 2.0**-23)


@pytest.mark.parametrize("heads,batch,prefix", LONG)
def test_bad_pages_deep_in_a_stretch(cuda, heads, batch, prefix):
    """A page in ten, and eight in a row behind the 16th tile, are not there."""
    own, got, want, kv = shared(cuda, np.random.default_rng(prefix + 1), heads, batch, prefix, bad=0.1)
    close(got, want, [kv], TOL16 + 30 * 8 * 2.0**-23)
    with pytest.raises(cuda.InvalidArgument) as e:
        own.check()
    assert e.value.status == 121


@pytest.mark.parametrize("heads,batch,prefix", LONG)
def test_maximum_that_rises_in_every_stretch(cuda, heads, batch, prefix):
    """Logits rise by 4 a page over 24 pages, again and again (or fall, for a negative query): the rescaling of
    the accumulators behind a stretch's first tile.  |logit| < 4 * 24 + 16: with 12 roundings of the products' sum
    and 3 of the scale, a weight is off by 15 * 2^-23 * 112 at most, and a weighted mean by twice that."""
    rng = np.random.default_rng(prefix + 2)
    kv = ko.rows(rng, 24 * 64, heads)
    kv[:, 0, :, 0] = (np.arange(24 * 64) // 64 * 4.0)[:, None]
    q = rng.standard_normal((batch, 4 * heads, 128)).astype(np.float16)
    q[:, :, 0] = np.sqrt(128.0) * np.where(rng.random((batch, 4 * heads)) < 0.3, -1.0, 1.0)
    own, got, want, kv = shared(cuda, rng, heads, batch, prefix, kv=kv, q=q, bad="rising")
    own.check()
    close(got, want, [kv], TOL16 + 30 * 8 * 2.0**-23 + 2 * 15 * 2.0**-23 * 112)
