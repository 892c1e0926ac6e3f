"""How exact the paged attention is where its arithmetic is under strain, against
64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import kv_oracle as ko
from test_gpu_kv_long import attention, counts_of, pool_of
from test_gpu_kv_pages import TOL16, close, dev, i32, quick_fill

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


def weighted(q, kv, counts):
    """One query row over tokens kv [n, 2, 128] with counts: the result and sum p |v| per channel, and 1 / sum exp."""
    x = kv[:, 0] @ q.astype(np.float64) / np.sqrt(128.0)
    e = counts * np.exp(x - x.max())
    p = e / e.sum()
    return p @ kv[:, 1], p @ np.abs(kv[:, 1]), 1 / e.sum()


def sink_and_tail(cuda, batch, heads, prefix, gaps):
    """One token whose logit is `gap` above a flat tail of the rest and whose V is near zero: the result is the
    tail's share.  A quarter of the rows each has its gap.  Checked on rows of the first and the last sequences."""
    rng = np.random.default_rng(42)
    pages = 8
    kv = ko.rows(rng, pages * 64, heads, 0.1)
    kv[:, 1] = (1.0 + 0.1 * rng.standard_normal(kv[:, 1].shape)).astype(np.float16)
    kv[:, 0, :, 0] = 0.0
    kv[0, 0, :, 0], kv[0, 1] = 1.0, 2.0**-10
    pre, pkv = pool_of(cuda, rng, "f16", heads, pages, kv)
    table = rng.integers(1, pages, -(-prefix // 64)).astype(np.int32)
    table[1] = 0
    counts = counts_of(table, prefix, pages)
    q = (0.1 * rng.standard_normal((batch, 4 * heads, 128))).astype(np.float16)
    q[:, :, 0] = np.tile(np.asarray(gaps) * np.sqrt(128.0), heads)
    own, _ = pool_of(cuda, rng, "int8", heads, 1)
    got = own.attention_shared(dev(q), i32(np.zeros((batch, 1))), i32([0] * batch), pre, i32(table), prefix)
    own.check()
    got = got[[0, 1, batch - 1]].double().cpu().numpy()
    for i, b in enumerate((0, 1, batch - 1)):
        for h in range(4 * heads):
            want, size, inv = weighted(q[b, h], pkv[:, :, h // 4], counts)
            yield got[i, h], want, size, inv, q[b, h], pkv[:, :, h // 4]


@pytest.mark.parametrize("batch,prefix", [(3, 32768), (64, 32768), (1216, 4096), (1216, 32768)])
def test_shared_tail_behind_a_dominant_token(cuda, batch, prefix):
    """A CTA's stretch is up to 256 tiles here.  A weight is rounded by 2^-11 of itself, or by 2^-32 of the largest
    (which is 1 / sum exp of the whole) where that is more; the result by 2^-11; a logit (|q k| summed < 21, 12
    additions cut by 2^-23, three roundings) by 2^-18, so the mean by twice that."""
    for got, want, size, inv, *_ in sink_and_tail(cuda, batch, 8, prefix, (8.0, 12.0, 16.0, 18.5)):
        n = min(prefix, 32768)
        bound = (2.0**-11 + 2 * 2.0**-18) * size + 2.0**-11 * np.abs(want) + n * 2.0**-32 * inv * 1.5 + 2.0**-25
        assert np.all(np.abs(got - want) < bound), (np.max(np.abs(got - want) / bound), want[0])


@pytest.mark.parametrize("heads,batch", [(8, 1216), (2, 4), (2, 64)])
def test_shared_sum_over_a_million_tokens(cuda, heads, batch):
    """Equal weights over 2^20 tokens with V of one sign, in stretches of 8192, 111 and 111 tiles: the tensor cores cut
    each of a tile's eight additions to the sum (by 2^-23 of it at most, and 2^-23 within the product), so no sum goes
    on for more than 256 tiles."""
    rng = np.random.default_rng(43)
    pages, prefix = 8, (1 << 20) + 77
    kv = ko.rows(rng, pages * 64, heads)
    kv[:, 1] = (1.0 + 0.1 * rng.standard_normal(kv[:, 1].shape)).astype(np.float16)
    pre, pkv = pool_of(cuda, rng, "f16", heads, pages, kv)
    table = rng.integers(0, pages, -(-prefix // 64)).astype(np.int32)
    counts = counts_of(table, prefix, pages)
    own, _ = pool_of(cuda, rng, "int8", heads, 1)
    got = own.attention_shared(dev(np.zeros((batch, 4 * heads, 128), np.float16)), i32(np.zeros((batch, 1))),
                               i32([0] * batch), pre, i32(table), prefix)
    own.check()
    want = np.repeat(np.tensordot(counts / counts.sum(), pkv[:, 1], 1), 4, 0)
    bound = (2.0**-11 + 2**-18 + 256 * 8 * 2 * 2.0**-23) * np.abs(want)
    err = np.abs(got.double().cpu().numpy() - want)
    assert np.all(err < bound), np.max(err / np.abs(want))


@pytest.mark.parametrize("heads,batch,prefix", [(8, 1216, 33000), (8, 1216, 70000), (1, 9472, 40000)])
def test_shared_stretches_in_several_sums(cuda, heads, batch, prefix):
    """Stretches that begin and end their sums several times: logits that rise from page to page, the dominant part in
    the first, the last or all of them, a bad page among them."""
    rng = np.random.default_rng(44)
    pages = 32
    kv = ko.rows(rng, pages * 64, heads)
    kv[:, 0, :, 0] = (np.arange(pages * 64) // 64 * 1.0)[:, None]
    pre, pkv = pool_of(cuda, rng, "f16", heads, pages, kv)
    total = -(-prefix // 64)
    table = (np.arange(total) * pages // total).astype(np.int32)
    table[total // 2] = -1
    counts = counts_of(table, prefix, pages)
    q = rng.standard_normal((batch, 4 * heads, 128)).astype(np.float16)
    q[:, :, 0] = np.tile(np.array([1.0, -1.0, 0.0, 0.5]) * np.sqrt(128.0), heads)
    own, okv = pool_of(cuda, rng, "int8", heads, 1)
    got = own.attention_shared(dev(q), i32(np.zeros((batch, 1))), i32([3] * batch), pre, i32(table), prefix)
    with pytest.raises(cuda.InvalidArgument) as e:
        own.check()
    assert e.value.status == 121
    both, pick = np.concatenate([pkv, okv]), sorted(rng.choice(batch, 20, replace=False)) + [batch - 1]
    counts = np.concatenate([counts, np.arange(64) < 3])
    want = np.stack([attention(q[b], both, counts) for b in pick])
    # (|logit| < 32 + 16: fifteen roundings of 2^-23 each, twice)
    close(got[pick], want, [both], TOL16 + 256 * 8 * 2 * 2.0**-23 + 2 * 15 * 2.0**-23 * 48)


# ------------------------------------------------------------ paged attention
def strict(got, q, kv, top):
    """One sequence's rows against 64 bits, channel by channel.  With s a row's V scale (1 in F16), a weight is off by
    2^-21 of itself (two halves of 11 bits, three roundings) or by 2^-31 of the head's largest weight x scale where
    that is more, but no weight by more than itself; with S = sum |q k| / sqrt(128) < 16 and |logit| < 32 of every
    row that counts, exp by 2e-5 (test_gpu_kv_pages.py) and so the mean by twice that."""
    got, worst = got.double().cpu().numpy(), 0.0
    for h in range(len(q)):
        k, v = kv[:, 0, h // 4], kv[:, 1, h // 4]
        x = k @ q[h].astype(np.float64) / np.sqrt(128.0)
        p = np.exp(x - x.max())
        s = np.max(np.abs(v), axis=1) / top if top else np.ones(len(v))
        off = 2.0**-21 * p + np.minimum(p, 2.0**-31 * np.max(p * s) / np.maximum(s, 1e-30))
        bound = (4e-5 * p + off) @ np.abs(v) / p.sum()
        worst = max(worst, np.max(np.abs(got[h] - p @ v / p.sum()) / np.maximum(bound, 1e-30)))
    assert worst < 1.0, worst


TOPS = {"f16": None, "int8": 127.0, "e4m3": 448.0}


@pytest.mark.parametrize("fmt", ko.FORMATS)
@pytest.mark.parametrize("n,at", [(513, 0), (513, 70), (513, 512), (4000, 1), (4000, 3000)])
@pytest.mark.parametrize("gap", [-20.0, -30.0, -60.0])
def test_loud_rows_that_count_little(cuda, fmt, n, at, gap):
    """One V of 6e4 among others of 1e-3, its logit far below theirs (or theirs far above it, where it comes first)."""
    rng = np.random.default_rng(45)
    kv = ko.rows(rng, n, 2)
    kv[:, 0, :, 0] = 0.0
    kv[:, 1] = (kv[:, 1].astype(np.float32) * 1e-3).astype(np.float16)
    kv[at, 0, :, 0] = gap
    kv[at, 1] = np.clip(rng.standard_normal((2, 128)) * 3e4, -6e4, 6e4).astype(np.float16)
    table, pages = ko.tables(rng, [n])
    cache = cuda.KVPages(pages=pages, kv_heads=2, format=fmt)
    cache.append(dev(kv), i32(table), i32([0]), offsets=i32([0, n]))
    q = (0.5 * rng.standard_normal((1, 8, 128))).astype(np.float32)
    q[:, :, 0] = np.sqrt(128.0)
    got = cache.attention(dev(q), i32(table), i32([n]))
    cache.check()
    strict(got[0], q[0], ko.stored(kv, fmt), TOPS[fmt])


@pytest.mark.parametrize("fmt", ko.FORMATS)
@pytest.mark.parametrize("lengths", [[77], [20011], [500, 1, 2048, 0, 777, 4096], [33] * 40])
def test_attention_channel_by_channel(cuda, fmt, lengths):
    rng = np.random.default_rng(46)
    cache, table, kvs = quick_fill(cuda, rng, fmt, 4, lengths)
    q = (0.7 * rng.standard_normal((len(lengths), 16, 128))).astype(np.float32)
    got = cache.attention(dev(q), i32(table), i32(lengths))
    cache.check()
    for b, kv in enumerate(kvs):
        if len(kv):
            strict(got[b], q[b], kv, TOPS[fmt])
        else:
            assert not got[b].any()


@pytest.mark.parametrize("heads,batch,tiles", [(8, 4, 4753), (8, 30, 9000), (8, 1216, 257), (8, 1216, 513)])
@pytest.mark.parametrize("slope", [0.0, 1.0, -1.0])
def test_shared_sums_that_end_and_begin_again(cuda, heads, batch, tiles, slope):
    """Stretches of 257, 486, 257 and 513 tiles: with one M tile the last sum of a single tile leaves one warpgroup
    none.  Equal weights, or logits that rise or fall by 32 along the prefix (|logit| < 32 + 5)."""
    rng = np.random.default_rng(47)
    pages, prefix = 32, tiles * 128 - 5
    kv = ko.rows(rng, pages * 64, heads, 0.3)
    kv[:, 0, :, 0] = (np.arange(pages * 64) // 64 * 1.0)[:, None]
    kv[:, 1] = (1.0 + 0.1 * rng.standard_normal(kv[:, 1].shape)).astype(np.float16)
    pre, pkv = pool_of(cuda, rng, "f16", heads, pages, kv)
    total = -(-prefix // 64)
    table = (np.arange(total) * pages // total).astype(np.int32)
    counts = counts_of(table, prefix, pages)
    q = (0.3 * rng.standard_normal((batch, 4 * heads, 128))).astype(np.float16)
    q[:, :, 0] = slope * np.sqrt(128.0)
    own, okv = pool_of(cuda, rng, "int8", heads, 1)
    got = own.attention_shared(dev(q), i32(np.zeros((batch, 1))), i32([2] * batch), pre, i32(table), prefix)
    own.check()
    both, pick = np.concatenate([pkv, okv]), sorted({0, 1, batch // 2, batch - 1})
    counts = np.concatenate([counts, np.arange(64) < 2])
    want = np.stack([attention(q[b], both, counts) for b in pick])
    close(got[pick], want, [both], TOL16 + 256 * 8 * 2 * 2.0**-23 + 2 * 15 * 2.0**-23 * 37)


@pytest.mark.parametrize("batch", [4, 64, 1216])
@pytest.mark.parametrize("q0", [1.0, 300.0, -300.0, 60000.0, -60000.0])
def test_shared_logits_that_grow_far(cuda, batch, q0):
    """Keys 8 t and one loud query channel: references that pass 2^20 in the middle of a stretch of 16 tiles (or begin
    above it, or fall).  Neighbouring logits are 0.7 |q0| apart, so all but a few take no weight."""
    rng = np.random.default_rng(48)
    heads, prefix = 8, 2048
    kv = ko.rows(rng, prefix, heads, 0.1)
    kv[:, 0] = 0
    kv[:, 0, :, 0] = (8.0 * np.arange(prefix))[:, None]
    pre, pkv = pool_of(cuda, rng, "f16", heads, prefix // 64, kv)
    own, _ = pool_of(cuda, rng, "int8", heads, 1)
    q = np.zeros((batch, 4 * heads, 128), np.float16)
    q[:, :, 0] = q0
    q[:, 1::4, 0] = 0.001  # (a row of small logits beside them in each warp)
    got = own.attention_shared(dev(q), i32(np.zeros((batch, 1))), i32([0] * batch), pre, i32(np.arange(prefix // 64)),
                               prefix)
    own.check()
    pick = sorted({0, batch // 2, batch - 1})
    want = np.stack([attention(q[b], pkv, np.ones(prefix)) for b in pick])
    # (|logit| of a row whose neighbours count is below 2^11 |q0| = 1450: 15 roundings of 2^-23 each, twice)
    close(got[pick], want, [pkv], TOL16 + (2 * 15 * 2.0**-23 * 1450 if q0 == 1.0 else 0.0))
