"""The paged KV cache on the GPU (hsb_kv_*) against its definition in 64 bits
(tests/kv_oracle.py): written pages bit for bit, rows read back, attention of
ragged batches and of batches with a shared prefix.

Tolerances, relative to the largest |v| in the cache.
F32 attention: with S = sum |q k| / sqrt(128) < 16 and |logit| < 32 for these
inputs, a logit is off by 2^-22 S (q as two F16 halves), 12 * 2^-24 S (128
rounded additions, their usual growth) and 3 * 2^-24 |logit| (scales), and its
exp2 by 2^-22: 2e-5 in all, so the weighted mean by at most twice that, 4e-5.
F16 shared: a weight's rounding to F16 (2^-11) and the output's (2^-11) on top."""
from __future__ import annotations

import numpy as np
import pytest

import kv_oracle as ko

pytestmark = pytest.mark.gpu
TOL32 = 4e-5
TOL16 = 4e-5 + 2 * 2.0**-11


def dev(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def i32(a):
    return dev(np.asarray(a, dtype=np.int32))


def filled(rng, fmt, heads, lengths, gap=-1, junk=0xFF):
    """(pool bytes, table, K/V per sequence in 64 bits): unwritten bytes hold junk (NaN in every format)."""
    table, pages = ko.tables(rng, lengths, gap=gap)
    pool = np.full((pages, heads, ko.PAGE_BYTES[fmt]), junk, dtype=np.uint8)
    kvs = []
    for b, n in enumerate(lengths):
        kv = ko.rows(rng, int(n), heads)
        for t in range(int(n)):
            ko.write_rows(pool, fmt, table[b, t // 64], t % 64, kv[t])
        kvs.append(ko.stored(kv, fmt))
    return pool, table, kvs


def quick_fill(cuda, rng, fmt, heads, lengths, gap=-1):
    """As filled, written by the library's own append (tested below)."""
    table, pages = ko.tables(rng, lengths, gap=gap)
    cache = cuda.KVPages(kv_heads=heads, format=fmt,
                         data=dev(np.full((pages, heads, ko.PAGE_BYTES[fmt]), 0xFF, dtype=np.uint8)))
    kv = ko.rows(rng, int(sum(lengths)), heads)
    offs = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    if len(kv):
        cache.append(dev(kv), i32(table), i32(np.zeros(len(lengths))), offsets=i32(offs))
    cache.check()
    values = ko.stored(kv, fmt)
    return cache, table, [values[offs[b]:offs[b + 1]] for b in range(len(lengths))]


def close(got, want, kvs, tol):
    top = max([float(np.max(np.abs(kv[:, 1]))) for kv in kvs if len(kv)] + [1e-30])
    got = got.double().cpu().numpy()
    assert np.all(np.isfinite(got))
    err = float(np.max(np.abs(got - want))) / top
    assert err < tol, err


# ------------------------------------------------------------------- write
@pytest.mark.parametrize("fmt", ko.FORMATS)
@pytest.mark.parametrize("heads,counts,starts", [
    (8, [1, 1, 1], [0, 63, 64]), (2, [0, 70, 0, 5, 1], [3, 60, 9, 128, 0]), (1, [130], [1]), (4, [33, 2], [0, 62])])
def test_append_is_the_format_bit_for_bit(cuda, fmt, heads, counts, starts):
    rng = np.random.default_rng(heads * 100 + len(counts))
    lengths = [s + n for s, n in zip(starts, counts)]
    table, pages = ko.tables(rng, lengths)
    pool = rng.integers(0, 256, (pages, heads, ko.PAGE_BYTES[fmt]), dtype=np.uint8)
    want = pool.copy()
    before, after = 2, 3  # rows of no sequence
    kv = ko.rows(rng, before + sum(counts) + after, heads)
    offs = before + np.concatenate([[0], np.cumsum(counts)])
    for b, n in enumerate(counts):
        for i in range(n):
            t = starts[b] + i
            ko.write_rows(want, fmt, table[b, t // 64], t % 64, kv[offs[b] + i])
    cache = cuda.KVPages(kv_heads=heads, format=fmt, data=dev(pool))
    cache.append(dev(kv), i32(table), i32(starts), offsets=i32(offs))
    cache.check()
    assert np.array_equal(cache.data.cpu().numpy(), want)


@pytest.mark.parametrize("fmt", ko.FORMATS)
def test_append_one_row_each_from_the_models_tensor(cuda, fmt):
    """[n][8][K 128 | V 128], the executor's current KV, as a strided view; many rows too."""
    rng = np.random.default_rng(5)
    for n in (5, 2500):  # few rows and the wide variant
        starts = rng.integers(0, 128, n)
        table = rng.permutation(2 * n).astype(np.int32).reshape(n, 2)
        pool = np.zeros((2 * n, 8, ko.PAGE_BYTES[fmt]), dtype=np.uint8) if n < 100 else None
        current = ko.rows(rng, n, 8).transpose(0, 2, 1, 3).copy()  # [n][8][2][128]
        cache = cuda.KVPages(pages=2 * n, kv_heads=8, format=fmt)
        cache.data.zero_()
        cache.append(dev(current).transpose(1, 2), i32(table), i32(starts))
        cache.check()
        kv = current.transpose(0, 2, 1, 3)
        if pool is not None:
            for i in range(n):
                ko.write_rows(pool, fmt, table[i, starts[i] // 64], starts[i] % 64, kv[i])
            assert np.array_equal(cache.data.cpu().numpy(), pool)
        got = cache.read(i32(starts), i32(table), seqs=i32(np.arange(n))).cpu().numpy()
        assert np.array_equal(got, ko.read_back(ko.stored(kv, fmt)))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_edges(cuda, fmt):
    """Zero rows, subnormals, the largest finite value, every finite F16 once, and non-finite values."""
    every = np.arange(65536, dtype=np.uint32).astype(np.uint16).view(np.float16)
    every = every[np.isfinite(every)]
    pad = np.zeros((-len(every)) % 256, dtype=np.float16)
    kv = np.concatenate([every, pad]).reshape(-1, 2, 1, 128)
    kv = np.concatenate([kv, np.zeros((1, 2, 1, 128), np.float16), np.full((1, 2, 1, 128), 65504, np.float16)])
    n = len(kv)
    table = i32(np.arange(-(-n // 64))[None])
    cache = cuda.KVPages(pages=-(-n // 64), kv_heads=1, format=fmt)
    pos = i32(np.arange(n))
    cache.append(dev(kv), table, i32([0]), offsets=i32([0, n]))
    cache.check()
    got = cache.read(pos, table).cpu().numpy()
    assert np.array_equal(got.view(np.uint16), ko.read_back(ko.stored(kv, fmt)).view(np.uint16))
    bad = ko.rows(np.random.default_rng(1), 3, 1)
    bad[1, 0, 0, 7], bad[1, 1, 0, 3], bad[1, 1, 0, 4] = np.nan, np.inf, -np.inf
    cache.append(dev(bad), table, i32([0]), offsets=i32([0, 3]))
    with pytest.raises(cuda.HsbError, match="nonfinite F16") as e:
        cache.check()
    assert e.value.status == 111
    got = cache.read(pos[:3].contiguous(), table).cpu().numpy()
    want = ko.read_back(ko.stored(bad, fmt))
    assert np.array_equal(got, want) and got[1, 0, 0, 7] == 0 and got[1, 1, 0, 3] == -got[1, 1, 0, 4] > 0
    cache.check()  # the error was forgotten


@pytest.mark.parametrize("fmt", ko.FORMATS)
def test_append_outside_the_pool_writes_nothing(cuda, fmt):
    rng = np.random.default_rng(3)
    pool = rng.integers(0, 256, (4, 2, ko.PAGE_BYTES[fmt]), dtype=np.uint8)
    kv = ko.rows(rng, 4, 2)
    for table, starts, status in (([[0], [4], [-1], [1]], [0, 0, 0, 0], 121), ([[0], [2], [3], [1]], [0, 64, -1, 0], 122)):
        want = pool.copy()
        for b in (0, 3):
            ko.write_rows(want, fmt, table[b][0], 0, kv[b])
        cache = cuda.KVPages(kv_heads=2, format=fmt, data=dev(pool))
        cache.append(dev(kv), i32(table), i32(starts))
        with pytest.raises(cuda.InvalidArgument) as e:
            cache.check()
        assert e.value.status == status
        assert np.array_equal(cache.data.cpu().numpy(), want)


# -------------------------------------------------------------------- read
@pytest.mark.parametrize("fmt", ko.FORMATS)
def test_read_rows_of_several_sequences(cuda, fmt):
    import torch

    rng = np.random.default_rng(11)
    pool, table, kvs = filled(rng, fmt, 2, [70, 1, 128])
    cache = cuda.KVPages(kv_heads=2, format=fmt, data=dev(pool))
    seqs = np.array([2, 0, 0, 1, 2, 2, 0])
    pos = np.array([127, 69, 0, 0, 64, 64, 63])
    want = ko.read_back(np.stack([kvs[s][p] for s, p in zip(seqs, pos)]))
    got = cache.read(i32(pos), i32(table), seqs=i32(seqs))
    cache.check()
    assert np.array_equal(got.cpu().numpy(), want)
    # only the first *count rows are written
    out = torch.full((7, 2, 2, 128), 9.0, dtype=torch.float16, device="cuda")
    cache.read(i32(pos), i32(table), seqs=i32(seqs), count=i32([4]), out=out)
    assert np.array_equal(out[:4].cpu().numpy(), want[:4]) and bool((out[4:] == 9).all())
    # sequence 0 without seqs; rows outside are zero and reported
    got = cache.read(i32([0, 200, 69]), i32(table)).cpu().numpy()
    assert np.array_equal(got[[0, 2]], ko.read_back(kvs[0][[0, 69]])) and not got[1].any()
    with pytest.raises(cuda.InvalidArgument) as e:
        cache.check()
    assert e.value.status == 122
    got = cache.read(i32([0, 64]), i32(table), seqs=i32([3, 1])).cpu().numpy()  # no such sequence; page -1
    assert not got.any()
    with pytest.raises(cuda.InvalidArgument):
        cache.check()
    assert cache.read(i32([]), i32(table)).shape[0] == 0


def test_read_feeds_the_packed_attention(cuda, ob):
    """union -> read -> pack -> attention_packed: an 8-bit history behind the selected path."""
    import torch

    rng = np.random.default_rng(21)
    n, kk, count = 700, 90, 96
    cache, table, (kv,) = quick_fill(cuda, rng, "int8", 8, [n])
    ids = np.stack([rng.permutation(n)[:kk] for _ in range(32)]).astype(np.int32)
    sizes = i32([kk] * 32)
    physical = cuda.gqa_physical_union(dev(ids), sizes, n)
    payload = cache.read(physical, i32(table))
    k = torch.empty(count * 4096, dtype=torch.int16, device="cuda")
    v = torch.empty_like(k)
    cuda.pack_gqa_workspace(dev(ids), sizes, [n - 1], physical, payload.view(torch.uint8), count, k, v)
    q = rng.standard_normal((32, 128)).astype(np.float32)
    out = cuda.attention_packed(dev(q), k, v, count, sizes=sizes).cpu().numpy()
    half = ko.read_back(kv).astype(np.float64)
    for h in range(32):
        x = half[ids[h]]
        want = ko.attention(q[4 * (h // 4):4 * (h // 4) + 4], x[:, 0, h // 4][:, None], x[:, 1, h // 4][:, None])[h % 4]
        assert np.max(np.abs(out[h] - want)) < 2e-3 * np.max(np.abs(want))


# --------------------------------------------------------------- attention
def attend(cuda, cache, table, lengths, q):
    out = cache.attention(dev(q), i32(table), i32(lengths))
    cache.check()
    return out


@pytest.mark.parametrize("fmt", ko.FORMATS)
@pytest.mark.parametrize("heads,lengths", [
    (8, [77]), (1, [0, 1, 31, 32, 33, 0, 63, 64, 65, 130, 0]), (2, [1]), (4, [200, 3]), (8, [0, 0, 0])])
def test_attention_short(cuda, fmt, heads, lengths):
    rng = np.random.default_rng(len(lengths) + heads)
    pool, table, kvs = filled(rng, fmt, heads, lengths, gap=10**6)
    cache = cuda.KVPages(kv_heads=heads, format=fmt, data=dev(pool))
    q = rng.standard_normal((len(lengths), 4 * heads, 128)).astype(np.float32)
    want = np.stack([ko.attention(q[b], kv[:, 0], kv[:, 1]) for b, kv in enumerate(kvs)])
    got = attend(cuda, cache, table, lengths, q)
    close(got, want, kvs, TOL32)
    for b, n in enumerate(lengths):
        if n == 0:
            assert not got[b].any()


@pytest.mark.parametrize("fmt", ko.FORMATS)
@pytest.mark.parametrize("heads,lengths", [
    (8, [20011]), (1, [9000, 0, 64 * 150, 1]), (2, list(range(1, 1200, 4))), (8, [500, 1, 2048, 0, 777, 4096])])
def test_attention_across_stretches(cuda, fmt, heads, lengths):
    """Runs that cross CTAs, many runs in one, long and short together."""
    rng = np.random.default_rng(sum(lengths) % 1000)
    cache, table, kvs = quick_fill(cuda, rng, fmt, heads, lengths)
    q = rng.standard_normal((len(lengths), 4 * heads, 128)).astype(np.float32)
    want = np.stack([ko.attention(q[b], kv[:, 0], kv[:, 1]) for b, kv in enumerate(kvs)])
    got = attend(cuda, cache, table, lengths, q)
    close(got, want, kvs, TOL32)
    again = attend(cuda, cache, table, lengths, q)
    assert bool((got == again).all())  # no order depends on timing


@pytest.mark.parametrize("fmt", ko.FORMATS)
@pytest.mark.parametrize("kv_scale,q_scale", [(1e-5, 1.0), (3000.0, 1e-4), (1.0, 1e-6)])
def test_attention_range(cuda, fmt, kv_scale, q_scale):
    """Small and large values keep their relative accuracy (logits stay below 32)."""
    rng = np.random.default_rng(8)
    lengths = [150]
    table, pages = ko.tables(rng, lengths)
    kv = ko.rows(rng, 150, 2, kv_scale)
    cache = cuda.KVPages(pages=pages, kv_heads=2, format=fmt)
    cache.append(dev(kv), i32(table), i32([0]), offsets=i32([0, 150]))
    values = ko.stored(kv, fmt)
    q = (rng.standard_normal((1, 8, 128)) * q_scale).astype(np.float32)
    q[0, 3] *= 100.0  # one head well above the rest of its group
    want = ko.attention(q[0], values[:, 0], values[:, 1])[None]
    close(attend(cuda, cache, table, lengths, q), want, [values], TOL32)


def test_attention_growing_maximum(cuda):
    """Logits that rise along the sequence: every tile changes the running maximum."""
    rng = np.random.default_rng(2)
    n = 640
    kv = ko.rows(rng, n, 1, 0.1)
    kv[:, 0] += (np.arange(n)[:, None, None] * 0.02).astype(np.float16)
    kv[:, 1] *= (1.0 + np.arange(n)[:, None, None]).astype(np.float16)  # V scales rise too
    q = np.full((1, 4, 128), 0.25, dtype=np.float32)
    for fmt in ko.FORMATS:
        table, pages = ko.tables(rng, [n])
        cache = cuda.KVPages(pages=pages, kv_heads=1, format=fmt)
        cache.append(dev(kv), i32(table), i32([0]), offsets=i32([0, n]))
        values = ko.stored(kv, fmt)
        want = ko.attention(q[0], values[:, 0], values[:, 1])[None]
        close(attend(cuda, cache, table, [n], q), want, [values], TOL32)


@pytest.mark.parametrize("fmt", ko.FORMATS)
def test_attention_bad_tables(cuda, fmt):
    """A page outside the pool leaves its tokens out; a length behind the table counts as none."""
    rng = np.random.default_rng(4)
    pool, table, kvs = filled(rng, fmt, 2, [200, 130, 64])
    q = rng.standard_normal((3, 8, 128)).astype(np.float32)
    cache = cuda.KVPages(kv_heads=2, format=fmt, data=dev(pool))
    broken = table.copy()
    broken[0, 1], broken[1, 2], broken[2, 0] = len(pool), -7, 2**31 - 1
    left = [np.delete(kvs[0], np.s_[64:128], 0), kvs[1][:128], kvs[2][:0]]
    want = np.stack([ko.attention(q[b], kv[:, 0], kv[:, 1]) for b, kv in enumerate(left)])
    got = cache.attention(dev(q), i32(broken), i32([200, 130, 64]))
    close(got, want, kvs, TOL32)
    with pytest.raises(cuda.InvalidArgument) as e:
        cache.check()
    assert e.value.status == 121
    got = cache.attention(dev(q), i32(table), i32([257, -1, 64]))
    want = np.stack([want[0] * 0, want[1] * 0, ko.attention(q[2], kvs[2][:, 0], kvs[2][:, 1])])
    close(got, want, kvs, TOL32)
    with pytest.raises(cuda.InvalidArgument) as e:
        cache.check()
    assert e.value.status == 122


@pytest.mark.parametrize("width", [5, 12, 13, 40])
def test_attention_is_the_same_however_the_work_is_split(cuda, width):
    """A wider table (of unused entries) makes the same runs whole CTAs' or stretches' work: only the
    order of the last sums differs."""
    rng = np.random.default_rng(35)
    lengths = [300, 0, 64, 1]
    cache, table, kvs = quick_fill(cuda, rng, "e4m3", 4, lengths, gap=7)
    table = np.concatenate([table, np.full((4, width - table.shape[1]), -5, np.int32)], 1)
    q = rng.standard_normal((4, 16, 128)).astype(np.float32)
    want = np.stack([ko.attention(q[b], kv[:, 0], kv[:, 1]) for b, kv in enumerate(kvs)])
    close(attend(cuda, cache, table, lengths, q), want, kvs, TOL32)


@pytest.mark.parametrize("fmt", ko.FORMATS)
def test_attention_many_sequences(cuda, fmt):
    """More sequences than lanes, warps or CTAs, most of them empty or a token long."""
    rng = np.random.default_rng(31)
    lengths = np.where(rng.random(5000) < 0.4, 0, rng.integers(1, 4, 5000))
    lengths[[17, 4999]] = 130, 200
    cache, table, kvs = quick_fill(cuda, rng, fmt, 1, lengths)
    q = rng.standard_normal((5000, 4, 128)).astype(np.float32)
    want = np.stack([ko.attention(q[b], kv[:, 0], kv[:, 1]) for b, kv in enumerate(kvs)])
    close(attend(cuda, cache, table, lengths, q), want, kvs, TOL32)


@pytest.mark.parametrize("factor", [1e30, 2e36])
def test_attention_huge_queries(cuda, factor):
    """Logits far above F16's and exp's range: the largest takes all the weight."""
    rng = np.random.default_rng(32)
    cache, table, kvs = quick_fill(cuda, rng, "f16", 1, [100])
    q = (rng.standard_normal((1, 4, 128)) * factor).astype(np.float32)
    want = np.stack([ko.attention(q[0].astype(np.float64), kvs[0][:, 0], kvs[0][:, 1])])
    close(attend(cuda, cache, table, [100], q), want, kvs, TOL32)


def test_attention_nan_query_stays_in_its_head(cuda):
    rng = np.random.default_rng(6)
    cache, table, kvs = quick_fill(cuda, rng, "int8", 1, [100])
    q = rng.standard_normal((1, 4, 128)).astype(np.float32)
    want = ko.attention(q[0], kvs[0][:, 0], kvs[0][:, 1])
    q[0, 2, 5] = np.nan
    got = cache.attention(dev(q), i32(table), i32([100])).cpu().numpy()[0]
    assert np.isnan(got[2]).all()
    keep = [0, 1, 3]
    assert np.max(np.abs(got[keep] - want[keep])) < TOL32 * np.max(np.abs(kvs[0][:, 1]))


def test_offsets_behind_4_gib(cuda):
    """Pages whose byte offset passes 32 bits, written, read and attended."""
    import torch

    pages = (5 << 30) // 32768
    cache = cuda.KVPages(pages=pages, kv_heads=1, format="f16")
    rng = np.random.default_rng(9)
    kv = ko.rows(rng, 130, 1)
    table = np.array([[pages - 1, 3, pages - 2]], dtype=np.int32)
    cache.append(dev(kv), i32(table), i32([0]), offsets=i32([0, 130]))
    assert np.array_equal(cache.read(i32(np.arange(130)), i32(table)).cpu().numpy(), kv)
    q = rng.standard_normal((1, 4, 128)).astype(np.float32)
    values = kv.astype(np.float64)
    want = ko.attention(q[0], values[:, 0], values[:, 1])[None]
    close(attend(cuda, cache, table, [130], q), want, [values], TOL32)
    q16 = dev(q.astype(np.float16))
    got = cache.attention_shared(q16, i32([[0]]), i32([0]), cache, i32(table[0]), 130)
    want = ko.attention(q[0].astype(np.float16), values[:, 0], values[:, 1])[None]
    close(got, want, [values], TOL16)
    del cache
    torch.cuda.empty_cache()


# ------------------------------------------------------------ shared prefix
def shared_case(cuda, seed, fmt, heads, prefix, lengths):
    rng = np.random.default_rng(seed)
    cache, table, kvs = quick_fill(cuda, rng, fmt, heads, lengths)
    pre, ptable, (pkv,) = quick_fill(cuda, rng, "f16", heads, [prefix])
    q = rng.standard_normal((len(lengths), 4 * heads, 128)).astype(np.float16)
    whole = [np.concatenate([pkv, kv]) for kv in kvs]
    want = np.stack([ko.attention(q[b], kv[:, 0], kv[:, 1]) for b, kv in enumerate(whole)])
    got = cache.attention_shared(dev(q), i32(table), i32(lengths), pre, i32(ptable[0]), prefix)
    cache.check()
    return got, want, whole


@pytest.mark.parametrize("fmt", ko.FORMATS)
@pytest.mark.parametrize("heads,prefix,lengths", [
    (8, 130, [5, 0, 64]), (1, 1, [0]), (2, 64, [1, 70]), (4, 63, [0] * 5), (1, 65, list(range(40)))])
def test_shared_small(cuda, fmt, heads, prefix, lengths):
    got, want, whole = shared_case(cuda, prefix, fmt, heads, prefix, lengths)
    close(got, want, whole, TOL16)


@pytest.mark.parametrize("heads,prefix,lengths", [
    (8, 5000, [3, 500, 0, 64, 129]), (1, 40001, [9] * 32), (2, 4096, list(range(33))), (8, 1000, [7] * 64),
    (1, 3001, [1] * 150), (4, 257, [200] * 65), (8, 200, [0, 1, 2] * 500), (2, 700, [3] * 97), (8, 64, [1] * 600)])
def test_shared_large(cuda, heads, prefix, lengths):
    got, want, whole = shared_case(cuda, prefix, "int8", heads, prefix, lengths)
    close(got, want, whole, TOL16)


def test_shared_growing_maximum(cuda):
    """Prefix logits that rise by hundreds along the prefix, own tokens above and below them."""
    rng = np.random.default_rng(12)
    n, heads = 900, 1
    pkv = ko.rows(rng, n, heads, 0.1)
    pkv[:, 0] += (np.arange(n)[:, None, None] * 0.05).astype(np.float16)
    table, pages = ko.tables(rng, [n])
    pre = cuda.KVPages(pages=pages, kv_heads=heads, format="f16")
    pre.append(dev(pkv), i32(table), i32([0]), offsets=i32([0, n]))
    cache, own, kvs = quick_fill(cuda, rng, "int8", heads, [20, 0, 3])
    # every second sequence's logits fall along the prefix instead
    q = np.stack([np.full((4, 128), s, dtype=np.float16) for s in (0.5, -0.5, 0.01)])
    pk = pkv.astype(np.float64)
    whole = [np.concatenate([pk, kv]) for kv in kvs]
    want = np.stack([ko.attention(q[b], kv[:, 0], kv[:, 1]) for b, kv in enumerate(whole)])
    got = cache.attention_shared(dev(q), i32(own), i32([20, 0, 3]), pre, i32(table[0]), n)
    # |logit| reaches 256 here: 3 * 2^-24 * 256 + 12 * 2^-24 * 256 is 2.3e-4 a weight
    close(got, want, whole, TOL16 + 2 * 2.3e-4)
    # the same for a batch of three M tiles, whose CTAs take several stretches
    many = 70
    table70, lengths = i32(np.zeros((many, 1))), i32(np.zeros(many))
    got = cache.attention_shared(dev(np.tile(q, (24, 1, 1))[:many]), table70, lengths, pre, i32(table[0]), n)
    want = [ko.attention(q[b], pk[:, 0], pk[:, 1]) for b in range(3)]
    close(got, np.stack([want[b % 3] for b in range(many)]), [pk], TOL16 + 2 * 2.3e-4)


def test_shared_nan_query_stays_in_its_row(cuda):
    rng = np.random.default_rng(33)
    cache, own, kvs = quick_fill(cuda, rng, "int8", 1, [10, 0, 5])
    pre, table, (pkv,) = quick_fill(cuda, rng, "f16", 1, [200])
    q = rng.standard_normal((3, 4, 128)).astype(np.float16)
    whole = [np.concatenate([pkv, kv]) for kv in kvs]
    want = np.stack([ko.attention(q[b], kv[:, 0], kv[:, 1]) for b, kv in enumerate(whole)])
    q[1, 2, 100] = np.nan
    got = cache.attention_shared(dev(q), i32(own), i32([10, 0, 5]), pre, i32(table[0]), 200).double().cpu().numpy()
    assert np.isnan(got[1, 2]).all()
    got[1, 2] = want[1, 2]
    assert np.max(np.abs(got - want)) < TOL16 * np.max(np.abs(pkv[:, 1]))


@pytest.mark.parametrize("batch", [3, 40])
def test_shared_nonfinite_keys(cuda, batch):
    """A NaN key anywhere in the prefix is NaN in every row of its head and no other's; an infinite one is NaN
    where its logit is +infinity and takes no weight where it is -infinity."""
    rng = np.random.default_rng(35)
    cache, own, _ = quick_fill(cuda, rng, "int8", 2, [0] * batch)
    pre, table, (pkv,) = quick_fill(cuda, rng, "f16", 2, [200])
    table = i32(table)
    q = rng.standard_normal((batch, 8, 128)).astype(np.float16)
    top = TOL16 * np.max(np.abs(pkv[:, 1]))
    rows = pkv.astype(np.float16)
    for t in list(range(9)) + [62, 63, 64, 65, 127, 128, 130, 199]:
        for value in (np.nan, np.inf):
            row = rows[t:t + 1].copy()
            row[0, 0, 1, 5] = value
            pre.append(dev(row), table, i32([t]))
            got = cache.attention_shared(dev(q), i32(own), i32([0] * batch), pre, table[0], 200).double().cpu().numpy()
            pre.append(dev(rows[t:t + 1].copy()), table, i32([t]))
            for b in range(batch):
                want = ko.attention(q[b, :4], pkv[:, 0, :1], pkv[:, 1, :1])
                assert np.max(np.abs(got[b, :4] - want)) < top
                gone = ko.attention(q[b, 4:], np.delete(pkv[:, 0, 1:], t, 0), np.delete(pkv[:, 1, 1:], t, 0))
                for h in range(4):
                    if np.isnan(value) or q[b, 4 + h, 5] > 0:
                        assert np.isnan(got[b, 4 + h]).all(), (t, value, b, h)
                    else:
                        assert np.max(np.abs(got[b, 4 + h] - gone[h])) < top, (t, value, b, h)
    pre.status.zero_()  # (the non-finite rows were reported)


@pytest.mark.parametrize("lengths", [[77, 200, 5], [3000, 4000, 100]])
@pytest.mark.parametrize("part", [0, 1])
def test_attention_nan_rows_stay_in_their_sequence(cuda, part, lengths):
    """A NaN in K or V of one token: that sequence's rows of that KV head, all NaN (K) or in that channel (V)."""
    rng = np.random.default_rng(36)
    cache, table, kvs = quick_fill(cuda, rng, "f16", 2, lengths)
    q = rng.standard_normal((3, 8, 128)).astype(np.float32)
    want = np.stack([ko.attention(q[b], kv[:, 0], kv[:, 1]) for b, kv in enumerate(kvs)])
    top = TOL32 * max(np.max(np.abs(kv[:, 1])) for kv in kvs)
    for t in (0, 1, 31, 32, 63, 64, lengths[1] - 1):
        row = kvs[1][t:t + 1].astype(np.float16)
        bad = row.copy()
        bad[0, part, 1, 9] = np.nan
        cache.append(dev(bad), i32(table[1:2]), i32([t]))
        got = cache.attention(dev(q), i32(table), i32(lengths)).double().cpu().numpy()
        cache.append(dev(row), i32(table[1:2]), i32([t]))
        lost = got[1, 4:] if part == 0 else got[1, 4:, 9]
        assert np.isnan(lost).all(), t
        lost[...] = want[1, 4:] if part == 0 else want[1, 4:, 9]
        assert np.max(np.abs(got - want)) < top, t
    cache.status.zero_()


def test_shared_padded_batch_and_long_own_lengths(cuda):
    """A padded batch (no own tokens, any query) beside one far longer own history than the prefix;
    a length behind the table counts as none and is reported."""
    rng = np.random.default_rng(34)
    lengths = [9000, 0, 0, 1, 0]
    got, want, whole = shared_case(cuda, 34, "e4m3", 2, 70, lengths)
    close(got, want, whole, TOL16)
    cache, own, kvs = quick_fill(cuda, rng, "f16", 2, [64, 64])
    pre, table, (pkv,) = quick_fill(cuda, rng, "f16", 2, [65])
    q = rng.standard_normal((2, 8, 128)).astype(np.float16)
    got = cache.attention_shared(dev(q), i32(own), i32([65, 64]), pre, i32(table[0]), 65)
    whole = [pkv, np.concatenate([pkv, kvs[1]])]
    close(got, np.stack([ko.attention(q[b], kv[:, 0], kv[:, 1]) for b, kv in enumerate(whole)]), whole, TOL16)
    with pytest.raises(cuda.InvalidArgument) as e:
        cache.check()
    assert e.value.status == 122


def test_shared_bad_prefix_page(cuda):
    rng = np.random.default_rng(13)
    cache, own, kvs = quick_fill(cuda, rng, "f16", 2, [10, 0])
    pre, table, (pkv,) = quick_fill(cuda, rng, "f16", 2, [300])
    q = rng.standard_normal((2, 8, 128)).astype(np.float16)
    broken = table[0].copy()
    broken[2] = -1
    left = np.delete(pkv, np.s_[128:192], 0)
    whole = [np.concatenate([left, kv]) for kv in kvs]
    want = np.stack([ko.attention(q[b], kv[:, 0], kv[:, 1]) for b, kv in enumerate(whole)])
    got = cache.attention_shared(dev(q), i32(own), i32([10, 0]), pre, i32(broken), 300)
    close(got, want, whole, TOL16)
    with pytest.raises(cuda.InvalidArgument) as e:
        cache.check()
    assert e.value.status == 121


@pytest.mark.parametrize("batch", [3, 64, 100])
@pytest.mark.parametrize("bad", [range(1, 24), range(0, 24, 2), range(0, 23), range(5, 7)])
def test_shared_many_bad_prefix_pages(cuda, batch, bad):
    """Tiles that are cleaned one after the other, faster than their products are issued."""
    rng = np.random.default_rng(38)
    heads, n = 2, 24 * 64 - 10
    pre, table, (pkv,) = quick_fill(cuda, rng, "f16", heads, [n])
    broken = table[0].copy()
    broken[list(bad)] = -1
    left = np.concatenate([pkv[i * 64:i * 64 + 64] for i in range(24) if i not in bad])
    cache, own, _ = quick_fill(cuda, rng, "int8", heads, [0] * batch)
    q = rng.standard_normal((batch, 4 * heads, 128)).astype(np.float16)
    want = np.stack([ko.attention(q[b], left[:, 0], left[:, 1]) for b in range(batch)])
    got = cache.attention_shared(dev(q), i32(own), i32([0] * batch), pre, i32(broken), n)
    close(got, want, [left], TOL16)
    with pytest.raises(cuda.InvalidArgument) as e:
        cache.check()
    assert e.value.status == 121


@pytest.mark.parametrize("prefix", [40, 170, 300])
def test_shared_ragged_prefix_of_many_runs(cuda, prefix):
    """Several short runs a CTA, each with a ragged last tile."""
    rng = np.random.default_rng(39)
    batch, heads = 1500, 8
    pre, table, (pkv,) = quick_fill(cuda, rng, "f16", heads, [prefix])
    cache, own, _ = quick_fill(cuda, rng, "int8", heads, [0] * batch)
    q = rng.standard_normal((batch, 4 * heads, 128)).astype(np.float16)
    want = np.stack([ko.attention(q[b], pkv[:, 0], pkv[:, 1]) for b in range(0, batch, 37)])
    got = cache.attention_shared(dev(q), i32(own), i32([0] * batch), pre, i32(table[0]), prefix)
    cache.check()
    close(got[::37], want, [pkv], TOL16)


# ---------------------------------------------------------- as used together
@pytest.mark.parametrize("fmt", ko.FORMATS)
def test_decode_steps_captured_and_eager(cuda, fmt):
    """A decode loop -- append, attend, attend behind a shared prefix -- eagerly on a
    stream of its own and as one captured graph replayed with lengths that grow."""
    import torch

    rng = np.random.default_rng(17)
    heads, batch, steps, prefix = 2, 5, 70, 150
    start = np.array([0, 63, 10, 128, 1])
    table, pages = ko.tables(rng, start + steps)
    pre, ptable, (pkv,) = quick_fill(cuda, rng, "f16", heads, [prefix])
    held = [ko.rows(rng, int(n), heads) for n in start]
    new = ko.rows(rng, steps * batch, heads).reshape(steps, batch, 2, heads, 128)
    qs = rng.standard_normal((steps, batch, 4 * heads, 128)).astype(np.float32)

    def fresh():
        c = cuda.KVPages(pages=pages, kv_heads=heads, format=fmt)
        c.data.fill_(0xFF)
        offs = np.concatenate([[0], np.cumsum(start)])
        c.append(dev(np.concatenate(held)), i32(table), i32(np.zeros(batch)), offsets=i32(offs))
        return c

    dt, dp = i32(table), i32(ptable[0])
    eager, other = fresh(), torch.cuda.Stream()
    kv_in, q_in = dev(new[0]), dev(qs[0])
    at, length = i32(start), i32(start + 1)
    graph, replayed = torch.cuda.CUDAGraph(), fresh()
    torch.cuda.synchronize()

    def step(c, kv, q, begin, n, **kw):
        c.append(kv, dt, begin, **kw)
        return c.attention(q, dt, n, **kw), c.attention_shared(q.half(), dt, n, pre, dp, prefix, **kw)

    with torch.cuda.graph(graph):
        g_out = step(replayed, kv_in, q_in, at, length)
    for i in range(steps):
        kv_in.copy_(dev(new[i]))
        q_in.copy_(dev(qs[i]))
        at.copy_(i32(start + i))
        length.copy_(i32(start + i + 1))
        graph.replay()
        torch.cuda.synchronize()
        args = dev(new[i]), dev(qs[i]), i32(start + i), i32(start + i + 1)
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            out = step(eager, *args)
        other.synchronize()
        for a, b in zip(out, g_out):
            assert bool((a == b).all())
        if i % 23 == 0:
            for b in range(batch):
                kv = ko.stored(np.concatenate([held[b], new[:i + 1, b]]), fmt)
                want = ko.attention(qs[i, b], kv[:, 0], kv[:, 1])
                close(out[0][b], want, [kv], TOL32)
                both = np.concatenate([pkv, kv])
                want = ko.attention(qs[i, b].astype(np.float16), both[:, 0], both[:, 1])
                close(out[1][b], want, [both], TOL16)
    eager.check()
    replayed.check()
    assert bool((eager.data == replayed.data).all())


def test_mirror_refuses_wrong_tensors(cuda):
    import torch

    cache = cuda.KVPages(4, kv_heads=2, format="int8")
    half = cuda.KVPages(4, kv_heads=2, format="f16")
    q, table, n = dev(np.zeros((3, 8, 128), np.float32)), i32(np.zeros((3, 2))), i32([0, 0, 0])
    rows = dev(np.zeros((3, 2, 2, 128), np.float16))
    for call in (lambda: cache.attention(q.half(), table, n), lambda: cache.attention(q[:2], table, n),
                 lambda: cache.attention(q.cpu(), table, n), lambda: cache.attention(q, table.long(), n),
                 lambda: cache.attention(q, table.T.contiguous().T, n), lambda: cache.attention(q, table[:, :0], n),
                 lambda: cache.attention(q, table, n[:2]), lambda: cache.attention(q, table, n, out=q),
                 lambda: cache.attention(q, table, n, out=torch.empty_like(q, dtype=torch.float16)),
                 lambda: cache.append(rows[:2], table, n), lambda: cache.append(rows.float(), table, n),
                 lambda: cache.append(rows[..., ::2], table, n), lambda: cache.append(rows, table, n, offsets=n),
                 lambda: cache.append(rows[:0], table, n),
                 lambda: cache.append(torch.zeros(3 * 513, dtype=torch.float16, device="cuda").view(3, 513)[:, 1:].view(3, 2, 2, 128), table, n),
                 lambda: cache.read(n.long(), table), lambda: cache.read(n, table, seqs=n[:2]),
                 lambda: cache.read(n, table, count=n), lambda: cache.read(n, table[0]),
                 lambda: cache.attention_shared(q, table, n, half, i32([0]), 64),
                 lambda: cache.attention_shared(q.half(), table, n, cache, i32([0]), 64),
                 lambda: cache.attention_shared(q.half(), table, n, half, i32([0]), 65),
                 lambda: cache.attention_shared(q.half(), table, n, half, i32([0]), 0)):
        with pytest.raises(cuda.InvalidArgument):
            call()
    cache.append(rows[:0], table, n, offsets=i32([0, 0, 0, 0]))  # no rows at all is not an error
    cache.check()


def test_calls_on_two_streams_at_once(cuda):
    """Two batches in flight on two streams, each call with memory of its own."""
    import torch

    rng = np.random.default_rng(19)
    streams = [torch.cuda.Stream() for _ in range(2)]
    cases, outs = [], []
    for i in range(2):
        lengths = [3000 + 17 * i, 5, 0, 900]
        cache, table, kvs = quick_fill(cuda, rng, "int8", 2, lengths)
        q = rng.standard_normal((4, 8, 128)).astype(np.float32)
        cases.append((cache, i32(table), i32(lengths), dev(q), kvs, q))
    torch.cuda.synchronize()
    for _ in range(20):
        for s, (cache, table, lengths, q, _, _) in zip(streams, cases):
            outs.append(cache.attention(q, table, lengths, stream=s))
    torch.cuda.synchronize()
    for n, out in enumerate(outs):
        _, _, _, _, kvs, q = cases[n % 2]
        want = np.stack([ko.attention(q[b], kv[:, 0], kv[:, 1]) for b, kv in enumerate(kvs)])
        close(out, want, kvs, TOL32)
