"""The paged KV cache on the CPU: the oracle's own formats against torch's
conversions, the library's refusals (before any CUDA work), and the even
split of work that the attention kernels share."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import kv_oracle as ko

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def lib():
    from hillserve_b200 import _capi

    return _capi.lib()


def test_e4m3_of_the_oracle():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().double().numpy()
    assert np.array_equal(codes, ko.E4M3, equal_nan=True)
    x = np.concatenate([np.linspace(-448, 448, 100001), ko.E4M3[:126], (ko.E4M3[:126] + ko.E4M3[1:127]) / 2, [-0.0]])
    want = torch.from_numpy(x.astype(np.float32)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(ko.e4m3_round(x.astype(np.float32)), want)


@pytest.mark.parametrize("fmt,rel", [("int8", 0.5 / 127), ("e4m3", 2.0**-4)])
def test_quantised_values_are_near(fmt, rel):
    """int8: half a step of max|x| / 127; e4m3: half a step of the value, or of its smallest step.
    The three F32 roundings (both quotients, the product) move a border by up to
    127 * 3 * 2^-24 steps: a share of 4.6e-5 of half a step."""
    x = ko.rows(np.random.default_rng(0), 50, 2)
    got, x64 = ko.stored(x, fmt), x.astype(np.float64)
    top = np.max(np.abs(x64), axis=-1, keepdims=True)
    bound = rel * top if fmt == "int8" else np.maximum(rel * np.abs(x64), 2.0**-10 * top / 448)
    assert np.all(np.abs(got - x64) <= bound * (1 + 4.6e-5))


def test_page_bytes(lib):
    assert [lib.hsb_kv_page_bytes(f) for f in (0, 1, 2)] == [ko.PAGE_BYTES[f] for f in ko.FORMATS]
    assert lib.hsb_kv_page_bytes(3) == lib.hsb_kv_page_bytes(-1) == 0


P, O = C.c_void_p(0x10000), C.c_void_p(0x20000)


def pool(data=0x10000, pages=4, fmt=1, heads=8):
    from hillserve_b200._capi import KvPages

    return C.byref(KvPages(data, pages, fmt, heads))


BAD_POOLS = [dict(data=0), dict(data=0x10008), dict(pages=0), dict(pages=1 << 31), dict(fmt=3), dict(fmt=-1),
             dict(heads=3), dict(heads=0), dict(heads=16)]


@pytest.mark.parametrize("bad", BAD_POOLS)
def test_bad_pools_are_refused(lib, bad):
    p = pool(**bad)
    assert lib.hsb_kv_append(p, P, 4, 2, P, None, P, P, 2, 2048, 128, None, None) == 120
    assert lib.hsb_kv_read(p, P, 4, 2, None, P, None, 5, P, None, None) == 120
    assert lib.hsb_kv_attention(p, P, 4, P, 2, P, P, P, 1 << 30, None, None) == 120
    assert lib.hsb_kv_attention_shared(p, P, 64, pool(), P, 4, P, 2, P, P, P, 1 << 30, None, None) == 120
    assert lib.hsb_kv_attention_shared(pool(fmt=0), P, 64, p, P, 4, P, 2, P, P, P, 1 << 30, None, None) == 120
    assert lib.hsb_last_error() == b"paged KV pool arguments"


def test_null_pools_are_refused(lib):
    assert lib.hsb_kv_append(None, P, 4, 2, P, None, P, P, 2, 2048, 128, None, None) == 120
    assert lib.hsb_kv_attention(None, P, 4, P, 2, P, P, P, 1 << 30, None, None) == 120


def call(lib, name, good, **change):
    args = dict(good)
    args.update(change)
    return getattr(lib, name)(*args.values())


def test_append_refusals(lib):
    good = dict(pages=pool(), table=P, width=4, batch=2, starts=P, offsets=None, k=P, v=P, rows=2, row=2048, head=128,
                status=None, stream=None)
    odd = C.c_void_p(0x10008)
    for change in (dict(table=None), dict(width=0), dict(batch=0), dict(starts=None), dict(k=None), dict(v=None),
                   dict(rows=0), dict(rows=3), dict(rows=1 << 31, offsets=P)):
        assert call(lib, "hsb_kv_append", good, **change) == 120, change
        assert lib.hsb_last_error() == b"paged KV append shape"
    for change in (dict(k=odd), dict(v=odd), dict(row=2044), dict(head=4)):
        assert call(lib, "hsb_kv_append", good, **change) == 120, change
        assert lib.hsb_last_error() == b"paged KV rows must be 16-byte aligned"
    for change in (dict(table=C.c_void_p(0x10002)), dict(starts=C.c_void_p(0x10001)),
                   dict(offsets=C.c_void_p(0x10002)), dict(status=C.c_void_p(0x10004))):
        assert call(lib, "hsb_kv_append", good, **change) == 120, change
        assert lib.hsb_last_error() == b"paged KV tables are misaligned"


def test_read_refusals(lib):
    good = dict(pages=pool(), table=P, width=4, batch=2, seqs=None, positions=P, count=None, rows=5, out=P, status=None,
                stream=None)
    for change in (dict(table=None), dict(width=0), dict(batch=0), dict(positions=None), dict(out=None), dict(rows=0),
                   dict(rows=1 << 31), dict(out=C.c_void_p(0x10002)), dict(seqs=C.c_void_p(0x10002)),
                   dict(positions=C.c_void_p(0x10001)), dict(count=C.c_void_p(0x10002)), dict(status=C.c_void_p(0x10004))):
        assert call(lib, "hsb_kv_read", good, **change) == 120, change


def test_attention_refusals(lib):
    size = lib.hsb_kv_attention_workspace_bytes(2, 8)
    good = dict(pages=pool(), table=P, width=4, lengths=P, batch=2, q=P, out=O, ws=P, size=size, status=None, stream=None)
    for change in (dict(table=None), dict(width=0), dict(lengths=None), dict(batch=0), dict(batch=(1 << 20) + 1),
                   dict(q=None), dict(out=None), dict(width=1 << 32), dict(width=1 << 27, batch=2),
                   dict(q=C.c_void_p(0x10008)), dict(out=C.c_void_p(0x20008)), dict(ws=C.c_void_p(0x10008)),
                   dict(table=C.c_void_p(0x10002)), dict(lengths=C.c_void_p(0x10002)), dict(status=C.c_void_p(0x10004)),
                   dict(out=P)):
        assert call(lib, "hsb_kv_attention", good, **change) == 120, change
    assert call(lib, "hsb_kv_attention", good, size=size - 1) == 3
    assert call(lib, "hsb_kv_attention", good, ws=None) == 3


def test_shared_refusals(lib):
    size = lib.hsb_kv_attention_shared_workspace_bytes(2, 8, 64)
    good = dict(prefix=pool(fmt=0), ptable=P, tokens=64, pages=pool(), table=P, width=4, lengths=P, batch=2, q=P, out=O,
                ws=P, size=size, status=None, stream=None)
    for change in (dict(prefix=pool(fmt=1)), dict(prefix=pool(fmt=0, heads=4)), dict(ptable=None), dict(tokens=0),
                   dict(table=None), dict(width=0), dict(lengths=None), dict(batch=0), dict(q=None), dict(out=None),
                   dict(q=C.c_void_p(0x10008)), dict(out=C.c_void_p(0x20008)), dict(ws=C.c_void_p(0x10008)),
                   dict(ptable=C.c_void_p(0x10002)), dict(batch=(1 << 20) + 1), dict(tokens=(1 << 30) + 1), dict(out=P)):
        assert call(lib, "hsb_kv_attention_shared", good, **change) == 120, change
    assert call(lib, "hsb_kv_attention_shared", good, size=size - 1) == 3
    assert call(lib, "hsb_kv_attention_shared", good, ws=None) == 3


def test_messages(lib):
    for code in (120, 121, 122):
        assert lib.hsb_status_message(code).startswith(b"paged KV ")


class Split:
    """The even split of kvattention.cuh, restated."""

    def __init__(self, units, n):
        self.each, self.more = units // n, units % n

    def begin(self, c):
        return self.each * c + min(c, self.more)

    def of(self, u):
        longer = (self.each + 1) * self.more
        return u // (self.each + 1) if u < longer else self.more + (u - longer) // self.each


@pytest.mark.parametrize("units", [1, 2, 7, 147, 148, 149, 1000, 4096 * 8 + 3])
@pytest.mark.parametrize("n", [1, 2, 16, 148])
def test_every_unit_has_the_stretch_that_holds_it(units, n):
    """The split's two formulas agree, so a run's folder finds its parts; empty stretches are the last ones."""
    s = Split(units, n)
    for u in {0, units - 1, units // 2, units // 3, min(units - 1, 5)}:
        assert 0 <= s.of(u) < n and s.begin(s.of(u)) <= u < s.begin(s.of(u) + 1)
    sizes = [s.begin(c + 1) - s.begin(c) for c in range(n)]
    assert s.begin(n) == units and sizes == sorted(sizes, reverse=True) and sizes[0] - sizes[-1] <= 1


def test_mirror_refusals():
    import hillserve_b200 as hsb

    with pytest.raises(hsb.InvalidArgument, match="unknown paged KV format"):
        hsb.KVPages(4, format="fp8", device="cpu")
    with pytest.raises(hsb.InvalidArgument, match="1, 2, 4 or 8"):
        hsb.KVPages(4, kv_heads=3, device="cpu")
    with pytest.raises(hsb.InvalidArgument, match="at least one page"):
        hsb.KVPages(0, device="cpu")
    for data in (torch.zeros(4, 8, 32768, dtype=torch.uint8), torch.zeros(4, 8, 16896, dtype=torch.int8),
                 torch.zeros(8, 8, 16896, dtype=torch.uint8)[::2], torch.zeros(0, 8, 16896, dtype=torch.uint8)):
        with pytest.raises(hsb.InvalidArgument, match="a int8 pool is uint8"):
            hsb.KVPages(kv_heads=8, format="int8", data=data)
    with pytest.raises(hsb.InvalidArgument, match="CUDA"):
        hsb.KVPages(4, device="cpu")
