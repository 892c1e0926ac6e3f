"""What the paged cache's calls record is neither lost nor made up when calls, pools and checks are on several streams."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from test_gpu_kv_pages import dev, i32

pytestmark = pytest.mark.gpu
SPIN = 100_000_000  # clocks: some 50 ms, well above what the host needs to enqueue a few calls


@pytest.fixture
def bad(cuda):
    """A call that records HSB_E_KV_PAGE for sequence `index` of a pool, and touches nothing."""
    rows = dev(np.zeros((4, 2, 1, 128), np.float16))
    starts = i32([0] * 4)
    tables = [i32(np.where(np.arange(4)[:, None] == i, 99, 0)) for i in range(4)]
    import torch

    torch.cuda.synchronize()

    def call(pool, index=0, stream=None):
        pool.append(rows, tables[index], starts, stream=stream)

    return call


def test_a_new_pool_is_ready_for_any_stream(cuda, bad):
    import torch

    other, busy = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(busy):
        held = [cuda.KVPages(1, kv_heads=1, format="f16") for _ in range(2)]
        bad(held[0], stream=other)
        torch.cuda.synchronize()
        del held  # (kernels and memory are at hand: getting them would wait for the device)
        torch.cuda._sleep(SPIN)
        pool = cuda.KVPages(1, kv_heads=1, format="f16")
        bad(pool, stream=other)
        torch.cuda.synchronize()
        with pytest.raises(cuda.InvalidArgument) as e:
            pool.check()
        assert e.value.status == 121
        fresh = cuda.KVPages(1, kv_heads=1, format="f16")
        fresh.check(stream=other)


def test_check_waits_for_every_stream(cuda, bad):
    import torch

    pool, other = cuda.KVPages(1, kv_heads=1, format="f16"), torch.cuda.Stream()
    with torch.cuda.stream(other):
        torch.cuda._sleep(SPIN)
    bad(pool, stream=other)
    with pytest.raises(cuda.InvalidArgument):
        pool.check()
    pool.check()


def test_check_of_one_stream_loses_nothing_of_another(cuda, bad):
    import torch

    pool = cuda.KVPages(1, kv_heads=1, format="f16")
    first, other, busy = (torch.cuda.Stream() for _ in range(3))
    bad(pool, 2, stream=first)
    first.synchronize()
    for s in (other, busy):
        with torch.cuda.stream(s):
            torch.cuda._sleep(SPIN if s is other else 3 * SPIN)
    bad(pool, 1, stream=other)
    with torch.cuda.stream(busy):
        with pytest.raises(cuda.InvalidArgument):
            pool.check(stream=first)
        other.synchronize()
        torch.cuda.synchronize()
        assert pool.status.tolist() == [121, 1]
        with pytest.raises(cuda.InvalidArgument):
            pool.check()
        pool.check()


def test_status_take(cuda):
    """The word comes back once; nothing recorded is no error; the index is kept until it is taken."""
    import torch
    from hillserve_b200 import _capi

    lib, word = _capi.lib(), i32([111, 7])
    s = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    at = C.c_void_p(word.data_ptr())
    assert lib.hsb_status_check(at, s) == 111 and word.tolist() == [111, 7]
    assert lib.hsb_status_take(at, s) == 111 and word.tolist() == [0, 0]
    assert lib.hsb_status_take(at, s) == 0 and lib.hsb_last_error() == b""
