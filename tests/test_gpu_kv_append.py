"""Edges of the paged write: starts that are no positions."""
from __future__ import annotations

import numpy as np
import pytest

import kv_oracle as ko
from test_gpu_kv_pages import dev, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("start", [-1, -64, -(2**31)])
def test_negative_starts_are_no_positions(cuda, start):
    """Also in a table so wide that the number read without its sign lies within it; later rows of such a sequence,
    which would come to positions from 0 on, are left out too."""
    import torch

    rng = np.random.default_rng(0)
    cache = cuda.KVPages(1, kv_heads=1, format="int8")
    cache.data.fill_(0x55)
    table = torch.zeros((1, (1 << 26) + 3), dtype=torch.int32, device="cuda")
    for n in (1, 70):
        cache.append(dev(ko.rows(rng, n, 1)), table, i32([start]), offsets=i32([0, n]))
        with pytest.raises(cuda.InvalidArgument) as e:
            cache.check()
        assert e.value.status == 122
        assert bool((cache.data == 0x55).all())
    cache.append(dev(ko.rows(rng, 1, 1)), table, i32([2**31 - 1]), offsets=i32([0, 1]))  # the last position
    cache.check()
    assert not bool((cache.data == 0x55).all())
    del table
    torch.cuda.empty_cache()
