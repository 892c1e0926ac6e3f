"""The paged attention's workspaces: any content before a call, one after another
in one workspace, captured and replayed."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from test_gpu_kv_pages import dev, i32, quick_fill

pytestmark = pytest.mark.gpu


def ptr(t):
    return C.c_void_p(t.data_ptr())


class Case:
    """A batch, its calls through the C ABI in a workspace that is given, and the results in workspaces of their own."""

    def __init__(self, cuda, seed, fmt, heads, lengths, prefix, width=0):
        rng = np.random.default_rng(seed)
        self.cache, table, _ = quick_fill(cuda, rng, fmt, heads, lengths)
        table = np.concatenate([table, np.full((len(lengths), width), -1, np.int32)], 1)
        self.pre, ptable, _ = quick_fill(cuda, rng, "f16", heads, [prefix])
        self.table, self.lengths, self.ptable = i32(table), i32(lengths), i32(ptable[0])
        self.batch, self.heads, self.prefix = len(lengths), heads, prefix
        self.q = dev(rng.standard_normal((self.batch, 4 * heads, 128)).astype(np.float32))
        self.q16 = self.q.half()
        self.want = self.cache.attention(self.q, self.table, self.lengths)
        self.want16 = self.cache.attention_shared(self.q16, self.table, self.lengths, self.pre, self.ptable, prefix)
        self.cache.check()

    def bytes(self, lib):
        return max(lib.hsb_kv_attention_workspace_bytes(self.batch, self.heads),
                   lib.hsb_kv_attention_shared_workspace_bytes(self.batch, self.heads, self.prefix))

    def run(self, lib, ws, out, out16):
        import torch

        s = C.c_void_p(torch.cuda.current_stream().cuda_stream)
        assert lib.hsb_kv_attention(self.cache._ref, ptr(self.table), self.table.shape[1], ptr(self.lengths), self.batch,
                                    ptr(self.q), ptr(out), ptr(ws), ws.numel(), ptr(self.cache.status), s) == 0
        assert lib.hsb_kv_attention_shared(self.pre._ref, ptr(self.ptable), self.prefix, self.cache._ref, ptr(self.table),
                                           self.table.shape[1], ptr(self.lengths), self.batch, ptr(self.q16), ptr(out16),
                                           ptr(ws), ws.numel(), ptr(self.cache.status), s) == 0


@pytest.mark.parametrize("junk", [0x00, 0xFF, 0x5A])
@pytest.mark.parametrize("captured", [False, True])
def test_calls_one_after_another_in_one_workspace(cuda, junk, captured):
    import torch
    from hillserve_b200 import _capi

    lib = _capi.lib()
    cases = [Case(cuda, 1, "int8", 8, [9000], 300), Case(cuda, 2, "f16", 2, [700, 0, 3000, 5], 5000, width=40),
             Case(cuda, 3, "e4m3", 4, [64] * 70, 1000), Case(cuda, 4, "int8", 1, [0, 0], 64)]
    ws = torch.full((max(c.bytes(lib) for c in cases),), junk, dtype=torch.uint8, device="cuda")
    order = [cases[(i * 3 + i // 4) % 4] for i in range(16)]
    outs = [(torch.empty_like(c.q), torch.empty_like(c.q16)) for c in order]

    def all_calls():
        for c, pair in zip(order, outs):
            c.run(lib, ws, *pair)

    if captured:
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            all_calls()
        ws.fill_(junk)
        for _ in range(3):
            graph.replay()
    else:
        all_calls()
    torch.cuda.synchronize()
    for i, (c, (out, out16)) in enumerate(zip(order, outs)):
        assert bool((out == c.want).all()) and bool((out16 == c.want16).all()), i
    for c in cases:
        c.cache.check()
