"""The paged attention's host+device arithmetic (csrc/kvattention.cuh), compiled
from the header itself by tests/cpp/kv_header_checks.cu and run on the host."""
from __future__ import annotations

import random
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    """Answers of the header's functions, a list of numbers a question."""
    from hillserve_b200 import build

    exe = tmp_path_factory.mktemp("kv_header") / "checks"
    subprocess.run([build.nvcc_path(), "-std=c++17", *build.ARCH, f"-I{build.CSRC}", f"-I{ROOT / 'include'}",
                    str(ROOT / "tests" / "cpp" / "kv_header_checks.cu"), "-o", str(exe)], check=True, timeout=300)

    def answers(questions):
        r = subprocess.run([str(exe)], input="\n".join(questions) + "\n", capture_output=True, text=True, timeout=60)
        assert r.returncode == 0, r.stderr
        got = [[int(x) for x in line.split()] for line in r.stdout.splitlines()]
        assert len(got) == len(questions)
        return got

    return answers


@pytest.mark.parametrize("grid", [1, 2, 7, 148, 160])
def test_a_place_never_names_partials_outside_the_grid(ask, grid):
    """Whatever a run's place word holds, its partials lie in the grid that could have left them."""
    rng = random.Random(grid)
    words = [0, 1, 0xFFFF, 0x10000, 0xFFFFFFFF, 0xFF, 0x80008000, grid, grid + 1, grid << 16, (grid - 1) << 16 | 1,
             (grid - 1) << 16 | 2, 1 << 16 | grid] + [rng.getrandbits(32) for _ in range(2000)]
    words += [rng.randrange(200) << 16 | rng.randrange(200) for _ in range(2000)]
    for word, (n,) in zip(words, ask([f"place {w} {grid}" for w in words])):
        if word == 0:
            assert n == 1
        else:
            assert n in (0, word & 0xFFFF) and (n == 0 or (word >> 16) + n <= grid), hex(word)


def test_a_cut_run_keeps_its_partials(ask):
    cuts = [(first, count) for first in range(148) for count in range(1, 149 - first, 13)]
    words = [w for (w,) in ask([f"cut {f} {c}" for f, c in cuts])]
    assert all(w for w, (f, c) in zip(words, cuts) if (f, c) != (0, 0))
    for (_, count), (n,) in zip(cuts, ask([f"place {w} 148" for w in words])):
        assert n == count


def test_status_take_refuses():
    import ctypes as C

    from hillserve_b200 import _capi

    lib = _capi.lib()
    for at in (None, C.c_void_p(0x10004)):
        assert lib.hsb_status_take(at, None) == lib.hsb_status_check(None, None) != 0


@pytest.mark.parametrize("n", [1, 2, 16, 148, 1184])
def test_the_split_as_compiled(ask, n):
    """Stretches follow one another over all units, differ by one unit at most, the longer ones first; the stretch of
    a unit is the one that holds it.  Up to the units of 2^27 table entries of 8 heads in halves, and their run costs."""
    rng = random.Random(n)
    units = [1, 2, 7, 147, 148, 149, 1000, 4096 * 8 + 3, (1 << 31) + (1 << 24)] + [rng.randrange(1, 1 << 31) for _ in range(20)]
    asked = [sorted({0, u - 1, u // 2, u // 3, min(u - 1, 5)} | {rng.randrange(u) for _ in range(20)}) for u in units]
    for u, at, got in zip(units, asked, ask([f"split {u} {n} " + " ".join(map(str, a)) for u, a in zip(units, asked)])):
        begins, of = got[:n + 1], got[n + 1:]
        sizes = [b - a for a, b in zip(begins, begins[1:])]
        assert begins[0] == 0 and begins[-1] == u and sizes == sorted(sizes, reverse=True) and sizes[0] - sizes[-1] <= 1
        assert len(of) == len(at) and all(begins[c] <= x < begins[c + 1] for c, x in zip(of, at))


def test_ranges_apart(ask):
    cases = [(a, n, b, m) for a in (100, 160) for n in (1, 16, 60, 61) for b in (80, 99, 100, 116, 160, 161, 220, 221)
             for m in (1, 20, 21, 80, 81)]
    for (a, n, b, m), (got,) in zip(cases, ask([f"apart {a} {n} {b} {m}" for a, n, b, m in cases])):
        assert got == (not set(range(a, a + n)) & set(range(b, b + m))), (a, n, b, m)


def test_overlapping_buffers_are_refused():
    """An attention's output inside its query, its workspace over either: all refused before any launch."""
    import ctypes as C

    from hillserve_b200 import _capi

    lib, batch, heads, base = _capi.lib(), 3, 2, 1 << 30
    P = C.c_void_p(1 << 20)
    at = lambda x: C.c_void_p(base + x)  # noqa: E731
    own = C.byref(_capi.KvPages(1 << 21, 4, 1, heads))
    pre = C.byref(_capi.KvPages(1 << 22, 4, 0, heads))
    for width, size, call in (
            (4, lib.hsb_kv_attention_workspace_bytes(batch, heads),
             lambda q, o, w, n: lib.hsb_kv_attention(own, P, 4, P, batch, q, o, w, n, None, None)),
            (2, lib.hsb_kv_attention_shared_workspace_bytes(batch, heads, 100),
             lambda q, o, w, n: lib.hsb_kv_attention_shared(pre, P, 100, own, P, 4, P, batch, q, o, w, n, None, None))):
        bytes_ = batch * 4 * heads * 128 * width
        far = at(1 << 28)
        for off in (0, 16, bytes_ - 16, 16 - bytes_):
            assert call(at(0), at(off), far, size) == 120
            assert lib.hsb_last_error() == b"paged KV attention output must not alias the query"
        for ws in (at(0), at(bytes_ - 16), at(-16 * (size // 16 - 1))):
            for q, o in ((at(0), far), (far, at(0))):
                assert call(q, o, ws, size) == 120
                assert lib.hsb_last_error() == b"paged KV attention workspace must not alias the query or the output"
