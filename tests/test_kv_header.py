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
