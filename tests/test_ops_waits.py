"""The operators' bounded waits (csrc/tc05.cuh): a wait that runs out says so,
and no kernel drops what it says."""
from __future__ import annotations

import ctypes
import re
import subprocess
from pathlib import Path

import pytest

from nesle_b200 import build

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "nesle_b200" / "csrc"


def dropped(text: str) -> list[str]:
    """Calls of mbar_wait and mbar_wait_warp that are a whole statement, behind an if or not."""
    text = re.sub(r"//.*", "", text)
    return [m.group(0).strip() for m in re.finditer(r"(?:[;{}]|\bif(?: constexpr)? \([^;{}]*\))\s*(?:tc::)?mbar_wait(?:_warp)?\([^;]*;", text)]


def test_a_dropped_wait_is_found():
    assert len(dropped("x = 1;\n    if (a && b(c)) tc::mbar_wait_warp(&bar, n & 1);  // long since\n")) == 1
    assert len(dropped("{ mbar_wait(&bar, 0); }")) == 1
    assert not dropped("if (!(ok = tc::mbar_wait(&full[i], 1))) break;\nok = tc::mbar_wait_warp(done, 0) && ok;\n"
                       "if (a && !tc::mbar_wait_warp(&b, 0)) { leave(); }\nreturn __all_sync(~0u, mbar_wait(b, parity));")


@pytest.mark.parametrize("source", sorted(p.name for p in CSRC.glob("ops_*")) + ["tc05.cuh"])
def test_no_kernel_drops_the_result_of_a_wait(source):
    """A wait that gave up and is not answered for leaves invalid outputs uncounted."""
    assert not dropped((CSRC / source).read_text())


@pytest.mark.gpu
def test_waits_run_out_and_say_so():
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    source, out = ROOT / "tests" / "native" / "wait_probe.cu", ROOT / "tests" / "native" / "_build" / "wait_probe.so"
    if not out.exists() or out.stat().st_mtime < max(source.stat().st_mtime, (CSRC / "tc05.cuh").stat().st_mtime):
        out.parent.mkdir(exist_ok=True)
        subprocess.run([build.nvcc(), "-std=c++20", "-O2", *build.ARCH, "-shared", "-Xcompiler", "-fPIC", "-o", str(out), str(source)],
                       check=True)
    lib = ctypes.CDLL(str(out))
    lib.run_wait_probe.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_longlong]
    got, took, limit = (ctypes.c_int * 32)(), ctypes.c_longlong(), 100_000
    assert lib.run_wait_probe(got, ctypes.byref(took), limit) == 0
    assert list(got) == [4] * 32  # only the phase that an arrival ended is over
    assert limit <= took.value < 1_000_000_000  # half a second at most, where the kernels wait a whole one
