"""The operators' C boundary (include/nesle_ops.h) without a GPU: the packed
argument blocks have the C layout, and every entry checks its arguments before
it touches a device."""
from __future__ import annotations

import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from nesle_b200 import _lib

ROOT = Path(__file__).resolve().parents[1]
BLOCKS = {"nesle_int8_args": _lib.INT8_ARGS, "nesle_orth_args": _lib.ORTH_ARGS,
          "nesle_delta_step_args": _lib.DELTA_STEP_ARGS, "nesle_delta_args": _lib.DELTA_ARGS}


@pytest.fixture(scope="module")
def lib():
    from nesle_b200 import build

    build.build()
    return _lib.load()


def members(name: str) -> list[str]:
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "nesle_ops.h").read_text(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1)
    out = []
    for declaration in body.split(";"):
        out += [x.strip().lstrip("*").split()[-1].lstrip("*") for x in declaration.split(",") if x.strip()]
    return out


@pytest.mark.parametrize("name", BLOCKS)
def test_argument_blocks_have_the_c_layout(name, tmp_path):
    """Every member at the offset that the struct format gives it."""
    if not shutil.which("gcc"):
        pytest.skip("gcc is not available")
    names = members(name)
    source = '#include <stdio.h>\n#include "nesle_ops.h"\nint main(void) {\n' + "".join(
        f'printf("%zu %zu\\n", offsetof({name}, {m}), sizeof((({name}*)0)->{m}));\n' for m in names) + "return 0; }\n"
    (tmp_path / "a.c").write_text(source)
    subprocess.run(["gcc", "-I", str(ROOT / "include"), "-o", str(tmp_path / "a"), str(tmp_path / "a.c")], check=True)
    want = [tuple(map(int, x.split())) for x in subprocess.run([str(tmp_path / "a")], capture_output=True, text=True,
                                                               check=True).stdout.splitlines()]
    letters = re.sub(r"\s", "", BLOCKS[name].format.lstrip("@"))
    assert len(letters) == len(names)
    import struct

    got = []
    for i, letter in enumerate(letters):
        size = struct.calcsize("@" + letter)
        got.append((struct.calcsize("@" + letters[:i + 1]) - size, size))
    assert got == want


def test_null_and_bad_arguments_are_refused(lib):
    invalid = _lib.NESLE_ERR_INVALID
    for name in ("nesle_int8_linear", "nesle_orthogonalize", "nesle_delta_step", "nesle_delta_scan",
                 "nesle_delta_scan_backward"):
        assert getattr(lib, name)(None, None) == invalid, name
        assert lib.nesle_last_error()
    assert lib.nesle_quantize_rows(None, 0, 4, 4, 4, None, 16, None, 0, None) == invalid
    assert lib.nesle_quantize_rows(1, 0, 4, 8, 4, 1, 16, 1, 0, None) == invalid  # rows overlap
    assert lib.nesle_ops_stalls(0, None) == invalid

    def delta(t=4, n=1, h=1, dk=16, dv=16, dtype=0):
        return _lib.DELTA_ARGS.pack(16, 16, 16, *(16,) * 9, dtype, 16, 16, *(1,) * 6, 0, 0, 0, 0, t, n, h, dk, dv, 1.0,
                                    *(0,) * 12, 0)

    assert lib.nesle_delta_scan(delta(dk=129), None) == invalid
    assert lib.nesle_delta_scan(delta(dv=0), None) == invalid
    assert lib.nesle_delta_scan(delta(dtype=9), None) == invalid
    assert lib.nesle_delta_scan(delta(), None) == invalid  # no output
    assert lib.nesle_delta_scan_backward(delta(t=0), None) == invalid
    assert lib.nesle_delta_scan(delta(n=0), None) == _lib.NESLE_OK  # nothing to do
    orth = _lib.ORTH_ARGS.pack(16, 0, 16, 4, 1, 1, 4, 4, 0, 1e-7, 16, 0, 0, 0)
    assert lib.nesle_orthogonalize(orth, None) == invalid  # no steps
    assert b"steps" in lib.nesle_last_error()


def test_sizes_of_what_a_scan_keeps(lib):
    args = _lib.DELTA_ARGS.pack(*(0,) * 25, 33, 5, 3, 40, 72, 0.0, *(0,) * 12, 0)
    assert lib.nesle_delta_checkpoint_floats(args) == 5 * 3 * 3 * 40 * 72  # a state for every 16 tokens begun
    assert lib.nesle_delta_error_floats(args) == 5 * 3 * 3 * 5 * 256       # 16 x 16 tiles
    assert lib.nesle_delta_error_floats(None) == 0


def test_tensors_that_are_not_on_a_gpu_are_refused():
    torch = pytest.importorskip("torch")
    from nesle_b200 import ops

    x = torch.zeros((2, 3, 16))
    with pytest.raises(ValueError, match="CUDA"):
        ops.quantize_rows(x)
    with pytest.raises(ValueError, match="CUDA"):
        ops.orthogonalize(x)
    with pytest.raises(ValueError, match="CUDA"):
        ops.delta_step(x, x, x, x[..., 0], x[..., 0], torch.zeros((2, 3, 16, 16)))
    with pytest.raises(ValueError, match="CUDA"):
        ops.int8_linear(x, None)
    with pytest.raises(ValueError, match="CUDA"):
        ops.Int8Weight(torch.zeros((4, 4), dtype=torch.int8), torch.zeros(4))


def test_tangents_are_refused_and_not_dropped():
    """A dual tensor does not require grad; a call on it would go on without its tangent."""
    torch = pytest.importorskip("torch")
    from torch.autograd import forward_ad

    from nesle_b200 import ops

    x = torch.ones(3)
    ops._no_grad_path("call", x, None)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, x)
        with pytest.raises(ValueError, match="forward-mode"):
            ops._no_grad_path("call", None, x, dual)
        with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
            ops._no_grad_path("call", dual)
        ops._no_grad_path("call", x, forward_ad.unpack_dual(dual).primal)


def test_pointers_off_their_elements_are_refused(lib):
    """Before a device is touched: a load there would fault.  Every pointer in turn, one byte off, or two where it is to 4-byte
    elements; the others are right, and sizes and strides those of a call that runs."""
    P = 1 << 20  # a pointer that only its alignment is looked at of

    def refused(call, names, elements):
        for i, name in enumerate(names):
            for off in {1, elements[i] // 2}:
                args = [P + off if i == j else P for j in range(len(names))]
                assert call(*args) == _lib.NESLE_ERR_INVALID, (name, off)
                assert b"aligned" in lib.nesle_last_error(), (name, off, lib.nesle_last_error())

    for dtype, size in ((0, 4), (1, 2), (2, 2)):
        refused(lambda x, scale: lib.nesle_quantize_rows(x, dtype, 4, 8, 8, P, 16, scale, 0, None), ("x", "scale"), (size, 4))
        refused(lambda xs, ws, bias, y: lib.nesle_int8_linear(
            _lib.INT8_ARGS.pack(P, 1, 16, xs, 1.0, P, P, 16, ws, bias, y, dtype, 8, 4, 16, 8, 0, 0, 0, 0), None),
            ("x_scale", "w_scale", "bias", "y"), (4, 4, 4, size))
        refused(lambda x: lib.nesle_orthogonalize(_lib.ORTH_ARGS.pack(x, dtype, 16, 4, 1, 1, 4, 4, 5, 1e-7, P, P, 1 << 30, 0), None),
                ("x",), (size,))
        refused(lambda q, k, v, g, beta, state, o: lib.nesle_delta_step(
            _lib.DELTA_STEP_ARGS.pack(q, k, v, *(16,) * 6, dtype, g, beta, *(1,) * 4, 0, 0, state, 256, 256, o, 2, 1, 16, 16, 1.0, 0), None),
            ("q", "k", "v", "g", "beta", "state", "o"), (size, size, size, 4, 4, 4, size))

        def scan(entry, q, k, v, g, beta, state, *rest):
            return entry(_lib.DELTA_ARGS.pack(q, k, v, *(32, 16, 16) * 3, dtype, g, beta, *(2, 1, 1) * 2, 0, 0, 0, state, 4, 2, 1, 16, 16,
                                              1.0, *rest, *(0,) * (12 - len(rest)), 0), None)

        names = ("q", "k", "v", "g", "beta", "state", "o", "final_state", "errors", "checkpoints")
        refused(lambda *p: scan(lib.nesle_delta_scan, *p), names, (size, size, size, 4, 4, 4, size, 4, 16, 4))
        names = ("q", "k", "v", "g", "beta", "errors", "checkpoints", "d_o", "d_final", "dq", "d_k", "d_v", "dg", "dbeta", "dstate")
        refused(lambda *p: scan(lib.nesle_delta_scan_backward, *p[:5], 0, 0, 0, *p[5:]), names,
                (size, size, size, 4, 4, 16, 16, size, 4, size, size, size, 4, 4, 4))


def test_outputs_on_the_memory_of_an_input_are_refused(lib):
    """At the C boundary; ops.py writes such an output elsewhere and copies.  The calls that this refuses reach no device."""
    far = 1 << 40

    def int8(y, **at):
        p = {"x": far, "x_scale": 2 * far, "w": 3 * far, "w_biased": 4 * far, "w_scale": 5 * far, "bias": 6 * far, **at}
        return lib.nesle_int8_linear(_lib.INT8_ARGS.pack(p["x"], 1, 2048, p["x_scale"], 1.0, p["w"], p["w_biased"], 512, p["w_scale"], p["bias"],
                                                         y, _lib.F32, 512, 40, 512, 100, 0, 0, 0, 0), None)

    y = 7 * far  # 40 rows of 400 bytes, 2,048 apart
    for name, size in (("x_scale", 160), ("w", 99 * 512 + 512), ("w_biased", 99 * 512 + 512), ("w_scale", 400), ("bias", 400)):
        size = -(-size // 16) * 16
        for at in (y, y + 39 * 2048 + 384, y - size + 16):
            assert int8(y, **{name: at}) == _lib.NESLE_ERR_OVERLAP, (name, at - y)
    # tokens, rows as far apart: bytes 0..511 of each against 0..399
    for at in (y, y + 384, y - 496, y + 39 * 2048 + 384, y - 39 * 2048, y + 2048 - 496):
        assert int8(y, x=at) == _lib.NESLE_ERR_OVERLAP, at - y
    assert b"y shares memory" in lib.nesle_last_error()

    def step(o, **at):  # 3 envs x 2 heads of 16 x 8, bf16
        p = {"q": far, "k": 2 * far, "v": 3 * far, "g": 4 * far, "beta": 5 * far, "reset": 6 * far, "state": 7 * far, **at}
        return lib.nesle_delta_step(_lib.DELTA_STEP_ARGS.pack(p["q"], p["k"], p["v"], 32, 16, 32, 16, 16, 8, _lib.BF16, p["g"], p["beta"], 2, 1, 2, 1,
                                                              p["reset"], 1, p["state"], 256, 128, o, 3, 2, 16, 8, 1.0, 0), None)

    o = 8 * far  # 96 bytes
    for name, size in (("q", 192), ("k", 192), ("v", 96), ("g", 24), ("beta", 24), ("reset", 3), ("state", 3072)):
        for at in (o, o + 92, o - (size - 1) // 4 * 4):
            assert step(o, **{name: at}) == _lib.NESLE_ERR_OVERLAP, (name, at - o)
