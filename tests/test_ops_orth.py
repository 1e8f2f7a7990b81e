"""Newton-Schulz orthogonalisation (nesle_b200.ops.orthogonalize) against 64 bits.

Error bound, in Frobenius norms.  A product of two matrices kept in 22 bits
errs by at most u = 2^-20 of the product of their norms: 2^-22 for each
operand, as much for what is stored, 2^-22 for sums in the tensor core's fp32.
With |X|_2 <= 1.21 a step's three products put at most
(2|a| + 3*1.46|b| + 5*2.1|c|) u |X|_F < 50 u |X|_F beside the new X, and each
later step multiplies what is there by at most a = 3.4445 (the derivative of
the quintic on [0, 1.21]).  Then one rounding to bf16."""
from __future__ import annotations

import threading

import pytest

torch = pytest.importorskip("torch")

from nesle_b200 import ops  # noqa: E402

A, B, C = 3.4445, -4.7750, 2.0315


@pytest.fixture(autouse=True, scope="module")
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from nesle_b200 import build

    build.build()


def exact(x, steps=5, eps=1e-7):
    """The 64-bit result and the bound on the error before the last rounding."""
    x = x.double()
    x = x / (torch.linalg.matrix_norm(x)[..., None, None] + eps)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    bound = torch.zeros(x.shape[:-2], dtype=torch.float64, device=x.device)
    for _ in range(steps):
        bound = A * bound + 50 * 2.0 ** -20 * torch.linalg.matrix_norm(x)
        g = x @ x.mT
        x = A * x + (B * g + C * (g @ g)) @ x
    return (x.mT if tall else x), bound


def check(out, x, steps=5):
    want, bound = exact(x, steps)
    assert out.dtype == torch.bfloat16 and out.shape == x.shape
    off = torch.linalg.matrix_norm(out.double() - want)
    assert bool((off <= bound + 2.0 ** -8 * torch.linalg.matrix_norm(want)).all()), (off, bound)


def momentum(*shape, seed=0, dtype=torch.float32, scale=1e-3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = min(shape[-2:])
    s = torch.exp(-3.0 * torch.arange(r, device="cuda") / r)
    x = torch.randn((*shape[:-1], r), generator=g, device="cuda") * s @ torch.randn((*shape[:-2], r, shape[-1]), generator=g,
                                                                                     device="cuda")
    return (scale * (x + 0.1 * torch.randn(shape, generator=g, device="cuda"))).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 50), (50, 1), (3, 5), (7, 256), (64, 64), (127, 129), (128, 128), (129, 127),
                                       (130, 64), (200, 1000), (256, 512), (512, 256), (512, 2048), (1000, 300), (333, 2049), (1100, 6500), (3700, 3600)])
def test_matches_64_bits(rows, cols):
    x = momentum(rows, cols, seed=rows + cols)
    check(ops.orthogonalize(x), x)
    assert ops.stalls() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(3, 96, 160), (2, 2, 65, 33), (5, 256, 256), (2, 300, 130)])
def test_batches_and_types(shape, dtype):
    x = momentum(*shape, seed=3, dtype=dtype, scale=0.1)
    check(ops.orthogonalize(x), x)


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [1, 2, 3, 8])
def test_steps(steps):
    x = momentum(150, 260, seed=steps)
    check(ops.orthogonalize(x, steps=steps), x, steps)


@pytest.mark.gpu
def test_strides():
    wide = momentum(300, 700, seed=1)
    for x in (wide.T, wide[10:110, 5:642], wide[::3, ::2], wide.T[::5], wide[:1].expand(40, 700)):
        check(ops.orthogonalize(x), x)
    batch = momentum(4, 60, 90, seed=2)
    check(ops.orthogonalize(batch.transpose(0, 1)), batch.transpose(0, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-4, 1.0, 1e30])
def test_the_scale_does_not_matter(scale):
    """Squares of 1e30 pass fp32; the norm is taken in 64 bits."""
    x = momentum(100, 140, seed=5, scale=1.0) * scale
    check(ops.orthogonalize(x), x)


@pytest.mark.gpu
def test_singular_values_move_to_one():
    q, _ = torch.linalg.qr(torch.randn((256, 256), device="cuda", dtype=torch.float64, generator=torch.Generator("cuda").manual_seed(1)))
    s = torch.linspace(0.05, 1.0, 256, device="cuda", dtype=torch.float64)
    out = ops.orthogonalize(((q * s) @ q.T).float()).double()
    values = torch.linalg.svdvals(out)
    assert 0.6 < float(values.min()) and float(values.max()) < 1.3


@pytest.mark.gpu
def test_zero_and_non_finite_matrices():
    x = momentum(4, 70, 90, seed=7)
    x[1] = 0
    x[2, 3, 4] = float("nan")
    x[3, 5, 6] = float("inf")
    out = ops.orthogonalize(x)
    check(out[:1], x[:1])
    assert int((out[1] != 0).sum()) == 0
    assert bool(torch.isnan(out[2]).all()) and not bool(torch.isfinite(out[3]).all())


@pytest.mark.gpu
def test_same_result_every_time_and_on_another_stream():
    x = momentum(512, 700, seed=9)
    first = ops.orthogonalize(x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = [ops.orthogonalize(x) for _ in range(5)]
    side.synchronize()
    assert all(torch.equal(first, y) for y in again)
    out = torch.empty_like(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.orthogonalize(x, out=out)
    graph.replay()
    assert torch.equal(out, first)


@pytest.mark.gpu
def test_empty_and_refusals():
    assert ops.orthogonalize(torch.empty((0, 4, 5), device="cuda")).shape == (0, 4, 5)
    assert ops.orthogonalize(torch.empty((2, 0, 5), device="cuda")).shape == (2, 0, 5)
    x = momentum(8, 12)
    for call in (
        lambda: ops.orthogonalize(x.cpu()),
        lambda: ops.orthogonalize(x.double()),
        lambda: ops.orthogonalize(x[0]),
        lambda: ops.orthogonalize(x, steps=0),
        lambda: ops.orthogonalize(x, eps=-1.0),
        lambda: ops.orthogonalize(x, out=torch.empty((8, 12), device="cuda")),
        lambda: ops.orthogonalize(x, out=torch.empty((12, 8), device="cuda", dtype=torch.bfloat16).T),
        lambda: ops.orthogonalize(x.clone().requires_grad_()),
    ):
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
def test_in_a_thread_that_has_made_no_cuda_call():
    x = momentum(130, 260, seed=11)
    want = ops.orthogonalize(x)
    out = torch.empty_like(want)
    torch.cuda.synchronize()
    thread = threading.Thread(target=lambda: ops.orthogonalize(x, out=out))
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@pytest.mark.gpu
def test_a_gradient_that_saved_out_is_refused_when_it_has_been_written():
    x = momentum(8, 12)
    out = torch.ones((8, 12), device="cuda", dtype=torch.bfloat16)
    a = torch.ones_like(out).requires_grad_()
    saved = (a * out).sum()
    ops.orthogonalize(x, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.backward()


@pytest.mark.gpu
def test_an_out_that_wants_a_gradient_is_refused():
    out = torch.ones((8, 12), device="cuda", dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(ValueError, match="no gradient"):
        ops.orthogonalize(momentum(8, 12), out=out)
    with torch.no_grad():
        assert torch.equal(ops.orthogonalize(momentum(8, 12), out=out), ops.orthogonalize(momentum(8, 12)))


@pytest.mark.gpu
def test_a_zero_matrix_stays_zero_without_eps():
    x = momentum(3, 40, 30, seed=13)
    x[1] = 0
    out = ops.orthogonalize(x, eps=0.0)
    assert int((out[1] != 0).sum()) == 0
    check(out[::2], x[::2])
    x[1, 0, 0] = float("nan")
    assert bool(torch.isnan(ops.orthogonalize(x, eps=0.0)[1]).all())


@pytest.mark.gpu
def test_steps_that_are_no_count_are_refused():
    x = momentum(8, 12)
    for steps in (2.5, 0, -3, 1 << 40, float("nan")):
        with pytest.raises(ValueError, match="steps"):
            ops.orthogonalize(x, steps=steps)
    assert torch.equal(ops.orthogonalize(x, steps=5.0), ops.orthogonalize(x))
