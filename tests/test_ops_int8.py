"""8-bit product (nesle_b200.ops.int8_linear, quantize_rows) against 64 bits.

The integer sum is exact, so an output differs from the 64-bit value by the
rounding of the epilogue alone: the sum to fp32 and three fp32 operations (at
most 4 * 2^-24 of the largest term) and one rounding to the output type."""
from __future__ import annotations

import threading

import pytest

torch = pytest.importorskip("torch")

from nesle_b200 import ops  # noqa: E402

UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}  # one rounding to nearest


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.fixture(autouse=True, scope="module")
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from nesle_b200 import build

    build.build()


def _weight(n, k, seed):
    g = _gen(seed)
    q = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    return q, torch.rand(n, generator=g, device="cuda") * 0.01 + 1e-4


def _check(y, xq, xs, q, ws, bias, relu):
    acc = xq.double() @ q.double().T
    terms = acc * xs * ws.double()
    want = terms + (bias.double() if bias is not None else 0.0)
    size = terms.abs() + (bias.double().abs() if bias is not None else 0.0)
    if relu:
        want = want.clamp(min=0)
    tol = want.abs() * UNIT[y.dtype] + size * 4 * 2.0 ** -24 + (2.0 ** -25 if y.dtype == torch.float16 else 0.0)
    assert y.shape == want.shape
    assert bool(((y.double() - want).abs() <= tol).all()), float(((y.double() - want).abs() - tol).max())


def _quantized(x):
    """IEEE divisions by tensors (torch turns a division by a number into a product with its reciprocal)."""
    most = x.float().abs().amax(1)
    scale = most / torch.full_like(most, 127.0)
    return torch.round(x.float() / torch.where(scale > 0, scale, 1.0)[:, None]).to(torch.int8), scale


SIZES = [(1, 2048, 512), (1, 1, 1), (2, 17, 3), (16, 64, 8), (17, 100, 9), (64, 256, 130), (65, 128, 16), (128, 128, 64),
         (129, 127, 65), (200, 130, 129), (257, 2048, 512), (1000, 300, 257), (300, 96, 2048), (20000, 64, 33),
         (19001, 200, 300), (9500, 130, 513), (20000, 16, 129), (6400, 1000, 700)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8])
def test_product_matches_64_bits(m, k, n, dtype):
    g = _gen(m * 7 + k)
    lo, hi = (0, 256) if dtype == torch.uint8 else (-128, 128)
    x = torch.randint(lo, hi, (m, k), generator=g, device="cuda", dtype=dtype)
    q, ws = _weight(n, k, 1)
    xs = torch.rand(m, generator=g, device="cuda") + 0.01
    bias = torch.randn(n, generator=g, device="cuda")
    w = ops.Int8Weight(q, ws)
    for out_dtype in (torch.bfloat16, torch.float32):
        _check(ops.int8_linear(x, w, xs, bias, out_dtype=out_dtype), x, xs.double()[:, None], q, ws, bias, False)
    _check(ops.int8_linear(x, w, 1 / 255, relu=True, out_dtype=torch.float16), x,
           float(torch.tensor(1 / 255, dtype=torch.float32)), q, ws, None, True)
    assert ops.stalls() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,value", [(torch.uint8, 255), (torch.int8, -128), (torch.int8, 127)])
def test_extreme_sums_are_exact(dtype, value):
    """Every byte at its extreme: the largest sums that the accumulators meet."""
    for m in (3, 130):
        k = 8192
        x = torch.full((m, k), value, dtype=dtype, device="cuda")
        q = torch.full((70, k), 127, dtype=torch.int8, device="cuda")
        q[1::2] = -127
        y = ops.int8_linear(x, ops.Int8Weight(q, torch.ones(70, device="cuda")), 1.0, out_dtype=torch.float32)
        want = (x.double() @ q.double().T).float()
        assert torch.equal(y, want)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [5, 300])
def test_strided_and_unaligned_operands(m):
    """Slices of a wider observation: rows further apart than they are long, starts off 16 bytes."""
    ram = torch.randint(0, 256, (m, 2048), generator=_gen(3), device="cuda", dtype=torch.uint8)
    for start, k in ((0, 100), (16, 1000), (1, 255), (2000, 48), (7, 2041)):
        x = ram[:, start:start + k]
        q, ws = _weight(40, k, start)
        out = torch.full((m, 64), 7.0, device="cuda", dtype=torch.bfloat16)
        ops.int8_linear(x, ops.Int8Weight(q, ws), 0.5, out=out[:, 3:43])
        _check(out[:, 3:43], x, 0.5, q, ws, None, False)
        assert bool((out[:, :3] == 7).all()) and bool((out[:, 43:] == 7).all())
    x = ram.T  # not unit stride: laid out again
    q, ws = _weight(40, m, 5)
    _check(ops.int8_linear(x, ops.Int8Weight(q, ws), 0.5), x, 0.5, q, ws, None, False)
    one = ram[:1].expand(m, 2048)
    q, ws = _weight(40, 2048, 6)
    _check(ops.int8_linear(one, ops.Int8Weight(q, ws), 0.5), one, 0.5, q, ws, None, False)


@pytest.mark.gpu
def test_empty_sizes():
    q, ws = _weight(6, 32, 1)
    w = ops.Int8Weight(q, ws)
    assert ops.int8_linear(torch.empty((0, 32), dtype=torch.uint8, device="cuda"), w, 1.0).shape == (0, 6)
    none = ops.Int8Weight(q[:, :0], ws)
    y = ops.int8_linear(torch.empty((5, 0), dtype=torch.int8, device="cuda"), none, 1.0, torch.arange(6.0, device="cuda"))
    assert torch.equal(y, torch.arange(6.0, device="cuda", dtype=torch.bfloat16).expand(5, 6))
    qq, ss = ops.quantize_rows(torch.empty((3, 0), device="cuda"))
    assert qq.shape == (3, 0) and torch.equal(ss, torch.zeros(3, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 64), (9, 1000), (4, 1024), (2, 4097), (3, 20000), (70, 512)])
def test_quantize_rows_is_exact(dtype, rows, cols):
    x = (torch.randn((rows, cols), generator=_gen(cols), device="cuda") * 3).to(dtype)
    if rows > 1:
        x[1] = 0
    q, s = ops.quantize_rows(x)
    want_q, want_s = _quantized(x)
    assert torch.equal(s, want_s) and torch.equal(q, want_q)
    wide = torch.randn((rows, 3 * cols + 5), generator=_gen(1), device="cuda").to(dtype)[:, 3:3 + cols]
    q, s = ops.quantize_rows(wide)
    want_q, want_s = _quantized(wide)
    assert torch.equal(s, want_s) and torch.equal(q, want_q)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [2048, 2047])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_rows_near_half_integers(cols, dtype):
    """Quotients at, and within a few units in the last place of, half integers, in rows of every magnitude that fp32 has."""
    exponents = torch.arange(-149, 122, device="cuda", dtype=torch.float64)[:, None]
    g = _gen(17)
    halves = torch.randint(-127, 127, (len(exponents), cols), generator=g, device="cuda").double() + 0.5
    near = halves * (1 + torch.randint(-4, 5, halves.shape, generator=g, device="cuda").double() * 2.0 ** -24)
    factor = 1 + torch.rand((len(exponents), 1), generator=g, device="cuda", dtype=torch.float64)
    near[:, 0] = 127
    x = (near * factor * 2.0 ** exponents).to(dtype)
    q, s = ops.quantize_rows(x)
    want_q, want_s = _quantized(x)
    finite = torch.isfinite(want_s)
    assert int(finite.sum()) > 250
    assert torch.equal(s[finite], want_s[finite]) and torch.equal(q[finite], want_q[finite])


@pytest.mark.gpu
@pytest.mark.parametrize("start", range(17))
def test_rows_that_start_anywhere(start):
    """Every offset from 16 bytes, of tokens whose rows are an odd number of bytes apart, and rows of results likewise."""
    ram = torch.randint(0, 256, (301, 407), generator=_gen(start), device="cuda", dtype=torch.uint8)
    k = 390 - 3 * start
    x = ram[:, start:start + k]
    q, ws = _weight(131, k, start)
    for dtype in (torch.bfloat16, torch.float32):
        out = torch.full((301, 200), 7.0, device="cuda", dtype=dtype)
        ops.int8_linear(x, ops.Int8Weight(q, ws), 0.5, out=out[:, start:start + 131])
        _check(out[:, start:start + 131], x, 0.5, q, ws, None, False)
        assert bool((out[:, :start] == 7).all()) and bool((out[:, start + 131:] == 7).all())


@pytest.mark.gpu
def test_quantize_rows_with_infinities_and_nan():
    x = torch.randn((4, 33), generator=_gen(0), device="cuda")
    x[1, 5], x[2, 6] = float("inf"), float("nan")
    q, s = ops.quantize_rows(x)
    assert torch.isinf(s[1]) and torch.isnan(s[2]) and torch.isfinite(s[[0, 3]]).all()
    assert int(q[1].abs().sum()) == 0 and int(q[2].abs().sum()) == 0
    qw, ws = _weight(8, 33, 1)
    y = ops.int8_linear(x, ops.Int8Weight(qw, ws))
    assert not torch.isfinite(y[1]).any() and not torch.isfinite(y[2]).any()
    assert torch.isfinite(y[[0, 3]]).all()


@pytest.mark.gpu
def test_floating_tokens_are_quantised_per_token():
    x = torch.randn((2, 70, 48), generator=_gen(2), device="cuda", dtype=torch.bfloat16)
    w = ops.Int8Weight.from_float(torch.randn((24, 48), generator=_gen(3), device="cuda"))
    q, s = ops.quantize_rows(x)
    assert q.shape == x.shape and s.shape == (2, 70)
    assert torch.equal(ops.int8_linear(x, w), ops.int8_linear(q, w, s))
    assert torch.equal(ops.int8_linear(x[0, 0], w), ops.int8_linear(x, w)[0, 0])


@pytest.mark.gpu
def test_on_another_stream_and_in_a_graph():
    x = torch.randint(0, 256, (500, 200), generator=_gen(2), device="cuda", dtype=torch.uint8)
    q, ws = _weight(96, 200, 4)
    w = ops.Int8Weight(q, ws)
    want = ops.int8_linear(x, w, 0.25)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y = ops.int8_linear(x, w, 0.25)
    side.synchronize()
    assert torch.equal(y, want)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.int8_linear(x, w, 0.25, out=out)
    x.fill_(3)
    graph.replay()
    assert torch.equal(out, ops.int8_linear(x, w, 0.25))


@pytest.mark.gpu
def test_in_a_thread_that_has_made_no_cuda_call():
    x = torch.randint(0, 256, (200, 64), generator=_gen(2), device="cuda", dtype=torch.uint8)
    q, ws = _weight(96, 64, 4)
    w, out = ops.Int8Weight(q, ws), torch.empty((200, 96), device="cuda", dtype=torch.bfloat16)
    want = ops.int8_linear(x, w, 0.25)
    torch.cuda.synchronize()
    thread = threading.Thread(target=lambda: ops.int8_linear(x, w, 0.25, out=out))
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert torch.equal(out, want)

@pytest.mark.gpu
def test_refusals():
    q, ws = _weight(8, 32, 1)
    w = ops.Int8Weight(q, ws)
    x = torch.zeros((4, 32), dtype=torch.uint8, device="cuda")
    for call in (
        lambda: ops.int8_linear(x.cpu(), w, 1.0),
        lambda: ops.int8_linear(x[:, :31], w, 1.0),
        lambda: ops.int8_linear(x, w),
        lambda: ops.int8_linear(x.to(torch.int16), w, 1.0),
        lambda: ops.int8_linear(x, w, torch.ones(3, device="cuda")),
        lambda: ops.int8_linear(x, w, torch.ones(4, device="cuda", dtype=torch.float64)),
        lambda: ops.int8_linear(x, w, 1.0, torch.ones(7, device="cuda")),
        lambda: ops.int8_linear(x, w, 1.0, out_dtype=torch.float64),
        lambda: ops.int8_linear(x, w, 1.0, out=torch.empty((4, 7), device="cuda")),
        lambda: ops.int8_linear(x, w, 1.0, out=torch.empty((8, 4), device="cuda").T),
        lambda: ops.int8_linear(x.float(), w, 1.0),
        lambda: ops.int8_linear(x.float().requires_grad_(), w),
        lambda: ops.Int8Weight(q.float(), ws),
        lambda: ops.Int8Weight(q, ws[:-1]),
        lambda: ops.quantize_rows(x),
        lambda: ops.int8_linear(torch.zeros((2, 40000), dtype=torch.uint8, device="cuda"),
                                ops.Int8Weight(torch.zeros((8, 40000), dtype=torch.int8, device="cuda"), ws), 1.0),
    ):
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("start", range(17))
@pytest.mark.parametrize("m", [1, 33, 64])
def test_few_rows_that_start_anywhere(m, start):
    ram = torch.randint(0, 256, (m, 1031), generator=_gen(start), device="cuda", dtype=torch.uint8)
    for k in (1 + start, 900 - start):
        for x in (ram[:, start:start + k], ram.view(torch.int8)[:, start:start + k]):
            q, ws = _weight(21, k, start)
            _check(ops.int8_linear(x, ops.Int8Weight(q, ws), 0.5, out_dtype=torch.float32), x, 0.5, q, ws, None, False)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [64, 63, 5000, 4999])
def test_quantize_rows_clamps_where_the_scale_is_subnormal(cols):
    """A scale of few units in the last place is rounded so coarsely that quotients pass 127: 190 units over 127 round to
    one unit.  They end at 127, not at what is left of them in 8 bits."""
    unit = 2.0 ** -149
    most = torch.cat([torch.arange(1, 700, device="cuda"), torch.tensor([4000, 16129, 100000], device="cuda")]).double()
    x = (torch.rand((len(most), cols), generator=_gen(4), device="cuda").double() * 2 - 1) * most[:, None]
    x[:, 0], x[:, 1] = most, -most
    x = (x.round() * unit).float()
    q, s = ops.quantize_rows(x)
    scale = ((most / 127).round() * unit).float()  # half to even, as IEEE division rounds it to a whole number of units
    quotient = x.double() / torch.where(scale > 0, scale, 1.0).double()[:, None]
    assert float(quotient.abs().max()) > 189
    assert torch.equal(s, scale) and torch.equal(q, quotient.float().round().clamp(-127, 127).to(torch.int8))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 130])
@pytest.mark.parametrize("dtype,k,value", [(torch.int8, 131071, -128), (torch.int8, 131056, -128), (torch.int8, 131071, 127),
                                           (torch.uint8, 33025, 255), (torch.uint8, 33024, 255)])
def test_extreme_sums_at_the_largest_k_are_exact(m, dtype, k, value):
    """128 * 128 * 131,071 and 255 * 255 * 33,025 (weights + 128) are just below 2^31."""
    x = torch.full((m, k), value, dtype=dtype, device="cuda")
    q = torch.full((5, k), -128, dtype=torch.int8, device="cuda")
    q[1::2] = 127
    y = ops.int8_linear(x, ops.Int8Weight(q, torch.ones(5, device="cuda")), 1.0, out_dtype=torch.float32)
    want = torch.tensor([float(k * value * int(w)) for w in q[:, 0]], device="cuda")  # rounded to fp32 once
    assert torch.equal(y, want.expand(m, 5))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,k", [(torch.int8, 131072), (torch.uint8, 33026)])
def test_sums_that_may_pass_32_bits_are_refused(dtype, k):
    w = ops.Int8Weight(torch.zeros((5, k), dtype=torch.int8, device="cuda"), torch.ones(5, device="cuda"))
    for m in (3, 130):
        with pytest.raises(ValueError, match="32-bit sums"):
            ops.int8_linear(torch.zeros((m, k), dtype=dtype, device="cuda"), w, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(40, 512, 256), (3000, 512, 256), (3000, 64, 32)])
def test_out_on_the_memory_of_the_tokens(m, k, n):
    """Other tiles still read the tokens when a tile's results are there."""
    room = torch.randint(0, 256, (m, k), generator=_gen(6), device="cuda", dtype=torch.uint8)
    x = room.clone()
    q, ws = _weight(n, k, 7)
    w = ops.Int8Weight(q, ws)
    want = ops.int8_linear(x, w, 0.5)
    out = room.view(torch.bfloat16)  # k bytes a row are k / 2 results
    assert out.shape == want.shape
    assert ops.int8_linear(room, w, 0.5, out=out) is out and torch.equal(out, want)
    both = torch.cat([x, torch.empty((m, 2 * n), dtype=torch.uint8, device="cuda")], 1)  # side by side in one record
    side = both[:, k:].view(torch.bfloat16)
    ops.int8_linear(both[:, :k], w, 0.5, out=side)
    assert torch.equal(side, want) and torch.equal(both[:, :k], x)
    scales = torch.rand(m, generator=_gen(8), device="cuda") + 0.1
    bias = torch.randn(n, generator=_gen(9), device="cuda")
    want = ops.int8_linear(x, w, scales, bias, out_dtype=torch.float32)
    store = torch.zeros((m, n), device="cuda")
    store[0] = bias
    assert torch.equal(ops.int8_linear(x, w, scales, store[0], out=store), want)


@pytest.mark.gpu
def test_a_gradient_that_saved_out_is_refused_when_it_has_been_written():
    q, ws = _weight(8, 32, 1)
    x, out = torch.ones((4, 32), dtype=torch.uint8, device="cuda"), torch.ones((4, 8), device="cuda")
    a = torch.ones_like(out).requires_grad_()
    saved = (a * out).sum()
    ops.int8_linear(x, ops.Int8Weight(q, ws), 1.0, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.backward()


@pytest.mark.gpu
def test_a_scale_that_wants_a_gradient_is_refused():
    q, ws = _weight(8, 32, 1)
    x, w = torch.ones((4, 32), dtype=torch.uint8, device="cuda"), ops.Int8Weight(q, ws)
    scale = torch.ones(4, device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="no gradient"):
        ops.int8_linear(x, w, scale)
    with torch.no_grad():
        assert torch.equal(ops.int8_linear(x, w, scale), ops.int8_linear(x, w, 1.0))


@pytest.mark.gpu
def test_an_out_that_wants_a_gradient_is_refused():
    q, ws = _weight(8, 32, 1)
    x, w = torch.ones((4, 32), dtype=torch.uint8, device="cuda"), ops.Int8Weight(q, ws)
    out = torch.ones((4, 8), device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="no gradient"):
        ops.int8_linear(x, w, 1.0, out=out)
    with torch.no_grad():
        assert torch.equal(ops.int8_linear(x, w, 1.0, out=out), ops.int8_linear(x, w, 1.0, out_dtype=torch.float32))


@pytest.mark.gpu
def test_no_columns_and_more_tokens_than_a_grid_holds():
    m, n = 65535 * 16 + 21, 6
    q, ws = _weight(n, 32, 1)
    bias = torch.arange(float(n), device="cuda")
    out = torch.full((m, 8), 7.0, device="cuda", dtype=torch.bfloat16)
    ops.int8_linear(torch.empty((m, 0), dtype=torch.int8, device="cuda"), ops.Int8Weight(q[:, :0], ws), torch.ones(m, device="cuda"),
                    bias, out=out[:, 1:7])
    assert torch.equal(out[:, 1:7], bias.to(torch.bfloat16).expand(m, n)) and bool((out[:, 0] == 7).all() and (out[:, 7] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("lead", [(), (3,), (2, 3), (2, 0, 4), (0,), (0, 5)])
@pytest.mark.parametrize("k", [0, 1, 20])
@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.bfloat16])
def test_any_leading_dimensions_and_none(lead, k, dtype):
    q, ws = _weight(6, k, 3) if k else (torch.empty((6, 0), dtype=torch.int8, device="cuda"), torch.ones(6, device="cuda"))
    w, bias = ops.Int8Weight(q, ws), torch.arange(6.0, device="cuda")
    x = torch.randint(0, 50, (*lead, k), generator=_gen(2), device="cuda").to(dtype)
    scale = None if dtype == torch.bfloat16 else torch.full(lead, 0.5, device="cuda")
    y = ops.int8_linear(x, w, scale, bias, out_dtype=torch.float32)
    assert y.shape == (*lead, 6)
    xq, xs = (x, scale) if scale is not None else ops.quantize_rows(x)
    assert xq.shape == x.shape and xs.shape == torch.Size(lead)
    rows = max(1, torch.Size(lead).numel()) if not lead else torch.Size(lead).numel()
    if rows:
        _check(y.reshape(rows, 6), xq.reshape(rows, k), xs.reshape(rows, 1).double(), q, ws, bias, False)
