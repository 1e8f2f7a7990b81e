"""The gated delta rule (nesle_b200.ops.delta_step, delta_scan) against the
recurrence token by token in 64 bits, its gradients against that recurrence's
derivative and against differences.

Tolerance.  Every output is a chain of fp32 sums of at most dk, dv or 16
products each; a sum of n products in fp32 is within n 2^-24 of the sum of their
magnitudes, and with keys of unit length and beta in (0, 1) a token's update
does not enlarge what came before.  Four such sums stand between the inputs and
any output (k.k, S k, the triangular solve, the read), on the way back as many
again: 8 (dk + dv + 16) 2^-24 of the tensor's largest magnitude, and one
rounding to the output's type."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from nesle_b200 import ops  # noqa: E402

NAMES = ("q", "k", "v", "g", "beta", "state")


@pytest.fixture(autouse=True, scope="module")
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from nesle_b200 import build

    build.build()


def inputs(t, n, h, dk, dv, dtype=torch.float32, p_reset=0.1, seed=0, decay=-2.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    k = normal(t, n, h, dk) + normal(1, n, h, dk)
    q = normal(t, n, h, dk)
    return {"q": (q / q.norm(dim=-1, keepdim=True)).to(dtype), "k": (k / k.norm(dim=-1, keepdim=True)).to(dtype),
            "v": normal(t, n, h, dv).to(dtype), "g": -torch.exp(normal(t, n, h) + decay),
            "beta": torch.sigmoid(normal(t, n, h)), "state": normal(n, h, dk, dv),
            "reset": torch.rand((t, n), generator=gen, device="cuda") < p_reset}


def reference(x, scale=None):
    """Token by token; differentiable, in the inputs' precision."""
    q, k, v, g, beta, state = (x[i] for i in NAMES)
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    out = []
    for t in range(q.shape[0]):
        state = torch.where(x["reset"][t][:, None, None, None], 0.0, torch.exp(g[t])[..., None, None] * state)
        u = beta[t][..., None] * (v[t] - torch.einsum("nhij,nhi->nhj", state, k[t]))
        state = state + torch.einsum("nhi,nhj->nhij", k[t], u)
        out.append(scale * torch.einsum("nhij,nhi->nhj", state, q[t]))
    return (torch.stack(out) if out else v[:0]), state


def close(got, want, dk, dv, what):
    want = want.double()
    tol = 8 * (dk + dv + 16) * 2.0 ** -24 * float(want.abs().max()) if want.numel() else 0.0
    if got.dtype != torch.float32:
        tol = tol + want.abs() * torch.finfo(got.dtype).eps / 2 + torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps
    assert got.shape == want.shape, what
    off = (got.double() - want).abs() - tol
    assert bool((off <= 0).all()), f"{what}: {float(off.max())} over the tolerance"


def check(x, train=True, seed=5, scale=None):
    dk, dv = x["q"].shape[-1], x["v"].shape[-1]
    wide = {i: (y.double().requires_grad_(train) if i != "reset" else y) for i, y in x.items()}
    want_o, want_s = reference(wide, scale)
    mine = {i: (y.detach().requires_grad_(train) if i != "reset" else y) for i, y in x.items()}
    o, s = ops.delta_scan(*(mine[i] for i in NAMES), mine["reset"], scale=scale)
    assert o.dtype == x["v"].dtype and s.dtype == torch.float32
    close(o.detach(), want_o.detach(), dk, dv, "o")
    close(s.detach(), want_s.detach(), dk, dv, "state")
    if not train:
        return
    gen = torch.Generator(device="cuda").manual_seed(seed)
    d_o = torch.randn(o.shape, generator=gen, device="cuda").to(o.dtype)
    d_s = torch.randn(s.shape, generator=gen, device="cuda")
    want = torch.autograd.grad([want_o, want_s], [wide[i] for i in NAMES], [d_o.double(), d_s.double()], allow_unused=True)
    got = torch.autograd.grad([o, s], [mine[i] for i in NAMES], [d_o, d_s])
    for i, a, b in zip(NAMES, got, want):
        assert a.dtype == x[i].dtype
        close(a, torch.zeros_like(a) if b is None else b, dk, dv, "d" + i)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [1, 2, 15, 16, 17, 31, 33, 64, 100])
@pytest.mark.parametrize("p_reset", [0.0, 0.15])
def test_lengths(t, p_reset):
    check(inputs(t, 3, 2, 64, 64, torch.bfloat16, p_reset, seed=t))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dk,dv", [(1, 1), (3, 5), (16, 16), (32, 32), (40, 72), (64, 16), (16, 128), (128, 32), (33, 65),
                                   (64, 64), (128, 128), (127, 127)])
def test_head_sizes_and_types(dk, dv, dtype):
    check(inputs(21, 2, 3, dk, dv, dtype, 0.08, seed=dk + dv))


@pytest.mark.gpu
@pytest.mark.parametrize("every", [1, 2, 5, 16])
def test_frequent_episode_ends(every):
    """Several episodes in one block of 16 tokens; at 1 every token stands alone."""
    x = inputs(40, 3, 1, 32, 48, torch.float32, 0.0, seed=every)
    x["reset"][::every] = True
    check(x)


@pytest.mark.gpu
def test_only_some_envs_restart():
    x = inputs(50, 4, 2, 64, 64, torch.bfloat16, 0.0, seed=1)
    x["reset"][0, 1] = x["reset"][49, 2] = True
    x["reset"][16:33, 3] = True
    check(x)


@pytest.mark.gpu
@pytest.mark.parametrize("decay", [-8.0, 1.0, 4.0])
def test_weak_and_strong_decays(decay):
    """From almost none to states that vanish from token to token; exp(g) underflows in the last."""
    check(inputs(48, 2, 2, 64, 64, torch.float32, 0.02, seed=3, decay=decay))


@pytest.mark.gpu
def test_repeated_keys():
    """The same key at every token with beta = 1: the system's matrix is all ones below the diagonal."""
    x = inputs(64, 2, 2, 64, 64, torch.float32, 0.0, seed=4)
    x["k"] = x["k"][:1].expand(64, -1, -1, -1).contiguous()
    x["beta"] = torch.ones_like(x["beta"])
    x["g"] = torch.zeros_like(x["g"])
    check(x)


@pytest.mark.gpu
def test_infinite_decay_is_a_gate_that_closes():
    x = inputs(20, 2, 2, 32, 32, torch.float32, 0.0, seed=6)
    x["g"][7, 0] = x["g"][16, 1] = float("-inf")
    o, s = ops.delta_scan(*(x[i] for i in NAMES), x["reset"])
    want_o, want_s = reference({i: (y if i == "reset" else y.double()) for i, y in x.items()})
    close(o, want_o, 32, 32, "o")
    close(s, want_s, 32, 32, "state")


@pytest.mark.gpu
def test_no_state_and_no_resets():
    x = inputs(30, 3, 2, 64, 32, torch.bfloat16, 0.0, seed=8)
    a, sa = ops.delta_scan(*(x[i] for i in NAMES[:5]))
    b, sb = ops.delta_scan(*(x[i] for i in NAMES[:5]), torch.zeros_like(x["state"]), x["reset"].to(torch.uint8))
    assert torch.equal(a, b) and torch.equal(sa, sb)


@pytest.mark.gpu
def test_nothing_passes_a_reset():
    """NaN and infinities of an ended episode, and of its state, stay in it, forward and back."""
    x = inputs(40, 2, 1, 64, 64, torch.float32, 0.0, seed=9)
    x["reset"][21] = True
    bad = {i: y.clone() for i, y in x.items()}
    bad["state"][:] = float("nan")
    for i in ("q", "k", "v"):
        bad[i][20] = float("inf")
        bad[i][3] = float("nan")
    bad["g"][18], bad["beta"][17] = float("nan"), float("nan")
    grads = []
    for y in (x, bad):
        leaf = {i: z.clone().requires_grad_() for i, z in y.items() if i != "reset"}
        o, s = ops.delta_scan(*(leaf[i] for i in NAMES), y["reset"])
        g = torch.autograd.grad([o[21:], s], [leaf[i] for i in NAMES[:5]], [torch.ones_like(o[21:]), torch.ones_like(s)])
        grads.append((o[21:], s, *(z[21:] for z in g)))
    for a, b in zip(*grads):
        assert bool(torch.isfinite(b).all()) and torch.equal(a, b)
    # and back: a NaN in the later episode's gradients does not reach the earlier one
    leaf = {i: z.clone().requires_grad_() for i, z in x.items() if i != "reset"}
    o, s = ops.delta_scan(*(leaf[i] for i in NAMES), x["reset"])
    d = torch.ones_like(o)
    d[25] = float("nan")
    g = torch.autograd.grad([o, s], [leaf[i] for i in NAMES], [d, torch.full_like(s, float("nan"))])
    for z in g[:5]:
        assert bool(torch.isfinite(z[:21]).all())
    assert bool(torch.isfinite(g[5]).all())


@pytest.mark.gpu
def test_gradient_against_differences():
    x = {i: (y if i == "reset" else y.double()) for i, y in inputs(19, 1, 2, 8, 8, torch.float32, 0.1, seed=10).items()}
    leaf = {i: y.float().requires_grad_() for i, y in x.items() if i != "reset"}
    o, s = ops.delta_scan(*(leaf[i] for i in NAMES), x["reset"])
    gen = torch.Generator(device="cuda").manual_seed(2)
    wo, wst = torch.randn(o.shape, generator=gen, device="cuda"), torch.randn(s.shape, generator=gen, device="cuda")
    grads = torch.autograd.grad([o, s], [leaf[i] for i in NAMES], [wo, wst])
    for i, grad in zip(NAMES, grads):
        way = torch.randn(grad.shape, generator=gen, device="cuda").double()
        sides = []
        for sign in (1, -1):
            y = dict(x, **{i: x[i] + sign * 1e-4 * way})
            ro, rs = reference(y)
            sides.append(float((ro * wo).sum() + (rs * wst).sum()))
        slope = (sides[0] - sides[1]) / 2e-4
        # central differences in 64 bits: an error of order 1e-8; the gradient's is fp32's
        assert abs(slope - float((grad.double() * way).sum())) <= 1e-4 * (abs(slope) + float(grad.double().norm() * way.norm()) * 0.1)


@pytest.mark.gpu
def test_strides():
    """Slices of one projection, env-major storage, expanded and unaligned tensors."""
    t, n, h, d = 37, 3, 2, 32
    x = inputs(t, n, h, d, d, torch.bfloat16, 0.1, seed=11)
    fused = torch.cat([x["q"], x["k"], x["v"]], -1)
    y = dict(x, q=fused[..., :d], k=fused[..., d:2 * d], v=fused[..., 2 * d:])
    check(y)
    odd = torch.cat([torch.zeros((t, n, h, 3), device="cuda", dtype=torch.bfloat16), fused], -1)
    check(dict(x, q=odd[..., 3:d + 3], k=odd[..., d + 3:2 * d + 3], v=odd[..., 2 * d + 3:]))
    check(dict(x, q=x["q"].transpose(0, 1).contiguous().transpose(0, 1), g=x["g"][:1].expand(t, n, h),
               reset=x["reset"][:, :1].expand(t, n), k=x["k"].transpose(2, 3).contiguous().transpose(2, 3)))


@pytest.mark.gpu
def test_long_sequence_and_many_heads():
    check(inputs(700, 2, 1, 64, 64, torch.bfloat16, 0.003, seed=12))
    check(inputs(5, 300, 3, 32, 32, torch.bfloat16, 0.05, seed=13), train=True)


def is_cut(t, n, h, dk, dv):
    return ops._scan_split(t, n, h, dk, dv, torch.cuda.current_device()) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,n,h,dk,dv", [(640, 1, 1, 64, 64), (801, 2, 2, 128, 128), (655, 1, 2, 32, 32), (999, 1, 1, 40, 72),
                                         (641, 2, 1, 33, 65), (700, 1, 1, 128, 16), (700, 1, 2, 16, 128), (650, 1, 1, 1, 3)])
def test_cut_sequences(t, n, h, dk, dv, dtype):
    """A few long sequences run as segments side by side, joined by one more product: S <- A S + B."""
    assert is_cut(t, n, h, dk, dv)
    check(inputs(t, n, h, dk, dv, dtype, 0.003, seed=t + dk), train=dtype == torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("decay", [-8.0, 3.0])
@pytest.mark.parametrize("p_reset", [0.0, 0.4])
def test_cut_sequences_of_weak_decays_and_many_episodes(decay, p_reset):
    assert is_cut(1030, 2, 1, 64, 64) and not is_cut(1030, 1024, 4, 64, 64) and not is_cut(64, 2, 1, 64, 64)
    check(inputs(1030, 2, 1, 64, 64, torch.float32, p_reset, seed=20, decay=decay), train=False)


@pytest.mark.gpu
def test_repeated_keys_in_cut_sequences():
    x = inputs(640, 1, 2, 64, 64, torch.float32, 0.0, seed=21)
    x["k"] = x["k"][:1].expand(640, -1, -1, -1).contiguous()
    x["beta"] = torch.ones_like(x["beta"])
    x["g"] = torch.zeros_like(x["g"])
    check(x, train=False)


@pytest.mark.gpu
def test_nothing_passes_a_reset_in_cut_sequences():
    """NaN of a state and of tokens stay in their episode, whatever segments it spans."""
    t = 900
    assert is_cut(t, 2, 1, 64, 64)
    x = inputs(t, 2, 1, 64, 64, torch.bfloat16, 0.0, seed=22)
    x["reset"][700] = True
    bad = {i: y.clone() for i, y in x.items()}
    bad["state"][:] = float("nan")
    bad["k"][300], bad["v"][690], bad["g"][400], bad["q"][699] = float("nan"), float("inf"), float("nan"), float("inf")
    for a, b in zip(*(ops.delta_scan(*(y[i] for i in NAMES), y["reset"]) for y in (x, bad))):
        a, b = (a[700:], b[700:]) if len(a) == t else (a, b)
        assert bool(torch.isfinite(b).all()) and torch.equal(a, b)


@pytest.mark.gpu
def test_cut_sequences_strides_streams_graphs_and_workspaces():
    t, n, h, d = 645, 2, 1, 32
    x = inputs(t, n, h, d, d, torch.bfloat16, 0.004, seed=23)
    odd = torch.cat([torch.zeros((t, n, h, 3), device="cuda", dtype=torch.bfloat16), x["q"], x["k"], x["v"]], -1)
    check(dict(x, q=odd[..., 3:d + 3], k=odd[..., d + 3:2 * d + 3], v=odd[..., 2 * d + 3:]), train=False)
    want = ops.delta_scan(*(x[i] for i in NAMES), x["reset"])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = [ops.delta_scan(*(x[i] for i in NAMES), x["reset"]) for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(a, b) for r in again for a, b in zip(want, r))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.delta_scan(*(x[i] for i in NAMES), x["reset"])
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    # the C entry: without a workspace one scan, with one that is not aligned a refusal
    o, s = torch.empty_like(want[0]), torch.empty_like(want[1])
    dev = torch.cuda.current_device()
    args = ops._scan_args(x["q"], x["k"], x["v"], x["g"], x["beta"], x["reset"], x["state"], d ** -0.5, dev, o.data_ptr(), s.data_ptr())
    ops._call("nesle_delta_scan_split", args, 0, torch.cuda.current_stream().cuda_stream)
    wide = {i: (y if i == "reset" else y.double()) for i, y in x.items()}
    for got, ref, name in zip((o, s), reference(wide), ("o", "state")):
        close(got, ref, d, d, name)
    with pytest.raises(ValueError, match="workspace"):
        ops._call("nesle_delta_scan_split", args, s.data_ptr() + 2, torch.cuda.current_stream().cuda_stream)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,h,dk,dv", [(1, 1, 64, 64), (5, 3, 64, 64), (33, 2, 128, 128), (4, 1, 1, 1), (7, 2, 40, 72), (3, 2, 33, 65),
                                       (2, 1, 16, 7), (300, 4, 32, 32)])
def test_step_is_the_recurrence(n, h, dk, dv, dtype):
    x = inputs(6, n, h, dk, dv, dtype, 0.2, seed=n + dk)
    state = x["state"].clone()
    got = [ops.delta_step(*(x[i][t] for i in NAMES[:5]), state, x["reset"][t]) for t in range(6)]
    want_o, want_s = reference({i: (y if i == "reset" else y.double()) for i, y in x.items()})
    close(torch.stack(got), want_o, dk, dv, "o")
    close(state, want_s, dk, dv, "state")


@pytest.mark.gpu
def test_step_strides_and_reset_of_a_broken_state():
    x = inputs(1, 9, 2, 64, 64, torch.bfloat16, 0.0, seed=3)
    store = torch.full((9, 3, 64 * 64 + 4), 5.0, device="cuda")
    state = store[:, 1:, :64 * 64].unflatten(2, (64, 64))
    state.copy_(x["state"])
    state[4] = float("nan")
    x["state"][4] = float("nan")
    x["reset"][0, 4] = True
    out = torch.empty((9, 2, 64), device="cuda", dtype=torch.bfloat16)
    ops.delta_step(*(x[i][0] for i in NAMES[:5]), state, x["reset"][0].to(torch.uint8), scale=0.5, out=out)
    x["state"][4] = 0
    want_o, want_s = reference({i: (y if i == "reset" else y.double()) for i, y in x.items()}, 0.5)
    close(out, want_o[0], 64, 64, "o")
    close(state, want_s, 64, 64, "state")
    assert bool((store[:, 0] == 5).all()) and bool((store[:, :, 64 * 64:] == 5).all())
    odd = torch.empty(9 * 2 * 64 * 64 + 1, device="cuda")[1:].view(9, 2, 64, 64)  # not on 16 bytes
    odd.copy_(x["state"])
    ops.delta_step(*(x[i][0] for i in NAMES[:5]), odd, x["reset"][0], scale=0.5, out=out)
    close(out, want_o[0], 64, 64, "o")
    close(odd, want_s, 64, 64, "state")


@pytest.mark.gpu
def test_rollout_steps_match_the_update_scan():
    """What the rollout computed step by step the update computes again at once."""
    x = inputs(40, 6, 2, 64, 64, torch.bfloat16, 0.05, seed=14)
    state = x["state"].clone()
    steps = torch.stack([ops.delta_step(*(x[i][t] for i in NAMES[:5]), state, x["reset"][t]) for t in range(40)])
    o, s = ops.delta_scan(*(x[i] for i in NAMES), x["reset"])
    close(s, state, 64, 64, "state")
    scale = float(o.float().abs().max())
    assert float((o.float() - steps.float()).abs().max()) <= 2 * 2.0 ** -8 * scale


@pytest.mark.gpu
def test_other_stream_graph_and_repeatability():
    x = inputs(50, 40, 2, 64, 64, torch.bfloat16, 0.02, seed=15)
    leaf = {i: y.clone().requires_grad_() for i, y in x.items() if i != "reset"}

    def once():
        o, s = ops.delta_scan(*(leaf[i] for i in NAMES), x["reset"])
        return (o.detach(), s.detach(), *torch.autograd.grad([o, s], [leaf[i] for i in NAMES], [torch.ones_like(o), torch.ones_like(s)]))

    first = once()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = [once() for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(a, b) for r in again for a, b in zip(first, r))
    state, out = x["state"].clone(), torch.empty((40, 2, 64), device="cuda", dtype=torch.bfloat16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.delta_step(*(x[i][0] for i in NAMES[:5]), state, x["reset"][0], out=out)
    state.copy_(x["state"])
    graph.replay()
    want = x["state"].clone()
    assert torch.equal(out, ops.delta_step(*(x[i][0] for i in NAMES[:5]), want, x["reset"][0])) and torch.equal(state, want)


@pytest.mark.gpu
def test_empty_sizes():
    x = inputs(0, 2, 2, 16, 16)
    leaf = {i: y.clone().requires_grad_() for i, y in x.items() if i != "reset"}
    o, s = ops.delta_scan(*(leaf[i] for i in NAMES), x["reset"])
    assert o.shape == (0, 2, 2, 16) and torch.equal(s, x["state"])
    g = torch.autograd.grad([o, s], [leaf["state"]], [torch.zeros_like(o), torch.full_like(s, 2.0)])
    assert bool((g[0] == 2).all())
    x = inputs(3, 0, 2, 16, 16)
    o, s = ops.delta_scan(*(x[i] for i in NAMES), x["reset"])
    assert o.shape == (3, 0, 2, 16) and s.shape == (0, 2, 16, 16)
    assert ops.delta_step(*(x[i][0] for i in NAMES[:5]), x["state"], x["reset"][0]).shape == (0, 2, 16)


@pytest.mark.gpu
def test_only_what_is_asked_for_has_a_gradient():
    x = inputs(20, 2, 2, 32, 32, seed=16)
    v = x["v"].clone().requires_grad_()
    o, s = ops.delta_scan(x["q"], x["k"], v, x["g"], x["beta"], x["state"], x["reset"])
    a = torch.autograd.grad(o.sum(), v, retain_graph=True)[0]
    b = torch.autograd.grad(s.sum(), v)[0]
    wide = {i: (y if i == "reset" else y.double()) for i, y in x.items()}
    wide["v"].requires_grad_()
    ro, rs = reference(wide)
    close(a, torch.autograd.grad(ro.sum(), wide["v"], retain_graph=True)[0], 32, 32, "dv of o")
    close(b, torch.autograd.grad(rs.sum(), wide["v"])[0], 32, 32, "dv of the state")


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    x = inputs(5, 1, 1, 16, 16, seed=17)
    q = x["q"].clone().requires_grad_()
    o, _ = ops.delta_scan(q, x["k"], x["v"], x["g"], x["beta"], x["state"])
    with pytest.raises(RuntimeError):
        torch.autograd.grad(o.square().sum(), q, create_graph=True)


@pytest.mark.gpu
def test_refusals():
    x = inputs(3, 2, 2, 16, 16)
    args = [x[i] for i in NAMES]

    def but(i, y):
        return [y if j == i else z for j, z in enumerate(args)]

    for bad in (but(0, args[0].cpu()), but(0, args[0].double()), but(1, args[1].half()), but(1, args[1][..., :8]), but(2, args[2][:2]),
                but(3, args[3].double()), but(4, args[4][:, :, :1]), but(5, args[5].half()), but(5, args[5][:1])):
        with pytest.raises(ValueError):
            ops.delta_scan(*bad, x["reset"])
    with pytest.raises(ValueError):
        ops.delta_scan(*args, x["reset"].float())
    with pytest.raises(ValueError):
        ops.delta_scan(*args, x["reset"][:2])
    wide = inputs(2, 1, 1, 129, 16)
    with pytest.raises(ValueError):
        ops.delta_scan(*(wide[i] for i in NAMES), wide["reset"])
    one = [x[i][0] for i in NAMES[:5]]
    for call in (
        lambda: ops.delta_step(*one, x["state"].half()),
        lambda: ops.delta_step(*one, x["state"].transpose(2, 3)),
        lambda: ops.delta_step(*one, x["state"][:1].expand(2, 2, 16, 16)),
        lambda: ops.delta_step(*one, x["state"], x["reset"]),
        lambda: ops.delta_step(*one, x["state"], out=torch.empty((2, 2, 16), device="cuda", dtype=torch.bfloat16)),
        lambda: ops.delta_step(*one, x["state"].clone().requires_grad_()),
    ):
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("on", ["q", "k", "v", "q of another env", "state"])
@pytest.mark.parametrize("dk", [32, 128])
def test_step_writes_out_on_the_memory_of_an_input(on, dk):
    """As if the output were written after everything has been read."""
    x = inputs(1, 300, 2, dk, dk, torch.float32, 0.0, seed=30)
    one = [x[i][0].clone() for i in NAMES[:5]]
    state = x["state"].clone()
    want = ops.delta_step(*one, state)
    again = x["state"].clone()
    if on == "q of another env":
        room = torch.cat([one[0], one[0][:1]])
        one[0], out = room[:-1], room[1:]
    else:
        out = again.view(-1)[5:5 + 300 * 2 * dk].view(300, 2, dk) if on == "state" else one["qkv".index(on)]
    got = ops.delta_step(*one, again, out=out)
    assert got is out and torch.equal(out, want)
    if on != "state":
        assert torch.equal(again, state)


@pytest.mark.gpu
@pytest.mark.parametrize("aliased", [False, True])
def test_a_gradient_that_saved_the_state_or_out_is_refused_after_a_step(aliased):
    """As after any torch operation in place; it would be that of the new values."""
    x = inputs(1, 2, 1, 16, 16, seed=31)
    one = [x[i][0] for i in NAMES[:5]]
    state, out = x["state"], one[2] if aliased else torch.ones((2, 1, 16), device="cuda")
    for written in (state, state[:1], out):  # a view is the same memory
        a = torch.ones_like(written).requires_grad_()
        saved = (a * written).sum()
        ops.delta_step(*one, state, out=out)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            saved.backward()
    a = torch.ones_like(one[0]).requires_grad_()
    saved = (a * one[0]).sum()
    ops.delta_step(*one, state)
    saved.backward()  # inputs are not written
    assert torch.equal(a.grad, one[0])
    with torch.inference_mode():
        state = x["state"].clone()
        want = ops.delta_step(*one, state)
    state.sum(), want.sum()
    ops.delta_step(*one, state)  # has no version to raise


@pytest.mark.gpu
def test_an_out_that_wants_a_gradient_is_refused():
    x = inputs(1, 2, 1, 16, 16, seed=32)
    out = torch.ones((2, 1, 16), device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="no gradient"):
        ops.delta_step(*(x[i][0] for i in NAMES[:5]), x["state"], out=out)
    with torch.no_grad():
        want = ops.delta_step(*(x[i][0] for i in NAMES[:5]), x["state"].clone())
        assert torch.equal(ops.delta_step(*(x[i][0] for i in NAMES[:5]), x["state"], out=out), want)


@pytest.mark.gpu
def test_tangents_are_refused():
    from torch.autograd import forward_ad

    x = inputs(1, 2, 1, 16, 16, seed=33)
    one = [x[i][0] for i in NAMES[:5]] + [x["state"]]
    q = torch.ones((4, 16), dtype=torch.int8, device="cuda")
    w = ops.Int8Weight(q, torch.ones(4, device="cuda"))
    with forward_ad.dual_level():
        for i in range(6):
            args = [forward_ad.make_dual(y, torch.ones_like(y)) if i == j else y for j, y in enumerate(one)]
            with pytest.raises(ValueError, match="forward-mode"):
                ops.delta_step(*args)
            with pytest.raises(NotImplementedError):
                ops.delta_scan(*(y[None] for y in args[:5]), args[5])
        ones = forward_ad.make_dual(torch.ones((4, 16), device="cuda"), torch.ones((4, 16), device="cuda"))
        for call in (lambda: ops.orthogonalize(ones), lambda: ops.quantize_rows(ones), lambda: ops.int8_linear(ones, w),
                     lambda: ops.int8_linear(q, w, 1.0, ones[0, :4]), lambda: ops.int8_linear(q, w, ones[:, 0])):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
        ops.delta_step(*one)


@pytest.mark.gpu
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("name", ["q", "k", "v", "g", "beta"])
@pytest.mark.parametrize("t,dk,dv,dtype", [(40, 64, 64, torch.bfloat16), (40, 64, 64, torch.float32), (40, 128, 128, torch.float16),
                                           (40, 40, 72, torch.bfloat16), (40, 33, 65, torch.float32), (700, 64, 64, torch.bfloat16)])
def test_what_is_not_finite_reaches_no_earlier_token(t, dk, dv, dtype, name, value):
    """As in the recurrence, token by token: a token that is not finite leaves those before it, and columns of the state that
    it does not reach, as they are; several in one block of 16, in the first token and in the last of the sequence."""
    x = inputs(t, 2, 2, dk, dv, dtype, 0.0, seed=34)
    assert is_cut(t, 2, 2, dk, dv) == (t == 700)
    for at, n in ((13, 0), (t - 1, 1)):
        x[name].view(t, 2, 2, -1)[at, n, 0, -1] = value
    x["v"][9, 0, 1, 2], x["v"][15, 0, 1, 3], x["v"][22, 0, 1, 2] = value, value, value  # columns of their own
    x["k"][16, 1, 1, 0] = value
    want_o, want_s = reference({i: (y if i == "reset" else y.double()) for i, y in x.items()})
    o, s = ops.delta_scan(*(x[i] for i in NAMES), x["reset"])
    for got, want, what in ((o, want_o, "o"), (s, want_s, "state")):
        finite = torch.isfinite(want)
        assert bool(finite.any()) and not bool(finite.all())
        assert torch.equal(torch.isfinite(got), finite), what
        close(torch.where(finite, got, 0), torch.where(finite, want, 0), dk, dv, what)


def segments(t, n, h, d, dtype):
    floats = ops._scan_split(t, n, h, d, d, torch.cuda.current_device(), ops._DTYPE[dtype])
    return 1 + floats // (n * h * (2 * d * d + 1))


@pytest.mark.gpu
def test_cutting_goes_by_what_an_sm_holds_of_the_type():
    """Heads of 128 in 16 and 32 bits by terms leave room for one block on an SM, in bfloat16 for two: sequences whose
    segments would come one after another anyway are left whole."""
    if torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("the counts are those of 148 SMs")
    wide = (torch.bfloat16, torch.float16, torch.float32)
    assert [segments(4096, 4, 4, 128, x) for x in wide] == [6, 8, 8]
    assert [segments(512, 4, 4, 128, x) for x in wide] == [6, 3, 3]
    assert [segments(4096, 4, 4, 64, x) for x in wide] == [15, 18, 18]
    assert [segments(1024, 8, 4, 128, x) for x in wide] == [1, 1, 1]
    assert [segments(4096, 12, 4, 128, x) for x in wide] == [3, 1, 1]
    for dtype in wide:  # what is cut so is the recurrence still
        check(inputs(512, 4, 4, 128, 128, dtype, 0.003, seed=35), train=False)
        check(inputs(1040, 1, 1, 64, 64, dtype, 0.003, seed=36), train=False)


@pytest.mark.gpu
def test_states_that_overlap_are_refused():
    x = inputs(1, 3, 2, 4, 5, seed=37)
    one = [x[i][0] for i in NAMES[:5]]
    room = torch.zeros(300, device="cuda")
    for strides in ((20, 20), (20, 40), (39, 20), (20, 50), (19, 100), (100, 19)):
        with pytest.raises(ValueError, match="overlap"):
            ops.delta_step(*one, room.as_strided((3, 2, 4, 5), (*strides, 5, 1)))
    want = x["state"].clone()
    o = ops.delta_step(*one, want)
    for strides in ((40, 20), (20, 60), (41, 20), (21, 63)):  # either dimension may be the outer one
        state = torch.zeros(200, device="cuda").as_strided((3, 2, 4, 5), (*strides, 5, 1))
        state.copy_(x["state"])
        assert torch.equal(ops.delta_step(*one, state), o) and torch.equal(state, want)
