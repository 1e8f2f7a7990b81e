"""The recurrent PPO loop (nesle_b200.memory_ppo) and its optimiser
(nesle_b200.muon): the rollout's 8-bit, step-by-step policy against the update's
bf16 sequence form, the env side replayed on the checker, and Muon against its
formula in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from nesle_b200 import build

    build.build()


def test_configuration_is_checked():
    from nesle_b200.memory_ppo import MemoryPPOConfig, MemoryPPOTrainer

    with pytest.raises(ValueError, match="whole sequences"):
        MemoryPPOTrainer(MemoryPPOConfig(num_envs=64, n_steps=24, batch_size=100))


def test_muon_refusals():
    from nesle_b200.muon import Muon

    with pytest.raises(ValueError):
        Muon([torch.nn.Parameter(torch.zeros(4))])
    with pytest.raises(ValueError):
        Muon([torch.nn.Parameter(torch.zeros(4, 4))], lr=-1.0)
    with pytest.raises(ValueError):
        Muon([torch.nn.Parameter(torch.zeros(4, 4))], momentum=1.0)
    with pytest.raises(ValueError):
        Muon([torch.nn.Parameter(torch.zeros(4, 4))], steps=0)


@pytest.mark.gpu
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_follows_its_formula(cuda, nesterov):
    from nesle_b200.muon import Muon

    gen = torch.Generator("cuda").manual_seed(1)
    shapes = [(96, 160), (160, 96), (96, 160), (33, 7)]
    params = [torch.nn.Parameter(torch.randn(s, generator=gen, device="cuda")) for s in shapes]
    want = [p.detach().double().clone() for p in params]
    momenta = [torch.zeros_like(x) for x in want]
    opt = Muon(params, lr=0.05, momentum=0.9, nesterov=nesterov, weight_decay=0.1)
    for _ in range(3):
        for i, p in enumerate(params):
            p.grad = torch.randn(p.shape, generator=gen, device="cuda")
            g = p.grad.double()
            momenta[i] = 0.9 * momenta[i] + g
            x = g + 0.9 * momenta[i] if nesterov else momenta[i]
            x = x / x.norm()
            x = x.T if x.shape[0] > x.shape[1] else x
            for _ in range(5):
                a = x @ x.T
                x = 3.4445 * x + (-4.7750 * a + 2.0315 * a @ a) @ x
            x = x.T if p.shape[0] > p.shape[1] else x
            want[i] = want[i] * (1 - 0.05 * 0.1) - 0.05 * max(1.0, p.shape[0] / p.shape[1]) ** 0.5 * x
        opt.step()
    for p, x in zip(params, want):
        # three steps of bf16 directions (2^-8 of entries below 1.3) and fp32 arithmetic on weights of order one
        size = max(1.0, p.shape[0] / p.shape[1]) ** 0.5
        assert float((p.detach().double() - x).abs().max()) <= 3 * 0.05 * size * 1.3 * 2.0 ** -8 + 12 * 5.0 * 2.0 ** -24
    opt.zero_grad(set_to_none=True)
    before = [p.detach().clone() for p in params]
    opt.step()  # nothing has a gradient
    assert all(torch.equal(a, b.detach()) for a, b in zip(before, params))


@pytest.mark.gpu
def test_sequence_form_agrees_with_the_rollout(cuda):
    """The update computes again what the rollout did: 8-bit weights (127 levels of a row's largest) and activations
    against bf16 ones, the same memory."""
    from nesle_b200.memory_ppo import MemoryPPOConfig, MemoryPPOTrainer

    tr = MemoryPPOTrainer(MemoryPPOConfig(num_envs=32, n_steps=12, batch_size=96, update_epochs=1))
    tr.rollout()
    with torch.no_grad():
        logits, value, state = tr.model(tr.obs_buf, tr.done_buf != 0, tr.first_state)
    logp = torch.log_softmax(logits, -1).gather(2, tr.act_buf[..., None]).squeeze(2)
    assert float((logp - tr.logp_buf).abs().max()) < 0.05
    assert float((value - tr.val_buf).abs().max()) < 0.1 * (1 + float(tr.val_buf.abs().max()))
    assert float((state - tr.state).norm() / state.norm()) < 0.1
    assert torch.isfinite(tr.state).all() and float(tr.state.abs().max()) > 0


@pytest.mark.gpu
def test_training_runs_and_env_side_replays_on_checker(cuda):
    from nesle_b200 import ops
    from nesle_b200 import workloads as w
    from nesle_b200.memory_ppo import MemoryPPOConfig, MemoryPPOTrainer
    from oracle import Oracle

    cfg = MemoryPPOConfig(num_envs=48, n_steps=8, batch_size=128, update_epochs=2)
    tr = MemoryPPOTrainer(cfg)
    wl = tr.wl
    o = Oracle(cfg.num_envs, cfg.frameskip, wl.rom.image, wl.snapshots, done_mode=wl.done_mode, done_args=wl.done_args,
               seed=wl.seed)
    masks = np.asarray(w.SIMPLE_MOVEMENT_MASKS, np.uint8)
    before = {n: p.detach().clone() for n, p in tr.model.named_parameters()}
    for _ in range(2):
        tr.rollout()
        acts, obs = tr.act_buf.cpu().numpy(), tr.obs_buf.cpu().numpy()
        for t in range(cfg.n_steps):
            np.testing.assert_array_equal(obs[t], o.get("ram"), err_msg=f"obs before step {t}")
            o.step(masks[acts[t]])
        assert np.isfinite(float(tr.update()["loss"]))
    changed = [n for n, p in tr.model.named_parameters() if not torch.equal(p.detach(), before[n])]
    assert set(changed) == set(before)  # every parameter has a gradient and moved
    assert all(torch.isfinite(p).all() for p in tr.model.parameters())
    assert ops.stalls() == 0


@pytest.mark.gpu
def test_a_reset_clears_the_memory_of_its_env(cuda):
    from nesle_b200.memory_ppo import MemoryPPOConfig, MemoryPPOTrainer

    tr = MemoryPPOTrainer(MemoryPPOConfig(num_envs=16, n_steps=4, batch_size=64))
    tr.rollout()
    reset = torch.zeros(16, dtype=torch.bool, device="cuda")
    reset[3] = True
    kept, cleared = tr.state.clone(), tr.state.clone()
    cleared[3] = 0
    a = tr.model.step(tr.obs, reset, kept)
    b = tr.model.step(tr.obs, torch.zeros_like(reset), cleared)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    # a memory decayed from nothing is nothing; the others are untouched by the flag
    assert torch.equal(kept, cleared)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_muon_keeps_its_momentum_in_32_bits(cuda, dtype):
    """A running sum of 40 gradients: each step rounds it twice, to 2^-24 of at most 20 gradients of below 6."""
    from nesle_b200.muon import Muon

    gen = torch.Generator("cuda").manual_seed(5)
    params = [torch.nn.Parameter(torch.randn(s, generator=gen, device="cuda").to(dtype)) for s in ((48, 96), (48, 96), (7, 5))]
    opt = Muon(params, lr=0.01, momentum=0.95)
    want = [torch.zeros(p.shape, device="cuda", dtype=torch.float64) for p in params]
    for _ in range(40):
        for i, p in enumerate(params):
            p.grad = torch.randn(p.shape, generator=gen, device="cuda").to(dtype)
            want[i] = 0.95 * want[i] + p.grad.double()
        opt.step()
    for p, x in zip(params, want):
        got = opt.state[p]["momentum"]
        assert got.dtype == torch.float32 and p.dtype == dtype and bool(torch.isfinite(p).all())
        assert float((got.double() - x).abs().max()) <= 40 * 2 * 2.0 ** -24 * 120
    again = Muon([torch.nn.Parameter(p.detach().clone()) for p in params], lr=0.5)
    again.load_state_dict(opt.state_dict())
    assert again.param_groups[0]["lr"] == 0.01
    for p, x in zip(again.param_groups[0]["params"], params):
        a, b = again.state[p]["momentum"], opt.state[x]["momentum"]
        assert a.dtype == torch.float32 and torch.equal(a, b) and a.data_ptr() != b.data_ptr()


def test_training_stops_where_a_kernel_has_given_up(monkeypatch):
    """The counter is read once an iteration; what it held before does not count."""
    from types import SimpleNamespace

    from nesle_b200 import memory_ppo, ops

    done = []
    trainer = SimpleNamespace(iteration=lambda: done.append(1) or {"loss": 1.0}, global_step=0,
                              batch=SimpleNamespace(synchronize=lambda: None))
    monkeypatch.setattr(memory_ppo, "MemoryPPOTrainer", lambda *a, **k: trainer)
    monkeypatch.setattr(ops, "stalls", lambda device: 3)
    assert memory_ppo.train_memory_ppo(None, 4) == [1.0] * 4
    done.clear()
    monkeypatch.setattr(ops, "stalls", lambda device: 3 + (len(done) >= 2))
    with pytest.raises(RuntimeError, match="iteration 2"):
        memory_ppo.train_memory_ppo(None, 4)
    assert len(done) == 2


@pytest.mark.parametrize("envs,steps,batch,want", [(2048, 128, 8192, 8192), (2048, 100, 8192, 8100), (256, 32, 8192, 8192), (48, 5, 8192, 240),
                                                   (3, 100, 64, 100)])
def test_the_command_takes_any_number_of_steps(monkeypatch, envs, steps, batch, want):
    """Minibatches of whole sequences, as many as --batch holds."""
    from nesle_b200 import memory_ppo

    seen = []
    monkeypatch.setattr(memory_ppo, "train_memory_ppo", lambda config, iterations, device: seen.append(config))
    assert memory_ppo.main(["--envs", str(envs), "--steps", str(steps), "--batch", str(batch)]) == 0
    assert (seen[0].num_envs, seen[0].n_steps, seen[0].batch_size) == (envs, steps, want)


@pytest.mark.gpu
def test_muon_passes_over_matrices_without_elements(cuda):
    from nesle_b200.muon import Muon

    params = [torch.nn.Parameter(torch.randn(s, device="cuda")) for s in ((4, 0), (0, 4), (3, 5))]
    before = params[2].detach().clone()
    for p in params:
        p.grad = torch.randn_like(p)
    Muon(params).step()
    assert not torch.equal(params[2].detach(), before)
