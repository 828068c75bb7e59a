"""LinearRecurrentPolicy: acting, replaying and training on the sequence
operators, through the learners, the trainer and the command line."""
import dataclasses
import json

import pytest
import torch

from rlgpuschedule_amd.agents.ppo import (A2CConfig, A2CLearner, PPOConfig,
                                          PPOLearner, replay_sequence)
from rlgpuschedule_amd.agents.rollout import (Collector, RolloutBuffer,
                                              TorchEnvAdapter)
from rlgpuschedule_amd.cli import main as cli_main
from rlgpuschedule_amd.env.gym_api import CpuVectorEnv
from rlgpuschedule_amd.env.spec import cluster16
from rlgpuschedule_amd.models.policy import (LinearRecurrentPolicy,
                                             evaluate_actions)
from rlgpuschedule_amd.trainer import CONFIGS, train

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def buffer(T, E, D, A, hidden, device, seed=0):
    """A rollout buffer of random steps with some episode ends."""
    g = torch.Generator().manual_seed(seed)
    buf = RolloutBuffer(T, E, D, A, device, hidden)
    buf.obs.copy_(torch.randn(T, E, D, generator=g))
    mask = torch.rand(T, E, A, generator=g) < 0.6
    act = torch.randint(0, A, (T, E), generator=g)
    mask.scatter_(-1, act.unsqueeze(-1), True)
    buf.mask.copy_(mask)
    buf.actions.copy_(act)
    buf.logp.copy_(-torch.rand(T, E, generator=g) * 2)
    buf.value.copy_(torch.randn(T, E, generator=g))
    buf.reward.copy_(torch.randn(T, E, generator=g))
    buf.done.copy_(torch.rand(T, E, generator=g) < 0.1)
    buf.last_value.copy_(torch.randn(E, generator=g))
    buf.h0.copy_(torch.randn(E, hidden, generator=g))
    return buf


def make(D, A, hidden, device, seed=0):
    torch.manual_seed(seed)
    return LinearRecurrentPolicy(D, A, hidden).to(device)


@pytest.mark.parametrize("device", DEVICES)
def test_steps_are_the_sequence(device):
    """forward, step and forward_sequence agree, across episode ends. Sizes
    are small: 32-bit products of up to 24 terms, so 1e-5 of values of
    order 1 is over a hundred roundings."""
    T, E, D, A, H = 40, 5, 9, 6, 24
    buf = buffer(T, E, D, A, H, device)
    pol = make(D, A, H, device)
    with torch.no_grad():
        logits, value, carry = pol.forward_sequence(buf.obs, buf.h0, buf.done)
        hx, hs, prev = buf.h0.clone(), buf.h0.clone(), None
        for t in range(T):
            lg, v, hx = pol(buf.obs[t], None, hx)
            torch.testing.assert_close(lg, logits[t], rtol=1e-5, atol=1e-5)
            torch.testing.assert_close(v, value[t], rtol=1e-5, atol=1e-5)
            hx = hx * (1.0 - buf.done[t].float()).unsqueeze(-1)
            lg2, v2 = pol.step(buf.obs[t], buf.mask[t], hs, prev)
            prev = buf.done[t]
            ok = buf.mask[t].bool()
            torch.testing.assert_close(lg2[ok], logits[t][ok], rtol=1e-5,
                                       atol=1e-5)
            assert (lg2[~ok] < -1e8).all()
        torch.testing.assert_close(hx, carry, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("device", DEVICES)
def test_replay_is_the_stepwise_replay(device):
    """replay_sequence's one scan gives the step-by-step replay's values and
    gradients."""
    T, E, D, A, H = 24, 4, 7, 5, 16
    buf = buffer(T, E, D, A, H, device, 1)
    pol = make(D, A, H, device, 1)
    w = [torch.randn(T, E, device=device) for _ in range(3)]
    params = list(pol.parameters())

    def loss_of(logp, ent, value):
        return (logp * w[0]).sum() + (ent * w[1]).sum() + (value * w[2]).sum()

    got = replay_sequence(pol, buf.obs, buf.mask, buf.actions, buf.h0,
                          buf.done)
    grads = torch.autograd.grad(loss_of(*got), params)
    hx, outs = buf.h0, []
    for t in range(T):
        logits, value, hx = pol(buf.obs[t], buf.mask[t], hx)
        outs.append((*evaluate_actions(logits, buf.actions[t]), value))
        hx = hx * (1.0 - buf.done[t].float()).unsqueeze(-1)
    want = [torch.stack(q) for q in zip(*outs)]
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-5)
    for a, b in zip(grads, torch.autograd.grad(loss_of(*want), params)):
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("algo", ["ppo", "a2c"])
def test_learners_update(device, algo):
    buf = buffer(16, 8, 9, 6, 32, device, 2)
    pol = make(9, 6, 32, device, 2)
    before = [p.detach().clone() for p in pol.parameters()]
    learner = (PPOLearner(pol, PPOConfig(epochs=2, minibatches=2))
               if algo == "ppo" else A2CLearner(pol, A2CConfig()))
    stats = learner.update(buf)
    assert all(torch.isfinite(torch.tensor(v)) for v in stats.values())
    for p, q in zip(pol.parameters(), before):
        assert torch.isfinite(p).all() and not torch.equal(p, q)


def test_collector_replays_what_it_acted():
    """The behaviour log probabilities and values of a rollout, and of the
    one after it, are those of the replay from its stored state."""
    spec = cluster16(horizon=12)     # episodes end within a rollout
    env = TorchEnvAdapter(CpuVectorEnv(spec, 3, trace_kind="philly",
                                       jobs_per_env=8, seed=3))
    pol = make(spec.obs_dim, spec.num_actions, 16, "cpu", 3)
    col = Collector(env, pol, 20, "cpu", seed=1)
    for _ in range(3):
        buf = col.collect()
        with torch.no_grad():
            logp, _, value = replay_sequence(pol, buf.obs, buf.mask,
                                             buf.actions, buf.h0, buf.done)
        torch.testing.assert_close(logp, buf.logp, rtol=1e-4, atol=1e-4)
        torch.testing.assert_close(value, buf.value, rtol=1e-4, atol=1e-4)
    assert buf.done.any()


def test_trainer_saves_and_resumes(tmp_path):
    cfg = dataclasses.replace(
        CONFIGS["c3_ppo_gru"], policy="linrec", spec=cluster16(), num_envs=4,
        jobs_per_env=8, rollout_T=8, use_hip_env=False, device="cpu",
        hidden=16)
    train(cfg, iterations=2, log_fn=None, out_dir=str(tmp_path), save_every=2)
    out = train(cfg, iterations=1, log_fn=None,
                resume=str(tmp_path / "policy_000002.pt"))
    assert isinstance(out["_policy"], LinearRecurrentPolicy)
    with pytest.raises(ValueError, match="linrec"):
        train(dataclasses.replace(cfg, algo="impala"), iterations=1)


def test_command_line(tmp_path, capsys):
    assert cli_main(["train", "--config", "c1_cpu_random", "--policy",
                     "linrec", "--iterations", "1", "--envs", "2",
                     "--jobs-per-env", "8"]) == 0
    from rlgpuschedule_amd.ckpt.io import save_policy
    cfg = CONFIGS["c1_cpu_random"]
    pol = LinearRecurrentPolicy(cfg.spec.obs_dim, cfg.spec.num_actions,
                                cfg.hidden)
    save_policy(tmp_path / "p.safetensors", pol, spec=cfg.spec)
    assert cli_main(["eval", "--config", "c1_cpu_random", "--policy", "linrec",
                     "--ckpt", str(tmp_path / "p.safetensors"), "--envs", "2",
                     "--episodes", "2", "--jobs-per-env", "10"]) == 0
    out = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    assert out["episodes"] >= 2


@pytest.mark.gpu
@pytest.mark.parametrize("algo", ["ppo", "a2c"])
def test_trainer_on_the_gpu_env(algo):
    cfg = dataclasses.replace(
        CONFIGS["c2_ppo_mlp"], policy="linrec", algo=algo, num_envs=64,
        jobs_per_env=16, rollout_T=16, hidden=64)
    out = train(cfg, iterations=3, log_fn=None)
    assert isinstance(out["_policy"], LinearRecurrentPolicy)
    assert out["_policy"].v.weight.is_cuda
    for p in out["_policy"].parameters():
        assert torch.isfinite(p).all()
