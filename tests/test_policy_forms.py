"""Linear recurrent policies beside policies of a user's own."""
import torch

from rlgpuschedule_amd.agents.ppo import (PPOConfig, PPOLearner,
                                          replay_sequence)
from rlgpuschedule_amd.agents.rollout import Collector, TorchEnvAdapter
from rlgpuschedule_amd.env.gym_api import CpuVectorEnv
from rlgpuschedule_amd.env.spec import cluster16


# --------------------------------------------------- policies of a user's own
class NamesakePolicy(torch.nn.Module):
    """A recurrent policy with methods of its own that happen to be called
    step and forward_sequence."""

    is_recurrent = True

    def __init__(self, obs_dim, num_actions, hidden=8):
        super().__init__()
        self.hidden = hidden
        self.cell = torch.nn.GRUCell(obs_dim, hidden)
        self.pi = torch.nn.Linear(hidden, num_actions)
        self.calls = []

    def step(self):
        self.calls.append("step")

    def forward_sequence(self, text):
        self.calls.append("forward_sequence")

    def forward(self, obs, mask=None, hx=None):
        hx = self.cell(obs, hx)
        logits = self.pi(hx)
        if mask is not None:
            logits = logits.masked_fill(mask == 0, -1e9)
        return logits, hx.sum(-1), hx

    def initial_state(self, batch, device):
        return torch.zeros(batch, self.hidden, device=device)


def test_methods_of_the_same_names_are_not_called():
    spec = cluster16(horizon=12)
    env = TorchEnvAdapter(CpuVectorEnv(spec, 3, trace_kind="philly",
                                       jobs_per_env=8, seed=3))
    torch.manual_seed(0)
    pol = NamesakePolicy(spec.obs_dim, spec.num_actions)
    col = Collector(env, pol, 20, "cpu", seed=1)
    for _ in range(2):
        buf = col.collect()
        with torch.no_grad():
            logp, _, value = replay_sequence(pol, buf.obs, buf.mask,
                                             buf.actions, buf.h0, buf.done)
        torch.testing.assert_close(logp, buf.logp, rtol=1e-4, atol=1e-4)
        torch.testing.assert_close(value, buf.value, rtol=1e-4, atol=1e-4)
    PPOLearner(pol, PPOConfig(epochs=1, minibatches=1)).update(buf)
    assert pol.calls == []
