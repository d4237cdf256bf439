"""A policy with a memory on the GPU: the step kernels of the rollout against the sequence kernels of the update, the captured rollout,
training, and the layer against its torch forms."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.gpu


def make(num_actors=256, horizon=24, units=64, **cfg):
    import _stub_env
    from airgym_amd.lib.agent.a2c_continuous import A2CAgent
    from airgym_amd.lib.utils import env_configurations  # noqa: F401
    import airgym_amd.envs  # noqa: F401
    p = _stub_env.ppo_params(num_actors=num_actors, horizon=horizon, units=(64, 64), env_name="hovering", device="cuda:0",
                             minibatch=num_actors * horizon // 2, **cfg)
    p["config"]["env_config"] = {"use_image": False, "ctl_mode": "rate", "seed": 3, "stagger_episode_phase": True}
    p["network"]["memory"] = {"units": units, "states": 16, "taps": 4}
    torch.manual_seed(0)
    return A2CAgent("run", p)


def test_layer_against_its_torch_forms():
    from airgym_amd.lib.network.ssm import SelectiveMemory
    torch.manual_seed(1)
    m = SelectiveMemory(18, units=48, states=16, taps=4)
    x, resets, dy = torch.randn(6, 24, 18), torch.rand(6, 24) < 0.1, torch.randn(6, 24, 18)
    out = m(x, None, resets)
    want = torch.autograd.grad(out, list(m.parameters()), dy)
    g = SelectiveMemory(18, units=48, states=16, taps=4).cuda()
    g.load_state_dict(m.state_dict())
    got_out = g(x.cuda(), None, resets.cuda())
    got = torch.autograd.grad(got_out, list(g.parameters()), dy.cuda())
    # both sides float32, every product a sum of at most 144 rows of terms of order one and 24 steps in a row; 2^-24 x 24 x 64
    assert torch.allclose(got_out.cpu(), out, rtol=0, atol=2.0 ** -24 * 24 * 64 * float(out.abs().max()))
    for (k, _), a, b in zip(m.named_parameters(), got, want):
        assert float((a.cpu() - b).abs().max()) <= 2.0 ** -24 * 144 * 64 * float(b.abs().max()), k


@pytest.mark.parametrize("graph", [False, True])
def test_update_sees_the_rollout(graph):
    """Eager and (from the second rollout on) replayed: the update's sequences give the rollout's own action means."""
    from airgym_amd.lib.network.ssm import RolloutMemory
    agent = make(use_hip_graph=graph)
    agent.init_tensors()
    agent.obs = agent.env_reset()
    agent.model.update_stats = False
    ended = 0
    for _ in range(4):
        batch = agent.play_steps()
        memory = RolloutMemory(agent.memory_start, batch["dones"], agent.horizon_length)
        ended += int(memory.resets[:, 1:].sum())
        n = agent.batch_size
        with torch.no_grad():
            for first, last in ((0, n), (n // 2, n)):
                mu, _, _ = agent.model.trunk(batch["obses"][first:last], memory=memory[first:last])
                # the same float32 sums in another order: about 2 x 64 roundings along a layer, five layers, 24 steps
                assert float((mu - batch["mus"][first:last]).abs().max()) <= 2.0 ** -24 * 128 * 5 * 24
    assert ended > 0                    # some episodes ended inside a rollout
    assert ("rollout" in agent._graphs) == graph


def test_training_runs_and_paths_are_named():
    agent = make(max_epochs=3, use_hip_graph=True)
    agent.train()
    assert torch.isfinite(agent.flat_param).all()
    paths = agent.compute_paths()
    assert "ag_selective_scan_step" in paths["rollout_step"] and "ag_selective_scan_fwd" in paths["update"]
    for k, p in agent.model.named_parameters():
        if k.startswith("memory."):
            assert torch.isfinite(p.grad).all() and p.grad.abs().max() > 0, k
