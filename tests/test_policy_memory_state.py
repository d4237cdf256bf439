"""When a policy's memory is kept and when it is cleared: the player's calls, checkpoints.  CPU."""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import _stub_env
from airgym_amd.lib.agent.a2c_continuous import A2CAgent
from airgym_amd.lib.agent.players import A2CPlayer

_stub_env.register()


def params(**kw):
    p = _stub_env.ppo_params(**kw)
    p["network"]["memory"] = {"units": 24, "states": 5, "taps": 3}
    p["config"]["player"] = {"games_num": 10 ** 6, "max_steps": 9, "print_stats": False}
    return p


def test_player_s_plain_call_remembers():
    """get_action(obs), step after step, is the sequence; `dones` forgets the envs it names and no others."""
    torch.manual_seed(0)
    player = A2CPlayer(params(num_actors=6))
    m, n = player.model, 6
    obs = torch.randn(7, n, player.obs_shape[0])
    resets = torch.zeros(n, 7, dtype=torch.bool)
    resets[2, 4] = resets[5, 4] = True
    got = []
    for t in range(7):
        got.append(player.get_action(obs[t], dones=resets[:, t]) if t == 4 else player.get_action(obs[t]))
    with torch.no_grad():
        flat = obs.transpose(0, 1).reshape(7 * n, -1)
        mu, _, _ = m.trunk(flat, memory={"state": m.memory.initial_state(n), "resets": resets})
    want = torch.clamp(mu, -1.0, 1.0).view(n, 7, -1)
    # one float32 computation in two orders: 24 channels, 32 units, 7 steps
    for t in range(7):
        assert torch.allclose(got[t], want[:, t], rtol=0, atol=1e-5), t
    alone = A2CPlayer(params(num_actors=6))
    alone.model.load_state_dict(m.state_dict())
    assert not torch.allclose(alone.get_action(obs[6]), got[6], rtol=0, atol=1e-4)


def test_player_s_run_starts_without_a_memory_of_the_run_before():
    torch.manual_seed(0)
    p = params(num_actors=6)
    player = A2CPlayer(p)
    seen = []
    first = player.get_action

    def spy(obs, is_deterministic=True, dones=None):
        seen.append((obs.clone(), first(obs, is_deterministic, dones)))
        return seen[-1][1]

    player.get_action = spy
    player.run()
    assert player.memory_state[1].abs().max() > 0
    player.run()
    assert len(seen) == 18
    fresh = A2CPlayer(p)
    fresh.model.load_state_dict(player.model.state_dict())
    obs, action = seen[9]                   # the second run's first step
    assert torch.allclose(fresh.get_action(obs), action, rtol=0, atol=1e-6)


def _trained(tmp_path, **kw):
    torch.manual_seed(1)
    agent = A2CAgent("run", params(num_actors=16, horizon=8, **kw))
    agent.init_tensors()
    agent.obs = agent.env_reset()
    agent.play_steps()
    fn = str(tmp_path / "ck")
    agent.save(fn)
    return agent, fn if os.path.exists(fn) else fn + ".pth"


def test_a_restore_into_a_live_agent_does_not_keep_another_policy_s_memory(tmp_path):
    """The envs go on with their own episodes; what was remembered of them came from the weights that are gone."""
    _, fn = _trained(tmp_path)
    live = A2CAgent("run", params(num_actors=16, horizon=8))
    live.init_tensors()
    live.obs = live.env_reset()
    live.play_steps()
    places = [t.data_ptr() for t in live.memory_state]
    assert live.memory_state[1].abs().max() > 0
    live.restore(fn)
    assert not any(t.any() for t in live.memory_state)
    assert [t.data_ptr() for t in live.memory_state] == places          # captured rollouts read them there
    player = A2CPlayer(params(num_actors=16))
    player.get_action(torch.randn(16, player.obs_shape[0]))
    player.restore(fn)
    assert not any(t.any() for t in player.memory_state)


def test_training_moves_every_parameter_of_the_memory():
    torch.manual_seed(2)
    agent = A2CAgent("run", params(num_actors=16, horizon=8, mini_epochs=2, max_epochs=2))
    before = {k: v.detach().clone() for k, v in agent.model.named_parameters() if k.startswith("memory.")}
    assert len(before) == 9
    agent.train()
    for k, v in agent.model.named_parameters():
        if k in before:
            assert torch.isfinite(v).all() and not torch.equal(v, before[k]), k


def test_update_sees_a_rollout_whose_episodes_end_inside(monkeypatch):
    """The env reports ends in the middle of the horizon; the update's sequences still give the rollout's own action means, and would not
    without the flags."""
    from airgym_amd.lib.network.ssm import RolloutMemory
    torch.manual_seed(3)
    step, calls = _stub_env.OracleVecEnv.step, [0]

    def ends(self, actions):
        obs, rew, done, info = step(self, actions)
        calls[0] += 1
        done = done.clone()
        done[calls[0] % 8::8] = 1
        return obs, rew, done, info

    monkeypatch.setattr(_stub_env.OracleVecEnv, "step", ends)
    agent = A2CAgent("run", params(num_actors=16, horizon=8))
    agent.init_tensors()
    agent.obs = agent.env_reset()
    agent.model.update_stats = False
    n = agent.batch_size
    for _ in range(3):
        batch = agent.play_steps()
        memory = RolloutMemory(agent.memory_start, batch["dones"], agent.horizon_length)
        assert int(memory.resets[:, 1:].any(1).sum()) == 14          # of 16: two end with the horizon's last step
        with torch.no_grad():
            for first, last in ((0, n), (n // 2, n)):
                mu, _, _ = agent.model.trunk(batch["obses"][first:last], memory=memory[first:last])
                assert torch.allclose(mu, batch["mus"][first:last], rtol=0, atol=1e-5)
            memory.resets = torch.zeros_like(memory.resets)
            mu, _, _ = agent.model.trunk(batch["obses"], memory=memory[0:n])
            assert not torch.allclose(mu, batch["mus"], rtol=0, atol=1e-4)


def test_paths_on_the_cpu_name_no_kernels():
    agent = A2CAgent("run", params(num_actors=8, horizon=4))
    agent.init_tensors()
    paths = agent.compute_paths()
    assert "memory: torch" in paths["rollout_step"] and "memory: torch" in paths["update"]
    assert not any("ag_" in v for v in (paths["rollout_step"], paths["update"], paths["optimizer"]))
