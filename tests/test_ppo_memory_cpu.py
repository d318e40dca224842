"""PPO with a memory and with dropout (ur3e_amd/rl/ppo.py, policy="memory", dropout=p) on the CPU: the rollout's steps are
the update's sequences, the update meets the rollout's masks, a memory is cut where an episode starts, and
replicas stay identical across two gloo ranks."""
import os

import numpy as np
import pytest
import torch
import torch.multiprocessing as mp

from ur3e_amd.rl.ppo import PPO, MemoryNet

from test_ppo_cpu import ToyEnv, _free_port


def test_memory_steps_are_its_sequence():
    torch.manual_seed(0)
    net = MemoryNet(6, (32, 16), heads=4, dropout=0.3, seed=5)
    b, t = 3, 11
    obs = torch.randn(b, t, 6)
    starts = torch.rand(b, t) < 0.2
    rows = torch.arange(b * t).view(b, t) + 1000
    s0 = torch.randn(b, 4, 8, 8)
    with torch.no_grad():
        seq = net.sequence(obs, s0, starts, rows)
        s = s0.clone()
        for i in range(t):
            look = net.step(obs[:, i], s, starts[:, i], rows[:, i], update=False)
            h = net.step(obs[:, i], s, starts[:, i], rows[:, i])
            torch.testing.assert_close(h, look, rtol=0, atol=0)
            torch.testing.assert_close(h, seq[:, i], rtol=1e-5, atol=1e-5)
        assert not torch.allclose(seq, net.sequence(obs, s0, starts, rows + 1))  # other numbers, other masks
        # the state in front of a start does not matter
        starts[:, 0] = True
        assert torch.equal(net.sequence(obs, s0, starts), net.sequence(obs, torch.zeros_like(s0), starts))


@pytest.mark.parametrize("policy,dropout", [("memory", 0.0), ("memory", 0.2), ("mlp", 0.2)])
def test_update_meets_the_rollout(policy, dropout):
    """before the first update step the policy's log-probabilities and values are the rollout's: same memories, same
    masks, whatever transitions a minibatch gathers; over two iterations"""
    algo = PPO(ToyEnv(8), n_steps=6, batch_size=12, n_epochs=2, device="cpu", policy=policy, dropout=dropout)
    for _ in range(2):
        algo.collect_rollouts()
        seen = {}
        inner = algo._loss

        def look(idx):
            if not seen:
                if algo.memory:
                    seq = [x[:, idx].transpose(0, 1) for x in (algo.buf_obs, algo.buf_act, algo.buf_start)]
                    numbers = algo._update_numbers[:, idx].transpose(0, 1) if dropout else None
                    flat = (idx[:, None] + algo._starts_at).flatten()
                    v, logp, _ = algo.policy.evaluate(seq[0], seq[1], [s[idx] for s in algo._began], seq[2] > 0, numbers)
                else:
                    flat = idx
                    v, logp, _ = algo.policy.evaluate(algo._obs_all[idx], algo._act_all[idx],
                                                      algo._update_numbers.view(-1)[idx])
                seen["logp"] = (logp - algo.buf_logp.flatten()[flat]).abs().max().item()
                seen["v"] = (v - algo.buf_val.flatten()[flat]).abs().max().item()
            return inner(idx)
        algo._loss = look
        before = [p.detach().clone() for p in algo.policy.parameters()]
        algo.train()
        algo._loss = inner
        assert seen["logp"] < 1e-4 and seen["v"] < 1e-4, seen
        assert all(torch.isfinite(p).all() for p in algo.policy.parameters())
        assert sum(not torch.equal(b, p) for b, p in zip(before, algo.policy.parameters())) > len(before) // 2
    assert (algo.buf_start[1:] > 0).any()  # episodes started inside the rollouts
    assert int(algo._first) == 2 * 6 * 8


def test_default_policy_is_unchanged_by_the_options():
    a = PPO(ToyEnv(4), n_steps=4, batch_size=8, n_epochs=1, device="cpu")
    b = PPO(ToyEnv(4), n_steps=4, batch_size=8, n_epochs=1, device="cpu", policy="mlp", dropout=0.0)
    a.learn(1)
    b.learn(1)
    assert all(torch.equal(x, y) for x, y in zip(a.policy.parameters(), b.policy.parameters()))
    assert not hasattr(a, "_pi")


def test_memory_refuses():
    kw = dict(n_steps=4, batch_size=8, device="cpu")
    with pytest.raises(ValueError, match="policy must be"):
        PPO(ToyEnv(4), policy="lstm", **kw)
    with pytest.raises(ValueError, match="dropout"):
        PPO(ToyEnv(4), dropout=1.0, **kw)
    with pytest.raises(ValueError, match="multiple of"):
        PPO(ToyEnv(4), policy="memory", n_steps=5, batch_size=8, device="cpu")
    with pytest.raises(ValueError, match="two layers"):
        PPO(ToyEnv(4), policy="memory", net_arch=(30, 16), **kw)
    with pytest.raises(ValueError, match="two layers"):
        PPO(ToyEnv(4), policy="memory", net_arch=(64,), **kw)


def _rank(rank, world, port, out):
    import torch.distributed as dist
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    algo = PPO(ToyEnv(4, seed=rank), n_steps=4, batch_size=8, n_epochs=2, device="cpu", seed=rank,
               group=dist.group.WORLD, policy="memory", dropout=0.1, net_arch=(32, 32))
    algo.learn(1)
    np.save(f"{out}.{rank}.npy", torch.cat([p.detach().reshape(-1) for p in algo.policy.parameters()]).numpy())
    dist.destroy_process_group()


def test_memory_replicas_stay_identical_gloo(tmp_path):
    out = str(tmp_path / "p")
    mp.spawn(_rank, args=(2, _free_port(), out), nprocs=2, join=True)
    np.testing.assert_array_equal(np.load(out + ".0.npy"), np.load(out + ".1.npy"))
