"""PPO's arguments for a memory and for dropout (ur3e_amd/rl/ppo.py) on the CPU."""
import pytest
import torch

from ur3e_amd.rl.ppo import PPO

from test_ppo_cpu import ToyEnv

KW = dict(n_steps=4, batch_size=8, n_epochs=1, device="cpu")


@pytest.mark.parametrize("heads", [0, -4])
def test_heads_are_refused(heads):
    with pytest.raises(ValueError, match="heads"):
        PPO(ToyEnv(4), policy="memory", heads=heads, **KW)


@pytest.mark.parametrize("policy", ["mlp", "memory"])
@pytest.mark.parametrize("seed", [-1, (1 << 64) - 1])
def test_dropout_takes_the_seeds_that_ppo_takes(policy, seed):
    """negative ones and those past 63 bits, as torch takes them, and the same masks twice"""
    both = [PPO(ToyEnv(4), policy=policy, dropout=0.2, net_arch=(32, 32), seed=seed, **KW) for _ in range(2)]
    for algo in both:
        algo.collect_rollouts()
    assert torch.equal(both[0].buf_val, both[1].buf_val)
