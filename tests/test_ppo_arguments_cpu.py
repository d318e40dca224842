"""PPO's arguments for a memory and for dropout (ur3e_amd/rl/ppo.py) on the CPU."""
import numpy as np
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
@pytest.mark.parametrize("seed,same", [(np.int64(5), 5), (-1, -1), ((1 << 64) - 1, (1 << 64) - 1)])
def test_dropout_takes_the_seeds_that_ppo_takes(policy, seed, same):
    """numpy's integers, negative ones and those past 63 bits, as torch.manual_seed takes them"""
    both = [PPO(ToyEnv(4), policy=policy, dropout=0.2, net_arch=(32, 32), seed=s, **KW) for s in (seed, same)]
    for algo in both:
        algo.collect_rollouts()
    assert torch.equal(both[0].buf_val, both[1].buf_val)
