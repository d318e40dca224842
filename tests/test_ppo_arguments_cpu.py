"""PPO's arguments for a memory and for dropout (ur3e_amd/rl/ppo.py) on the CPU."""
import pytest

from ur3e_amd.rl.ppo import PPO

from test_ppo_cpu import ToyEnv

KW = dict(n_steps=4, batch_size=8, n_epochs=1, device="cpu")


@pytest.mark.parametrize("heads", [0, -4])
def test_heads_are_refused(heads):
    with pytest.raises(ValueError, match="heads"):
        PPO(ToyEnv(4), policy="memory", heads=heads, **KW)
