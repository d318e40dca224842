"""GPU: PPO with a memory and dropout (ur3e_amd/rl/ppo.py) on the batched env through the HIP operators: the captured
update lands where the eager one does, and the update meets the rollout's memories and masks."""
import pytest

pytestmark = pytest.mark.gpu


def _algo(policy, dropout, graphs, n=64, n_steps=4, batch_size=32):
    from ur3e_amd.envs.vec_env import UR3eVecEnv
    from ur3e_amd.envs.vec_normalize import VecNormalize
    from ur3e_amd.rl.ppo import PPO
    venv = UR3eVecEnv(num_envs=n, device=0, seed=0, max_episode_steps=3)
    env = VecNormalize(venv, norm_obs=True, norm_reward=False, clip_obs=10.0)
    return venv, PPO(env, n_steps=n_steps, batch_size=batch_size, n_epochs=2, device="cuda:0", seed=0, graphs=graphs,
                     policy=policy, dropout=dropout)


@pytest.mark.parametrize("policy,dropout", [("memory", 0.0), ("memory", 0.1), ("mlp", 0.1)])
def test_graph_update_matches_eager(policy, dropout):
    """The captured minibatch, replayed after a second rollout with eager work in between, gives the gradients of the
    eager one.  (The parameters themselves are no measure: Adam divides a gradient by its own size, so one that is
    rounding alone moves its parameter by up to the learning rate, 3e-4, in either direction.)"""
    import torch
    venv, algo = _algo(policy, dropout, graphs=True)
    algo.learn(1)
    assert algo._graphs is not None
    algo.collect_rollouts()
    # what train() lays out before its minibatches
    total = algo.n_steps * algo.n_envs
    algo._adv_s.copy_(algo.adv.reshape(-1))
    algo._ret_s.copy_(algo.ret.reshape(-1))
    torch.add(algo._numbers[:algo.n_steps], algo._first - total, out=algo._update_numbers)
    g = torch.Generator().manual_seed(0)
    for r in range(4):
        idx = torch.randperm(algo.n_envs if algo.memory else total, generator=g)[:algo._g_idx.numel()].cuda()
        algo._g_idx.copy_(idx)
        algo._graphs[0].replay()
        torch.cuda.synchronize()
        replayed = algo._flat_grad.clone()
        algo._backward(idx)
        eager = algo._flat_grad.clone()
        # at most 512 terms a sum, in whatever order
        assert (replayed - eager).abs().max() <= 512 * 2.0 ** -24 * eager.abs().max(), r
        assert torch.isfinite(eager).all() and eager.abs().max() > 0
    venv.close()


@pytest.mark.parametrize("policy,dropout", [("memory", 0.2), ("mlp", 0.2)])
def test_update_meets_the_rollout(policy, dropout):
    import torch
    venv, algo = _algo(policy, dropout, graphs=False, n=96, n_steps=16, batch_size=64)
    algo.collect_rollouts()
    assert (algo.buf_start[1:] > 0).any()
    numbers = algo._numbers[:16]
    with torch.no_grad():
        if algo.memory:
            seq = [x.transpose(0, 1) for x in (algo.buf_obs, algo.buf_act, algo.buf_start)]
            v, logp, _ = algo.policy.evaluate(seq[0], seq[1], algo._began, seq[2] > 0, numbers.transpose(0, 1))
            want = [x.transpose(0, 1).flatten() for x in (algo.buf_val, algo.buf_logp)]
        else:
            v, logp, _ = algo.policy.evaluate(algo.buf_obs.flatten(0, 1), algo.buf_act.flatten(0, 1), numbers.flatten())
            want = [algo.buf_val.flatten(), algo.buf_logp.flatten()]
    venv.close()
    # float products of 256 terms in another order, values of order 1 and log-probabilities of order 10
    assert (v - want[0]).abs().max().item() < 1e-3
    assert (logp - want[1]).abs().max().item() < 1e-3
