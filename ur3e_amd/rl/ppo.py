"""Device-resident PPO driving the batched env.

Replaces `stable_baselines3.PPO("MlpPolicy", VecNormalize(venv), ...)` as configured in
gymnasium_src/scripts/regular_rl/rl/train_rl.py:60-73 with gymnasium_src/config/config_rl.yml
(net_arch [256, 256], lr 3e-4, batch 256, n_epochs 30, gamma 0.99, gae_lambda 0.95, ent_coef 0.01;
SB3 defaults for the rest: clip_range 0.2, vf_coef 0.5, max_grad_norm 0.5, Adam eps 1e-5,
normalize_advantage, state-independent log_std initialised to 0, tanh MLPs with orthogonal init).
No feature extractor: train_rl.py:123 reads `hyperparameters.get("feature_encoder")` while the
yml key is `feature_extractor`, so the reference's transformer / frame-stack branch (:26-35) is
never taken and the policy is the plain MLP above.  SB3 itself is not installed in this image; the algorithm follows stable_baselines3==2.x
(`PPO.train`, `OnPolicyAlgorithm.collect_rollouts`, `RolloutBuffer.compute_returns_and_advantage`).

MI355X layout: the env, the on-device VecNormalize, the rollout buffer and the policy all live on
one GPU and share torch's current stream, so a rollout step is env kernel -> normalisation kernel ->
policy forward with no host round trip.  With several ranks (one process per GPU) each rank steps its
own env shard and keeps a policy replica; gradients are flattened into ONE buffer and all-reduced
(averaged) per minibatch, a single RCCL call over xGMI instead of one per parameter tensor.

Beyond the reference's MLP (`policy="mlp"`, the default) there is a policy that remembers (`policy="memory"`: attention
with a decaying state, ur3e_amd/rl/ops.py, in the place of the reference's sequence feature extractor over
stacked frames, train_rl.py:26-35), and dropout (`dropout=p`) for either.  The memory is carried from step to step of a
rollout, cut where an episode starts, and the update runs over whole rollouts of a few envs from the states their
rollouts began with.  A dropped unit is a function of the transition's number, so every epoch of the update
drops what the rollout dropped and the probability ratio measures the policy's change alone.

The env object only needs `num_envs`, `action_space` (low/high), `reset_torch()` and
`step_torch(actions) -> (obs f32, reward, terminated, truncated, terminal_obs f32)`: the GPU
`VecNormalize` provides it, and tests use a CPU stand-in with the same interface.
"""
from __future__ import annotations

import math
import time

import torch
import torch.nn as nn

from . import ops


def _mlp(sizes, gain):
    layers = []
    for i in range(len(sizes) - 1):
        lin = nn.Linear(sizes[i], sizes[i + 1])
        nn.init.orthogonal_(lin.weight, gain=gain)
        nn.init.zeros_(lin.bias)
        layers += [lin, nn.Tanh()]
    return nn.Sequential(*layers)


class ActorCritic(nn.Module):
    """SB3 ActorCriticPolicy for a Box action space with net_arch=[256, 256]: separate pi / vf MLPs
    over the flattened observation, Gaussian head with a state-independent log_std.  `rows` (transition numbers)
    turn dropout on: hidden units of a transition are dropped by its number (ops.keyed_dropout)."""

    def __init__(self, obs_dim: int, act_dim: int, net_arch=(256, 256), log_std_init: float = 0.0,
                 dropout: float = 0.0, seed: int = 0):
        super().__init__()
        self.dropout, self.seed = dropout, seed
        self.pi_net = _mlp([obs_dim, *net_arch], gain=math.sqrt(2))
        self.vf_net = _mlp([obs_dim, *net_arch], gain=math.sqrt(2))
        self.action_net = nn.Linear(net_arch[-1], act_dim)
        self.value_net = nn.Linear(net_arch[-1], 1)
        nn.init.orthogonal_(self.action_net.weight, gain=0.01)
        nn.init.zeros_(self.action_net.bias)
        nn.init.orthogonal_(self.value_net.weight, gain=1.0)
        nn.init.zeros_(self.value_net.bias)
        self.log_std = nn.Parameter(torch.full((act_dim,), float(log_std_init)))

    def _hidden(self, net, obs, rows, substream):
        if rows is None or not self.dropout:
            return net(obs)
        for i, layer in enumerate(net):
            obs = layer(obs)
            if isinstance(layer, nn.Tanh):
                obs = ops.keyed_dropout(obs, self.dropout, self.seed, rows, substream + i)
        return obs

    def mean(self, obs, rows=None):
        return self.action_net(self._hidden(self.pi_net, obs, rows, PI_STREAM))

    def normal(self, mean):
        # validate_args=False: the argument checks synchronise with the host every rollout step
        return torch.distributions.Normal(mean, self.log_std.exp().expand_as(mean), validate_args=False)

    def dist(self, obs, rows=None):
        return self.normal(self.mean(obs, rows))

    def value(self, obs, rows=None):
        return self.value_net(self._hidden(self.vf_net, obs, rows, VF_STREAM)).squeeze(-1)

    def evaluate(self, obs, actions, rows=None):
        d = self.dist(obs, rows)
        return self.value(obs, rows), d.log_prob(actions).sum(-1), d.entropy().sum(-1)


# substreams of the dropout masks: one for each place of a network
PI_STREAM, VF_STREAM = 0, 1 << 16


class MemoryNet(nn.Module):
    """A trunk that remembers: tanh encoder, attention with a decaying state (`heads` heads of width / heads
    channels, each normalised to unit mean square), projected and added to the encoder's output, tanh layer.
    `sequence` runs over [B, T, obs] from a state, `step` one token of N envs."""

    def __init__(self, obs_dim: int, net_arch=(256, 256), heads: int = 4, dropout: float = 0.0, seed: int = 0,
                 substream: int = 0):
        super().__init__()
        width = net_arch[0]
        if heads < 1:
            raise ValueError(f"heads must be at least 1, got {heads}")
        if len(net_arch) != 2 or width % heads or width // heads > ops.MAX_DIM:
            raise ValueError(f"a memory needs two layers, the first of {heads} heads of at most {ops.MAX_DIM} "
                             f"channels: net_arch={tuple(net_arch)}")
        self.heads, self.dim = heads, width // heads
        self.dropout, self.seed, self.substream = dropout, seed, substream
        gain = math.sqrt(2)
        self.encoder = _mlp([obs_dim, width], gain)
        self.qkv = nn.Linear(width, 3 * width, bias=False)
        self.out = nn.Linear(width, width, bias=False)
        self.tail = _mlp([width, net_arch[1]], gain)
        nn.init.orthogonal_(self.qkv.weight)
        nn.init.orthogonal_(self.out.weight)
        # the heads forget over 4 to 256 steps
        over = torch.linspace(2.0, 8.0, heads) if heads > 1 else torch.tensor([5.0])
        self.register_buffer("log_decay", torch.log1p(-torch.exp2(-over)))

    def state(self, n: int, device):
        """n empty memories"""
        return torch.zeros((n, self.heads, self.dim, self.dim), dtype=torch.float32, device=device)

    def _qkv(self, e):
        return self.qkv(e).unflatten(-1, (3, self.heads, self.dim)).unbind(-3)

    def _merge(self, e, y, rows):
        y = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + 1e-6)
        y = self.out(y.flatten(-2))
        if rows is None or not self.dropout:
            h = e + y
        else:
            h = ops.keyed_dropout(y, self.dropout, self.seed, rows, self.substream, residual=e)
        return self.tail(h)

    def sequence(self, obs, state, starts, rows=None):
        e = self.encoder(obs)
        y, _ = ops.decay_attention(*self._qkv(e), self.log_decay, initial_state=state, starts=starts)
        return self._merge(e, y, rows)

    def step(self, obs, state, starts=None, rows=None, next_state=None, update=True):
        e = self.encoder(obs)
        y = ops.decay_attention_step(*self._qkv(e), self.log_decay, state, starts=starts, next_state=next_state,
                                     update=update)
        return self._merge(e, y, rows)


class MemoryActorCritic(nn.Module):
    """ActorCritic with a memory in each trunk"""

    def __init__(self, obs_dim: int, act_dim: int, net_arch=(256, 256), log_std_init: float = 0.0,
                 dropout: float = 0.0, seed: int = 0, heads: int = 4):
        super().__init__()
        self.pi_net = MemoryNet(obs_dim, net_arch, heads, dropout, seed, PI_STREAM)
        self.vf_net = MemoryNet(obs_dim, net_arch, heads, dropout, seed, VF_STREAM)
        self.action_net = nn.Linear(net_arch[-1], act_dim)
        self.value_net = nn.Linear(net_arch[-1], 1)
        nn.init.orthogonal_(self.action_net.weight, gain=0.01)
        nn.init.zeros_(self.action_net.bias)
        nn.init.orthogonal_(self.value_net.weight, gain=1.0)
        nn.init.zeros_(self.value_net.bias)
        self.log_std = nn.Parameter(torch.full((act_dim,), float(log_std_init)))

    normal = ActorCritic.normal

    def evaluate(self, obs, actions, states, starts, rows=None):
        """obs [B, T, .], actions [B, T, .], states = (pi, vf) in front of the first token, starts [B, T]; every result
        flattened to B * T"""
        d = self.normal(self.action_net(self.pi_net.sequence(obs, states[0], starts, rows)).flatten(0, 1))
        v = self.value_net(self.vf_net.sequence(obs, states[1], starts, rows)).flatten()
        return v, d.log_prob(actions.flatten(0, 1)).sum(-1), d.entropy().sum(-1)


def compute_gae(rewards, values, episode_starts, last_values, dones, gamma, lam):
    """RolloutBuffer.compute_returns_and_advantage: rewards/values/episode_starts [T, N];
    `dones` are the done flags after the last step. Returns (advantages, returns)."""
    T = rewards.shape[0]
    adv = torch.zeros_like(rewards)
    last = torch.zeros_like(last_values)
    for t in reversed(range(T)):
        if t == T - 1:
            nonterm = 1.0 - dones.to(rewards.dtype)
            nv = last_values
        else:
            nonterm = 1.0 - episode_starts[t + 1]
            nv = values[t + 1]
        delta = rewards[t] + gamma * nv * nonterm - values[t]
        last = delta + gamma * lam * nonterm * last
        adv[t] = last
    return adv, adv + values


class PPO:
    def __init__(self, env, n_steps: int = 16, batch_size: int = 256, n_epochs: int = 30, learning_rate: float = 3e-4,
                 gamma: float = 0.99, gae_lambda: float = 0.95, clip_range: float = 0.2, ent_coef: float = 0.01,
                 vf_coef: float = 0.5, max_grad_norm: float = 0.5, net_arch=(256, 256), device=None, seed: int = 0,
                 group=None, graphs=None, policy: str = "mlp", dropout: float = 0.0, heads: int = 4):
        """policy: "mlp" or "memory"; dropout: probability of dropping a hidden unit; heads: of the memory.  With a
        memory a minibatch is the whole rollouts of batch_size / n_steps envs."""
        if policy not in ("mlp", "memory"):
            raise ValueError(f"policy must be 'mlp' or 'memory', got {policy!r}")
        if not 0.0 <= dropout < 1.0:
            raise ValueError(f"dropout must be in [0, 1), got {dropout}")
        self.memory = policy == "memory"
        if self.memory and batch_size % n_steps:
            raise ValueError(f"a memory's minibatch is whole rollouts: batch_size ({batch_size}) must be a multiple of "
                             f"n_steps ({n_steps})")
        self.env = env
        self.n_envs = env.num_envs
        self.device = torch.device(device) if device is not None else torch.device("cpu")
        low = torch.as_tensor(env.action_space.low, dtype=torch.float32, device=self.device)
        high = torch.as_tensor(env.action_space.high, dtype=torch.float32, device=self.device)
        self.low, self.high = low, high
        self.obs_dim = env.observation_space.shape[0]
        self.act_dim = low.numel()
        self.n_steps, self.batch_size, self.n_epochs = n_steps, batch_size, n_epochs
        self.gamma, self.lam, self.clip, self.ent_coef, self.vf_coef = gamma, gae_lambda, clip_range, ent_coef, vf_coef
        self.max_grad_norm = max_grad_norm
        self.group = group
        torch.manual_seed(seed)
        kw = dict(dropout=dropout, seed=seed % (1 << 64))  # (a mask's key; torch takes negative seeds as well)
        self.policy = (MemoryActorCritic(self.obs_dim, self.act_dim, net_arch, heads=heads, **kw) if self.memory else
                       ActorCritic(self.obs_dim, self.act_dim, net_arch, **kw)).to(self.device)
        if group is not None:  # identical replicas: broadcast rank 0's initial weights
            import torch.distributed as dist
            for p in self.policy.parameters():
                dist.broadcast(p.data, src=0, group=group)
        # gradients live in ONE flat buffer (each parameter's .grad is a view of it): the multi-rank
        # average is a single all-reduce on that buffer, with no flatten / unflatten copies
        params = list(self.policy.parameters())
        self._flat_grad = torch.zeros(sum(p.numel() for p in params), dtype=torch.float32, device=self.device)
        off = 0
        for p in params:
            p.grad = self._flat_grad[off:off + p.numel()].view_as(p)
            off += p.numel()
        # on the GPU the minibatch update is replayed from HIP graphs (a batch-256 update is a few
        # hundred tiny kernels, launch-bound when issued one by one); Adam keeps its step count on
        # the device for that (capturable)
        self.use_graphs = (self.device.type == "cuda") if graphs is None else bool(graphs)
        self.opt = torch.optim.Adam(params, lr=learning_rate, eps=1e-5, capturable=self.use_graphs)
        self._graphs = None
        self.gen = torch.Generator(device=self.device)
        self.gen.manual_seed(seed)
        T, N, f = n_steps, self.n_envs, dict(dtype=torch.float32, device=self.device)
        self.buf_obs = torch.zeros((T, N, self.obs_dim), **f)
        self.buf_act = torch.zeros((T, N, self.act_dim), **f)
        self.buf_rew = torch.zeros((T, N), **f)
        self.buf_start = torch.zeros((T, N), **f)
        self.buf_val = torch.zeros((T, N), **f)
        self.buf_logp = torch.zeros((T, N), **f)
        self._noise = torch.zeros((T, N, self.act_dim), **f)
        # transition (t, n) of the running rollout has number _first + t * N + n
        self.dropout = dropout
        self._first = torch.zeros((), dtype=torch.int64, device=self.device)
        self._numbers = torch.arange((T + 1) * N, device=self.device).view(T + 1, N)
        if self.memory:
            # pi's and vf's memories in front of the current observation; vf's behind it; what the rollout began with
            self._pi, self._vf, self._vf_next = (self.policy.pi_net.state(N, self.device) for _ in range(3))
            self._began = (torch.empty_like(self._pi), torch.empty_like(self._vf))
        self._obs = None
        self._start = torch.ones(N, **f)
        self.num_timesteps = 0
        self.stats = {}

    # -- rollout ---------------------------------------------------------------
    def _rows(self, t: int):
        """numbers of the transitions at rollout index t (None: nothing is dropped)"""
        return self._first + self._numbers[t] if self.dropout else None

    def _current_value(self):
        """the critic on the current observation"""
        if not self.memory:
            return self.policy.value(self._obs, self._rows(0))
        h = self.policy.vf_net.step(self._obs, self._vf, self._start > 0, self._rows(0), next_state=self._vf_next)
        return self.policy.value_net(h).squeeze(-1)

    def _rollout_step(self, t: int):
        """One env step at rollout index t (persistent tensors; no host synchronisation).
        Launch count is what limits a 4,096-env rollout step, so: the sampling noise and the
        log-probabilities are handled for the whole rollout at once (log_std is constant during a
        rollout: log N(mean + std*eps) = -eps^2/2 - log_std - log(2 pi)/2), and the value of the next
        observation and of the terminal observation share one critic pass over 2N rows."""
        N = self.n_envs
        obs = self._obs
        if self.memory:
            h = self.policy.pi_net.step(obs, self._pi, self._start > 0, self._rows(t))
            act = self.policy.action_net(h) + self._std * self._noise[t]
        else:
            act = self.policy.mean(obs, self._rows(t)) + self._std * self._noise[t]
        clipped = torch.maximum(torch.minimum(act, self.high), self.low)
        nobs, rew, term, trunc, tobs = self.env.step_torch(clipped.to(torch.float64))
        term, trunc = term.bool(), trunc.bool()
        if self.memory:
            # behind this observation: what the terminal observation would be worth, and the next one's value
            self._vf, self._vf_next = self._vf_next, self._vf
            end = self.policy.vf_net.step(tobs.to(torch.float32), self._vf, None, self._rows(t), update=False)
            nxt = self.policy.vf_net.step(nobs, self._vf, term | trunc, self._rows(t + 1), next_state=self._vf_next)
            v2 = self.policy.value_net(torch.cat([nxt, end])).squeeze(-1)
        else:
            self._vin[:N].copy_(nobs)
            self._vin[N:].copy_(tobs)
            rows = torch.cat([self._rows(t + 1), self._rows(t)]) if self.dropout else None
            v2 = self.policy.value(self._vin, rows)
        # SB3 timeout bootstrap: truncated-not-terminated envs get gamma * V(terminal obs); evaluated
        # for every env and masked, so the rollout never waits on the host for an any()
        rew = rew.to(torch.float32) + self.gamma * torch.where(trunc & ~term, v2[N:], torch.zeros_like(v2[N:]))
        self.buf_obs[t].copy_(obs)
        self.buf_act[t].copy_(act)
        self.buf_rew[t].copy_(rew)
        self.buf_start[t].copy_(self._start)
        self.buf_val[t].copy_(self._val)
        self._val.copy_(v2[:N])
        self._obs.copy_(nobs)  # the env reuses its output buffers: copy, never alias
        self._start.copy_((term | trunc).to(torch.float32))

    @torch.no_grad()
    def collect_rollouts(self):
        if self._obs is None:
            self._obs = self.env.reset_torch().to(torch.float32).clone()
            self._val = self._current_value()
            self._vin = torch.empty((2 * self.n_envs, self.obs_dim), dtype=torch.float32, device=self.device)
        else:  # the critic changed in train(): value the carried-over observation with the new one
            self._val = self._current_value()
        if self.memory:
            self._began[0].copy_(self._pi)
            self._began[1].copy_(self._vf)
        # all sampling noise of the rollout in one draw
        self._noise.normal_(generator=self.gen)
        self._std = self.policy.log_std.exp()
        for t in range(self.n_steps):
            self._rollout_step(t)
        ls = self.policy.log_std
        self.buf_logp.copy_(-0.5 * self._noise.pow(2).sum(-1) - (ls.sum() + 0.5 * math.log(2 * math.pi) * ls.numel()))
        last_val = self._val
        self.adv, self.ret = compute_gae(self.buf_rew, self.buf_val, self.buf_start, last_val, self._start > 0,
                                         self.gamma, self.lam)
        self.num_timesteps += self.n_steps * self.n_envs
        self._first += self.n_steps * self.n_envs

    # -- update ----------------------------------------------------------------
    def _allreduce_grads(self):
        import torch.distributed as dist
        dist.all_reduce(self._flat_grad, group=self.group)
        self._flat_grad /= dist.get_world_size(self.group)

    def _loss(self, idx):
        """SB3 PPO.train minibatch loss (clipped surrogate, value MSE, entropy bonus)."""
        if self.memory:
            # idx: envs, each with its whole rollout
            seq = [x[:, idx].transpose(0, 1) for x in (self.buf_obs, self.buf_act, self.buf_start)]
            numbers = self._update_numbers[:, idx].transpose(0, 1) if self.dropout else None
            v, logp, ent = self.policy.evaluate(seq[0], seq[1], [s[idx] for s in self._began], seq[2] > 0, numbers)
            idx = (idx[:, None] + self._starts_at).flatten()  # of the flat buffers below, in the same order
        else:
            numbers = self._update_numbers.view(-1)[idx] if self.dropout else None
            v, logp, ent = self.policy.evaluate(self._obs_all[idx], self._act_all[idx], numbers)
        adv = self._adv_s[idx]
        if adv.numel() > 1:
            adv = (adv - adv.mean()) / (adv.std() + 1e-8)
        ratio = torch.exp(logp - self._logp_all[idx])
        pg = -torch.min(adv * ratio, adv * ratio.clamp(1 - self.clip, 1 + self.clip)).mean()
        vf = torch.nn.functional.mse_loss(self._ret_s[idx], v)
        ent_loss = -ent.mean()
        return pg + self.ent_coef * ent_loss + self.vf_coef * vf, pg, vf, ent_loss

    def _backward(self, idx):
        self._flat_grad.zero_()
        loss, pg, vf, ent_loss = self._loss(idx)
        loss.backward()
        return pg.detach(), vf.detach(), ent_loss.detach()

    def _apply(self):
        nn.utils.clip_grad_norm_(self.policy.parameters(), self.max_grad_norm)
        self.opt.step()

    def _minibatch_eager(self, idx):
        out = self._backward(idx)
        if self.group is not None:
            self._allreduce_grads()
        self._apply()
        return out

    def _capture(self):
        """Two graphs per minibatch: (zero grads, forward, backward) and (clip, Adam step); the
        multi-rank gradient average runs between them as one eager RCCL all-reduce."""
        ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(ga):
            self._g_out = self._backward(self._g_idx)
        with torch.cuda.graph(gb, pool=ga.pool()):
            self._apply()
        self._graphs = (ga, gb)

    def _minibatch_graph(self, idx):
        self._g_idx.copy_(idx)
        self._graphs[0].replay()
        if self.group is not None:
            self._allreduce_grads()
        self._graphs[1].replay()
        return self._g_out

    def train(self):
        T, N = self.n_steps, self.n_envs
        B = self.batch_size // T if self.memory else self.batch_size
        total = T * N
        self._obs_all = self.buf_obs.reshape(total, -1)
        self._act_all = self.buf_act.reshape(total, -1)
        self._logp_all = self.buf_logp.reshape(-1)
        if getattr(self, "_adv_s", None) is None:  # persistent: the graphs read these addresses
            self._adv_s = torch.empty(total, dtype=torch.float32, device=self.device)
            self._ret_s = torch.empty(total, dtype=torch.float32, device=self.device)
            self._g_idx = torch.zeros(B, dtype=torch.long, device=self.device)
            self._update_numbers = torch.empty_like(self._numbers[:T])
            self._starts_at = torch.arange(0, total, N, device=self.device)
        # the numbers that the rollout drew its masks with
        torch.add(self._numbers[:T], self._first - total, out=self._update_numbers)
        self._adv_s.copy_(self.adv.reshape(-1))
        self._ret_s.copy_(self.ret.reshape(-1))
        last = None
        warm = 0
        for _ in range(self.n_epochs):
            perm = torch.randperm(N if self.memory else total, generator=self.gen, device=self.device)
            for s in range(0, perm.numel(), B):
                idx = perm[s:s + B]
                if not self.use_graphs or idx.numel() != B:
                    last = self._minibatch_eager(idx)
                elif self._graphs is None and warm < 3:
                    # warm-up before capture (torch.cuda.graphs): real minibatch updates, run on a
                    # side stream so that autograd and the BLAS handles settle outside the capture
                    side = torch.cuda.Stream(device=self.device)
                    side.wait_stream(torch.cuda.current_stream(self.device))
                    with torch.cuda.stream(side):
                        last = self._minibatch_eager(idx)
                    torch.cuda.current_stream(self.device).wait_stream(side)
                    warm += 1
                else:
                    if self._graphs is None:
                        self._capture()
                    last = self._minibatch_graph(idx)
        if last is not None:
            self.stats = dict(zip(("policy_gradient_loss", "value_loss", "entropy_loss"), (float(x) for x in last)))

    def learn(self, iterations: int = 1):
        """Returns per-iteration wall times {rollout_s, train_s}."""
        times = []
        for _ in range(iterations):
            t0 = time.perf_counter()
            self.collect_rollouts()
            if self.device.type == "cuda":
                torch.cuda.synchronize(self.device)
            t1 = time.perf_counter()
            self.train()
            if self.device.type == "cuda":
                torch.cuda.synchronize(self.device)
            times.append({"rollout_s": t1 - t0, "train_s": time.perf_counter() - t1})
        return times
