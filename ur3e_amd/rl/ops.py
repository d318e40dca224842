"""Operators of a policy with memory (include/ur3e_policy.h).

`decay_attention` and `decay_attention_step` are the memory: linear attention whose state, one [dk, dv] matrix
a head, decays by a factor of that head's own,

    S_t = a_t S_{t-1} + k_t v_t^T,   a_t = 0 where an episode starts at t, else exp(log_decay[head])
    o_t = scale * S_t^T q_t

over whole sequences (a PPO update, a demonstration, a history to warm up on), with gradients, or one token
at a time (a rollout step).  `keyed_dropout` is dropout whose mask is a function of (seed, row id,
substream, column) alone: the update that revisits a transition drops what the rollout dropped, in whatever
order the minibatch gathers it, and no mask is stored.  They stand in for the reference's sequence
feature extractor over stacked frames (gymnasium_src/scripts/regular_rl/rl/train_rl.py:26-35).

GPU tensors go through the HIP library, on torch's current stream of their device, whatever the current
device is; a missing library raises.  CPU tensors are computed with elementary torch operations.  The calls
never synchronise and may be captured into HIP graphs, forward and backward; RuntimeError where an eager graph of the
default stream still holds one of the leaves, which torch cannot capture a backward pass of.  Wrong arguments raise
ValueError (TypeError for what is no tensor) before any launch.  Gradients are not differentiable again, and
forward-mode derivatives are refused on the GPU (ValueError); the CPU path carries them.
Results do not depend on timing: the same call gives the same bits.
"""
from __future__ import annotations

import importlib.util
import math
import os

import torch

from .. import runtime as rt

MAX_DIM = 128  # channels of a head (UR3E_ATTN_MAX_DIM)

_ext = None


def _c():
    """the binding (csrc/ur3e_policy_torch.cpp): checks, kernels and gradients; raises when it is not built"""
    global _ext
    if _ext is None:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "_lib", "ur3e_policy_torch.so")
        if not os.path.exists(path):
            raise RuntimeError(f"policy operators missing: {path} (run __graft_entry__.build())")
        rt.load_library()
        spec = importlib.util.spec_from_file_location("ur3e_policy_torch", path)
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        _ext = mod
    return _ext


def _tensor(what, name, x):
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{what}: {name} must be a torch tensor, got {type(x).__name__}")


def _scale(q):
    return q.shape[-1] ** -0.5 if q.dim() and q.shape[-1] else 1.0


def _attention_cpu(q, k, v, log_decay, s0, starts, lengths, scale):
    """token after token, in float32; autograd differentiates it"""
    b, t, h, dk = q.shape
    grp = h // k.shape[2]
    kf = k.float().repeat_interleave(grp, 2)
    vf = v.float().repeat_interleave(grp, 2)
    qf = q.float() * scale
    decay = log_decay.exp().view(1, h, 1, 1)
    s = qf.new_zeros((b, h, dk, v.shape[3])) if s0 is None else s0.clone()
    zero = qf.new_zeros(())
    if lengths is not None:
        # (in front of the loop: a zero gradient times padding that is not finite would not be zero)
        here = (torch.arange(t, device=q.device) < lengths[:, None]).view(b, t, 1, 1)
        qf, kf, vf = (torch.where(here, x, zero) for x in (qf, kf, vf))
    outs = []
    for i in range(t):
        old = s * decay
        if starts is not None:
            old = torch.where((starts[:, i] != 0).view(b, 1, 1, 1), zero, old)
        new = old + kf[:, i, :, :, None] * vf[:, i, :, None, :]
        o = (new * qf[:, i, :, :, None]).sum(2)
        if lengths is not None:
            real = i < lengths
            new = torch.where(real.view(b, 1, 1, 1), new, s)
            o = torch.where(real.view(b, 1, 1), o, zero)
        s = new
        outs.append(o)
    out = torch.stack(outs, 1) if outs else qf.new_zeros((b, 0, h, v.shape[3]))
    return out.to(q.dtype), s


def decay_attention(q, k, v, log_decay, initial_state=None, starts=None, lengths=None, scale=None,
                    return_state=False):
    """Attention with a decaying state over sequences; differentiable in q, k, v and initial_state.

    q [B, T, H, dk], k [B, T, Hk, dk], v [B, T, Hk, dv]: float32, bfloat16 or float16 (all the same), 1 to 128
      channels, any strides (a rollout buffer [T, B, ...] is passed as its transpose).  Query head h reads key
      / value head h // (H // Hk).
    log_decay [H] float32, at most 0 (not checked): a head's state is multiplied by exp(log_decay) a token; 0 never
      forgets, -inf keeps the token alone (of states that are finite).  A constant: it gets no gradient.
    initial_state [B, H, dk, dv] float32: the state in front of the first token (default 0).
    starts [B, T] bool or uint8: nonzero where an episode starts; the state in front of that token is dropped.
    lengths [B] int32: the tokens of each sequence (clamped to [0, T]); the rest of a row is padding, which is
      not read, leaves the state alone and gets zeros in the output and the gradients.
    scale: of the outputs, default dk ** -0.5.

    Returns (out [B, T, H, dv] of q's type, state): the state [B, H, dk, dv] float32 behind each sequence's
    last token, or None without `return_state`.  States and sums are float32.  On the GPU, with 16-bit tokens, a float32
    operand of a product is taken to 17 bits: the scores, the state where it is read out, and keys that enter a state which is
    not returned (to 25 bits where it is); outputs and gradients are then rounded to 8 bits (bfloat16) or 11 (float16).
    With float32 tokens every product is float32.
    What a NaN or an infinity reaches by the formula is not finite (a NaN where the formula may say infinity); nothing else
    is touched by it.
    B * H must be below 2**22 and T at most 2**30; with shared heads (H != Hk) or less than 4 channels, B * T * H times a
    quarter of the channels, rounded up, below 2**32 - 256.
    """
    _tensor("decay_attention", "q", q)
    if scale is None:
        scale = _scale(q)
    if q.is_cuda:
        return _c().decay_attention(q, k, v, log_decay, initial_state, starts, lengths, scale, return_state)
    _c().check_sequences(q, k, v, log_decay, initial_state, starts, lengths, scale)
    out, state = _attention_cpu(q, k, v, log_decay.detach(), initial_state, starts, lengths, scale)
    return out, (state if return_state else None)


def decay_attention_step(q, k, v, log_decay, state, starts=None, scale=None, next_state=None, update=True):
    """One token of `decay_attention` for B sequences: q [B, H, dk], k [B, Hk, dk], v [B, Hk, dv], starts [B];
    state [B, H, dk, dv] float32, contiguous.  Returns out [B, H, dv].

    The new state overwrites `state`, or goes to `next_state` (a buffer like `state` that does not overlap
    it), or nowhere with update=False (the value of a terminal observation: a look without a step).  No gradients:
    ValueError where one would be recorded.
    """
    _tensor("decay_attention_step", "q", q)
    if scale is None:
        scale = _scale(q)
    if q.is_cuda:
        return _c().decay_attention_step(q, k, v, log_decay, state, starts, scale, next_state, update)
    _c().check_step(q, k, v, log_decay, state, starts, scale, next_state, update)
    with torch.no_grad():
        out, new = _attention_cpu(q.unsqueeze(1), k.unsqueeze(1), v.unsqueeze(1), log_decay, state,
                                  None if starts is None else starts.unsqueeze(1), None, scale)
        if update:
            (state if next_state is None else next_state).copy_(new)
    return out[:, 0]


# -- keyed dropout ---------------------------------------------------------------


def keep_count(p: float) -> int:
    """How many of the 65,536 values of a 16-bit draw keep an element: the drop probability is
    1 - keep_count(p) / 65536, and what is kept is multiplied by 65536 / keep_count(p)."""
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"keyed_dropout: p must be in [0, 1], got {p}")
    return int(math.floor((1.0 - p) * 65536.0 + 0.5))


def _philox_cpu(seed, rows, blocks, substream, first=0):
    """Philox4x32-10 words [rows, blocks, 4] of the blocks from `first` on, in int64 (the wrapped products keep the words' bits)"""
    m = 0xFFFFFFFF
    c0 = torch.arange(first, first + blocks).expand(rows.numel(), blocks)
    c1 = (rows & m)[:, None].expand_as(c0)
    c2 = ((rows >> 32) & m)[:, None].expand_as(c0)
    c3 = torch.full_like(c0, substream)
    k0, k1 = seed & m, seed >> 32
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & m) ^ c1 ^ k0, p1 & m, ((p0 >> 32) & m) ^ c3 ^ k1, p0 & m
        k0, k1 = (k0 + 0x9E3779B9) & m, (k1 + 0xBB67AE85) & m
    return torch.stack([c0, c1, c2, c3], -1)


def _dropout_cpu(x, residual, rows, count, seed, substream):
    r, c = x.shape
    rows = torch.arange(r) if rows is None else rows
    w = _philox_cpu(seed, rows, (c + 7) // 8, substream)
    keep = torch.stack([w & 0xFFFF, w >> 16], -1).view(r, -1)[:, :c] < count
    y = torch.where(keep, x.float() * (65536.0 / count if count else 0.0), torch.zeros(()))
    if residual is not None:
        y = y + residual.float()
    return y.to(x.dtype)


def keyed_dropout(x, p, seed, rows=None, substream=0, residual=None):
    """y = x * keep / P(keep) (+ residual), differentiable in x and residual.

    x [..., C] float32, bfloat16 or float16; residual like x.  Whether column c of row r (rows of x, its leading
    dimensions flattened) is kept is a fixed function of seed (an int in [0, 2**64)), rows[r], substream (an
    int in [0, 2**32): one per place in a network) and c: Philox4x32-10 with the row's id in its counter.
    rows: int64 ids, as many as x has rows and of any values (the same id twice: the same mask twice); default
    0, 1, 2, ...  p in [0, 1] is rounded to a multiple of 2**-16 and the scale follows the rounded value
    (`keep_count`); what is dropped is 0 whatever it held, p = 1 drops everything.
    """
    _tensor("keyed_dropout", "x", x)
    count = keep_count(p)
    if type(seed) is not int or not 0 <= seed < 1 << 64:
        raise ValueError(f"keyed_dropout: seed must be an int in [0, 2**64), got {seed!r}")
    if type(substream) is not int or not 0 <= substream < 1 << 32:
        raise ValueError(f"keyed_dropout: substream must be an int in [0, 2**32), got {substream!r}")
    if x.is_cuda:
        return _c().keyed_dropout(x, count, seed, rows, substream, residual)
    _c().check_dropout(x, rows, residual)
    if x.numel() == 0:
        return x.clone() if residual is None else x + residual
    y = _dropout_cpu(x.reshape(-1, x.shape[-1]), None if residual is None else residual.reshape(-1, x.shape[-1]),
                     None if rows is None else rows.reshape(-1), count, seed, substream)
    return y.view(x.shape)
