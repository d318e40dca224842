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
never synchronise and may be captured into HIP graphs.  Wrong arguments raise ValueError before any launch.
"""
from __future__ import annotations

import ctypes
import math

import torch

from .. import runtime as rt

MAX_DIM = 128
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class TokensC(ctypes.Structure):
    _fields_ = [("p", ctypes.c_void_p), ("sb", ctypes.c_longlong), ("st", ctypes.c_longlong),
                ("sh", ctypes.c_longlong)]


class AttnC(ctypes.Structure):
    _fields_ = [("b", ctypes.c_int), ("t", ctypes.c_int), ("heads", ctypes.c_int), ("kv_heads", ctypes.c_int),
                ("dk", ctypes.c_int), ("dv", ctypes.c_int), ("dtype", ctypes.c_int), ("scale", ctypes.c_float),
                ("q", TokensC), ("k", TokensC), ("v", TokensC), ("log_decay", ctypes.c_void_p),
                ("s0", ctypes.c_void_p), ("starts", ctypes.c_void_p), ("starts_sb", ctypes.c_longlong),
                ("starts_st", ctypes.c_longlong), ("lengths", ctypes.c_void_p)]


_bound = None


def _lib():
    global _bound
    if _bound is None:
        L = rt.load_library()
        vp, sz, ll = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_longlong
        L.ur3e_attn_workspace.argtypes = [vp, ctypes.c_int, ctypes.POINTER(sz)]
        L.ur3e_attn_forward.argtypes = [vp, vp, vp, vp, sz, vp]
        L.ur3e_attn_backward.argtypes = [vp, vp, vp, vp, vp, vp, vp, vp, sz, vp]
        L.ur3e_attn_step.argtypes = [vp, vp, vp, vp, vp]
        L.ur3e_keyed_dropout.argtypes = [ctypes.c_int, ll, ctypes.c_int, vp, ll, vp, ll, vp, ll, vp,
                                         ctypes.c_ulonglong, ctypes.c_uint, ctypes.c_int, vp]
        _bound = L
    return _bound


def _stream(device):
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _p(t):
    return None if t is None else t.data_ptr()


def _tok(t):
    """[b, t, heads, d] tensor with contiguous channels"""
    return TokensC(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2))


def _unit(t):
    """the tensor, with the channels of a token next to each other"""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _tokens_like(ref, heads, d):
    """an empty [b, t, heads, d] in the memory order of `ref` (sequence- or time-major)"""
    b, t = ref.shape[:2]
    if t > 1 and b > 1 and ref.stride(1) > ref.stride(0):
        return ref.new_empty((t, b, heads, d)).transpose(0, 1)
    return ref.new_empty((b, t, heads, d))


def _check_qkv(what, q, k, v, log_decay, starts, scale, dims):
    for n, x in (("q", q), ("k", k), ("v", v), ("log_decay", log_decay)):
        if not isinstance(x, torch.Tensor):
            raise ValueError(f"{what}: {n} must be a torch tensor")
    if q.dtype not in _DTYPES:
        raise ValueError(f"{what}: q must be float32, bfloat16 or float16, got {q.dtype}")
    lead = q.shape[:-2]
    if q.dim() != dims or k.dim() != dims or v.dim() != dims:
        raise ValueError(f"{what}: q, k and v must have {dims} dimensions, got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    for n, x in (("k", k), ("v", v)):
        if x.dtype != q.dtype or x.device != q.device:
            raise ValueError(f"{what}: {n} is {x.dtype} on {x.device}, q {q.dtype} on {q.device}")
        if x.shape[:-2] != lead:
            raise ValueError(f"{what}: {n} has leading sizes {tuple(x.shape[:-2])}, q {tuple(lead)}")
    h, hk = q.shape[-2], k.shape[-2]
    if hk < 1 or h < 1 or h % hk or v.shape[-2] != hk:
        raise ValueError(f"{what}: {h} query heads over {hk} key heads and {v.shape[-2]} value heads: the key and "
                         "value heads must be as many, and divide the query heads")
    if k.shape[-1] != q.shape[-1]:
        raise ValueError(f"{what}: q has {q.shape[-1]} channels, k {k.shape[-1]}")
    for n, x in (("q and k", q), ("v", v)):
        if not 1 <= x.shape[-1] <= MAX_DIM:
            raise ValueError(f"{what}: {n} must have 1 to {MAX_DIM} channels, got {x.shape[-1]}")
    if log_decay.dtype != torch.float32 or log_decay.device != q.device or tuple(log_decay.shape) != (h,):
        raise ValueError(f"{what}: log_decay must be a float32 tensor of shape ({h},) on {q.device}")
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what}: log_decay is a constant of the heads and gets no gradient; detach it")
    if starts is not None:
        if not isinstance(starts, torch.Tensor) or starts.dtype not in (torch.bool, torch.uint8) \
                or starts.device != q.device or starts.shape != lead:
            raise ValueError(f"{what}: starts must be a bool or uint8 tensor of shape {tuple(lead)} on {q.device}")
    if not math.isfinite(scale):
        raise ValueError(f"{what}: scale must be finite, got {scale}")


def _check_state(what, name, s, shape, device):
    if not isinstance(s, torch.Tensor) or s.dtype != torch.float32 or s.device != device or tuple(s.shape) != shape:
        raise ValueError(f"{what}: {name} must be a float32 tensor of shape {shape} on {device}")


def _args(q, k, v, log_decay, s0, starts, lengths, scale):
    b, t, h, dk = q.shape
    a = AttnC()
    a.b, a.t, a.heads, a.kv_heads, a.dk, a.dv = b, t, h, k.shape[2], dk, v.shape[3]
    a.dtype = _DTYPES[q.dtype]
    a.scale = scale
    a.q, a.k, a.v = _tok(q), _tok(k), _tok(v)
    a.log_decay = _p(log_decay)
    a.s0 = _p(s0)
    if starts is not None:
        a.starts, a.starts_sb, a.starts_st = _p(starts), starts.stride(0), starts.stride(1)
    a.lengths = _p(lengths)
    return a


def _workspace(L, a, backward, device):
    n = ctypes.c_size_t()
    rt._check(L.ur3e_attn_workspace(ctypes.byref(a), backward, ctypes.byref(n)), L)
    return torch.empty(n.value, dtype=torch.uint8, device=device) if n.value else None


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, s0, log_decay, starts, lengths, scale, return_state):
        L = _lib()
        out = _tokens_like(q, q.shape[2], v.shape[3])
        final = q.new_empty((q.shape[0], q.shape[2], q.shape[3], v.shape[3]), dtype=torch.float32) if return_state else None
        with torch.cuda.device(q.device):
            a = _args(q, k, v, log_decay, s0, starts, lengths, scale)
            ws = _workspace(L, a, 0, q.device)
            rt._check(L.ur3e_attn_forward(ctypes.byref(a), ctypes.byref(_tok(out)), _p(final), _p(ws),
                                          0 if ws is None else ws.numel(), _stream(q.device)), L)
        ctx.save_for_backward(q, k, v, s0, log_decay, starts, lengths)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return out, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dfinal):
        q, k, v, s0, log_decay, starts, lengths = ctx.saved_tensors
        L = _lib()
        if dout is None:
            dout = torch.zeros_like(v[:, :, :1]).expand(-1, -1, q.shape[2], -1)
        dout = _unit(dout)
        if dfinal is not None:
            dfinal = dfinal.contiguous()
        dq = _tokens_like(q, *q.shape[2:])
        dk = _tokens_like(k, *k.shape[2:])
        dv = _tokens_like(v, *v.shape[2:])
        ds0 = torch.empty_like(s0) if s0 is not None and ctx.needs_input_grad[3] else None
        with torch.cuda.device(q.device):
            a = _args(q, k, v, log_decay, s0, starts, lengths, ctx.scale)
            ws = _workspace(L, a, 1, q.device)
            rt._check(L.ur3e_attn_backward(ctypes.byref(a), ctypes.byref(_tok(dout)), _p(dfinal),
                                           ctypes.byref(_tok(dq)), ctypes.byref(_tok(dk)), ctypes.byref(_tok(dv)),
                                           _p(ds0), _p(ws), 0 if ws is None else ws.numel(), _stream(q.device)), L)
        return dq, dk, dv, ds0, None, None, None, None, None


def _attention_cpu(q, k, v, log_decay, s0, starts, lengths, scale):
    """token after token, in float32; autograd differentiates it"""
    b, t, h, dk = q.shape
    grp = h // k.shape[2]
    kf = k.float().repeat_interleave(grp, 2)
    vf = v.float().repeat_interleave(grp, 2)
    qf = q.float() * scale
    decay = log_decay.exp().view(1, h, 1, 1)
    s = qf.new_zeros((b, h, dk, v.shape[3])) if s0 is None else s0
    zero = qf.new_zeros(())
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
    log_decay [H] float32: a head's state is multiplied by exp(log_decay) a token; 0 never forgets, -inf keeps
      the token alone.  A constant: it gets no gradient.
    initial_state [B, H, dk, dv] float32: the state in front of the first token (default 0).
    starts [B, T] bool or uint8: nonzero where an episode starts; the state in front of that token is dropped.
    lengths [B] int32: the tokens of each sequence (clamped to [0, T]); the rest of a row is padding, which is
      not read, leaves the state alone and gets zeros in the output and the gradients.
    scale: of the outputs, default dk ** -0.5.

    Returns (out [B, T, H, dv] of q's type, state): the state [B, H, dk, dv] float32 behind each sequence's
    last token, or None without `return_state`.  States and sums are float32.
    """
    what = "decay_attention"
    if scale is None:
        scale = q.shape[-1] ** -0.5 if isinstance(q, torch.Tensor) and q.dim() and q.shape[-1] else 1.0
    scale = float(scale)
    _check_qkv(what, q, k, v, log_decay, starts, scale, 4)
    b, t, h, dk = q.shape
    if initial_state is not None:
        _check_state(what, "initial_state", initial_state, (b, h, dk, v.shape[3]), q.device)
        initial_state = initial_state.contiguous()
    if lengths is not None:
        if not isinstance(lengths, torch.Tensor) or lengths.dtype != torch.int32 or lengths.device != q.device \
                or tuple(lengths.shape) != (b,):
            raise ValueError(f"{what}: lengths must be an int32 tensor of shape ({b},) on {q.device}")
        lengths = lengths.contiguous()
    log_decay = log_decay.detach().contiguous()
    if q.device.type == "cpu":
        out, state = _attention_cpu(q, k, v, log_decay, initial_state, starts, lengths, scale)
        return out, (state if return_state else None)
    if starts is not None and starts.dtype == torch.bool:
        starts = starts.view(torch.uint8)
    return _DecayAttention.apply(_unit(q), _unit(k), _unit(v), initial_state, log_decay, starts, lengths, scale,
                                 bool(return_state))


def _overlap(x, y):
    n = x.numel() * x.element_size()
    return abs(x.data_ptr() - y.data_ptr()) < n


@torch.no_grad()
def decay_attention_step(q, k, v, log_decay, state, starts=None, scale=None, next_state=None, update=True):
    """One token of `decay_attention` for B sequences: q [B, H, dk], k [B, Hk, dk], v [B, Hk, dv], starts [B];
    state [B, H, dk, dv] float32, contiguous.  Returns out [B, H, dv].

    The new state overwrites `state`, or goes to `next_state` (a buffer like `state` that does not overlap
    it), or nowhere with update=False (the value of a terminal observation: a look without a step).  No gradients.
    """
    what = "decay_attention_step"
    if scale is None:
        scale = q.shape[-1] ** -0.5 if isinstance(q, torch.Tensor) and q.dim() and q.shape[-1] else 1.0
    scale = float(scale)
    _check_qkv(what, q, k, v, log_decay, starts, scale, 3)
    b, h, dk = q.shape
    shape = (b, h, dk, v.shape[2])
    _check_state(what, "state", state, shape, q.device)
    if not state.is_contiguous():
        raise ValueError(f"{what}: state must be contiguous")
    if next_state is not None:
        if not update:
            raise ValueError(f"{what}: next_state without an update")
        _check_state(what, "next_state", next_state, shape, q.device)
        if not next_state.is_contiguous():
            raise ValueError(f"{what}: next_state must be contiguous")
        if next_state.data_ptr() != state.data_ptr() and _overlap(state, next_state):
            raise ValueError(f"{what}: next_state overlaps state")
    to = (state if next_state is None else next_state) if update else None
    q, k, v = (_unit(x).unsqueeze(1) for x in (q, k, v))
    log_decay = log_decay.detach().contiguous()
    if q.device.type == "cpu":
        out, new = _attention_cpu(q, k, v, log_decay, state, None if starts is None else starts.view(b, 1), None, scale)
        if to is not None:
            to.copy_(new)
        return out[:, 0]
    if starts is not None:
        starts = (starts.view(torch.uint8) if starts.dtype == torch.bool else starts).unsqueeze(1)
    L = _lib()
    out = q.new_empty((b, 1, h, v.shape[3]))
    with torch.cuda.device(q.device):
        a = _args(q, k, v, log_decay, None, starts, None, scale)
        rt._check(L.ur3e_attn_step(ctypes.byref(a), ctypes.byref(_tok(out)), _p(state), _p(to), _stream(q.device)), L)
    return out[:, 0]


# -- keyed dropout ---------------------------------------------------------------


def keep_count(p: float) -> int:
    """How many of the 65,536 values of a 16-bit draw keep an element: the drop probability is
    1 - keep_count(p) / 65536, and what is kept is multiplied by 65536 / keep_count(p)."""
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"keyed_dropout: p must be in [0, 1], got {p}")
    return int(math.floor((1.0 - p) * 65536.0 + 0.5))


def _philox_cpu(seed, rows, blocks, substream):
    """Philox4x32-10 words [rows, blocks, 4] in int64 (the wrapped products keep the words' bits)"""
    m = 0xFFFFFFFF
    c0 = torch.arange(blocks).expand(rows.numel(), blocks)
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


def _dropout_2d(x, residual, rows, count, seed, substream):
    """x [r, c] (contiguous columns) -> y [r, c]"""
    if x.device.type == "cpu":
        return _dropout_cpu(x, residual, rows, count, seed, substream)
    L = _lib()
    y = x.new_empty(x.shape)
    with torch.cuda.device(x.device):
        rt._check(L.ur3e_keyed_dropout(_DTYPES[x.dtype], x.shape[0], x.shape[1], _p(x), x.stride(0), _p(residual),
                                       0 if residual is None else residual.stride(0), _p(y), y.stride(0), _p(rows),
                                       seed, substream, count, _stream(x.device)), L)
    return y


def _rows2d(x):
    """x as [rows, columns] with contiguous columns, without a copy where its strides allow it"""
    x = x.reshape(-1, x.shape[-1]) if x.dim() != 2 else x
    return _unit(x)


class _KeyedDropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, rows, count, seed, substream):
        ctx.save_for_backward(rows)
        ctx.key = (count, seed, substream)
        y = _dropout_2d(_rows2d(x), None if residual is None else _rows2d(residual), rows, count, seed, substream)
        return y.view(x.shape)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        rows, = ctx.saved_tensors
        dx = None
        if ctx.needs_input_grad[0]:
            dx = _dropout_2d(_rows2d(dy), None, rows, *ctx.key).view(dy.shape)
        return dx, (dy if ctx.needs_input_grad[1] else None), None, None, None, None


def keyed_dropout(x, p, seed, rows=None, substream=0, residual=None):
    """y = x * keep / P(keep) (+ residual), differentiable in x and residual.

    x [..., C] float32, bfloat16 or float16; residual like x.  Whether column c of row r (rows of x, its leading
    dimensions flattened) is kept is a fixed function of seed (an int in [0, 2**64)), rows[r], substream (an
    int in [0, 2**32): one per place in a network) and c: Philox4x32-10 with the row's id in its counter.
    rows: int64 ids, as many as x has rows and of any values (the same id twice: the same mask twice); default
    0, 1, 2, ...  p in [0, 1] is rounded to a multiple of 2**-16 and the scale follows the rounded value
    (`keep_count`); what is dropped is 0 whatever it held, p = 1 drops everything.
    """
    what = "keyed_dropout"
    if not isinstance(x, torch.Tensor) or x.dtype not in _DTYPES or x.dim() < 1:
        raise ValueError(f"{what}: x must be a float32, bfloat16 or float16 tensor of at least one dimension")
    count = keep_count(p)
    if not isinstance(seed, int) or not 0 <= seed < 1 << 64:
        raise ValueError(f"{what}: seed must be an int in [0, 2**64), got {seed!r}")
    if not isinstance(substream, int) or not 0 <= substream < 1 << 32:
        raise ValueError(f"{what}: substream must be an int in [0, 2**32), got {substream!r}")
    n = math.prod(x.shape[:-1])
    if rows is not None:
        if not isinstance(rows, torch.Tensor) or rows.dtype != torch.int64 or rows.device != x.device \
                or rows.numel() != n:
            raise ValueError(f"{what}: rows must be {n} int64 ids on {x.device}")
        rows = rows.reshape(-1).contiguous()
    if residual is not None and (not isinstance(residual, torch.Tensor) or residual.dtype != x.dtype
                                 or residual.device != x.device or residual.shape != x.shape):
        raise ValueError(f"{what}: residual must be like x: {tuple(x.shape)} {x.dtype} on {x.device}")
    if x.numel() == 0:
        return x.clone() if residual is None else x + residual
    return _KeyedDropout.apply(x, residual, rows, count, seed, substream)
