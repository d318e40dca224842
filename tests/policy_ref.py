"""The policy operators (ur3e_amd/rl/ops.py) from their definitions in 64 bits, token after token, and the
rounding error that a 32-bit evaluation may have.  Test infrastructure only."""
import math

import numpy as np
import torch

HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}


def attention(q, k, v, log_decay, s0=None, starts=None, lengths=None, scale=1.0, dout=None, dfinal=None,
              magnitude=False):
    """{"out", "state"} and, with dout, {"dq", "dk", "dv", "ds0"}, float64 on the CPU.  magnitude: the same sums over the
    absolute values of their terms, which bounds what rounding can do to them."""
    def c(x):
        x = x.detach().cpu().double()
        return x.abs() if magnitude else x
    q, k, v = c(q), c(k), c(v)
    b, t, h, dk = q.shape
    hk, dv = k.shape[2], v.shape[3]
    grp = h // hk
    k, v = k.repeat_interleave(grp, 2), v.repeat_interleave(grp, 2)
    decay = torch.exp(log_decay.detach().cpu().double()).expand(b, h)
    starts = None if starts is None else starts.cpu() != 0
    n = torch.full((b,), t) if lengths is None else lengths.cpu().long().clamp(0, t)

    def a(i):
        """what token i multiplies the state by: 1 for padding"""
        f = decay.clone()
        if starts is not None:
            f[starts[:, i]] = 0.0
        f[i >= n] = 1.0
        return f[..., None, None]

    def drop(x, i):
        """where the factor is 0 nothing is left, whatever was there"""
        return torch.where(a(i) == 0, torch.zeros((), dtype=torch.float64), a(i) * x)

    def real(x, i):
        return torch.where((i < n).view(b, *[1] * (x.dim() - 1)), x, torch.zeros((), dtype=torch.float64))

    s = torch.zeros((b, h, dk, dv), dtype=torch.float64) if s0 is None else c(s0)
    out = torch.zeros((b, t, h, dv), dtype=torch.float64)
    grad = dout is not None
    if grad:
        do = c(dout)
        dq, dkk, dvv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for i in range(t):
        s = drop(s, i) + real(k[:, i, :, :, None] * v[:, i, :, None, :], i)
        out[:, i] = real(scale * (q[:, i, :, :, None] * s).sum(2), i)
        if grad:
            dq[:, i] = real(scale * (s * do[:, i, :, None, :]).sum(3), i)
    res = {"out": out, "state": s}
    if grad:
        g = torch.zeros_like(s) if dfinal is None else c(dfinal)
        for i in range(t - 1, -1, -1):
            g = g + real(scale * q[:, i, :, :, None] * do[:, i, :, None, :], i)
            dkk[:, i] = real((g * v[:, i, :, None, :]).sum(3), i)
            dvv[:, i] = real((g * k[:, i, :, :, None]).sum(2), i)
            g = drop(g, i)
        res.update(dq=dq, dk=dkk.view(b, t, hk, grp, dk).sum(3), dv=dvv.view(b, t, hk, grp, dv).sum(3), ds0=g)
    return res


def roundings(t, dk, dv, log_decay, heads=1):
    """How many roundings of 2^-24 a term of the sums can meet: the longest dot product (dk or dv terms), 16 + 16 terms of
    a chunk's two products, the sum over shared heads, a dozen factors; and for every chunk of 16 tokens the state's
    decay (the factor: 2 for exp, |16 l| for its argument, 1 for itself; 1 for the product), one more addition per
    token, and the joins of a split axis (as many again at most)."""
    f = log_decay[torch.isfinite(log_decay)]
    big = 16.0 * f.abs().max().item() if f.numel() else 0.0
    return max(dk, dv) + 44 + heads + 2 * math.ceil(t / 16) * (4 + big) + t


def bound(dtype, exact, magnitude, n):
    """|error| of a value of `dtype`: half a step where it leaves the kernel, n roundings of the sums, and, for
    16-bit tensors, two operands (scores, state) held as two parts of 8 bits each (2^-17 either)"""
    u = HALF_STEP[dtype]
    inner = n * 2.0 ** -24 + (2.0 ** -16 if dtype != torch.float32 else 0.0)
    tiny = 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -126
    return u * exact.abs() + (1 + u) * inner * magnitude + tiny


def check(got, exact, magnitude, n, what):
    got_d = got.detach().cpu().double()
    assert got_d.shape == exact.shape, (what, got_d.shape, exact.shape)
    err = (got_d - exact).abs()
    lim = bound(got.dtype, exact, magnitude, n)
    assert torch.isfinite(got_d).all(), f"{what}: not finite"
    over = (err / lim).max().item() if err.numel() else 0.0
    assert over <= 1.0, f"{what}: {over:.3g} times the bound"


def philox(seed, rows, cols, substream=0):
    """16-bit draws [rows, cols] of Philox4x32-10, in numpy's 64-bit integers"""
    u = np.uint64
    rows = np.asarray(rows, dtype=np.int64).astype(u)[:, None]
    nb = -(-cols // 8)
    low, sh = u(0xFFFFFFFF), u(32)
    c = [np.broadcast_to(np.arange(nb, dtype=u), (rows.shape[0], nb)), np.broadcast_to(rows & low, (rows.shape[0], nb)),
         np.broadcast_to(rows >> sh, (rows.shape[0], nb)), np.full((rows.shape[0], nb), substream, u)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        p, r = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(r >> sh) ^ c[1] ^ u(k[0]), r & low, (p >> sh) ^ c[3] ^ u(k[1]), p & low]
        k = [(k[0] + 0x9E3779B9) % (1 << 32), (k[1] + 0xBB67AE85) % (1 << 32)]
    words = np.stack(c, -1)
    return np.stack([words & u(0xFFFF), words >> u(16)], -1).reshape(rows.shape[0], -1)[:, :cols].astype(np.int64)
