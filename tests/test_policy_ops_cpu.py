"""The policy operators (ur3e_amd/rl/ops.py) without a GPU: the CPU path against the 64-bit definitions, the
generator's published known answers, what is refused, and the C entries' own refusals."""
import ctypes

import numpy as np
import pytest
import torch

from ur3e_amd.rl import ops

import policy_ref as ref


def make(b, t, h, hk, dk, dv, dtype=torch.float32, seed=0, starts=0.0, ragged=False, state=True):
    g = torch.Generator().manual_seed(seed)
    x = dict(q=torch.randn((b, t, h, dk), generator=g).to(dtype), k=torch.randn((b, t, hk, dk), generator=g).to(dtype),
             v=torch.randn((b, t, hk, dv), generator=g).to(dtype),
             log_decay=torch.log(torch.linspace(0.6, 0.99, h)),
             initial_state=torch.randn((b, h, dk, dv), generator=g) if state else None,
             starts=torch.rand((b, t), generator=g) < starts if starts else None,
             lengths=torch.randint(0, t + 1, (b,), generator=g, dtype=torch.int32) if ragged else None)
    return x


def exact(x, dout=None, dfinal=None, scale=None):
    a = (x["q"], x["k"], x["v"], x["log_decay"], x["initial_state"], x["starts"], x["lengths"],
         x["q"].shape[-1] ** -0.5 if scale is None else scale, dout, dfinal)
    return ref.attention(*a), ref.attention(*a, magnitude=True)


@pytest.mark.parametrize("b,t,h,hk,dk,dv", [(2, 1, 1, 1, 1, 1), (3, 7, 4, 2, 5, 3), (1, 33, 2, 2, 16, 8)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_cpu_matches_definition(b, t, h, hk, dk, dv, dtype):
    x = make(b, t, h, hk, dk, dv, dtype, starts=0.2, ragged=True)
    g = torch.Generator().manual_seed(1)
    dout, dfinal = torch.randn((b, t, h, dv), generator=g).to(dtype), torch.randn((b, h, dk, dv), generator=g)
    leaves = [x[n].requires_grad_() for n in ("q", "k", "v", "initial_state")]
    out, state = ops.decay_attention(**x, return_state=True)
    grads = torch.autograd.grad([out, state], leaves, [dout, dfinal])
    e, m = exact(x, dout, dfinal)
    n = ref.roundings(t, dk, dv, x["log_decay"], h // hk)
    for got, name in zip((out, state, *grads), ("out", "state", "dq", "dk", "dv", "ds0")):
        ref.check(got, e[name], m[name], n, name)


def test_step_cpu_is_the_sequence_token_by_token():
    x = make(3, 9, 4, 2, 6, 5, starts=0.3)
    out, state = ops.decay_attention(**x, return_state=True)
    s = x["initial_state"].clone()
    for i in range(9):
        a = (x["q"][:, i], x["k"][:, i], x["v"][:, i], x["log_decay"])
        before = s.clone()
        look = ops.decay_attention_step(*a, s, starts=x["starts"][:, i], update=False)
        assert torch.equal(s, before)
        nxt = torch.empty_like(s)
        other = ops.decay_attention_step(*a, s, starts=x["starts"][:, i], next_state=nxt)
        assert torch.equal(s, before)
        o = ops.decay_attention_step(*a, s, starts=x["starts"][:, i])
        assert torch.equal(o, look) and torch.equal(o, other) and torch.equal(s, nxt)
        torch.testing.assert_close(o, out[:, i], rtol=0, atol=1e-6)
    torch.testing.assert_close(s, state, rtol=0, atol=1e-6)


def test_attention_empty():
    for b, t in ((0, 5), (3, 0)):
        x = make(b, t, 2, 1, 4, 3)
        out, state = ops.decay_attention(**x, return_state=True)
        assert out.shape == (b, t, 2, 3) and torch.equal(state, x["initial_state"])


BAD = [
    (dict(q=torch.zeros(2, 3, 4)), "dimensions"),
    (dict(q=torch.zeros((2, 3, 4, 5), dtype=torch.float64)), "float32, bfloat16 or float16"),
    (dict(k=torch.zeros((2, 3, 2, 5), dtype=torch.bfloat16)), "k is"),
    (dict(k=torch.zeros(2, 4, 2, 5)), "leading sizes"),
    (dict(k=torch.zeros(2, 3, 3, 5), v=torch.zeros(2, 3, 3, 6)), "divide the query heads"),
    (dict(v=torch.zeros(2, 3, 4, 6)), "as many"),
    (dict(k=torch.zeros(2, 3, 2, 4)), "channels"),
    (dict(v=torch.zeros(2, 3, 2, 129)), "1 to 128"),
    (dict(v=torch.zeros(2, 3, 2, 0)), "1 to 128"),
    (dict(log_decay=torch.zeros(3)), "log_decay"),
    (dict(log_decay=torch.zeros(4, dtype=torch.float64)), "log_decay"),
    (dict(log_decay=torch.zeros(4, requires_grad=True)), "gets no gradient"),
    (dict(initial_state=torch.zeros(2, 4, 6, 5)), "initial_state"),
    (dict(initial_state=torch.zeros((2, 4, 5, 6), dtype=torch.bfloat16)), "initial_state"),
    (dict(starts=torch.zeros(2, 3)), "starts"),
    (dict(starts=torch.zeros((3, 2), dtype=torch.bool)), "starts"),
    (dict(lengths=torch.zeros(2, dtype=torch.int64)), "lengths"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths"),
    (dict(scale=float("nan")), "scale"),
]


@pytest.mark.parametrize("change,says", BAD)
def test_attention_refuses(change, says):
    x = dict(q=torch.zeros(2, 3, 4, 5), k=torch.zeros(2, 3, 2, 5), v=torch.zeros(2, 3, 2, 6), log_decay=torch.zeros(4))
    ops.decay_attention(**x)
    with pytest.raises(ValueError, match=says):
        ops.decay_attention(**{**x, **change})


def test_step_refuses():
    x = dict(q=torch.zeros(2, 4, 5), k=torch.zeros(2, 2, 5), v=torch.zeros(2, 2, 6), log_decay=torch.zeros(4),
             state=torch.zeros(2, 4, 5, 6))
    ops.decay_attention_step(**x)
    big = torch.zeros(3, 4, 5, 6)
    for change, says in ((dict(state=torch.zeros(2, 4, 6, 5)), "state"),
                         (dict(state=torch.zeros(2, 4, 6, 5).transpose(2, 3)), "contiguous"),
                         (dict(state=big[:2], next_state=big[1:]), "overlaps"),
                         (dict(next_state=torch.zeros(2, 4, 5, 6), update=False), "without an update"),
                         (dict(starts=torch.zeros((2, 1), dtype=torch.bool)), "starts"),
                         (dict(q=torch.zeros(2, 1, 4, 5)), "dimensions")):
        with pytest.raises(ValueError, match=says):
            ops.decay_attention_step(**{**x, **change})


@pytest.mark.parametrize("name", ["q", "k", "v", "state"])
def test_step_refuses_gradients(name):
    """a step that autograd would take for a constant is refused; under no_grad the same call runs"""
    x = dict(q=torch.ones(2, 2, 4), k=torch.ones(2, 2, 4), v=torch.ones(2, 2, 4), log_decay=torch.zeros(2),
             state=torch.zeros(2, 2, 4, 4))
    x[name].requires_grad_()
    with pytest.raises(ValueError, match="no gradients"):
        ops.decay_attention_step(**x)
    with torch.no_grad():
        out = ops.decay_attention_step(**x)
    assert not out.requires_grad and (out == 2.0).all() and (x["state"].detach() == 1.0).all()


def test_philox_known_answers():
    """Random123's kat_vectors for philox4x32 with 10 rounds"""
    kat = [(0, (0, 0), 0, "6627e8d5 e169c58d bc57ac4c 9b00dbd8"),
           ((1 << 64) - 1, (0xffffffff, 0xffffffffffffffff), 0xffffffff, "408f276d 41c83b0e a20bc7c6 6d5451fd")]
    m = 0xffffffff
    for seed, (block, row), sub, want in kat:
        rows = torch.tensor([row - (1 << 64) if row >= 1 << 63 else row])
        if block == 0:
            got = ops._philox_cpu(seed, rows, 1, sub)[0, 0].tolist()
            assert [f"{w:08x}" for w in got] == want.split()
            d = ref.philox(seed, rows.numpy(), 8, sub)[0]
            assert [f"{d[2 * i] | d[2 * i + 1] << 16:08x}" for i in range(4)] == want.split()
        else:  # a block number that no row is wide enough for: the rounds alone, in Python's integers
            c, k = [block, row & m, row >> 32, sub], [seed & m, seed >> 32]
            for _ in range(10):
                p, r = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
                c = [(r >> 32) ^ c[1] ^ k[0], r & m, (p >> 32) ^ c[3] ^ k[1], p & m]
                k = [(k[0] + 0x9E3779B9) & m, (k[1] + 0xBB67AE85) & m]
            assert [f"{w:08x}" for w in c] == want.split()


@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_dropout_cpu_matches_definition(p, dtype):
    g = torch.Generator().manual_seed(3)
    x = torch.randn((5, 13), generator=g).to(dtype).requires_grad_()
    res = torch.randn((5, 13), generator=g).to(dtype).requires_grad_()
    rows = torch.tensor([3, -1, 3, 1 << 40, 0])
    seed = 0xDEADBEEF12345678
    count = ops.keep_count(p)
    assert abs(count / 65536 - (1 - p)) <= 2.0 ** -17
    keep = torch.from_numpy(ref.philox(seed, rows.numpy(), 13, 7) < count)
    assert torch.equal(keep[0], keep[2])
    y = ops.keyed_dropout(x, p, seed, rows, 7, residual=res)
    up = 65536 / count if count else 0.0
    e = torch.where(keep, x.double() * up, 0.0) + res.double()
    # the scale, the product and the sum each round to 2^-24; the value once to its type
    ref.check(y, e, torch.where(keep, x.double().abs() * up, 0.0) + res.double().abs(), 3, "y")
    dy = torch.randn((5, 13), generator=g).to(dtype)
    dx, dres = torch.autograd.grad(y, [x, res], dy)
    assert torch.equal(dres, dy)
    ref.check(dx, torch.where(keep, dy.double() * up, 0.0), dy.double().abs() * max(up, 1), 3, "dx")


def test_dropout_drops_what_is_not_finite_and_shapes():
    x = torch.full((4, 3, 8), float("nan"))
    assert torch.equal(ops.keyed_dropout(x, 1.0, 1), torch.zeros(4, 3, 8))
    y = ops.keyed_dropout(torch.ones(4, 3, 8), 0.5, 1)
    assert torch.equal(y.view(12, 8), ops.keyed_dropout(torch.ones(12, 8), 0.5, 1))
    assert torch.equal(ops.keyed_dropout(torch.ones(8), 0.5, 1), y[0, 0])
    assert ops.keyed_dropout(torch.ones(0, 8), 0.5, 1).shape == (0, 8)
    assert ops.keyed_dropout(torch.ones(3, 0), 0.5, 1).shape == (3, 0)


def test_dropout_refuses():
    x = torch.zeros(4, 6)
    for a, kw, says in (((x.double(), 0.1, 0), {}, "float32, bfloat16 or float16"), ((x, 1.1, 0), {}, "p must be"),
                        ((x, float("nan"), 0), {}, "p must be"), ((x, 0.1, -1), {}, "seed"), ((x, 0.1, 1 << 64), {}, "seed"),
                        ((x, 0.1, 1.5), {}, "seed"), ((x, 0.1, 0), dict(substream=1 << 32), "substream"),
                        ((x, 0.1, 0), dict(rows=torch.zeros(3, dtype=torch.int64)), "rows"),
                        ((x, 0.1, 0), dict(rows=torch.zeros(4, dtype=torch.int32)), "rows"),
                        ((x, 0.1, 0), dict(residual=torch.zeros(4, 1)), "residual"),
                        ((x, 0.1, 0), dict(residual=x.half()), "residual")):
        with pytest.raises(ValueError, match=says):
            ops.keyed_dropout(*a, **kw)


class TokensC(ctypes.Structure):
    _fields_ = [("p", ctypes.c_void_p), ("sb", ctypes.c_longlong), ("st", ctypes.c_longlong),
                ("sh", ctypes.c_longlong)]


class AttnC(ctypes.Structure):
    _fields_ = [("b", ctypes.c_int), ("t", ctypes.c_int), ("heads", ctypes.c_int), ("kv_heads", ctypes.c_int),
                ("dk", ctypes.c_int), ("dv", ctypes.c_int), ("dtype", ctypes.c_int), ("scale", ctypes.c_float),
                ("q", TokensC), ("k", TokensC), ("v", TokensC), ("log_decay", ctypes.c_void_p),
                ("s0", ctypes.c_void_p), ("starts", ctypes.c_void_p), ("starts_sb", ctypes.c_longlong),
                ("starts_st", ctypes.c_longlong), ("lengths", ctypes.c_void_p)]


def test_c_entries_refuse_before_any_launch():
    """every refusal of the C entries comes from the host (no GPU here); empty calls succeed"""
    from ur3e_amd import runtime as rt
    L = rt.load_library()
    EINVAL = -1
    vp, sz, ll, ip = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_longlong, ctypes.c_int
    L.ur3e_attn_workspace.argtypes = [vp, ip, vp]
    L.ur3e_attn_forward.argtypes = [vp, vp, vp, vp, sz, vp]
    L.ur3e_attn_backward.argtypes = [vp] * 8 + [sz, vp]
    L.ur3e_attn_step.argtypes = [vp] * 5
    L.ur3e_keyed_dropout.argtypes = [ip, ll, ip, vp, ll, vp, ll, vp, ll, vp, ctypes.c_ulonglong, ctypes.c_uint, ip, vp]

    def attn(**kw):
        a = AttnC()
        a.b, a.t, a.heads, a.kv_heads, a.dk, a.dv, a.dtype, a.scale = 1, 4, 2, 1, 8, 8, 0, 1.0
        a.q = a.k = a.v = TokensC(4096, 64, 16, 8)
        a.log_decay = 4096
        for n, x in kw.items():
            setattr(a, n, x)
        return a
    tok = TokensC(4096, 64, 16, 8)
    null = TokensC(None, 64, 16, 8)

    def fwd(a, out=tok, ws=None, n=0):
        return L.ur3e_attn_forward(ctypes.byref(a) if a else None, ctypes.byref(out) if out else None, None, ws, n, None)
    for a in (None, attn(dtype=3), attn(dtype=-1), attn(b=-1), attn(t=-1), attn(heads=0), attn(kv_heads=0),
              attn(heads=3, kv_heads=2), attn(dk=0), attn(dk=129), attn(dv=0), attn(dv=129), attn(log_decay=None),
              attn(q=null), attn(k=null), attn(v=null), attn(b=1 << 22),
              attn(q=TokensC(4096, 64, -16, 8)), attn(starts_st=-1)):
        assert fwd(a) == EINVAL and L.ur3e_last_error()
    assert fwd(attn(), TokensC(4096, 64, -16, 8)) == EINVAL
    assert fwd(attn(), None) == EINVAL and fwd(attn(), null) == EINVAL
    assert fwd(attn(b=0)) == 0
    n = ctypes.c_size_t()
    long = attn(t=10500)
    assert L.ur3e_attn_workspace(ctypes.byref(long), 0, ctypes.byref(n)) == 0 and n.value > 0
    assert fwd(long) == EINVAL and fwd(long, ws=4096, n=n.value - 1) == EINVAL and fwd(long, ws=None, n=n.value) == EINVAL
    assert L.ur3e_attn_workspace(ctypes.byref(long), 0, None) == EINVAL
    r = ctypes.byref
    assert L.ur3e_attn_backward(r(attn()), r(tok), None, r(tok), r(tok), None, None, None, 0, None) == EINVAL
    assert L.ur3e_attn_backward(r(attn()), r(null), None, r(tok), r(tok), r(tok), None, None, 0, None) == EINVAL
    one = attn(t=1)
    assert L.ur3e_attn_step(r(attn()), r(tok), 4096, None, None) == EINVAL
    assert L.ur3e_attn_step(r(one), r(tok), None, None, None) == EINVAL
    assert L.ur3e_attn_step(r(attn(t=1, lengths=4096)), r(tok), 4096, None, None) == EINVAL

    def drop(dtype=0, rows=2, cols=8, x=4096, y=4096, count=100):
        return L.ur3e_keyed_dropout(dtype, rows, cols, x, 8, None, 0, y, 8, None, 1, 0, count, None)
    assert [drop(dtype=3), drop(rows=-1), drop(cols=-1), drop(x=None), drop(y=None), drop(count=-1), drop(count=65537),
            drop(rows=1 << 40)] == [EINVAL] * 8
    assert drop(rows=0) == 0 and drop(cols=0) == 0
