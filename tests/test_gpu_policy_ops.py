"""GPU: the policy operators (ur3e_amd/rl/ops.py) against their definitions in 64 bits, within the error that
rounding allows (tests/policy_ref.py), at the sizes and masks where they can go wrong."""
import numpy as np
import pytest
import torch

import policy_ref as ref

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def rand(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g).to(dtype)


def make(b, t, h, hk, dk, dv, dtype, seed=0, starts=0.0, lengths=None, state=True, time_major=False, decay=None):
    """inputs on the GPU (made on the CPU), and dout / dfinal"""
    g = torch.Generator().manual_seed(seed)

    def tok(heads, d):
        x = rand(g, b, t, heads, d, dtype=dtype)
        return x.transpose(0, 1).contiguous().cuda().transpose(0, 1) if time_major else x.cuda()
    x = dict(q=tok(h, dk), k=tok(hk, dk), v=tok(hk, dv),
             log_decay=(torch.log(torch.linspace(0.6, 0.998, h)) if decay is None else torch.tensor(decay)).cuda(),
             initial_state=rand(g, b, h, dk, dv).cuda() if state else None,
             starts=(torch.rand((b, t), generator=g) < starts).cuda() if starts else None,
             lengths=None if lengths is None else torch.tensor(lengths, dtype=torch.int32).cuda())
    return x, tok(h, dv), rand(g, b, h, dk, dv).cuda()


def run(x, dout, dfinal, **kw):
    from ur3e_amd.rl import ops
    names = [n for n in ("q", "k", "v", "initial_state") if x[n] is not None]
    leaves = {n: x[n].detach().requires_grad_() for n in names}
    out, state = ops.decay_attention(**{**x, **leaves}, return_state=True, **kw)
    grads = torch.autograd.grad([out, state], list(leaves.values()), [dout, dfinal])
    return dict(out=out, state=state, **{{"q": "dq", "k": "dk", "v": "dv", "initial_state": "ds0"}[n]: gr
                                         for n, gr in zip(names, grads)})


def check_all(x, dout, dfinal, got=None, scale=None):
    got = run(x, dout, dfinal) if got is None else got
    b, t, h, dk = x["q"].shape
    a = (x["q"], x["k"], x["v"], x["log_decay"], x["initial_state"], x["starts"], x["lengths"],
         dk ** -0.5 if scale is None else scale, dout, dfinal)
    e, m = ref.attention(*a), ref.attention(*a, magnitude=True)
    n = ref.roundings(t, dk, x["v"].shape[3], x["log_decay"].cpu(), h // x["k"].shape[2])
    for name, y in got.items():
        ref.check(y, e[name], m[name], n, name)
    return got


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("b,t,h,hk,dk,dv", [
    (1, 1, 1, 1, 1, 1), (2, 2, 2, 1, 3, 5), (3, 15, 4, 4, 16, 16), (2, 16, 4, 2, 32, 32), (5, 17, 4, 4, 64, 64),
    (1, 33, 6, 2, 40, 72), (2, 50, 2, 2, 128, 128), (1, 47, 2, 1, 127, 65), (2, 31, 3, 3, 8, 128), (2, 31, 3, 3, 128, 8),
    (1, 64, 2, 2, 17, 33), (1, 300, 2, 2, 64, 64), (2, 531, 2, 1, 24, 48)])
def test_attention_sizes(b, t, h, hk, dk, dv, dtype):
    """every tile width, whole and ragged chunks of 16, one to several waves along a sequence (t >= 256)"""
    check_all(*make(b, t, h, hk, dk, dv, DT[dtype], seed=t))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("first", range(1, 129, 8))
def test_attention_every_channel_count(first, dtype):
    """keys and values of 1 to 128 channels, each with another partner: rows that end anywhere in a lane's load"""
    for d in range(first, first + 8):
        dv = (d * 37) % 128 + 1
        check_all(*make(1, 19, 2, 1, d, dv, DT[dtype], seed=d))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dk,dv", [(2, 3), (3, 66), (66, 1), (3, 3), (100, 70), (45, 45)])
def test_attention_odd_rows_in_splits(dk, dv, dtype):
    """rows of less than four channels and rows that fill no tile, over several waves a sequence, ragged, with starts"""
    check_all(*make(3, 400, 4, 2, dk, dv, DT[dtype], seed=dk, starts=0.02, lengths=[400, 0, 333]))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("t,starts,time_major", [(16, 0.3, True), (37, 0.1, False), (40, 1.0, True), (400, 0.02, False),
                                                 (400, 0.5, True)])
def test_attention_starts_and_lengths(t, starts, time_major, dtype):
    b = 5
    lengths = [t, 0, 1, t - 1, t // 2]
    x, dout, dfinal = make(b, t, 4, 2, 32, 48, DT[dtype], seed=7, starts=starts, lengths=lengths, time_major=time_major)
    x["starts"][0, 0] = True
    x["starts"][3, 0] = False
    got = check_all(x, dout, dfinal)
    assert got["out"][1].abs().max() == 0 and got["dk"][2, 1:].abs().max() == 0
    assert torch.equal(got["state"][1], x["initial_state"][1])
    assert torch.equal(got["ds0"][1], dfinal[1])
    assert got["ds0"][0].abs().max() == 0
    x["starts"] = x["starts"].to(torch.uint8) * 3
    again = run(x, dout, dfinal)
    assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("t,dk,dv", [(1500, 16, 16), (1700, 33, 20)])
def test_attention_many_splits_of_one_sequence(t, dk, dv):
    """more than 32 splits: the join's waves hand the state on to each other, through decays and starts"""
    check_all(*make(1, t, 1, 1, dk, dv, torch.float32, seed=t, starts=0.004, decay=[-0.002]))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_attention_exact_over_hundreds_of_splits(dtype):
    """more than 512 splits, two rounds of the join.  Without decay and with values of -1, 0 and 1 every sum is a whole number:
    the state stays below 2^11 (three are drawn, so it is a walk of 0.67 sqrt(t) = 180 on average), exact in any of the kernel's
    forms, and so do the outputs in float; a 16-bit output is the exact one rounded once."""
    from ur3e_amd.rl import ops
    t, d = 70000, 16
    g = torch.Generator().manual_seed(1)
    q, k, v, do = (torch.randint(-1, 2, (1, t, 1, d), generator=g).float() for _ in range(4))
    starts = torch.zeros((1, t), dtype=torch.bool)
    starts[0, [0, 30001, 30002]] = True
    leaves = [z.to(DT[dtype]).cuda().requires_grad_() for z in (q, k, v)]
    s0 = torch.full((1, 1, d, d), float("nan"), device="cuda")
    out, state = ops.decay_attention(*leaves, torch.zeros(1, device="cuda"), initial_state=s0, starts=starts.cuda(), scale=1.0,
                                     return_state=True)
    grads = torch.autograd.grad(out, leaves, do.to(DT[dtype]).cuda())
    q, k, v, do = (z[0, :, 0].double() for z in (q, k, v, do))
    segs = [(0, 30001), (30001, 30002), (30002, t)]
    eo, eq, ek, ev = (torch.zeros(t, d, dtype=torch.float64) for _ in range(4))
    for lo, hi in segs:
        s = (k[lo:hi, :, None] * v[lo:hi, None, :]).cumsum(0)
        gs = (q[lo:hi, :, None] * do[lo:hi, None, :]).flip(0).cumsum(0).flip(0)
        eo[lo:hi] = (q[lo:hi, :, None] * s).sum(1)
        eq[lo:hi] = (s * do[lo:hi, None, :]).sum(2)
        ek[lo:hi] = (gs * v[lo:hi, None, :]).sum(2)
        ev[lo:hi] = (gs * k[lo:hi, :, None]).sum(1)
        assert max(s.abs().max(), gs.abs().max()) < 2 ** 11
    assert torch.equal(state.cpu().double()[0, 0], s[-1])
    for got, e in zip((out, *grads), (eo, eq, ek, ev)):
        assert torch.equal(got.detach().cpu()[0, :, 0], e.float().to(DT[dtype]))


@pytest.mark.parametrize("small", ["q", "k", "v"])
@pytest.mark.parametrize("t", [16, 300])
def test_attention_half_below_its_normal_range(small, t):
    """one operand's elements lie below 2^-14, where half has fewer bits, but has them: nothing is taken for zero.  The others
    are of the size that keeps sums of 300 products below 2^16."""
    x, dout, dfinal = make(1, t, 2, 2, 32, 32, torch.float16, seed=t, decay=[-0.1, -0.5])
    size = {n: 2.0 ** 4 for n in ("q", "k", "v")}
    size[small] = 2.0 ** -17
    for n, f in size.items():
        x[n] = (x[n].float() * f).half()
    x["initial_state"] *= size["k"] * size["v"]
    got = check_all(x, dout, dfinal)
    assert got["out"].abs().max() > 2.0 ** -12 and got["d" + small].abs().max() > 1.0


def test_attention_lengths_are_clamped():
    x, dout, dfinal = make(3, 20, 2, 2, 16, 16, torch.float32, lengths=[-5, 99, 20])
    got = run(x, dout, dfinal)
    y = dict(x, lengths=torch.tensor([0, 20, 20], dtype=torch.int32).cuda())
    want = run(y, dout, dfinal)
    assert all(torch.equal(got[n], want[n]) for n in got)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_attention_decay_ends(dtype):
    """exp(log_decay) = 0 keeps the token alone, 1 never forgets, and 1 - 2^-12 forgets slowly"""
    x, dout, dfinal = make(2, 300, 3, 3, 32, 32, DT[dtype], decay=[float("-inf"), 0.0, -2.0 ** -12])
    got = check_all(x, dout, dfinal)
    s = x["q"].shape[-1] ** -0.5
    alone = (x["q"][:, :, 0].double() * x["k"][:, :, 0].double()).sum(-1, keepdim=True) * s * x["v"][:, :, 0].double()
    scale = (x["q"][:, :, 0].double() * x["k"][:, :, 0].double()).abs().sum(-1, keepdim=True) * s * x["v"][:, :, 0].double().abs()
    ref.check(got["out"][:, :, 0], alone.cpu(), scale.cpu(), 64, "alone")


@pytest.mark.parametrize("t", [32, 300])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_attention_what_masks_hide_stays_hidden(t, dtype, value):
    """padding, the tokens and the state in front of a start, and later tokens never reach a token, whatever they hold"""
    x, dout, dfinal = make(2, t, 2, 2, 32, 32, DT[dtype], lengths=[t, t - 5], starts=0.0)
    cut = t - 13  # inside a chunk of 16
    starts = torch.zeros((2, t), dtype=torch.bool, device="cuda")
    starts[:, cut] = True
    x["starts"] = starts
    clean = check_all(x, dout, dfinal)
    a = (x["q"], x["k"], x["v"], x["log_decay"], x["initial_state"], x["starts"], x["lengths"], 32 ** -0.5, dout, dfinal)
    e, m = ref.attention(*a), ref.attention(*a, magnitude=True)
    n = ref.roundings(t, 32, 32, x["log_decay"].cpu())
    # in front of the start
    y = {name: z.clone() for name, z in x.items()}
    for z in ("q", "k", "v"):
        y[z][:, cut - 1] = value
        y[z][:, 3, 0, 1] = value
    y["initial_state"][:, 0, 2, 3] = value
    d2 = dout.clone()
    d2[:, cut - 1] = value
    got = run(y, d2, dfinal)
    for z in ("out", "dq", "dk", "dv"):
        ref.check(got[z][:, cut:], e[z][:, cut:], m[z][:, cut:], n, z)
    ref.check(got["state"], e["state"], m["state"], n, "state")
    # padding of the second sequence
    y = {name: z.clone() for name, z in x.items()}
    d2 = dout.clone()
    for z in (y["q"], y["k"], y["v"], d2):
        z[1, t - 5:] = value
    got = run(y, d2, dfinal)
    for z in got:
        assert torch.equal(got[z], clean[z]), z
    # a later token: outputs in front of it
    y = {name: z.clone() for name, z in x.items()}
    for z in ("q", "k", "v"):
        y[z][:, 9] = value
    got = run(y, dout, dfinal)
    ref.check(got["out"][:, :9], e["out"][:, :9], m["out"][:, :9], n, "in front of a later token")
    assert not torch.isfinite(got["out"][:, 9]).any()


def test_attention_strides():
    """views of a fused projection (offset, unaligned), keys shared by all heads through an expanded view, channels
    that are not contiguous, and expanded output gradients"""
    from ur3e_amd.rl import ops
    g = torch.Generator().manual_seed(0)
    b, t, h, d = 3, 35, 4, 20
    qkv = rand(g, t, b, h * 3 * d + 3).cuda()
    parts = [qkv[..., i * h * d + 1:(i + 1) * h * d + 1].unflatten(-1, (h, d)).transpose(0, 1) for i in range(3)]
    ld = torch.log(torch.linspace(0.5, 0.9, h)).cuda()
    x = dict(q=parts[0], k=parts[1], v=parts[2], log_decay=ld, initial_state=None, starts=None, lengths=None)
    got = run(x, rand(g, b, t, h, d).cuda(), rand(g, b, h, d, d).cuda())
    y = {n: z.contiguous() if torch.is_tensor(z) else z for n, z in x.items()}
    g = torch.Generator().manual_seed(0)
    rand(g, t, b, h * 3 * d + 3)
    want = check_all(y, rand(g, b, t, h, d).cuda(), rand(g, b, h, d, d).cuda())
    for n in want:
        torch.testing.assert_close(got[n], want[n], rtol=1e-5, atol=1e-5)
    # one key for all heads
    k1 = rand(g, b, t, 1, d).cuda().requires_grad_()
    v = rand(g, b, t, h, d).cuda()
    out, _ = ops.decay_attention(parts[0], k1.expand(-1, -1, h, -1), v, ld)
    dk, = torch.autograd.grad(out.sum(), [k1])
    e = [ref.attention(parts[0], k1.expand(-1, -1, h, -1), v, ld, scale=d ** -0.5, dout=torch.ones(b, t, h, d), magnitude=i)
         for i in (False, True)]
    n = ref.roundings(t, d, d, ld.cpu(), h)
    ref.check(out, e[0]["out"], e[1]["out"], n, "expanded k")
    ref.check(dk, e[0]["dk"].sum(2, keepdim=True), e[1]["dk"].sum(2, keepdim=True), n, "expanded dk")
    # channels in the slow dimension
    q2 = parts[0].contiguous().transpose(2, 3).contiguous().transpose(2, 3)
    assert q2.stride(-1) != 1
    out2, _ = ops.decay_attention(q2, k1.expand(-1, -1, h, -1), v, ld)
    torch.testing.assert_close(out2, out, rtol=1e-5, atol=1e-5)


def test_attention_offsets_past_32_bits():
    """tokens that lie 2^29 elements apart: byte and element offsets past 32 bits"""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    g = torch.Generator().manual_seed(0)
    step, t = 1 << 29, 10
    buf = torch.empty(step * (t - 1) + 64, dtype=torch.bfloat16, device="cuda")
    q, k, v = (buf.as_strided((1, t, 1, 16), (0, step, 16, 1), 16 * i) for i in range(3))
    small = [rand(g, 1, t, 1, 16, dtype=torch.bfloat16).cuda() for _ in range(3)]
    for a, s in zip((q, k, v), small):
        a.copy_(s)
    from ur3e_amd.rl import ops
    ld = torch.tensor([-0.1], device="cuda")
    # such tokens are taken one by one, so the sums run in another order than for the small tensors: each side
    # is held to the definition, not to the other's bits
    e, m = (ref.attention(*small, ld, scale=0.25, magnitude=i) for i in (False, True))
    n = ref.roundings(t, 16, 16, ld.cpu())
    for args in ((q, k, v), small):
        for got, name in zip(ops.decay_attention(*args, ld, return_state=True), ("out", "state")):
            ref.check(got, e[name], m[name], n, name)


def test_attention_differences():
    """the output is linear in each of q, k, v and the state, so a difference of any size is the gradient's"""
    x, dout, dfinal = make(2, 45, 4, 2, 24, 40, torch.float32, starts=0.1, lengths=[45, 30])
    base = run(x, dout, dfinal)

    def loss(y):
        from ur3e_amd.rl import ops
        o, s = ops.decay_attention(**y, return_state=True)
        return (o.double() * dout.double()).sum() + (s.double() * dfinal.double()).sum()
    l0 = loss(x)
    g = torch.Generator().manual_seed(9)
    for n, dn in (("q", "dq"), ("k", "dk"), ("v", "dv"), ("initial_state", "ds0")):
        d = rand(g, *x[n].shape).cuda()
        diff = loss(dict(x, **{n: x[n] + d})) - l0
        lin = (base[dn].double() * d.double()).sum()
        size = (base[dn].double() * d.double()).abs().sum() + l0.abs()
        # ~1e2 roundings of 2^-24 in every value, and the sum x + d rounded once
        assert (diff - lin).abs() <= 300 * 2.0 ** -24 * size * 10, (n, diff.item(), lin.item())


def test_attention_repeats_bit_for_bit():
    x, dout, dfinal = make(3, 777, 6, 2, 48, 96, torch.bfloat16, starts=0.02, lengths=[777, 500, 3])
    a, b = run(x, dout, dfinal), run(x, dout, dfinal)
    assert all(torch.equal(a[n], b[n]) for n in a)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("b,h,hk,dk,dv", [(1, 1, 1, 1, 1), (1, 4, 4, 64, 64), (5, 6, 2, 40, 72), (3, 2, 1, 127, 65), (7, 3, 3, 128, 128),
                                          (2, 4, 4, 16, 6)])
def test_step(b, h, hk, dk, dv, dtype):
    from ur3e_amd.rl import ops
    t = 4
    x, _, _ = make(b, t, h, hk, dk, dv, DT[dtype], starts=0.3, time_major=True)
    x["starts"][:, 0] = False
    a = (x["q"], x["k"], x["v"], x["log_decay"], x["initial_state"], x["starts"], None, dk ** -0.5)
    e, m = ref.attention(*a), ref.attention(*a, magnitude=True)
    n = ref.roundings(t, dk, dv, x["log_decay"].cpu())
    s = x["initial_state"].clone()
    for i in range(t):
        args = (x["q"][:, i], x["k"][:, i], x["v"][:, i], x["log_decay"])
        before = s.clone()
        look = ops.decay_attention_step(*args, s, starts=x["starts"][:, i], update=False)
        nxt = torch.full_like(s, float("nan"))
        other = ops.decay_attention_step(*args, s, starts=x["starts"][:, i], next_state=nxt)
        assert torch.equal(s, before)
        o = ops.decay_attention_step(*args, s, starts=x["starts"][:, i])
        assert torch.equal(o, look) and torch.equal(o, other) and torch.equal(s, nxt)
        ref.check(o, e["out"][:, i], m["out"][:, i], n, f"out {i}")
    ref.check(s, e["state"], m["state"], n, "state")


def test_step_start_drops_what_is_not_finite():
    from ur3e_amd.rl import ops
    s = torch.full((2, 1, 8, 8), float("nan"), device="cuda")
    s[1] = 1.0
    q, k, v = (torch.ones((2, 1, 8), device="cuda") for _ in range(3))
    starts = torch.tensor([True, False], device="cuda")
    o = ops.decay_attention_step(q, k, v, torch.zeros(1, device="cuda"), s, starts=starts, scale=1.0)
    assert torch.equal(o, torch.tensor([8.0, 16.0], device="cuda").view(2, 1, 1).expand(2, 1, 8))
    assert torch.equal(s[0], torch.ones((1, 8, 8), device="cuda"))


def test_streams_and_graphs():
    """on a side stream, and captured (forward and backward) into two graphs replayed in turn with eager work between
    them, each replay equal to the eager result on the same inputs"""
    shapes = [(2, 700, 4, 2, 64, 64), (3, 20, 2, 2, 32, 32)]
    cases = [make(*s, torch.float32, seed=i, starts=0.01) for i, s in enumerate(shapes)]
    eager = [run(*c) for c in cases]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = [run(*c) for c in cases]
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(eager, on_side):
        assert all(torch.equal(a[n], b[n]) for n in a)
    graphs, outs = [], []
    for c in cases:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(run(*c))
        graphs.append(gr)
    for r in range(4):
        for i, (x, dout, dfinal) in enumerate(cases):
            x["q"].copy_(x["q"].roll(1, 0) * 0.9)
            want = run(x, dout, dfinal)
            graphs[i].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(want[n], outs[i][n]) for n in want), (r, i)


def test_capture_refuses_leaves_of_a_live_eager_graph():
    """a captured backward pass cannot reach leaves whose gradients belong to an eager graph of the default stream"""
    from ur3e_amd.rl import ops
    w = torch.randn((8, 24), device="cuda", requires_grad=True)
    x = torch.randn((2, 5, 8), device="cuda")
    ld = torch.zeros(2, device="cuda")

    def loss():
        q, k, v = (x @ w).unflatten(-1, (3, 2, 4)).unbind(-3)
        return ops.keyed_dropout(ops.decay_attention(q, k, v, ld)[0].flatten(-2), 0.5, 1).sum()

    def drop():
        return ops.keyed_dropout(x @ w, 0.5, 1)
    for f in (loss, drop):
        alive = f()
        gr = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="eager graph"):
            with torch.cuda.graph(gr):
                f()
        gr = torch.cuda.CUDAGraph()
        with torch.no_grad(), torch.cuda.graph(gr):  # the forward pass alone is free
            y = f()
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, alive.detach())
        del alive, y, gr
    want, = torch.autograd.grad(loss(), [w])
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got, = torch.autograd.grad(loss(), [w])
    for _ in range(3):
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_nothing_to_do(dtype):
    """no sequences, no tokens, no rows, no columns"""
    from ur3e_amd.rl import ops
    for b, t, h, hk, dk, dv in ((0, 5, 4, 2, 8, 2), (3, 0, 4, 2, 8, 2), (0, 0, 2, 2, 64, 64), (3, 0, 2, 2, 64, 64)):
        x, dout, dfinal = make(b, t, h, hk, dk, dv, DT[dtype], starts=0.5, lengths=[0] * b)
        got = run(x, dout, dfinal)
        assert torch.equal(got["state"], x["initial_state"]) and torch.equal(got["ds0"], dfinal)
        assert all(got[n].shape == y.shape for n, y in (("out", dout), ("dq", x["q"]), ("dk", x["k"]), ("dv", x["v"])))
        x, dout, dfinal = make(b, t, h, hk, dk, dv, DT[dtype], state=False)
        assert run(x, dout, dfinal)["state"].abs().sum() == 0
    s = torch.zeros((0, 2, 8, 8), device="cuda")
    q = torch.zeros((0, 2, 8), device="cuda", dtype=DT[dtype])
    assert ops.decay_attention_step(q, q, q, torch.zeros(2, device="cuda"), s).shape == (0, 2, 8)
    for shape in ((0, 8), (8, 0), (2, 3, 0), (0, 2, 8), (0,), (0, 0)):
        z = torch.zeros(shape, device="cuda", dtype=DT[dtype], requires_grad=True)
        y = ops.keyed_dropout(z, 0.5, 1, residual=z)
        g, = torch.autograd.grad(y.sum(), [z])
        assert y.shape == g.shape == z.shape


def test_two_calls_at_once():
    """calls on two streams that overlap on the card share nothing"""
    cases = [make(2, 3000, 4, 4, 64, 64, torch.bfloat16, seed=i, starts=0.001) for i in range(2)]
    want = [run(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(run(*cases[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(g[n], want[i][n]) for n in g)


def test_differentiable_once_and_too_large():
    from ur3e_amd.rl import ops
    x, dout, _ = make(1, 4, 1, 1, 8, 8, torch.float32, state=False)
    q = x["q"].requires_grad_()
    out, _ = ops.decay_attention(q, x["k"], x["v"], x["log_decay"])
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(out, [q], dout, create_graph=True)
    y = ops.keyed_dropout(q, 0.5, 1)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(y, [q], torch.ones_like(y), create_graph=True)
    big = torch.zeros((1, 1, 1, 8), device="cuda").expand(1 << 22, 1, 1, 8)
    with pytest.raises(ValueError, match="2\\^22"):
        ops.decay_attention(big, big, big, x["log_decay"])


def test_gradients_of_some_inputs():
    """a gradient is the same whichever of the others are asked for, and an unused output counts as zero"""
    from ur3e_amd.rl import ops
    x, dout, dfinal = make(2, 40, 4, 2, 24, 40, torch.float32)
    full = run(x, dout, dfinal)
    for n, dn in (("q", "dq"), ("k", "dk"), ("v", "dv"), ("initial_state", "ds0")):
        leaf = x[n].detach().requires_grad_()
        out, state = ops.decay_attention(**{**x, n: leaf}, return_state=True)
        g, = torch.autograd.grad([out, state], [leaf], [dout, dfinal])
        assert torch.equal(g, full[dn])
        g1, = torch.autograd.grad(ops.decay_attention(**{**x, n: leaf}, return_state=True)[0], [leaf], dout)
        g2, = torch.autograd.grad(ops.decay_attention(**{**x, n: leaf}, return_state=True)[1], [leaf], dfinal, allow_unused=True)
        size = full[dn].abs().max()
        assert (g1 + (0 if g2 is None else g2) - g).abs().max() <= 64 * 2.0 ** -24 * size * 40


# -- keyed dropout -----------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("r,c", [(1, 1), (3, 7), (5, 8), (19, 9), (6, 15), (4, 256), (129, 101), (7, 1024)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.73, 1.0])
def test_dropout(r, c, p, dtype):
    from ur3e_amd.rl import ops
    g = torch.Generator().manual_seed(r)
    x, res, dy = (rand(g, r, c, dtype=DT[dtype]).cuda() for _ in range(3))
    rows = torch.randint(-2 ** 62, 2 ** 62, (r,), generator=g)
    rows[-1] = rows[0]
    seed, sub = 0xFEDCBA9876543210, 0xABCDEF01
    count = ops.keep_count(p)
    keep = torch.from_numpy(ref.philox(seed, rows.numpy(), c, sub) < count)
    up = 65536 / count if count else 0.0
    xl, rl = x.detach().requires_grad_(), res.detach().requires_grad_()
    xd, rd, dyd = (z.cpu().double() for z in (x, res, dy))

    def kept(z):
        return torch.where(keep, z * up, torch.zeros((), dtype=torch.float64))
    for residual in (None, rl):
        y = ops.keyed_dropout(xl, p, seed, rows.cuda(), sub, residual=residual)
        gr = torch.autograd.grad(y, [xl] if residual is None else [xl, rl], dy)
        e = kept(xd) + (0 if residual is None else rd)
        ref.check(y, e, kept(xd.abs()) + (0 if residual is None else rd.abs()), 3, "y")
        ref.check(gr[0], kept(dyd), kept(dyd.abs()), 3, "dx")
        if residual is not None:
            assert torch.equal(gr[1], dy)
    if p == 1.0:
        assert torch.equal(ops.keyed_dropout(torch.full_like(x, float("nan")), p, seed), torch.zeros_like(x))


def test_dropout_rows_strides_and_default_ids():
    from ur3e_amd.rl import ops
    g = torch.Generator().manual_seed(0)
    x = rand(g, 64, 40).cuda()
    y = ops.keyed_dropout(x, 0.4, 99)
    perm = torch.randperm(64, generator=g).cuda()
    assert torch.equal(ops.keyed_dropout(x[perm], 0.4, 99, perm), y[perm])
    assert torch.equal(ops.keyed_dropout(x.view(8, 8, 40), 0.4, 99), y.view(8, 8, 40))
    wide = rand(g, 64, 60).cuda()
    for view in (wide[:, 1:41], wide[:, 4:44], wide.t().contiguous().t()[:, 3:43]):
        assert torch.equal(ops.keyed_dropout(view, 0.4, 99, residual=view), ops.keyed_dropout(view.contiguous(), 0.4, 99, residual=view.contiguous()))
    xl = x.detach().requires_grad_()
    gs, = torch.autograd.grad(ops.keyed_dropout(xl, 0.4, 99).sum(), [xl])  # an expanded gradient
    assert torch.equal(gs != 0, torch.from_numpy(ref.philox(99, np.arange(64), 40) < ops.keep_count(0.4)).cuda())


def test_dropout_graph():
    from ur3e_amd.rl import ops
    x = torch.randn((300, 72), device="cuda")
    rows = torch.arange(300, device="cuda")
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        y = ops.keyed_dropout(x, 0.3, 5, rows)
    for i in range(4):
        x.normal_()
        rows += 300
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.keyed_dropout(x, 0.3, 5, rows))
