"""GPU: the policy operators (ur3e_amd/rl/ops.py) where their kernels' variants, slabs and splits meet."""
import pytest
import torch

import policy_variants as pv
from test_gpu_policy_ops import DT, check_all, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("b,t", [(2, 40), (300, 20)])
def test_a_value_that_is_not_finite_stays_in_its_slab(b, t, dtype):
    """66 channels leave two for the last slab, fewer than a load of a lane.  A NaN in channel 50 has its slab go token by token; the
    channels from 60 on, which the last slab owns, are rounded as without it, bit for bit: no channel is two slabs'."""
    x, dout, dfinal = make(b, t, 2, 1, 66, 66, DT[dtype], seed=b, starts=0.05, lengths=[t, t - 3] * (b // 2))
    clean = run(x, dout, dfinal)

    def planted(z):
        z = z.clone()
        z[:, 3, :, 50] = float("nan")
        return z
    got = run(dict(x, v=planted(x["v"])), dout, dfinal)
    assert not torch.isfinite(got["out"][:, 3, :, 50]).any()
    for n in ("out", "state"):
        assert torch.equal(got[n][..., 60:], clean[n][..., 60:]), n
    got = run(dict(x, k=planted(x["k"])), dout, dfinal)
    assert torch.equal(got["dq"][..., 60:], clean["dq"][..., 60:])
    got = run(dict(x, q=planted(x["q"])), dout, dfinal)
    assert torch.equal(got["dk"][..., 60:], clean["dk"][..., 60:])
    got = run(x, planted(dout), dfinal)
    for n in ("dv", "ds0"):
        assert torch.equal(got[n][..., 60:], clean[n][..., 60:]), n


def tokens(g, dtype, b, t, h, d):
    return torch.randn((b, t, h, d), device="cuda", generator=g).to(dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("b,h,t,d", [
    (64, 4, 4000, 8),     # a few splits of 500 tokens and more, few elements
    (1, 1, 10500, 16),    # hundreds of splits of one sequence
    (64, 4, 4000, 33),    # a few splits, many elements
])
def test_what_is_not_finite_is_not_lost_between_splits(b, h, t, d, dtype):
    """The decay over a split of 368 tokens of a factor of 3/4, or over 32 shorter ones, is less than any float.  A NaN in the state
    is there behind it all the same, forwards and backwards, up to an episode's start and not past it."""
    g = torch.Generator(device="cuda").manual_seed(t + d)
    cut = t - 700
    x = dict(q=tokens(g, DT[dtype], b, t, h, d), k=tokens(g, DT[dtype], b, t, h, d), v=tokens(g, DT[dtype], b, t, h, d),
             log_decay=torch.full((h,), 0.75, device="cuda").log(), initial_state=torch.zeros((b, h, d, d), device="cuda"),
             starts=None, lengths=None)
    dout = tokens(g, DT[dtype], b, t, h, d)
    dfinal = torch.zeros_like(x["initial_state"])
    starts = torch.zeros((b, t), dtype=torch.bool, device="cuda")
    starts[:, cut] = True

    def nan_at(z, *at):
        z = z.clone()
        z[at] = float("nan")
        return z

    def gone(z):
        return not torch.isfinite(z).any()

    def whole(z):
        return torch.isfinite(z).all()
    # forwards: a value of the first token, and the state in front of it
    for change in (dict(v=nan_at(x["v"], 0, 0, slice(None), 1)),
                   dict(initial_state=nan_at(x["initial_state"], 0, slice(None), 0, 1))):
        got = run({**x, **change}, dout, dfinal)
        assert gone(got["out"][0, :, :, 1]) and whole(got["out"][0, :, :, 2:]) and whole(got["out"][1:])
        assert gone(got["dq"][0, :, :, 0]) and whole(got["dq"][1:]) and whole(got["dk"][:, 1:])
        assert gone(got["state"][0, :, 0, 1]) and whole(got["state"][1:]) and whole(got["state"][0, :, :, 2:])
        got = run({**x, **change, "starts": starts}, dout, dfinal)
        assert gone(got["out"][0, :cut, :, 1]) and whole(got["out"][:, cut:])
        assert gone(got["dq"][0, :cut, :, 0]) and whole(got["dq"][:, cut:]) and whole(got["state"])
    # backwards: the last output's gradient, and the last state's
    starts = starts.roll(700 - cut, 1)
    cut = 700
    for do, df in ((nan_at(dout, 0, t - 1, slice(None), 1), dfinal), (dout, nan_at(dfinal, 0, slice(None), 0, 1))):
        got = run(x, do, df)
        assert gone(got["dv"][0, :, :, 1]) and whole(got["dv"][0, :, :, 2:]) and whole(got["dv"][1:])
        assert gone(got["dk"][0, :, :, 0]) and whole(got["dk"][1:]) and whole(got["dq"][:, :t - 1])
        assert gone(got["ds0"][0, :, 0, 1]) and whole(got["ds0"][1:]) and whole(got["ds0"][0, :, :, 2:])
        got = run(dict(x, starts=starts), do, df)
        assert gone(got["dv"][0, cut:, :, 1]) and whole(got["dv"][:, :cut])
        assert gone(got["dk"][0, cut:, :, 0]) and whole(got["dk"][:, :cut]) and whole(got["ds0"])


def test_forward_mode_is_refused():
    """a tangent that the kernels would drop is refused, in the inputs and in the gradients of a backward pass"""
    import torch.autograd.forward_ad as fwd
    from ur3e_amd.rl import ops
    x, dout, dfinal = make(2, 5, 2, 1, 8, 8, torch.float32, state=True)
    ld = x["log_decay"]
    leaf = x["q"].detach().requires_grad_()
    with fwd.dual_level():
        def dual(z):
            return fwd.make_dual(z, torch.ones_like(z))
        for n in ("q", "k", "v", "initial_state", "log_decay"):
            with pytest.raises(ValueError, match="forward-mode"):
                ops.decay_attention(**dict(x, **{n: dual(x[n])}))
        with pytest.raises(ValueError, match="forward-mode"):
            ops.decay_attention(dual(leaf), x["k"], x["v"], ld)
        with pytest.raises(ValueError, match="forward-mode"):
            ops.decay_attention_step(x["q"][:, 0], x["k"][:, 0], dual(x["v"])[:, 0], ld, x["initial_state"])
        with pytest.raises(ValueError, match="forward-mode"):
            ops.keyed_dropout(dual(x["q"]), 0.5, 1)
        out, _ = ops.decay_attention(leaf, x["k"], x["v"], ld)
        with pytest.raises(ValueError, match="forward-mode"):
            torch.autograd.grad(out, [leaf], dual(dout))
        y = ops.keyed_dropout(leaf, 0.5, 1)
        with pytest.raises(ValueError, match="forward-mode"):
            torch.autograd.grad(y, [leaf], dual(torch.ones_like(y)))
        # switched off, a tangent is nothing to carry
        q = dual(x["q"])
        with fwd._set_fwd_grad_enabled(False):
            off, _ = ops.decay_attention(q, x["k"], x["v"], ld)
        assert torch.equal(off, out)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_exact_over_two_rounds_of_the_join(dtype):
    """More than 512 splits, which the 16 waves of the join take in two rounds.  Without decay, with q, k, v and dout of -1, 0 and 1 and an
    initial state of whole numbers, every sum is a whole number; the states stay below 2^11, exact in any of the kernel's forms,
    and an output is the exact one rounded once."""
    from ur3e_amd.rl import ops
    t, d = 80000, 16
    assert all(pv.splits(1, t, 1, d, d, 2 if dtype != "f32" else 4, False, back)[0] > 512 for back in (False, True))
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v, do = (torch.randint(-1, 2, (t, d), device="cuda", generator=g).double() for _ in range(4))
    s0, df = (torch.randint(-9, 10, (d, d), device="cuda", generator=g).double() for _ in range(2))
    starts = torch.zeros((1, t), dtype=torch.bool, device="cuda")
    ends = [30001, 30002, t]  # of the episodes; the last one runs over both rounds
    starts[0, ends[:-1]] = True
    leaves = [z.to(DT[dtype]).view(1, t, 1, d).requires_grad_() for z in (q, k, v)]
    state0 = s0.float().view(1, 1, d, d).requires_grad_()
    out, state = ops.decay_attention(*leaves, torch.zeros(1, device="cuda"), initial_state=state0, starts=starts, scale=1.0,
                                     return_state=True)
    grads = torch.autograd.grad([out, state], leaves + [state0],
                                [do.to(DT[dtype]).view(1, t, 1, d), df.float().view(1, 1, d, d)])
    want = [torch.empty((t, d), dtype=torch.float64, device="cuda") for _ in range(4)]
    lo = 0
    for hi in ends:
        s = (k[lo:hi, :, None] * v[lo:hi, None, :]).cumsum(0)
        if lo == 0:
            s = s + s0
        gs = (q[lo:hi, :, None] * do[lo:hi, None, :]).flip(0).cumsum(0).flip(0)
        if hi == t:
            gs = gs + df
        if lo == 0:
            gs0 = gs[0]
        want[0][lo:hi] = (q[lo:hi, :, None] * s).sum(1)
        want[1][lo:hi] = (s * do[lo:hi, None, :]).sum(2)
        want[2][lo:hi] = (gs * v[lo:hi, None, :]).sum(2)
        want[3][lo:hi] = (gs * k[lo:hi, :, None]).sum(1)
        assert max(s.abs().max(), gs.abs().max()) < 2 ** 11
        lo = hi
    assert torch.equal(state.double()[0, 0], s[-1]) and torch.equal(grads[3].double()[0, 0], gs0)
    for got, e in zip((out, *grads[:3]), want):
        assert torch.equal(got.detach()[0, :, 0], e.float().to(DT[dtype]))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("t,far", [(40, "tokens"), (200, "tokens"), (40, "starts")])
def test_tokens_far_apart_one_by_one(t, far, dtype):
    """Tokens (or starts) so far apart that 16 of them are past the 2^30 bytes of an offset are taken one by one: both directions, with
    starts, padding, an initial state and, at 200, several splits"""
    size = 4 if dtype == "f32" else 2
    step = (1 << 26) // size + 64 if far == "tokens" else (1 << 25) + 8
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    x, dout, dfinal = make(2, t, 4, 2, 20, 24, DT[dtype], seed=t, starts=0.05, lengths=[t, t - 9])
    if far == "tokens":
        assert pv.splits(2, t, 4, 20, 24, size, True, False)[0] == (1 if t == 40 else pv.splits(2, t, 4, 20, 24, size, True, True)[0])
        buf = torch.empty(step * (t - 1) + 2 * 1024, dtype=DT[dtype], device="cuda")
        at = 0
        for n in ("q", "k", "v"):
            b, _, h, d = x[n].shape
            y = buf.as_strided((b, t, h, d), (h * d, step, d, 1), at)
            at += b * h * d
            y.copy_(x[n])
            x[n] = y
        assert at <= 2 * 1024
    else:
        y = torch.empty(step * (t - 1) + 8, dtype=torch.bool, device="cuda").as_strided((2, t), (1, step))
        y.copy_(x["starts"])
        x["starts"] = y
    check_all(x, dout, dfinal)
