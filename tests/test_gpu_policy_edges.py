"""GPU: the policy operators (ur3e_amd/rl/ops.py) where their kernels' variants, slabs and splits meet."""
import pytest
import torch

from test_gpu_policy_ops import DT, make, run

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
