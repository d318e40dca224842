"""The policy operators (ur3e_amd/rl/ops.py) without a GPU: derivatives and padding where they can go wrong."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from ur3e_amd.rl import ops

from test_policy_ops_cpu import make


def test_forward_mode_is_refused_before_a_launch():
    """The binding refuses tensors with a tangent, which the kernels would drop, before it looks for a GPU."""
    c = ops._c()
    x = make(2, 3, 2, 1, 4, 5)
    q, k, v, s = (x[n] for n in ("q", "k", "v", "initial_state"))
    ld = x["log_decay"]
    with fwd.dual_level():
        def dual(z):
            return fwd.make_dual(z, torch.ones_like(z))
        for a in ((dual(q), k, v, s), (q, dual(k), v, s), (q, k, dual(v), s), (q, k, v, dual(s))):
            with pytest.raises(ValueError, match="forward-mode"):
                c.decay_attention(*a[:3], ld, a[3], None, None, 1.0, True)
            with pytest.raises(ValueError, match="forward-mode"):
                c.decay_attention_step(*(z[:, 0] for z in a[:3]), ld, a[3], None, 1.0, None, True)
        with pytest.raises(ValueError, match="forward-mode"):
            c.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s, None, 1.0, dual(s), True)
        for a in ((dual(q), None), (q, dual(q))):
            with pytest.raises(ValueError, match="forward-mode"):
                c.keyed_dropout(a[0], 100, 1, None, 0, a[1])
        # a constant, on the CPU as well
        with pytest.raises(ValueError, match="log_decay"):
            ops.decay_attention(q, k, v, dual(ld))
        # the CPU path carries the rest: the output is linear in v
        out, _ = ops.decay_attention(q, k, dual(v), ld)
        lin, _ = ops.decay_attention(q, k, torch.ones_like(v), ld)
        torch.testing.assert_close(fwd.unpack_dual(out).tangent, lin)


def grads_of(x, dout, dfinal):
    names = ("q", "k", "v", "initial_state")
    leaves = {n: x[n].detach().requires_grad_() for n in names}
    out, state = ops.decay_attention(**{**x, **leaves}, return_state=True)
    return dict(zip(("out", "state", "dq", "dk", "dv", "ds0"),
                    (out, state, *torch.autograd.grad([out, state], list(leaves.values()), [dout, dfinal]))))


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_padding_is_not_read(value):
    """whatever the padding and its output gradients hold: the same outputs and gradients, and zeros for the padding"""
    x = make(3, 9, 4, 2, 6, 5, starts=0.2)
    x["lengths"] = torch.tensor([9, 4, 0], dtype=torch.int32)
    g = torch.Generator().manual_seed(2)
    dout, dfinal = torch.randn((3, 9, 4, 5), generator=g), torch.randn((3, 4, 6, 5), generator=g)
    clean = grads_of(x, dout, dfinal)
    y = {n: z.clone() for n, z in x.items()}
    d2 = dout.clone()
    for z in (y["q"], y["k"], y["v"], d2):
        z[1, 4:] = value
        z[2] = value
    y["starts"][1, 4:] = True
    y["starts"][2] = True
    got = grads_of(y, d2, dfinal)
    for n, z in got.items():
        assert torch.equal(z, clean[n]), n
    for n in ("out", "dq", "dk", "dv"):
        assert got[n][1, 4:].abs().max() == 0 and got[n][2].abs().max() == 0


def test_what_starts_hide_has_no_gradient_of_what_is_behind():
    """values that are not finite in front of a start, and behind it: each side's results are as without them"""
    x = make(2, 8, 2, 2, 4, 4)
    x["starts"] = torch.zeros((2, 8), dtype=torch.bool)
    x["starts"][:, 5] = True
    g = torch.Generator().manual_seed(3)
    dout, dfinal = torch.randn((2, 8, 2, 4), generator=g), torch.randn((2, 2, 4, 4), generator=g)
    clean = grads_of(x, dout, dfinal)
    for token, side in ((2, slice(5, 8)), (6, slice(0, 5))):
        y = {n: z.clone() if torch.is_tensor(z) else z for n, z in x.items()}
        d2 = dout.clone()
        for z in (y["q"], y["k"], y["v"], d2):
            z[:, token] = float("nan")
        got = grads_of(y, d2, dfinal)
        for n in ("out", "dq", "dk", "dv"):
            assert torch.equal(got[n][:, side], clean[n][:, side]), (token, n)
        hidden = "state" if token == 2 else "ds0"
        assert torch.equal(got[hidden], clean[hidden])


def test_no_tokens_return_a_state_of_their_own():
    x = make(3, 0, 2, 1, 4, 3)
    _, state = ops.decay_attention(**x, return_state=True)
    assert torch.equal(state, x["initial_state"])
    state.zero_()
    assert x["initial_state"].abs().max() > 0


def test_philox_known_answers_of_any_block():
    """Random123's kat_vectors for philox4x32 with 10 rounds: counters and keys of ones, and of pi's digits"""
    for first, row, sub, seed, want in (
            (0, 0, 0, 0, "6627e8d5 e169c58d bc57ac4c 9b00dbd8"),
            (0xffffffff, -1, 0xffffffff, (1 << 64) - 1, "408f276d 41c83b0e a20bc7c6 6d5451fd"),
            (0x243f6a88, 0x13198a2e85a308d3, 0x03707344, 0x299f31d0a4093822, "d16cfe09 94fdcceb 5001e420 24126ea1")):
        words = ops._philox_cpu(seed, torch.tensor([row]), 1, sub, first=first)[0, 0].tolist()
        assert [f"{w:08x}" for w in words] == want.split()
