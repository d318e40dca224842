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
