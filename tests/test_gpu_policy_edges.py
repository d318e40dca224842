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
