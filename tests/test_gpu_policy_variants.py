"""GPU: every kernel that decay_attention can launch (tests/policy_variants.py) against the definition in 64 bits, computed on the
GPU token after token."""
import pytest
import torch

import policy_ref as ref
import policy_variants as pv
from test_gpu_policy_ops import DT, run

pytestmark = pytest.mark.gpu


def definition(x, dout, dfinal, scale, magnitude):
    """the sums of policy_ref.attention, by products of 64-bit matrices"""
    def c(z):
        z = z.detach().double()
        return (z.abs() if magnitude else z).transpose(0, 1).contiguous()  # time in front
    q, k, v, do = (c(z) for z in (x["q"], x["k"], x["v"], dout))
    t, b, h, dk = q.shape
    hk, dv = k.shape[2], v.shape[3]
    grp = h // hk
    here = (torch.arange(t, device="cuda")[:, None] < x["lengths"]).double()[:, :, None, None]
    q, k, v, do = q * here, k * here, v * here, do * here
    kw, vw = k.repeat_interleave(grp, 2), v.repeat_interleave(grp, 2)
    a = torch.exp(x["log_decay"].double()) * torch.where(x["starts"].t(), 0.0, 1.0)[:, :, None]
    a = torch.where(here[:, :, :, 0] > 0, a, 1.0)[..., None, None]
    s = torch.zeros((b, h, dk, dv), dtype=torch.float64, device="cuda")
    if x["initial_state"] is not None:
        s = s + (x["initial_state"].double().abs() if magnitude else x["initial_state"].double())
    out = torch.empty((t, b, h, dv), dtype=torch.float64, device="cuda")
    dq, dkk, dvv = torch.empty_like(q), torch.empty_like(kw), torch.empty_like(vw)
    for i in range(t):
        s = a[i] * s + kw[i, :, :, :, None] * vw[i, :, :, None, :]
        out[i] = (scale * q[i, :, :, None, :] @ s)[:, :, 0]
        dq[i] = scale * (s @ do[i, :, :, :, None])[..., 0]
    g = dfinal.double().abs() if magnitude else dfinal.double()
    for i in range(t - 1, -1, -1):
        g = g + scale * q[i, :, :, :, None] * do[i, :, :, None, :]
        dkk[i] = (g @ vw[i, :, :, :, None])[..., 0] * here[i]
        dvv[i] = (kw[i, :, :, None, :] @ g)[:, :, 0] * here[i]
        g = a[i] * g
    res = dict(out=out, dq=dq, dk=dkk.view(t, b, hk, grp, dk).sum(3), dv=dvv.view(t, b, hk, grp, dv).sum(3))
    return dict({n: z.transpose(0, 1).cpu() for n, z in res.items()}, state=s.cpu(), ds0=g.cpu())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vc", pv.CLASSES)
@pytest.mark.parametrize("kc", pv.CLASSES)
def test_every_kernel(kc, vc, dtype):
    from ur3e_amd.rl import ops
    for case in pv.calls(kc, vc):
        b, t, h, hk, dk, dv, state = case
        print(dtype, case, flush=True)
        gen = torch.Generator(device="cuda").manual_seed(t + dk + dv)

        def tok(*shape, dt=DT[dtype]):
            return torch.randn(shape, device="cuda", generator=gen).to(dt)
        lengths = torch.randint(0, t + 1, (b,), device="cuda", generator=gen, dtype=torch.int32)
        lengths[0] = t
        x = dict(q=tok(b, t, h, dk), k=tok(b, t, hk, dk), v=tok(b, t, hk, dv),
                 log_decay=torch.log(torch.linspace(0.6, 0.998, h)).cuda(),
                 initial_state=tok(b, h, dk, dv, dt=torch.float32) if state else None,
                 starts=torch.rand((b, t), device="cuda", generator=gen) < 0.02, lengths=lengths)
        dout, dfinal = tok(b, t, h, dv), tok(b, h, dk, dv, dt=torch.float32)
        if state:
            got = run(x, dout, dfinal)
        else:  # the outputs alone, and no state's gradient
            leaves = {n: x[n].requires_grad_() for n in ("q", "k", "v")}
            out, none = ops.decay_attention(**{**x, **leaves})
            assert none is None
            got = dict(zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, list(leaves.values()), dout))))
            dfinal.zero_()
        e, m = (definition(x, dout, dfinal, dk ** -0.5, i) for i in (False, True))
        n = ref.roundings(t, dk, dv, x["log_decay"].cpu(), h // hk)
        for name, y in got.items():
            ref.check(y, e[name], m[name], n, f"{case} {name}")
