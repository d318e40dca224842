"""The calls of tests/test_gpu_policy_variants.py reach every kernel of the walk, and the rules that say so are the library's."""
import ctypes

import pytest

import policy_variants as pv
from test_policy_ops_cpu import AttnC, TokensC


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_the_list_reaches_every_kernel(dtype):
    reached = set()
    for kc in pv.CLASSES:
        for vc in pv.CLASSES:
            for b, t, h, hk, dk, dv, state in pv.calls(kc, vc):
                reached |= pv.kernels(b, t, h, dk, dv, dtype, True, state, True)
    assert reached == pv.every(dtype)


def sizes():
    out = {c for kc in pv.CLASSES for vc in pv.CLASSES for c in pv.calls(kc, vc)}
    # the rule's edges, and lengths up to a demonstration's and beyond
    out |= {(b, t, h, h, d, d, True) for b in (1, 3, 32, 700) for t in (127, 128, 191, 192, 777, 10500, 80000)
            for h, d in ((1, 16), (4, 64))}
    return sorted(out)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("ragged", [False, True])
def test_splits_are_the_librarys(dtype, ragged):
    """by the bytes of workspace that they need"""
    from ur3e_amd import runtime as rt
    L = rt.load_library()
    L.ur3e_attn_workspace.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p]
    es = 4 if dtype == "f32" else 2

    def up(x):
        return (x + 255) // 256 * 256
    for b, t, h, hk, dk, dv, _ in sizes():
        a = AttnC()
        a.b, a.t, a.heads, a.kv_heads, a.dk, a.dv, a.scale = b, t, h, hk, dk, dv, 1.0
        a.dtype = ("f32", "bf16", "f16").index(dtype)
        a.q = a.k = a.v = TokensC(4096, 1, 1, 1)
        a.log_decay = 4096
        a.lengths = 4096 if ragged else None
        n = ctypes.c_size_t()
        for backward in (0, 1):
            assert L.ur3e_attn_workspace(ctypes.byref(a), backward, ctypes.byref(n)) == 0
            s, _ = pv.splits(b, t, h, dk, dv, es, ragged, backward)
            want = up(b * h * s * (pv.room(dk * dv) + 1) * 4) if s > 1 else 0
            if backward:
                want *= 2
                if hk != h:
                    want += up(b * t * h * dk * 4) + up(b * t * h * dv * 4)
            assert n.value == want, (b, t, h, hk, dk, dv, backward)
