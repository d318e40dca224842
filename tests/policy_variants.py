"""Which kernels a call of decay_attention runs (the rules of ur3e_policy.hip, restated), and a list of calls that reaches every one
of them.  Test infrastructure only."""
import math

CLASSES = (16, 32, 64, 128)
# an odd count of channels in each class of key and value tiles
KEYS = {16: 13, 32: 27, 64: 57, 128: 99}
VALUES = {16: 13, 32: 27, 64: 57, 128: 99}
OTHER = {16: 9, 32: 20, 64: 60, 128: 70}


def tiles(kdim, vdim):
    def pow2(d):
        return 1 if d <= 16 else 2 if d <= 32 else 4 if d <= 64 else 8
    kt = pow2(kdim)
    vt = min(pow2(vdim), 2 if kt == 8 else 4)
    return kt, vt, -(-vdim // (16 * vt))


def splits(b, t, h, dk, dv, es, ragged, backward):
    """(splits, tokens of each)"""
    waves = b * h * tiles(dk, dv)[2]
    if backward:
        waves = 3 * waves if dk == dv else min(waves, 2 * b * h * tiles(dv, dk)[2])
    if t < (128 if es == 4 else 192):
        return 1, max(t, 1)

    def length(n):
        return (-(-t // n) + 15) // 16 * 16
    least = 32
    while least * least * 4 < t:
        least += 16
    once, again = 2048 // waves, 4096 // waves
    ln = length(once) if once > 1 else t
    if ragged and again > 1:
        even = 8 * dk * dv // ((dk + dv) * es)
        ln = min(ln, max(length(again), (even + 15) // 16 * 16))
    if ln >= t:
        return 1, t
    ln = max(ln, least)
    n = -(-t // ln)
    return (n, ln) if n > 1 else (1, t)


def room(elems):
    return (elems + 3) // 4 * 4


def kernels(b, t, h, dk, dv, dtype, ragged, state, grad):
    """the walks (dtype, KT, VT, STATE, H, FINE) and the joins of a call"""
    es = 4 if dtype == "f32" else 2
    out = set()

    def walk(kdim, vdim, nw, n, is_state, fine):
        kt, vt, slabs = tiles(kdim, vdim)
        while vt > 1 and b * h * nw * slabs * n <= 1024:
            vt //= 2
            slabs = -(-vdim // (16 * vt))
        pairs = es == 2 and kt < 8 and t > 16
        out.add((dtype, kt, vt, is_state, 2 if pairs else 1, True if es == 4 else fine))
        if is_state:
            elems = kdim * vdim
            out.add("join" if b * h * nw * elems >= 64 * 4096 else "join of several waves" if n > 32 else "join of one wave")
    n, _ = splits(b, t, h, dk, dv, es, ragged, False)
    if n > 1:
        walk(dk, dv, 1, n, True, state)
    walk(dk, dv, 1, n, False, state)
    if grad:
        n, _ = splits(b, t, h, dk, dv, es, ragged, True)
        if n > 1:
            walk(dk, dv, 2, n, True, state)
        if dk == dv:
            walk(dv, dk, 3, n, False, state)
        else:
            walk(dv, dk, 2, n, False, False)
            walk(dk, dv, 1, n, False, state)
    return out


def every(dtype):
    """all that are compiled for a type"""
    es = 4 if dtype == "f32" else 2
    out = {"join", "join of one wave", "join of several waves"}
    for kt in (1, 2, 4, 8):
        for vt in (1, 2, 4) if kt < 8 else (1, 2):
            for fine in (True,) if es == 4 else (True, False):
                pairs = es == 2 and kt < 8
                out.add((dtype, kt, vt, True, 2 if pairs else 1, fine))
                out.add((dtype, kt, vt, False, 1, fine))
                if pairs:
                    out.add((dtype, kt, vt, False, 2, fine))
    return out


def calls(kc, vc):
    """[(b, t, h, hk, dk, dv, state)] for a class of key and a class of value channels: one tile of tokens, several, and several
    splits, each with enough waves that the widest tiles stay; sequences that few waves share take the narrow ones"""
    dk, dv = KEYS[kc], VALUES[vc]
    out = []
    for state in (True, False) if kc == vc else (True,):
        for h, hk, t in ((4, 4, 16), (4, 2, 33)):
            out.append((257, t, h, hk, dk, dv, state))
        slabs = tiles(dk, dv)[2]
        out.append((600 // 4 // slabs, 200, 4, 2, dk, dv, state))
        out.append((600 // 4 // slabs, 200, 4, 4, OTHER[kc], OTHER[vc], state))
    if kc != vc:
        out.append((600 // 4 // slabs, 200, 4, 2, dk, dv, False))
    out.append((1, 200 if kc != vc else 1500, 2, 1, OTHER[kc], OTHER[vc], True))
    return out
