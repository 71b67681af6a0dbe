"""Refusals of the balance loss and the per-expert counts (no device)."""
import naiwa_moe as nm
from naiwa_moe._lib import E_INVALID, E_UNSUPPORTED


def _counts(**a):
    d = dict(ids=4096, ids_ld=0, T=8, k=2, E=8, mask=None, counts=4096, bad=None)
    d.update(a)
    return nm.lib().naiwa_expert_counts(d["ids"], d["ids_ld"], d["T"], d["k"], d["E"], d["mask"], d["counts"], d["bad"], 0)


def _forward(**a):
    d = dict(x=4096, dt=nm.F32, ld=0, ids=4096, ids_ld=0, T=8, E=8, k=2, mask=None, counts=4096, valid=4096, probs=4096,
             loss=4096)
    d.update(a)
    return nm.lib().naiwa_router_balance(d["x"], d["dt"], d["ld"], d["ids"], d["ids_ld"], d["T"], d["E"], d["k"], d["mask"],
                                         d["counts"], d["valid"], d["probs"], d["loss"], 0)


def _backward(**a):
    d = dict(x=4096, dt=nm.F32, ld=0, counts=4096, valid=4096, T=8, E=8, k=2, mask=None, g=4096, d=4096, dld=0, flags=0)
    d.update(a)
    return nm.lib().naiwa_router_balance_backward(d["x"], d["dt"], d["ld"], d["counts"], d["valid"], d["T"], d["E"],
                                                  d["k"], d["mask"], d["g"], d["d"], d["dld"], d["flags"], 0)


def test_counts_refuse():
    for bad in (dict(T=-1), dict(k=0), dict(E=0), dict(ids_ld=1), dict(ids_ld=-2), dict(ids=None), dict(counts=None)):
        assert _counts(**bad) == E_INVALID, bad
    for bad in (dict(E=1025), dict(T=1 << 40), dict(T=1 << 30, k=2)):
        assert _counts(**bad) == E_UNSUPPORTED, bad


def test_forward_refuses():
    for bad in (dict(T=-1), dict(k=0), dict(E=0), dict(E=-8), dict(ids_ld=1), dict(ld=7), dict(ld=-1), dict(x=None),
                dict(ids=None), dict(counts=None), dict(valid=None), dict(probs=None), dict(loss=None)):
        assert _forward(**bad) == E_INVALID, bad
    for bad in (dict(E=1025), dict(dt=nm.F16), dict(dt=nm.Q8_0), dict(T=1 << 31)):
        assert _forward(**bad) == E_UNSUPPORTED, bad


def test_backward_refuses():
    for bad in (dict(T=-1), dict(k=0), dict(E=0), dict(ld=7), dict(dld=7), dict(dld=-1), dict(flags=2), dict(x=None),
                dict(counts=None), dict(valid=None), dict(g=None), dict(d=None), dict(x=1 << 20, d=1 << 20, dld=12)):
        assert _backward(**bad) == E_INVALID, bad
    for bad in (dict(E=1025), dict(dt=nm.F16), dict(T=1 << 31)):
        assert _backward(**bad) == E_UNSUPPORTED, bad
    assert _backward(T=0) == 0   # nothing to write, and no device call
