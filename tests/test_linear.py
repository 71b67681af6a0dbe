"""Refusals of the sorted tokens' and the 16-bit products' entry points (no device): made-up addresses that
nothing may touch."""
import ctypes as C

import pytest

import naiwa_moe as nm
from naiwa_moe._lib import E_INVALID, E_UNSUPPORTED, LinearWeights

A = [(i + 1) << 36 for i in range(12)]   # addresses far apart


def call(name, args, order, **changes):
    bad = set(changes) - set(args)
    assert not bad, bad
    a = {**args, **changes}
    return getattr(nm.lib(), name)(*[a[k] for k in order.split()], 0)


def sort(**c):
    d = dict(ids=A[0], ids_ld=0, T=8, k=2, E=8, mask=None, perm=A[1], inv=A[2], offsets=A[3], bad=None)
    return call("naiwa_expert_sort", d, "ids ids_ld T k E mask perm inv offsets bad", **c)


def to(**c):
    d = dict(x=A[0], dt=nm.BF16, ld=0, inv=A[1], T=8, k=2, H=16, rows=A[2], rows_ld=0)
    return call("naiwa_tokens_to_experts", d, "x dt ld inv T k H rows rows_ld", **c)


def back(**c):
    d = dict(y=A[0], dt=nm.BF16, ld=0, inv=A[1], w=None, w_ld=0, T=8, k=2, H=16, out=A[2], od=nm.F32, out_ld=0, flags=0)
    return call("naiwa_tokens_from_experts", d, "y dt ld inv w w_ld T k H out od out_ld flags", **c)


def back_grad(**c):
    d = dict(d=A[0], dd=nm.F32, d_ld=0, y=A[1], dt=nm.BF16, ld=0, inv=A[2], w=A[3], w_ld=0, T=8, k=2, H=16, dy=A[4], dy_ld=0,
             dw=A[5], dw_ld=0)
    return call("naiwa_tokens_from_experts_backward", d, "d dd d_ld y dt ld inv w w_ld T k H dy dy_ld dw dw_ld", **c)


def router(**c):
    d = dict(x=A[0], dt=nm.F32, ld=0, ids=A[1], ids_ld=0, dw=A[2], dw_ld=0, T=8, E=8, k=2, mode=0, mask=None, d=A[3], dld=0,
             flags=0)
    return call("naiwa_router_topk_backward", d, "x dt ld ids ids_ld dw dw_ld T E k mode mask d dld flags", **c)


def weights(w=A[0], bias=None, ld=0, stride=0, experts=4, n=32, k=48, dtype=nm.BF16):
    return C.byref(LinearWeights(w, bias, ld, stride, experts, n, k, dtype))


def forward(**c):
    d = dict(w=weights(), u=None, x=A[1], x_ld=0, o=A[2], rows=8, act=nm.ACT_NONE, r=None, r_ld=0, out=A[3], od=nm.BF16,
             out_ld=0, pre=None, pre_up=None, pre_ld=0)
    return call("naiwa_linear", d, "w u x x_ld o rows act r r_ld out od out_ld pre pre_up pre_ld", **c)


def input_grad(**c):
    d = dict(w=weights(), u=None, dy=A[1], dy_up=None, dy_ld=0, o=A[2], rows=8, act=nm.ACT_SILU, pre=None, pre_up=None,
             pre_ld=0, dx=A[3], dx_up=None, dd=nm.BF16, dx_ld=0, flags=0)
    return call("naiwa_linear_input_grad", d, "w u dy dy_up dy_ld o rows act pre pre_up pre_ld dx dx_up dd dx_ld flags", **c)


def weight_grad(**c):
    d = dict(dy=A[0], dy_ld=0, x=A[1], x_ld=0, dt=nm.F16, o=A[2], experts=4, rows=8, n=32, k=48, dw=A[3], wd=nm.F32, ld=0,
             stride=0, db=None, flags=0)
    return call("naiwa_linear_weight_grad", d, "dy dy_ld x x_ld dt o experts rows n k dw wd ld stride db flags", **c)


def act(**c):
    d = dict(d=A[0], p=A[1], q=None, dt=nm.F32, rows=8, n=32, ld=0, act=nm.ACT_SILU, dp=A[2], dq=None)
    return call("naiwa_act_backward", d, "d p q dt rows n ld act dp dq", **c)


INVALID = [
    (sort, [dict(T=-1), dict(k=0), dict(E=0), dict(ids_ld=1), dict(ids_ld=-2), dict(ids=None), dict(perm=None),
            dict(inv=None), dict(offsets=None)]),
    (to, [dict(T=-1), dict(k=0), dict(H=0), dict(ld=15), dict(rows_ld=-16), dict(x=None), dict(inv=None), dict(rows=None),
          dict(rows=A[0]), dict(rows=A[0] + 2 * 16 * 8 - 2), dict(rows=A[0] - 2 * 16 * 16 + 2)]),
    (back, [dict(T=-1), dict(k=0), dict(H=0), dict(ld=15), dict(out_ld=15), dict(w_ld=1), dict(y=None), dict(inv=None),
            dict(out=None), dict(flags=2), dict(out=A[0], od=nm.BF16), dict(out=A[0] + 2 * 16 * 16 - 4)]),
    (back_grad, [dict(T=-1), dict(k=0), dict(H=0), dict(d_ld=15), dict(ld=15), dict(dy_ld=15), dict(w_ld=1), dict(dw_ld=1),
                 dict(d=None), dict(y=None), dict(inv=None), dict(dy=A[0]), dict(dy=A[1], dy_ld=24), dict(dy=A[1] + 2)]),
    (router, [dict(T=-1), dict(k=0), dict(E=0), dict(ld=7), dict(dld=7), dict(ids_ld=1), dict(dw_ld=1), dict(flags=2),
              dict(x=None), dict(ids=None), dict(dw=None), dict(d=None), dict(d=A[0], dld=12)]),
    (forward, [dict(w=None), dict(w=weights(w=None)), dict(w=weights(n=0)), dict(w=weights(k=0)), dict(w=weights(experts=0)),
               dict(w=weights(ld=47)), dict(w=weights(ld=-48)), dict(w=weights(stride=32 * 48 - 1)), dict(u=weights(n=16)),
               dict(u=weights(k=32)), dict(u=weights(experts=3)), dict(u=weights(dtype=nm.F16)), dict(x_ld=47), dict(r_ld=31),
               dict(out_ld=31), dict(pre_ld=31), dict(rows=-1), dict(o=None), dict(x=None), dict(out=None), dict(pre_up=A[5]),
               dict(out=A[1]), dict(out=A[0] + 4 * 32 * 48 * 2 - 2), dict(pre=A[3]), dict(pre=A[1]), dict(r=A[3] + 2),
               dict(r=A[3], r_ld=40), dict(u=weights(w=A[4]), pre=A[5], pre_up=A[5] + 64), dict(u=weights(w=A[3])),
               dict(w=weights(bias=A[3]))]),
    (input_grad, [dict(w=None), dict(w=weights(n=0)), dict(u=weights(w=A[4])), dict(dy_up=A[5]), dict(dy_ld=31),
                  dict(pre_ld=47), dict(dx_ld=47), dict(rows=-1), dict(o=None), dict(dy=None), dict(dx=None), dict(flags=2),
                  dict(pre_up=A[5], dx_up=A[6]), dict(pre=A[4], pre_up=A[5]), dict(pre=A[4], dx_up=A[5]),
                  dict(pre=A[4], flags=1), dict(dx=A[1]), dict(dx=A[0]), dict(pre=A[3]),
                  dict(pre=A[4], pre_up=A[5], dx_up=A[3]), dict(pre=A[4], pre_up=A[5], dx_up=A[4])]),
    (weight_grad, [dict(experts=0), dict(rows=-1), dict(n=0), dict(k=0), dict(dy_ld=31), dict(x_ld=47), dict(ld=47),
                   dict(stride=32 * 48 - 1), dict(o=None), dict(dy=None), dict(x=None), dict(dw=None), dict(flags=2),
                   dict(dw=A[0]), dict(dw=A[1]), dict(db=A[3]), dict(db=A[0])]),
    (act, [dict(rows=-1), dict(n=0), dict(ld=31), dict(d=None), dict(p=None), dict(dp=None), dict(q=A[3]), dict(dq=A[3]),
           dict(dp=A[0] + 4), dict(q=A[3], dq=A[2]), dict(q=A[3], dq=A[1] + 4)]),
]
UNSUPPORTED = [
    (sort, [dict(E=4097), dict(T=1 << 31), dict(T=1 << 30, k=2)]),
    (to, [dict(dt=nm.Q8_0), dict(T=1 << 31)]),
    (back, [dict(dt=nm.Q8_0), dict(od=nm.F16), dict(dt=nm.F32, od=nm.BF16), dict(T=1 << 31)]),
    (back_grad, [dict(dt=nm.Q8_0), dict(dd=nm.F16), dict(T=1 << 31)]),
    (router, [dict(E=1025), dict(k=33), dict(dt=nm.F16), dict(mode=3), dict(mode=-1), dict(T=1 << 31)]),
    (forward, [dict(w=weights(dtype=nm.F32)), dict(w=weights(experts=4097)), dict(w=weights(ld=(1 << 21) + 1)), dict(act=7),
               dict(od=nm.F16), dict(rows=1 << 31), dict(x_ld=(1 << 21) + 1), dict(w=weights(stride=(1 << 48) + 1))]),
    (input_grad, [dict(w=weights(dtype=nm.Q8_0)), dict(act=7), dict(dd=nm.F16), dict(rows=1 << 31),
                  dict(dy_ld=(1 << 21) + 1)]),
    (weight_grad, [dict(dt=nm.F32), dict(wd=nm.BF16), dict(rows=1 << 31), dict(experts=4097), dict(n=(1 << 21) + 1),
                   dict(k=(1 << 21) + 1)]),
    (act, [dict(dt=nm.Q8_0), dict(act=7), dict(rows=1 << 31)]),
]


def cases(table):
    return [pytest.param(f, c, id=f"{f.__name__}-{i}-" + "-".join(c)) for f, all_ in table for i, c in enumerate(all_)]


@pytest.mark.parametrize("f,change", cases(INVALID))
def test_invalid(f, change):
    assert f(**change) == E_INVALID


@pytest.mark.parametrize("f,change", cases(UNSUPPORTED))
def test_unsupported(f, change):
    assert f(**change) == E_UNSUPPORTED


def test_calls_of_nothing():
    for rc in (to(T=0), back(T=0), back_grad(T=0), back_grad(dy=None, dw=None), router(T=0), forward(rows=0),
               input_grad(rows=0), act(rows=0)):
        assert rc == 0
