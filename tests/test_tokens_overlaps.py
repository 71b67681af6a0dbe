"""Sorted tokens: outputs over memory that the call reads, or over each other, are refused (no device: made-up addresses that
nothing may touch)."""
import pytest

import naiwa_moe as nm
from naiwa_moe._lib import E_INVALID
from test_linear import A, back, back_grad, sort, to

# T = 8 tokens of k = 2, H = 16: 64 bytes of ids, inv and weights, 8 of a mask


@pytest.mark.parametrize("change", [
    dict(perm=A[0]), dict(perm=A[0] + 60), dict(perm=A[0] - 60), dict(inv=A[0]), dict(inv=A[0] + 60), dict(offsets=A[0] - 32),
    dict(offsets=A[0] + 60), dict(bad=A[0]), dict(bad=A[0] + 60), dict(perm=A[5], mask=A[5]), dict(inv=A[5] + 4, mask=A[5]),
    dict(offsets=A[5], mask=A[5]), dict(bad=A[5], mask=A[5]), dict(inv=A[1]), dict(inv=A[1] + 60), dict(offsets=A[1] + 60),
    dict(offsets=A[2] - 32), dict(bad=A[1]), dict(bad=A[2] + 60), dict(bad=A[3] + 32), dict(perm=A[0] + 64, ids_ld=4),
])
@pytest.mark.parametrize("T", [8, 5000])
def test_sort(change, T):
    assert sort(T=T, **change) == E_INVALID


@pytest.mark.parametrize("f,change", [
    (to, dict(rows=A[1])), (to, dict(rows=A[1] + 60)), (to, dict(rows=A[1] - 2 * 16 * 16 + 2)),
    (back, dict(out=A[1])), (back, dict(out=A[1] + 60)), (back, dict(out=A[4], w=A[4])), (back, dict(out=A[4] + 60, w=A[4])),
    (back, dict(out=A[4] - 508, w=A[4])), (back, dict(out=A[4] - 508, w=A[4], flags=1)),
    (back_grad, dict(dw=A[0])), (back_grad, dict(dw=A[0] + 508)), (back_grad, dict(dw=A[1])), (back_grad, dict(dw=A[1] + 508)),
    (back_grad, dict(dw=A[2])), (back_grad, dict(dw=A[2] + 60)), (back_grad, dict(dw=A[3])), (back_grad, dict(dw=A[3] + 4)),
    (back_grad, dict(dw=A[4])), (back_grad, dict(dw=A[4] + 508)), (back_grad, dict(dy=A[2])), (back_grad, dict(dy=A[3] + 60)),
    (back_grad, dict(dy=A[2] - 510, dw=None)), (back_grad, dict(dy=A[3], dw=None)), (back_grad, dict(dw=A[3], dy=None)),
    (back_grad, dict(dw=A[0] + 4, dy=None)), (back_grad, dict(dy=A[0], dw=None, y=None)),
])
def test_rows(f, change):
    assert f(**change) == E_INVALID
