"""Products whose tiles would not fit a launch's 2^32 threads are refused (no device: made-up addresses that nothing may touch)."""
import pytest

from naiwa_moe._lib import E_UNSUPPORTED
from test_linear import forward, input_grad, weight_grad, weights

B = [(i + 1) << 48 for i in range(6)]   # addresses far apart, for arrays of terabytes
MOST = (1 << 31) - 1


@pytest.mark.parametrize("f,change", [
    (forward, dict(w=weights(w=B[0], experts=1, n=16, k=16), o=None, rows=MOST, x=B[1], out=B[2])),
    (forward, dict(w=weights(w=B[0], experts=4096, n=1 << 21, k=8), o=B[3], rows=4096, x=B[1], out=B[2])),
    (forward, dict(w=weights(w=B[0], experts=1, n=1 << 21, k=1 << 21), o=None, rows=1 << 24, x=B[1], out=B[2])),
    (input_grad, dict(w=weights(w=B[0], experts=1, n=16, k=16), o=None, rows=MOST, dy=B[1], dx=B[2])),
    (input_grad, dict(w=weights(w=B[0], experts=1, n=16, k=1 << 21), o=None, rows=1 << 24, dy=B[1], dx=B[2])),
    (weight_grad, dict(experts=4096, n=1, k=1 << 21, o=B[3], dy=B[1], x=B[2], dw=B[4])),
    (weight_grad, dict(experts=4096, n=1 << 21, k=1 << 21, o=B[3], dy=B[1], x=B[2], dw=B[4])),
])
def test_refused(f, change):
    assert f(**change) == E_UNSUPPORTED
