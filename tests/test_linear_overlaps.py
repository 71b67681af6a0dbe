"""Products and gradients: outputs over the offsets are refused (no device: made-up addresses that nothing may touch)."""
import pytest

from naiwa_moe._lib import E_INVALID
from test_linear import A, forward, input_grad, weight_grad, weights

# four experts: 20 bytes of offsets, at A[2]; 8 rows of 32 and 48 16-bit values: 512 and 768 bytes
O = A[2]


@pytest.mark.parametrize("f,change", [
    (forward, dict(out=O)), (forward, dict(out=O + 16)), (forward, dict(out=O - 508)), (forward, dict(pre=O)),
    (forward, dict(pre=O + 16)), (forward, dict(u=weights(w=A[4]), pre_up=O - 508)), (forward, dict(out=O, r=O)),
    (input_grad, dict(dx=O)), (input_grad, dict(dx=O + 16)), (input_grad, dict(dx=O - 764)),
    (input_grad, dict(pre=A[4], pre_up=A[5], dx_up=O + 16)),
    (weight_grad, dict(dw=O)), (weight_grad, dict(dw=O + 16)), (weight_grad, dict(dw=O - 4 * 32 * 48 * 4 + 4)),
    (weight_grad, dict(db=O)), (weight_grad, dict(db=O + 16)), (weight_grad, dict(db=O - 4 * 32 * 4 + 4)),
    (weight_grad, dict(dw=O, rows=0, dy=None, x=None)), (weight_grad, dict(db=O, rows=0, dy=None, x=None)),
])
def test_outputs_over_the_offsets(f, change):
    assert f(**change) == E_INVALID
