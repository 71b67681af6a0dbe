"""Row lengths past the documented limits are refused, those at the limit are not (no device: no rows, or an empty sort's)."""
import pytest

from naiwa_moe._lib import E_UNSUPPORTED
from test_linear import A, back, back_grad, forward, input_grad, to, weights

FAR, LONG = 1 << 21, 1 << 28


@pytest.mark.parametrize("f,change", [
    (forward, dict(out_ld=FAR)), (forward, dict(r=A[5], r_ld=FAR)), (forward, dict(pre=A[5], pre_ld=FAR)), (forward, dict(x_ld=FAR)),
    (input_grad, dict(dx_ld=FAR)), (input_grad, dict(pre=A[5], pre_ld=FAR)), (input_grad, dict(dy_ld=FAR)),
    (to, dict(ld=LONG)), (to, dict(rows_ld=LONG)), (back, dict(ld=LONG)), (back, dict(out_ld=LONG)), (back_grad, dict(d_ld=LONG)),
    (back_grad, dict(ld=LONG)), (back_grad, dict(dy_ld=LONG)),
], ids=lambda v: v.__name__ if callable(v) else "-".join(v))
def test_row_lengths(f, change):
    none = {"T" if f in (to, back, back_grad) else "rows": 0}
    assert f(**change, **none) == 0
    longer = {k: v + 1 if k.endswith("ld") else v for k, v in change.items()}
    assert f(**longer) == E_UNSUPPORTED
    assert f(**{k: 1 << 62 if k.endswith("ld") else v for k, v in change.items()}) == E_UNSUPPORTED


def test_features_past_a_row_length():
    assert forward(w=weights(experts=1, n=FAR, k=8), rows=0) == 0
    assert forward(w=weights(experts=1, n=FAR + 1, k=8)) == E_UNSUPPORTED
    assert forward(w=weights(experts=1, n=(1 << 31) - 1, k=1)) == E_UNSUPPORTED


def test_hidden_sizes_and_pairs():
    for f in (to, back, back_grad):
        assert f(T=0, H=1 << 24) == 0 and f(H=(1 << 24) + 1) == E_UNSUPPORTED
        assert f(T=(1 << 31) // 4, k=4) == E_UNSUPPORTED
