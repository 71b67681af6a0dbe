"""Row lengths of the activation's gradient: packed rows have the limit that stated ones have (no device: no rows, or refused)."""
import pytest

import naiwa_moe as nm
from naiwa_moe._lib import E_UNSUPPORTED
from test_linear import act

FAR = 1 << 21


@pytest.mark.parametrize("dt", [nm.F32, nm.BF16, nm.F16])
def test_packed_rows_have_a_limit(dt):
    assert act(dt=dt, n=FAR, rows=0) == 0
    assert act(dt=dt, n=FAR, ld=FAR, rows=0) == 0
    for n in (FAR + 1, (1 << 31) - 8, (1 << 31) - 7, (1 << 31) - 3, (1 << 31) - 1):
        for rows in (0, 1):
            assert act(dt=dt, n=n, rows=rows) == E_UNSUPPORTED
            assert act(dt=dt, n=n, ld=n, rows=rows) == E_UNSUPPORTED
    assert act(dt=dt, ld=FAR + 1) == E_UNSUPPORTED
