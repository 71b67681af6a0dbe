"""The routed weights' gradient over memory that the call reads is refused (no device: made-up addresses that nothing may touch)."""
import pytest

import naiwa_moe as nm
from naiwa_moe._lib import E_INVALID
from test_linear import A, router

# T = 8 rows of E = 8 f32 logits, k = 2: logits at A[0], ids A[1], dw A[2]; 256 bytes of logits, 64 of ids and dw
LOGITS, IDS, DW, MASK = A[0], A[1], A[2], A[4]


@pytest.mark.parametrize("change", [
    dict(d=LOGITS + 4), dict(d=LOGITS + 32), dict(d=LOGITS + 252), dict(d=LOGITS - 252), dict(d=LOGITS, dld=12),
    dict(d=LOGITS, ld=12), dict(d=LOGITS + 16, ld=12, dld=12), dict(d=LOGITS + 2, dt=nm.BF16), dict(d=LOGITS + 126, dt=nm.BF16),
    dict(d=IDS), dict(d=IDS + 60), dict(d=IDS - 252), dict(d=DW), dict(d=DW + 60), dict(d=DW - 252),
    dict(d=MASK, mask=MASK), dict(d=MASK + 4, mask=MASK), dict(d=MASK - 252, mask=MASK), dict(d=DW + 64, dw_ld=16),
])
@pytest.mark.parametrize("mode,flags", [(0, 0), (0, 1), (2, 0), (2, 1)])
def test_refused(change, mode, flags):
    assert router(mode=mode, flags=flags, **change) == E_INVALID
