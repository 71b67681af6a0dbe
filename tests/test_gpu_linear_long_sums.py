"""Products of few rows and few features with long sums: parts of the tiles, aligned and not, at the rule's edges.  Tolerances as in
test_gpu_linear."""
import pytest

import test_gpu_linear as base
from test_gpu_linear_kinds import ADDED, GATED, PLAIN, WHOLE

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,n,k,experts,kind,how", [
    (1, 1, 40000, 1, "dense", PLAIN), (1, 32, 100000, 1, "dense", ADDED), (3, 16, 8200, 1, "dense", WHOLE), (64, 32, 20008, 1, "dense", GATED),
    (200, 7, 4104, 1, "dense", PLAIN), (40, 200, 6144, 1, "dense", GATED), (16, 24, 20000, 8, "all", GATED), (200, 40, 8192, 5, "some", WHOLE),
    (1, 1, 40001, 1, "dense", PLAIN), (5, 33, 1537, 1, "dense", ADDED), (64, 200, 2501, 1, "dense", GATED), (200, 16, 4097, 1, "dense", WHOLE),
    (130, 9, 20001, 3, "all", WHOLE), (5, 65, 1535, 1, "dense", GATED), (70, 33, 4099, 4, "one", GATED),
    (6, 30, 2046, 1, "dense", PLAIN), (6, 30, 4098, 1, "dense", ADDED),                    # rows of 4, not 16 bytes
    (1, 14336, 1001, 1, "dense", PLAIN), (2, 7001, 1301, 2, "all", WHOLE),
])
def test_linear(gpu, rows, n, k, experts, kind, how):
    base.test_linear(gpu, rows, n, k, experts, kind, *how)
