"""The sort around the number of experts that its own tables hold (2048), and at
the most that it takes; plain implementation and tolerances of
test_gpu_sort_rows."""
import pytest

import test_gpu_sort_rows as rows

pytestmark = rows.pytestmark


@pytest.mark.parametrize("E", [2047, 2048, 2049, 16383, 16384])
@pytest.mark.parametrize("T,K", [(1, 16), (300, 4), (3000, 8)])
def test_many_experts(gpu, E, T, K):
    for n, kind in enumerate(("mixed", "all", "one", "none")):
        print(f"sort T={T} K={K} E={E} {kind}", flush=True)
        ids = rows.routes(T, E, K, T + n, kind)
        x, w = rows.data(T, 64, K, n)
        rows.check_sort(rows.sort(gpu, ids, x, E, True, w, True), ids, x, E, True, w, True)
