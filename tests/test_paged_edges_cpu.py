"""CPU: the float64 restatements at the edges that test_gpu_paged_edges.py takes the kernels to."""

import numpy as np

from oracle import paged as opg


def test_eviction_ranks_protected_slots_before_any_weight():
    """Worked out by hand: of 6 slots 3 stay, two of them protected ones with small weights behind infinite
    weights in lower slots."""
    k = np.arange(6 * 16, dtype=float).reshape(1, 1, 6, 16)
    acc = np.array([[[np.inf, np.nan, np.inf, 0.5, 0.1, np.inf]]])
    pos = np.array([[[3, 4, 5, 0, 9, 6]]])
    k1, _, a, p, n = opg.evict(k, k, np.array([[0]]), [6], acc, pos, [3], [9], 1)
    assert n == [3]
    # slots 3 (position 0) and 4 (position 9) are protected, slot 0 is the lowest of the infinite ones;
    # 3 and 4 move into the holes 1 and 2
    assert p[0, 0].tolist() == [3, 0, 9] and a[0, 0].tolist() == [np.inf, 0.5, 0.1]
    np.testing.assert_array_equal(k1[0, 0, :3], k[0, 0, [0, 3, 4]])
