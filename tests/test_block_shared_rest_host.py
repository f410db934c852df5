"""Which items of a plan with shared prefixes hold their weights in two terms (no GPU needed)."""

import numpy as np
import pytest

from mjolnir_b200 import _lib


@pytest.mark.parametrize("few,rest", [(0, [0, 0]), (2, [1, 0]), (3, [1, 0]), (6, [1, 1])])
def test_groups_with_rows_of_the_decode_kernel(few, rest):
    groups = [(1, 2, 512), (4, 2, 1024)]
    q, kv = [2] * 6, [700, 600, 590, 80, 1500, 1300]
    work, joins = np.zeros((500, 8), np.int32), np.zeros((100, 12), np.int32)
    nw, *_ = _lib.block_shared_plan(q, kv, [2] * few, groups, 8, 2, 128, True, 148, 300, work, joins)
    of = {first: r for (first, _, _), r in zip(groups, rest)}
    for s, _, _, _, _, span, two, last in work[:nw].tolist():
        assert two == (of[s] if span else 0) and last == 0
