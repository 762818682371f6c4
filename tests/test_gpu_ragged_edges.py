"""Edges of the ragged operators: bounds and lengths that cannot be right, caps and scales of any size, weights far below
the largest."""

import pytest
import torch

from tests.test_gpu_kv_cache import Cache, append_op, ints, random_rows, run_op

pytestmark = pytest.mark.gpu

MOST, LEAST = 2**31 - 1, -(2**31)
BAD = 64  # bit 6 of the status word


# ------------------------------------------------------------------ append
@pytest.mark.parametrize(
    "bounds,good",
    [([0, 3, 10, 10], [0]), ([0, 3, MOST, MOST], [0]), ([-2, 3, 6, 8], [1, 2]), ([LEAST, 3, 6, 8], [1, 2]), ([0, 5, 3, 8], [0, 2]),
     ([0, 9, 9, 8], [])],
    ids=str,
)  # fmt: skip
def test_append_skips_sequences_whose_bounds_are_not_right(bounds, good):
    """Rows that the tensor does not have, or an end before its beginning: the sequence is left as it is, the others are appended."""
    from tests.attention64 import append

    cache = Cache([90, 75, 140], 2, seed=1)
    k, v = random_rows(2, 8, 2), random_rows(3, 8, 2)
    want = [[x.clone() for x in part] for part in (cache.codes, cache.scales)]
    for s in good:
        for which, x in enumerate((k, v)):
            fresh = x[bounds[s] : bounds[s + 1]].float()
            append(want[0][which], want[1][which], fresh, cache.table[s], cache.plain[s] - len(fresh))
    run_op(append_op(cache, k, v, ints(bounds)), status=BAD)
    for which in range(2):
        assert torch.equal(cache.scales[which], want[1][which]) and torch.equal(cache.codes[which], want[0][which])


@pytest.mark.parametrize("length", [LEAST, LEAST + 1, -1, 2, 193, MOST])
def test_append_skips_lengths_that_are_not_right(length):
    """Of any size: fewer tokens than the new ones, or more than the table has room for."""
    from tests.attention64 import append

    cache = Cache([90, 75, 140], 2, seed=4)
    k, v = random_rows(5, 8, 2), random_rows(6, 8, 2)
    bounds = [0, 3, 6, 8]
    want = [[x.clone() for x in part] for part in (cache.codes, cache.scales)]
    for s in (0, 2):
        for which, x in enumerate((k, v)):
            fresh = x[bounds[s] : bounds[s + 1]].float()
            append(want[0][which], want[1][which], fresh, cache.table[s], cache.plain[s] - len(fresh))
    cache.lengths[1] = length
    run_op(append_op(cache, k, v, ints(bounds)), status=BAD)
    for which in range(2):
        assert torch.equal(cache.scales[which], want[1][which]) and torch.equal(cache.codes[which], want[0][which])


@pytest.mark.parametrize("bounds", [(128, 300), (128, 100)])
def test_append_notes_bounds_behind_the_last_rows(bounds):
    """More sequences than a CTA looks up at once; those behind the first 128 have no rows, and no CTA to look for any."""
    from tests.attention64 import append

    cache = Cache([70] * 300, 1, seed=28)
    k, v = random_rows(29, 128, 1), random_rows(30, 128, 1)
    want = [[x.clone() for x in part] for part in (cache.codes, cache.scales)]
    for s in range(128):
        for which, x in enumerate((k, v)):
            append(want[0][which], want[1][which], x[s : s + 1].float(), cache.table[s], 69)
    run_op(append_op(cache, k, v, ints([*range(129), *[128] * 170, *bounds])), status=BAD)
    for which in range(2):
        assert torch.equal(cache.scales[which], want[1][which]) and torch.equal(cache.codes[which], want[0][which])
