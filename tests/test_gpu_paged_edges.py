"""Attention on pages at the edges of its definition, against oracle/paged.py in float64: scores and values that are infinite."""
import math

import pytest
import torch

from tensor_parallel_amd import paged
from test_gpu_paged import BF16, DEV, F16, Batch, check_attend

pytestmark = pytest.mark.gpu


def infinite_keys(batch, b, positions):
    """Keys of sequence b whose score with any row is -inf (the queries' first element is 1)."""
    batch.q[:, :, 0] = 1.0
    for j in positions:
        batch.k[batch.table[b][j // batch.page], :, j % batch.page, 0] = -math.inf


CASES = [
    # counts, lengths, positions of the last sequence with a score of -inf
    ([1], [1], [0]), ([1], [40], range(40)), ([1, 3], [9, 70], range(68)), ([1, 4], [9, 4], range(3)), ([1], [9000], range(9000)), ([2], [9000], range(8990)), ([2], [9000], range(8999)),
    ([1], [600], range(600)), ([40], [40], range(11)), ([40], [40], [0]), ([30], [3000], range(2985)), ([300], [300], range(290)), ([1, 60], [700, 60], range(60)),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("counts,lengths,positions", CASES)
def test_scores_of_minus_infinity(dtype, D, counts, lengths, positions):
    """A row all of whose scores are -inf has no softmax: NaN, whole, cut and joined; one that has a finite score goes by that; zeros are for rows that see no position."""
    batch = Batch(counts, lengths, 4, 2, D, 16, dtype, seed=40)
    infinite_keys(batch, len(counts) - 1, positions)
    got = check_attend(batch, max_new=max(counts), max_length=max(lengths))
    first, n, length = batch.seqs[-1]
    for i in range(n):
        assert bool(got[first + i].isnan().all()) == all(j in positions for j in range(length - n + i + 1))


def test_rows_before_position_zero_are_zeros_beside_scores_of_minus_infinity():
    for counts, lengths in (([4], [2]), ([40], [25]), ([3, 1], [1, 0])):
        batch = Batch(counts, lengths, 4, 2, 64, 16, BF16, seed=41)
        infinite_keys(batch, 0, [0])
        got = check_attend(batch)
        before = counts[0] - lengths[0]
        assert (got[:before] == 0).all() and got[before].isnan().all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("counts,lengths", [([1, 4], [70, 133]), ([1], [600]), ([50, 40], [50, 161]), ([3], [9000]), ([40], [5000])])
def test_infinite_values_of_small_probability_do_not_vanish(dtype, D, counts, lengths):
    """Values that are not finite at positions whose probability is below what the dtype holds (e^-200 and less, but not zero): the rows that see them are not finite in their columns (the value itself,
    or the NaN of zero times it), and no other row or column is touched."""
    batch = Batch(counts, lengths, 4, 2, D, 16, dtype, seed=42, spread=0.1)
    b, n, new = len(counts) - 1, lengths[-1], counts[-1]
    batch.q[:, :, 0] = 16.0
    placed = {3: (n - 1, math.inf), 5: (max(n - 2, 0), -math.inf), 7: (n - 1 - new // 2, math.nan), 11: (n - new, math.inf), 13: (n // 2, -math.inf)}
    for column, (j, value) in placed.items():
        batch.k[batch.table[b][j // 16], :, j % 16, 0] = -15.0 * D**0.5
        batch.v[batch.table[b][j // 16], :, j % 16, column] = value
    got = paged.attend(batch.q.to(DEV), **batch.on(), max_new=max(counts), max_length=max(lengths)).cpu().double()
    want, weight = batch.want(D**-0.5)
    tol = batch.tolerance(want, weight, D**-0.5)
    finite = torch.isfinite(want)
    first, count, length = batch.seqs[b]
    for column, (j, value) in placed.items():
        for i in range(count):
            sees = j <= length - count + i
            assert bool(torch.isfinite(got[first + i, :, column]).any()) != sees, (column, i)
    assert torch.equal(torch.isfinite(got), finite)
    assert ((got - want).abs() - tol)[finite].max() <= 0
