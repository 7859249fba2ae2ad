"""The eviction's oracle on cases worked out by hand."""
import numpy as np

from evict_oracle import Evicting


def _cache(lengths, table, counts, weights, page=2):
    pool = np.arange(len(counts) * page * 3).reshape(len(counts), page, 3)
    return Evicting(table, lengths, counts, page, [pool], weights=weights), pool


def test_the_heaviest_and_the_recent_stay_in_order():
    c, pool = _cache([7], [[3, 0, 5, 1]], [1, 1, 0, 1, 0, 1], [[.1, .9, .2, .9, .5, .0, .0, .0]])
    assert c.evict([4], 1) == [[1, 3, 4, 6, -1, -1, -1, -1]]
    assert c.weights == [[.9, .9, .5, 0., 0., 0., 0., .0]]
    assert c.table == [[3, 0, -1, -1]] and c.lengths == [4] and c.counts == [1, 0, 0, 1, 0, 0]
    assert np.array_equal(c.pools[0][3], [pool[3, 1], pool[0, 1]]) and np.array_equal(c.pools[0][0], [pool[5, 0], pool[1, 0]])


def test_ties_go_to_the_first_and_nan_is_above_all():
    c, _ = _cache([4], [[0, 1]], [1, 1], [[1., 1., float("nan"), 1.]])
    assert c.evict([2], 0) == [[0, 2, -1, -1]]


def test_shared_pages_stay():
    c, _ = _cache([6, 5], [[0, 1, 2], [0, 3, 4]], [2, 1, 1, 1, 1], [[0, 0, 5, 6, 7, 8.], [9, 9, 1, 2, 3, 0]])
    assert c.evict([1, 3], 2) == [[0, 1, 5, -1, -1, -1], [0, 1, 3, 4, -1, -1]]
    assert c.lengths == [3, 4] and c.counts == [2, 1, 0, 1, 0]


def test_rows_within_their_budgets_are_left():
    c, pool = _cache([3, 0], [[0, 1], [-1, -1]], [1, 1], [[1., 2., 3., 4.], [0.] * 4])
    assert c.evict([3, -2], 9) == [[0, 1, 2, -1], [-1] * 4]
    assert c.table == [[0, 1], [-1, -1]] and c.lengths == [3, 0] and np.array_equal(c.pools[0], pool)


def test_nothing_stays():
    c, _ = _cache([3], [[1, 0]], [1, 1], [[1., 2., 3., 4.]])
    assert c.evict([-1], 5) == [[-1] * 4]
    assert c.table == [[-1, -1]] and c.lengths == [0] and c.counts == [0, 0] and c.weights == [[0., 0., 0., 4.]]
