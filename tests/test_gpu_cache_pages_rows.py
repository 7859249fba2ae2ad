"""Forks of tables with more rows than a planning workgroup keeps the forks' claims of in LDS (4096), against
pages_oracle.py to the bit."""
import numpy as np
import pytest

from test_gpu_cache_pages import Both

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [4096, 4097, 9000])
def test_forks_of_tables_of_many_rows(rows):
    """Children named several times, rows outside, parents that are empty, more forks than the workgroup has
    threads; twice, so that the second call finds the first one's claims where its own go."""
    c = Both(rows, 3, 20000, 4, shapes=((4,),), seed=rows)
    rng = np.random.default_rng(rows)
    c.reserve([int(x) for x in rng.integers(0, 12, 1200)] + [0] * (rows - 1200))
    for _ in range(2):
        n = 2500
        parents = [int(x) for x in rng.integers(-1, 1300, n)]
        children = [int(x) for x in rng.integers(1000, rows + 2, n)]
        children[7:12] = [rows - 1] * 5
        c.fork(parents, children)
        c.free([int(x) for x in rng.integers(0, rows, 500)])
