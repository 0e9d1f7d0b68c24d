"""Eviction from long sequences: counts over several blocks of bit words, sums of which thousands share their first digits, and tables whose bits need more than a small
block's shared memory."""
import numpy as np
import pytest

from tests import helpers as H

torch = pytest.importorskip("torch")
from tests.test_gpu_paged import Cache, _ints  # noqa: E402
from tests.test_gpu_paged_evict import _evict  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from ironmill_b200 import ops
    return ops.Device(0)


KINDS = {
    "equal": lambda rng, shape: np.ones(shape),
    "eleven bits": lambda rng, shape: 1 + rng.random(shape) / 4,                        # sign, exponent and two bits are the same
    "twenty-two bits": lambda rng, shape: 1 + rng.integers(0, 1024, shape) * 2.0 ** -23,  # the last ten alone differ, many are equal
    "one in two": lambda rng, shape: rng.integers(0, 2, shape) * 3.0,
    "any": lambda rng, shape: np.exp(3 * rng.standard_normal(shape)),
}


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("budget, recent", [(12000, 500), (19999, 1), (9001, 0), (300, 300), (1030, 7)])
def test_twenty_thousand_rows(dev, kind, budget, recent):
    rng = H.rng_for("evict-20000", budget)
    c = Cache(dev, rng, [20000, 8200], [20000, 8200], kv_heads=1, dim=8, page=128)
    _evict(dev, c, rng, budget, recent, weights=KINDS[kind](rng, (1, 2, 1, c.table.shape[1] * 128)).astype(np.float32))


@pytest.mark.parametrize("budget, recent", [(1000, 100), (140000, 3000)])
def test_tables_of_two_hundred_thousand_rows_of_which_few_are_there(dev, budget, recent):
    """A short sequence, and one whose length passes what is there: its sums move, rows that are not there do not."""
    rng = H.rng_for("evict-200000", budget)
    c = Cache(dev, rng, [3000, 2500], [3000, 150000], kv_heads=1, dim=8, page=256)
    c.table = np.concatenate([c.table, np.full((2, 200000 // 256), -1)], 1)
    c.table[1, 500:503] = c.table[1, :3]
    c.table[1, :3] = -1
    c.kv.point_at(_ints(c.table), _ints(c.lengths))
    _evict(dev, c, rng, budget, recent, weights=rng.random((1, 2, 1, c.table.shape[1] * 256)).astype(np.float32))
