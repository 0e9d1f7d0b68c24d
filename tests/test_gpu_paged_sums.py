"""Sums of attention weights where rows are not numbers, where scores lie far apart, and in tables of which little is there (tests/oracle_paged_more.py)."""
import numpy as np
import pytest

from tests import helpers as H
from tests import oracle_paged_more as om

torch = pytest.importorskip("torch")
from tests.test_gpu_paged import Cache, _ints, _np, _randn  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from ironmill_b200 import ops
    return ops.Device(0)


@pytest.mark.parametrize("max_len", ["said", "longer", "none"])
@pytest.mark.parametrize("dtype, dim, heads, nodes", [("f16", 128, 8, 3), ("bf16", 64, 4, 8), ("f16", 256, 4, 2), ("bf16", 128, 8, 40), ("f16", 64, 16, 40), ("f16", 256, 8, 9)])
def test_a_row_that_is_not_a_number_reaches_only_the_positions_that_it_sees(dev, dtype, dim, heads, nodes, max_len):
    """Every node sees itself alone; a query of the first node is NaN. Pages that are not there get nothing from it either."""
    from ironmill_b200 import ops
    rng = H.rng_for("sums-nan-row", dim + nodes)
    c = Cache(dev, rng, [70 + nodes, 50 + nodes], [70, 50], dim=dim, page=16, dtype=dtype)
    c.table[0, 2] = -1
    c.kv.point_at(_ints(c.table), _ints(c.lengths))
    mask = np.array([1 << i for i in range(nodes)] * 2, dtype=np.uint64)[:, None]
    q = _randn(rng, (2 * nodes, heads, dim), dtype)
    q[0, 1] = float("nan")
    sums = torch.zeros((2, 2, c.table.shape[1] * 16), device="cuda")
    starts = [0, nodes, 2 * nodes]
    ops.paged_attention_weights(c.kv, 0, q, _ints(starts), nodes, 0.1, sums, mask=torch.from_numpy(mask.view(np.int64)).cuda(),
                                max_len={"said": 70 + nodes, "longer": 9000, "none": 0}[max_len])
    with np.errstate(invalid="ignore"):
        _, _, _, want = om.attention(_np(c.k[0]), _np(c.v[0]), c.table, c.lengths, starts, _np(q), 0.1, mask, np.zeros(sums.shape))
    bad = np.isnan(want)
    assert bad[0, 0, :32].all() and not bad[0, 0, 32:48].any() and bad[0, 0, 48:71].all() and not bad[0, 0, 71:].any() and not bad[0, 1].any() and not bad[1].any()
    got = _np(sums)
    assert (np.isnan(got) == bad).all()
    # sums of `heads` weights of at most one each: scores to 2^-15, the exponential and the norm to 2^-18
    assert np.abs(got - want)[~bad].max() <= nodes * heads * 2.0 ** -14
