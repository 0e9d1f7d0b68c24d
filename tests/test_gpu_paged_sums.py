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


@pytest.mark.parametrize("dtype, dim", [("f16", 128), ("bf16", 64), ("bf16", 256)])
@pytest.mark.parametrize("new, heads, max_len", [(1, 8, 0), (1, 8, 400), (2, 8, 9000), (26, 8, 400), (64, 8, 400)])
@pytest.mark.parametrize("scale2", [4.0, -0.5, 2.0 ** -7])
def test_sums_of_scores_that_are_exact_and_far_apart(dev, dtype, dim, new, heads, max_len, scale2):
    """Queries and keys of small whole numbers: their products are exact, and thousands apart. Every row's weights add up to one."""
    from ironmill_b200 import ops
    rng = H.rng_for("sums-exact", dim + new)
    lengths = [300, 40]
    c = Cache(dev, rng, [n + new for n in lengths], lengths, dim=dim, page=16, dtype=dtype)
    c.k.copy_(torch.from_numpy(rng.integers(-4, 5, c.k.shape)))
    q = torch.from_numpy(rng.integers(-4, 5, (2 * new, heads, dim))).to(device="cuda", dtype=c.k.dtype)
    scale = float(np.float32(scale2 * np.log(2.0)))
    rows = c.table.shape[1] * 16
    sums = torch.zeros((2, 2, rows), device="cuda")
    starts = [0, new, 2 * new]
    ops.paged_attention_weights(c.kv, 0, q, _ints(starts), new, scale, sums, max_len=max_len)
    _, _, dot, want = om.attention(_np(c.k[0]), _np(c.v[0]), c.table, c.lengths, starts, _np(q), scale, None, np.zeros(sums.shape))
    most = np.abs(np.einsum("thd,phrd->thpr", _np(q)[:, ::heads // 2], _np(c.k[0]))).max() * abs(scale2)
    # A weight is 2^(score + norm): the score and the maximum in the norm are rounded twice each (products with the scale; sums with a logarithm), by 2^-24 of the largest score; the
    # scale's own rounding, 2^-23, counts for the distance to the maximum, below 150 where a weight is not zero; the exponential, the logarithm and the sums 2^-18.
    rel = np.log(2) * (4 * 2.0 ** -24 * most + 150 * 2.0 ** -23) + 2.0 ** -18 + (new * heads + rows) * 2.0 ** -24
    assert rel < 2e-3
    got = _np(sums)
    assert (np.abs(got - want) <= rel * want + 2.0 ** -120).all(), (np.abs(got - want) / want.clip(1e-30)).max()
    assert np.abs(got.sum(-1) - new * heads / 2).max() <= rel * new * heads / 2
