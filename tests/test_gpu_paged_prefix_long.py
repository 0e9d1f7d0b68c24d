"""Attention over shared prefixes where some sequences have far more rows of their own (or groups more shared ones) than the others: against the plain restatement
in 64 bits, and against the time of the call that knows nothing of groups."""
import numpy as np
import pytest

from tests import helpers as H

torch = pytest.importorskip("torch")
from tests.test_gpu_paged import Cache, _ints, _randn, _tree  # noqa: E402
from tests.test_gpu_paged_prefix import _cache, _check  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from ironmill_b200 import ops
    return ops.Device(0)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim, heads, kv_heads", [(64, 8, 2), (128, 8, 2), (256, 4, 2), (128, 5, 1)])
def test_long_sequences_of_no_group_beside_short_ones(dev, dtype, dim, heads, kv_heads):
    rng = H.rng_for("long-lone", dim + heads)
    groups, pages = [3, 4], [20, 18]
    new = [1] * 12
    c = _cache(dev, rng, groups, pages, [int(x) for x in rng.integers(0, 90, 7)], new, page=64, before=(1340, 3), after=(700, 1100, 1025), dim=dim, kv_heads=kv_heads, dtype=dtype)
    _check(dev, c, rng, groups, pages, new, heads, dtype, first=2)
    _check(dev, c, rng, groups, pages, new, heads, dtype, first=2, max_prefix=0, max_len=0)      # nothing said: everything may be long
    _check(dev, c, rng, groups, pages, new, heads, dtype, first=2, max_prefix=100, max_len=200)  # too little said: slower, the same results


@pytest.mark.parametrize("dim, dtype", [(64, "bf16"), (128, "f16"), (256, "bf16")])
def test_so_many_long_sequences_that_a_share_has_several(dev, dim, dtype):
    """Items that a share has all of, items cut in two, shares that go on behind short sequences in between."""
    rng = H.rng_for("long-many", dim)
    after = [int(x) for x in rng.choice([1050, 1200, 1337, 40, 0], 150)]
    pages = [10 if dim != 256 else 5]
    c = _cache(dev, rng, [2], pages, [5, 60], [1] * 152, page=128, after=after, dim=dim, kv_heads=2, dtype=dtype)
    _check(dev, c, rng, [2], pages, [1] * 152, 2, dtype)


@pytest.mark.parametrize("seqs, long_ones", [(400, 3), (130, 1), (700, 2)])
def test_long_sequences_far_apart_in_the_list(dev, seqs, long_ones):
    rng = H.rng_for("long-far", seqs)
    after = [int(x) for x in rng.integers(0, 20, seqs)]
    for i in range(long_ones):
        after[(i + 1) * seqs // (long_ones + 1) - (i == 0)] = 2900 + i
    after[-1] = 2500
    c = _cache(dev, rng, [2], [45], [5, 60], [1] * (seqs + 2), page=64, after=after, dim=64, kv_heads=1, dtype="f16")
    _check(dev, c, rng, [2], [45], [1] * (seqs + 2), 2, "f16")


@pytest.mark.parametrize("dim, nodes", [(128, 3), (64, 4), (256, 9)])
def test_trees_of_long_sequences_and_pages_that_are_not_there(dev, dim, nodes):
    rng = H.rng_for("long-trees", dim)
    new = [nodes] * 5
    c = _cache(dev, rng, [3], [22], [0, 33, 7], new, page=64, after=(1300, 1450), dim=dim, kv_heads=2)
    c.table[4, 7], c.table[3, 2:5] = -1, 1 << 30
    c.kv.point_at(_ints(c.table), _ints(c.lengths))
    mask = np.concatenate([_tree(rng, nodes) for _ in range(5)])
    _check(dev, c, rng, [3], [22], new, 8, "f16", mask=mask, strided=True, lead=2, trail=3)


@pytest.mark.parametrize("page", [5, 100])
def test_long_groups_of_wide_heads_beside_short_ones(dev, page):
    """Heads of 256 read their shared rows in tiles of 16 rows: one group behind far more than the others."""
    rng = H.rng_for("long-groups", page)
    groups = [9] + [2] * 20
    pages = [-(-3500 // page)] + [int(x) for x in rng.integers(0, 90 // page + 2, 20)]
    new = [1] * 49
    c = _cache(dev, rng, groups, pages, [int(x) for x in rng.integers(0, 60, 49)], new, page=page, dim=256, kv_heads=2, dtype="bf16")
    _check(dev, c, rng, groups, pages, new, 8, "bf16")


def test_infinities_where_nobody_looks_in_long_sequences(dev):
    for dtype, dim in (("f16", 128), ("bf16", 64), ("f16", 256)):
        rng = H.rng_for("long-nan", dim)
        new = [3, 3, 3]
        c = _cache(dev, rng, [2], [24], [9, 20], new, page=64, after=(1500,), dim=dim, dtype=dtype)
        mask = np.array([[1], [3], [5]] * 3, dtype=np.uint64)      # nobody sees node 1 but itself
        for x in (c.k, c.v):
            x[0, c.table[2, 1501 // 64], :, 1501 % 64] = np.inf
            x[0, c.table[2, 1503 // 64], :, 1503 % 64:] = np.nan   # behind the last row
        got, want = _check(dev, c, rng, [2], [24], new, 8, dtype, mask=mask, finite=False)
        keep = np.array([True] * 7 + [False, True])
        assert np.isfinite(want[keep]).all() and np.abs(got - want)[keep].max() < 2e-2


def test_a_captured_call_follows_sequences_that_become_long(dev):
    from ironmill_b200 import ops
    from tests import oracle_paged as op
    from tests.test_gpu_paged import _np
    rng = H.rng_for("long-graph")
    c = _cache(dev, rng, [3], [20], [10, 20, 30], [1] * 5, page=64, after=(1400, 1400))
    q = _randn(rng, (5, 8, 128), "f16")
    starts, bounds, pages, lengths = _ints(range(6)), _ints([0, 3]), _ints([20]), _ints(c.lengths)
    c.kv.point_at(_ints(c.table), lengths)
    scratch, out = ops.paged_prefix_attention_scratch(c.kv, 8, 1, 1, 3), torch.zeros_like(q)
    call = lambda: ops.paged_prefix_attention(c.kv, 0, q, starts, 1, 0.1, bounds, 3, pages, max_prefix=1280, max_len=1401, out=out, scratch=scratch)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for lens in ([1290, 1300, 1310, 1400, 1400], [1290, 1300, 1310, 5, 0], [1290, 1300, 1310, 20, 1333], [1280, 1290, 1300, 1024, 1023]):
        lengths.copy_(_ints(lens)), q.copy_(_randn(rng, q.shape, "f16"))
        graph.replay()
        want, _, _ = op.attention(_np(c.k[0]), _np(c.v[0]), c.table, lens, list(range(6)), _np(q), 0.1)
        assert np.abs(_np(out) - want).max() < 2e-3


def _best_us(call):
    call()
    best = float("inf")
    for _ in range(5):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        for _ in range(10):
            call()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b) * 100)
    return best


@pytest.mark.parametrize("seqs", [4, 63])
def test_one_long_sequence_is_shared_out_over_the_gpu(dev, seqs):
    """Users behind an instruction and one user of no group with as many rows: about the time of paged_attention, which reads the instruction for every one of them (a CTA
    per KV head for the long sequence took six times that for four users, twice for 63)."""
    from ironmill_b200 import ops
    rng = H.rng_for("long-time", seqs)
    prefix = 30016 if seqs == 4 else 8192
    c = Cache(dev, rng, [prefix + 128] + [128] * (seqs - 1) + [30016], [prefix + 100] * seqs + [30000], page=64, kv_heads=8, filled=False)
    shared = prefix // 64
    own = c.table[1:seqs, :2].copy()
    c.table = np.concatenate([c.table, np.full((seqs + 1, 2), -1)], 1)
    c.table[1:seqs, :shared], c.table[1:seqs, shared:shared + 2] = c.table[0, :shared], own
    c.kv.point_at(_ints(c.table), _ints(c.lengths))
    q, starts, bounds, pages = _randn(rng, (seqs + 1, 32, 128), "f16"), _ints(range(seqs + 2)), _ints([0, seqs]), _ints([shared])
    longest = max(c.lengths) + 1
    groups = _best_us(lambda: ops.paged_prefix_attention(c.kv, 0, q, starts, 1, 0.1, bounds, seqs, pages, max_prefix=prefix, max_len=longest))
    plain = _best_us(lambda: ops.paged_attention(c.kv, 0, q, starts, 1, 0.1, max_len=longest))
    assert groups < 1.3 * plain, (groups, plain)
