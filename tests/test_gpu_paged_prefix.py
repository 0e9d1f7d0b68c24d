"""Attention of sequences that share their first pages against the plain restatement in 64 bits (tests/oracle_paged.py), which knows nothing of groups."""
import numpy as np
import pytest

from tests import helpers as H
from tests import oracle_paged as op

torch = pytest.importorskip("torch")
from tests.test_gpu_paged import TYPES, Cache, _ints, _np, _randn, _starts, _tolerance, _tree  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from ironmill_b200 import ops
    return ops.Device(0)


def _shared(c, groups, pages):
    """The sequences of every group (counts) get the first one's first pages, `pages` of them."""
    at = 0
    for n, k in zip(groups, pages):
        c.table[at:at + n, :k] = c.table[at, :k]
        at += n
    c.kv.point_at(_ints(c.table), _ints(c.lengths))


def _check(dev, c, rng, groups, pages, new, heads, dtype, mask=None, lead=0, trail=0, first=0, layer=0, max_len=None, max_prefix=None, scale=None, strided=False, finite=True, max_new=None,
           max_group_new=None, q=None):
    """groups: sequences of each; first: sequences before the first group."""
    from ironmill_b200 import ops
    _, _, nkv, page, dim = c.k.shape
    starts = _starts(new, lead)
    n = starts[-1] + trail
    scale = dim ** -0.5 if scale is None else scale
    if q is None:
        q = _randn(rng, (n, heads, dim), dtype)
    if strided:
        q = torch.cat([q, torch.zeros_like(q)], 1)[:, :heads]
    full = None
    if mask is not None:
        full = np.zeros((n, mask.shape[1]), dtype=np.uint64)
        full[starts[0]:starts[-1]] = mask
    bounds = [first + sum(groups[:i]) for i in range(len(groups) + 1)]
    of_group = [starts[b] - starts[a] for a, b in zip(bounds, bounds[1:])]
    out = torch.full((n, 2 * heads if strided else heads, dim), 7.0, dtype=TYPES[dtype], device="cuda")[:, :heads]
    got = _np(ops.paged_prefix_attention(
        c.kv, layer, q, _ints(starts), max_new or max(new), scale, _ints(bounds), max_group_new or max(of_group + [1]), _ints(pages),
        max_prefix=max_prefix if max_prefix is not None else max(list(pages) + [0]) * page, mask=None if mask is None else torch.from_numpy(full.view(np.int64)).cuda(),
        max_len=max_len if max_len is not None else max(a + b for a, b in zip(c.lengths, new)), out=out))
    kn, vn = _np(c.k[layer]), _np(c.v[layer])
    with np.errstate(invalid="ignore", over="ignore"):
        want, mass, dot = op.attention(kn, vn, c.table, c.lengths, starts, _np(q), scale, full)
    edge = np.ones(n, dtype=bool)
    edge[starts[0]:starts[-1]] = False
    assert (got[edge] == 7.0).all()
    got, want, mass, dot = got[~edge], want[~edge], mass[~edge], dot[~edge]
    if finite:
        vmax = np.abs(vn[np.isfinite(vn)]).max()
        off = np.abs(got - want)
        # as for one sequence; the shared rows' weights go by the rows of the whole group
        rows = max([max_new or max(new)] + [max_group_new or max(of_group + [1])]) * heads // nkv
        tol = _tolerance(want, mass, dot, dtype, dim, vmax, max(a + b for a, b in zip(c.lengths, new)), rows)
        assert (off <= tol).all(), (off - tol).max()
    return got, want


def _cache(dev, rng, groups, pages, rest, new, page=16, before=(), after=(), **more):
    """Sequences of `groups`, the first `before` and the last `after` of none; rest: rows of their own."""
    prefix = [0] * len(before) + [k * page for n, k in zip(groups, pages) for _ in range(n)] + [0] * len(after)
    lengths = [a + b for a, b in zip(prefix, list(before) + list(rest) + list(after))]
    c = Cache(dev, rng, [a + b for a, b in zip(lengths, new)], lengths, page=page, **more)
    at = len(before)
    for n, k in zip(groups, pages):
        c.table[at:at + n, :k] = c.table[at, :k]
        at += n
    c.kv.point_at(_ints(c.table), _ints(c.lengths))
    return c


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads, kv_heads", [(4, 4), (8, 2), (5, 1), (24, 2), (16, 1), (40, 1)])
def test_one_token_each_in_groups_of_all_sizes(dev, dtype, dim, heads, kv_heads):
    rng = H.rng_for("prefix-decode", dim + heads)
    groups, pages = [1, 5, 3, 12], [4, 0, 9, 13]
    rest = [int(x) for x in rng.integers(0, 90, 21)]
    c = _cache(dev, rng, groups, pages, rest, [1] * 21, kv_heads=kv_heads, dim=dim, dtype=dtype)
    _check(dev, c, rng, groups, pages, [1] * 21, heads, dtype)


@pytest.mark.parametrize("heads, kv_heads, seqs", [(8, 2, 4), (8, 2, 5), (8, 2, 32), (8, 2, 33), (8, 1, 40), (8, 2, 70)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_tiles_of_16_of_128_and_of_256_rows(dev, dtype, heads, kv_heads, seqs):
    rng = H.rng_for("prefix-tiles", seqs)
    c = _cache(dev, rng, [seqs], [40], [int(x) for x in rng.integers(0, 40, seqs)], [1] * seqs, kv_heads=kv_heads, dtype=dtype)
    _check(dev, c, rng, [seqs], [40], [1] * seqs, heads, dtype)


@pytest.mark.parametrize("page", [1, 5, 24, 64, 100])
def test_prefixes_end_inside_a_tile(dev, page):
    rng = H.rng_for("prefix-pages", page)
    groups, pages = [3, 2], [-(-190 // page), -(-33 // page)]
    c = _cache(dev, rng, groups, pages, [0, 5, 70, 1, 129], [1, 2, 9, 5, 1], page=page)
    _check(dev, c, rng, groups, pages, [1, 2, 9, 5, 1], 8, "f16")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim, heads, kv_heads", [(128, 8, 2), (64, 6, 2), (256, 4, 1)])
@pytest.mark.parametrize("nodes", [2, 7, 26, 65])
def test_trees_behind_a_shared_prefix(dev, dtype, dim, heads, kv_heads, nodes):
    rng = H.rng_for("prefix-trees", nodes + dim)
    groups, pages = [2, 3], [5, 11]
    c = _cache(dev, rng, groups, pages, [0, 33, 7, 100, 1], [nodes] * 5, kv_heads=kv_heads, dim=dim, page=32, dtype=dtype)
    mask = np.concatenate([_tree(rng, nodes) for _ in range(5)])
    _check(dev, c, rng, groups, pages, [nodes] * 5, heads, dtype, mask=mask)


def test_sequences_of_no_group_before_and_behind_and_idle_ones(dev):
    rng = H.rng_for("prefix-outside")
    groups, pages, new = [2, 0, 3], [3, 7, 6], [4, 1, 0, 7, 1, 1, 0, 3, 2]
    for dtype in ("f16", "bf16"):
        c = _cache(dev, rng, groups, pages, [10, 0, 5, 90, 31], new, before=(70, 3), after=(0, 200), dtype=dtype)
        _check(dev, c, rng, groups, pages, new, 8, dtype, lead=3, trail=2, first=2, strided=True)


def test_no_groups_at_all(dev):
    rng = H.rng_for("prefix-none")
    c = _cache(dev, rng, [], [], [], [1, 5], before=(40, 300))
    _check(dev, c, rng, [], [], [1, 5], 8, "f16", first=2)
    _check(dev, c, rng, [0, 0], [2, 3], [1, 5], 8, "f16", first=1)       # groups without sequences


def test_long_prefixes_are_cut_into_shares(dev):
    rng = H.rng_for("prefix-long")
    for dtype, seqs, dim in (("f16", 3, 128), ("bf16", 9, 64), ("bf16", 40, 128)):
        c = _cache(dev, rng, [seqs, 1], [150, 70], [300] * seqs + [4000], [1] * (seqs + 1), page=64, dim=dim, dtype=dtype)
        _check(dev, c, rng, [seqs, 1], [150, 70], [1] * (seqs + 1), 4, dtype)
        _check(dev, c, rng, [seqs, 1], [150, 70], [1] * (seqs + 1), 4, dtype, max_len=0, max_prefix=0)
        _check(dev, c, rng, [seqs, 1], [150, 70], [1] * (seqs + 1), 4, dtype, max_len=100, max_prefix=17)    # too small: slower, the same results


def test_many_groups_and_many_sequences(dev):
    rng = H.rng_for("prefix-many")
    groups = [int(x) for x in rng.integers(0, 4, 300)]
    pages = [int(x) for x in rng.integers(0, 6, 300)]
    n = sum(groups)
    new = [int(x) for x in rng.integers(0, 3, n)]
    c = _cache(dev, rng, groups, pages, [int(x) for x in rng.integers(0, 60, n)], new, kv_heads=1, dim=64)
    _check(dev, c, rng, groups, pages, new, 2, "f16", max_len=0, max_new=2)


def test_rows_that_see_nothing_and_pages_that_are_not_there(dev):
    rng = H.rng_for("prefix-empty")
    for heads, seqs in ((4, 2), (16, 6)):
        c = _cache(dev, rng, [seqs, 1], [2, 0], [0] * seqs + [0], [5] * (seqs + 1))
        mask = np.zeros((5 * (seqs + 1), 1), dtype=np.uint64)
        mask[-2, 0] = 5
        got, _ = _check(dev, c, rng, [seqs, 1], [2, 0], [5] * (seqs + 1), heads, "f16", mask=mask)
        assert (got[-5:-2] == 0).all() and (got[-1] == 0).all() and (got[-2] != 0).all() and (got[:-5] != 0).any((1, 2)).all()
        c.table[:seqs, 1] = 1 << 29
        c.kv.point_at(_ints(c.table), _ints(c.lengths))
        _check(dev, c, rng, [seqs, 1], [2, 0], [5] * (seqs + 1), heads, "f16", mask=mask)
        c.table[:seqs, :2] = -1
        c.kv.point_at(_ints(c.table), _ints(c.lengths))
        got, _ = _check(dev, c, rng, [seqs, 1], [2, 0], [5] * (seqs + 1), heads, "f16", mask=mask)
        assert (got[:-5] == 0).all()


def test_infinities_and_nan_in_shared_and_own_rows(dev):
    """Rows that nobody sees (behind the last one of a page, nodes that are no ancestors) do not matter; a NaN in a shared row reaches every token of the group."""
    for dtype, dim, seqs in (("f16", 128, 2), ("bf16", 64, 9), ("bf16", 128, 40), ("f16", 256, 3)):
        rng = H.rng_for("prefix-nan", dim + seqs)
        c = _cache(dev, rng, [seqs], [6], [20] * seqs, [3] * seqs, page=16, dtype=dtype)  if dim == 128 else _cache(dev, rng, [seqs], [6], [20] * seqs, [3] * seqs, page=16, dtype=dtype, dim=dim)
        mask = np.array([[1], [3], [5]] * seqs, dtype=np.uint64)        # nobody sees node 1 but itself
        for s in range(seqs):
            for x in (c.k, c.v):
                x[0, c.table[s, 7], :, 7:] = np.nan                    # rows 119 .. 127: the sequence ends at row 119
                x[0, c.table[s, 7], :, 5] = np.inf                     # node 1
        got, want = _check(dev, c, rng, [seqs], [6], [3] * seqs, 8, dtype, mask=mask, finite=False)
        keep = np.arange(3 * seqs) % 3 != 1
        assert np.isfinite(want[keep]).all() and np.abs(got - want)[keep].max() < 2e-2
        c.v[0, c.table[0, 2], 1, 3, 7] = np.nan
        got, want = _check(dev, c, rng, [seqs], [6], [3] * seqs, 8, dtype, mask=mask, finite=False)
        bad = np.isnan(want[keep])
        assert bad[:, 4:, 7].all() and bad.sum() == bad.shape[0] * 4 and (np.isnan(got[keep]) == bad).all()
        assert np.abs(got[keep] - want[keep])[~bad].max() < 2e-2


def test_scores_far_apart_between_the_shared_rows_and_the_others(dev):
    for seqs in (2, 12, 40):
        rng = H.rng_for("prefix-far", seqs)
        c = _cache(dev, rng, [seqs], [8], [40] * seqs, [2] * seqs)
        first = _ints(c.table[0, :8]).long()
        c.k[:, first] *= 30
        for scale in (1.0, -0.5, 0.0):
            _check(dev, c, rng, [seqs], [8], [2] * seqs, 8, "f16", scale=scale)
        c.k[:, first] /= 900
        c.k *= 30
        _check(dev, c, rng, [seqs], [8], [2] * seqs, 8, "f16", scale=1.0)


def test_more_new_tokens_than_announced_are_left_alone(dev):
    from ironmill_b200 import ops
    rng = H.rng_for("prefix-announced")
    c = _cache(dev, rng, [3], [4], [10, 10, 10], [6, 6, 6])
    q = _randn(rng, (18, 8, 128), "f16")
    out = torch.full_like(q, 7.0)
    ops.paged_prefix_attention(c.kv, 0, q, _ints([0, 6, 12, 18]), 4, 0.1, _ints([0, 3]), 13, _ints([4]), out=out)
    want, _, _ = op.attention(_np(c.k[0]), _np(c.v[0]), c.table, c.lengths, [0, 6, 12, 18], _np(q), 0.1)
    told = np.array([t % 6 < 4 and t < 13 for t in range(18)])
    assert np.abs(_np(out) - want)[told].max() < 2e-3 and (_np(out)[~told] == 7.0).all()


def test_what_the_arrays_say_is_checked_on_the_device(dev):
    """Starts that decrease or pass the arrays, group numbers out of range, prefixes longer than the table: something comes out or nothing, inside the arrays."""
    from ironmill_b200 import ops
    rng = H.rng_for("prefix-bad")
    c = _cache(dev, rng, [2, 2], [2, 2], [5, 5, 5, 5], [1, 1, 1, 1])
    q = _randn(rng, (4, 4, 128), "f16")
    for starts, bounds, pages in (([0, 1, 2, 3, 9], [0, 2, 4], [2, 2]), ([3, 2, 1, 0, 4], [0, 2, 4], [2, 2]), ([0, 1, 2, 3, 4], [0, 99, 4], [2, 2]), ([0, 1, 2, 3, 4], [-5, 2, 1 << 30], [2, 2]),
                                  ([0, 1, 2, 3, 4], [4, 2, 0], [2, 2]), ([0, 1, 2, 3, 4], [0, 2, 4], [1 << 30, -4])):
        out = ops.paged_prefix_attention(c.kv, 0, q, _ints(starts), 1, 0.1, _ints(bounds), 2, _ints(pages))
        torch.cuda.synchronize()
        assert out.shape == q.shape
    good = ops.paged_prefix_attention(c.kv, 0, q, _ints([0, 1, 2, 3, 4]), 1, 0.1, _ints([0, 2, 4]), 2, _ints([2, 2]))
    want, _, _ = op.attention(_np(c.k[0]), _np(c.v[0]), c.table, c.lengths, [0, 1, 2, 3, 4], _np(q), 0.1)
    assert np.abs(_np(good) - want).max() < 2e-3


def test_a_captured_call_follows_lengths_prefixes_and_tables(dev):
    from ironmill_b200 import ops
    rng = H.rng_for("prefix-graph")
    c = _cache(dev, rng, [6, 3], [5, 9], [20] * 9, [1] * 9)
    q = _randn(rng, (9, 8, 128), "f16")
    starts, bounds, pages, lengths, table = _ints(range(10)), _ints([0, 6, 9]), _ints([5, 9]), _ints(c.lengths), _ints(c.table)
    c.kv.point_at(table, lengths)
    scratch = ops.paged_prefix_attention_scratch(c.kv, 8, 1, 2, 9)
    out = torch.zeros_like(q)
    call = lambda: ops.paged_prefix_attention(c.kv, 0, q, starts, 1, 0.1, bounds, 9, pages, out=out, scratch=scratch)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for new_bounds, new_pages in (([0, 6, 9], [5, 9]), ([0, 6, 9], [2, 0]), ([0, 5, 9], [5, 0]), ([6, 9, 9], [9, 3])):
        bounds.copy_(_ints(new_bounds)), pages.copy_(_ints(new_pages)), q.copy_(_randn(rng, q.shape, "f16"))
        lens = [int(x) - int(rng.integers(0, 9)) for x in c.lengths]
        lengths.copy_(_ints(lens))
        graph.replay()
        want, _, _ = op.attention(_np(c.k[0]), _np(c.v[0]), c.table, lens, list(range(10)), _np(q), 0.1)
        assert np.abs(_np(out) - want).max() < 2e-3


def test_two_calls_at_once_on_streams_of_their_own(dev):
    from ironmill_b200 import ops
    rng = H.rng_for("prefix-streams")
    c = _cache(dev, rng, [20], [60], [200] * 20, [1] * 20)
    qs = [_randn(rng, (20, 8, 128), "f16") for _ in range(2)]
    args = (_ints(range(21)), 1, 0.1, _ints([0, 20]), 20, _ints([60]))
    alone = [ops.paged_prefix_attention(c.kv, 0, q, *args) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    for _ in range(5):
        got = []
        for q, st in zip(qs, streams):
            with torch.cuda.stream(st):
                got.append(ops.paged_prefix_attention(c.kv, 0, q, *args))
        torch.cuda.synchronize()
        for a, b in zip(got, alone):
            assert (a == b).all()


def test_no_tokens_and_one_sequence_alone(dev):
    from ironmill_b200 import ops
    rng = H.rng_for("prefix-alone")
    c = _cache(dev, rng, [1], [3], [7], [1])
    _check(dev, c, rng, [1], [3], [1], 4, "f16")
    q = torch.zeros((0, 4, 128), dtype=torch.float16, device="cuda")
    assert ops.paged_prefix_attention(c.kv, 0, q, _ints([0, 0]), 1, 0.1, _ints([0, 1]), 1, _ints([3])).shape == q.shape


@pytest.mark.parametrize("seqs, nodes", [(3, 1), (12, 1), (40, 1), (4, 26)])
def test_calls_in_a_row_follow_what_the_ones_before_them_wrote(dev, seqs, nodes):
    """Appending and attending in turns on one stream, without waiting: each call finds what those before it wrote, whatever starts beside what."""
    from ironmill_b200 import ops
    rng = H.rng_for("prefix-chain", seqs + nodes)
    c = _cache(dev, rng, [seqs], [30], [8] * seqs, [nodes] * seqs, page=32)
    starts, n = _ints(_starts([nodes] * seqs)), seqs * nodes
    steps = [(_randn(rng, (n, 8, 128), "f16"), _randn(rng, (n, 2, 128), "f16"), _randn(rng, (n, 2, 128), "f16")) for _ in range(6)]
    got = []
    for q, k, v in steps:
        ops.paged_append(c.kv, 0, k, v, starts)
        got.append(ops.paged_prefix_attention(c.kv, 0, q, starts, nodes, 0.1, _ints([0, seqs]), n, _ints([30])))
    torch.cuda.synchronize()
    for (q, k, v), out in zip(steps, got):
        ops.paged_append(c.kv, 0, k, v, starts)
        torch.cuda.synchronize()
        want, _, _ = op.attention(_np(c.k[0]), _np(c.v[0]), c.table, c.lengths, _starts([nodes] * seqs), _np(q), 0.1)
        assert np.abs(_np(out) - want).max() < 2e-3


@pytest.mark.parametrize("seqs, nodes", [(3, 1), (40, 1), (6, 26)])
def test_a_layer_of_pages_that_lie_apart(dev, seqs, nodes):
    rng = H.rng_for("prefix-apart", seqs + nodes)
    c = _cache(dev, rng, [seqs], [9], [int(x) for x in rng.integers(0, 300, seqs)], [nodes] * seqs, page=32, layers=3, apart=True, dtype="bf16")
    _check(dev, c, rng, [seqs], [9], [nodes] * seqs, 8, "bf16", layer=1, strided=True)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_few_shared_rows_in_small_tiles_and_many_in_large_ones_agree(dev, dim):
    """The same call by either kernel: what is announced of the prefix decides."""
    rng = H.rng_for("prefix-either", dim)
    for seqs in (5, 9, 20):
        c = _cache(dev, rng, [seqs], [6], [int(x) for x in rng.integers(0, 60, seqs)], [1] * seqs, page=64, dim=dim)
        for most in (6 * 64, 0, 1, 100000):
            _check(dev, c, rng, [seqs], [6], [1] * seqs, 8, "f16", max_prefix=most, max_len=0)
