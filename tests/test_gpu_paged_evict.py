"""Sums of attention weights over a paged cache, and eviction by them, against the plain restatement in 64 bits (tests/oracle_paged_more.py)."""
import numpy as np
import pytest

from tests import helpers as H
from tests import oracle_paged_more as om

torch = pytest.importorskip("torch")
from tests.test_gpu_paged import TYPES, Cache, _ints, _np, _randn, _starts, _tolerance, _tree  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from ironmill_b200 import ops
    return ops.Device(0)


# ------------------------------------------------------------------------------------------------ attention with sums
def _check(dev, c, rng, new, heads, dtype, mask=None, lead=0, trail=0, layer=0, max_len=None, scale=None, cols=None, strided=False, finite=True, q=None, calls=1):
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
    rows = cols or c.table.shape[1] * page
    sums = torch.from_numpy(rng.random((len(new), 2 * nkv if strided else nkv, rows + (3 if strided else 0)))).float().cuda()
    sums = sums[:, :nkv, :rows]
    before = _np(sums)
    out = torch.full((n, 2 * heads if strided else heads, dim), 7.0, dtype=TYPES[dtype], device="cuda")[:, :heads]
    kwargs = dict(mask=None if mask is None else torch.from_numpy(full.view(np.int64)).cuda(), max_len=max_len if max_len is not None else max(a + b for a, b in zip(c.lengths, new)))
    for _ in range(calls):
        got = _np(ops.paged_attention_weights(c.kv, layer, q, _ints(starts), max(new), scale, sums, out=out, **kwargs))
    plain = ops.paged_attention(c.kv, layer, q, _ints(starts), max(new), scale, **kwargs)
    kn, vn = _np(c.k[layer]), _np(c.v[layer])
    with np.errstate(invalid="ignore", over="ignore"):
        want, mass, dot, total = om.attention(kn, vn, c.table, c.lengths, starts, _np(q), scale, full, before)
        if calls > 1:
            _, _, _, total = om.attention(kn, vn, c.table, c.lengths, starts, _np(q), scale, full, total)
    edge = np.ones(n, dtype=bool)
    edge[starts[0]:starts[-1]] = False
    assert (got[edge] == 7.0).all()
    if finite:
        assert (got[~edge] == _np(plain)[~edge]).all()
        vmax = np.abs(vn[np.isfinite(vn)]).max()
        count = max(a + b for a, b in zip(c.lengths, new))
        tol = _tolerance(want, mass, dot, dtype, dim, vmax, count, max(new) * heads // nkv)
        assert (np.abs(got - want)[~edge] <= tol[~edge]).all()
        # A weight: scores off by (dim + 8) 2^-23 of the magnitudes in them, twice that relative to the weight (and once more, when the scores are computed again for the
        # sums), the exponential, the norm and their product 2^-18; a sum of as many f32 as there are rows, and the sum that was there.
        most, rows_of = dot[~edge].max() if (~edge).any() else 0.0, max(new) * heads // nkv
        rel = 4 * (dim + 8) * 2.0 ** -23 * most + 2.0 ** -18 + (rows_of + 2) * 2.0 ** -24
        off = np.abs(_np(sums) - total)
        assert (off <= rel * np.abs(total) + calls * 2.0 ** -24 * np.abs(before) + 2.0 ** -120).all(), (off / np.abs(total).clip(1e-30)).max()
    return got[~edge], _np(sums), total, before


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads, kv_heads", [(4, 4), (8, 2), (5, 1), (24, 2), (16, 1), (40, 1)])
def test_sums_of_one_token_of_sequences_of_all_lengths(dev, dtype, dim, heads, kv_heads):
    rng = H.rng_for("sums-decode", dim + heads)
    lengths = [0, 1, 15, 16, 17, 63, 64, 65, 200, 130]
    c = Cache(dev, rng, [n + 1 for n in lengths], lengths, kv_heads=kv_heads, dim=dim, page=16, dtype=dtype)
    _check(dev, c, rng, [1] * len(lengths), heads, dtype, calls=2)


@pytest.mark.parametrize("dtype, dim, heads, kv_heads", [("f16", 128, 8, 2), ("bf16", 64, 5, 1), ("f16", 256, 6, 3), ("bf16", 128, 16, 1), ("f16", 128, 40, 1)])
def test_sums_of_short_contexts_announced_as_long_and_of_long_ones_as_short(dev, dtype, dim, heads, kv_heads):
    rng = H.rng_for("sums-announced", dim + heads)
    lengths = [0, 1, 15, 16, 63, 64, 65, 200, 130]
    c = Cache(dev, rng, [6000] + [n + 2 for n in lengths[1:]], lengths, kv_heads=kv_heads, dim=dim, page=16, dtype=dtype)
    for most in (0, 40, 6002):
        _check(dev, c, rng, [1] * len(lengths), heads, dtype, max_len=most)
    c = Cache(dev, rng, [5001, 301], [5000, 300], kv_heads=kv_heads, dim=dim, page=64, dtype=dtype)
    for most in (0, 100, 5001, 3000):
        _check(dev, c, rng, [1, 1], heads, dtype, max_len=most)


@pytest.mark.parametrize("page", [1, 5, 24, 64, 100])
@pytest.mark.parametrize("heads", [2, 8])
def test_sums_with_pages_of_any_size(dev, page, heads):
    rng = H.rng_for("sums-pages", page)
    lengths = [700, 3, 129, 64]
    c = Cache(dev, rng, [n + 9 for n in lengths], lengths, page=page)
    _check(dev, c, rng, [1, 9, 2, 5], heads, "f16")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim, heads, kv_heads", [(128, 8, 2), (64, 6, 2), (256, 4, 1), (128, 7, 1)])
@pytest.mark.parametrize("nodes", [2, 7, 26, 65])
def test_sums_of_trees(dev, dtype, dim, heads, kv_heads, nodes):
    rng = H.rng_for("sums-trees", nodes + dim + heads)
    lengths = [0, 33, 300]
    c = Cache(dev, rng, [n + nodes for n in lengths], lengths, kv_heads=kv_heads, dim=dim, page=32, dtype=dtype)
    _check(dev, c, rng, [nodes] * 3, heads, dtype, mask=np.concatenate([_tree(rng, nodes) for _ in lengths]))


@pytest.mark.parametrize("new", [[3], [17, 5], [130, 1, 64]])
@pytest.mark.parametrize("before", [0, 1, 500])
def test_sums_of_portions_of_prompts(dev, new, before):
    rng = H.rng_for("sums-prompt", sum(new) + before)
    lengths = [before + 10 * i for i in range(len(new))]
    c = Cache(dev, rng, [a + b for a, b in zip(lengths, new)], lengths, page=16, dtype="bf16")
    _check(dev, c, rng, new, 8, "bf16", calls=2)


@pytest.mark.parametrize("heads, nodes", [(8, 1), (8, 26), (8, 64)])
def test_sums_of_long_contexts_in_shares(dev, heads, nodes):
    rng = H.rng_for("sums-long", nodes)
    lengths = [9000, 1, 4321]
    c = Cache(dev, rng, [n + nodes for n in lengths], lengths, page=64, dtype="bf16")
    _check(dev, c, rng, [nodes] * 3, heads, "bf16", mask=np.concatenate([_tree(rng, nodes) for _ in lengths]) if nodes > 1 else None)


@pytest.mark.parametrize("heads, new", [(4, [5, 0, 1, 2, 0]), (16, [40, 0, 1, 17, 0])])
def test_idle_sequences_other_tokens_and_rows_behind_the_last_are_left_alone(dev, heads, new):
    rng = H.rng_for("sums-idle", heads)
    c = Cache(dev, rng, [150, 50, 200, 60, 40], [100, 50, 0, 33, 40], page=48)
    _check(dev, c, rng, new, heads, "f16", lead=3, trail=2, strided=True, layer=0)
    _, sums, _, before = _check(dev, c, rng, new, heads, "f16", cols=90)
    assert (sums[1] == before[1]).all() and (sums[4] == before[4]).all() and (sums[2, :, 1:] == before[2, :, 1:]).all()


@pytest.mark.parametrize("heads, nodes", [(4, 5), (16, 40)])
def test_sums_of_rows_that_see_nothing_and_of_pages_that_are_not_there(dev, heads, nodes):
    rng = H.rng_for("sums-empty", nodes)
    c = Cache(dev, rng, [nodes, 30 + nodes, 64 + nodes], [0, 30, 64])
    c.table[2, 1], c.table[1, 0] = 1 << 30, -7
    c.kv.point_at(_ints(c.table), _ints(c.lengths))
    mask = np.zeros((3 * nodes, 1), dtype=np.uint64)
    mask[2, 0] = 5
    for most in (None, 0):
        _, sums, total, _ = _check(dev, c, rng, [nodes] * 3, heads, "f16", mask=mask, max_len=most)
        assert (sums[0, :, 3:nodes] == 0).all() and (total[0, :, 3:nodes] == 0).all()       # new rows that nobody sees start at zero


@pytest.mark.parametrize("heads, nodes", [(4, 3), (8, 26), (8, 64)])
def test_nan_and_infinities_where_nobody_looks_do_not_reach_the_sums(dev, heads, nodes):
    for dtype, dim in (("f16", 128), ("bf16", 64)):
        rng = H.rng_for("sums-nan", dim + nodes)
        c = Cache(dev, rng, [70 + nodes], [70], page=16, dtype=dtype, dim=dim)
        mask = _tree(rng, nodes)
        mask[:, 0] &= ~np.uint64(6)                 # nobody sees nodes 1 and 2
        for node, value in ((1, np.nan), (2, np.inf)):
            r = 70 + node
            for x in (c.k, c.v):
                x[0, c.table[0, r // 16], :, r % 16] = value
        last = 70 + nodes
        for x in (c.k, c.v):
            x[0, c.table[0, (last - 1) // 16], :, (last - 1) % 16 + 1:] = np.nan
        for most in (None, 0):
            _check(dev, c, rng, [nodes], heads, dtype, mask=mask, max_len=most)


def test_sums_of_scores_far_apart(dev):
    for new, heads in ([1], 8), ([26], 8), ([64], 8):
        rng = H.rng_for("sums-far", new[0])
        c = Cache(dev, rng, [300 + new[0]], [300])
        c.k *= 8
        for scale in (4.0, -0.5, 0.0):
            _check(dev, c, rng, new, heads, "f16", scale=scale)


@pytest.mark.parametrize("heads, new", [(8, 1), (8, 30)])
def test_a_captured_call_with_sums_follows_lengths(dev, heads, new):
    from ironmill_b200 import ops
    rng = H.rng_for("sums-graph", new)
    c = Cache(dev, rng, [400, 500, 90], [300, 400, 50])
    q, starts, lengths = _randn(rng, (3 * new, heads, 128), "f16"), _ints([0, new, 2 * new, 3 * new]), _ints(c.lengths)
    c.kv.point_at(_ints(c.table), lengths)
    sums = torch.zeros((3, 2, c.table.shape[1] * 16), device="cuda")
    scratch, out = ops.paged_attention_weights_scratch(c.kv, heads, new, 530), torch.zeros_like(q)
    call = lambda: ops.paged_attention_weights(c.kv, 0, q, starts, new, 0.1, sums, max_len=530, out=out, scratch=scratch)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for lens in ([300, 400, 50], [0, 17, 1], [370, 470, 60]):
        lengths.copy_(_ints(lens)), q.copy_(_randn(rng, q.shape, "f16")), sums.zero_()
        graph.replay()
        want, _, _, total = om.attention(_np(c.k[0]), _np(c.v[0]), c.table, lens, [0, new, 2 * new, 3 * new], _np(q), 0.1, None, np.zeros(sums.shape))
        assert np.abs(_np(out) - want).max() < 2e-3 and np.abs(_np(sums) - total).max() < 1e-4
        assert abs(float(sums.sum()) - 3 * new * heads) < 1e-2


@pytest.mark.parametrize("dtype, dim, heads, new", [("f16", 128, 8, 1), ("bf16", 64, 6, 2), ("f16", 256, 4, 3)])
def test_sums_where_the_scores_have_no_room(dev, dtype, dim, heads, new):
    """A table of five million rows, of which little is there, and no word of it: scores of so many are not kept, they are computed again."""
    rng = H.rng_for("sums-no-room", dim)
    c = Cache(dev, rng, [300 + new, 77 + new], [300, 77], dim=dim, page=256, dtype=dtype)
    c.table = np.concatenate([c.table, np.full((2, 20000), -1)], 1)
    c.kv.point_at(_ints(c.table), _ints(c.lengths))
    _check(dev, c, rng, [new, new], heads, dtype, max_len=0, cols=400)


@pytest.mark.parametrize("heads, new", [(8, 1), (8, 26), (8, 64)])
def test_sums_in_a_layer_of_pages_that_lie_apart(dev, heads, new):
    rng = H.rng_for("sums-apart", new)
    c = Cache(dev, rng, [700 + new, 90 + new], [700, 90], page=32, layers=3, apart=True, dtype="bf16")
    _check(dev, c, rng, [new, new], heads, "bf16", layer=2)


# ------------------------------------------------------------------------------------------------ eviction
def _evict(dev, c, rng, budget, recent, weights=None, strided=False):
    from ironmill_b200 import ops
    layers, _, nkv, page, _ = c.k.shape
    rows = c.table.shape[1] * page
    shape = (layers, len(c.lengths), nkv, rows)
    if weights is None:
        weights = np.exp(rng.standard_normal(shape)) * (rng.random(shape) > 0.1)
    w = torch.from_numpy(np.asarray(weights)).float().cuda()
    if strided:
        w = torch.cat([w, w + 1], 1)[:, :len(c.lengths)]
    w_out = torch.full((layers + (1 if strided else 0), len(c.lengths), nkv, rows), 7.0, device="cuda")[:layers]
    ko, vo, want = _np(c.k), _np(c.v), np.full(shape, 7.0)
    lengths, got = ops.paged_evict(c.kv, w, budget, recent, weights_out=w_out)
    lens = om.evict(ko, vo, c.table, c.lengths, _np(w), want, budget, recent)
    assert got is w_out and lengths.tolist() == lens.tolist()
    assert np.array_equal(_np(got), want, equal_nan=True)
    assert np.array_equal(_np(c.k), ko, equal_nan=True) and np.array_equal(_np(c.v), vo, equal_nan=True)
    return lengths, got


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [8, 64, 80, 128, 256])
@pytest.mark.parametrize("budget, recent", [(40, 8), (40, 0), (40, 40), (1, 0), (1, 1), (300, 299)])
def test_eviction_keeps_the_heaviest_and_the_last(dev, dtype, dim, budget, recent):
    rng = H.rng_for("evict", dim + budget)
    lengths = [0, 1, 39, 40, 41, 42, 80, 333]
    c = Cache(dev, rng, lengths, lengths, kv_heads=3, dim=dim, page=7, dtype=dtype, layers=2)
    _evict(dev, c, rng, budget, recent)


@pytest.mark.parametrize("budget, recent", [(1000, 32), (1800, 900), (1999, 1), (500, 500), (1024, 0)])
def test_eviction_of_long_sequences(dev, budget, recent):
    rng = H.rng_for("evict-long", budget)
    c = Cache(dev, rng, [2000, 1024, 1500], [2000, 1024, 1500], kv_heads=2, dim=64, page=64, layers=2, apart=True)
    _evict(dev, c, rng, budget, recent, strided=True)


def test_recent_rows_that_move_by_less_than_a_batch(dev):
    """Targets of the recent rows lie over the sources of others."""
    for n, budget, recent, dim in ((700, 699, 600, 128), (700, 640, 600, 256), (513, 500, 500, 8), (400, 270, 270, 80)):
        rng = H.rng_for("evict-shift", n + budget)
        c = Cache(dev, rng, [n], [n], dim=dim, page=16)
        _evict(dev, c, rng, budget, recent)


@pytest.mark.parametrize("kind", ["zeros", "ties", "ordered", "reversed", "negative", "special", "tiny"])
def test_sums_of_all_kinds(dev, kind):
    rng = H.rng_for("evict-kinds", len(kind))
    c = Cache(dev, rng, [600, 77], [600, 77], page=32)
    shape = (1, 2, 2, c.table.shape[1] * 32)
    line = np.arange(shape[3], dtype=np.float64)
    w = {"zeros": np.zeros(shape), "ties": rng.integers(0, 4, shape).astype(np.float64), "ordered": np.broadcast_to(line, shape), "reversed": np.broadcast_to(-line, shape),
         "negative": rng.standard_normal(shape), "special": rng.choice([0.0, -0.0, np.inf, -np.inf, np.nan, 1.0, 2.0], shape), "tiny": rng.integers(0, 9, shape) * 2.0 ** -149}[kind]
    for budget, recent in ((200, 50), (60, 0), (3, 2)):
        c = Cache(dev, rng, [600, 77], [600, 77], page=32)
        _evict(dev, c, rng, budget, recent, weights=np.ascontiguousarray(w))


def test_eviction_where_pages_are_missing_and_lengths_pass_the_table(dev):
    rng = H.rng_for("evict-bad")
    c = Cache(dev, rng, [64, 64, 64], [64, 60, 40])
    c.table[0, 1], c.table[1, 3], c.table[2, 0] = 1 << 30, -7, -1
    c.lengths = [1000, 60, -3]
    c.kv.point_at(_ints(c.table), _ints(c.lengths))
    _evict(dev, c, rng, 24, 10)


def test_nothing_to_evict_and_no_sequences(dev):
    from ironmill_b200 import ops
    rng = H.rng_for("evict-none")
    c = Cache(dev, rng, [30, 20], [30, 20])
    _evict(dev, c, rng, 30, 5)
    _evict(dev, c, rng, 1 << 20, 1 << 19)
    kv = ops.PagedKV(dev, c.k, c.v, _ints(np.zeros((0, 3))), _ints(np.zeros(0)))
    lengths, w = ops.paged_evict(kv, torch.zeros((1, 0, 2, 48), device="cuda"), 5, 1)
    assert lengths.numel() == 0 and w.numel() == 0


def test_a_captured_eviction_follows_lengths_and_sums(dev):
    from ironmill_b200 import ops
    rng = H.rng_for("evict-graph")
    c = Cache(dev, rng, [300, 200], [300, 200], layers=2)
    lengths, w = _ints(c.lengths), torch.zeros((2, 2, 2, c.table.shape[1] * 16), device="cuda")
    c.kv.point_at(_ints(c.table), lengths)
    w_out, len_out = torch.zeros_like(w), torch.zeros_like(lengths)
    call = lambda: ops.paged_evict(c.kv, w, 100, 20, weights_out=w_out, lengths_out=len_out)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for lens in ([300, 200], [120, 101], [90, 280]):
        lengths.copy_(_ints(lens)), w.copy_(torch.rand(w.shape)), w_out.fill_(7.0)
        ko, vo, want = _np(c.k), _np(c.v), np.full(w.shape, 7.0)
        graph.replay()
        assert len_out.tolist() == om.evict(ko, vo, c.table, lens, _np(w), want, 100, 20).tolist()
        assert (_np(w_out) == want).all() and (_np(c.k) == ko).all() and (_np(c.v) == vo).all()


# ------------------------------------------------------------------------------------------------ together, as a server uses them
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new", [1, 12])
def test_a_run_of_appending_attending_weighing_and_evicting(dev, dtype, new):
    """Two sequences over two layers and several steps: positions go on counting while the caches stay within their budget. Nothing waits in between."""
    from ironmill_b200 import ops
    rng = H.rng_for("evict-run", new)
    budget, recent, steps, heads, page = 40, 10, 6, 8, 16
    c = Cache(dev, rng, [budget + 2 * new + 8] * 2, [20, 45], kv_heads=2, page=page, layers=2, dtype=dtype)
    rows = c.table.shape[1] * page
    starts, position = [0, new, 2 * new], [20, 45]
    angle = np.arange(200)[:, None] * 1e4 ** (-np.arange(64) / 64)
    cos, sin = (torch.from_numpy(f(angle)).float().cuda() for f in (np.cos, np.sin))
    norm = (1 + _randn(rng, (128,), "f32", 0.1)).float()
    w = [torch.rand((2, 2, 2, rows), device="cuda"), torch.zeros((2, 2, 2, rows), device="cuda")]
    k64, v64, w64 = _np(c.k), _np(c.v), _np(w[0])
    lens = list(c.lengths)
    lengths = _ints(lens)
    ins, outs = [], []
    for _ in range(steps):
        at = np.concatenate([np.arange(p, p + new) for p in position])
        x = [(_randn(rng, (2 * new, heads, 128), dtype), _randn(rng, (2 * new, 2, 128), dtype), _randn(rng, (2 * new, 2, 128), dtype)) for _ in range(2)]
        ins.append((at, x))
        c.kv.point_at(c.kv.page_table, lengths)
        for layer, (q, k, v) in enumerate(x):
            q = ops.paged_append(c.kv, layer, k, v, _ints(starts), q=q, cos=cos, sin=sin, positions=_ints(at), q_norm=norm, k_norm=norm)
            outs.append((q, ops.paged_attention_weights(c.kv, layer, q, _ints(starts), new, 0.088, w[0][layer], max_len=rows)))
        c.kv.point_at(c.kv.page_table, lengths + new)
        lengths, _ = ops.paged_evict(c.kv, w[0], budget, recent, weights_out=w[1])
        w.reverse()
        position = [p + new for p in position]
    torch.cuda.synchronize()
    # the same from the restatement: what the kernels rounded (rotated queries and keys) is taken from it, so that both choose among the same sums up to f32
    for step, (at, x) in enumerate(ins):
        for layer, (q, k, v) in enumerate(x):
            turned, _, _ = om.append(k64[layer], v64[layer], c.table, lens, starts, _np(k), _np(v), _np(q), _np(cos), _np(sin), 128, False, [at], _np(norm), _np(norm), 1e-6)
            k64[layer] = np.where(k64[layer] == 0, 0, torch.from_numpy(k64[layer]).to(TYPES[dtype]).double().numpy())
            got_q, got = outs[2 * step + layer]
            assert np.abs(_np(got_q) - turned).max() < 0.05
            want, mass, dot, w64[layer] = om.attention(k64[layer], v64[layer], c.table, lens, starts, _np(got_q), 0.088, None, w64[layer])
            assert np.abs(_np(got) - want).max() < (3e-2 if dtype == "bf16" else 4e-3)
        lens = [n + new for n in lens]
        out64 = np.zeros_like(w64)
        lens = om.evict(k64, v64, c.table, lens, w64, out64, budget, recent).tolist()
        w64 = out64
    assert lengths.tolist() == lens
    for s, n in enumerate(lens):
        assert np.abs(_np(w[0])[:, s, :, :n] - w64[:, s, :, :n]).max() < 1e-2
