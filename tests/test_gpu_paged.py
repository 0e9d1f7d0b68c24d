"""The paged cache's operators and beam selection on the GPU against their plain restatement in 64 bits (tests/oracle_paged.py)."""
import numpy as np
import pytest

from tests import helpers as H
from tests import oracle_paged as op

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


@pytest.fixture(scope="module")
def dev():
    from ironmill_b200 import ops
    return ops.Device(0)


def _np(t):
    return t.detach().double().cpu().numpy()


def _ints(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def _randn(rng, shape, dtype, scale=1.0):
    return torch.from_numpy(rng.standard_normal(shape) * scale).to(device="cuda", dtype=TYPES[dtype])


class Cache:
    """A pool of pages in no order, with a table for sequences of `room` rows each."""

    def __init__(self, dev, rng, room, lengths, kv_heads=2, dim=128, page=16, dtype="f16", layers=1, apart=False, filled=True):
        from ironmill_b200 import ops
        need = [-(-r // page) for r in room]
        width, total = max(max(need), 1) + 1, sum(need) + 2
        order = rng.permutation(total)
        table = np.full((len(room), width), -1)
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n]
            at += n
        shape = (layers, total, kv_heads, page, dim)
        if apart:   # keys and values of a page side by side, all layers of it too
            pool = torch.zeros((total, layers, 2, kv_heads, page, dim), dtype=TYPES[dtype], device="cuda")
            self.k, self.v = pool[:, :, 0].transpose(0, 1), pool[:, :, 1].transpose(0, 1)
        else:
            self.k, self.v = (torch.zeros(shape, dtype=TYPES[dtype], device="cuda") for _ in range(2))
        if filled:
            for x in (self.k, self.v):
                x.copy_(_randn(rng, shape, dtype))
        self.table, self.lengths, self.page = table, list(lengths), page
        self.kv = ops.PagedKV(dev, self.k, self.v, _ints(table), _ints(lengths))


def _starts(new, lead=0):
    return [lead + sum(new[:i]) for i in range(len(new) + 1)]


# ------------------------------------------------------------------------------------------------ append
def _check_append(dev, c, rng, new, heads, dtype, rotary, neighbours=False, table="f16", positions=None, lead=0, trail=0, layer=0, in_place=False, max_pos=None):
    from ironmill_b200 import ops
    _, pages, nkv, page, dim = c.k.shape
    starts = _starts(new, lead)
    n = starts[-1] + trail
    qkv = _randn(rng, (n, heads + 2 * nkv, dim), dtype)
    q, k, v = qkv.split([heads, nkv, nkv], 1)
    most = max_pos or max(a + b for a, b in zip(c.lengths, new)) + 1
    angle = np.arange(most)[:, None] * 1e4 ** (-2.0 * np.arange(dim // 2) / max(rotary, 2))
    cos, sin = (torch.from_numpy(f(angle)).to(device="cuda", dtype=TYPES[table]) for f in (np.cos, np.sin))
    ko, vo = _np(c.k), _np(c.v)
    qn, kn, vn = _np(q), _np(k), _np(v)
    kwargs = dict(cos=cos, sin=sin, rotary_dim=rotary, neighbours=neighbours) if rotary else {}
    if heads:
        out = q if in_place else torch.full((n, heads, dim), 7.0, dtype=TYPES[dtype], device="cuda")
        kwargs.update(q=q, q_out=out)
    ops.paged_append(c.kv, layer, k, v, _ints(starts), positions=None if positions is None else _ints(positions), **kwargs)
    want = op.append(ko[layer], vo[layer], c.table, c.lengths, starts, kn, vn, qn if heads else None, _np(cos), _np(sin), rotary, neighbours, positions)
    # two products and a sum in f32 (each off by at most 2^-24 of its terms, here at most sqrt(2) * 6), then one rounding of the result
    eps = torch.finfo(TYPES[dtype]).eps / 2
    near = lambda a, b: (np.abs(a - b) <= eps * np.abs(b) * (1 + 1e-3) + 12 * 2.0 ** -23 + 2.0 ** -25).all()  # noqa: E731
    assert near(_np(c.k), ko)
    assert (_np(c.v) == vo).all()
    if heads:
        got, before = _np(out), qn if in_place else np.full(qn.shape, 7.0)
        want = np.where(np.isnan(want), before, want)
        assert near(got, want)
        untouched = np.ones(n, dtype=bool)
        untouched[starts[0]:starts[-1]] = False
        assert (got[untouched] == before[untouched]).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim, rotary, neighbours", [(128, 128, False), (128, 64, False), (128, 64, True), (64, 64, True), (64, 24, False), (256, 256, False), (80, 80, False),
                                                     (80, 36, False), (80, 38, True), (8, 8, False), (8, 2, True), (128, 0, False)])
def test_append_matches_the_formula(dev, dtype, dim, rotary, neighbours):
    rng = H.rng_for("append", dim * 1000 + rotary)
    c = Cache(dev, rng, [40, 9, 70, 1], [30, 0, 33, 0], kv_heads=3, dim=dim, page=7, dtype=dtype)
    _check_append(dev, c, rng, [10, 5, 0, 1], 5, dtype, rotary, neighbours, "f32" if dim % 16 else "f16")


def test_append_without_queries_in_a_layer_of_pages_that_lie_apart(dev):
    rng = H.rng_for("append-apart")
    c = Cache(dev, rng, [100, 100], [64, 13], page=16, layers=3, apart=True)
    _check_append(dev, c, rng, [1, 1], 0, "f16", 128, layer=2)


def test_append_rotates_queries_in_place_and_leaves_other_tokens_alone(dev):
    for rotary in (128, 40):
        rng = H.rng_for("append-place", rotary)
        c = Cache(dev, rng, [30, 30, 30], [0, 7, 29], dtype="bf16")
        _check_append(dev, c, rng, [3, 4, 1], 9, "bf16", rotary, lead=2, trail=3, in_place=True)


def test_append_at_the_depths_of_a_tree_and_outside_the_tables(dev):
    rng = H.rng_for("append-tree")
    c = Cache(dev, rng, [60, 60], [20, 41])
    _check_append(dev, c, rng, [6, 6], 4, "f16", 128, positions=[20, 21, 21, 22, 22, 23, 41, 42, -1, 42, 1 << 30, 43], max_pos=43)


def test_append_past_the_table_and_to_pages_that_are_not_there(dev):
    rng = H.rng_for("append-bad")
    c = Cache(dev, rng, [32, 32, 32], [30, 16, 0], page=16)     # the table holds 48 rows, its last column names no page
    c.table[1, 1] = 99
    c.table[2, 0] = -5
    c.lengths[0] = 46
    c.kv.point_at(_ints(c.table), _ints([46, 16, -3]))
    c.lengths[2] = -3
    _check_append(dev, c, rng, [4, 3, 20], 4, "f16", 128, max_pos=60)


def test_append_finds_the_sequence_of_a_token_among_many(dev):
    rng = H.rng_for("append-many")
    n = 1500
    new = rng.integers(0, 3, n).tolist()
    c = Cache(dev, rng, [4] * n, rng.integers(0, 3, n).tolist(), kv_heads=1, dim=8, page=2)
    _check_append(dev, c, rng, new, 1, "f16", 8)


# ------------------------------------------------------------------------------------------------ attention
def _tolerance(out, mass, dot, dtype, dim, vmax, count, rows=1):
    """Scores: dim products summed in f32 and two factors, off by (dim + 8) 2^-23 of the sum of their magnitudes (relative to a weight: twice that);
    exponentials, sums and the join 2^-18; weights as two 16-bit terms 2^-16 (bf16) or 2^-21 and half the smallest fp16 number, 2^-25, each; one
    rounding. More than 128 rows of a KV head: weights in one 16-bit term, each off by half a step of its type, and so their sum over |values|."""
    eps = torch.finfo(TYPES[dtype]).eps / 2
    score = 2 * (dim + 8) * 2.0 ** -23 * dot[..., None]
    weights = eps * (1 + 2.0 ** -7) if rows > 128 and dim < 256 else 2.0 ** -16 if dtype == "bf16" else 2.0 ** -21
    tiny = 0.0 if dtype == "bf16" else count * 2.0 ** -25 * vmax + 2.0 ** -25
    return eps * np.abs(out) * (1 + 1e-3) + (score + weights + 2.0 ** -18) * mass + tiny


def _tree(rng, n, words=None):
    """Bits of ancestors and itself of a random tree of n nodes, int64 [n, words]."""
    words = words or -(-n // 64)
    sees, rows = [], []
    for t in range(n):
        sees.append((sees[int(rng.integers(max(0, t - 6), t))] if t else 0) | 1 << t)
        rows.append([(sees[t] >> 64 * w) & (1 << 64) - 1 for w in range(words)])
    return np.array(rows, dtype=np.uint64)


def _check_attention(dev, c, rng, new, heads, dtype, mask=None, lead=0, trail=0, layer=0, max_len=None, max_new=None, scale=None, q=None, strided=False, finite=True):
    from ironmill_b200 import ops
    _, pages, nkv, page, dim = c.k.shape
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
    out = torch.full((n, 2 * heads if strided else heads, dim), 7.0, dtype=TYPES[dtype], device="cuda")[:, :heads]
    got = ops.paged_attention(c.kv, layer, q, _ints(starts), max_new or max(new), scale, mask=None if mask is None else torch.from_numpy(full.view(np.int64)).cuda(),
                              max_len=max_len if max_len is not None else max(a + b for a, b in zip(c.lengths, new)), out=out)
    got = _np(got)
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
        tol = _tolerance(want, mass, dot, dtype, dim, vmax, max(a + b for a, b in zip(c.lengths, new)), (max_new or max(new)) * heads // nkv)
        assert (off <= tol).all(), (off - tol).max()
    return got, want


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads, kv_heads", [(4, 4), (8, 2), (5, 1), (24, 2), (16, 1), (40, 1)])
def test_one_token_of_sequences_of_all_lengths(dev, dtype, dim, heads, kv_heads):
    rng = H.rng_for("decode", dim + heads)
    lengths = [0, 1, 15, 16, 17, 63, 64, 65, 200, 130]
    c = Cache(dev, rng, [n + 1 for n in lengths], lengths, kv_heads=kv_heads, dim=dim, page=16, dtype=dtype)
    _check_attention(dev, c, rng, [1] * len(lengths), heads, dtype)


@pytest.mark.parametrize("dtype, dim, heads, kv_heads", [("f16", 128, 8, 2), ("bf16", 64, 5, 1), ("f16", 256, 6, 3), ("bf16", 128, 16, 1)])
def test_short_contexts_where_long_ones_are_announced(dev, dtype, dim, heads, kv_heads):
    """Nothing says that the contexts are short: they go by shares of all tiles instead of a cluster per item; NaN and missing pages too."""
    rng = H.rng_for("announced-long", dim + heads)
    lengths = [0, 1, 15, 16, 63, 64, 65, 200, 130]
    c = Cache(dev, rng, [6000] + [n + 2 for n in lengths[1:]], lengths, kv_heads=kv_heads, dim=dim, page=16, dtype=dtype)
    c.table[7, 3] = 1 << 20
    c.kv.point_at(_ints(c.table), _ints(lengths))
    _check_attention(dev, c, rng, [1] * len(lengths), heads, dtype, max_len=0)
    mask = np.array([[1], [2]] * len(lengths), dtype=np.uint64)      # no node sees the other one
    for i, n in enumerate(lengths):
        for x in (c.k, c.v):
            x[0, c.table[i, n // 16], :, n % 16] = 1.0 if i % 2 else -1.0
            x[0, c.table[i, (n + 1) // 16], :, (n + 1) % 16] = np.nan if i % 3 == 0 else 2.0
    mask[1::2] = 1
    _check_attention(dev, c, rng, [2] * len(lengths), heads, dtype, mask=mask, max_len=0)
    _check_attention(dev, c, rng, [2] * len(lengths), heads, dtype, mask=mask)


@pytest.mark.parametrize("page", [1, 5, 8, 24, 64, 100, 256])
def test_pages_of_any_size_end_inside_a_tile(dev, page):
    rng = H.rng_for("pages", page)
    lengths = [700, 3, 129, 64]
    c = Cache(dev, rng, [n + 9 for n in lengths], lengths, page=page)
    _check_attention(dev, c, rng, [1, 9, 2, 5], 8, "f16")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim, heads, kv_heads", [(128, 8, 2), (64, 6, 2), (256, 4, 1), (128, 7, 1), (128, 16, 2)])
@pytest.mark.parametrize("nodes", [2, 7, 26, 64, 65, 130])
def test_trees(dev, dtype, dim, heads, kv_heads, nodes):
    rng = H.rng_for("trees", nodes + dim + heads)
    lengths = [0, 33, 300]
    c = Cache(dev, rng, [n + nodes for n in lengths], lengths, kv_heads=kv_heads, dim=dim, page=32, dtype=dtype)
    mask = np.concatenate([_tree(rng, nodes) for _ in lengths])
    _check_attention(dev, c, rng, [nodes] * len(lengths), heads, dtype, mask=mask)


def test_trees_of_different_sizes_and_a_sequence_without_any(dev):
    rng = H.rng_for("trees-ragged")
    new, lengths = [5, 0, 17, 1, 40], [100, 50, 0, 77, 128]
    c = Cache(dev, rng, [a + b for a, b in zip(lengths, new)], lengths, page=48)
    mask = np.concatenate([_tree(rng, n, 1) for n in new if n])
    _check_attention(dev, c, rng, new, 8, "f16", mask=mask, lead=3, trail=2, strided=True)


@pytest.mark.parametrize("new", [[3], [17, 5], [300, 1, 64], [129]])
@pytest.mark.parametrize("before", [0, 1, 500])
def test_portions_of_prompts_are_causal(dev, new, before):
    rng = H.rng_for("prompt", sum(new) + before)
    lengths = [before + 10 * i for i in range(len(new))]
    c = Cache(dev, rng, [a + b for a, b in zip(lengths, new)], lengths, page=16, dtype="bf16")
    _check_attention(dev, c, rng, new, 8, "bf16")


def test_rows_whose_mask_leaves_nothing_are_zero(dev):
    rng = H.rng_for("empty")
    c = Cache(dev, rng, [10, 40], [0, 30])
    mask = np.zeros((10, 1), dtype=np.uint64)
    mask[2, 0] = 5
    got, _ = _check_attention(dev, c, rng, [5, 5], 4, "f16", mask=mask)
    assert (got[[0, 1, 3, 4]] == 0).all() and (got[5:] != 0).all()


def test_a_mask_of_more_and_of_fewer_words_than_the_tree_has(dev):
    rng = H.rng_for("words")
    c = Cache(dev, rng, [170], [50])
    _check_attention(dev, c, rng, [70], 4, "f16", mask=_tree(rng, 70, 5))
    few = np.full((70, 1), (1 << 64) - 1, dtype=np.uint64)     # nodes from 64 on are seen by nobody; bits past the tree mean nothing
    _check_attention(dev, c, rng, [70], 4, "f16", mask=few)
    _check_attention(dev, c, rng, [9], 4, "f16", mask=few[:9])


def test_pages_that_are_not_there_and_lengths_past_the_table_read_nothing(dev):
    rng = H.rng_for("bad-pages")
    c = Cache(dev, rng, [64, 64, 64, 64], [60, 40, 20, 64])
    c.table[0, 1], c.table[1, 0], c.table[2, :] = 1 << 30, -7, -1
    c.lengths = [60, 40, -9, 1000]
    c.kv.point_at(_ints(c.table), _ints(c.lengths))
    got, _ = _check_attention(dev, c, rng, [2, 2, 2, 2], 8, "f16", max_len=0)
    assert (got[4:6] == 0).all()


def test_infinities_and_nan_in_rows_that_are_not_seen(dev):
    for dtype, dim, nodes, heads in (("f16", 128, 26, 8), ("bf16", 64, 5, 4), ("f16", 256, 3, 4), ("bf16", 128, 64, 8)):
        rng = H.rng_for("nan", dim)
        c = Cache(dev, rng, [70 + nodes], [70], page=16, dtype=dtype)
        mask = _tree(rng, nodes)
        mask[:, 0] &= ~np.uint64(6)                 # nobody sees nodes 1 and 2
        for node, value in ((1, np.nan), (2, np.inf)):
            r = 70 + node
            for x in (c.k, c.v):
                x[0, c.table[0, r // 16], :, r % 16] = value
        # what a page holds behind the last row, too
        last = 70 + nodes
        for x in (c.k, c.v):
            x[0, c.table[0, (last - 1) // 16], :, (last - 1) % 16 + 1:] = np.nan
        _check_attention(dev, c, rng, [nodes], heads, dtype, mask=mask)


def test_a_nan_reaches_the_rows_that_see_it_and_no_other(dev):
    rng = H.rng_for("nan-seen")
    c = Cache(dev, rng, [200], [150], page=16)
    r = 150 + 3
    c.v[0, c.table[0, r // 16], 0, r % 16, 5] = np.nan
    got, want = _check_attention(dev, c, rng, [9], 8, "f16", finite=False)
    bad = np.isnan(want)
    assert bad[3:, :4, 5].all() and bad.sum() == 6 * 4
    assert (np.isnan(got) == bad).all()
    assert np.abs(got - want)[~bad].max() < 2e-3


def test_largest_values_and_scores_far_apart(dev):
    rng = H.rng_for("far")
    c = Cache(dev, rng, [300], [290])
    c.v.copy_(torch.where(c.v > 0, 65504.0, -65504.0))
    c.k *= 8
    _check_attention(dev, c, rng, [4], 8, "f16", scale=4.0)
    _check_attention(dev, c, rng, [4], 8, "f16", scale=-0.5)
    _check_attention(dev, c, rng, [4], 8, "f16", scale=0.0)
    for nodes in (9, 40):           # the tensor cores' tiles, narrow and wide
        c = Cache(dev, rng, [330], [290])
        c.k *= 8
        mask = _tree(rng, nodes)
        for scale in (4.0, -0.5, 0.0):
            _check_attention(dev, c, rng, [nodes], 8, "f16", scale=scale, mask=mask)
            _check_attention(dev, c, rng, [nodes], 8, "f16", scale=scale)
        c.v.copy_(torch.where(c.v > 0, 65504.0, -65504.0))
        _check_attention(dev, c, rng, [nodes], 8, "f16", scale=4.0)


@pytest.mark.parametrize("heads, new", [(2, 1), (2, 11), (40, 1)])
@pytest.mark.parametrize("dim", [64, 256])
def test_more_sequences_than_threads(dev, heads, new, dim):
    """Shares of 700 sequences: places found in several rounds; nothing says that the contexts are short."""
    rng = H.rng_for("many", heads + new)
    n = 700
    lengths = rng.integers(0, 150, n).tolist()
    counts = [int(x) for x in rng.integers(0, new + 1, n)]
    c = Cache(dev, rng, [a + b for a, b in zip(lengths, counts)] + [], lengths, kv_heads=1, dim=dim, page=32)
    wide = np.concatenate([c.table, np.full((n, 60), -1)], 1)
    c.kv.point_at(_ints(wide), _ints(lengths))
    c.table = wide
    _check_attention(dev, c, rng, counts, heads, "f16", max_len=0, max_new=new)


@pytest.mark.parametrize("heads, nodes", [(8, 10), (16, 40)])
def test_tensor_core_tiles_with_missing_pages_and_empty_rows(dev, heads, nodes):
    rng = H.rng_for("tc-bad", nodes)
    lengths = [200, 40, 0, 64]
    c = Cache(dev, rng, [n + nodes for n in lengths], lengths, page=16)
    c.table[0, 1], c.table[0, 12], c.table[1, 0], c.table[2, :] = 1 << 30, -7, 99999, -1
    c.kv.point_at(_ints(c.table), _ints(lengths))
    mask = np.concatenate([_tree(rng, nodes) for _ in lengths])
    mask[3 * nodes + 2] = 0
    got, _ = _check_attention(dev, c, rng, [nodes] * 4, heads, "f16", mask=mask)
    assert (got[2 * nodes:3 * nodes] == 0).all()            # a sequence without any page
    mask = np.zeros((nodes, 1), dtype=np.uint64)            # an empty cache, and nodes that see nothing but for one
    mask[5] = 33
    c = Cache(dev, rng, [nodes], [0])
    got, _ = _check_attention(dev, c, rng, [nodes], heads, "f16", mask=mask)
    assert (np.delete(got, 5, 0) == 0).all() and (got[5] != 0).all()


@pytest.mark.parametrize("dtype, nodes", [("f16", 1), ("bf16", 26), ("bf16", 64)])
def test_long_contexts_are_cut_into_shares_and_joined(dev, dtype, nodes):
    rng = H.rng_for("long", nodes)
    lengths = [9000, 1, 4321]
    c = Cache(dev, rng, [n + nodes for n in lengths], lengths, page=64, dtype=dtype)
    mask = np.concatenate([_tree(rng, nodes) for _ in lengths]) if nodes > 1 else None
    _check_attention(dev, c, rng, [nodes] * 3, 4, dtype, mask=mask)


def test_more_new_tokens_than_announced_are_left_alone(dev):
    from ironmill_b200 import ops
    rng = H.rng_for("announced")
    c = Cache(dev, rng, [300], [100])
    q = _randn(rng, (64, 8, 128), "f16")
    out = torch.full_like(q, 7.0)
    ops.paged_attention(c.kv, 0, q, _ints([0, 64]), 4, 0.1, out=out)
    want, _, _ = op.attention(_np(c.k[0]), _np(c.v[0]), c.table, [100], [0, 64], _np(q), 0.1)
    assert np.abs(_np(out[:4]) - want[:4]).max() < 2e-3 and (out[4:] == 7.0).all()


def test_token_starts_past_the_arrays_are_left_alone(dev):
    from ironmill_b200 import ops
    rng = H.rng_for("starts")
    c = Cache(dev, rng, [50, 50], [10, 20])
    q = _randn(rng, (2, 4, 128), "f16")
    out = torch.full_like(q, 7.0)
    ops.paged_attention(c.kv, 0, q, _ints([0, 1, 3]), 2, 0.1, out=out)     # the second sequence claims a token that is not there
    assert (out[0] != 7.0).any() and (out[1] == 7.0).all()
    ops.paged_attention(c.kv, 0, q, _ints([1, 0, 2]), 2, 0.1, out=out)     # it decreases
    torch.cuda.synchronize()


def test_page_offsets_past_32_bits(dev):
    from ironmill_b200 import ops
    pages, page = 40, 64
    stride = 1 << 27                                       # elements from page to page: the last lie 5 G elements in
    rng = H.rng_for("offsets")
    pool = torch.zeros(pages * stride, dtype=torch.float16, device="cuda")
    k = pool.as_strided((1, pages, 2, page, 128), (pages * stride, stride, page * 128, 128, 1))
    v = pool[1 << 20:].as_strided((1, pages, 2, page, 128), (pages * stride, stride, page * 128, 128, 1))
    table = np.array([[39, 2, 35, 17], [38, 37, 0, 36]])
    kv = ops.PagedKV(dev, k, v, _ints(table), _ints([0, 0]))
    rows = _randn(rng, (2 * 240, 2, 128), "f16")
    vals = _randn(rng, (2 * 240, 2, 128), "f16")
    ops.paged_append(kv, 0, rows, vals, _ints([0, 240, 480]))
    kn, vn = np.zeros((pages, 2, page, 128)), np.zeros((pages, 2, page, 128))
    op.append(kn, vn, table, [0, 0], [0, 240, 480], _np(rows), _np(vals))
    for i in range(pages):
        assert (_np(k[0, i]) == kn[i]).all() and (_np(v[0, i]) == vn[i]).all()
    kv.point_at(_ints(table), _ints([239, 230]))
    q = _randn(rng, (2, 8, 128), "f16")
    out = ops.paged_attention(kv, 0, q, _ints([0, 1, 2]), 1, 0.1, max_len=240)
    want, mass, dot = op.attention(kn, vn, table, [239, 230], [0, 1, 2], _np(q), 0.1)
    assert (np.abs(_np(out) - want) <= _tolerance(want, mass, dot, "f16", 128, 6, 240)).all()
    lens = ops.paged_keep(kv, _ints([[0, 9], [5, 7]]), _ints([2, 2]))
    torch.cuda.synchronize()
    assert lens.tolist() == [241, 232] and (_np(k[0, 36, :, 38]) == kn[36, :, 43]).all()


def test_no_tokens_and_no_sequences(dev):
    from ironmill_b200 import ops
    rng = H.rng_for("none")
    c = Cache(dev, rng, [10], [5])
    q = torch.empty((0, 4, 128), dtype=torch.float16, device="cuda")
    assert ops.paged_attention(c.kv, 0, q, _ints([0, 0]), 1, 0.1).shape == (0, 4, 128)
    ops.paged_append(c.kv, 0, q[:, :2], q[:, :2], _ints([0, 0]))
    kv = ops.PagedKV(dev, c.k, c.v, _ints(np.zeros((0, 2))), _ints([]))
    assert ops.paged_keep(kv, _ints(np.zeros((0, 1))), _ints([])).shape == (0,)
    assert ops.paged_attention(kv, 0, _randn(rng, (2, 4, 128), "f16"), _ints([0]), 1, 0.1).shape == (2, 4, 128)
    score, _, _ = ops.beam_select(dev, torch.empty((0, 2, 10), device="cuda"), torch.empty((0, 2), device="cuda"), 2)
    assert score.shape == (0, 2)
    assert (_np(c.k) != 0).any()


# ------------------------------------------------------------------------------------------------ keep, reorder
@pytest.mark.parametrize("page, layers, dim, apart", [(16, 1, 128, False), (5, 3, 64, True), (64, 2, 72, False), (1, 2, 8, False)])
def test_keep_moves_the_accepted_path_in_every_layer(dev, page, layers, dim, apart):
    from ironmill_b200 import ops
    rng = H.rng_for("keep", page)
    lengths = [0, 7, 31, 100, 12, 3]
    c = Cache(dev, rng, [n + 40 for n in lengths], lengths, page=page, layers=layers, dim=dim, apart=apart, dtype="bf16")
    accepted = np.zeros((6, 12), dtype=np.int64)
    counts = [3, 0, 12, 1, 99, -4]
    for i, n in enumerate([3, 0, 12, 1, 12, 0]):
        accepted[i, :n] = np.sort(rng.choice(40, n, replace=False))
    kn, vn = _np(c.k), _np(c.v)
    lens = ops.paged_keep(c.kv, _ints(accepted), _ints(counts))
    want = op.keep(kn, vn, c.table, lengths, accepted, counts)
    assert lens.tolist() == want.tolist()
    assert (_np(c.k) == kn).all() and (_np(c.v) == vn).all()


def test_keep_with_long_paths_bad_places_and_pages(dev):
    from ironmill_b200 import ops
    rng = H.rng_for("keep-bad")
    c = Cache(dev, rng, [1200, 64, 64], [3, 40, 30], page=16)
    accepted = np.zeros((3, 600), dtype=np.int64)
    accepted[0] = np.sort(rng.choice(np.arange(1, 1190), 600, replace=False))
    accepted[1, :4] = [1, 1 << 30, -5, 6]
    accepted[2, :4] = [1, 3, 18, 20]
    c.table[2, 3] = 5000                      # rows 48..63 are not there
    c.kv.point_at(_ints(c.table), _ints(c.lengths))
    kn, vn = _np(c.k), _np(c.v)
    lens = ops.paged_keep(c.kv, _ints(accepted), _ints([600, 4, 4]))
    assert lens.tolist() == op.keep(kn, vn, c.table, c.lengths, accepted, [600, 4, 4]).tolist()
    assert (_np(c.k) == kn).all() and (_np(c.v) == vn).all()


@pytest.mark.parametrize("beams, page, layers, dim, apart", [(4, 16, 2, 128, False), (1, 16, 1, 64, False), (7, 5, 3, 72, True), (8, 64, 1, 128, False), (100, 3, 1, 8, False)])
def test_reorder_copies_last_pages_of_parents_with_several_children(dev, beams, page, layers, dim, apart):
    from ironmill_b200 import ops
    rng = H.rng_for("reorder", beams)
    groups = 3
    lengths = np.repeat(rng.integers(0, 3 * page, groups), beams)
    if beams == 7:
        lengths = rng.integers(0, 3 * page, groups * beams)        # beams that ended earlier
    c = Cache(dev, rng, [int(n) // page * page + page for n in lengths], lengths.tolist(), page=page, layers=layers, dim=dim, apart=apart)
    for parents in (rng.integers(0, beams, groups * beams), np.tile(np.arange(beams), groups), np.full(groups * beams, beams - 1), rng.integers(-1, beams + 1, groups * beams)):
        kn, vn = _np(c.k), _np(c.v)
        table, lens = ops.paged_reorder(c.kv, _ints(parents), beams)
        want_t, want_l = op.reorder(kn, vn, c.table, lengths, parents, beams)
        assert (table.cpu().numpy() == want_t).all() and lens.tolist() == want_l.tolist()
        assert (_np(c.k) == kn).all() and (_np(c.v) == vn).all()


def test_reorder_with_full_tables(dev):
    from ironmill_b200 import ops
    rng = H.rng_for("reorder-full")
    c = Cache(dev, rng, [16, 16, 16], [16, 16, 16], page=8)
    kv = ops.PagedKV(dev, c.k, c.v, _ints(c.table)[:, :2], _ints([16, 16, 5]))
    kn, vn = _np(c.k), _np(c.v)
    table, lens = ops.paged_reorder(kv, _ints([0, 0, 1]), 3)
    want_t, want_l = op.reorder(kn, vn, c.table[:, :2], [16, 16, 5], [0, 0, 1], 3)
    assert (table.cpu().numpy() == want_t).all() and lens.tolist() == want_l.tolist() == [16, 16, 16]
    assert (_np(c.k) == kn).all()


# ------------------------------------------------------------------------------------------------ selection
def _check_select(dev, logits, scores, picks, done=None, end_token=-1):
    from ironmill_b200 import ops
    got = ops.beam_select(dev, logits, scores, picks, done=done, end_token=end_token)
    score, parent, token = (x.cpu().numpy() for x in got)
    with np.errstate(all="ignore"):
        want = op.select(_np(logits), _np(scores), picks, None if done is None else done.cpu().numpy(), end_token)
    # a thread sums up to vocab / 256 exponentials (at least eight slots each) in f32, each off by 2^-21; then the score is rounded
    slack = (logits.shape[2] / 256 + 64) * 2.0 ** -24 + 2.0 ** -20
    for g, rows in enumerate(want):
        for i, (value, beam, tok) in enumerate(rows[:picks]):
            near = [r[0] for j, r in enumerate(rows) if j != i and r[1] != beam]
            if np.isfinite(value) and any(abs(value - n) < 2 * slack for n in near):
                continue                       # two beams' values nearer than their sums are exact: either order is right
            assert (parent[g, i], token[g, i]) == (beam, tok), (g, i, rows)
            if np.isfinite(value):
                assert abs(score[g, i] - value) <= slack + 2.0 ** -24 * abs(value)
            else:
                assert score[g, i] == -np.inf
    return got


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("groups, beams, vocab, picks", [(1, 1, 1, 1), (1, 4, 7, 64), (3, 2, 500, 4), (2, 5, 2049, 10), (1, 8, 32768, 16), (40, 3, 1001, 3), (60, 8, 700, 5), (1, 3, 90000, 6), (1, 7, 20011, 64), (5, 2, 65536, 2), (1, 64, 4096, 64), (2, 4, 151936, 8)])
def test_selection(dev, dtype, groups, beams, vocab, picks):
    rng = H.rng_for("select", vocab + beams)
    _check_select(dev, _randn(rng, (groups, beams, vocab), dtype, 3.0), _randn(rng, (groups, beams), "f32", 2.0), picks)


def test_selection_ties_go_to_the_lowest_beam_and_token(dev):
    x = torch.zeros((2, 3, 5000), device="cuda")
    x[1, :, 4321] = 1.0
    x[1, :, 77] = 1.0
    _, parent, token = _check_select(dev, x, torch.zeros((2, 3), device="cuda"), 8)
    assert parent[0].tolist() == [0] * 8 and token[0].tolist() == list(range(8))
    assert list(zip(parent[1].tolist(), token[1].tolist()))[:6] == [(0, 77), (0, 4321), (1, 77), (1, 4321), (2, 77), (2, 4321)]
    rng = H.rng_for("select-ties")
    few = torch.from_numpy(rng.integers(0, 4, (2, 4, 30000)).astype(np.float32)).cuda()    # thousands of equal values
    few[:, 1:] = few[:, :1]
    for dtype in TYPES.values():
        _check_select(dev, few.to(dtype), torch.zeros((2, 4), device="cuda"), 16)


def test_selection_of_masked_vocabularies(dev):
    rng = H.rng_for("select-masked")
    for dtype in ("f16", "bf16", "f32"):
        x = _randn(rng, (2, 2, 9000), dtype, 2.0)
        lowest = torch.finfo(x.dtype).min
        allowed = torch.zeros(9000, dtype=torch.bool, device="cuda")
        allowed[[3, 4500, 8999]] = True
        scores = torch.tensor([[0.0, -1.0], [0.0, -np.inf]], device="cuda")
        _, parent, token = _check_select(dev, torch.where(allowed, x, -np.inf), scores, 8)
        assert token[0].tolist()[6:] == [-1, -1] and sorted(token[1].tolist()[:3]) == [3, 4500, 8999] and token[1].tolist()[3:] == [-1] * 5
        assert (parent[1, :3] == 0).all()
        if dtype != "bf16":   # (bf16's lowest value is below f32's range with a score added: -inf once rounded)
            _check_select(dev, torch.where(allowed, x, lowest), scores * 0.5, 8)


def test_selection_leaves_out_beams_without_a_distribution(dev):
    rng = H.rng_for("select-nan")
    x = _randn(rng, (1, 5, 3000), "f32", 2.0)
    x[0, 0, 17], x[0, 1, 2999], x[0, 2] = np.nan, np.inf, -np.inf
    scores = torch.tensor([[5.0, 5.0, 5.0, np.nan, 0.0]], device="cuda")
    _, parent, _ = _check_select(dev, x, scores, 10)
    assert (parent == 4).all()
    x[0, 4, 5] = np.nan
    score, parent, token = _check_select(dev, x, scores, 10)
    assert (score == -np.inf).all() and (parent == -1).all() and (token == -1).all()


def test_selection_with_finished_beams(dev):
    rng = H.rng_for("select-done")
    x = _randn(rng, (3, 4, 6000), "f16", 3.0)
    x[0, 1] = np.nan                                     # a finished beam's logits are not read
    done = torch.tensor([[0, 1, 0, 0], [1, 1, 1, 1], [0, 0, 0, 0]], dtype=torch.bool, device="cuda")
    scores = _randn(rng, (3, 4), "f32")
    _, parent, token = _check_select(dev, x, scores, 6, done=done, end_token=2)
    assert token[1].tolist() == [2, 2, 2, 2, -1, -1]


def test_selection_of_rows_that_lie_apart_and_start_anywhere(dev):
    rng = H.rng_for("select-strides")
    for dtype in ("f16", "f32"):
        x = _randn(rng, (2 * 3 * 1003 + 1,), dtype, 3.0)[1:].view(2, 3, 1003)[:, :, :997]
        _check_select(dev, x, _randn(rng, (2, 3), "f32"), 6)


# ------------------------------------------------------------------------------------------------ together, streams, graphs
def test_draft_and_verify_as_plain_decoding(dev):
    """Tokens that go in one by one, and the same ones as nodes of a tree of which a path is kept: the same rows and outputs."""
    from ironmill_b200 import ops
    heads, nkv, dim, page, layers, steps = 8, 2, 128, 16, 2, 4
    rng = H.rng_for("verify")
    lengths = [21, 5]
    parent_of = [-1, 0, 0, 1, 2, 2, 4]                       # a tree of seven nodes; kept: 0 -> 2 -> 4 -> 6
    path, depth = [0, 2, 4, 6], [0, 1, 1, 2, 2, 2, 3]
    angle = np.arange(200)[:, None] * 1e4 ** (-2.0 * np.arange(dim // 2) / dim)
    cos, sin = (torch.from_numpy(f(angle)).cuda().half() for f in (np.cos, np.sin))
    c = Cache(dev, rng, [n + 40 for n in lengths], lengths, layers=layers, page=page)
    other = Cache(dev, H.rng_for("verify"), [n + 40 for n in lengths], lengths, layers=layers, page=page)
    assert (c.table == other.table).all() and (c.k == other.k).all()
    x = {n: _randn(rng, (layers, 2, 7, h, dim), "f16") for n, h in (("q", heads), ("k", nkv), ("v", nkv))}
    mask = np.zeros((14, 1), dtype=np.int64)
    for t in range(7):
        mask[t, 0] = 1 << t | (int(mask[parent_of[t], 0]) if parent_of[t] >= 0 else 0)
    mask[7:] = mask[:7]
    positions = _ints([n + d for n in lengths for d in depth])
    starts = _ints([0, 7, 14])
    tree_out = []
    for layer in range(layers):
        q, k, v = (x[n][layer].reshape(14, -1, dim) for n in "qkv")
        q = ops.paged_append(c.kv, layer, k, v, starts, q=q, cos=cos, sin=sin, positions=positions)
        tree_out.append(ops.paged_attention(c.kv, layer, q, starts, 7, dim ** -0.5, mask=torch.from_numpy(mask).cuda()).view(2, 7, heads, dim))
    c.kv.point_at(c.kv.page_table, ops.paged_keep(c.kv, _ints([path, path]), _ints([4, 3])))
    assert c.kv.lengths.tolist() == [25, 8]
    one = _ints([0, 1, 2])
    for i in range(steps):
        for layer in range(layers):
            q, k, v = (x[n][layer][:, path[i]].contiguous() for n in "qkv")
            q = ops.paged_append(other.kv, layer, k, v, one, q=q, cos=cos, sin=sin)
            out = ops.paged_attention(other.kv, layer, q, one, 1, dim ** -0.5)
            # the same rows in another order of sums: both within an f16 rounding of outputs of size one
            assert (out - tree_out[layer][:, path[i]]).abs().max() <= 2.0 ** -9
        other.kv.point_at(other.kv.page_table, other.kv.lengths + 1)
    for s, n in enumerate([25, 8]):
        for r in range(n):
            p = c.table[s, r // page]
            assert (c.k[:, p, :, r % page] == other.k[:, p, :, r % page]).all() and (c.v[:, p, :, r % page] == other.v[:, p, :, r % page]).all()


def test_a_beam_search_over_shared_pages(dev):
    """Steps of append, attention, selection and reordering against the same search with a contiguous cache per beam in plain arithmetic."""
    from ironmill_b200 import ops
    heads, nkv, dim, page, beams, vocab, steps = 4, 2, 64, 4, 4, 300, 9
    rng = H.rng_for("beams")
    prompt = 10
    embed, head = _randn(rng, (vocab, 3, dim), "f32"), _randn(rng, (heads * dim, vocab), "f32", 0.3)
    shared, own = prompt // page, -(-(prompt + steps) // page) + 1
    pages = shared + beams * own
    k, v = (_randn(rng, (1, pages, nkv, page, dim), "f16") for _ in range(2))
    table = np.array([list(range(shared)) + list(range(shared + b * own, shared + b * own + own)) for b in range(beams)])
    for x in (k, v):                                                     # the rows of the prompt's last page
        for b in range(1, beams):
            x[0, table[b, shared]] = x[0, table[0, shared]]
    kv = ops.PagedKV(dev, k, v, _ints(table), _ints([prompt] * beams))
    gather = lambda x, b: np.concatenate([_np(x[0, p]).transpose(1, 0, 2) for p in table[b]])[:prompt]  # noqa: E731
    plain = [(gather(k, b), gather(v, b), [], 0.0 if b == 0 else -np.inf) for b in range(beams)]
    scores = torch.tensor([[p[3] for p in plain]], dtype=torch.float32, device="cuda")
    tokens = torch.zeros(beams, dtype=torch.long, device="cuda")
    said, starts = [], _ints(range(beams + 1))
    for step in range(steps):
        e = embed[tokens].half()
        kn, vn, q = e[:, :1].repeat(1, nkv, 1), e[:, 1:2].repeat(1, nkv, 1), e[:, 2:].repeat(1, heads, 1)
        ops.paged_append(kv, 0, kn, vn, starts)
        out = ops.paged_attention(kv, 0, q, starts, 1, dim ** -0.5)
        kv.point_at(kv.page_table, kv.lengths + 1)
        logits = (out.float().view(beams, -1) @ head).view(1, beams, vocab)
        scores, parent, token = ops.beam_select(dev, logits, scores, beams)
        # the same step over contiguous rows
        rows = []
        for b, (pk, pv, _, _) in enumerate(plain):
            pk, pv = np.concatenate([pk, _np(kn[b:b + 1])]), np.concatenate([pv, _np(vn[b:b + 1])])
            o = np.zeros((heads, dim))
            for h in range(heads):
                s = pk[:, h // 2] @ _np(q[b, h]) * dim ** -0.5
                w = np.exp(s - s.max())
                o[h] = w @ pv[:, h // 2] / w.sum()
            assert np.abs(o - _np(out[b])).max() <= 2.0 ** -9, (step, b)
            rows.append((pk, pv))
        best = op.select(_np(logits), np.array([[p[3] for p in plain]]), beams)[0]
        assert parent[0].tolist() == [r[1] for r in best[:beams]] and token[0].tolist() == [r[2] for r in best[:beams]]
        plain = [(rows[b][0], rows[b][1], plain[b][2] + [t], value) for value, b, t in best[:beams]]
        kv.point_at(*ops.paged_reorder(kv, parent[0], beams))
        tokens = token[0].long()
    got = kv.page_table.cpu().numpy()
    for b in range(beams):
        rows = np.concatenate([_np(k[0, p]).transpose(1, 0, 2) for p in got[b]])[:prompt + steps]
        assert (rows == plain[b][0]).all()


def _calls(dev, c, rng, nodes):
    from ironmill_b200 import ops
    n = len(c.lengths) * nodes
    q, k, v = _randn(rng, (n, 8, 128), "f16"), _randn(rng, (n, 2, 128), "f16"), _randn(rng, (n, 2, 128), "f16")
    starts = _ints([nodes * i for i in range(len(c.lengths) + 1)])
    scratch = ops.paged_attention_scratch(c.kv, 8, nodes)
    x, scores = _randn(rng, (2, 3, 5000), "f32"), _randn(rng, (2, 3), "f32")
    select = ops.beam_select_scratch(dev, 2, 3, 5000, 6)

    def run():
        ops.paged_append(c.kv, 0, k, v, starts)
        out = ops.paged_attention(c.kv, 0, q, starts, nodes, 0.09, scratch=scratch)
        return [out, *ops.beam_select(dev, x, scores, 6, scratch=select)]
    return run, q


def test_on_a_stream_of_its_own_and_in_a_graph_that_is_replayed(dev):
    rng = H.rng_for("graph")
    c = Cache(dev, rng, [900, 300, 64], [880, 250, 40])
    run, q = _calls(dev, c, rng, 11)
    want = [x.clone() for x in run()]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = run()
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for _ in range(3):
        for x in outs:
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, outs))
    # what the device arrays say at the time of the replay is what counts
    c.kv.lengths.copy_(_ints([100, 200, 1]))
    graph.replay()
    torch.cuda.synchronize()
    fresh = run()
    assert all(torch.equal(a, b) for a, b in zip(fresh, outs)) and not torch.equal(want[0], outs[0])


def test_two_streams_with_scratch_of_their_own(dev):
    rng = H.rng_for("streams")
    runs = []
    for i in range(2):
        c = Cache(dev, rng, [2000, 2000], [1900 - i, 1500])
        runs.append(_calls(dev, c, rng, 9)[0])
    want = [[x.clone() for x in r()] for r in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in runs]
    for _ in range(10):
        got = []
        for s, r in zip(streams, runs):
            with torch.cuda.stream(s):
                got.append(r())
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_refusals_on_a_device(dev):
    from ironmill_b200 import CudaSysError, ops
    rng = H.rng_for("refusals")
    c = Cache(dev, rng, [9000], [40], page=64)
    q = _randn(rng, (1, 4, 128), "f16")
    with pytest.raises(CudaSysError, match="scratch"):
        ops.paged_attention(c.kv, 0, q, _ints([0, 1]), 1, 0.1, scratch=torch.empty(64, dtype=torch.uint8, device="cuda"))
    with pytest.raises(CudaSysError, match="scratch"):
        ops.beam_select(dev, torch.zeros((1, 9, 10), device="cuda"), torch.zeros((1, 9), device="cuda"), 1, scratch=torch.empty(8, dtype=torch.uint8, device="cuda"))
    with pytest.raises(CudaSysError, match="layer"):
        ops.paged_append(c.kv, 1, q[:, :2].contiguous(), q[:, 2:].contiguous(), _ints([0, 1]))
    for call in (lambda: ops.paged_attention(c.kv, 0, q.bfloat16(), _ints([0, 1]), 1, 0.1), lambda: ops.paged_attention(c.kv, 0, q, _ints([0, 1, 2]), 1, 0.1),
                 lambda: ops.paged_attention(c.kv, 0, q.transpose(1, 2), _ints([0, 1]), 1, 0.1), lambda: ops.paged_append(c.kv, 0, q, q, _ints([0, 1])),
                 lambda: ops.paged_keep(c.kv, _ints([[0]]), _ints([0, 0])), lambda: c.kv.point_at(c.kv.page_table, _ints([1, 2]))):
        with pytest.raises(AssertionError):
            call()


def test_expanded_tensors_are_refused(dev):
    """A stride of zero means packed to the kernels: an axis that a caller has expanded must not reach them."""
    from ironmill_b200 import ops
    rng = H.rng_for("expanded")
    c = Cache(dev, rng, [40, 40, 40, 40], [20, 20, 20, 20], layers=2)
    row, scores = torch.zeros((1, 1, 100), device="cuda"), torch.zeros((2, 4), device="cuda")
    parents = _ints([0, 0, 0, 0])
    shared = c.kv.page_table[:1].expand(4, -1)
    for call in (lambda: ops.beam_select(dev, row.expand(2, 4, 100), scores, 4), lambda: ops.beam_select(dev, row.expand(1, 4, 100), scores[:1], 4),
                 lambda: ops.beam_select(dev, row.expand(2, 1, 100), scores[:, :1].contiguous(), 4), lambda: c.kv.point_at(shared, c.kv.lengths),
                 lambda: ops.PagedKV(dev, c.k[:1].expand(2, -1, -1, -1, -1), c.v[:1].expand(2, -1, -1, -1, -1), c.kv.page_table, c.kv.lengths),
                 lambda: ops.PagedKV(dev, c.k[:, :1].expand(-1, 9, -1, -1, -1), c.v[:, :1].expand(-1, 9, -1, -1, -1), c.kv.page_table, c.kv.lengths),
                 lambda: ops.paged_reorder(c.kv, parents, 4, table_out=_ints([[0] * shared.shape[1]]).expand(4, -1))):
        with pytest.raises(AssertionError):
            call()
    assert c.kv.num_seqs == 4 and c.kv.struct.table_width == shared.shape[1]
    want = ops.beam_select(dev, row.expand(2, 4, 100).contiguous(), scores, 4)  # what the caller writes instead
    assert want[1].tolist() == [[0, 0, 0, 0]] * 2 and want[2].tolist() == [[0, 1, 2, 3]] * 2


# ------------------------------------------------------------------------------------------------ many units on the tensor cores
@pytest.mark.parametrize("seqs, heads, kv_heads, dim, dtype, most", [
    (40, 8, 2, 128, "f16", 10), (40, 12, 1, 128, "bf16", 40), (45, 16, 2, 64, "f16", 33), (37, 24, 1, 64, "bf16", 5), (450, 20, 1, 128, "f16", 2), (430, 132, 1, 64, "bf16", 2)])
def test_tensor_core_tiles_of_more_units_than_a_warp_has_lanes(dev, seqs, heads, kv_heads, dim, dtype, most):
    """Narrow and wide tiles of more units than a warp has lanes, and than a block has threads; some sequences have no new token."""
    rng = H.rng_for("units", seqs + heads)
    lengths = rng.integers(0, 300, seqs).tolist()
    new = [most, *(int(x) for x in rng.integers(0, most + 1, seqs - 1))]
    c = Cache(dev, rng, [a + b for a, b in zip(lengths, new)], lengths, kv_heads=kv_heads, dim=dim, page=24, dtype=dtype)
    first = _check_attention(dev, c, H.rng_for("units-q"), new, heads, dtype)[0]
    for _ in range(3):
        assert (_check_attention(dev, c, H.rng_for("units-q"), new, heads, dtype)[0] == first).all()


# ------------------------------------------------------------------------------------------------ rows that are not finite, beside others
def _exact(kv, seq, q, scale, mask):
    """Attention of a sequence's new tokens q [new, heads, dim] in 64 bits on the GPU, with the sums that bounds on rounding need: (out, mass, dot)."""
    k, v = kv.k_pages[0], kv.v_pages[0]
    new, heads, dim = q.shape
    before, page, nkv = int(kv.lengths[seq]), k.shape[2], k.shape[1]
    row = torch.arange(before + new, device="cuda")
    at = kv.page_table[seq].long()[row // page]
    sees = torch.ones((new, before + new), dtype=torch.bool, device="cuda")
    sees[:, before:] = (mask[:, None, 0] >> torch.arange(new, device="cuda")) & 1 == 1
    out, mass, dot = (torch.zeros(s, dtype=torch.float64, device="cuda") for s in (q.shape, q.shape, q.shape[:2]))
    for h in range(heads):
        kk, vv = (x[at, h * nkv // heads, row % page].double() for x in (k, v))
        x = (q[:, h].double() @ torch.where(sees.any(0)[:, None], kk, 0.0).T * scale).masked_fill(~sees, -np.inf)
        w = torch.softmax(x, 1)
        vv = torch.where(sees.any(0)[:, None], vv, 0.0)
        out[:, h], mass[:, h] = w @ vv, w @ vv.abs()
        dot[:, h] = (q[:, h].double().abs() @ torch.where(sees.any(0)[:, None], kk, 0.0).abs().T).masked_fill(~sees, 0.0).amax(1) * scale
    return [_np(x) for x in (out, mass, dot)]


@pytest.mark.parametrize("seqs, before, heads, dtype", [(12, 24000, 8, "f16"), (12, 24000, 64, "bf16"), (3, 20000, 8, "bf16"), (60, 150, 8, "f16"), (60, 150, 64, "f16"), (1, 70000, 64, "f16")])
def test_nodes_that_nobody_sees_may_hold_anything_in_long_batches(dev, seqs, before, heads, dtype):
    """NaN and infinities in drafted rows of some sequences: long ones, whose repair takes its time, whole items and parts of them. Every row of every
    sequence against 64 bits, and the sequences without them bit by bit as they are without."""
    from ironmill_b200 import ops
    rng = H.rng_for("odd", before + heads)
    nodes, nkv, dim, page = 32, 8, 128, 64
    lengths = [before - 17 * i % 40 for i in range(seqs)]
    shared, own = 96, 2
    table = np.array([[*rng.integers(0, shared, -(-(before + nodes) // page) + 1)] for _ in range(seqs)])
    for i, n in enumerate(lengths):                                       # the drafted rows' pages are a sequence's own
        table[i, n // page:n // page + own] = shared + own * i + np.arange(own)
    torch.manual_seed(before)
    k, v = (torch.randn((1, shared + own * seqs, nkv, page, dim), device="cuda").to(TYPES[dtype]) for _ in range(2))
    kv = ops.PagedKV(dev, k, v, _ints(table), _ints(lengths))
    q = torch.randn((seqs * nodes, heads, dim), device="cuda").to(TYPES[dtype])
    starts, scale = _ints(np.arange(seqs + 1) * nodes), dim ** -0.5
    mask = np.concatenate([_tree(rng, nodes) for _ in range(seqs)])
    mask[:, 0] &= ~np.uint64(0b110000)                                    # nobody sees nodes 4 and 5
    mask = torch.from_numpy(mask.view(np.int64)).cuda()
    run = lambda: ops.paged_attention(kv, 0, q, starts, nodes, scale, mask=mask, max_len=before + nodes)  # noqa: E731
    clean = run()
    odd = [i for i in range(seqs) if i % 5 in (0, 3)]
    for i in odd:
        for node, value in ((4, np.nan), (5, np.inf)):
            r = lengths[i] + node
            k[0, table[i, r // page], i % nkv, r % page, 7] = value
            v[0, table[i, r // page], :, r % page, 100] = value
    got = run()
    rest = torch.tensor([i not in odd for i in range(seqs)]).cuda().repeat_interleave(nodes)
    assert torch.equal(got[rest], clean[rest])
    for i in {*odd[:3], *range(min(seqs, 3)), seqs - 1}:
        want, mass, dot = _exact(kv, i, q[i * nodes:i * nodes + nodes], scale, mask[i * nodes:i * nodes + nodes])
        tol = _tolerance(want, mass, dot, dtype, dim, float(v.float().nan_to_num(0, 0, 0).abs().max()), before + nodes, nodes * heads // nkv)
        assert (np.abs(_np(got[i * nodes:i * nodes + nodes]) - want) <= tol).all(), i


# ------------------------------------------------------------------------------------------------ equal beams
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("groups, beams, vocab", [(1, 8, 50257), (2, 3, 1001), (5, 16, 50257), (40, 5, 1003), (3, 7, 130001), (2, 2, 4099)])
@pytest.mark.parametrize("lead", [0, 1])
def test_equal_beams_tie_wherever_their_rows_start(dev, dtype, groups, beams, vocab, lead):
    """Beams with the same logits and scores have the same values to the last bit: a token's beams come in order, at rows of every alignment."""
    from ironmill_b200 import ops
    rng = H.rng_for("equal", vocab + beams)
    row = _randn(rng, (groups, 1, vocab), dtype)     # sums of many terms of like size, whose roundings follow their order
    for g in range(groups):                          # the two best tokens of a group
        row[g, 0, (17 * g + 5) % vocab], row[g, 0, vocab - 1 - g] = 6.0, 5.75
    x = torch.empty(groups * beams * vocab + lead, dtype=TYPES[dtype], device="cuda")[lead:].view(groups, beams, vocab)
    x.copy_(row)
    score, parent, token = (t.cpu() for t in ops.beam_select(dev, x, torch.full((groups, beams), -1.25, device="cuda"), 2 * beams))
    for g in range(groups):
        assert parent[g].tolist() == [*range(beams)] * 2
        assert token[g].tolist() == [(17 * g + 5) % vocab] * beams + [vocab - 1 - g] * beams
        assert len(set(score[g, :beams].tolist())) == len(set(score[g, beams:].tolist())) == 1


# ------------------------------------------------------------------------------------------------ long flat tails
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads, new, dim", [(1, 1, 128), (16, 1, 64), (4, 1, 256), (8, 4, 128), (8, 4, 64), (16, 16, 128), (16, 16, 64)])
@pytest.mark.parametrize("low, rows", [(-17.0625, 100003), (-17.375, 100003), (-21.0, 100003), (-12.0, 900)])
@pytest.mark.parametrize("sink_last", [False, True])
def test_a_long_tail_of_small_weights_beside_one_large_one(dev, dtype, heads, new, dim, low, rows, sink_last):
    """A row that takes nearly all of the weight and has a value of zero, and a tail whose weights (2^-17 to 2^-30 of it) are what the outputs come from."""
    from ironmill_b200 import ops
    page = 64
    pages = -(-(rows + new) // page)
    low = torch.tensor(low).to(TYPES[dtype]).item()
    k, v = (torch.zeros((1, pages, 1, page, dim), dtype=TYPES[dtype], device="cuda") for _ in range(2))
    kr, vr = k.view(-1, dim), v.view(-1, dim)              # (one KV head, pages in order)
    kr[:rows, 0], vr[:rows] = low, 1.0
    sink = rows - 1 if sink_last else 0
    kr[sink, 0], vr[sink] = 0.0, 0.0
    kr[rows:, 0] = -1000.0                                 # the new rows take nothing: 2^-1442
    kv = ops.PagedKV(dev, k, v, _ints(np.arange(pages)[None]), _ints([rows]))
    q = torch.zeros((new, heads, dim), dtype=TYPES[dtype], device="cuda")
    q[:, :, 0] = 1.0
    got = _np(ops.paged_attention(kv, 0, q, _ints([0, new]), new, 1.0, max_len=rows + new))
    # a score is one product: off by 2^-24 of it where it is scaled to powers of two, and again where the maximum is taken off; the
    # exponential, the sum and the join 2^-18; two 16-bit terms 2^-16 (bf16) or 2^-21, one 2^-9 or 2^-12; what of an fp16 weight is below 2^-37 of the largest; one rounding
    tail = np.exp(float(low)) * (rows - 1)
    want, eps = tail / (1 + tail), torch.finfo(TYPES[dtype]).eps / 2
    weights = eps if heads * new > 128 else 2.0 ** -16 if dtype == "bf16" else 2.0 ** -21
    tol = eps * want * (1 + 1e-3) + (weights + 2.0 ** -18 + 4 * abs(low) * 1.45 * 2.0 ** -24) * want
    tol += rows * 2.0 ** -37 + 2.0 ** -25 if dtype == "f16" else 0.0
    assert np.abs(got - want).max() <= tol, (got.min(), got.max(), want, tol)


# ------------------------------------------------------------------------------------------------ lengths that the table cannot hold
@pytest.mark.parametrize("nodes, heads", [(1, 4), (9, 8), (40, 16)])
def test_negative_lengths_count_as_zero_and_long_ones_as_the_table(dev, nodes, heads):
    """On pages that are all there: every operator does what it does at the lengths that these count as."""
    from ironmill_b200 import ops
    runs = []
    for lengths in ([-1, 20, -(1 << 31), 5000], [0, 20, 0, 64]):
        rng = H.rng_for("lengths", nodes)
        c = Cache(dev, rng, [64] * 4, [0, 20, 0, 64], page=16)
        table = c.table[:, :4]
        c.kv.point_at(_ints(table), _ints(lengths))
        q, k, v = _randn(rng, (4 * nodes, heads, 128), "f16"), _randn(rng, (4 * nodes, 2, 128), "f16"), _randn(rng, (4 * nodes, 2, 128), "f16")
        angle = np.arange(200)[:, None] * 1e4 ** (-2.0 * np.arange(64) / 128)
        cos, sin = (torch.from_numpy(f(angle)).cuda().half() for f in (np.cos, np.sin))
        starts = _ints(np.arange(5) * nodes)
        got = [ops.paged_append(c.kv, 0, k, v, starts, q=q, cos=cos, sin=sin), c.k.clone(), c.v.clone()]
        got.append(ops.paged_attention(c.kv, 0, q, starts, nodes, 0.09, max_len=0))
        got += [ops.paged_keep(c.kv, _ints([[0, 5, 9]] * 4), _ints([3] * 4)), c.k.clone(), c.v.clone()]
        got += [*ops.paged_reorder(c.kv, _ints([1, 1, 0, 0]), 4), c.k.clone(), c.v.clone()]
        runs.append(got)
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    k0 = runs[0][1]
    assert k0[0, table[0, 0], :, 0].any() and runs[0][4].tolist() == [3, 23, 3, 67]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("groups, beams, vocab, picks", [(1, 3, 30001, 16), (2, 12, 5001, 64), (1, 1, 1025, 7), (30, 8, 20003, 9)])
def test_thousands_of_equal_logits_in_rows_that_start_anywhere(dev, dtype, groups, beams, vocab, picks):
    from ironmill_b200 import ops
    rng = H.rng_for("few", vocab)
    few = rng.integers(0, 4, (groups, vocab))
    x = torch.from_numpy(np.repeat(few[:, None], beams, 1)).to(device="cuda", dtype=TYPES[dtype])
    x[:, :, 2::5] = -np.inf
    few[:, 2::5] = -1
    _, parent, token = ops.beam_select(dev, x, torch.zeros((groups, beams), device="cuda"), picks)
    for g in range(groups):
        assert parent[g].tolist() == [0] * picks and token[g].tolist() == np.flatnonzero(few[g] == 3)[:picks].tolist()


# ------------------------------------------------------------------------------------------------ ragged batches in wide tiles
def _no_wait_ran_out(dev):
    from ironmill_b200._lib import check, lib
    check(lib().im_cuda_device_check_error(dev.handle))


@pytest.mark.parametrize("dtype, dim, heads, kv_heads, new, most, max_new", [
    ("bf16", 128, 32, 4, [200] + [1] * 31, 900, 200), ("f16", 128, 12, 3, [1] * 40 + [90], 700, 90), ("f16", 64, 20, 1, [1] * 60, 900, 21), ("bf16", 64, 16, 4, [0, 40, 3, 0, 17, 1, 1, 2, 33] * 4, 800, 60),
    ("bf16", 128, 16, 4, [33, 1, 33, 1, 1, 33, 1, 1, 1, 33, 1], 3000, 33), ("f16", 128, 24, 3, [20, 5, 17, 16, 2], 5000, 40), ("bf16", 128, 32, 4, [80], 589, 130)])
def test_wide_tiles_that_few_rows_of_a_sequence_fill(dev, dtype, dim, heads, kv_heads, new, most, max_new):
    """Portions of prompts beside single tokens: a CTA has items one after the other whose rows leave half of its warps without any."""
    rng = H.rng_for("ragged", most + heads)
    lengths = [most, *rng.integers(0, most, len(new) - 1).tolist()]
    c = Cache(dev, rng, [a + b for a, b in zip(lengths, new)], lengths, kv_heads=kv_heads, dim=dim, page=48, dtype=dtype)
    first = _check_attention(dev, c, H.rng_for("ragged-q"), new, heads, dtype, max_new=max_new)[0]
    _no_wait_ran_out(dev)
    masks = np.concatenate([_tree(rng, n, -(-max_new // 64)) for n in new if n])
    _check_attention(dev, c, H.rng_for("ragged-q"), new, heads, dtype, max_new=max_new, mask=masks, max_len=0)
    _no_wait_ran_out(dev)
    assert (_check_attention(dev, c, H.rng_for("ragged-q"), new, heads, dtype, max_new=max_new)[0] == first).all()
