"""Appending to a paged cache with norms per head and positions of several axes, against the plain restatement in 64 bits (tests/oracle_paged_more.py)."""
import numpy as np
import pytest

from tests import helpers as H
from tests import oracle_paged_more as om

torch = pytest.importorskip("torch")
from tests.test_gpu_paged import TYPES, Cache, _ints, _np, _randn, _starts  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from ironmill_b200 import ops
    return ops.Device(0)


def _check(dev, c, rng, new, heads, dtype, rotary, neighbours=False, table="f16", axes=1, axis=None, positions=None, norms="qk", norm_type=None, eps=1e-6, lead=0, trail=0, layer=0,
           in_place=False, max_pos=None, scale=1.0):
    from ironmill_b200 import ops
    nkv, dim = c.k.shape[2], c.k.shape[4]
    starts = _starts(new, lead)
    n = starts[-1] + trail
    qkv = _randn(rng, (n, heads + 2 * nkv, dim), dtype, scale)
    q, k, v = qkv.split([heads, nkv, nkv], 1)
    most = max_pos or max(a + b for a, b in zip(c.lengths, new)) + 1
    angle = np.arange(most)[:, None] * 1e4 ** (-2.0 * np.arange(dim // 2) / max(rotary, 2))
    cos, sin = (torch.from_numpy(f(angle)).to(device="cuda", dtype=TYPES[table]) for f in (np.cos, np.sin))
    weights = {x: _randn(rng, (dim,), norm_type or dtype, 0.3) + 1 if x in norms else None for x in "qk"}
    if positions is None and axes > 1:
        positions = rng.integers(0, most, (axes, n))
    ko, vo, qn, kn, vn = _np(c.k), _np(c.v), _np(q), _np(k), _np(v)
    kwargs = dict(cos=cos, sin=sin, rotary_dim=rotary, neighbours=neighbours) if rotary else {}
    if heads:
        out = q if in_place else torch.full((n, heads, dim), 7.0, dtype=TYPES[dtype], device="cuda")
        kwargs.update(q=q, q_out=out, q_norm=weights["q"])
    if axis is not None:
        kwargs.update(pair_axis=bytes(axis), positions=_ints(positions))
    elif positions is not None:
        kwargs.update(positions=_ints(positions[0]))
    ops.paged_append(c.kv, layer, k, v, _ints(starts), k_norm=weights["k"], eps=eps, **kwargs)
    f = lambda x: None if x is None else _np(x)  # noqa: E731
    with np.errstate(invalid="ignore", divide="ignore"):
        want, mass_k, mass_q = om.append(ko[layer], vo[layer], c.table, c.lengths, starts, kn, vn, qn if heads else None, _np(cos), _np(sin), rotary, neighbours, positions, f(weights["q"]),
                                         f(weights["k"]), eps, axis)
    # A norm: a sum of dim squares and its factors, half of that behind the square root, the library's root, two products: (dim / 2 + 8) 2^-24 relative; two
    # products and a sum of a rotation 3 2^-24 of their magnitudes; one rounding.
    step, f32 = torch.finfo(TYPES[dtype]).eps / 2, (dim / 2 + 12) * 2.0 ** -24

    def near(got, exact, mass):
        same = np.isnan(got) & np.isnan(exact)
        return (same | (np.abs(got - exact) <= step * np.abs(exact) * (1 + 1e-3) + f32 * mass + 2.0 ** -25)).all()

    full = np.zeros(ko.shape)
    full[layer] = mass_k
    assert near(_np(c.k), ko, full)
    assert (_np(c.v) == vo).all()
    if heads:
        got, before = _np(out), qn if in_place else np.full(qn.shape, 7.0)
        touched = mass_q.any((1, 2))
        assert near(got[touched], want[touched], mass_q[touched]) and (got[~touched] == before[~touched]).all()
        return got, touched


def _sections(half, parts):
    return [min(len(parts) - 1, next(a for a in range(len(parts)) if i < sum(parts[:a + 1]) or a == len(parts) - 1)) for i in range(half)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("norms", ["qk", "q", "k", ""])
@pytest.mark.parametrize("dim, rotary, neighbours", [(128, 128, False), (128, 64, False), (128, 64, True), (64, 64, True), (64, 24, False), (256, 256, False), (80, 80, False),
                                                     (80, 36, False), (80, 38, True), (8, 8, False), (8, 2, True), (128, 0, False), (200, 90, False)])
def test_norms_and_two_axes_match_the_formula(dev, dtype, norms, dim, rotary, neighbours):
    rng = H.rng_for("append-normed", dim * 1000 + rotary + len(norms))
    c = Cache(dev, rng, [40, 9, 70, 1], [30, 0, 33, 0], kv_heads=3, dim=dim, page=7, dtype=dtype)
    axis = [int(x) for x in rng.integers(0, 2, rotary // 2)] if rotary else None
    _check(dev, c, rng, [10, 5, 0, 1], 5, dtype, rotary, neighbours, "f32" if dim % 16 else "f16", axes=2 if rotary else 1, axis=axis, norms=norms,
           norm_type="f32" if dim == 64 else None)


@pytest.mark.parametrize("axes", [1, 2, 3, 4])
@pytest.mark.parametrize("mixed", [False, True])
@pytest.mark.parametrize("dim, rotary, neighbours", [(128, 128, False), (256, 256, True), (64, 44, False)])
def test_axes_in_runs_and_in_turns(dev, axes, mixed, dim, rotary, neighbours):
    rng = H.rng_for("append-axes", axes * 10 + mixed + dim)
    c = Cache(dev, rng, [200, 90], [100, 3], dim=dim, page=16)
    half = rotary // 2
    axis = [i % axes for i in range(half)] if mixed else _sections(half, [half // (axes + 1)] * axes)
    _check(dev, c, rng, [60, 77], 4, "f16", rotary, neighbours, axes=axes, axis=axis, table="f32", positions=rng.integers(0, 200, (axes, 137)))


def test_a_section_may_be_empty(dev):
    rng = H.rng_for("append-same")
    c = Cache(dev, rng, [50], [20])
    _check(dev, c, rng, [10], 4, "f16", 128, axes=3, axis=_sections(64, [16, 0, 48]), positions=rng.integers(0, 31, (3, 10)), norms="")


def test_a_position_outside_the_table_on_any_axis_leaves_the_token_alone(dev):
    rng = H.rng_for("append-outside")
    c = Cache(dev, rng, [60], [20])
    positions = np.array([[1, 2, 3, 4, 43, -1], [1, 43, 3, 4, 5, 6], [1, 2, -5, 42, 5, 6]])
    _, touched = _check(dev, c, rng, [6], 4, "f16", 128, axes=3, axis=[i % 3 for i in range(64)], positions=positions, max_pos=43)
    assert touched.tolist() == [True, False, False, True, False, False]


def test_in_place_other_tokens_and_a_layer_that_lies_apart(dev):
    for rotary, neighbours in ((128, False), (40, True), (44, False)):
        rng = H.rng_for("append-place", rotary)
        c = Cache(dev, rng, [30, 30, 30], [0, 7, 29], dtype="bf16", layers=2, apart=True)
        _check(dev, c, rng, [3, 4, 1], 9, "bf16", rotary, neighbours, lead=2, trail=3, in_place=True, layer=1)


def test_keys_alone_and_values_that_stay_as_they_are(dev):
    rng = H.rng_for("append-keys")
    c = Cache(dev, rng, [100, 100], [64, 13])
    _check(dev, c, rng, [1, 1], 0, "f16", 128)


def test_small_and_large_heads_and_heads_of_zeros(dev):
    """The mean lies far below eps, and far above it; a head of zeros stays one."""
    for dtype, scale, eps in (("f16", 2.0 ** -12, 1e-5), ("bf16", 1e4, 1e-6), ("f16", 0.0, 1e-6), ("bf16", 2.0 ** -30, 0.0)):
        rng = H.rng_for("append-scale", int(eps * 1e7))
        c = Cache(dev, rng, [20], [3], dtype=dtype)
        if scale == 0.0:
            from ironmill_b200 import ops
            z = torch.zeros((4, 6, 128), dtype=TYPES[dtype], device="cuda")
            got = ops.paged_append(c.kv, 0, z[:, 4:], z[:, 4:], _ints([0, 4]), q=z[:, :4], q_norm=torch.ones(128, dtype=TYPES[dtype], device="cuda"), eps=eps)
            assert (got == 0).all()
        else:
            _check(dev, c, rng, [4], 4, dtype, 128, eps=eps, scale=scale)


def test_many_tokens_go_by_small_blocks(dev):
    rng = H.rng_for("append-many")
    new = [300, 0, 400, 5]
    c = Cache(dev, rng, [a + 3 for a in new], [3] * 4, kv_heads=1, page=32, dtype="bf16")
    _check(dev, c, rng, new, 5, "bf16", 128, axes=3, axis=_sections(64, [16, 24, 24]), table="f32")


def test_without_norms_and_axes_the_plain_append_runs(dev):
    """One axis named for every pair is the same as none."""
    from ironmill_b200 import ops
    rng = H.rng_for("append-plain")
    x = _randn(rng, (6, 8, 128), "f16")
    angle = np.arange(40)[:, None] * 1e4 ** (-np.arange(64) / 64)
    cos, sin = (torch.from_numpy(f(angle)).half().cuda() for f in (np.cos, np.sin))
    at = _ints([9, 1, 2, 30, 4, 5])
    got = []
    for more in (dict(positions=at), dict(positions=at[None], pair_axis=bytes(64))):
        c = Cache(dev, H.rng_for("append-plain-cache"), [30], [20])
        q = ops.paged_append(c.kv, 0, x[:, 4:6], x[:, 6:], _ints([0, 6]), q=x[:, :4], cos=cos, sin=sin, **more)
        got.append((q, c.k, c.v))
    # the same formula, contracted differently: a step of the type at most
    for a, b in zip(*got):
        assert ((a.float() - b.float()).abs() <= 2.0 ** -10 * b.float().abs() + 2.0 ** -21).all()


def test_no_tokens(dev):
    from ironmill_b200 import ops
    c = Cache(dev, H.rng_for("append-none"), [30], [20])
    x, cos = torch.zeros((0, 8, 128), dtype=torch.float16, device="cuda"), torch.ones((9, 64), dtype=torch.float16, device="cuda")
    w = torch.ones(128, dtype=torch.float16, device="cuda")
    before = c.k.clone()
    q = ops.paged_append(c.kv, 0, x[:, :2], x[:, 2:4], _ints([0, 0]), q=x[:, 4:], cos=cos, sin=cos, positions=torch.zeros((3, 0), dtype=torch.int32, device="cuda"), q_norm=w, k_norm=w,
                         pair_axis=bytes([i % 3 for i in range(64)]))
    assert q.shape == (0, 4, 128) and (c.k == before).all()


def test_heads_of_which_some_lie_in_other_rows_of_a_wider_tensor(dev):
    """Parts of one row per token, as a projection leaves them, tokens far apart; norm weights of another type than the cache's are f32."""
    rng = H.rng_for("append-wide")
    for dim, norm_type in ((128, "f32"), (64, None), (96, "f32")):
        c = Cache(dev, rng, [50, 20], [40, 0], dim=dim, kv_heads=2, dtype="bf16")
        _check(dev, c, rng, [9, 20], 6, "bf16", dim, axes=3, axis=[i * 3 // (dim // 2) for i in range(dim // 2)], norm_type=norm_type, table="f32")
