"""How exact single tokens behind a shared prefix are: as exact as the same tokens through paged_attention, however many sequences share it."""
import numpy as np
import pytest

from tests import helpers as H
from tests import oracle_paged as op

torch = pytest.importorskip("torch")
from tests.test_gpu_paged import _ints, _np, _randn  # noqa: E402
from tests.test_gpu_paged_prefix import _cache  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    from ironmill_b200 import ops
    return ops.Device(0)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim, seqs", [(128, 20), (128, 40), (128, 70), (64, 40), (256, 40)])
def test_single_tokens_lose_nothing_by_sharing(dev, dtype, dim, seqs):
    from ironmill_b200 import ops
    rng = H.rng_for("prefix-exact", dim + seqs)
    c = _cache(dev, rng, [seqs], [40], [int(x) for x in rng.integers(0, 40, seqs)], [1] * seqs, page=32, dim=dim, dtype=dtype)
    q, starts, scale = _randn(rng, (seqs, 8, dim), dtype), _ints(range(seqs + 1)), dim ** -0.5
    shared = ops.paged_prefix_attention(c.kv, 0, q, starts, 1, scale, _ints([0, seqs]), seqs, _ints([40]), max_len=1400)      # (the whole table: what is shared goes by tiles)
    alone = ops.paged_attention(c.kv, 0, q, starts, 1, scale)
    want, _, _ = op.attention(_np(c.k[0]), _np(c.v[0]), c.table, c.lengths, list(range(seqs + 1)), _np(q), scale)
    off = [np.linalg.norm(_np(x) - want) / np.linalg.norm(want) for x in (shared, alone)]
    # both round an output once: the root of a mean square of at most half a step, 2^-8 or 2^-11; a weight of one 16-bit term would make that 1.4 times as much
    assert off[1] < torch.finfo(c.k.dtype).eps / 2 and off[0] < 1.1 * off[1], off
