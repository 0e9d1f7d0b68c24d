"""What appending with positions of several axes refuses in Python: axes that no positions are given for."""
import numpy as np
import pytest

from tests import helpers as H

torch = pytest.importorskip("torch")
from tests.test_gpu_paged import Cache, _ints, _randn  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pair_axis, positions", [([0, 1] * 32, [[1, 2, 3]]), ([0] * 63 + [1], [[1, 2, 3]]), ([0, 1] * 32, None), ([0] * 64, [1, 2, 3]), ([0] * 63, [[1, 2, 3]])])
def test_axes_without_positions_are_refused(pair_axis, positions):
    from ironmill_b200 import ops
    rng = H.rng_for("append-axes-refused")
    c = Cache(ops.Device(0), rng, [20], [4])
    x = _randn(rng, (3, 4, 128), "f16")
    cos = torch.ones((9, 64), dtype=torch.float16, device="cuda")
    before = c.k.clone()
    with pytest.raises(AssertionError):
        ops.paged_append(c.kv, 0, x[:, :2], x[:, 2:], _ints([0, 3]), cos=cos, sin=cos, positions=None if positions is None else _ints(np.array(positions)), pair_axis=pair_axis)
    assert (c.k == before).all()
    ops.paged_append(c.kv, 0, x[:, :2], x[:, 2:], _ints([0, 3]), cos=cos, sin=cos, positions=_ints([[1, 2, 3]]), pair_axis=[0] * 64)    # one axis, named
    assert not (c.k == before).all()
