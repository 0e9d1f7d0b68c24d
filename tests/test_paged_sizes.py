"""Sizes whose products pass 64 bits are refused, not taken for small ones (arguments are checked before the device)."""
import pytest

from tests.test_paged import GOOD, PTR, _attend, _kv, _message, lib  # noqa: F401
from tests.test_paged_more import _prefix, _weights

WIDE = dict(heads=1 << 30, qs=1 << 37, os=1 << 37, out=1 << 60, n=3)


@pytest.mark.parametrize("call", [_attend, _prefix, _weights])
@pytest.mark.parametrize("max_new, seqs", [(1 << 30, 512), (1 << 30, 1 << 10), (1 << 29, 1 << 20), ((1 << 31) - 1, 3)])
def test_new_tokens_of_all_sequences(lib, call, max_new, seqs):  # noqa: F811
    more = dict(ss=1 << 8, w=1 << 59) if call is _weights else {}
    assert "too many" in _message(lib, call(lib, _kv(num_seqs=seqs), **WIDE, max_new=max_new, **more))


@pytest.mark.parametrize("group_new, groups", [(1 << 30, 512), (1 << 29, 1 << 20), ((1 << 31) - 1, 3)])
def test_new_tokens_of_all_groups(lib, group_new, groups):  # noqa: F811
    assert "too many" in _message(lib, _prefix(lib, _kv(), **WIDE, group_new=group_new, groups=groups))


def test_as_many_as_there_may_be(lib):  # noqa: F811
    """2^24 tiles of 16 rows: two KV heads of two query heads, 2^13 sequences of 2^13 new tokens."""
    more = dict(n=3, max_new=1 << 13)
    assert _message(lib, _attend(lib, _kv(num_seqs=1 << 13), **more)) == GOOD
    assert "too many" in _message(lib, _attend(lib, _kv(num_seqs=(1 << 13) + 1), **more))
    assert "too many" in _message(lib, _attend(lib, _kv(num_seqs=1 << 13), **dict(more, max_new=(1 << 13) + 1)))


def test_sums_of_sequences_too_far_apart(lib):  # noqa: F811
    assert "overlap" in _message(lib, _weights(lib, _kv(num_seqs=1 << 22), ss=1 << 40, w=1 << 59, max_new=1))
    assert _message(lib, _weights(lib, _kv(num_seqs=1 << 10), ss=1 << 30, w=1 << 59, max_new=1, out=1 << 60, q=PTR)) == GOOD
