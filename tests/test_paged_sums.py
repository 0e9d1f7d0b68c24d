"""Where the sums of attention weights may lie, seen without a GPU (arguments are checked before the device)."""
import pytest

from tests.test_paged import GOOD, PTR, _kv, _message, lib  # noqa: F401
from tests.test_paged_more import _weights

SPAN = 4 * (2 * 128 + 64 + 64)      # bytes of the sums: three sequences of two heads of 64 rows


@pytest.mark.parametrize("change", [
    dict(w=3 * PTR), dict(w=3 * PTR + 44), dict(w=3 * PTR - SPAN + 4),                  # the page table: three rows of four
    dict(w=4 * PTR), dict(w=4 * PTR + 8), dict(w=4 * PTR - SPAN + 4),                   # lengths
    dict(start=17 * PTR), dict(start=17 * PTR - 12), dict(start=17 * PTR + SPAN - 4),   # four starts
    dict(mask=17 * PTR, words=2), dict(mask=17 * PTR - 40, words=2), dict(mask=17 * PTR + SPAN - 8, words=2)])
def test_sums_over_what_says_where_rows_lie_are_refused(lib, change):  # noqa: F811
    assert "table" in _message(lib, _weights(lib, _kv(), **change))


@pytest.mark.parametrize("change", [
    dict(w=3 * PTR + 48), dict(w=3 * PTR - SPAN), dict(w=4 * PTR + 12), dict(w=4 * PTR - SPAN), dict(start=17 * PTR - 16), dict(start=17 * PTR + SPAN),
    dict(mask=17 * PTR - 48, words=2), dict(mask=17 * PTR + SPAN, words=2)])
def test_sums_may_lie_right_beside_it(lib, change):  # noqa: F811
    assert _message(lib, _weights(lib, _kv(), **change)) == GOOD


def test_rows_of_a_page_table_that_lie_apart_count_as_a_whole(lib):  # noqa: F811
    assert "table" in _message(lib, _weights(lib, _kv(table_stride=100), w=3 * PTR + 800))
    assert _message(lib, _weights(lib, _kv(table_stride=100), w=3 * PTR + 816)) == GOOD


@pytest.mark.parametrize("tokens, row", [(1, 512), (2, 512), (5, 512), (5, 640)])
def test_sums_may_lie_right_behind_and_right_before_queries_and_outputs(lib, tokens, row):  # noqa: F811
    """Four heads of 128 columns of two bytes a token, rows apart by `row` elements: the last one ends with its heads."""
    end = 2 * row * (tokens - 1) + 1024
    shape = dict(n=tokens, qs=row, os=row, q=6 * PTR)
    for at in (6 * PTR, 9 * PTR):
        for w, word in ((at + end, GOOD), (at + end - 4, "queries or the outputs"), (at - SPAN, GOOD), (at - SPAN + 4, "queries or the outputs")):
            assert word in _message(lib, _weights(lib, _kv(), **dict(shape, w=w))), (at, w)
