"""What the paged cache's operators and beam selection refuse, seen without a GPU (arguments are checked before the device), and their plain
restatement on cases small enough to check by hand."""
import ctypes as C

import numpy as np
import pytest

from tests import oracle_paged as op

PTR = 1 << 20  # stands for device memory: nothing is launched


@pytest.fixture(scope="module")
def lib():
    from ironmill_b200 import _lib, build
    build.build()
    return _lib.lib()


def _kv(**more):
    from ironmill_b200._lib import PagedKvStruct
    kv = PagedKvStruct()
    for k, v in dict(dict(k_dev=PTR, v_dev=2 * PTR, num_layers=2, num_pages=10, num_kv_heads=2, page_size=16, head_dim=128, dtype=0, num_seqs=3,
                          page_table_dev=3 * PTR, table_width=4, seq_len_dev=4 * PTR), **more).items():
        setattr(kv, k, v)
    return kv


def _message(lib, rc):
    assert rc == -1, rc
    return lib.im_cuda_last_error().decode()


def _append(lib, kv, **more):
    a = dict(dict(layer=0, k=PTR, ks=256, v=PTR, vs=256, start=PTR, n=3, q=PTR, qs=512, qo=PTR, qos=512, heads=4, cos=PTR, sin=PTR, table=0, max_pos=9, rot=128, nb=0,
                  pos=None), **more)
    return lib.im_cuda_paged_append(None, C.addressof(kv) if kv is not None else None, *a.values(), None)


def _attend(lib, kv, **more):
    a = dict(dict(layer=0, q=PTR, qs=512, out=5 * PTR, os=512, heads=4, start=PTR, n=3, max_new=1, mask=None, words=0, scale=0.1, max_len=0, scratch=PTR, size=1 << 30), **more)
    return lib.im_cuda_paged_attention(None, C.addressof(kv) if kv is not None else None, *a.values(), None)


def _select(lib, **more):
    a = dict(dict(x=PTR, dtype=1, stride=0, groups=2, beams=4, vocab=100, score=PTR, done=None, end=-1, picks=4, so=5 * PTR, po=PTR, to=PTR, scratch=PTR, size=1 << 30), **more)
    return lib.im_cuda_beam_select(None, *a.values(), None)


GOOD = "dev is NULL"  # what a call says whose arguments are right, where there is no device


def test_right_arguments_are_only_short_of_a_device(lib):
    assert _message(lib, _append(lib, _kv())) == GOOD
    assert _message(lib, _append(lib, _kv(), q=None, qo=None, heads=0, rot=0, cos=None, sin=None)) == GOOD
    assert _message(lib, _attend(lib, _kv())) == GOOD
    assert _message(lib, _select(lib)) == GOOD
    kv = _kv()
    assert _message(lib, lib.im_cuda_paged_keep(None, C.addressof(kv), PTR, 4, PTR, 5 * PTR, None)) == GOOD
    assert _message(lib, lib.im_cuda_paged_reorder(None, C.addressof(kv), PTR, 3, 5 * PTR, 0, 6 * PTR, None)) == GOOD


@pytest.mark.parametrize("change, word", [
    (dict(dtype=1), "dtype 1"), (dict(num_layers=0), "shape"), (dict(num_pages=0), "shape"), (dict(page_size=0), "shape"), (dict(table_width=0), "shape"), (dict(num_seqs=-1), "shape"),
    (dict(head_dim=100), "head_dim"), (dict(head_dim=264), "head_dim"), (dict(k_dev=None), "NULL"), (dict(seq_len_dev=None), "NULL"), (dict(page_table_dev=None), "NULL"),
    (dict(v_dev=PTR), "same place"), (dict(k_dev=PTR + 8), "16-byte"), (dict(table_width=1 << 30), "too long"), (dict(page_stride=4096 - 8), "strides"),
    (dict(page_stride=4097), "strides"), (dict(layer_stride=4096), "overlap"), (dict(table_stride=3), "overlap"), (dict(num_pages=1 << 30, page_size=1 << 20, table_width=1), "shape")])
def test_caches_that_are_refused(lib, change, word):
    kv = _kv(**change)
    for call in (lambda: _append(lib, kv), lambda: _attend(lib, kv), lambda: lib.im_cuda_paged_keep(None, C.addressof(kv), PTR, 4, PTR, 5 * PTR, None),
                 lambda: lib.im_cuda_paged_reorder(None, C.addressof(kv), PTR, 3, 5 * PTR, 0, 6 * PTR, None)):
        assert word in _message(lib, call())


def test_layers_inside_pages_are_taken(lib):
    assert _message(lib, _attend(lib, _kv(layer_stride=4096, page_stride=8192))) == GOOD


@pytest.mark.parametrize("change, word", [
    (dict(layer=2), "layer"), (dict(layer=-1), "layer"), (dict(k=None), "bad argument"), (dict(n=-1), "bad argument"), (dict(qo=None), "queries"), (dict(heads=0), "queries"),
    (dict(ks=248), "keys"), (dict(vs=260), "keys"), (dict(k=PTR + 2), "keys"), (dict(qs=8), "queries"), (dict(q=PTR + 4), "queries"), (dict(rot=130), "rotary"), (dict(rot=3), "rotary"),
    (dict(cos=None), "tables"), (dict(table=2), "tables"), (dict(max_pos=0), "tables"), (dict(cos=PTR + 8), "aligned"), (dict(nb=2), "neighbours")])
def test_appends_that_are_refused(lib, change, word):
    assert word in _message(lib, _append(lib, _kv(), **change))


@pytest.mark.parametrize("change, word", [
    (dict(layer=2), "layer"), (dict(q=None), "bad argument"), (dict(max_len=-1), "bad argument"), (dict(heads=3), "multiple"), (dict(heads=0), "multiple"), (dict(max_new=0), "max_new"),
    (dict(qs=500), "queries"), (dict(os=8), "queries"), (dict(out=PTR + 8), "queries"), (dict(mask=PTR, words=0), "mask"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(out=PTR), "over the queries"), (dict(max_new=1 << 30), "too many")])
def test_attention_that_is_refused(lib, change, word):
    assert word in _message(lib, _attend(lib, _kv(), **change))


def test_heads_that_attention_is_not_built_for(lib):
    assert "64, 128 and 256" in _message(lib, _attend(lib, _kv(head_dim=96)))
    assert lib.im_cuda_paged_attention_scratch_bytes(None, C.addressof(_kv()), 4, 1, 0) == 0


@pytest.mark.parametrize("change, word", [
    (dict(dtype=3), "dtype"), (dict(beams=0), "beams"), (dict(beams=65), "beams"), (dict(vocab=0), "tokens"), (dict(groups=-1), "groups"), (dict(picks=0), "picks"), (dict(picks=65), "picks"),
    (dict(groups=40000), "65535"), (dict(stride=99), "overlap"), (dict(x=None), "NULL"), (dict(x=PTR + 2), "aligned"), (dict(done=PTR, end=100), "end_token"),
    (dict(done=PTR, end=-1), "end_token"), (dict(so=None), "NULL"), (dict(so=PTR + 28), "old ones")])
def test_selections_that_are_refused(lib, change, word):
    assert word in _message(lib, _select(lib, **change))


def test_results_may_not_lie_over_what_is_read(lib):
    kv = _kv()
    at = C.addressof(kv)
    assert "old ones" in _message(lib, lib.im_cuda_paged_keep(None, at, PTR, 4, PTR, 4 * PTR + 8, None))
    assert "accepted" in _message(lib, lib.im_cuda_paged_keep(None, at, PTR, 4, 5 * PTR, PTR + 47, None))
    assert "accepted" in _message(lib, lib.im_cuda_paged_keep(None, at, PTR, 4, 5 * PTR, 5 * PTR - 11, None))
    assert "parents" in _message(lib, lib.im_cuda_paged_reorder(None, at, PTR, 3, 5 * PTR, 0, PTR + 8, None))
    assert "each other" in _message(lib, lib.im_cuda_paged_reorder(None, at, PTR, 3, 5 * PTR, 0, 5 * PTR + 44, None))
    assert "old one" in _message(lib, lib.im_cuda_paged_reorder(None, at, PTR, 3, 3 * PTR + 16, 0, PTR, None))
    assert "old ones" in _message(lib, lib.im_cuda_paged_reorder(None, at, PTR, 3, PTR, 0, 4 * PTR, None))
    assert "groups of 2" in _message(lib, lib.im_cuda_paged_reorder(None, at, PTR, 2, PTR, 0, PTR, None))
    assert "overlap" in _message(lib, lib.im_cuda_paged_reorder(None, at, PTR, 3, PTR, 3, PTR, None))
    assert "bad argument" in _message(lib, lib.im_cuda_paged_keep(None, at, PTR, 0, PTR, PTR, None))


@pytest.mark.parametrize("change, word", [
    (dict(qos=520), "other tokens"), (dict(qo=PTR + 1024), "other tokens"), (dict(q=PTR + 1024), "other tokens"), (dict(qs=1024, qos=1024, qo=PTR + 1008), "other tokens"),
    (dict(qs=1024, qos=1024, qo=PTR + 2048 - 16), "other tokens"), (dict(qs=1024, qos=1024, qo=PTR + 1024), GOOD), (dict(qos=520, n=1), GOOD), (dict(qo=PTR + 3 * 1024 - 16), "other tokens"),
    (dict(qo=PTR + 3 * 1024), GOOD), (dict(n=(1 << 31) - 1, qs=1 << 40, qos=1 << 40), GOOD), (dict(n=(1 << 31) - 1, qs=1 << 40, qos=(1 << 40) - 8), "other tokens"),
    (dict(heads=1 << 21, qs=1 << 40, qos=1 << 40), "heads")])
def test_rotated_queries_over_other_tokens_queries(lib, change, word):
    assert word in _message(lib, _append(lib, _kv(), **change))


@pytest.mark.parametrize("change, word", [
    (dict(out=PTR + 1024), "over the queries"), (dict(q=PTR + 1024, out=PTR), "over the queries"), (dict(os=520, out=PTR + 16), "over the queries"),
    (dict(qs=1024, os=1024, out=PTR + 1024), GOOD), (dict(qs=1024, os=1024, out=PTR + 1040), "over the queries"), (dict(qs=1024, os=1024, out=PTR + 1008), "over the queries")])
def test_outputs_over_the_queries(lib, change, word):
    assert word in _message(lib, _attend(lib, _kv(), **change))


# ------------------------------------------------------------------------------------------------ the restatement itself
def test_plain_reorder_by_hand():
    # beams with rows [0 0 | 0 .], pages of two: page 9 shared, last pages 0..2; children of beams 1, 1, 2: beam 0 is childless
    keys = np.zeros((1, 10, 1, 2, 1))
    keys[0, :3, 0, 0, 0] = [10, 11, 12]
    values = -keys
    table = np.array([[9, 0], [9, 1], [9, 2]])
    new, lens = op.reorder(keys, values, table, np.array([3, 3, 3]), [1, 1, 2], 3)
    assert new.tolist() == [[9, 1], [9, 0], [9, 2]] and lens.tolist() == [3, 3, 3]
    assert keys[0, :3, 0, 0, 0].tolist() == [11, 11, 12] and values[0, 0, 0, 0, 0] == -11


def test_plain_keep_by_hand():
    keys = np.arange(8.0).reshape(1, 2, 1, 4, 1)
    values = keys.copy()
    lens = op.keep(keys, values, np.array([[1, 0]]), [2], np.array([[0, 2, 5]]), [3])
    # rows 2.. are 6 7 | 0 1 2 3: places 0, 2 stay or move to 1; place 5 is row 7
    assert lens.tolist() == [5] and keys.reshape(-1).tolist() == [3, 1, 2, 3, 4, 5, 6, 0]


def test_plain_selection_by_hand():
    x = np.log(np.array([[[0.5, 0.25, 0.25], [0.2, 0.2, 0.6]]]))
    best = op.select(x, np.array([[0.0, -1.0]]), 3)[0]
    assert [(b, t) for _, b, t in best[:3]] == [(0, 0), (0, 1), (0, 2)]
    best = op.select(x, np.array([[0.0, -0.1]]), 3, done=np.array([[False, True]]), end_token=1)[0]
    assert [(b, t) for _, b, t in best[:3]] == [(1, 1), (0, 0), (0, 1)]


def test_plain_attention_by_hand():
    keys = np.zeros((2, 1, 2, 1))
    values = np.array([[[[1.0], [2.0]]], [[[4.0], [8.0]]]])
    table, q = np.array([[1, 0]]), np.ones((2, 1, 1))
    out, _, _ = op.attention(keys, values, table, [2], [0, 2], q, 1.0)
    assert np.allclose(out.ravel(), [13 / 3, 15 / 4])
    out, _, _ = op.attention(keys, values, table, [0], [0, 2], q, 1.0, mask=np.array([[2], [0]]))
    assert out.ravel().tolist() == [8.0, 0.0]


# ------------------------------------------------------------------------------------------------ keeping over the page table
@pytest.mark.parametrize("out, table, word", [
    (3 * PTR, {}, "page table"), (3 * PTR - 8, {}, "page table"), (3 * PTR + 47, {}, "page table"), (3 * PTR + 48, {}, GOOD), (3 * PTR - 12, {}, GOOD),
    (3 * PTR + 76, dict(table_stride=8), "page table"), (3 * PTR + 80, dict(table_stride=8), GOOD), (3 * PTR, dict(num_seqs=0), GOOD)])
def test_new_lengths_over_the_page_table_are_refused(lib, out, table, word):
    kv = _kv(**table)
    assert word in _message(lib, lib.im_cuda_paged_keep(None, C.addressof(kv), PTR, 4, PTR, out, None))
