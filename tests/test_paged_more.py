"""What the paged cache's further operators refuse, seen without a GPU (arguments are checked before the device), and their plain restatement on cases small
enough to check by hand."""
import ctypes as C

import numpy as np
import pytest

from tests import oracle_paged_more as om
from tests.test_paged import GOOD, PTR, _kv, _message

F32, F16, BF16 = 1, 0, 2


@pytest.fixture(scope="module")
def lib():
    from ironmill_b200 import _lib, build
    build.build()
    return _lib.lib()


def _call(lib, fn, kv, packed):
    return getattr(lib, fn)(None, C.addressof(kv) if kv is not None else None, packed, None)


def _append(lib, kv, **more):
    from ironmill_b200._lib import APPEND_ARGS
    a = dict(dict(k=PTR, v=PTR, q=PTR, qo=PTR, start=PTR, pos=PTR, cos=PTR, sin=PTR, qn=PTR, kn=PTR, axis=0, ks=256, vs=256, qs=512, qos=512, layer=0, n=3, heads=4, table=0, max_pos=9, rot=128, nb=0,
                  norm=0, axes=1, eps=1e-6), **more)
    return _call(lib, "im_cuda_paged_append_normed", kv, APPEND_ARGS.pack(*a.values()))


ATTN = dict(q=PTR, out=9 * PTR, start=PTR, mask=0, scratch=PTR, size=1 << 40, qs=512, os=512, layer=0, heads=4, n=3, max_new=1, words=0, max_len=0, scale=0.1)


def _prefix(lib, kv, **more):
    from ironmill_b200._lib import PREFIX_ARGS
    a = dict(dict(ATTN, bounds=PTR, pages=PTR, groups=2, group_new=3, prefix=0), **more)
    return _call(lib, "im_cuda_paged_prefix_attention", kv, PREFIX_ARGS.pack(*a.values()))


def _weights(lib, kv, **more):
    from ironmill_b200._lib import WEIGHTS_ARGS
    a = dict(dict(ATTN, w=17 * PTR, ss=128, sh=64, rows=64), **more)
    return _call(lib, "im_cuda_paged_attention_weights", kv, WEIGHTS_ARGS.pack(*a.values()))


def _evict(lib, kv, **more):
    from ironmill_b200._lib import EVICT_ARGS
    a = dict(dict(w=17 * PTR, wo=33 * PTR, lens=5 * PTR, wl=384, ws=128, wh=64, ol=384, os=128, oh=64, budget=10, recent=3), **more)
    return _call(lib, "im_cuda_paged_evict", kv, EVICT_ARGS.pack(*a.values()))


def test_right_arguments_are_only_short_of_a_device(lib):
    for f in (_append, _prefix, _weights, _evict):
        assert _message(lib, f(lib, _kv())) == GOOD
        assert _message(lib, f(lib, _kv(num_seqs=0))) == GOOD
    assert _message(lib, _append(lib, _kv(), q=0, qo=0, heads=0, qn=0, rot=0, cos=0, sin=0, pos=0)) == GOOD
    assert _message(lib, _append(lib, _kv(), n=0)) == GOOD
    assert _message(lib, _prefix(lib, _kv(), groups=0, bounds=0, pages=0)) == GOOD
    assert _message(lib, _prefix(lib, _kv(), n=0)) == GOOD and _message(lib, _weights(lib, _kv(), n=0)) == GOOD


def test_the_packed_structs_are_those_of_the_header(tmp_path):
    """Sizes and offsets as a C compiler sees them."""
    import os
    import subprocess
    from ironmill_b200 import _lib, build
    fields = {"im_paged_append_args": ("APPEND_ARGS", "k_dev v_dev q_dev q_out_dev token_start_dev position_dev cos_dev sin_dev q_norm_dev k_norm_dev pair_axis_host k_stride v_stride q_stride "
                                       "q_out_stride layer num_tokens num_heads table_dtype max_pos rotary_dim neighbours norm_dtype num_axes eps"),
              "im_paged_prefix_args": ("PREFIX_ARGS", " ".join("attention." + x for x in "q_dev out_dev token_start_dev mask_dev scratch_dev scratch_bytes q_stride out_stride layer num_heads num_tokens "
                                       "max_new mask_words max_len scale".split()) + " group_start_dev prefix_pages_dev num_groups max_group_new max_prefix"),
              "im_paged_weights_args": ("WEIGHTS_ARGS", " ".join("attention." + x for x in "q_dev out_dev token_start_dev mask_dev scratch_dev scratch_bytes q_stride out_stride layer num_heads num_tokens "
                                        "max_new mask_words max_len scale".split()) + " weights_dev seq_stride head_stride rows"),
              "im_paged_evict_args": ("EVICT_ARGS", "weights_dev weights_out_dev seq_len_out_dev layer_stride seq_stride head_stride out_layer_stride out_seq_stride out_head_stride budget recent")}
    lines = []
    for struct, (_, names) in fields.items():
        lines.append(f'printf("{struct} size %zu\\n", sizeof({struct}));')
        lines += [f'printf("{struct} {n} %zu\\n", offsetof({struct}, {n}));' for n in names.split()]
    src = tmp_path / "offsets.c"
    src.write_text('#include <stdio.h>\n#include "ironmill_cuda.h"\nint main(void) {' + "\n".join(lines) + "return 0;}\n")
    subprocess.run(["gcc", "-I", build.INCLUDE, str(src), "-o", str(tmp_path / "offsets")], check=True)
    got = {}
    for line in subprocess.run([str(tmp_path / "offsets")], capture_output=True, text=True, check=True).stdout.splitlines():
        s, n, v = line.split()
        got[s, n] = int(v)
    import struct as st
    for name, (packer, names) in fields.items():
        p = getattr(_lib, packer)
        assert p.size == got[name, "size"], name
        names = names.split()
        floats = {"eps", "attention.scale"}
        for i, n in enumerate(names):
            values = [0.0 if x in floats else 0 for x in names]
            values[i] = 1.0 if n in floats else 1
            raw = p.pack(*values)
            at = next(j for j, b in enumerate(raw) if b)
            assert (at - 2 if n in floats else at) == got[name, n], (name, n)      # the float 1.0 is 00 00 80 3f
    assert os.path.exists(build.INCLUDE) and st.calcsize("P") == 8


@pytest.mark.parametrize("change, word", [
    (dict(qn=PTR, q=0, qo=0, heads=0), "without queries"), (dict(norm=BF16), "norm weights are"), (dict(norm=7), "norm weights are"), (dict(norm=F32), GOOD), (dict(qn=0, kn=0, norm=7), GOOD),
    (dict(qn=PTR + 8), "16-byte"), (dict(kn=PTR + 2), "16-byte"), (dict(eps=-1e-6), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(eps=0.0), GOOD),
    (dict(axes=0), "axes"), (dict(axes=5), "axes"), (dict(axes=2), "the axis of every pair"), (dict(axes=2, axis=PTR, pos=0), "the axis of every pair"),
    (dict(axes=2, axis=PTR, rot=0), "the axis of every pair"), (dict(rot=127), "rotary_dim"), (dict(rot=130), "rotary_dim"), (dict(nb=2), "neighbours"), (dict(cos=0), "tables"),
    (dict(sin=PTR + 4), "16-byte"), (dict(table=BF16), "tables"), (dict(ks=248), "apart"), (dict(qos=504), "apart"), (dict(v=PTR + 2), "apart"), (dict(layer=2), "layer"), (dict(layer=-1), "layer"),
    (dict(k=0), "bad argument"), (dict(start=0), "bad argument"), (dict(n=-1), "bad argument"), (dict(qo=PTR + 1024), "other tokens"), (dict(max_pos=0), "tables")])
def test_append_refuses(lib, change, word):
    assert word in _message(lib, _append(lib, _kv(), **change))


@pytest.mark.parametrize("change, word", [
    (dict(groups=-1), "groups"), (dict(group_new=0), "groups"), (dict(bounds=0), "first sequences"), (dict(pages=0), "first sequences"), (dict(prefix=-1), "max_prefix"),
    (dict(groups=1 << 23, group_new=1 << 8), "too many"), (dict(max_new=0), "max_new"), (dict(heads=3), "multiple"), (dict(heads=0), "multiple"), (dict(words=0, mask=PTR), "mask"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(max_len=-1), "bad argument"), (dict(q=0), "bad argument"), (dict(out=PTR), "over the queries"), (dict(os=504), "apart"), (dict(q=PTR + 8), "apart"),
    (dict(layer=9), "layer")])
def test_prefix_attention_refuses(lib, change, word):
    assert word in _message(lib, _prefix(lib, _kv(), **change))
    if "group" not in " ".join(change) and "bounds" not in change and "pages" not in change and "prefix" not in change:
        assert word in _message(lib, _weights(lib, _kv(), **change))


@pytest.mark.parametrize("change, word", [
    (dict(w=0), "NULL"), (dict(w=17 * PTR + 2), "4-byte"), (dict(rows=0), "overlap"), (dict(sh=63), "overlap"), (dict(ss=127), "overlap"), (dict(w=PTR), "queries or the outputs"),
    (dict(w=9 * PTR + 2048), "queries or the outputs"), (dict(w=9 * PTR + 4096), GOOD), (dict(ss=0), "overlap"), (dict(sh=-64), "overlap"), (dict(sh=1 << 50), "overlap")])
def test_attention_with_sums_refuses(lib, change, word):
    assert word in _message(lib, _weights(lib, _kv(), **change))


@pytest.mark.parametrize("change, word", [
    (dict(budget=0), "budget"), (dict(recent=-1), "budget"), (dict(recent=11), "budget"), (dict(recent=10), GOOD), (dict(w=0), "bad argument"), (dict(wo=0), "bad argument"), (dict(lens=0), "bad argument"),
    (dict(wh=63), "apart"), (dict(ws=127), "apart"), (dict(wl=383), "apart"), (dict(oh=63), "apart"), (dict(os=127), "apart"), (dict(ol=383), "apart"), (dict(w=17 * PTR + 1), "4-byte"),
    (dict(wo=17 * PTR), "over what is read"), (dict(wo=17 * PTR + 4 * 767), "over what is read"), (dict(wo=17 * PTR + 4 * 768), GOOD), (dict(wo=4 * PTR), "over what is read"), (dict(wo=3 * PTR), "over what is read"),
    (dict(lens=17 * PTR), "new lengths"), (dict(lens=4 * PTR), "new lengths"), (dict(lens=3 * PTR), "new lengths"), (dict(lens=33 * PTR + 8), "new lengths")])
def test_eviction_refuses(lib, change, word):
    assert word in _message(lib, _evict(lib, _kv(), **change))


def test_eviction_refuses_tables_that_its_bits_do_not_hold(lib):
    assert "page tables" in _message(lib, _evict(lib, _kv(table_width=(1 << 15) + 1), wh=1 << 30, oh=1 << 30, ws=1 << 32, os=1 << 32, wl=1 << 34, ol=1 << 34))


@pytest.mark.parametrize("f", [_append, _prefix, _weights, _evict])
def test_calls_refuse_what_no_cache_is(lib, f):
    for change, word in ((dict(dtype=F32), "fp16 or bf16"), (dict(num_kv_heads=0), "heads"), (dict(k_dev=0), "NULL"), (dict(page_table_dev=0), "NULL"), (dict(head_dim=100), "head_dim"), (dict(table_width=0), "shape")):
        message = _message(lib, f(lib, _kv(**change), **(dict(qn=0, kn=0) if f is _append else {})))
        assert word in message or "shape" in message, (change, message)
    fn = {_append: "im_cuda_paged_append_normed", _prefix: "im_cuda_paged_prefix_attention", _weights: "im_cuda_paged_attention_weights", _evict: "im_cuda_paged_evict"}[f]
    assert "NULL" in _message(lib, _call(lib, fn, _kv(), None))
    assert "NULL" in _message(lib, f(lib, None))


@pytest.mark.parametrize("fn, n", [("im_cuda_paged_prefix_attention_scratch_bytes", 4), ("im_cuda_paged_attention_weights_scratch_bytes", 3)])
def test_scratch_sizes_without_a_device_are_none(lib, fn, n):
    assert getattr(lib, fn)(None, C.addressof(_kv()), *[1] * n) == 0


# ------------------------------------------------------------------------------------------------ the restatement itself
def test_plain_norm_and_axes_by_hand():
    x = np.array([[3.0, 4.0, 0.0, 0.0]])
    assert np.allclose(om.norm(x, np.array([1.0, 2.0, 1.0, 1.0]), 0.0), [[3 / 2.5, 8 / 2.5, 0, 0]])
    cos, sin = np.array([[1.0, 1.0], [0.0, 0.0]]), np.array([[0.0, 0.0], [1.0, 1.0]])
    y, _ = om.turn(np.array([[1.0, 2.0, 3.0, 4.0]]), cos, sin, [0, 1], 4, False, [0, 1])       # pair 0 stays, pair 1 (columns 1, 3) turns by a right angle
    assert y.tolist() == [[1.0, -4.0, 3.0, 2.0]]
    y, _ = om.turn(np.array([[1.0, 2.0, 3.0, 4.0]]), cos, sin, [1, 0], 4, True, [0, 1])
    assert y.tolist() == [[-2.0, 1.0, 3.0, 4.0]]


def test_plain_sums_by_hand():
    keys, values = np.zeros((2, 1, 2, 1)), np.ones((2, 1, 2, 1))
    sums = np.full((1, 1, 4), 5.0)
    _, _, _, got = om.attention(keys, values, np.array([[1, 0]]), [2], [0, 2], np.ones((2, 1, 1)), 1.0, weights=sums)
    assert np.allclose(got, [[[5 + 1 / 3 + 1 / 4, 5 + 1 / 3 + 1 / 4, 1 / 3 + 1 / 4, 1 / 4]]])


def test_plain_eviction_by_hand():
    keys = np.arange(8.0).reshape(1, 2, 1, 4, 1)
    values = -keys
    weights = np.array([[[[1.0, 9.0, 3.0, 3.0, 7.0, 3.0, 0.0, 0.0]]]])
    out = np.zeros_like(weights)
    lens = om.evict(keys, values, np.array([[0, 1]]), [8], weights, out, 5, 2)
    # of rows 0 .. 5 the three heaviest are 1, 4 and (the lowest of three equal ones) 2: rows 1 and 2 stay, 4 takes the place of 0; 6 and 7 follow
    assert lens.tolist() == [5] and keys.reshape(-1)[:5].tolist() == [4, 1, 2, 6, 7] and values.reshape(-1)[:5].tolist() == [-4, -1, -2, -6, -7]
    assert out.reshape(-1).tolist() == [7, 9, 3, 0, 0, 0, 0, 0]
