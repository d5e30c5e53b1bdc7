"""The C entry points of the attention, page and scoring operators refuse bad
arguments before any CUDA call (no GPU needed)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from ie_tpq import _lib
from ie_tpq.kv_attention import _ARGS


def args(**kw):
    a = _lib.AttentionArgs()
    base = dict(q=4096, q_token_stride=256, q_head_stride=64, k_cache=4096, v_cache=4096,
                cache_slots=64, slot_stride=128, head_stride=64, block_tables=4096,
                table_stride=4, table_width=4, context_lens=4096, out=4096, out_token_stride=256,
                tokens=2, seqs=2, dtype=_lib.IE_DT_BF16, heads=4, kv_heads=2, head_dim=64,
                block_size=16, scale=0.125)
    base.update(kw)
    for name, value in base.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("kw", [
    dict(dtype=3), dict(heads=0), dict(kv_heads=3), dict(head_dim=0), dict(head_dim=257),
    dict(tokens=-1), dict(tokens=3), dict(seqs=1), dict(seqs=-1), dict(block_size=0),
    dict(table_width=1 << 30), dict(table_width=-1), dict(cache_slots=-1),
    dict(cache_slots=1 << 31), dict(window=-1), dict(sinks=-1), dict(max_query_len=-1),
    dict(max_context_len=-1), dict(scale=float("inf")),
    dict(scale=0.0), dict(scale=-0.1), dict(scale=float("nan")), dict(q=None),
    dict(out=None), dict(block_tables=None), dict(context_lens=None), dict(k_cache=None),
    dict(q=4097), dict(v_cache=4097), dict(out_token_stride=100), dict(prefix_len=1),
    dict(tokens=0, seqs=0, cu_seqlens_q=4096, window=-5)])
def test_window_attention(kw):
    a = args(**kw)
    assert _lib.lib().ie_window_attention(ctypes.byref(a), None, 0, None) == _lib.IE_ERR_INVALID
    assert _lib.last_error().startswith("window_attention")


@pytest.mark.parametrize("kw", [
    dict(tokens=(1 << 62) + 2, seqs=(1 << 62) + 2), dict(tokens=1 << 62, seqs=1 << 62),
    dict(tokens=(1 << 62) + 2, seqs=2, cu_seqlens_q=4096),
    dict(table_width=(1 << 60) + 4), dict(table_width=1 << 59, block_size=32),
    dict(table_width=1 << 33, block_size=(1 << 31) - 1)])
def test_sizes_whose_products_wrap(kw):
    a = args(**kw)
    for entry, name in ((_lib.lib().ie_window_attention, "window_attention"),
                        (_lib.lib().ie_shared_prefix_attention, "shared_prefix_attention")):
        assert entry(ctypes.byref(a), None, 0, None) == _lib.IE_ERR_INVALID
        assert _lib.last_error().startswith(name + ": a table of" if "table_width" in kw else
                                            f"{name}: {kw['tokens']} query tokens")
    assert _lib.lib().ie_attention_workspace_size(ctypes.byref(a)) == 0


@pytest.mark.parametrize("kw", [dict(window=4), dict(sinks=4), dict(prefix_len=65),
                                dict(prefix_len=-1), dict(heads=3)])
def test_shared_prefix_attention(kw):
    a = args(**kw)
    assert _lib.lib().ie_shared_prefix_attention(ctypes.byref(a), None, 0, None) == _lib.IE_ERR_INVALID
    assert _lib.last_error().startswith("shared_prefix_attention")


def test_workspace_that_is_missing_or_small():
    lib = _lib.lib()
    for a, entry in ((args(table_width=1 << 16), lib.ie_window_attention),
                     (args(table_width=4096, prefix_len=4096), lib.ie_shared_prefix_attention)):
        need = lib.ie_attention_workspace_size(ctypes.byref(a))
        assert need > 0
        for at, size in ((None, 0), (None, need), (4096, need - 1), (4104, need)):
            assert entry(ctypes.byref(a), at, size, None) == _lib.IE_ERR_INVALID
    assert lib.ie_attention_workspace_size(None) == 0
    assert lib.ie_attention_workspace_size(ctypes.byref(args(heads=3))) == 0
    assert lib.ie_window_attention(None, None, 0, None) == _lib.IE_ERR_INVALID


@pytest.mark.parametrize("cu", [None, 4096])
@pytest.mark.parametrize("dtype", [_lib.IE_DT_BF16, _lib.IE_DT_F32])
def test_a_window_without_limit_is_planned_like_none(cu, dtype):
    lib = _lib.lib()
    one = dict(tokens=1, seqs=1, heads=2, kv_heads=1, table_width=4096, table_stride=4096,
               cu_seqlens_q=cu, dtype=dtype)
    want = lib.ie_attention_workspace_size(ctypes.byref(args(**one)))
    assert want > 0
    for window, sinks in ((2 ** 63 - 1, 4), (2 ** 63 - 1, 2 ** 63 - 1), (1, 2 ** 63 - 1),
                          (65536, 0), (65535, 1)):
        a = args(window=window, sinks=sinks, **one)
        assert lib.ie_attention_workspace_size(ctypes.byref(a)) == want


@pytest.mark.parametrize("head_dim", [1, 33, 255])
def test_odd_head_sizes_leave_room_for_aligned_pairs(head_dim):
    """The parts' (m, l) pairs follow an odd number of f32 sums on an 8-byte boundary."""
    a = args(tokens=1, seqs=1, heads=1, kv_heads=1, head_dim=head_dim, q_token_stride=head_dim,
             q_head_stride=head_dim, out_token_stride=head_dim, slot_stride=head_dim,
             head_stride=head_dim, dtype=_lib.IE_DT_F32, table_width=12, table_stride=12)
    need = _lib.lib().ie_attention_workspace_size(ctypes.byref(a))     # three parts
    assert need == 16 + (3 * head_dim + 1) * 4 + 3 * 8


def test_nothing_to_do_is_not_an_error():
    a = args(tokens=0, seqs=0)
    assert _lib.lib().ie_window_attention(ctypes.byref(a), None, 0, None) == _lib.IE_OK
    assert _lib.lib().ie_shared_prefix_attention(ctypes.byref(a), None, 0, None) == _lib.IE_OK
    assert _lib.lib().ie_copy_pages(None, 0, 16, 4, None, None, 0, None) == _lib.IE_OK
    assert _lib.lib().ie_token_logprobs(None, 8, 2, 0, 8, None, 0, None, None, None, None,
                                        None) == _lib.IE_OK


def test_packed_arguments_have_the_structure_layout():
    names = [n for n, _ in _lib.AttentionArgs._fields_]
    values = list(range(1, len(names))) + [0.5]
    a = _lib.AttentionArgs.from_buffer_copy(_ARGS.pack(*values))
    assert [getattr(a, n) for n in names] == values


def copy(src, dst, pages=8, nbytes=32, caches=(4096, 8192)):
    ptr = (ctypes.c_void_p * len(caches))(*caches)
    s, d = np.asarray(src, dtype=np.int32), np.asarray(dst, dtype=np.int32)
    return _lib.lib().ie_copy_pages(ptr, len(caches), nbytes, pages, s.ctypes.data, d.ctypes.data,
                                    s.size, None)


@pytest.mark.parametrize("kw", [
    dict(src=[8], dst=[0]), dict(src=[0], dst=[-1]), dict(src=[0, 1], dst=[2, 2]),
    dict(src=[0, 1], dst=[3, 0]), dict(src=[1], dst=[1]), dict(src=[0], dst=[1], nbytes=0),
    dict(src=[0], dst=[1], nbytes=3), dict(src=[0], dst=[1], nbytes=1 << 29),
    dict(src=[0], dst=[1], pages=-1), dict(src=[0], dst=[5000], pages=5000),
    dict(src=[0], dst=[1], caches=(4096, 0)), dict(src=[0], dst=[1], caches=(4097, 4096))])
def test_copy_pages(kw):
    assert copy(**kw) == _lib.IE_ERR_INVALID
    assert _lib.last_error().startswith("copy_pages")


@pytest.mark.parametrize("pages", [
    np.array([2 ** 32 + 1, 2]), np.array([2 ** 31]), np.array([1.0, 2.0]), [1.5], [2 ** 40],
    [2 ** 70], np.array([-2 ** 32]), [-1], [True], np.array([2 ** 63], dtype=np.uint64), ["1"]])
def test_page_numbers_are_not_cast(pages):
    from ie_tpq.kv_pages import KVPagePool

    pool = KVPagePool.__new__(KVPagePool)     # its copy_pages refuses before it needs a cache
    with pytest.raises(ValueError):
        pool.copy_pages(pages, pages)


def test_page_numbers_of_any_integer_type():
    from ie_tpq.kv_pages import _page_numbers

    for pages in ([3, 0, 2], (3, 0, 2), np.array([3, 0, 2], dtype=np.uint8),
                  np.array([3, 9, 0, 9, 2], dtype=np.int64)[::2], np.array([3, 0, 2], dtype=">i4")):
        got = _page_numbers("src", pages)
        assert got.dtype == np.int32 and got.flags.c_contiguous and got.tolist() == [3, 0, 2]
    assert _page_numbers("src", []).shape == (0,)


def logprobs(**kw):
    a = dict(logits=4096, ld=100, dtype=_lib.IE_DT_F32, rows=2, vocab=100, tokens=4096, top=5,
             logprobs=4096, entropy=4096, top_logprobs=4096, top_tokens=4096, stream=None)
    a.update(kw)
    return _lib.lib().ie_token_logprobs(*a.values())


@pytest.mark.parametrize("kw", [
    dict(rows=-1), dict(vocab=0), dict(vocab=2097153, ld=1 << 22), dict(top=65), dict(top=-1),
    dict(vocab=4, top=5), dict(ld=-1), dict(dtype=4), dict(logits=None), dict(tokens=None),
    dict(logprobs=None), dict(entropy=None), dict(top_logprobs=None), dict(top_tokens=None),
    dict(logits=4098)])
def test_token_logprobs(kw):
    assert logprobs(**kw) == _lib.IE_ERR_INVALID
    assert _lib.last_error().startswith("token_logprobs")
