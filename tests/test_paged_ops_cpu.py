"""Descriptors and arguments of the paged cache operators are checked before the context is used, so
a stand-in handle that is never dereferenced reaches the checks without a GPU."""
import ctypes as C

import pytest


def _cache(U, **k):
    return U.CacheDesc(**{**dict(dtype=U.T_F16, n_layer=1, n_head_kv=2, head_dim=64, page=16, n_pages=4, n_seq=1, max_pages=4), **k})


@pytest.mark.parametrize("bad", [dict(dtype=0), dict(page=0), dict(page=48), dict(head_dim=0), dict(head_dim=260), dict(n_head_kv=0),
                                 dict(n_pages=0), dict(n_seq=0), dict(max_pages=-1), dict(pos_stride=12), dict(head_stride=-8),
                                 dict(pos_stride=32), dict(page=256, max_pages=1 << 24)])
def test_cache_descriptions(bad):
    import ulb_capi as U
    L, f = U.lib(), C.c_void_p(16)
    c = C.byref(_cache(U, **bad))
    d = C.byref(U.TreeDesc(4, 1, 1, 1, 0, 0.1))
    for rc in (L.ulb_tree_attention(f, c, d, f, f, f, f, f, f, f, None, f, None), L.ulb_pages_copy(f, c, f, f, f, 1),
               L.ulb_pages_compact(f, c, f, f, f, f, f, f, 1), L.ulb_pages_create(f, c, f, f, C.byref(C.c_void_p()))):
        assert rc in (U.EINVAL, U.EUNSUPPORTED)
        assert L.ulb_last_error().startswith(b"ulb_")


def test_null_arguments_and_empty_calls():
    import ulb_capi as U
    L, f = U.lib(), C.c_void_p(16)
    c = C.byref(_cache(U))
    assert L.ulb_use_stream(None, None) == U.EINVAL
    assert L.ulb_rope_create(f, None, None, C.byref(C.c_void_p())) == U.EINVAL
    assert L.ulb_rope_apply(f, None, U.T_F32, f, 0, 0, f, 1, 1, 0, f, 0, 0) == U.EINVAL
    assert L.ulb_rope_append(f, None, c, U.T_F32, f, 0, f, 0, f, 0, 1, f, f, f, f, 1, f, f, f) == U.EINVAL
    assert L.ulb_tree_attention(f, c, None, f, f, f, f, f, f, f, None, f, None) == U.EINVAL
    assert L.ulb_logits_process(f, None) == U.EINVAL
    assert L.ulb_pages_reserve(None, 0, 0, 1) == U.EINVAL
    assert L.ulb_pages_fork(None, 0, 1, 1) == U.EINVAL
    assert L.ulb_pages_truncate(None, 0, 0) == U.EINVAL
    assert L.ulb_pages_defrag(None, None) == U.EINVAL
    assert L.ulb_pages_info(None, None, None, -1, None) == U.EINVAL
    assert L.ulb_rope_free(None) == U.OK and L.ulb_pages_free(None) == U.OK
    # nothing to do is no error, whatever the pointers
    d = U.TreeDesc(4, 0, 0, 0, 0, 0.1)
    assert L.ulb_tree_attention(f, c, C.byref(d), None, None, None, None, None, None, None, None, None, None) == U.OK
    assert L.ulb_pages_copy(f, c, None, None, None, 0) == U.OK
    a = U.LogitsArgs(U.T_F32, 100, 0, 0, 0, 100, 100, 0, 0)
    assert L.ulb_logits_process(f, C.byref(a)) == U.OK


@pytest.mark.parametrize("bad", [dict(n_head=3), dict(n_head=0), dict(rows=-1), dict(mask_words=-1), dict(scale=0.0),
                                 dict(scale=float("inf")), dict(n_head=2 * 65), dict(mask_words=1)])
def test_tree_descriptions(bad):
    import ulb_capi as U
    L, f = U.lib(), C.c_void_p(16)
    d = U.TreeDesc(**{**dict(n_head=4, rows=1, max_rows=1, max_len=1, mask_words=0, scale=0.1), **bad})
    assert L.ulb_tree_attention(f, C.byref(_cache(U)), C.byref(d), f, f, f, f, f, f, f, None, f, None) in (U.EINVAL, U.EUNSUPPORTED)
    assert b"ulb_tree_attention" in L.ulb_last_error()


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(V=0), dict(ld_in=99), dict(ld_out=10), dict(rows=-1), dict(mask_words=-1)])
def test_logits_arguments(bad):
    import ulb_capi as U
    L = U.lib()
    a = U.LogitsArgs(dtype=U.T_F32, V=100, n_seq=1, rows=1, max_rows=1, ld_in=100, ld_out=100, in_=16, out=16, row_start=16)
    for k, v in bad.items():
        setattr(a, k, v)
    assert L.ulb_logits_process(C.c_void_p(16), C.byref(a)) in (U.EINVAL, U.EUNSUPPORTED)
    assert b"ulb_logits_process" in L.ulb_last_error()


def _addresses(n, odd):
    """n addresses, the one of number `odd` two bytes off."""
    return [C.c_void_p(66 if i == odd else 64) for i in range(n)]


@pytest.mark.parametrize("i", range(6))
def test_tree_arrays_at_odd_addresses(i):
    import ulb_capi as U
    f, d = C.c_void_p(64), U.TreeDesc(4, 1, 1, 1, 1, 0.1)
    table, start, prefix, length, mask, lse = _addresses(6, i)
    assert U.lib().ulb_tree_attention(f, C.byref(_cache(U)), C.byref(d), f, f, f, table, start, prefix, length, mask, f, lse) == U.EINVAL
    assert b"unaligned" in U.lib().ulb_last_error()


@pytest.mark.parametrize("i", range(5))
def test_page_move_arrays_at_odd_addresses(i):
    import ulb_capi as U
    f, c = C.c_void_p(64), C.byref(_cache(U))
    a = _addresses(5, i)
    if i == 0:
        assert U.lib().ulb_pages_copy(f, c, f, f, a[0], 1) == U.EINVAL
    else:
        assert U.lib().ulb_pages_compact(f, c, f, f, *a[1:], 1) == U.EINVAL
    assert b"unaligned" in U.lib().ulb_last_error()


@pytest.mark.parametrize("name", ["row_start", "params", "history", "history_start", "prompt", "node_tokens", "mask", "bias_start",
                                  "bias_tokens", "bias_values", "allow", "row_allow"])
def test_logits_arrays_at_odd_addresses(name):
    import ulb_capi as U
    a = U.LogitsArgs(dtype=U.T_F32, V=100, n_seq=1, rows=1, max_rows=1, ld_in=100, ld_out=100, mask_words=1, n_allow=1)
    for n, t in U.LogitsArgs._fields_:
        if t is C.c_void_p:
            setattr(a, n, 64)
    setattr(a, name, 66)
    assert U.lib().ulb_logits_process(C.c_void_p(64), C.byref(a)) == U.EINVAL
    assert b"unaligned" in U.lib().ulb_last_error()
