"""Descriptors and arguments of the head norms, the quantised cache and the prompt attention are checked before
the context is used, so a stand-in handle that is never dereferenced reaches the checks without a GPU."""
import ctypes as C

import pytest


def _quant(U, **k):
    return U.QuantDesc(**{**dict(format=U.T_Q8_0, dtype=U.T_F16, n_head_kv=2, head_dim=64, page=16, n_pages=4, n_seq=1, max_pages=4), **k})


@pytest.mark.parametrize("bad", [dict(format=2), dict(dtype=0), dict(page=0), dict(page=48), dict(head_dim=0), dict(head_dim=96),
                                 dict(head_dim=512), dict(n_head_kv=0), dict(n_pages=0), dict(n_seq=0), dict(max_pages=-1),
                                 dict(page=256, max_pages=1 << 24)])
def test_quantised_cache_descriptions(bad):
    import ulb_capi as U
    L, f = U.lib(), C.c_void_p(16)
    c = C.byref(_quant(U, **bad))
    d = C.byref(U.TreeDesc(4, 1, 1, 1, 0, 0.1))
    a = C.byref(U.QuantAppendArgs())
    for rc in (L.ulb_quant_attention(f, c, d, f, f, f, f, f, f, f, None, f, None), L.ulb_quant_append(f, f, c, a),
               L.ulb_quant_read(f, c, 1, f, f, f, f, f, 1, f, f), L.ulb_quant_row_bytes(c, C.byref(C.c_int())),
               L.ulb_quant_pages(c, 1, C.byref(U.CacheDesc()))):
        assert rc in (U.EINVAL, U.EUNSUPPORTED)
        assert L.ulb_last_error().startswith(b"ulb_quant_")


@pytest.mark.parametrize("fmt,dim,want", [(8, 64, 80), (8, 128, 144), (8, 256, 272), (3, 64, 48), (3, 128, 80), (3, 256, 160)])
def test_row_bytes_and_the_pools_as_16_bit_elements(fmt, dim, want):
    import ulb_capi as U
    d = _quant(U, format=fmt, head_dim=dim, n_pages=7, page=64)
    assert d.row_bytes == want
    v = d.pages_view(3)
    assert (v.dtype, v.n_layer, v.n_head_kv, v.head_dim, v.page, v.n_pages) == (U.T_F16, 3, 2, want // 2, 64, 7)
    with pytest.raises(U.UlbError):
        d.pages_view(0)


def test_null_arguments_and_empty_calls():
    import ulb_capi as U
    L, f = U.lib(), C.c_void_p(16)
    c = C.byref(_quant(U))
    assert L.ulb_norm_rope_apply(f, None, C.byref(U.NormRopeArgs()), f, f) == U.EINVAL
    assert L.ulb_norm_rope_apply(f, f, None, f, f) == U.EINVAL
    assert L.ulb_norm_rope_grad(f, None, C.byref(U.NormRopeArgs()), f, f, f, f, f, f) == U.EINVAL
    assert L.ulb_quant_append(f, None, c, C.byref(U.QuantAppendArgs())) == U.EINVAL
    assert L.ulb_quant_append(f, f, c, None) == U.EINVAL
    assert L.ulb_quant_read(None, c, 1, f, f, f, f, f, 1, f, f) == U.EINVAL
    assert L.ulb_quant_read(f, c, 1, f, f, f, f, None, 1, f, f) == U.EINVAL
    assert L.ulb_quant_read(f, c, 1, C.c_void_p(8), f, f, f, f, 1, f, f) == U.EINVAL
    assert L.ulb_quant_read(f, c, 1, f, f, f, C.c_void_p(18), f, 1, f, f) == U.EINVAL
    assert L.ulb_quant_read(f, c, 8, f, f, f, f, f, 1, f, f) == U.EUNSUPPORTED
    assert L.ulb_quant_attention(f, c, None, f, f, f, f, f, f, f, None, f, None) == U.EINVAL
    assert L.ulb_quant_attention(f, None, C.byref(U.TreeDesc(4, 1, 1, 1, 0, 0.1)), f, f, f, f, f, f, f, None, f, None) == U.EINVAL
    assert L.ulb_prompt_attention(f, None, f, f, f, f, f, f, None) == U.EINVAL
    # nothing to do is no error, whatever the pointers
    assert L.ulb_quant_attention(f, c, C.byref(U.TreeDesc(4, 0, 0, 0, 0, 0.1)), *[None] * 10) == U.OK
    assert L.ulb_quant_read(f, c, 1, None, None, None, None, None, 0, None, None) == U.OK
    d = U.PromptDesc(U.T_F16, 4, 2, 64, 0, 0, 0, 0, 0, 0.1)
    assert L.ulb_prompt_attention(f, C.byref(d), *[None] * 7) == U.OK


@pytest.mark.parametrize("bad", [dict(n_head=3), dict(n_head=0), dict(rows=-1), dict(mask_words=-1), dict(scale=0.0),
                                 dict(scale=float("nan")), dict(n_head=2 * 65), dict(mask_words=1)])
def test_rows_of_quantised_attention(bad):
    import ulb_capi as U
    L, f = U.lib(), C.c_void_p(16)
    d = U.TreeDesc(**{**dict(n_head=4, rows=1, max_rows=1, max_len=1, mask_words=0, scale=0.1), **bad})
    assert L.ulb_quant_attention(f, C.byref(_quant(U)), C.byref(d), f, f, f, f, f, f, f, None, f, None) in (U.EINVAL, U.EUNSUPPORTED)
    assert b"ulb_quant_attention" in L.ulb_last_error()


@pytest.mark.parametrize("at", [0, 1, 2, 9])
def test_unaligned_pointers_of_quantised_attention(at):
    import ulb_capi as U
    L, f = U.lib(), C.c_void_p(16)
    d = U.TreeDesc(4, 1, 1, 1, 0, 0.1)
    p = [f] * 7 + [None, f, None]
    p[at if at < 9 else 8] = C.c_void_p(24)
    assert L.ulb_quant_attention(f, C.byref(_quant(U)), C.byref(d), *p) == U.EINVAL
    for i in (3, 4, 5, 6, 9):
        p = [f] * 7 + [None, f, None]
        p[i] = C.c_void_p(18)
        assert L.ulb_quant_attention(f, C.byref(_quant(U)), C.byref(d), *p) == U.EINVAL


@pytest.mark.parametrize("bad", [dict(dtype=0), dict(head_dim=72), dict(n_head=3), dict(n_head_kv=0), dict(n_seq=-1), dict(q_rows=-1),
                                 dict(max_k=-1), dict(scale=0.0), dict(q_row=4 * 64 + 4), dict(k_row=64), dict(v_row=-8),
                                 dict(n_head=130)])
def test_prompt_descriptions(bad):
    import ulb_capi as U
    L, f = U.lib(), C.c_void_p(16)
    d = U.PromptDesc(**{**dict(dtype=U.T_F16, n_head=4, n_head_kv=2, head_dim=64, n_seq=1, q_rows=1, k_rows=1, max_q=1, max_k=1, scale=0.1), **bad})
    assert L.ulb_prompt_attention(f, C.byref(d), f, f, f, f, f, f, None) in (U.EINVAL, U.EUNSUPPORTED)
    assert b"ulb_prompt_attention" in L.ulb_last_error()


@pytest.mark.parametrize("at,addr", [(0, 8), (1, 8), (2, 8), (3, 18), (4, 18), (5, 8), (6, 18), (0, 0), (1, 0), (3, 0), (5, 0)])
def test_prompt_pointers(at, addr):
    import ulb_capi as U
    L, f = U.lib(), C.c_void_p(16)
    d = U.PromptDesc(U.T_F16, 4, 2, 64, 1, 1, 1, 1, 1, 0.1)
    p = [f] * 6 + [None]
    p[at] = C.c_void_p(addr) if addr else None
    assert L.ulb_prompt_attention(f, C.byref(d), *p) == U.EINVAL
