"""The serving operators refuse bad arguments before they touch a GPU: each
call below is right but for one argument."""
import ctypes

import numpy as np
import pytest

import kokopop_b200 as kb

FAKE = 0x10000  # aligned, never read: the checks come first
P = FAKE


def _cache(**kw):
    a = dict(k_ptr=P, v_ptr=P, dtype=kb.DTYPE_F16, n_pages=4, page_size=16, n_kv_heads=2, head_dim=64)
    a.update(kw)
    return kb.PagedCache(**a)


def _tables(**kw):
    a = dict(ctx=P, n_seqs=2, page_size=16, max_pages=4, ctx_len=P, new_len=P, free_pages=P, n_free=8, free_range=P,
             table=P, seq_len=P + 32, cu_new=P + 48, n_tokens=2, slots=P, positions=P, status=P + 64, stream=0)
    a.update(kw)
    return kb.load_library().kk_page_tables_device(*a.values())


def _append(**kw):
    a = dict(ctx=P, cache=_cache(), n_tokens=2, slots=P, dtype=kb.DTYPE_F32, k=P, k_stride=128, v=P, v_stride=128,
             stream=0)
    a.update(kw)
    return kb.load_library().kk_cache_append_device(*a.values())


def _attend(**kw):
    a = dict(ctx=P, cache=_cache(), n_seqs=2, seq_len=P, cu_new=P, n_tokens=2, max_new=1, max_len=9, table=P,
             max_pages=4, q=P, q_stride=256, n_heads=4, scale=0.1, window=0, out=P, out_stride=256, stream=0)
    a.update(kw)
    return kb.load_library().kk_paged_attention_device(*a.values())


def _q4(**kw):
    a = dict(ctx=P, n_rows=1, n_out=8, n_in=128, group=32, w=P, scales=P, dtype=kb.DTYPE_F32, x=P, x_stride=128,
             bias=None, out=P, out_stride=8, stream=0)
    a.update(kw)
    return kb.load_library().kk_q4_matvec_device(*a.values())


BAD_CACHE = [dict(k_ptr=0), dict(v_ptr=0), dict(k_ptr=P + 8), dict(dtype=kb.DTYPE_F32), dict(dtype=99),
             dict(n_pages=0), dict(page_size=0), dict(n_kv_heads=0), dict(head_dim=0), dict(head_dim=60),
             dict(head_dim=136), dict(token_stride=129), dict(page_stride=-8), dict(head_stride=4)]


@pytest.mark.parametrize("call,bad", [
    (_tables, b) for b in (dict(ctx=None), dict(ctx_len=None), dict(new_len=None), dict(free_pages=None),
                           dict(free_range=None), dict(table=None), dict(seq_len=None), dict(cu_new=None),
                           dict(slots=None), dict(status=None), dict(n_seqs=0), dict(page_size=0), dict(max_pages=0),
                           dict(n_free=-1), dict(n_tokens=-1), dict(status=P + 4), dict(free_range=P + 72),
                           dict(seq_len=P + 4), dict(cu_new=P), dict(new_len=P + 36), dict(ctx_len=P + 56))
] + [
    (_append, b) for b in (dict(ctx=None), dict(cache=None), dict(slots=None), dict(k=None), dict(v=None),
                           dict(n_tokens=-1), dict(dtype=7), dict(k=P + 4), dict(k_stride=120), dict(v_stride=130),
                           dict(dtype=kb.DTYPE_F16, v_stride=132))
] + [
    (_attend, b) for b in (dict(ctx=None), dict(cache=None), dict(seq_len=None), dict(cu_new=None), dict(table=None),
                           dict(q=None), dict(out=None), dict(n_seqs=0), dict(n_tokens=-1), dict(n_tokens=1 << 31),
                           dict(max_new=-1), dict(max_len=-1), dict(max_pages=0), dict(n_heads=3), dict(n_heads=0),
                           dict(scale=float("nan")), dict(window=-1), dict(q=P + 2), dict(out=P + 8),
                           dict(q_stride=248), dict(q_stride=257), dict(out_stride=260))
] + [
    (_q4, b) for b in (dict(ctx=None), dict(w=None), dict(scales=None), dict(x=None), dict(out=None),
                       dict(n_rows=-1), dict(n_out=0), dict(n_in=0), dict(group=16), dict(group=96),
                       dict(n_in=144), dict(dtype=5), dict(w=P + 4), dict(x=P + 8), dict(x_stride=120),
                       dict(x_stride=130), dict(out_stride=7), dict(out=P + 2), dict(bias=P + 2), dict(scales=P + 1),
                       dict(n_rows=1 << 20))
] + [(c, dict(cache=_cache(**b))) for b in BAD_CACHE for c in (_append, _attend)])
def test_one_bad_argument_is_refused_with_a_message(call, bad):
    L = kb.load_library()
    assert call(**bad) == kb.KK_ERROR_INVALID_ARGUMENT
    assert L.kk_last_error().decode()


def test_no_tokens_is_no_work():
    """Without a row there is nothing to read: no pointer is needed."""
    assert _append(n_tokens=0, slots=None, k=None, v=None) == kb.KK_OK
    assert _attend(n_tokens=0, q=None, out=None) == kb.KK_OK
    assert _q4(n_rows=0, x=None, out=None) == kb.KK_OK


def test_the_python_methods_raise():
    c = kb.Context.__new__(kb.Context)
    c.L, c.h = kb.load_library(), None
    for call in (lambda: c.cache_append_device(_cache(), 1, P, kb.DTYPE_F32, P, 128, P, 128),
                 lambda: c.paged_attention_device(_cache(), 1, P, P, 1, 1, 1, P, 1, P, 256, 4, 0.1, 0, P, 256),
                 lambda: c.q4_matvec_device(1, 8, 32, 32, P, P, kb.DTYPE_F32, P, 32, 0, P, 8),
                 lambda: c.page_tables_device(1, 16, 4, P, P, P, 1, P, P, P, P, 1, P, 0, P + 64)):
        with pytest.raises(kb.KKError) as e:
            call()
        assert e.value.code == kb.KK_ERROR_INVALID_ARGUMENT


def test_the_cache_structure_has_the_headers_layout():
    c = kb.PagedCache(1, 2, kb.DTYPE_BF16, 3, 4, 5, 8)
    assert ctypes.sizeof(c) == 64
    assert (c.page_stride, c.token_stride, c.head_stride) == (4 * 5 * 8, 40, 8)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_q4_pack_is_the_nearest_of_its_grid(group):
    rng = np.random.default_rng(group)
    w = rng.normal(0.0, 1.0, (7, 384)).astype(np.float32)
    w[2, :group] = 0.0  # a group of zeros has scale 0
    q, s = kb.q4_pack(w, group)
    assert q.dtype == np.uint8 and q.shape == (7, 192) and s.dtype == np.float16 and s.shape == (7, 384 // group)
    assert s[2, 0] == 0.0
    back = kb.q4_unpack(q, s, group)
    step = np.repeat(s.astype(np.float32), group, axis=1)
    # half a step, and what rounding the scale to half takes from the 7 steps of the largest
    assert (np.abs(back - w) <= step * (0.5 + 7 * 2.0 ** -11) + 1e-6).all()
    assert back[0, 5] == ((q[0, 2] >> 4) - 8.0) * np.float32(s[0, 0])


def test_q4_pack_refuses_other_shapes():
    for w, group in ((np.zeros(64), 32), (np.zeros((2, 48)), 32), (np.zeros((2, 64)), 16)):
        with pytest.raises(kb.KKError):
            kb.q4_pack(w, group)
