"""Arguments of the serving operators that no kernel could take safely are
refused before a GPU is touched."""
import numpy as np
import pytest

import kokopop_b200 as kb
from test_serving_abi import P, _append, _attend, _q4, _tables

TOP = 2 ** 31 - 1


@pytest.mark.parametrize("call,bad", [
    (_tables, dict(n_seqs=2 ** 30, n_free=0, seq_len=P + 2 ** 34, cu_new=P + 2 ** 35, status=P + 2 ** 36)),
    (_attend, dict(n_seqs=2 ** 30)),
    (_attend, dict(n_seqs=TOP)),
    # a chunk of k, or a block of outputs, past the last one would not fit 32 bits
    (_q4, dict(n_in=TOP // 128 * 128, x_stride=2 ** 31)),
    (_q4, dict(n_in=2 ** 31 - 65408, x_stride=2 ** 31)),
    (_q4, dict(n_out=TOP, out_stride=2 ** 31)),
    (_q4, dict(n_out=2 ** 31 - 65535, out_stride=2 ** 31)),
])
def test_sizes_whose_indices_pass_32_bits_are_refused(call, bad):
    assert call(**bad) == kb.KK_ERROR_INVALID_ARGUMENT
    assert "out of range" in kb.load_library().kk_last_error().decode()


@pytest.mark.parametrize("call,bad", [
    (_tables, {name: P + 2 ** 20 + 2}) for name in ("ctx_len", "new_len", "free_pages", "free_range", "table", "seq_len",
                                                    "cu_new", "positions", "status")
] + [(_attend, {name: P + 2}) for name in ("seq_len", "cu_new", "table")] + [(c, dict(slots=P + 4))
                                                                            for c in (_tables, _append)])
def test_arrays_that_are_not_aligned_to_their_type_are_refused(call, bad):
    assert call(**bad) == kb.KK_ERROR_INVALID_ARGUMENT
    assert "aligned" in kb.load_library().kk_last_error().decode()


def test_status_and_its_self_test_refuse_bad_arguments():
    L = kb.load_library()
    for rc in (L.kk_serving_status(None, None), L.kk_serving_wait_selftest(None, 1000, None),
               L.kk_serving_wait_selftest(P, 0, None), L.kk_serving_wait_selftest(P, 2000001, None)):
        assert rc == kb.KK_ERROR_INVALID_ARGUMENT
        assert L.kk_last_error().decode()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 7 * 65520.0, -1e30])
def test_q4_pack_refuses_weights_that_no_scale_holds(bad):
    """They would come back as NaN. 7 x 65504 still has a scale."""
    w = np.ones((3, 64), np.float32)
    w[1, 40] = 7 * 65504.0
    q, s = kb.q4_pack(w, 32)
    assert kb.q4_unpack(q, s, 32)[1, 40] == 7 * 65504.0
    w[2, 5] = bad
    with pytest.raises(kb.KKError) as e:
        kb.q4_pack(w, 32)
    assert e.value.code == kb.KK_ERROR_INVALID_ARGUMENT
