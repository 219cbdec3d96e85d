"""Edges of the serving operators: requests longer than their tables, idle
slots, weights and values at the ends of their types. Definitions and
tolerances as in test_gpu_serving.py unless a test says otherwise."""
import numpy as np
import pytest

from test_gpu_serving import _attend_plain, _attend_run, _attend_setup

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("page,cols", [(16, 64), (256, 4), (24, 43)])
@pytest.mark.parametrize("new", [[1, 1, 1], [40, 3, 40]])
def test_attention_of_requests_past_their_tables(ctx, page, cols, new):
    """Positions past the table's last page count as masked: with a window
    some queries, or all of a tile's, have nothing left to see. The last
    request's length is the largest that a length can be."""
    heads, kv, dim, held = 8, 2, 128, page * cols
    k, v, table, q = _attend_setup([held] * 3, new, heads, kv, dim, page, "token", "bf16", extra_cols=0)
    assert table.shape[1] == cols
    for lens in ([held + 576, held + 17, 2 ** 31 - 1], [200000, held + 1, 2 ** 31 - 2]):
        for window in (0, 8, 30, 100, 600):
            want, tol = _attend_plain(k, v, table, lens, new, q, heads, 0.1, window, "bf16")
            for hint in (max(lens), held):
                got = _attend_run(ctx, k, v, table, lens, new, q, heads, 0.1, window, "bf16", max_len=hint)
                assert (np.abs(got - want) <= tol).all(), (lens, window)
                if 0 < window <= 100:
                    assert (got[-new[2]:] == 0.0).all()
