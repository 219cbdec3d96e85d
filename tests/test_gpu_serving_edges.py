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


@pytest.mark.parametrize("n,new,keys,tops", [(600, 1, 1 << 20, 4), (148, 20, 1 << 18, 1)])
def test_attention_rounds_small_weights_as_finely_as_large_ones_in_half(ctx, n, new, keys, tops):
    """Keys of weight 1.4 2^-24 against a largest of 1 (in each of the row
    kernel's warps), whose values are 1 where the largest's are 0, so that
    they are all of the output. A weight's rounding and the output's are 2^-11
    each; the products of 16 keys and the sum so far are cut at 2^-24 of the
    largest of the 17, a step; in the row kernel, a lane's sums of the weights
    round at 2^-24, a step. (As fractions of 1 the weights would be
    subnormals of half, 2^-24 each: 29 % off.) All requests share pages."""
    dim, page = 8, 128
    k = torch.zeros(keys // page, page, 1, dim, dtype=torch.float16, device="cuda")
    v = torch.ones_like(k)
    k.view(-1, dim)[0:16 * tops:16, 0] = 8.0
    v.view(-1, dim)[0:16 * tops:16] = 0.0
    q = torch.zeros(n * new, 1, dim, dtype=torch.float16, device="cuda")
    q[..., 0] = 1.0
    table = np.repeat(np.arange(keys // page)[None], n, axis=0)
    scale = float((24.0 - np.log2(1.4)) * np.log(2.0) / 8.0)
    got = _attend_run(ctx, k, v, table, [keys] * n, [new] * n, q, 1, scale, 0, "f16")
    seen = np.tile(np.arange(keys - new, keys) + 1.0, n)[:, None, None] - tops
    want = seen * 1.4 * 2.0 ** -24 / (tops + seen * 1.4 * 2.0 ** -24)
    steps = keys // tops // 16
    tol = 2.0 ** -10 + 17 * steps * 2.0 ** -24 + (steps * 2.0 ** -24 if new == 1 else 0.0)
    assert (np.abs(got / want - 1.0) <= tol).all(), (float(np.abs(got / want - 1.0).max()), tol)
