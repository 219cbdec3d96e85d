"""Forms of the serving operators that their other tests leave out: pages of
8 tokens and of 48, scales of 0 and below, every layout of the 4-bit product.
Same definitions and tolerances as there."""
import numpy as np
import pytest

from test_gpu_serving import (_attend_check, _attend_plain, _attend_run, _attend_setup,
                              test_q4_product_matches_the_definition as q4_check)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [8, 48])
@pytest.mark.parametrize("new", [[1, 1, 1], [70, 33, 1]])
def test_attention_with_pages_of_half_a_step_and_of_no_power_of_two(ctx, dim, page, new):
    """A step of one row is two pages of 8, a third of a page of 48; a chunk's
    is 16 pages of 8. One page is missing in the middle of a step."""
    lens, heads, kv = [300, 77, 129], 8, 2
    for window in (0, 50):
        _attend_check(ctx, lens, new, heads, kv, dim, page, window, "token", "f16")
    k, v, table, q = _attend_setup(lens, new, heads, kv, dim, page, "head", "bf16", seed=3)
    table[0, 1], table[0, 288 // page], table[2, 0] = -1, k.shape[0], -7
    for window in (0, 50):
        want, tol = _attend_plain(k, v, table, lens, new, q, heads, 0.1, window, "bf16")
        got = _attend_run(ctx, k, v, table, lens, new, q, heads, 0.1, window, "bf16")
        assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("scale", [-0.11, 0.0])
@pytest.mark.parametrize("new", [[1, 2], [150, 64]])
def test_attention_with_a_scale_of_zero_or_below(ctx, scale, new):
    """Also where the mask and a missing page leave some keys of a row, and
    where they leave none."""
    lens, heads, kv, dim, page = [300, 64], 4, 2, 64, 16
    k, v, table, q = _attend_setup(lens, new, heads, kv, dim, page, "token", "f16", seed=5)
    table[0, 4] = -1
    table[1, :] = -1
    for window in (0, 40):
        want, tol = _attend_plain(k, v, table, lens, new, q, heads, scale, window, "f16")
        got = _attend_run(ctx, k, v, table, lens, new, q, heads, scale, window, "f16")
        assert (np.abs(got - want) <= tol).all()
        assert (got[new[0]:] == 0.0).all()


# from 4736 outputs on, two warps of a block lie along them, from 16384 on four
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 8, 9, 16])
@pytest.mark.parametrize("n_out,n_in,group", [(4735, 96, 32), (4736, 320, 64), (4739, 2176, 128), (16383, 96, 32),
                                              (16384, 160, 32), (16401, 2176, 64)])
def test_q4_product_in_every_layout(ctx, n_out, n_in, group, rows, dtype):
    q4_check(ctx, rows, n_out, n_in, group, rows % 2 == 1, dtype)
