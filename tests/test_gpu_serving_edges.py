"""Edges of the serving operators: requests longer than their tables, idle
slots, weights and values at the ends of their types. Definitions and
tolerances as in test_gpu_serving.py unless a test says otherwise."""
import numpy as np
import pytest

from test_gpu_serving import DT, KK, UNIT, _attend_check, _attend_plain, _attend_run, _attend_setup, _stream

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


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 9])
def test_q4_product_of_the_largest_values_is_finite_where_the_definition_is(ctx, dtype, rows):
    """A group's sum of x (q - 8) can pass the largest float although its
    product with the scale does not."""
    n_out, n_in, group = 40, 256, 128
    big = torch.finfo(DT[dtype]).max
    x = torch.full((rows, n_in), big, device="cuda").to(DT[dtype])
    x[:, 1::3] *= -0.25
    x[:, group:] *= 2.0 ** -20
    w = torch.zeros(n_out, n_in // 2, dtype=torch.uint8, device="cuda")  # every weight -8
    w[1::2] = 0xff                                                       # or 7
    sc = torch.full((n_out, n_in // group), 2.0 ** -11, device="cuda").half()
    out = torch.empty(rows, n_out, dtype=DT[dtype], device="cuda")
    ctx.q4_matvec_device(rows, n_out, n_in, group, w.data_ptr(), sc.data_ptr(), KK[dtype], x.data_ptr(), n_in, 0,
                         out.data_ptr(), n_out, _stream())
    torch.cuda.synchronize()
    q = torch.full((n_out, n_in), -8.0, dtype=torch.float64, device="cuda")
    q[1::2] = 7.0
    q *= 2.0 ** -11
    want, size = x.double() @ q.T, x.double().abs() @ q.abs().T
    assert float(want.abs().max()) < torch.finfo(torch.float32).max
    tol = (n_in + 4) * 2.0 ** -23 * size + UNIT[dtype] * want.abs()
    assert bool(((out.double() - want).abs() <= tol).all())


def test_q4_product_of_small_values_keeps_their_bits(ctx):
    """F32 rows around 2^-100: nothing but the 32-bit sums rounds, apart from
    what of a product of an x below 2^-115 is below the smallest float (2^-149,
    2^11 times that in the result, times the scale)."""
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    rows, n_out, n_in, group = 3, 70, 640, 64
    x = torch.randn(rows, n_in, device="cuda", generator=g) * 2.0 ** -100
    w = torch.randint(0, 256, (n_out, n_in // 2), dtype=torch.uint8, device="cuda", generator=g)
    sc = torch.rand(n_out, n_in // group, device="cuda", generator=g).half()
    out = torch.empty(rows, n_out, device="cuda")
    ctx.q4_matvec_device(rows, n_out, n_in, group, w.data_ptr(), sc.data_ptr(), KK["f32"], x.data_ptr(), n_in, 0,
                         out.data_ptr(), n_out, _stream())
    torch.cuda.synchronize()
    q = torch.empty(n_out, n_in, dtype=torch.float64, device="cuda")
    q[:, 0::2], q[:, 1::2] = (w.long() % 16 - 8).double(), (w.long() // 16 - 8).double()
    q *= sc.double().repeat_interleave(group, dim=1)
    want, size = x.double() @ q.T, x.double().abs() @ q.abs().T
    tol = (n_in + 4) * 2.0 ** -23 * size + 3 * n_in * 2.0 ** -138
    assert bool(((out.double() - want).abs() <= tol).all())
    rel = float((out.double() - want).norm(dim=1).div(want.norm(dim=1)).max())
    assert rel <= n_in ** 0.5 * 2.0 ** -23, rel


@pytest.mark.parametrize("new,slots,at", [(1, 64, 37), (70, 64, 0), (70, 300, 299)])
def test_idle_slots_do_not_change_the_division_of_the_keys(ctx, new, slots, at):
    """A request alone and the same one among slots without new tokens (some
    with keys in the cache): one division of its keys, so the same bits."""
    k, v, table, q = _attend_setup([5000], [new], 8, 2, 64, 16, "token", "bf16")
    alone = _attend_run(ctx, k, v, table, [5000], [new], q, 8, 0.125, 0, "bf16")
    lens, news = [i % 2 * 40 for i in range(slots)], [0] * slots
    lens[at], news[at] = 5000, new
    many = np.repeat(table, slots, axis=0)
    got = _attend_run(ctx, k, v, many, lens, news, q, 8, 0.125, 0, "bf16")
    np.testing.assert_array_equal(got, alone)


@pytest.mark.parametrize("new", [(5, 8), (12, 12)])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_many_short_requests_on_either_kernel(ctx, dim, new):
    """Up to 32 rows on average, and 48: heads of 128 change kernels between."""
    rng = np.random.default_rng(dim)
    new = rng.integers(new[0], new[1] + 1, 160).tolist()
    lens = [int(n + rng.integers(0, 60)) for n in new]
    for window in (0, 20):
        _attend_check(ctx, lens, new, 8, 2, dim, 16, window, "token", "f16")
