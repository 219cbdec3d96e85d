"""The serving operators of a token model against plain implementations in 64
bits: page tables and slots, the cache append, attention over the paged cache
and the products with 4-bit weights, at the sizes and masks where they can go
wrong. Tolerances follow from the roundings each operator documents."""
import numpy as np
import pytest

import kokopop_b200 as kb

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
KK = {"f32": kb.DTYPE_F32, "f16": kb.DTYPE_F16, "bf16": kb.DTYPE_BF16}
UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # relative rounding, to nearest, at most


def _i32(v):
    return torch.tensor(np.asarray(v, np.int64).astype(np.int32), device="cuda")


def _stream():
    return torch.cuda.current_stream().cuda_stream or kb.STREAM_LEGACY


# ---------------------------------------------------------------------------
# page tables
# ---------------------------------------------------------------------------

def _tables_plain(c, m, page, cols, free, head, end, table, n_tokens):
    table = table.copy()
    slots = np.full(n_tokens, -1, np.int64)
    positions = np.full(n_tokens, -1, np.int32)
    cu, short, at = [0], 0, 0
    for r, (a, k) in enumerate(zip(c, m)):
        a, k = max(a, 0), max(k, 0)
        for col in range(-(-a // page), min(-(-(a + k) // page), cols)):
            table[r, col] = free[head] if head < end else -1
            short += head >= end
            head += head < end
        for p in range(a, a + k):
            pg = table[r, p // page] if p // page < cols else -1
            slots[at] = pg * page + p % page if pg >= 0 else -1
            positions[at] = p
            at += 1
        cu.append(cu[-1] + k)
    seq = [max(a, 0) + max(k, 0) for a, k in zip(c, m)]
    return table, np.array(seq), np.array(cu), slots, positions, np.array([head, end, short])


def _tables_run(ctx, c, m, page, cols, free, rng2, table, n_tokens, with_positions=True):
    n = len(c)
    d_table, d_free, d_range = _i32(table), _i32(free), _i32(rng2)
    seq, cu, status = _i32(np.zeros(n)), _i32(np.zeros(n + 1)), _i32(np.zeros(3))
    slots = torch.full((n_tokens,), -7, dtype=torch.int64, device="cuda")
    pos = torch.full((n_tokens,), -7, dtype=torch.int32, device="cuda")
    d_c, d_m = _i32(c), _i32(m)
    ctx.page_tables_device(n, page, cols, d_c.data_ptr(), d_m.data_ptr(), d_free.data_ptr(), len(free),
                           d_range.data_ptr(), d_table.data_ptr(), seq.data_ptr(), cu.data_ptr(), n_tokens,
                           slots.data_ptr(), pos.data_ptr() if with_positions else 0, status.data_ptr(), _stream())
    torch.cuda.synchronize()
    return [x.cpu().numpy() for x in (d_table, seq, cu, slots, pos, status)]


TABLES = [
    # lengths before, new lengths, page, table width, free pages, extra rows
    ([0], [1], 16, 4, 8, 0),
    ([0], [0], 16, 4, 8, 0),
    ([15, 16, 17], [1, 1, 1], 16, 3, 8, 0),
    ([5, 0, 31, 32], [0, 0, 0, 0], 16, 4, 4, 5),
    ([3, 0, 100, 64], [130, 1, 0, 64], 32, 8, 20, 7),
    ([7, 0, 2], [9, 5, 1], 1, 20, 64, 0),
    ([10, 20, 30], [40, 40, 40], 24, 9, 2, 3),       # the free pages run out
    ([10, 20, 30], [40, 40, 40], 24, 2, 50, 0),      # the table is too narrow
    ([10, 500], [40, 9], 24, 2, 50, 0),              # one request is past its table already
    ([-3, 4], [5, -2], 4, 4, 9, 1),                  # negative lengths count as 0
    ([0, 0], [20000, 3], 128, 200, 400, 0),
    ([10, 20], [30, 30], 16, 8, 0, 0),               # no free page at all
]


@pytest.mark.parametrize("c,m,page,cols,n_free,extra", TABLES)
def test_page_tables_match_the_definition(ctx, c, m, page, cols, n_free, extra):
    rng = np.random.default_rng(len(c) * 1000 + page)
    free = rng.permutation(10 * n_free + 5)[:n_free] + 1000
    table = rng.integers(0, 900, (len(c), cols))
    n_tokens = sum(max(k, 0) for k in m) + extra
    want = _tables_plain(c, m, page, cols, free, 0, n_free, table, n_tokens)
    got = _tables_run(ctx, c, m, page, cols, free, [0, n_free], table, n_tokens)
    for name, x, y in zip(("table", "seq_len", "cu_new", "slots", "positions", "status"), got, want):
        np.testing.assert_array_equal(x, y, err_msg=name)


@pytest.mark.parametrize("n", [4095, 4096, 4097, 9000])
def test_page_tables_of_many_requests_in_several_chunks(ctx, n):
    rng = np.random.default_rng(n)
    c, m = rng.integers(0, 200, n).tolist(), rng.integers(0, 40, n).tolist()
    free = rng.permutation(n * 3)
    table = rng.integers(0, 900, (n, 16))
    want = _tables_plain(c, m, 16, 16, free, 5, n * 3 - 2, table, sum(m) + 1)
    got = _tables_run(ctx, c, m, 16, 16, free, [5, n * 3 - 2], table, sum(m) + 1)
    for x, y in zip(got, want):
        np.testing.assert_array_equal(x, y)


def test_page_tables_status_is_the_next_calls_free_range(ctx):
    """Two steps: the pages the first takes are not given out again, and the
    missing pages of the second are counted. positions may be left out."""
    free = np.arange(100, 107)
    table = np.full((2, 4), -1)
    t1 = _tables_run(ctx, [0, 0], [20, 5], 8, 4, free, [0, 7], table, 25)
    np.testing.assert_array_equal(t1[5], [4, 7, 0])
    t2 = _tables_run(ctx, t1[1].tolist(), [9, 20], 8, 4, free, t1[5][:2], t1[0], 29, with_positions=False)
    want = _tables_plain(t1[1].tolist(), [9, 20], 8, 4, free, 4, 7, t1[0], 29)
    for i in (0, 1, 2, 3, 5):
        np.testing.assert_array_equal(t2[i], want[i])
    np.testing.assert_array_equal(t2[5], [7, 7, 1])
    assert (t2[4] == -7).all()


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------

def _cache(n_pages, page, kv, dim, dtype, layout, fill=None, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    shape = (n_pages, page, kv, dim) if layout == "token" else (n_pages, kv, page, dim)
    made = []
    for _ in range(2):
        x = torch.empty(shape, dtype=DT[dtype], device="cuda")
        x.normal_(generator=g) if fill is None else x.fill_(fill)
        made.append(x if layout == "token" else x.transpose(1, 2))
    return made


def _view(k, v, dtype):
    return kb.PagedCache(k.data_ptr(), v.data_ptr(), KK[dtype], k.shape[0], k.shape[1], k.shape[2], k.shape[3],
                         k.stride(0), k.stride(1), k.stride(2))


@pytest.mark.parametrize("tokens,kv,dim,page,layout,source,dtype", [
    (1, 1, 8, 1, "token", "f32", "f16"),
    (1, 12, 64, 16, "head", "f16", "f16"),
    (7, 3, 24, 5, "token", "bf16", "f16"),
    (33, 8, 128, 16, "head", "f32", "bf16"),
    (300, 2, 96, 32, "token", "f16", "bf16"),
    (1025, 4, 40, 64, "head", "bf16", "bf16"),
])
def test_append_writes_each_row_to_its_slot_and_nothing_else(ctx, tokens, kv, dim, page, layout, source, dtype):
    rng = np.random.default_rng(tokens)
    n_pages = tokens // page + 3
    k, v = _cache(n_pages, page, kv, dim, dtype, layout)
    slots = rng.permutation(n_pages * page)[:tokens].astype(np.int64)
    slots[rng.random(tokens) < 0.1] = -1                      # tokens without a page
    slots[rng.random(tokens) < 0.05] = n_pages * page + 3      # and past the cache
    qkv = torch.randn(tokens, 4 * kv + 2, dim, device="cuda")  # rows of a wider projection, strided
    qkv[0, 0, 0], qkv[0, kv, 1] = float("nan"), float("inf")
    qkv[0, 1 if kv > 1 else 0, 2] = 1e30                       # overflows half to infinity
    qkv = qkv.to(DT[source])
    src_k, src_v = qkv[:, :kv], qkv[:, kv:2 * kv]
    want_k, want_v = k.clone(), v.clone()
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < n_pages * page:
            want_k[s // page, s % page] = src_k[t].to(DT[dtype])
            want_v[s // page, s % page] = src_v[t].to(DT[dtype])
    d_slots = torch.tensor(slots, device="cuda")
    ctx.cache_append_device(_view(k, v, dtype), tokens, d_slots.data_ptr(), KK[source], src_k.data_ptr(),
                            qkv.stride(0), src_v.data_ptr(), qkv.stride(0), _stream())
    torch.cuda.synchronize()
    for got, want in ((k, want_k), (v, want_v)):
        np.testing.assert_array_equal(got.float().cpu().numpy(), want.float().cpu().numpy())


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def _attend_plain(k, v, table, lens, new, q, heads, scale, window, dtype):
    """Output in 64 bits and the tolerance of each value: the weights' and
    the output's rounding (unit u each, of sum p |v| / sum p and of |out|),
    the 32-bit score (a sum of head_dim products, so head_dim + 8 roundings of
    scale |q| . |k|, twice: numerator and denominator; 2^-21 for exp2), the
    32-bit sums over the keys, and for half weights the subnormal spacing
    2^-25 against a largest weight of 1."""
    page, kv, dim = k.shape[1:]
    u = UNIT[dtype]
    outs, tols = [], []
    at = 0
    for r, (n, m) in enumerate(zip(lens, new)):
        j = np.arange(min(n, table.shape[1] * page))
        pg = table[r][j // page]
        j = j[(pg >= 0) & (pg < k.shape[0])]
        jj = torch.tensor(j, device="cuda", dtype=torch.int64)
        at_page = torch.tensor(table[r][j // page], device="cuda", dtype=torch.int64)
        kk, vv = k[at_page, jj % page].double(), v[at_page, jj % page].double()
        for t in range(m):
            p = n - m + t
            seen = jj <= p
            if window:
                seen &= jj > p - window
            o, e = torch.zeros(heads, dim, device="cuda").double(), torch.zeros(heads, dim, device="cuda").double()
            if bool(seen.any()):
                ks, vs = kk[seen], vv[seen]
                qq = q[at + t].double().view(kv, heads // kv, dim)
                s = torch.einsum("hgd,jhd->hgj", qq, ks) * scale
                size = float(torch.einsum("hgd,jhd->hgj", qq.abs(), ks.abs()).max()) * abs(scale)
                w = torch.softmax(s, dim=2)
                o = torch.einsum("hgj,jhd->hgd", w, vs).reshape(heads, dim)
                mass = torch.einsum("hgj,jhd->hgd", w, vs.abs()).reshape(heads, dim)
                c32 = 2 * ((dim + 8) * 2.0 ** -24 * size + 2.0 ** -21) + len(ks) * 2.0 ** -23
                e = (u + c32) * mass + u * o.abs() + 2.0 ** -25
                if dtype == "f16":
                    e = e + len(ks) * 2.0 ** -25 * float(vs.abs().max())
            outs.append(o)
            tols.append(e)
        at += m
    if not outs:
        return np.zeros((0, heads, dim)), np.zeros((0, heads, dim))
    return torch.stack(outs).cpu().numpy(), torch.stack(tols).cpu().numpy()


def _attend_setup(lens, new, heads, kv, dim, page, layout, dtype, seed=0, extra_cols=1, spare=2):
    rng = np.random.default_rng(seed)
    held = [-(-n // page) for n in lens]
    n_pages = sum(held) + spare
    order = rng.permutation(n_pages)
    table = np.full((len(lens), max(held + [1]) + extra_cols), -1, np.int64)
    at = 0
    for r, h in enumerate(held):
        table[r, :h] = order[at:at + h]
        at += h
    k, v = _cache(n_pages, page, kv, dim, dtype, layout, seed=seed + 1)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed + 2)
    q = torch.empty(sum(new), heads, dim, dtype=DT[dtype], device="cuda").normal_(generator=g)
    return k, v, table, q


def _attend_run(ctx, k, v, table, lens, new, q, heads, scale, window, dtype, pad_rows=0, max_new=None, max_len=None,
                stream=None):
    t = q.shape[0] + pad_rows
    qq = torch.cat([q, torch.full((pad_rows,) + q.shape[1:], float("nan"), dtype=q.dtype, device="cuda")])
    out = torch.full_like(qq, 77.0)
    d_len, d_cu, d_table = _i32(lens), _i32(np.cumsum([0] + list(new))), _i32(table)
    torch.cuda.synchronize()
    ctx.paged_attention_device(_view(k, v, dtype), len(lens), d_len.data_ptr(), d_cu.data_ptr(), t,
                               max(new) if max_new is None else max_new, max(lens) if max_len is None else max_len,
                               d_table.data_ptr(), table.shape[1], qq.data_ptr(), qq.stride(0), heads, scale, window,
                               out.data_ptr(), out.stride(0), _stream() if stream is None else stream)
    torch.cuda.synchronize()
    assert (out[q.shape[0]:] == 77.0).all()  # rows past the last new token are left alone
    return out[:q.shape[0]].double().cpu().numpy()


def _attend_check(ctx, lens, new, heads, kv, dim, page, window, layout, dtype, seed=0, **kw):
    k, v, table, q = _attend_setup(lens, new, heads, kv, dim, page, layout, dtype, seed)
    want, tol = _attend_plain(k, v, table, lens, new, q, heads, dim ** -0.5, window, dtype)
    got = _attend_run(ctx, k, v, table, lens, new, q, heads, dim ** -0.5, window, dtype, **kw)
    assert np.isfinite(got).all()
    worst = np.abs(got - want) / tol
    assert worst.max(initial=0.0) <= 1.0, float(worst.max())


ATTEND = [
    # lengths, new, heads, kv heads, dim, page, window, layout, type
    ([1], [1], 1, 1, 8, 16, 0, "token", "f16"),
    ([130], [1], 12, 12, 64, 16, 0, "token", "f16"),
    ([130], [130], 12, 12, 64, 16, 0, "head", "bf16"),
    ([17, 1, 400, 33], [1, 1, 1, 1], 32, 8, 128, 16, 0, "token", "bf16"),
    ([17, 1, 400, 33], [1, 1, 1, 1], 32, 8, 128, 16, 0, "token", "f16"),
    ([5, 0, 64, 9], [5, 0, 1, 0], 6, 2, 96, 32, 0, "head", "f16"),             # requests without new tokens
    ([100, 257, 63], [33, 57, 63], 28, 4, 128, 32, 0, "token", "bf16"),
    ([100, 257, 63], [33, 57, 63], 28, 4, 128, 32, 40, "token", "f16"),
    ([300, 80], [20, 7], 4, 4, 40, 24, 1, "token", "f16"),                      # a window of the token itself
    ([300, 80], [20, 7], 4, 4, 72, 1, 129, "head", "bf16"),                     # pages of one token
    ([90, 41], [3, 41], 20, 1, 64, 5, 0, "token", "bf16"),                      # more heads on a key than a tile's rows
    ([259], [129], 40, 2, 128, 64, 0, "head", "f16"),
    ([700, 523], [300, 211], 8, 2, 128, 128, 0, "token", "bf16"),
    ([700, 523], [300, 211], 8, 2, 64, 64, 200, "head", "f16"),
    ([513, 640, 128, 129], [257, 128, 128, 1], 16, 16, 64, 16, 0, "token", "bf16"),
    ([600], [256], 24, 8, 80, 256, 0, "token", "f16"),
]


@pytest.mark.parametrize("case", ATTEND, ids=lambda c: "-".join(map(str, c[2:])))
def test_attention_matches_the_definition(ctx, case):
    _attend_check(ctx, *case)


@pytest.mark.parametrize("window", [0, 700])
@pytest.mark.parametrize("new", [1, 70])
def test_attention_over_a_long_cache_in_pieces(ctx, window, new):
    """Few rows over thousands of keys, divided along the keys."""
    _attend_check(ctx, [5003, 2100], [new, 1], 8, 2, 128, 32, window, "token", "bf16")


@pytest.mark.parametrize("window", [0, 30])
def test_attention_of_many_short_requests(ctx, window):
    """Enough requests and few enough rows and keys for the row kernel."""
    rng = np.random.default_rng(7)
    new = rng.integers(1, 13, 80).tolist()
    lens = [int(n + rng.integers(0, 90)) for n in new]
    _attend_check(ctx, lens, new, 16, 4, 64, 16, window, "token", "bf16")


def test_attention_hints_do_not_change_what_is_computed(ctx):
    """max_new and max_len only choose the division of the work: too small
    or too large, the result is within the same tolerances."""
    for hints in ((1, 1), (1, 100000), (5000, 1), (0, 0)):
        _attend_check(ctx, [900, 333, 64], [130, 2, 1], 8, 2, 64, 16, 0, "token", "f16", max_new=hints[0],
                      max_len=hints[1])


def test_attention_repeats_bit_for_bit_and_leaves_padding_rows(ctx):
    lens, new = [3000, 41, 1500], [1, 1, 1]
    k, v, table, q = _attend_setup(lens, new, 16, 4, 128, 16, "token", "bf16")
    first = _attend_run(ctx, k, v, table, lens, new, q, 16, 0.1, 0, "bf16", pad_rows=5)
    for _ in range(5):
        np.testing.assert_array_equal(_attend_run(ctx, k, v, table, lens, new, q, 16, 0.1, 0, "bf16", pad_rows=5),
                                      first)


@pytest.mark.parametrize("page,new", [(16, [1, 3]), (24, [1, 3]), (64, [150, 90])])
def test_attention_ignores_what_lies_in_masked_places(ctx, page, new):
    """Cells past each request's tokens and pages outside every table hold
    NaN and infinities; missing pages (-1, or an index past the cache) drop
    their tokens; a request whose pages are all missing gives 0."""
    lens = [200, 333]
    k, v, table, q = _attend_setup(lens, new, 8, 2, 128, page, "token", "f16")
    used = {int(table[r][j // page]) * page + j % page for r, n in enumerate(lens) for j in range(n)}
    for cache, bad in ((k, float("nan")), (v, float("inf"))):
        flat = cache.view(-1, *cache.shape[2:])
        for s in range(flat.shape[0]):
            if s not in used:
                flat[s] = bad
                if s % 3 == 0:
                    flat[s] = -float("inf")
                if s % 3 == 1:
                    flat[s] = float("nan")
    table[0, 1], table[1, 2] = -1, k.shape[0] + 5
    for window in (0, 90):
        want, tol = _attend_plain(k, v, table, lens, new, q, 8, 0.125, window, "f16")
        got = _attend_run(ctx, k, v, table, lens, new, q, 8, 0.125, window, "f16")
        assert (np.abs(got - want) <= tol).all()
    table[1, :] = -1
    got = _attend_run(ctx, k, v, table, lens, new, q, 8, 0.125, 0, "f16")
    assert (got[new[0]:] == 0.0).all()
    # fewer tokens in the cache than new ones: the queries before the first key give 0
    want, tol = _attend_plain(k, v, table, [2, 1], new, q, 8, 0.125, 0, "f16")
    got = _attend_run(ctx, k, v, table, [2, 1], new, q, 8, 0.125, 0, "f16")
    assert (np.abs(got - want) <= tol).all()


def test_attention_passes_a_nan_that_a_query_sees(ctx):
    lens, new = [50], [1]
    k, v, table, q = _attend_setup(lens, new, 4, 4, 64, 16, "token", "bf16")
    k[table[0, 1], 3, 2] = float("nan")
    got = _attend_run(ctx, k, v, table, lens, new, q, 4, 0.1, 0, "bf16")
    assert np.isnan(got[0, 2]).all() and np.isfinite(got[0, [0, 1, 3]]).all()


@pytest.mark.parametrize("new", [1, 140])
def test_attention_with_offsets_past_32_bits(ctx, new):
    """Pages a little over 2^30 values apart: the third begins past 2^31."""
    kv, dim, page, stride = 2, 64, 128, (1 << 30) + 8
    big = [torch.empty(2 * stride + page * kv * dim, dtype=torch.float16, device="cuda") for _ in range(2)]
    caches = [torch.as_strided(b, (3, page, kv, dim), (stride, kv * dim, dim, 1)) for b in big]
    for c in caches:
        c.normal_()
    lens = [300]
    table = np.array([[2, 0, 1]])
    q = torch.randn(new, 4, dim, device="cuda").half()
    want, tol = _attend_plain(*caches, table, lens, [new], q, 4, 0.125, 0, "f16")
    got = _attend_run(ctx, *caches, table, lens, [new], q, 4, 0.125, 0, "f16")
    assert (np.abs(got - want) <= tol).all()


def test_attention_on_a_side_stream_and_strided_rows(ctx):
    """q and out as parts of wider rows, on a stream of the caller's; a call
    on another stream right after it shares the context's workspace."""
    lens, new, heads, kv, dim = [4000, 3500], [1, 1], 8, 2, 64
    k, v, table, q = _attend_setup(lens, new, heads, kv, dim, 16, "token", "f16")
    want, tol = _attend_plain(k, v, table, lens, new, q, heads, 0.125, 0, "f16")
    wide = torch.full((2, heads + 2 * kv, dim), 9.0, dtype=torch.float16, device="cuda")
    wide[:, :heads] = q
    outs = [torch.full((2, heads + 1, dim), 9.0, dtype=torch.float16, device="cuda") for _ in range(2)]
    d_len, d_cu, d_table = _i32(lens), _i32([0, 1, 2]), _i32(table)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s, out in zip(streams, outs):
        ctx.paged_attention_device(_view(k, v, "f16"), 2, d_len.data_ptr(), d_cu.data_ptr(), 2, 1, 4000,
                                   d_table.data_ptr(), table.shape[1], wide.data_ptr(), wide.stride(0), heads, 0.125,
                                   0, out.data_ptr(), out.stride(0), s.cuda_stream)
    torch.cuda.synchronize()
    for out in outs:
        assert (np.abs(out[:, :heads].double().cpu().numpy() - want) <= tol).all()
        assert (out[:, heads:] == 9.0).all()


# ---------------------------------------------------------------------------
# 4-bit products
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("rows,n_out,n_in,group,bias,dtype", [
    (1, 1, 32, 32, False, "f32"),
    (1, 512, 768, 32, True, "f32"),
    (3, 17, 160, 32, True, "f16"),
    (1, 4096, 4096, 64, False, "f16"),
    (8, 100, 320, 64, False, "bf16"),
    (9, 33, 384, 128, True, "f32"),
    (16, 129, 2048, 128, True, "bf16"),
    (37, 65, 96, 32, False, "f16"),
    (5, 2048, 768, 64, True, "f32"),
    (2, 31, 8192, 128, False, "f32"),
    (2, 40, 24704, 128, False, "f16"),
])
def test_q4_product_matches_the_definition(ctx, rows, n_out, n_in, group, bias, dtype):
    """Against 64 bits: any order of n_in 32-bit additions (each at most one
    unit in the last place, 2^-23) of the absolute products, the scaling of a
    group's sum and the bias, and the output's rounding."""
    g = torch.Generator(device="cuda")
    g.manual_seed(n_out + n_in)
    w = torch.randint(0, 256, (n_out, n_in // 2), dtype=torch.uint8, device="cuda", generator=g)
    sc = (torch.randn(n_out, n_in // group, device="cuda", generator=g) * 0.02).half()
    x = torch.randn(rows, n_in + 8, device="cuda", generator=g)
    if dtype == "f32":
        x *= torch.logspace(-20, 20, rows, device="cuda")[:, None]  # the whole range, not half's
    x = x.to(DT[dtype])[:, :n_in]
    b = torch.randn(n_out, device="cuda", generator=g) if bias else None
    out = torch.full((rows, n_out + 3), 5.0, dtype=DT[dtype], device="cuda")
    ctx.q4_matvec_device(rows, n_out, n_in, group, w.data_ptr(), sc.data_ptr(), KK[dtype], x.data_ptr(), x.stride(0),
                         b.data_ptr() if bias else 0, out.data_ptr(), out.stride(0), _stream())
    torch.cuda.synchronize()
    q = torch.empty(n_out, n_in, dtype=torch.float64, device="cuda")
    q[:, 0::2], q[:, 1::2] = (w.long() % 16 - 8).double(), (w.long() // 16 - 8).double()
    q *= sc.double().repeat_interleave(group, dim=1)
    want, size = x.double() @ q.T, x.double().abs() @ q.abs().T
    if bias:
        want, size = want + b.double(), size + b.double().abs()
    tol = (n_in + 4) * 2.0 ** -23 * size + UNIT[dtype] * want.abs() + 1e-30
    if dtype == "f16":
        tol = tol + 2.0 ** -25
    got = out[:, :n_out].double()
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / tol).max())
    if dtype == "f32" and n_in >= 768:
        # independent roundings grow with the square root of their number
        rel = float((got - want).norm(dim=1).div(want.norm(dim=1)).max())
        assert rel <= n_in ** 0.5 * 2.0 ** -23, rel
    assert (out[:, n_out:] == 5.0).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_q4_product_is_exact_on_whole_numbers(ctx, dtype):
    """Small whole numbers and a scale of 1 leave nothing to round."""
    rng = np.random.default_rng(5)
    n_out, n_in = 50, 256
    q = rng.integers(0, 16, (n_out, n_in))
    w = torch.tensor((q[:, 0::2] | q[:, 1::2] << 4).astype(np.uint8), device="cuda")
    sc = torch.ones(n_out, n_in // 32, device="cuda").half()
    x = np.zeros((3, n_in))
    x[:, ::17] = rng.integers(-1, 2, (3, len(range(0, n_in, 17))))
    d_x = torch.tensor(x, device="cuda").to(DT[dtype])
    out = torch.empty(3, n_out, dtype=DT[dtype], device="cuda")
    ctx.q4_matvec_device(3, n_out, n_in, 32, w.data_ptr(), sc.data_ptr(), KK[dtype], d_x.data_ptr(), n_in, 0,
                         out.data_ptr(), n_out, _stream())
    torch.cuda.synchronize()
    np.testing.assert_array_equal(out.double().cpu().numpy(), x @ (q - 8.0).T)


def test_q4_product_passes_infinities_and_nan_of_its_row_only(ctx):
    w = torch.full((20, 64), 0x99, dtype=torch.uint8, device="cuda")  # every weight 1
    sc = torch.ones(20, 1, device="cuda").half()
    for dtype in ("f32", "f16", "bf16"):
        x = torch.ones(3, 128, dtype=DT[dtype], device="cuda")
        x[0, 77], x[1, 5] = float("nan"), float("inf")
        out = torch.empty(3, 20, dtype=DT[dtype], device="cuda")
        ctx.q4_matvec_device(3, 20, 128, 128, w.data_ptr(), sc.data_ptr(), KK[dtype], x.data_ptr(), 128, 0,
                             out.data_ptr(), 20, _stream())
        torch.cuda.synchronize()
        assert bool(out[0].isnan().all()) and bool((out[2] == 128).all())
        assert bool((out[1] == float("inf")).all()), dtype
