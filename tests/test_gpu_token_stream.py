"""The example that runs the serving operators together, against a dense
64-bit evaluation of the same model without a cache, and what the operators
promise about streams, graphs and device-side failures."""
import os
import sys

import numpy as np
import pytest

import kokopop_b200 as kb

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
import token_stream as ts  # noqa: E402


def _dense_logits(weights, embedding, ids):
    """Logits of every token of one sequence, in 64 bits."""
    w = {k: torch.from_numpy(v[2]).cuda().double() for k, v in weights.items()}
    x = torch.from_numpy(embedding).cuda().double()[torch.tensor(ids, device="cuda")]
    t, half = len(ids), ts.DIM // 2
    pos = torch.arange(t, device="cuda").double()[:, None, None]
    a = pos * 10000.0 ** (-torch.arange(half, device="cuda").double() / half)

    def norm(x):
        return (x - x.mean(-1, keepdim=True)) / (x.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt()

    def rotate(x):
        u, v = x[..., :half], x[..., half:]
        return torch.cat([u * a.cos() - v * a.sin(), u * a.sin() + v * a.cos()], -1)

    hide = torch.triu(torch.ones(t, t, device="cuda", dtype=torch.bool), 1)
    for i in range(ts.LAYERS):
        qkv = (norm(x) @ w[f"{i}.qkv"].T).view(t, -1, ts.DIM)
        q, k, v = rotate(qkv[:, :ts.HEADS]), rotate(qkv[:, ts.HEADS:ts.HEADS + ts.KV_HEADS]), qkv[:, -ts.KV_HEADS:]
        g = ts.HEADS // ts.KV_HEADS
        s = torch.einsum("qhd,khd->hqk", q, k.repeat_interleave(g, 1)) * ts.DIM ** -0.5
        p = torch.softmax(s.masked_fill(hide, -np.inf), -1)
        o = torch.einsum("hqk,khd->qhd", p, v.repeat_interleave(g, 1)).reshape(t, -1)
        x = x + o @ w[f"{i}.out"].T
        x = x + torch.nn.functional.gelu(norm(x) @ w[f"{i}.up"].T) @ w[f"{i}.down"].T
    return norm(x) @ w["logits"].T


def test_the_example_matches_a_dense_evaluation():
    """Each of about 9 values a layer is rounded to half (2^-11 relative at
    most): over the layers their independent errors add to sqrt(9 L) 2^-11 of
    the values' size; four times that bounds the logits' relative error in
    the 2-norm."""
    weights, embedding = ts.make_weights(3)
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, ts.VOCAB, n) for n in (1, 17, 130, 64, 33)]
    steps = 9
    m = ts.TokenStream(weights, embedding, len(prompts), 130 + steps + 1)
    try:
        tokens, logits = m.generate(prompts, steps)
        assert int(m.status[0][2]) == 0
        assert m.length.tolist() == [len(p) + steps for p in prompts]
        for r, p in enumerate(prompts):
            ids = list(p) + tokens[r].tolist()[:steps]
            want = _dense_logits(weights, embedding, ids)[len(p) - 1:]
            got = logits[r].double()
            rel = float((got - want).norm() / want.norm())
            assert rel <= 4 * (9 * ts.LAYERS) ** 0.5 * 2.0 ** -11, (r, rel)
    finally:
        m.close()


def test_the_example_gives_out_each_page_once():
    weights, embedding = ts.make_weights(5)
    m = ts.TokenStream(weights, embedding, 4, 64)
    try:
        m.generate([np.arange(n) for n in (16, 15, 1, 40)], 20)
        used = m.table[m.table >= 0].tolist()
        assert len(used) == len(set(used)) == sum(-(-(n + 20) // ts.PAGE) for n in (16, 15, 1, 40))
        assert sorted(used) == sorted(m.free[:len(used)].tolist())
    finally:
        m.close()


def _decode_setup(n, length, page, heads, kv, dim):
    g = torch.Generator(device="cuda")
    g.manual_seed(n)
    pages = n * -(-length // page)
    k, v = (torch.empty(pages, page, kv, dim, dtype=torch.float16, device="cuda").normal_(generator=g) for _ in "kv")
    q = torch.empty(n, heads, dim, dtype=torch.float16, device="cuda").normal_(generator=g)
    table = torch.randperm(pages, device="cuda", generator=g, dtype=torch.int32).view(n, -1)
    lens = torch.full((n,), length, dtype=torch.int32, device="cuda")
    cu = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    view = kb.PagedCache(k.data_ptr(), v.data_ptr(), kb.DTYPE_F16, pages, page, kv, dim)
    return view, q, table, lens, cu, (k, v)


def _attend(ctx, s, out, stream, max_new=1):
    view, q, table, lens, cu, _ = s
    ctx.paged_attention_device(view, q.shape[0], lens.data_ptr(), cu.data_ptr(), q.shape[0], max_new, int(lens.max()),
                               table.data_ptr(), table.shape[1], q.data_ptr(), q.stride(0), q.shape[1], 0.125, 0,
                               out.data_ptr(), out.stride(0), stream)


def test_a_captured_step_replays_with_new_lengths_and_inputs(ctx):
    """Tables, append, attention and a product captured once; the replay takes
    the lengths and values that then lie in the buffers, and equals direct
    calls. (A captured attention is not divided along the keys.)"""
    n, heads, kv, dim, page, cols = 3, 4, 2, 64, 16, 40
    dev = dict(device="cuda")
    k, v = (torch.zeros(n * cols, page, kv, dim, dtype=torch.float16, **dev) for _ in "kv")
    view = kb.PagedCache(k.data_ptr(), v.data_ptr(), kb.DTYPE_F16, n * cols, page, kv, dim)
    free, rng2 = torch.arange(n * cols, dtype=torch.int32, **dev), torch.tensor([0, n * cols], dtype=torch.int32, **dev)
    length, one = torch.zeros(n, dtype=torch.int32, **dev), torch.ones(n, dtype=torch.int32, **dev)
    table = torch.full((n, cols), -1, dtype=torch.int32, **dev)
    seq, cu = torch.zeros(n, dtype=torch.int32, **dev), torch.zeros(n + 1, dtype=torch.int32, **dev)
    status, slots = torch.zeros(3, dtype=torch.int32, **dev), torch.zeros(n, dtype=torch.int64, **dev)
    kv_new, q = torch.zeros(n, 2 * kv, dim, **dev), torch.zeros(n, heads, dim, dtype=torch.float16, **dev)
    out, y = torch.zeros_like(q), torch.zeros(n, 96, dtype=torch.float16, **dev)
    w, sc = kb.q4_pack(np.random.default_rng(0).normal(size=(96, heads * dim)).astype(np.float32), 64)
    w, sc = torch.from_numpy(w).cuda(), torch.from_numpy(sc).cuda()

    def step(stream):
        ctx.page_tables_device(n, page, cols, length.data_ptr(), one.data_ptr(), free.data_ptr(), n * cols,
                               rng2.data_ptr(), table.data_ptr(), seq.data_ptr(), cu.data_ptr(), n, slots.data_ptr(),
                               0, status.data_ptr(), stream)
        ctx.cache_append_device(view, n, slots.data_ptr(), kb.DTYPE_F32, kv_new.data_ptr(), 2 * kv * dim,
                                kv_new[:, kv:].data_ptr(), 2 * kv * dim, stream)
        ctx.paged_attention_device(view, n, seq.data_ptr(), cu.data_ptr(), n, 1, cols * page, table.data_ptr(), cols,
                                   q.data_ptr(), heads * dim, heads, 0.125, 0, out.data_ptr(), heads * dim, stream)
        ctx.q4_matvec_device(n, 96, heads * dim, 64, w.data_ptr(), sc.data_ptr(), kb.DTYPE_F16, out.data_ptr(),
                             heads * dim, 0, y.data_ptr(), 96, stream)

    def inputs(i):
        g = torch.Generator(device="cuda")
        g.manual_seed(i)
        kv_new.normal_(generator=g)
        q.normal_(generator=g)

    def run(do):
        for x in (k, v):
            x.zero_()
        table.fill_(-1)
        length.zero_()
        rng2[0] = 0
        got = []
        for i in range(20):
            inputs(i)
            do()
            torch.cuda.synchronize()
            got.append((out.clone(), y.clone(), slots.clone()))
            length.copy_(seq)
            rng2.copy_(status[:2])
        return got

    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    direct = run(lambda: step(kb.STREAM_LEGACY))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(torch.cuda.current_stream().cuda_stream)
    replayed = run(graph.replay)
    for a, b in zip(direct, replayed):
        assert torch.equal(a[2], b[2])
        # pieces and no pieces round alike but for the order of the sums
        assert float((a[0].double() - b[0].double()).abs().max()) <= 4 * 2.0 ** -11 * float(a[0].abs().max())
        assert float((a[1].double() - b[1].double()).norm()) <= 2.0 ** -8 * float(a[1].double().norm())


def test_calls_on_two_streams_share_the_workspace_in_order(ctx):
    """Divided attention on one context from two streams in turn, without a
    wait between them, gives what each gives alone."""
    a, b = _decode_setup(2, 6000, 16, 8, 2, 64), _decode_setup(5, 3000, 32, 8, 2, 64)
    want = []
    for s in (a, b):
        out = torch.zeros_like(s[1])
        _attend(ctx, s, out, kb.STREAM_LEGACY)
        torch.cuda.synchronize()
        want.append(out.clone())
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[torch.zeros_like(s[1]) for _ in range(10)] for s in (a, b)]
    torch.cuda.synchronize()
    for i in range(10):
        for j, s in enumerate((a, b)):
            _attend(ctx, s, outs[j][i], streams[j].cuda_stream)
    torch.cuda.synchronize()
    for j in range(2):
        for o in outs[j]:
            assert torch.equal(o, want[j])


def test_a_workspace_that_cannot_grow_is_reported_and_the_next_call_works():
    L = kb.load_library()
    c = kb.Context(0)
    try:
        s = _decode_setup(2, 6000, 16, 8, 2, 64)
        out = torch.zeros_like(s[1])
        torch.cuda.synchronize()
        assert L.kk_inject_allocation_failures(1) == kb.KK_OK
        with pytest.raises(kb.KKError) as e:
            _attend(c, s, out, kb.STREAM_LEGACY)
        assert e.value.code == kb.KK_ERROR_INFERENCE and "cudaMalloc" in str(e.value)
        assert L.kk_inject_allocation_failures(0) == kb.KK_OK
        _attend(c, s, out, kb.STREAM_LEGACY)
        torch.cuda.synchronize()
        first = out.clone()
        assert bool(first.isfinite().all()) and float(first.abs().max()) > 0
        n = [kb.ctypes.c_uint64(0), kb.ctypes.c_uint64(0)]
        L.kk_allocation_count(kb.ctypes.byref(n[0]))
        _attend(c, s, out, kb.STREAM_LEGACY)  # warm: nothing is allocated
        L.kk_allocation_count(kb.ctypes.byref(n[1]))
        torch.cuda.synchronize()
        assert n[0].value == n[1].value and torch.equal(out, first)
    finally:
        L.kk_inject_allocation_failures(0)
        c.close()


def test_the_decoder_is_unchanged_beside_the_serving_calls(ctx):
    """Serving calls between two decoder forwards of one context leave its
    results bit for bit."""
    from kokopop_b200 import workload as W
    ctx.upload(W.config2_weights())
    utts = [W.make_utterance(np.random.default_rng(9), t) for t in (7, 12)]
    want = ctx.decoder_forward(utts)
    s = _decode_setup(3, 5000, 16, 8, 2, 64)
    out = torch.zeros_like(s[1])
    _attend(ctx, s, out, torch.cuda.Stream().cuda_stream)
    for x, y in zip(ctx.decoder_forward(utts), want):
        np.testing.assert_array_equal(x, y)
    torch.cuda.synchronize()
