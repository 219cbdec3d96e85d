"""Cases and plain forms of the language-model serving operators.

A text model that feeds the synthesis front end token by token keeps a paged
key / value cache beside it. One step of it needs four operators:

  tables   pages and slots of the step's new tokens, from the request lengths
  append   the new tokens' keys and values into the paged cache
  attend   attention of the new tokens over the paged cache
  q4       products of a few rows with a 4-bit weight matrix

`listed()` gives the cases, `draw()` more of the same ranges, `prepare()` the
inputs, `run()` one pass: in elementary torch operations, or with `own` set
through the library. `exact()` is the definition in 64 bits.
"""
import math
import random

import numpy as np
import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}

# Sizes of the largest listed cases; draws stay inside them.
_MAX_TOKENS = 900000        # new tokens of one "tables" pass
_MAX_APPEND = 12000000      # values of K (and of V) that one "append" pass writes
_MAX_PAIRS = 8e8            # padded query head x key pairs of one "attend" pass
_MAX_CACHE = 300000000      # padded K values that one "attend" pass may read
_MAX_WEIGHT = 170000000     # 4-bit weights of one "q4" pass


def listed():
    return [
        # 64 streams that each take one token: the page tables of every decoding step
        {"name": "tables-decode", "op": "tables", "n": 64, "page": 16, "ctx": 2000, "new_lo": 1, "new_hi": 1,
         "max_pages": 256},
        # a server that takes in long prompts of many requests at once, some of them idle
        {"name": "tables-prefill", "op": "tables", "n": 2048, "page": 32, "ctx": 5000, "new_lo": 0, "new_hi": 1023,
         "max_pages": 512},
        # one decoding step of 64 streams: 64 tokens scattered over the cache
        {"name": "append-decode", "op": "append", "tokens": 64, "kv_heads": 8, "dim": 128, "page": 16,
         "layout": "token", "source": "bf16", "dtype": "bf16"},
        # prompts cut to chunks: thousands of tokens from 32-bit activations into a 16-bit cache
        {"name": "append-prefill", "op": "append", "tokens": 16381, "kv_heads": 12, "dim": 64, "page": 64,
         "layout": "head", "source": "f32", "dtype": "f16"},
        # one stream of a small model, a sentence of 130 tokens in the cache, one new token
        {"name": "attend-one", "op": "attend", "n": 1, "heads": 12, "kv_heads": 12, "dim": 64, "page": 16,
         "len_lo": 130, "len_hi": 130, "new_lo": 1, "new_hi": 1, "window": 0, "layout": "token", "dtype": "f16"},
        # 64 streams of mixed lengths, one token each, eight key heads shared by four query heads each
        {"name": "attend-decode", "op": "attend", "n": 64, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "len_lo": 17, "len_hi": 4099, "new_lo": 1, "new_hi": 1, "window": 0, "layout": "token", "dtype": "bf16"},
        # a few very long conversations, one token each: the long axis has to be split
        {"name": "attend-long", "op": "attend", "n": 7, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "len_lo": 30011, "len_hi": 65000, "new_lo": 1, "new_hi": 1, "window": 0, "layout": "head", "dtype": "bf16"},
        # short continuations of running streams with a sliding window, odd lengths
        {"name": "attend-window", "op": "attend", "n": 9, "heads": 28, "kv_heads": 4, "dim": 128, "page": 32,
         "len_lo": 700, "len_hi": 4500, "new_lo": 5, "new_hi": 131, "window": 1024, "layout": "token",
         "dtype": "f16"},
        # chunks of long prompts over what is cached already: the largest amount of arithmetic
        {"name": "attend-chunk", "op": "attend", "n": 3, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "len_lo": 5000, "len_hi": 7300, "new_lo": 1500, "new_hi": 2048, "window": 0, "layout": "token",
         "dtype": "bf16"},
        # one token through a linear layer of the encoder's size, 32-bit activations, with a bias
        {"name": "q4-small", "op": "q4", "rows": 1, "out": 512, "in": 768, "group": 32, "bias": True, "dtype": "f32"},
        # one stream through a square layer
        {"name": "q4-one", "op": "q4", "rows": 1, "out": 4096, "in": 4096, "group": 64, "bias": False,
         "dtype": "f16"},
        # eight streams through a wide layer, the largest weight
        {"name": "q4-wide", "op": "q4", "rows": 8, "out": 24576, "in": 8192, "group": 128, "bias": False,
         "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    """A size from lo to hi, spread over its logarithm; off the multiples of 1024, which every tile divides."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return v - (v % 1024 == 0)


def _cost(case):
    w = work(case)
    return w["bytes"] + w["flops"] / 256


def draw(rng):
    most = {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0), _cost(c))
    while True:
        case = _draw(rng)
        if _cost(case) <= most[case["op"]]:
            return case


def _draw(rng):
    op = rng.choice(["tables", "append", "attend", "attend", "attend", "q4"])
    if op == "tables":
        n = _log(rng, 1, 4096)
        hi = min(_log(rng, 1, 4000), _MAX_TOKENS // n)
        page = rng.choice([16, 32, 64, 128, 24])
        ctx = _log(rng, 1, 20000)
        return {"op": op, "n": n, "page": page, "ctx": ctx, "new_lo": rng.choice([0, hi]) if hi > 1 else 1,
                "new_hi": hi, "max_pages": -(-(ctx + hi) // page) + rng.randrange(9)}
    if op == "append":
        heads, dim = rng.choice([1, 2, 4, 8, 12, 16]), rng.choice([64, 96, 128])
        return {"op": op, "tokens": _log(rng, 1, _MAX_APPEND // (heads * dim)), "kv_heads": heads, "dim": dim,
                "page": rng.choice([16, 32, 64, 128, 24]), "layout": rng.choice(["token", "head"]),
                "source": rng.choice(["f32", "f16", "bf16"]), "dtype": rng.choice(["f16", "bf16"])}
    if op == "attend":
        heads, kv = rng.choice([(12, 12), (16, 16), (32, 8), (32, 4), (28, 4), (8, 1), (6, 2)])
        dim = rng.choice([64, 96, 128])
        n = _log(rng, 1, 128)
        hi = min(_log(rng, 64, 65000), _MAX_CACHE // (n * kv * dim))
        hi = max(hi, 32)
        new = 1 if rng.random() < 0.4 else _log(rng, 2, 2048)
        new = max(1, min(new, hi, int(_MAX_PAIRS / (n * heads * hi))))
        return {"op": op, "n": n, "heads": heads, "kv_heads": kv, "dim": dim, "page": rng.choice([16, 32, 64, 128]),
                "len_lo": max(1, new, int(hi * rng.choice([0.1, 0.5, 0.9]))), "len_hi": hi,
                "new_lo": rng.randint(1, new), "new_hi": new, "window": rng.choice([0, 0, 0, _log(rng, 33, 5000)]),
                "layout": rng.choice(["token", "head"]), "dtype": rng.choice(["f16", "bf16"])}
    group = rng.choice([32, 64, 128])
    n_in = group * (_log(rng, 256, 24576) // group | 1)  # no wider tile divides the row
    return {"op": op, "rows": _log(rng, 1, 16), "out": min(_log(rng, 256, 24576) | 1, _MAX_WEIGHT // n_in), "in": n_in,
            "group": group, "bias": rng.random() < 0.5, "dtype": rng.choice(["f32", "f16", "bf16"])}


def _between(case, lo, hi, n, salt):
    """n whole numbers from lo to hi that the case alone decides."""
    r = random.Random(repr((salt, sorted((k, v) for k, v in case.items() if k != "name"))))
    return [r.randint(lo, hi) for _ in range(n)]


def _lengths(case):
    """(tokens in the cache before the pass, new tokens) of each request."""
    n = case["n"]
    new = _between(case, case["new_lo"], case["new_hi"], n, "new")
    if case["op"] == "tables":
        return _between(case, 0, case["ctx"], n, "ctx"), new
    new[0] = case["new_hi"]
    total = _between(case, case["len_lo"], case["len_hi"], n, "len")
    total[-1] = case["len_hi"]
    return [max(0, t - m) for t, m in zip(total, new)], new


def _cells(case):
    """(query, key) pairs under the mask and keys that are read, over all requests."""
    pairs = keys = 0
    for c, m in zip(*_lengths(case)):
        w = case["window"] or c + m
        pairs += sum(min(c + t + 1, w) for t in range(m))
        keys += min(c + m, w + m - 1)
    return pairs, keys


def work(case):
    if case["op"] == "tables":
        c, m = _lengths(case)
        t, p = sum(m), case["page"]
        pages = sum(-(-(a + b) // p) - -(-a // p) for a, b in zip(c, m))
        return {"bytes": 16 * len(c) + 12 * t + 8 * pages, "flops": 0}
    if case["op"] == "append":
        n = 2 * case["tokens"] * case["kv_heads"] * case["dim"]
        return {"bytes": n * (_DT[case["source"]].itemsize + 2) + 8 * case["tokens"], "flops": 0}
    if case["op"] == "attend":
        pairs, keys = _cells(case)
        t = sum(_lengths(case)[1])
        return {"bytes": 2 * case["dim"] * (2 * t * case["heads"] + 2 * keys * case["kv_heads"]),
                "flops": 4 * case["dim"] * case["heads"] * pairs}
    n = case["out"] * case["in"]
    e = _DT[case["dtype"]].itemsize
    return {"bytes": n // 2 + 2 * (n // case["group"]) + e * case["rows"] * (case["in"] + case["out"]),
            "flops": 2 * n * case["rows"]}


def _cache(case, n_pages, g):
    """A filled cache, as [pages, page, heads, dim] whatever order its memory has."""
    h, p, d = case["kv_heads"], case["page"], case["dim"]
    shape = (n_pages, p, h, d) if case["layout"] == "token" else (n_pages, h, p, d)
    made = []
    for _ in range(2):
        x = torch.empty(shape, dtype=_DT[case["dtype"]], device="cuda").normal_(generator=g)
        made.append(x if case["layout"] == "token" else x.transpose(1, 2))
    return made


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case}
    if case["op"] == "tables":
        c, m = _lengths(case)
        n, p, cols = case["n"], case["page"], case["max_pages"]
        used = sum(-(-a // p) for a in c)
        need = sum(-(-(a + b) // p) - -(-a // p) for a, b in zip(c, m))
        order = torch.randperm(used + need + 64, device="cuda", generator=g, dtype=torch.int32)
        held = _ints([-(-a // p) for a in c])
        at = torch.arange(cols, device="cuda", dtype=torch.int32)[None] < held[:, None]
        table = torch.full((n, cols), -1, dtype=torch.int32, device="cuda")
        table[at] = order[:used]
        s.update(ctx_len=_ints(c), new_len=_ints(m), free=order[used:].clone(), table=table,
                 free_range=_ints([0, need + 64]), n_tokens=sum(m))
        t = s["n_tokens"]
        s.update(seq_len=_ints([0] * n), cu_new=_ints([0] * (n + 1)), status=_ints([0] * 3),
                 slots=torch.empty(t, dtype=torch.int64, device="cuda"),
                 positions=torch.empty(t, dtype=torch.int32, device="cuda"))
    elif case["op"] == "append":
        t, p = case["tokens"], case["page"]
        pages = -(-t // p) + 16
        s["k_cache"], s["v_cache"] = _cache(case, pages, g)
        order = torch.randperm(pages, device="cuda", generator=g)
        # runs of tokens fill pages in order; the tokens of a decoding step lie each on a page of its own
        i = torch.arange(t, device="cuda")
        s["slots"] = order[i // p] * p + i % p if t > 256 else torch.randperm(pages * p, device="cuda", generator=g)[:t]
        both = torch.empty((t, 2, case["kv_heads"], case["dim"]), dtype=_DT[case["source"]], device="cuda")
        both.normal_(generator=g)
        s["k"], s["v"] = both[:, 0], both[:, 1]  # as one projection writes them
    elif case["op"] == "attend":
        c, m = _lengths(case)
        n, p, t = case["n"], case["page"], sum(m)
        held = [-(-(a + b) // p) for a, b in zip(c, m)]
        order = torch.randperm(sum(held) + 8, device="cuda", generator=g, dtype=torch.int32)
        at = torch.arange(max(held) + 2, device="cuda", dtype=torch.int32)[None] < _ints(held)[:, None]
        table = torch.full(tuple(at.shape), -1, dtype=torch.int32, device="cuda")
        table[at] = order[:sum(held)]
        s["k_cache"], s["v_cache"] = _cache(case, sum(held) + 8, g)
        q = torch.empty((t, case["heads"], case["dim"]), dtype=_DT[case["dtype"]], device="cuda").normal_(generator=g)
        s.update(table=table, q=q, out=torch.empty_like(q), seq_len=_ints([a + b for a, b in zip(c, m)]),
                 cu_new=_ints([0] + np.cumsum(m).tolist()), max_new=max(m), max_len=max(a + b for a, b in zip(c, m)),
                 scale=case["dim"] ** -0.5)
    else:
        o, i, r = case["out"], case["in"], case["rows"]
        s["w"] = torch.randint(0, 256, (o, i // 2), dtype=torch.uint8, device="cuda", generator=g)
        sc = torch.rand((o, i // case["group"]), device="cuda", generator=g)
        s["scales"] = ((0.5 + sc) * (0.2 / math.sqrt(i))).half()
        s["x"] = torch.empty((r, i), dtype=_DT[case["dtype"]], device="cuda").normal_(generator=g)
        s["bias"] = torch.empty(o, device="cuda").normal_(generator=g) if case["bias"] else None
        s["out"] = torch.empty((r, o), dtype=_DT[case["dtype"]], device="cuda")
    return s


def _plain_tables(s):
    p, cols, t = s["case"]["page"], s["case"]["max_pages"], s["n_tokens"]
    c, m = s["ctx_len"].long(), s["new_len"].long()
    n = c.numel()
    old = (c + p - 1) // p
    need = (((c + m + p - 1) // p).clamp(max=cols) - old).clamp(min=0)
    first = need.cumsum(0) - need
    cu = torch.zeros(n + 1, dtype=torch.int64, device="cuda")
    cu[1:] = m.cumsum(0)
    head, end = s["free_range"][0].long(), s["free_range"][1].long()
    j = torch.arange(cols, device="cuda")[None] - old[:, None]
    at = head + first[:, None] + j
    page = torch.where(at < end, s["free"][at.clamp(0, s["free"].numel() - 1)], -1)
    s["table"].copy_(torch.where((j >= 0) & (j < need[:, None]), page, s["table"]))
    row = torch.repeat_interleave(torch.arange(n, device="cuda"), m, output_size=t)
    pos = c[row] + torch.arange(t, device="cuda") - cu[row]
    col = pos // p
    page = s["table"][row, col.clamp(max=cols - 1)].long()
    slots = torch.where((col < cols) & (page >= 0), page * p + pos % p, -1)
    total = need.sum()
    took = torch.minimum(total, end - head)
    status = torch.stack([head + took, end, total - took])
    return {"table": s["table"], "seq_len": (c + m).int(), "cu_new": cu.int(), "slots": slots,
            "positions": pos.int(), "status": status.int()}


def _plain_append(s):
    p = s["case"]["page"]
    at = (s["slots"] // p, s["slots"] % p)
    s["k_cache"][at] = s["k"].to(s["k_cache"].dtype)
    s["v_cache"][at] = s["v"].to(s["v_cache"].dtype)
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attend(s):
    case = s["case"]
    n, h, kv, d, p = case["n"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    g, t, m = h // kv, s["q"].shape[0], s["max_new"]
    pages = -(-s["max_len"] // p)
    table = s["table"][:, :pages].clamp(min=0)
    k = s["k_cache"][table].reshape(n, pages * p, kv, d).transpose(1, 2).float()
    v = s["v_cache"][table].reshape(n, pages * p, kv, d).transpose(1, 2).float()
    cu = s["cu_new"].long()
    new = cu[1:] - cu[:-1]
    step = torch.arange(m, device="cuda")
    q = s["q"][(cu[:-1, None] + step).clamp(max=t - 1)].float()
    q = q.reshape(n, m, kv, g, d).permute(0, 2, 1, 3, 4).reshape(n, kv, m * g, d)
    score = (q @ k.transpose(2, 3)).mul_(s["scale"]).view(n, kv, m, g, pages * p)
    pos = (s["seq_len"].long() - new)[:, None] + step
    key = torch.arange(pages * p, device="cuda")
    seen = key <= pos[..., None]
    if case["window"]:
        seen &= key > pos[..., None] - case["window"]
    score.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    prob = score.sub_(top).exp_()
    total = prob.sum(-1, keepdim=True)
    out = (prob.view(n, kv, m * g, pages * p) @ v).view(n, kv, m, g, d) / total.clamp(min=1e-30)
    out = out.permute(0, 2, 1, 3, 4).reshape(n * m, h, d)
    row = torch.repeat_interleave(torch.arange(n, device="cuda"), new, output_size=t)
    return out[row * m + torch.arange(t, device="cuda") - cu[row]].to(s["q"].dtype)


def _plain_q4(s):
    o, half = s["w"].shape
    q = torch.stack([s["w"] & 15, s["w"] >> 4], dim=-1).view(o, -1, s["case"]["group"]).float() - 8
    w = (q * s["scales"].float()[..., None]).view(o, 2 * half)
    y = s["x"].float() @ w.T
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["x"].dtype)


_handle = {}


def _library():
    """The library's context and data types, and the stream that torch works on."""
    if not _handle:
        import kokopop_b200 as kb
        _handle.update(kb=kb, ctx=kb.Context(torch.cuda.current_device()),
                       dt={torch.float32: kb.DTYPE_F32, torch.float16: kb.DTYPE_F16, torch.bfloat16: kb.DTYPE_BF16})
    kb = _handle["kb"]
    return kb, _handle["ctx"], _handle["dt"], torch.cuda.current_stream().cuda_stream or kb.STREAM_LEGACY


def _paged(kb, dt, s):
    k = s["k_cache"]
    return kb.PagedCache(s["k_cache"].data_ptr(), s["v_cache"].data_ptr(), dtype=dt[k.dtype], n_pages=k.shape[0],
                         page_size=k.shape[1], n_kv_heads=k.shape[2], head_dim=k.shape[3], page_stride=k.stride(0),
                         token_stride=k.stride(1), head_stride=k.stride(2))


def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        return {"tables": _plain_tables, "append": _plain_append, "attend": _plain_attend, "q4": _plain_q4}[op](s)
    kb, ctx, dt, stream = _library()
    if op == "tables":
        ctx.page_tables_device(s["case"]["n"], s["case"]["page"], s["case"]["max_pages"], s["ctx_len"].data_ptr(),
                               s["new_len"].data_ptr(), s["free"].data_ptr(), s["free"].numel(),
                               s["free_range"].data_ptr(), s["table"].data_ptr(), s["seq_len"].data_ptr(),
                               s["cu_new"].data_ptr(), s["n_tokens"], s["slots"].data_ptr(),
                               s["positions"].data_ptr(), s["status"].data_ptr(), stream)
        return {k: s[k] for k in ("table", "seq_len", "cu_new", "slots", "positions", "status")}
    if op == "append":
        ctx.cache_append_device(_paged(kb, dt, s), s["k"].shape[0], s["slots"].data_ptr(), dt[s["k"].dtype],
                                s["k"].data_ptr(), s["k"].stride(0), s["v"].data_ptr(), s["v"].stride(0), stream)
        return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if op == "attend":
        q, out = s["q"], s["out"]
        ctx.paged_attention_device(_paged(kb, dt, s), s["case"]["n"], s["seq_len"].data_ptr(),
                                   s["cu_new"].data_ptr(), q.shape[0], s["max_new"], s["max_len"],
                                   s["table"].data_ptr(), s["table"].shape[1], q.data_ptr(), q.stride(0), q.shape[1],
                                   s["scale"], s["case"]["window"], out.data_ptr(), out.stride(0), stream)
        return out
    x, out = s["x"], s["out"]
    ctx.q4_matvec_device(x.shape[0], out.shape[1], x.shape[1], s["case"]["group"], s["w"].data_ptr(),
                         s["scales"].data_ptr(), dt[x.dtype], x.data_ptr(), x.stride(0),
                         s["bias"].data_ptr() if s["bias"] is not None else 0, out.data_ptr(), out.stride(0), stream)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "tables":
        c, m = _lengths(case)
        p, cols = case["page"], case["max_pages"]
        free, table = s["free"].cpu().numpy(), s["table"].cpu().numpy()
        head, end = s["free_range"].tolist()
        slots, positions, short = [], [], 0
        for b, (a, k) in enumerate(zip(c, m)):
            for col in range(-(-a // p), min(-(-(a + k) // p), cols)):
                table[b, col] = free[head] if head < end else -1
                short += head >= end
                head += head < end
            pos = np.arange(a, a + k)
            page = table[b, np.minimum(pos // p, cols - 1)].astype(np.int64)
            slots.append(np.where((pos // p < cols) & (page >= 0), page * p + pos % p, -1))
            positions.append(pos)
        return {"table": table, "seq_len": np.array(c, np.int32) + np.array(m, np.int32),
                "cu_new": np.cumsum([0] + m).astype(np.int32), "slots": np.concatenate(slots),
                "positions": np.concatenate(positions).astype(np.int32),
                "status": np.array([head, end, short], np.int32)}
    if case["op"] == "append":
        return _plain_append({**s, "k": s["k"].double(), "v": s["v"].double(), "k_cache": s["k_cache"].double(),
                              "v_cache": s["v_cache"].double()})
    if case["op"] == "attend":
        kv, p, out = case["kv_heads"], case["page"], []
        for b, (c, m) in enumerate(zip(*_lengths(case))):
            at = s["table"][b, :-(-(c + m) // p)].long()
            k, v = (s[x][at].reshape(-1, kv, case["dim"])[:c + m].double() for x in ("k_cache", "v_cache"))
            q = s["q"][s["cu_new"][b]:s["cu_new"][b + 1]].double()
            pos = torch.arange(c, c + m, device="cuda")[:, None]
            key = torch.arange(c + m, device="cuda")[None]
            hide = (key > pos) | (key <= pos - (case["window"] or c + m))
            o = torch.empty_like(q)
            for head in range(case["heads"]):
                j = head // (case["heads"] // kv)
                a = (q[:, head] @ k[:, j].T * s["scale"]).masked_fill_(hide, -math.inf)
                o[:, head] = torch.softmax(a, dim=1) @ v[:, j]
            out.append(o)
        return torch.cat(out)
    w = s["w"].long()
    q = torch.empty((case["out"], case["in"]), dtype=torch.float64, device="cuda")
    q[:, 0::2], q[:, 1::2] = (w % 16 - 8).double(), (w // 16 - 8).double()
    q *= s["scales"].double().repeat_interleave(case["group"], dim=1)
    y = s["x"].double() @ q.T
    return y + s["bias"].double() if case["bias"] else y
