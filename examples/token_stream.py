"""A small decoder-only token model served with the paged-cache operators.

Several requests of different lengths run together, as the text model in front
of the synthesis would: their prompts in one pass, then a token each per step.
A step is

    page tables -> per layer: qkv product -> cache append -> attention ->
                   output product -> feed-forward products -> logits

with 4-bit weights, a paged F16 cache and everything on the device, the free
pages included: no length is read back. Weights are random; the point is how
the calls fit together.

    python examples/token_stream.py [--requests 6] [--steps 24]
"""
from __future__ import annotations

import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import kokopop_b200 as kb  # noqa: E402

VOCAB, HIDDEN, LAYERS, HEADS, KV_HEADS, DIM, FFN = 178, 512, 2, 8, 2, 64, 2048
GROUP, PAGE = 64, 16


def make_weights(seed: int = 0):
    """{name: (bytes, scales, float32 values of the 4-bit weights)} and the embedding."""
    rng = np.random.default_rng(seed)
    shapes = {"logits": (VOCAB, HIDDEN)}
    for i in range(LAYERS):
        shapes[f"{i}.qkv"] = ((HEADS + 2 * KV_HEADS) * DIM, HIDDEN)
        shapes[f"{i}.out"] = (HIDDEN, HEADS * DIM)
        shapes[f"{i}.up"] = (FFN, HIDDEN)
        shapes[f"{i}.down"] = (HIDDEN, FFN)
    weights = {}
    for name, (n_out, n_in) in shapes.items():
        w = rng.normal(0.0, n_in ** -0.5, (n_out, n_in)).astype(np.float32)
        weights[name] = kb.q4_pack(w, GROUP) + (kb.q4_unpack(*kb.q4_pack(w, GROUP), GROUP),)
    return weights, rng.normal(0.0, 1.0, (VOCAB, HIDDEN)).astype(np.float32)


def rotate(x: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
    """Rotary positions on [tokens, heads, DIM], in 32 bits."""
    half = DIM // 2
    freq = 10000.0 ** (-torch.arange(half, device=x.device, dtype=torch.float32) / half)
    a = positions[:, None, None].float() * freq
    u, v = x.float()[..., :half], x.float()[..., half:]
    return torch.cat([u * a.cos() - v * a.sin(), u * a.sin() + v * a.cos()], dim=-1)


def norm(x: torch.Tensor) -> torch.Tensor:
    return torch.nn.functional.layer_norm(x.float(), x.shape[-1:])


class TokenStream:
    """The requests' cache and lengths on the device, and one step of them all."""

    def __init__(self, weights, embedding, n_requests: int, max_tokens: int, device: int = 0):
        self.ctx = kb.Context(device)
        self.device = torch.device("cuda", device)
        to = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(self.device)  # noqa: E731
        self.w = {k: (to(q), to(s.view(np.int16)), q.shape[0], 2 * q.shape[1]) for k, (q, s, _) in weights.items()}
        self.embedding = to(embedding)
        self.n, self.cols = n_requests, -(-max_tokens // PAGE)
        pages = n_requests * self.cols
        shape = (LAYERS, 2, pages, PAGE, KV_HEADS, DIM)
        self.cache = torch.empty(shape, dtype=torch.float16, device=self.device)
        self.views = [kb.PagedCache(self.cache[i, 0].data_ptr(), self.cache[i, 1].data_ptr(), kb.DTYPE_F16, pages, PAGE,
                                    KV_HEADS, DIM) for i in range(LAYERS)]
        ints = lambda n, fill=0: torch.full((n,), fill, dtype=torch.int32, device=self.device)  # noqa: E731
        self.free = torch.randperm(pages, device=self.device, dtype=torch.int32)
        self.table = ints(n_requests * self.cols, -1).view(n_requests, self.cols)
        self.length, self.seq_len, self.cu_new = ints(n_requests), ints(n_requests), ints(n_requests + 1)
        self.status = [ints(3), ints(3)]  # the free range left, used in turn
        self.status[0][1] = pages
        self.longest = 0

    def product(self, name: str, x: torch.Tensor, stream: int) -> torch.Tensor:
        w, scales, n_out, n_in = self.w[name]
        x = x.half().contiguous()
        out = torch.empty((x.shape[0], n_out), dtype=torch.float16, device=self.device)
        self.ctx.q4_matvec_device(x.shape[0], n_out, n_in, GROUP, w.data_ptr(), scales.data_ptr(), kb.DTYPE_F16,
                                  x.data_ptr(), n_in, 0, out.data_ptr(), n_out, stream)
        return out

    def step(self, tokens: torch.Tensor, new: torch.Tensor, max_new: int) -> torch.Tensor:
        """tokens: the new tokens of all requests, one after another; new: how
        many of each request (int32, on the device). Returns the logits of
        every token."""
        stream = torch.cuda.current_stream(self.device).cuda_stream or kb.STREAM_LEGACY
        t = tokens.shape[0]
        self.longest += max_new
        slots = torch.empty(t, dtype=torch.int64, device=self.device)
        positions = torch.empty(t, dtype=torch.int32, device=self.device)
        before, after = self.status
        self.ctx.page_tables_device(self.n, PAGE, self.cols, self.length.data_ptr(), new.data_ptr(),
                                    self.free.data_ptr(), self.free.shape[0], before.data_ptr(), self.table.data_ptr(),
                                    self.seq_len.data_ptr(), self.cu_new.data_ptr(), t, slots.data_ptr(),
                                    positions.data_ptr(), after.data_ptr(), stream)
        x = self.embedding[tokens]
        for i in range(LAYERS):
            qkv = self.product(f"{i}.qkv", norm(x), stream).view(t, HEADS + 2 * KV_HEADS, DIM)
            q = rotate(qkv[:, :HEADS], positions).half()
            k = rotate(qkv[:, HEADS:HEADS + KV_HEADS], positions)
            v = qkv[:, HEADS + KV_HEADS:].float()
            self.ctx.cache_append_device(self.views[i], t, slots.data_ptr(), kb.DTYPE_F32, k.data_ptr(),
                                         KV_HEADS * DIM, v.data_ptr(), KV_HEADS * DIM, stream)
            o = torch.empty_like(q)
            self.ctx.paged_attention_device(self.views[i], self.n, self.seq_len.data_ptr(), self.cu_new.data_ptr(), t,
                                            max_new, self.longest, self.table.data_ptr(), self.cols, q.data_ptr(),
                                            HEADS * DIM, HEADS, DIM ** -0.5, 0, o.data_ptr(), HEADS * DIM, stream)
            x = x + self.product(f"{i}.out", o.view(t, HEADS * DIM), stream).float()
            h = torch.nn.functional.gelu(self.product(f"{i}.up", norm(x), stream).float())
            x = x + self.product(f"{i}.down", h, stream).float()
        logits = self.product("logits", norm(x), stream)
        # the next step starts from the new lengths and the pages left
        self.length, self.seq_len = self.seq_len, self.length
        self.status = [after, before]
        return logits

    def generate(self, prompts, steps: int):
        """Greedy continuations: ([steps + 1 tokens of each request], logits of
        each step, the prompts' last token's first)."""
        new = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device=self.device)
        tokens = torch.tensor(np.concatenate(prompts), dtype=torch.int64, device=self.device)
        ends = new.cumsum(0) - 1
        logits = [self.step(tokens, new, max(len(p) for p in prompts))[ends]]
        one = torch.ones_like(new)
        out = [logits[0].argmax(-1)]
        for _ in range(steps):
            logits.append(self.step(out[-1], one, 1))
            out.append(logits[-1].argmax(-1))
        self.ctx.serving_status(torch.cuda.current_stream(self.device).cuda_stream or kb.STREAM_LEGACY)
        return torch.stack(out, dim=1), torch.stack(logits, dim=1)

    def close(self):
        torch.cuda.synchronize(self.device)
        self.ctx.close()


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--requests", type=int, default=6)
    ap.add_argument("--steps", type=int, default=24)
    a = ap.parse_args()
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, VOCAB, rng.integers(1, 130)) for _ in range(a.requests)]
    weights, embedding = make_weights()
    m = TokenStream(weights, embedding, a.requests, max(len(p) for p in prompts) + a.steps + 1)
    tokens, _ = m.generate(prompts, a.steps)
    for p, t in zip(prompts, tokens.tolist()):
        print(f"prompt of {len(p):3d} tokens -> {t}")
    print("free pages left:", int(m.status[0][1] - m.status[0][0]), "missing:", int(m.status[0][2]))
    m.close()


if __name__ == "__main__":
    main()
