"""Continuous decoding with the token-scaled products and the paged cache.

A small Llama-shaped model with random weights: every product is int8 with a
scale per token and per output channel (`quantize_rows`, `matmul_rows`), the
keys and values live in int8 pages (`kv_append`), and attention reads those
pages (`paged_attention`).  Ragged prompts go through in one call; then all
sequences decode together, one token each, in a CUDA graph that holds the whole
step.  At the end the logits are compared with the same model in plain fp32.

    python examples/paged_decode.py [--layers 4 --dim 1024 --steps 64 ...]
"""
from __future__ import annotations

import argparse
import importlib
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
lq = importlib.import_module("llama2-min-inference_b200")

TYPES = {"f32": (torch.float32, lq.F32), "f16": (torch.float16, lq.F16), "bf16": (torch.bfloat16, lq.BF16)}


class Rows:
    """Memory for up to `rows` int8 rows of `cols` with a scale each, and its descriptor."""

    def __init__(self, rows: int, cols: int):
        self.q = torch.empty(rows, lq.row8_pitch(cols), dtype=torch.int8, device="cuda")
        self.s = torch.empty(rows, device="cuda")
        self.desc = lq.QuantizedTensor(q=self.q.data_ptr(), s=self.s.data_ptr(), rows=rows, cols=cols, group_size=cols,
                                       kind=lq.KIND_ROW8)

    def fill(self, x: torch.Tensor, dtype: int):
        self.desc.rows = x.shape[0]
        lq.quantize_rows(self.desc, x.data_ptr(), x.shape[1], dtype, x.stride(0))
        return self.desc


class Linear:
    """y = x W^T with W int8, a scale per row of W and per row of x."""

    def __init__(self, weight: torch.Tensor):
        self.weight = weight  # fp32, for the comparison at the end
        self.rows = Rows(*weight.shape)
        self.rows.fill(weight, lq.F32)

    def __call__(self, x: "lq.QuantizedTensor", dtype) -> torch.Tensor:
        d, n = self.weight.shape
        y = torch.empty(x.rows, d, dtype=dtype[0], device="cuda")
        lq.matmul_rows(y.data_ptr(), x, self.rows.desc, n, d, dtype[1])
        return y


def norm(x):
    f = x.float()
    return (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-5)).to(x.dtype)


class Model:
    def __init__(self, a, seed: int = 0):
        self.a, self.dtype = a, TYPES[a.dtype]
        self.hs = a.dim // a.heads
        gen = torch.Generator(device="cuda").manual_seed(seed)

        def linear(d, n):
            return Linear(torch.randn(d, n, generator=gen, device="cuda") * n**-0.5)

        width = (a.heads + 2 * a.kv_heads) * self.hs
        self.embed = torch.randn(a.vocab, a.dim, generator=gen, device="cuda").to(self.dtype[0])
        self.layers = [dict(qkv=linear(width, a.dim), o=linear(a.dim, a.dim), up=linear(2 * a.hidden, a.dim),
                            down=linear(a.dim, a.hidden)) for _ in range(a.layers)]
        self.head = linear(a.vocab, a.dim)
        self.rope = torch.from_numpy(lq.rope_table(a.max_context, self.hs)).cuda()
        # the cache: one pool of pages per layer, a sequence's pages anywhere in it
        per = -(-a.max_context // a.page)
        self.n_pages = per * a.seqs
        self.pages = torch.randperm(self.n_pages, generator=gen, device="cuda").to(torch.int32).view(a.seqs, per)
        cell = a.kv_heads * 2
        self.pools = []
        for _ in self.layers:
            codes = torch.empty(self.n_pages * cell * self.hs * a.page, dtype=torch.int8, device="cuda")
            scales = torch.empty(self.n_pages * cell, device="cuda")
            self.pools.append((codes, scales, lq.PagedKV(codes=codes.data_ptr(), scales=scales.data_ptr(),
                                                         n_pages=self.n_pages, page_size=a.page,
                                                         n_kv_heads=a.kv_heads, head_size=self.hs)))
        rows = a.seqs * a.prompt  # the most rows of one call
        self.xq = {n: Rows(rows, n) for n in {a.dim, a.hidden}}

    def batch(self, row_start, context, max_rows):
        return lq.KVBatch(row_start=row_start.data_ptr(), context=context.data_ptr(), pages=self.pages.data_ptr(),
                          n_seqs=self.a.seqs, n_rows=0, max_pages=self.pages.shape[1], max_rows=max_rows,
                          max_context=self.a.max_context)

    def forward(self, tokens, batch, last):
        """Logits of rows `last` after the batch's new tokens, which the cache then holds."""
        a, hs, (torch_type, code) = self.a, self.hs, self.dtype
        size = torch_type.itemsize
        x = self.embed[tokens]
        batch.n_rows = x.shape[0]
        for layer, (_, _, pool) in zip(self.layers, self.pools):
            qkv = layer["qkv"](self.xq[a.dim].fill(norm(x), code), self.dtype)
            at, ld = qkv.data_ptr(), qkv.stride(0)
            lq.kv_append(pool, batch, lq.KVRows(
                q=at, k=at + a.heads * hs * size, v=at + (a.heads + a.kv_heads) * hs * size, q_out=at, ld_q=ld, ld_k=ld,
                ld_v=ld, ld_q_out=ld, n_heads=a.heads, type=code, rope=self.rope.data_ptr(), rope_rows=a.max_context,
                rope_mode=lq.ROPE_PAIRS))
            out = torch.empty_like(x)
            lq.paged_attention(out.data_ptr(), at, a.heads, pool, batch, code, hs**-0.5, a.dim, ld)
            x = x + layer["o"](self.xq[a.dim].fill(out, code), self.dtype)
            gate, up = layer["up"](self.xq[a.dim].fill(norm(x), code), self.dtype).chunk(2, -1)
            x = x + layer["down"](self.xq[a.hidden].fill(torch.nn.functional.silu(gate) * up, code), self.dtype)
        return self.head(self.xq[a.dim].fill(norm(x[last]), code), (torch.float32, lq.F32))

    def plain(self, tokens):
        """fp32 logits at every position of one sequence, nothing quantized."""
        a, hs, n = self.a, self.hs, len(tokens)
        cos, sin = self.rope.view(-1, hs // 2, 2)[:n].unbind(-1)

        def turn(x):  # [n, heads, hs]
            u, v = x[..., ::2], x[..., 1::2]
            c, s = cos[:, None], sin[:, None]
            return torch.stack((u * c - v * s, u * s + v * c), -1).flatten(-2)

        x = self.embed[tokens].float()
        for layer in self.layers:
            q, k, v = (norm(x) @ layer["qkv"].weight.T).view(n, -1, hs).split((a.heads, a.kv_heads, a.kv_heads), 1)
            k, v = (t.repeat_interleave(a.heads // a.kv_heads, 1) for t in (turn(k), v))
            score = torch.einsum("qhd,khd->hqk", turn(q), k) * hs**-0.5
            score.masked_fill_(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), float("-inf"))
            x = x + torch.einsum("hqk,khd->qhd", score.softmax(-1), v).reshape(n, -1) @ layer["o"].weight.T
            gate, up = (norm(x) @ layer["up"].weight.T).chunk(2, -1)
            x = x + (torch.nn.functional.silu(gate) * up) @ layer["down"].weight.T
        return norm(x) @ self.head.weight.T


def arguments(argv=None):
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--dtype", choices=sorted(TYPES), default="bf16", help="of the activations")
    for name, value in dict(layers=4, dim=1024, hidden=2752, heads=16, kv_heads=4, vocab=2000, seqs=8, prompt=200, page=32,
                            steps=64).items():
        p.add_argument("--" + name.replace("_", "-"), type=int, default=value)
    a = p.parse_args(argv)
    a.max_context = a.prompt + a.steps + 1
    return a


def main(argv=None):
    a = arguments(argv)
    torch.backends.cuda.matmul.allow_tf32 = False  # of the plain model
    stream = torch.cuda.Stream()  # torch's work and the library's are ordered on it
    with torch.cuda.stream(stream):
        lq.set_stream(stream.cuda_stream)
        try:
            return generate(a, stream)
        finally:
            lq.sync()
            lq.set_stream(None)


def generate(a, stream):
    model = Model(a)
    # ragged prompts, the longest of a.prompt tokens
    lengths = [max(1, a.prompt * (s + 1) // a.seqs) for s in range(a.seqs)]
    gen = torch.Generator(device="cuda").manual_seed(1)
    prompts = [torch.randint(a.vocab, (n,), generator=gen, device="cuda") for n in lengths]
    starts = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).cuda()
    context = torch.tensor(lengths, dtype=torch.int32).cuda()
    logits = model.forward(torch.cat(prompts), model.batch(starts, context, max(lengths)), starts[1:].long() - 1)
    token = logits.argmax(-1)
    got_tokens, got_logits = [token.clone()], [logits.clone()]

    # one decode step: lengths and tokens stay on the device, so it can be replayed
    one = torch.arange(a.seqs + 1, dtype=torch.int32, device="cuda")
    batch, every = model.batch(one, context, 1), torch.arange(a.seqs, device="cuda")

    def step():
        context.add_(1)
        out = model.forward(token, batch, every)
        token.copy_(out.argmax(-1))
        return out

    got_logits.append(step().clone())  # not captured: the first step sets up what is allocated once
    got_tokens.append(token.clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step()
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    for _ in range(a.steps - 1):
        graph.replay()
        got_logits.append(out.clone())
        got_tokens.append(token.clone())
    end.record()
    lq.sync()  # reports errors that kernels found

    tokens, logits = torch.stack(got_tokens, 1), torch.stack(got_logits, 1)
    worst = 0.0
    for s, prompt in enumerate(prompts):
        plain = model.plain(torch.cat((prompt, tokens[s, :-1])))[len(prompt) - 1:]
        worst = max(worst, ((logits[s] - plain).norm() / plain.norm()).item())
    ms = begin.elapsed_time(end) / max(a.steps - 1, 1)
    print(f"{a.seqs} sequences, prompts of {min(lengths)} to {max(lengths)}, {a.steps} steps: {ms:.3f} ms per step, "
          f"logits within {worst:.3f} (relative, rms) of plain fp32")
    return {"tokens": tokens.cpu(), "context": context.cpu(), "lengths": lengths, "error": worst, "ms": ms}


if __name__ == "__main__":
    main()
