"""A layer's calls one right after another, each launched while the one before still
runs: the same bits as with a wait after every call."""
import numpy as np
import pytest

from gpu_util import lq
from paged_ref import KINDS, Batch, cache_struct, torch_type
from test_rows_gpu import empty_row8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("seqs,prompt,kv_heads,group,hs,page", [(1, 3, 16, 1, 128, 64), (5, 60, 4, 4, 64, 16), (33, 2, 32, 1, 64, 32)])
def test_steps(cuda, dtype, seqs, prompt, kv_heads, group, hs, page):
    torch, kind, tt = cuda, KINDS[dtype], torch_type(cuda, dtype)
    rng = np.random.default_rng(seqs)
    heads, steps = kv_heads * group, 24
    width, dim = (heads + 2 * kv_heads) * hs, heads * hs
    layout = Batch(rng, [prompt] * seqs, [prompt + steps] * seqs, page)
    pages = torch.from_numpy(layout.pages.astype(np.int32)).cuda()
    rope = torch.from_numpy(lq.rope_table(prompt + steps, hs)).cuda()
    w, wq, ws = empty_row8(torch, width, dim)
    wv = torch.from_numpy(rng.standard_normal((width, dim)).astype(np.float32)).cuda() * dim**-0.5
    lq.quantize_rows(w, wv.data_ptr(), dim)
    first = torch.from_numpy(rng.standard_normal((seqs * prompt, dim)).astype(np.float32)).cuda().to(tt)
    x, xq, xs = empty_row8(torch, seqs * prompt, dim)
    qkv = torch.empty(seqs * prompt, width, dtype=tt, device="cuda")
    out = torch.empty(seqs * prompt, dim, dtype=tt, device="cuda")

    def run(wait):
        codes = torch.zeros(layout.n_pages, kv_heads, 2, hs * page, dtype=torch.int8, device="cuda")
        scales = torch.zeros(layout.n_pages, kv_heads, 2, device="cuda")
        cache = cache_struct(codes, scales, kv_heads, hs, page)
        context = torch.full((seqs,), prompt, dtype=torch.int32, device="cuda")
        rows, h, got = prompt, first, []
        for step in range(steps):
            n = seqs * rows
            start = torch.arange(0, n + 1, rows, dtype=torch.int32, device="cuda")
            batch = lq.KVBatch(row_start=start.data_ptr(), context=context.data_ptr(), pages=pages.data_ptr(), n_seqs=seqs,
                               n_rows=n, max_pages=layout.max_pages, max_rows=rows, max_context=prompt + steps)
            x.rows = n
            at, size = qkv.data_ptr(), qkv.element_size()
            lq.quantize_rows(x, h.data_ptr(), dim, kind)
            wait()
            lq.matmul_rows(at, x, w, dim, width, kind)
            wait()
            lq.kv_append(cache, batch, lq.KVRows(
                q=at, k=at + heads * hs * size, v=at + (heads + kv_heads) * hs * size, q_out=at, ld_q=width, ld_k=width,
                ld_v=width, ld_q_out=width, n_heads=heads, type=kind, rope=rope.data_ptr(), rope_rows=prompt + steps,
                rope_mode=lq.ROPE_PAIRS))
            wait()
            lq.paged_attention(out.data_ptr(), at, heads, cache, batch, kind, ld_q=width)
            wait()
            got.append(out[:n].clone())
            h = out[:n].view(seqs, rows, dim)[:, -1] * (1.0 + 0.1 * step)  # the scales of pages grow
            rows = 1
            context += 1
        torch.cuda.synchronize()
        return torch.cat(got), codes, scales

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        lq.set_stream(stream.cuda_stream)
        try:
            want = run(lq.sync)
            for _ in range(8):
                assert all(torch.equal(a, b) for a, b in zip(run(lambda: None), want))
        finally:
            lq.sync()
            lq.set_stream(None)
