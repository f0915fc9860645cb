"""The paged int8 cache in numpy and 64 bits: page layout, random caches and
batches, append, attention with its error bounds, and their device copies."""
from __future__ import annotations

import numpy as np

from gpu_util import lq

KINDS = {"f32": lq.F32, "f16": lq.F16, "bf16": lq.BF16}
# half a unit in the last place, relative
HALF_ULP = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}


def torch_type(torch, dtype):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]


def k_index(hs, P):
    t, d = np.arange(P)[:, None], np.arange(hs)[None]
    return (d // 16 * P + t) * 16 + d % 16


def v_index(hs, P):
    t, d = np.arange(P)[:, None], np.arange(hs)[None]
    return (t // 16 * hs + d) * 16 + t % 16


class Batch:
    """rows[s] new tokens of a sequence whose context with them is ctx[s]."""

    def __init__(self, rng, rows, ctx, page, spare=2, max_pages=None):
        self.rows, self.ctx, self.page = list(rows), list(ctx), page
        need = [-(-max(c, 0) // page) for c in ctx]
        self.n_pages = sum(need) + spare
        self.max_pages = max(max(need), 1) if max_pages is None else max_pages
        order = rng.permutation(self.n_pages)
        # slots past a sequence's pages hold page numbers that must not be used
        self.pages = np.full((len(rows), self.max_pages), 2**31 - 1, np.int64)
        at = 0
        for s, n in enumerate(need):
            self.pages[s, :n] = order[at:at + n]
            at += n
        self.row_start = np.concatenate([[0], np.cumsum(rows)])
        self.n_rows = int(self.row_start[-1])

    def places(self):
        """(row, sequence, position) of every row that is a token."""
        for s, (n, c) in enumerate(zip(self.rows, self.ctx)):
            for i in range(n):
                if c - n + i >= 0:
                    yield int(self.row_start[s]) + i, s, c - n + i

    def device(self, torch, max_rows=None, max_context=None):
        keep = [torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()
                for a in (self.row_start, self.ctx, self.pages)]
        b = lq.KVBatch(row_start=keep[0].data_ptr(), context=keep[1].data_ptr(), pages=keep[2].data_ptr(),
                       n_seqs=len(self.rows), n_rows=self.n_rows, max_pages=self.max_pages,
                       max_rows=max(self.rows) if max_rows is None else max_rows,
                       max_context=max(max(self.ctx), 0) if max_context is None else max_context)
        return b, keep


def random_cache(rng, n_pages, kv_heads, hs, page):
    codes = np.clip(np.rint(rng.standard_normal((n_pages, kv_heads, 2, hs * page)) * 42), -127, 127).astype(np.int8)
    scales = ((rng.random((n_pages, kv_heads, 2)) + 0.5) / 42).astype(np.float32)
    return codes, scales


def cache_struct(codes_t, scales_t, kv_heads, hs, page):
    return lq.PagedKV(codes=codes_t.data_ptr(), scales=scales_t.data_ptr(), n_pages=codes_t.shape[0],
                      page_size=page, n_kv_heads=kv_heads, head_size=hs)


def sequence_kv(codes, scales, batch, s, h, hs):
    """K and V codes and scales of a sequence's context: [ctx, hs] and [ctx]."""
    P, c = batch.page, max(batch.ctx[s], 0)
    p = batch.pages[s, : -(-c // P)].astype(np.int64)
    k = codes[p, h, 0][:, k_index(hs, P)].reshape(-1, hs)[:c].astype(np.float64)
    v = codes[p, h, 1][:, v_index(hs, P)].reshape(-1, hs)[:c].astype(np.float64)
    sk, sv = (np.repeat(scales[p, h, i].astype(np.float64), P)[:c] for i in (0, 1))
    return k, v, sk, sv


def attention(q, codes, scales, batch, dtype, scale):
    """out, lse and the bound of out's and lse's errors, all in 64 bits.

    q [rows, heads, hs] holds values of the type.  With x* the kernels' value
    of x: q* is a fixed-point or split form within eq * max|q| of q, so a
    score is off by ds <= |scale| * sk * eq * max|q| * sum|code| plus four fp32
    roundings of its own sum of magnitudes; a weight p by a factor
    1 + ds + 2^-20 (exponential, sums and rescaling) and by its own form's
    step, 2^-22 of the row's largest p * sv for fp32 and 2^-11 of itself plus
    2^-15 of that for the 16-bit types; out by both, twice (numerator and
    denominator), and by its last rounding.
    """
    eq = 2.0**-22 if dtype == "f32" else 2.0**-14
    n, heads, hs = q.shape
    kv_heads = codes.shape[1]
    g = heads // kv_heads
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    lse, ltol = np.full((n, heads), -np.inf), np.zeros((n, heads))
    by_seq = {}
    for row, s, pos in batch.places():
        by_seq.setdefault(s, []).append((row, pos))
    for s, places in by_seq.items():
        for h in range(kv_heads):
            k, v, sk, sv = sequence_kv(codes, scales, batch, s, h, hs)
            kv, vv = k * sk[:, None], v * sv[:, None]
            size = np.abs(k).sum(1) * sk * abs(scale)
            for row, pos in places:
                m = pos + 1
                for e in range(h * g, (h + 1) * g):
                    x = q[row, e]
                    sc = kv[:m] @ x * scale
                    ds = (size[:m] * np.abs(x).max() * eq
                          + 4 * 2.0**-24 * abs(scale) * (np.abs(kv[:m]) @ np.abs(x))).max()
                    top = sc.max()
                    p = np.exp(sc - top)
                    l = p.sum()
                    out[row, e] = p @ vv[:m] / l
                    lse[row, e] = top + np.log(l)
                    rel = 2 * (ds + 2.0**-20)
                    mag = p @ np.abs(vv[:m]) / l
                    fixed = (p * sv[:m]).max() * np.abs(v[:m]).sum(0) / l
                    step = 2.0**-22 * fixed if dtype == "f32" else 2.0**-11 * mag + 2.0**-15 * fixed
                    tol[row, e] = (rel * (mag + np.abs(out[row, e])) + 2 * step
                                   + 2 * HALF_ULP[dtype] * np.abs(out[row, e]) + 1e-7 * HALF_ULP[dtype])
                    ltol[row, e] = rel + 2.0**-21 * (abs(top) + abs(np.log(l)) + 1)
    return out, lse, tol, ltol
