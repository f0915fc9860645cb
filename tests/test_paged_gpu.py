"""kv_append and paged_attention against 64 bits: lengths from nothing to
several pages, pages that end inside tiles, every page size, odd head layouts,
ragged rows, strides, rows that attend to nothing, stale and unused pages."""
import math

import numpy as np
import pytest

from gpu_util import lq
from paged_ref import (HALF_ULP, KINDS, Batch, attention, cache_struct, k_index, random_cache, torch_type, v_index)

pytestmark = pytest.mark.gpu


# ---- attention -----------------------------------------------------------------

def run_attention(torch, q, codes, scales, batch, dtype, hs, scale=None, ld_q=None, ld_out=None, fill=7.0, dev=None):
    kv_heads = codes.shape[1]
    heads = q.shape[1]
    tc, ts = torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda()
    c = cache_struct(tc, ts, kv_heads, hs, batch.page)
    b, keep = batch.device(torch) if dev is None else dev
    w = heads * hs
    ld_q, ld_out = ld_q or w, ld_out or w
    n = batch.n_rows
    qt = torch.zeros(max(n, 1), ld_q, device="cuda", dtype=torch_type(torch, dtype))
    qt[:n, :w] = torch.from_numpy(q.reshape(n, w)).cuda().to(qt.dtype)
    out = torch.full((max(n, 1), ld_out), fill, device="cuda", dtype=qt.dtype)
    lse = torch.full((max(n, 1), heads), fill, device="cuda")
    lq.paged_attention(out.data_ptr(), qt.data_ptr(), heads, c, b, KINDS[dtype], scale, ld_out, ld_q, lse.data_ptr())
    lq.sync()
    assert bool((out[:, w:] == fill).all())
    qv = qt[:n, :w].double().cpu().numpy().reshape(n, heads, hs)
    return qv, out[:n, :w].double().cpu().numpy().reshape(n, heads, hs), lse[:n].double().cpu().numpy()


def check_attention(torch, rng, rows, ctx, kv_heads, group, hs, page, dtype, q_scale=2.0, scale=None, **kw):
    batch = Batch(rng, rows, ctx, page)
    codes, scales = random_cache(rng, batch.n_pages, kv_heads, hs, page)
    used = np.zeros(batch.n_pages, bool)
    for s, c in enumerate(batch.ctx):
        used[batch.pages[s, : -(-max(c, 0) // page)].astype(np.int64)] = True
    scales[~used] = np.nan  # what no sequence holds must not matter
    q = rng.standard_normal((batch.n_rows, kv_heads * group, hs)) * q_scale
    scale = 1 / math.sqrt(hs) if scale is None else scale
    qv, out, lse = run_attention(torch, q, codes, scales, batch, dtype, hs, scale, **kw)
    want, wlse, tol, ltol = attention(qv, codes, scales, batch, dtype, scale)
    # stated per element: nothing is scaled to fit
    assert np.all(np.abs(out - want) <= tol), (np.abs(out - want) / np.maximum(tol, 1e-30)).max()
    empty = np.isinf(wlse)
    assert np.array_equal(empty, np.isneginf(lse))
    assert np.all(np.abs(lse[~empty] - wlse[~empty]) <= ltol[~empty])
    assert not out[empty].any()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_attend_lengths(cuda, dtype, page):
    """One new token, contexts around every boundary, in one call."""
    rng = np.random.default_rng(page)
    ctx = [1, 2, 3, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 257, 300, 511, 513, 700]
    check_attention(cuda, rng, [1] * len(ctx), ctx, 2, 1, 64, page, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hs", [16, 48, 64, 80, 96, 128, 176, 256])
@pytest.mark.parametrize("kv_heads,group", [(3, 1), (2, 4), (1, 7), (1, 8), (1, 20)])
def test_attend_heads(cuda, dtype, hs, kv_heads, group):
    rng = np.random.default_rng(hs * 10 + group)
    check_attention(cuda, rng, [1, 1, 1], [37, 150, 90], kv_heads, group, hs, 32, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv_heads,group,hs,page", [(2, 1, 128, 64), (1, 8, 128, 16), (2, 3, 48, 32), (1, 1, 256, 128),
                                                    (1, 5, 64, 16)])
def test_attend_ragged_rows(cuda, dtype, kv_heads, group, hs, page):
    """Prompts, decodes and an idle sequence together; rows behind a context."""
    rng = np.random.default_rng(hs + page)
    rows = [1, 33, 0, 70, 5, 128, 2, 17, 1]
    ctx = [140, 33, 50, 200, 6, 130, 2, 64, 1]
    check_attention(cuda, rng, rows, ctx, kv_heads, group, hs, page, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_long_split(cuda, dtype):
    """Few rows, a long axis: the work is split and joined."""
    rng = np.random.default_rng(5)
    check_attention(cuda, rng, [1, 2], [5000, 3001], 2, 2, 128, 64, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_long_prompt(cuda, dtype):
    rng = np.random.default_rng(6)
    check_attention(cuda, rng, [300, 1], [700, 900], 1, 2, 128, 64, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,ctx", [([4, 1], [2, 0]), ([3], [-1]), ([40, 1], [20, 5]), ([0, 0], [3, 0]), ([1, 90], [0, 0])])
def test_attend_empty_rows(cuda, dtype, rows, ctx):
    """Rows before position 0 and sequences without tokens: zeros, lse -inf."""
    rng = np.random.default_rng(sum(rows))
    check_attention(cuda, rng, rows, ctx, 2, 2, 64, 16, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attend_peaked_and_flat(cuda, dtype):
    """Scores that span hundreds (one key takes all), and all-zero queries."""
    rng = np.random.default_rng(8)
    check_attention(cuda, rng, [1, 40], [600, 90], 1, 2, 128, 64, dtype, q_scale=40.0)
    check_attention(cuda, rng, [1, 40], [600, 90], 1, 2, 128, 64, dtype, q_scale=0.0)


def test_attend_scale_sign_and_strides(cuda):
    rng = np.random.default_rng(9)
    check_attention(cuda, rng, [1, 20], [77, 90], 2, 2, 64, 32, "f32", scale=-0.2, ld_q=4 * 64 + 3, ld_out=4 * 64 + 1)
    check_attention(cuda, rng, [1, 20], [77, 90], 2, 2, 64, 32, "bf16", scale=0.0, ld_q=4 * 64 + 3, ld_out=4 * 64 + 1)


@pytest.mark.parametrize("rows,ctx", [(1, 700), (50, 120)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_non_finite(cuda, dtype, rows, ctx):
    """A query with a NaN or an infinity, or a page whose scale is NaN, gives NaN
    to the rows that see it and to no others; an infinite or NaN scale after a
    sequence's end gives nothing."""
    torch = cuda
    rng = np.random.default_rng(ctx)
    hs, page = 64, 16
    batch = Batch(rng, [rows, 3], [ctx, 60], page)
    codes, scales = random_cache(rng, batch.n_pages, 1, hs, page)
    q = rng.standard_normal((batch.n_rows, 2, hs))
    q[0, 0, 5], q[rows, 1, 7] = np.nan, np.inf
    _, out, lse = run_attention(torch, q, codes, scales, batch, dtype, hs)
    nan = np.zeros((batch.n_rows, 2), bool)
    nan[0, 0] = nan[rows, 1] = True
    assert np.array_equal(np.isnan(out).all(-1), nan) and np.array_equal(np.isnan(out).any(-1), nan)
    assert np.array_equal(np.isnan(lse), nan)
    q = rng.standard_normal((batch.n_rows, 2, hs))
    p = int(batch.pages[1, 3])  # positions 48 .. 59 of the second sequence
    scales[p] = np.nan
    _, out, lse = run_attention(torch, q, codes, scales, batch, dtype, hs)
    assert np.isnan(out[rows:]).all() and not np.isnan(out[:rows]).any()


@pytest.mark.parametrize("rows,ctx", [([1, 1], [40, 70]), ([30, 9], [40, 70])])
def test_attend_bad_device_arguments(cuda, rows, ctx):
    """A page number past the cache or negative, rows past max_rows, a context
    past max_context: an error status at the next sync, no access outside."""
    torch = cuda
    rng = np.random.default_rng(3)
    hs, page = 64, 16
    for what in range(5):
        batch = Batch(rng, rows, ctx, page)
        codes, scales = random_cache(rng, batch.n_pages, 1, hs, page)
        q = rng.standard_normal((batch.n_rows, 1, hs))
        kw = {}
        if what == 0:
            batch.pages[1, 2] = batch.n_pages
        elif what == 1:
            batch.pages[0, 0] = -1
        elif what == 2:
            kw["max_rows"] = max(rows) - 1
        elif what == 3:
            kw["max_context"] = max(ctx) - 1
        else:
            batch.max_pages = 3
            batch.pages = batch.pages[:, :3].copy()
        with pytest.raises(lq.LlamaQError) as e:
            run_attention(torch, q, codes, scales, batch, "f32", hs, dev=batch.device(torch, **kw))
        assert e.value.code == lq.EINVAL
        lq.sync()  # reported once


def test_attend_same_bits_every_time(cuda):
    """Splits are joined in one order: repeated calls, other streams and a graph
    give the same bits."""
    torch = cuda
    rng = np.random.default_rng(11)
    hs, page, heads = 128, 64, 8
    for rows, ctx in (([1, 1, 1], [3000, 40, 1500]), ([200, 1], [900, 30])):
        batch = Batch(rng, rows, ctx, page)
        codes, scales = random_cache(rng, batch.n_pages, 4, hs, page)
        tc, ts = torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda()
        c = cache_struct(tc, ts, 4, hs, page)
        b, keep = batch.device(torch)
        q = torch.randn(batch.n_rows, heads * hs, device="cuda")
        out, lse = torch.empty_like(q), torch.empty(batch.n_rows, heads, device="cuda")

        def step():
            lq.paged_attention(out.data_ptr(), q.data_ptr(), heads, c, b, lse_ptr=lse.data_ptr())

        step()
        lq.sync()
        want, wlse = out.clone(), lse.clone()
        st = torch.cuda.Stream()
        lq.set_stream(st.cuda_stream)
        try:
            step()
            lq.sync()
            lq.graph_begin()
            step()
            g = lq.graph_end()
            for _ in range(20):
                out.fill_(3.0)
                torch.cuda.synchronize()
                lq.graph_launch(g)
                lq.sync()
                assert torch.equal(out, want) and torch.equal(lse, wlse)
            lq.graph_destroy(g)
        finally:
            lq.set_stream(None)


# ---- append --------------------------------------------------------------------

def rotate(x, pos, rope, mode):
    """x [heads, hs] in 64 bits."""
    if mode is None:
        return x
    c, s = rope[pos, :, 0], rope[pos, :, 1]
    y = np.empty_like(x)
    if mode == "pairs":
        a, b = x[:, 0::2], x[:, 1::2]
        y[:, 0::2], y[:, 1::2] = a * c - b * s, a * s + b * c
    else:
        h = x.shape[1] // 2
        a, b = x[:, :h], x[:, h:]
        y[:, :h], y[:, h:] = a * c - b * s, a * s + b * c
    return y


class Appender:
    """A cache on the device and its reference: the values every code stands for."""

    def __init__(self, torch, rng, n_pages, kv_heads, hs, page, dtype, mode, group=2, positions=2048):
        self.torch, self.rng, self.dtype, self.mode = torch, rng, dtype, mode
        self.kv_heads, self.hs, self.page, self.heads = kv_heads, hs, page, kv_heads * group
        self.codes = torch.randint(-127, 128, (n_pages, kv_heads, 2, hs * page), dtype=torch.int8, device="cuda")
        self.scales = torch.full((n_pages, kv_heads, 2), float("nan"), device="cuda")  # fresh memory holds anything
        self.rope = lq.rope_table(positions, hs)
        self.rope_t = torch.from_numpy(self.rope).cuda()

    def call(self, batch, scale=1.0, pad=0, in_place=False, outs=True, queries=True, dev=None, rope_rows=None, edit=None):
        torch, hs = self.torch, self.hs
        kw, qw, n = self.kv_heads * hs, self.heads * hs, max(batch.n_rows, 1)
        dt = torch_type(torch, self.dtype)

        def rnd(w):
            return (torch.from_numpy(self.rng.standard_normal((n, w + pad)) * scale).cuda().to(dt))

        kv = (torch.from_numpy(self.rng.standard_normal((n, 2 * kw + pad)) * scale).cuda().to(dt))
        q = rnd(qw)
        if edit:
            edit(kv)
        q_in = q.clone()
        q_out = q if in_place else torch.full_like(q, 7.0)
        k_out, v_out = (torch.full((n, kw + pad), 7.0, device="cuda", dtype=dt) for _ in range(2))
        size = kv.element_size()
        r = lq.KVRows(q=q.data_ptr() if queries else None, k=kv.data_ptr(), v=kv.data_ptr() + kw * size,
                      q_out=q_out.data_ptr() if queries else None, k_out=k_out.data_ptr() if outs else None,
                      v_out=v_out.data_ptr() if outs else None, ld_q=qw + pad, ld_k=2 * kw + pad, ld_v=2 * kw + pad,
                      ld_q_out=qw + pad, ld_kv_out=kw + pad, n_heads=self.heads, type=KINDS[self.dtype],
                      rope=self.rope_t.data_ptr() if self.mode else None,
                      rope_rows=self.rope.shape[0] if rope_rows is None else rope_rows,
                      rope_mode=lq.ROPE_HALVES if self.mode == "halves" else lq.ROPE_PAIRS)
        c = cache_struct(self.codes, self.scales, self.kv_heads, hs, self.page)
        b, keep = batch.device(torch) if dev is None else dev
        before = self.codes.cpu().numpy().copy(), self.scales.cpu().numpy().copy()
        lq.kv_append(c, b, r)
        lq.sync()
        f = lambda t: t.double().cpu().numpy()  # noqa: E731
        self.after = self.codes.cpu().numpy(), self.scales.cpu().numpy()
        kvv = f(kv)
        return (f(q_in)[:, :qw].reshape(n, self.heads, hs), kvv[:, :kw].reshape(n, self.kv_heads, hs),
                kvv[:, kw:2 * kw].reshape(n, self.kv_heads, hs), f(q_out)[:, :qw].reshape(n, self.heads, hs),
                f(k_out)[:, :kw].reshape(n, self.kv_heads, hs), f(v_out)[:, :kw].reshape(n, self.kv_heads, hs), before)

    def check(self, batch, **kw):
        hs, P, H = self.hs, self.page, self.kv_heads
        q, k, v, q_out, k_out, v_out, (codes0, scales0) = self.call(batch, **kw)
        codes, scales = self.after
        u = 2.0**-24
        want_codes_known = np.zeros(codes.shape, bool)  # bytes this call may change
        new = {}  # (page, which) -> [(offset, row, rotated)]
        tokens = list(batch.places())
        rope = self.rope.astype(np.float64)
        for row, s, pos in tokens:
            x = rotate(k[row], pos, rope, self.mode)
            mag = 2 * np.abs(k[row]).max(1, keepdims=True)
            p = int(batch.pages[s, pos // P])
            new.setdefault((p, 0), []).append((pos % P, row, x, mag))
            new.setdefault((p, 1), []).append((pos % P, row, v[row], 0 * mag))
            if kw.get("queries", True):
                want = rotate(q[row], pos, rope, self.mode)
                tol = (3 * u * 2 * np.abs(q[row]).max(1, keepdims=True) if self.mode else 0) + np.abs(want) * HALF_ULP[self.dtype] * 1.01 + 1e-7
                assert np.all(np.abs(q_out[row] - want) <= tol)
        index = [k_index(hs, P), v_index(hs, P)]
        for (p, w), items in new.items():
            first = min(t for t, *_ in items)
            for h in range(H):
                peak = max(np.abs(x[h]).max() for _, _, x, _ in items)
                near = max(m[h].max() for *_, m in items) * 3 * u  # of a rotated value
                old = float(scales0[p, h, w]) if first > 0 else 0.0
                want = max(old, peak / 127) or float(np.float32(1e-8))
                got = float(scales[p, h, w])
                assert abs(got - want) <= want * 2 * u + near / 127
                kept = codes0[p, h, w][index[w][:first]].astype(np.float64)
                now = codes[p, h, w][index[w][:first]].astype(np.float64)
                if got == old:
                    assert np.array_equal(kept, now)
                else:
                    assert np.all(np.abs(now - kept * (old / got)) <= 0.5 + 127 * 4 * u)
                want_codes_known[p, h, w][index[w][:first]] = True
                for t, row, x, m in items:
                    c = codes[p, h, w][index[w][t]].astype(np.float64)
                    assert np.all(np.abs(c - x[h] / got) <= 0.5 + 127 * 2 * u + near / got)
                    assert np.abs(c).max() <= 127
                    want_codes_known[p, h, w][index[w][t]] = True
                    if kw.get("outs", True):
                        o = (k_out, v_out)[w][row, h]
                        assert np.all(np.abs(o - c * got) <= np.abs(c * got) * (u + HALF_ULP[self.dtype]) * 1.01)
        # nothing else moved
        assert np.array_equal(codes[~want_codes_known], codes0[~want_codes_known])
        touched = np.zeros(scales.shape, bool)
        for p, w in new:
            touched[p, :, w] = True
        assert np.array_equal(scales[~touched], scales0[~touched], equal_nan=True)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("mode", ["pairs", "halves", None])
@pytest.mark.parametrize("page,hs,kv_heads", [(16, 128, 2), (64, 48, 3), (128, 64, 1), (32, 256, 1)])
def test_append_in_steps(cuda, dtype, mode, page, hs, kv_heads):
    """Prompts, then single tokens (growing and not), then a chunk: every call
    against the codes and scales it found."""
    rng = np.random.default_rng(page + hs)
    rows = [[5, 0, 40, page], [1, 1, 1, 1], [1, 0, 1, 1], [page + 3, 2, 1, 2 * page]]
    ctx = np.zeros(4, int)
    full = [sum(r[s] for r in rows) for s in range(4)]
    layout = Batch(rng, [0] * 4, full, page)
    a = Appender(cuda, rng, layout.n_pages, kv_heads, hs, page, dtype, mode)
    for i, r in enumerate(rows):
        ctx = ctx + r
        b = Batch(rng, r, ctx, page, max_pages=layout.max_pages)
        b.pages, b.n_pages = layout.pages, layout.n_pages
        a.check(b, scale=[1.0, 3.0, 0.1, 2.0][i], pad=[0, 3, 8, 1][i])


def test_append_single_tokens_through_pages(cuda):
    rng = np.random.default_rng(2)
    layout = Batch(rng, [0, 0], [40, 37], 16)
    a = Appender(cuda, rng, layout.n_pages, 2, 64, 16, "f32", "pairs")
    for t in range(1, 37):
        b = Batch(rng, [1, 1], [t + 3 if t > 1 else 1, t], 16, max_pages=layout.max_pages)
        if t == 1:
            b = Batch(rng, [4, 1], [4, 1], 16, max_pages=layout.max_pages)
        b.pages = layout.pages
        a.check(b, scale=1.0 + 0.05 * t)


@pytest.mark.parametrize("mode", ["pairs", "halves"])
def test_append_in_place_and_without(cuda, mode):
    rng = np.random.default_rng(4)
    b = Batch(rng, [3, 30], [9, 30], 32)
    a = Appender(cuda, rng, b.n_pages, 2, 96, 32, "bf16", mode)
    a.scales.fill_(0.001)
    a.check(b, in_place=True)
    a.check(b, queries=False)
    a.check(b, outs=False)


def test_append_empty(cuda):
    """No rows, rows before position 0, a sequence without tokens."""
    rng = np.random.default_rng(5)
    for rows, ctx in (([0, 0], [3, 0]), ([4, 1], [2, 0]), ([2], [-5])):
        b = Batch(rng, rows, ctx, 16)
        a = Appender(cuda, rng, b.n_pages, 1, 64, 16, "f32", "pairs")
        a.scales.fill_(0.01)
        a.check(b)


def test_append_zeros_and_non_finite(cuda):
    torch = cuda
    rng = np.random.default_rng(6)
    b = Batch(rng, [20, 2], [20, 2], 16)
    a = Appender(torch, rng, b.n_pages, 1, 64, 16, "f32", None, group=1)
    a.check(b, scale=0.0)
    assert np.all(a.after[1][b.pages[0, :2].astype(int)] == np.float32(1e-8))

    def edit(kv):
        kv[3, 7] = float("nan")       # key of token 3 of sequence 0: page 0
        kv[18, 64 + 5] = float("inf")  # value of token 18: page 1

    a.call(b, edit=edit)
    codes, scales = a.after
    p0, p1 = b.pages[0, :2].astype(int)
    assert np.isnan(scales[p0, 0, 0]) and np.isfinite(scales[p0, 0, 1])
    assert np.isnan(scales[p1, 0, 1]) and np.isfinite(scales[p1, 0, 0])
    assert not codes[p0, 0, 0].any()
    # it stays until the page is begun again
    b2 = Batch(rng, [1, 0], [21, 2], 16, max_pages=b.max_pages)
    b2.pages = b.pages
    a.call(b2)
    assert np.isnan(a.after[1][p1, 0, 1])
    a.check(b)
    assert np.isfinite(a.after[1]).any()


def test_append_bad_device_arguments(cuda):
    torch = cuda
    rng = np.random.default_rng(7)
    for what in range(6):
        b = Batch(rng, [3, 20], [9, 40], 16)
        kw, call = {}, {}
        if what == 0:
            b.pages[1, 2] = b.n_pages
        elif what == 1:
            b.pages[0, 0] = -7
        elif what == 2:
            kw["max_rows"] = 19
        elif what == 3:
            kw["max_context"] = 39
        elif what == 4:
            b.max_pages = 2
            b.pages = b.pages[:, :2].copy()
        else:
            call["rope_rows"] = 39
        a = Appender(torch, rng, b.n_pages, 1, 64, 16, "f32", "pairs")
        with pytest.raises(lq.LlamaQError) as e:
            a.call(b, dev=b.device(torch, **kw), **call)
        assert e.value.code == lq.EINVAL
        lq.sync()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_then_attend(cuda, dtype):
    """The pair as a decode step uses it: what was appended is what is read."""
    torch = cuda
    rng = np.random.default_rng(8)
    hs, page = 64, 32
    full = [50, 33]
    layout = Batch(rng, [0, 0], full, page)
    a = Appender(torch, rng, layout.n_pages, 2, hs, page, dtype, "pairs", group=2)
    ctx = np.zeros(2, int)
    for rows in ([30, 20], [1, 1], [17, 10], [1, 1], [1, 1]):
        ctx = ctx + rows
        b = Batch(rng, rows, ctx, page, max_pages=layout.max_pages)
        b.pages = layout.pages
        _, _, _, q_rot, _, _, _ = a.call(b)
        codes, scales = a.after
        qv, out, lse = run_attention(torch, q_rot, codes, scales, b, dtype, hs)
        want, wlse, tol, ltol = attention(qv, codes, scales, b, dtype, 1 / math.sqrt(hs))
        assert np.all(np.abs(out - want) <= tol) and np.all(np.abs(lse - wlse) <= ltol)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("seqs,kv_heads,group", [(1, 1, 1), (33, 1, 1), (70, 2, 1), (70, 1, 6), (300, 1, 1), (300, 1, 2), (500, 1, 1)])
def test_attend_bound_far_above_the_contexts(cuda, dtype, seqs, kv_heads, group):
    """Many sequences, idle and long ones among them, and a max_context that none
    comes near: how they are split follows from the contexts themselves."""
    rng = np.random.default_rng(seqs)
    ctx = [int(x) for x in rng.integers(0, 400, seqs)]
    ctx[seqs // 2] = 3000
    rows = [int(x) for x in rng.integers(0, 2, seqs)]
    rows[seqs // 2] = 1
    batch = Batch(rng, rows, ctx, 64)
    codes, scales = random_cache(rng, batch.n_pages, kv_heads, 64, 64)
    q = rng.standard_normal((batch.n_rows, kv_heads * group, 64)) * 2
    for bound in (3000, 100000):
        qv, out, lse = run_attention(cuda, q, codes, scales, batch, dtype, 64, 0.125,
                                     dev=batch.device(cuda, max_context=bound))
        want, wlse, tol, ltol = attention(qv, codes, scales, batch, dtype, 0.125)
        assert np.all(np.abs(out - want) <= tol), (np.abs(out - want) / np.maximum(tol, 1e-30)).max()
        empty = np.isinf(wlse)
        assert np.array_equal(empty, np.isneginf(lse)) and not out[empty].any()
        assert np.all(np.abs(lse[~empty] - wlse[~empty]) <= ltol[~empty])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("group,hs,page", [(2, 128, 64), (1, 64, 16), (3, 128, 16)])
def test_prompts_same_bits_many_times(cuda, dtype, group, hs, page):
    """Prompts that end in the middle of tiles, over and over with the GPU busy:
    every launch gives the first one's bits, which are right."""
    rng = np.random.default_rng(group)
    rows, ctx = [300, 1, 129, 64], [700, 900, 129, 65]
    batch = Batch(rng, rows, ctx, page)
    codes, scales = random_cache(rng, batch.n_pages, 4, hs, page)
    heads = 4 * group
    q = rng.standard_normal((batch.n_rows, heads, hs)) * 2
    tc, ts = cuda.from_numpy(codes).cuda(), cuda.from_numpy(scales).cuda()
    c = cache_struct(tc, ts, 4, hs, page)
    b, keep = batch.device(cuda)
    qt = cuda.from_numpy(q.reshape(batch.n_rows, heads * hs)).cuda().to(torch_type(cuda, dtype))
    outs = [cuda.empty_like(qt) for _ in range(9)]
    wrong = cuda.zeros(1, device="cuda", dtype=cuda.int64)
    for n in range(40):
        for out in outs[n > 0:]:
            lq.paged_attention(out.data_ptr(), qt.data_ptr(), heads, c, b, KINDS[dtype], hs**-0.5)
        lq.sync()
        for out in outs[1:]:
            wrong += (out != outs[0]).sum()
        cuda.cuda.synchronize()
    assert int(wrong) == 0
    qv = qt.double().cpu().numpy().reshape(-1, heads, hs)
    want, _, tol, _ = attention(qv, codes, scales, batch, dtype, hs**-0.5)
    got = outs[0].double().cpu().numpy().reshape(want.shape)
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hs", [16, 32, 48, 80, 96, 112, 144, 240])
def test_attend_prompt_head_sizes(cuda, dtype, hs):
    """Prompts at head sizes between the usual ones."""
    check_attention(cuda, np.random.default_rng(hs), [150, 40], [333, 41], 2, 2, hs, 32, dtype)
