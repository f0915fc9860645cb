"""paged_attention where weights, page scales and queries span many orders of
magnitude: an attention sink over thousands of small weights, pages whose value
scales lie up to 2^30 apart, seen and unseen ones."""
import math

import numpy as np
import pytest

from paged_ref import HALF_ULP, Batch, attention, k_index, random_cache, sequence_kv, v_index
from test_paged_gpu import run_attention

pytestmark = pytest.mark.gpu


def sink_cache(rng, batch, kv_heads, hs, page, where):
    """Keys that one direction of q tells apart: dim 0 of token `where` of every
    sequence holds 127, of the others -8 to 8; the rest is small.  The sink's
    values are zero, the others' all of one sign."""
    codes, scales = random_cache(rng, batch.n_pages, kv_heads, hs, page)
    k = rng.integers(-3, 4, (batch.n_pages, kv_heads, page, hs)).astype(np.int8)
    k[..., 0] = rng.integers(-8, 9, k.shape[:-1])
    v = rng.integers(20, 101, k.shape).astype(np.int8)
    for s in range(len(batch.rows)):
        p = int(batch.pages[s, where // page])
        k[p, :, where % page, 0] = 127
        v[p, :, where % page] = 0
    codes[:, :, 0][:, :, k_index(hs, page)] = k
    codes[:, :, 1][:, :, v_index(hs, page)] = v
    scales[:] = np.float32(1 / 127)
    return codes, scales


def bound(q, codes, scales, batch, dtype, scale, step, floor, every):
    """out in 64 bits, and what its error may be: scores as in paged_ref.attention;
    every weight off by `step` of itself, and `every` weight, or those of 32
    neighbouring tokens (the others are measured against something smaller), by
    `floor` of the row's largest p * s_V; the last rounding."""
    eq = 2.0**-22 if dtype == "f32" else 2.0**-14
    n, heads, hs = q.shape
    g = heads // codes.shape[1]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for s in range(len(batch.rows)):
        for h in range(codes.shape[1]):
            k, v, sk, sv = sequence_kv(codes, scales, batch, s, h, hs)
            kv, vv = k * sk[:, None], v * sv[:, None]
            size = np.abs(k).sum(1) * sk * abs(scale)
            for i in range(batch.rows[s]):
                row, m = batch.row_start[s] + i, batch.ctx[s] - batch.rows[s] + i + 1
                for e in range(h * g, h * g + g):
                    x = q[row, e]
                    sc = kv[:m] @ x * scale
                    ds = (size[:m] * np.abs(x).max() * eq
                          + 4 * 2.0**-24 * abs(scale) * (np.abs(kv[:m]) @ np.abs(x))).max()
                    p = np.exp(sc - sc.max())
                    p /= p.sum()
                    out[row, e] = p @ vv[:m]
                    mag = p @ np.abs(vv[:m])
                    count = np.abs(v[:m]).sum(0) if every else 32 * 127
                    tol[row, e] = ((2 * (ds + 2.0**-20) + step) * 2 * mag + count * floor * (p * sv[:m]).max()
                                   + 2 * HALF_ULP[dtype] * np.abs(out[row, e]) + 1e-30)
    return out, tol


# the type's range: from here on values round to infinity; half the distance of its smallest values
LARGEST = {"f32": 2.0**128, "f16": 65520.0, "bf16": 2.0**128}
SMALL = {"f32": 2.0**-150, "f16": 2.0**-25, "bf16": 2.0**-134}


def agree(out, want, tol, dtype):
    """Within tol, where the type's range allows: past it a value rounds to
    infinity, below its normal numbers to a multiple of the smallest."""
    tol = tol + SMALL[dtype]
    over = np.abs(want) >= LARGEST[dtype]
    assert np.all(np.isinf(out[over]) | (np.abs(want[over]) - tol[over] < LARGEST[dtype]))
    assert np.all(np.sign(out[over]) == np.sign(want[over]))
    err = np.abs(out[~over] - want[~over])
    near = np.isinf(out[~over]) & (np.abs(want[~over]) + tol[~over] >= LARGEST[dtype])
    assert np.all((err <= tol[~over]) | near), np.nanmax(err / tol[~over])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("name,seqs,rows,ctx,kv_heads,group", [
    ("split, one row", 1, 1, 4000, 2, 1), ("split, eight rows", 1, 2, 4000, 1, 4),
    ("whole contexts, one row", 60, 1, 1100, 8, 1), ("whole contexts, eight rows", 30, 1, 1100, 16, 2),
])
def test_attend_sink(cuda, dtype, page, name, seqs, rows, ctx, kv_heads, group):
    """One key takes most of the sum and gives nothing to the output, which is what
    thousands of others 11 to 13 nats lower leave."""
    check_sink(cuda, dtype, page, seqs, rows, ctx, kv_heads, group)


def check_sink(cuda, dtype, page, seqs, rows, ctx, kv_heads, group, hs=64, where=5):
    rng = np.random.default_rng(ctx + page)
    batch = Batch(rng, [rows] * seqs, [ctx] * seqs, page)
    codes, scales = sink_cache(rng, batch, kv_heads, hs, page, where)
    q = rng.standard_normal((batch.n_rows, kv_heads * group, hs)) * 0.1
    q[..., 0] = 12 * math.sqrt(hs)  # the sink's key is 1 there, the others' about 0
    qv, out, _ = run_attention(cuda, q, codes, scales, batch, dtype, hs, 1 / math.sqrt(hs))
    # a weight's own form: 24 or more fixed bits in blocks of 32, or one or two f16,
    # whose smallest step is 2^-24 where the largest weight is 2^6 (fp32: 2^11) or more
    many = rows * group > 32
    step = 2.0**-21 if dtype == "f32" else 2.0**-11
    floor = (2.0**-36, 2.0**-31)[dtype != "f32"] if many else (2.0**-31, 2.0**-24)[dtype != "f32"]
    want, tol = bound(qv, codes, scales, batch, dtype, 1 / math.sqrt(hs), step, floor, many)
    agree(out, want, tol, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("group", [1, 4])
@pytest.mark.parametrize("order", ["falling", "rising", "mixed"])
def test_attend_page_scales_apart(cuda, dtype, group, order):
    """Two pages in one step of 32 tokens, their value scales 2^0 to 2^30 apart;
    contexts that end in the first, the second or later: what a row does not see
    has no say, and a page it hardly attends to takes nothing from the others."""
    rng = np.random.default_rng(group)
    hs, page, kv_heads = 64, 16, 2
    ctx = [1, 5, 16, 17, 20, 32, 33, 50, 64, 80, 100]
    batch = Batch(rng, [1] * len(ctx), ctx, page)
    codes, scales = random_cache(rng, batch.n_pages, kv_heads, hs, page)
    spread(rng, batch, scales, order)
    q = rng.standard_normal((batch.n_rows, kv_heads * group, hs)) * 2
    # the slots past a context's last page: a page of the largest scale, unseen
    qv, out, lse = run_attention(cuda, q, codes, scales, batch, dtype, hs, 0.125)
    want, wlse, tol, ltol = attention(qv, codes, scales, batch, dtype, 0.125)
    agree(out, want, tol, dtype)
    assert np.all(np.abs(lse - wlse) <= ltol)


def spread(rng, batch, scales, order):
    for s, c in enumerate(batch.ctx):
        n = -(-c // batch.page)
        k = {"falling": -np.arange(n) * 30 // max(n - 1, 1), "rising": np.arange(n) * 30 // max(n - 1, 1),
             "mixed": rng.permutation(n) * 30 // max(n - 1, 1)}[order]
        p = batch.pages[s, :n].astype(np.int64)
        scales[p, :, 1] = (2.0 ** (k - 15))[:, None] * (1 + rng.random((n, scales.shape[1])))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attend_unseen_half_of_a_step(cuda, dtype):
    """Rows of one tile that see one or both of two pages: the second's scale,
    2^30 times the first's, is nothing to rows before it."""
    rng = np.random.default_rng(3)
    hs, page = 64, 16
    batch = Batch(rng, [8], [20], page)  # positions 12 .. 19
    codes, scales = random_cache(rng, batch.n_pages, 1, hs, page)
    scales[int(batch.pages[0, 1]), :, 1] = 2.0**25
    q = rng.standard_normal((8, 1, hs)) * 2
    qv, out, _ = run_attention(cuda, q, codes, scales, batch, dtype, hs, 0.125)
    want, _, tol, _ = attention(qv, codes, scales, batch, dtype, 0.125)
    agree(out, want, tol, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,ctx,group,hs,page,where", [
    (40, 4000, 1, 64, 16, 5), (40, 3000, 4, 64, 64, 2900), (300, 700, 1, 64, 32, 0), (40, 1500, 1, 128, 64, 700),
    (40, 1500, 1, 192, 16, 700)])
def test_attend_sink_prompt(cuda, dtype, rows, ctx, group, hs, page, where):
    """The same from a prompt's rows, the sink at the start, within and near the end."""
    check_sink(cuda, dtype, page, 1, rows, ctx, 1, group, hs, where)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("order", ["falling", "rising", "mixed"])
@pytest.mark.parametrize("group,hs,page", [(1, 64, 16), (2, 128, 64), (1, 192, 32)])
def test_attend_page_scales_apart_prompt(cuda, dtype, order, group, hs, page):
    """Value scales 2^0 to 2^30 apart before, behind and at the rows' positions."""
    rng = np.random.default_rng(hs)
    batch = Batch(rng, [100, 40, 150], [100, 333, 260], page)
    codes, scales = random_cache(rng, batch.n_pages, 2, hs, page)
    spread(rng, batch, scales, order)
    q = rng.standard_normal((batch.n_rows, 2 * group, hs)) * 2
    qv, out, lse = run_attention(cuda, q, codes, scales, batch, dtype, hs, hs**-0.5)
    want, wlse, tol, ltol = attention(qv, codes, scales, batch, dtype, hs**-0.5)
    agree(out, want, tol, dtype)
    assert np.all(np.abs(lse - wlse) <= ltol)


@pytest.mark.parametrize("rows,ctx", [([60], [200]), ([9, 200], [9, 200])])
def test_attend_prompt_blind_to_later_pages(cuda, rows, ctx):
    """Rows before a page have the same bits whatever that page's scales are."""
    rng = np.random.default_rng(7)
    hs, page = 64, 16
    batch = Batch(rng, rows, ctx, page)
    codes, scales = random_cache(rng, batch.n_pages, 1, hs, page)
    q = rng.standard_normal((batch.n_rows, 1, hs)) * 2
    last = int(batch.pages[-1, (ctx[-1] - 1) // page])  # positions 192 .. 199
    for dtype in ("f32", "f16", "bf16"):
        outs = []
        for factor in (1.0, 2.0**20, np.nan):
            other = scales.copy()
            other[last] *= np.float32(factor)
            outs.append(run_attention(cuda, q, codes, other, batch, dtype, hs, 0.125)[1:])
        for out, lse in outs[1:]:
            assert np.array_equal(out[:-8], outs[0][0][:-8]) and np.array_equal(lse[:-8], outs[0][1][:-8])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,ctx,hs", [([1], [300], 64), ([50], [120], 128), ([40, 3], [300, 50], 256)])
@pytest.mark.parametrize("size", [1e-20, 1e20, 3e37])
def test_attend_queries_of_any_size(cuda, dtype, rows, ctx, hs, size):
    """Queries near the ends of fp32's range whose scores, by the scale, are ordinary."""
    rng = np.random.default_rng(hs)
    batch = Batch(rng, rows, ctx, 32)
    codes, scales = random_cache(rng, batch.n_pages, 1, hs, 32)
    q = np.clip(rng.standard_normal((batch.n_rows, 1, hs)), -5, 5) * size
    scale = 2 / size / math.sqrt(hs)
    qv, out, lse = run_attention(cuda, q, codes, scales, batch, dtype, hs, scale)
    want, wlse, tol, ltol = attention(qv, codes, scales, batch, dtype, scale)
    assert np.all(np.abs(out - want) <= tol), (np.abs(out - want) / tol).max()
    assert np.all(np.abs(lse - wlse) <= ltol)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hs,group,page", [(256, 1, 64), (144, 2, 16)])
def test_attend_long_prompt_wide_heads(cuda, dtype, hs, group, page):
    """Heads above 128 dims, prompts of several row tiles behind a context and not."""
    rng = np.random.default_rng(hs)
    batch = Batch(rng, [300, 170], [500, 170], page)
    codes, scales = random_cache(rng, batch.n_pages, 1, hs, page)
    q = rng.standard_normal((batch.n_rows, group, hs)) * 2
    qv, out, lse = run_attention(cuda, q, codes, scales, batch, dtype, hs, hs**-0.5)
    want, wlse, tol, ltol = attention(qv, codes, scales, batch, dtype, hs**-0.5)
    assert np.all(np.abs(out - want) <= tol), (np.abs(out - want) / tol).max()
    assert np.all(np.abs(lse - wlse) <= ltol)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,ctx,group,page", [([1], [3000], 1, 64), ([1, 2], [90, 33], 4, 16), ([60], [200], 2, 32)])
@pytest.mark.parametrize("size", [2.0**-105, 2.0**115])
def test_attend_values_of_any_size(cuda, dtype, rows, ctx, group, page, size):
    """Values near the ends of fp32's range keep their bits: a power of two in the
    scales is one in the outputs."""
    rng = np.random.default_rng(page)
    hs = 64
    batch = Batch(rng, rows, ctx, page)
    codes, scales = random_cache(rng, batch.n_pages, 2, hs, page)
    q = rng.standard_normal((batch.n_rows, 2 * group, hs)) * 2
    far = scales.copy()
    far[:, :, 1] *= np.float32(size)
    qv, out, lse = run_attention(cuda, q, codes, far, batch, dtype, hs, 0.125)
    want, wlse, tol, ltol = attention(qv, codes, scales, batch, dtype, 0.125)
    assert np.all(np.abs(out / size - want) <= tol), (np.abs(out / size - want) / tol).max()
    assert np.all(np.abs(lse - wlse) <= ltol)
