"""What quantize_rows, matmul_rows, kv_append and paged_attention refuse, before
any device is touched (CPU only)."""
import numpy as np
import pytest


def refused(lq, call, *args, code=None, **kw):
    with pytest.raises(lq.LlamaQError) as e:
        call(*args, **kw)
    assert e.value.code == (lq.EINVAL if code is None else code)
    assert lq.last_error()


def row8(lq, rows, cols, **kw):
    f = dict(q=256, s=256, rows=rows, cols=cols, group_size=cols, kind=lq.KIND_ROW8)
    return lq.QuantizedTensor(**{**f, **kw})


def test_quantize_rows(lq):
    out = row8(lq, 2, 64)
    refused(lq, lq.quantize_rows, out, 256, 0)
    refused(lq, lq.quantize_rows, out, 256, 131073)
    refused(lq, lq.quantize_rows, out, 256, 64, 3)
    refused(lq, lq.quantize_rows, out, 256, 64, lq.F32, 63)
    refused(lq, lq.quantize_rows, out, None, 64)
    refused(lq, lq.quantize_rows, out, 258, 64)
    refused(lq, lq.quantize_rows, row8(lq, 2, 64, q=8), 256, 64)
    refused(lq, lq.quantize_rows, row8(lq, 2, 64, s=None), 256, 64)
    refused(lq, lq.quantize_rows, row8(lq, -1, 64), 256, 64)


def test_matmul_rows(lq):
    x, w = row8(lq, 2, 64), row8(lq, 5, 64)
    refused(lq, lq.matmul_rows, 256, x, w, 65, 5)
    refused(lq, lq.matmul_rows, 256, x, w, 64, 6)
    refused(lq, lq.matmul_rows, 256, x, w, 64, 5, 9)
    refused(lq, lq.matmul_rows, 256, x, w, 64, 5, lq.F32, 4)
    refused(lq, lq.matmul_rows, None, x, w, 64, 5)
    refused(lq, lq.matmul_rows, 257, x, w, 64, 5, lq.BF16)
    refused(lq, lq.matmul_rows, 256, row8(lq, 2, 64, kind=lq.KIND_ACT8), w, 64, 5)
    refused(lq, lq.matmul_rows, 256, x, row8(lq, 5, 64, kind=lq.KIND_INT8), 64, 5)
    refused(lq, lq.matmul_rows, 256, row8(lq, 2, 64, group_size=32), w, 64, 5)
    refused(lq, lq.matmul_rows, 256, x, row8(lq, 5, 64, q=264), 64, 5)
    refused(lq, lq.matmul_rows, 256, row8(lq, 2, 131073), row8(lq, 5, 131073), 131073, 5)


def paged(lq, **kw):
    f = dict(codes=256, scales=256, n_pages=10, page_size=16, n_kv_heads=2, head_size=64)
    return lq.PagedKV(**{**f, **kw})


def seqs(lq, **kw):
    f = dict(row_start=256, context=256, pages=256, n_seqs=2, n_rows=3, max_pages=4, max_rows=2, max_context=50)
    return lq.KVBatch(**{**f, **kw})


BAD_CACHE = [dict(page_size=24), dict(page_size=0), dict(page_size=256), dict(head_size=0), dict(head_size=24),
             dict(head_size=272), dict(n_kv_heads=0), dict(n_kv_heads=3), dict(codes=None), dict(codes=264),
             dict(scales=None), dict(scales=260), dict(n_pages=-1)]
BAD_BATCH = [dict(row_start=None), dict(context=None), dict(pages=None), dict(row_start=258), dict(n_rows=-1),
             dict(n_seqs=-1), dict(max_pages=-1), dict(max_rows=-1), dict(max_context=-1)]


def test_attention(lq):
    ok = (256, 256, 4, paged(lq), seqs(lq))
    for kw in BAD_CACHE:
        refused(lq, lq.paged_attention, 256, 256, 4, paged(lq, **kw), seqs(lq), lq.F32, 0.1, 1 << 20, 1 << 20)
    for kw in BAD_BATCH:
        refused(lq, lq.paged_attention, 256, 256, 4, paged(lq), seqs(lq, **kw))
    refused(lq, lq.paged_attention, 256, 256, 4, paged(lq), seqs(lq, n_seqs=70000), code=lq.EUNSUPPORTED)
    refused(lq, lq.paged_attention, 256, 256, 0, *ok[3:])
    refused(lq, lq.paged_attention, 256, 256, 5, *ok[3:])
    refused(lq, lq.paged_attention, *ok, 7)
    refused(lq, lq.paged_attention, *ok, lq.F32, float("nan"))
    refused(lq, lq.paged_attention, *ok, lq.F32, float("inf"))
    refused(lq, lq.paged_attention, *ok, lq.F32, 0.1, 255)
    refused(lq, lq.paged_attention, *ok, lq.F32, 0.1, 256, 255)
    refused(lq, lq.paged_attention, None, 256, *ok[2:])
    refused(lq, lq.paged_attention, 256, None, *ok[2:])
    refused(lq, lq.paged_attention, 258, 256, *ok[2:])
    refused(lq, lq.paged_attention, *ok, lse_ptr=258)


def rows(lq, **kw):
    f = dict(q=256, k=256, v=256, q_out=256, k_out=256, v_out=256, ld_q=256, ld_k=128, ld_v=128, ld_q_out=256,
             ld_kv_out=128, n_heads=4, type=lq.F32, rope=256, rope_rows=50, rope_mode=lq.ROPE_PAIRS)
    return lq.KVRows(**{**f, **kw})


def test_append(lq):
    for kw in BAD_CACHE:
        big = dict(ld_q=1 << 20, ld_k=1 << 20, ld_v=1 << 20, ld_q_out=1 << 20, ld_kv_out=1 << 20)
        refused(lq, lq.kv_append, paged(lq, **kw), seqs(lq), rows(lq, **big))
    for kw in BAD_BATCH:
        refused(lq, lq.kv_append, paged(lq), seqs(lq, **kw), rows(lq))
    for kw in (dict(k=None), dict(v=None), dict(q_out=None), dict(ld_q=255), dict(ld_k=127), dict(ld_v=127),
               dict(ld_q_out=255), dict(ld_kv_out=127), dict(n_heads=5), dict(type=3), dict(rope_mode=2),
               dict(rope_rows=-1), dict(rope=260), dict(k=258), dict(v_out=257)):
        refused(lq, lq.kv_append, paged(lq), seqs(lq), rows(lq, **kw))
    with pytest.raises(lq.LlamaQError):
        lq.check(lq.lib().kv_append(paged(lq), seqs(lq), None))


def test_rope_table(lq):
    t = lq.rope_table(40, 48)
    p, i = np.arange(40)[:, None], np.arange(24)[None]
    a = p * 10000.0 ** (-2 * i / 48)
    # fp32 angles up to 39: half an ulp of the frequency and of the product
    assert np.abs(t - np.stack((np.cos(a), np.sin(a)), -1)).max() <= 40 * 4 * 2.0**-24
    refused(lq, lq.rope_table, 4, 47)
    refused(lq, lq.rope_table, -1, 48)
