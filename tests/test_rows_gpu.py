"""quantize_rows and matmul_rows against 64 bits, at the sizes where they can
go wrong: one row and many, one column, rows that end inside a 16-byte piece or
a tile, row strides, unaligned pointers, zero and non-finite rows."""
import numpy as np
import pytest

from gpu_util import lq
from paged_ref import HALF_ULP, KINDS, torch_type

pytestmark = pytest.mark.gpu


def row8(torch, q, s):
    """A ROW8 tensor of codes [rows, cols] on the device, padding zero."""
    rows, cols = q.shape
    t = torch.zeros(rows, lq.row8_pitch(cols), dtype=torch.int8, device="cuda")
    t[:, :cols] = torch.from_numpy(q).cuda()
    ts = torch.from_numpy(s.astype(np.float32)).cuda()
    return lq.QuantizedTensor(q=t.data_ptr(), s=ts.data_ptr(), rows=rows, cols=cols, group_size=cols,
                              kind=lq.KIND_ROW8), (t, ts)


def empty_row8(torch, rows, cols):
    t = torch.full((rows, lq.row8_pitch(cols)), 99, dtype=torch.int8, device="cuda")
    ts = torch.full((rows,), 99.0, device="cuda")
    return lq.QuantizedTensor(q=t.data_ptr(), s=ts.data_ptr(), rows=rows), t, ts


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,n,extra,shift", [
    (1, 1, 0, 0), (3, 15, 0, 0), (2, 288, 0, 0), (5, 1000, 24, 0), (4, 1001, 3, 1), (1, 4096, 0, 0),
    (7, 11008, 0, 0), (2, 20001, 0, 3), (300, 77, 1, 0),
])
def test_quantize_rows(cuda, dtype, rows, n, extra, shift):
    torch = cuda
    rng = np.random.default_rng(rows * 7919 + n)
    ld = n + extra
    buf = torch.from_numpy(rng.standard_normal(rows * ld + 8) * 3).cuda().to(torch_type(torch, dtype))
    x = buf[shift:shift + rows * ld].view(rows, ld)
    x[0, :n] = 0  # a zero row
    out, q, s = empty_row8(torch, rows, n)
    lq.quantize_rows(out, x.data_ptr(), n, KINDS[dtype], ld)
    lq.sync()
    assert (out.cols, out.group_size, out.kind) == (n, n, lq.KIND_ROW8)
    xv = x[:, :n].double().cpu().numpy()
    qv, sv = q.cpu().numpy().astype(np.float64), s.cpu().numpy().astype(np.float64)
    assert not qv[:, n:].any()  # the padding
    peak = np.abs(xv).max(1)
    want = np.where(peak > 0, peak / 127, np.float64(np.float32(1e-8)))
    assert np.all(np.abs(sv - want) <= want * 2.0**-24)
    # a code is the nearest integer to x / s; x / s carries one fp32 rounding
    assert np.all(np.abs(qv[:, :n] - xv / sv[:, None]) <= 0.5 + 127 * 2.0**-23)
    assert np.abs(qv).max() <= 127 and (np.abs(qv[peak > 0]).max(1) == 127).all()
    # bit for bit the fp32 formula
    x32 = xv.astype(np.float32)
    s32 = np.where(peak > 0, np.abs(x32).max(1) / np.float32(127), np.float32(1e-8)).astype(np.float32)
    assert np.array_equal(s.cpu().numpy(), s32)
    assert np.array_equal(q.cpu().numpy()[:, :n], np.rint(x32 / s32[:, None]).astype(np.int8))


def test_quantize_rows_non_finite(cuda):
    torch = cuda
    x = torch.randn(4, 100, device="cuda")
    x[1, 99], x[2, 0] = float("nan"), float("-inf")
    out, q, s = empty_row8(torch, 4, 100)
    lq.quantize_rows(out, x.data_ptr(), 100)
    w, keep = row8(torch, np.ones((5, 100), np.int8), np.ones(5))
    y = torch.empty(4, 5, device="cuda")
    lq.matmul_rows(y.data_ptr(), out, w, 100, 5)
    lq.sync()
    assert s.isnan().tolist() == [False, True, True, False]
    assert not q[1:3].any()
    assert y.isnan().all(1).tolist() == [False, True, True, False]


SHAPES = [
    # rows, n, d: one of everything; the tiny configuration; ends inside tiles
    (1, 1, 1), (1, 288, 768), (1, 4096, 4096), (2, 31, 33), (3, 100, 129), (7, 768, 288), (8, 4096, 1000),
    (9, 513, 127), (15, 1000, 2000), (16, 128, 128), (17, 144, 4097), (31, 5120, 640), (33, 2048, 300), (64, 8192, 1024),
    (65, 640, 385), (100, 4096, 4096), (128, 256, 256), (129, 1000, 1111), (255, 4097, 513), (257, 288, 768),
    (700, 1000, 1500), (1030, 272, 2304), (300, 16384, 40), (2048, 64, 64),
]


@pytest.mark.parametrize("rows,n,d", SHAPES)
def test_matmul_rows_exact(cuda, rows, n, d):
    """fp32 out: the integer dot is exact, so the result is bit for bit
    fl(fl(dot) * fl(sx * sw))."""
    torch = cuda
    rng = np.random.default_rng(rows * 31 + n * 7 + d)
    xq = rng.integers(-127, 128, (rows, n)).astype(np.int8)
    wq = rng.integers(-127, 128, (d, n)).astype(np.int8)
    xs, ws = (rng.random(m).astype(np.float32) + 0.5 for m in (rows, d))
    x, keep_x = row8(torch, xq, xs)
    w, keep_w = row8(torch, wq, ws)
    y = torch.full((rows, d), float("nan"), device="cuda")
    lq.matmul_rows(y.data_ptr(), x, w, n, d)
    lq.sync()
    # the dots in fp64: below 2^53, exact
    dot = (keep_x[0][:, :n].double() @ keep_w[0][:, :n].double().T).cpu().numpy()
    want = dot.astype(np.float32) * (xs[:, None] * ws[None])
    assert np.array_equal(y.cpu().numpy(), want)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,n,d,extra", [(1, 1000, 515, 5), (5, 288, 768, 8), (40, 640, 300, 1), (200, 320, 777, 3),
                                            (513, 1024, 1000, 0)])
def test_matmul_rows_types_and_strides(cuda, dtype, rows, n, d, extra):
    """Each type; rows of xout further apart than d, what lies between untouched."""
    torch = cuda
    rng = np.random.default_rng(rows + n + d)
    xq = rng.integers(-127, 128, (rows, n)).astype(np.int8)
    wq = rng.integers(-127, 128, (d, n)).astype(np.int8)
    xs, ws = (rng.random(m).astype(np.float32) / 500 for m in (rows, d))
    x, keep_x = row8(torch, xq, xs)
    w, keep_w = row8(torch, wq, ws)
    y = torch.full((rows, d + extra), 7.0, device="cuda", dtype=torch_type(torch, dtype))
    lq.matmul_rows(y.data_ptr(), x, w, n, d, KINDS[dtype], d + extra)
    lq.sync()
    assert bool((y[:, d:] == 7.0).all())
    want = xq.astype(np.float64) @ wq.astype(np.float64).T * (xs.astype(np.float64)[:, None] * ws.astype(np.float64)[None])
    tol = np.abs(want) * (3 * 2.0**-24 * 1.001 + (HALF_ULP[dtype] * 1.01 if dtype != "f32" else 0))
    assert np.all(np.abs(y[:, :d].double().cpu().numpy() - want) <= tol + (2.0**-25 if dtype == "f16" else 0))


@pytest.mark.parametrize("rows", [1, 20, 300])
def test_matmul_rows_largest_codes(cuda, rows):
    """Every code 127 at the longest row: the int32 sum stays in range."""
    torch = cuda
    n, d = 131072, 130
    x, keep_x = row8(torch, np.full((rows, n), 127, np.int8), np.ones(rows))
    w, keep_w = row8(torch, np.full((d, n), -127, np.int8), np.ones(d))
    y = torch.empty(rows, d, device="cuda")
    lq.matmul_rows(y.data_ptr(), x, w, n, d)
    lq.sync()
    assert bool((y == float(np.float32(-127.0 * 127 * n))).all())


@pytest.mark.parametrize("rows", [1, 8, 24, 200])
def test_matmul_rows_graph_and_streams(cuda, rows):
    """Captured and replayed on a stream of its own, and again and again: the
    same bits (workspaces are left as they were found)."""
    torch = cuda
    n, d = 2048, 1153
    rng = np.random.default_rng(rows)
    xv = torch.randn(rows, n, device="cuda")
    w, keep_w = row8(torch, rng.integers(-127, 128, (d, n)).astype(np.int8), np.full(d, 0.01))
    out, q, s = empty_row8(torch, rows, n)
    y = torch.empty(rows, d, device="cuda")

    def step():
        lq.quantize_rows(out, xv.data_ptr(), n)
        lq.matmul_rows(y.data_ptr(), out, w, n, d)

    step()
    lq.sync()
    want = y.clone()
    st = torch.cuda.Stream()
    lq.set_stream(st.cuda_stream)
    try:
        step()
        lq.sync()
        assert torch.equal(y, want)
        lq.graph_begin()
        step()
        g = lq.graph_end()
        for _ in range(20):
            y.fill_(float("nan"))
            torch.cuda.synchronize()
            lq.graph_launch(g)
            lq.sync()
            assert torch.equal(y, want)
        lq.graph_destroy(g)
        for _ in range(50):
            step()
        lq.sync()
        assert torch.equal(y, want)
    finally:
        lq.set_stream(None)


@pytest.mark.parametrize("rows", [1, 64])
def test_matmul_rows_right_after_its_inputs(cuda, rows):
    """Weights and activations quantized by the calls just before are seen."""
    torch = cuda
    n, d = 4096, 2048
    wv, xv = torch.randn(d, n, device="cuda"), torch.randn(rows, n, device="cuda")
    w, wq, ws = empty_row8(torch, d, n)
    x, xq, xs = empty_row8(torch, rows, n)
    y = torch.empty(rows, d, device="cuda")
    for k in range(5):
        wq.zero_(), xq.zero_()
        lq.quantize_rows(w, wv.data_ptr(), n)
        lq.quantize_rows(x, xv.data_ptr(), n)
        lq.matmul_rows(y.data_ptr(), x, w, n, d)
        lq.sync()
        dot = xq[:, :n].double() @ wq[:, :n].double().T
        want = dot.float() * (xs[:, None] * ws[None])
        assert torch.equal(y, want)
        wv.mul_(-1.5)


def test_no_rows(cuda):
    x = lq.QuantizedTensor(rows=0)
    lq.quantize_rows(x, None, 64)
    w, keep = row8(cuda, np.ones((3, 64), np.int8), np.ones(3))
    lq.matmul_rows(None, x, w, 64, 3)
    lq.sync()
