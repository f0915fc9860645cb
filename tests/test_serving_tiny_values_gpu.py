"""Rows and pages whose largest value is a few of fp32's smallest steps: the scale
is rounded to whole steps, and codes stay within 127 in the value's sign."""
import numpy as np
import pytest

from gpu_util import lq
from paged_ref import Batch
from test_paged_gpu import Appender
from test_rows_gpu import empty_row8

pytestmark = pytest.mark.gpu

STEP = np.float64(2.0**-149)


def want_codes(x):
    """rint(x / s) kept to 127, s = max|x| / 127 in fp32 (0: 1e-8)."""
    s = np.float32(np.abs(x).max() / 127)  # of whole steps, once rounded: as fp32 divides
    if s == 0:
        s = np.float32(1e-8)
    return np.clip(np.rint(x / np.float64(s)), -127, 127), s


@pytest.mark.parametrize("peak", [1, 63, 64, 100, 127, 128, 190, 191, 300, 5000, 20000, 2**21, 2**24])
def test_quantize_rows_subnormal(cuda, peak):
    torch = cuda
    x = np.linspace(-peak, peak, 77).round() * STEP
    out, q, s = empty_row8(torch, 1, 77)
    xt = torch.from_numpy(x.astype(np.float32)).cuda()
    lq.quantize_rows(out, xt.data_ptr(), 77)
    lq.sync()
    codes, scale = want_codes(x)
    assert s.cpu().numpy()[0] == scale
    assert np.array_equal(q.cpu().numpy()[0, :77], codes)


@pytest.mark.parametrize("rows", [1, 5])
@pytest.mark.parametrize("peak", [64, 190, 300, 5000])
def test_append_subnormal(cuda, rows, peak):
    torch = cuda
    rng = np.random.default_rng(peak)
    b = Batch(rng, [rows], [rows], 16)
    a = Appender(torch, rng, b.n_pages, 1, 64, 16, "f32", None, group=1)
    x = torch.from_numpy((rng.integers(-peak, peak + 1, (rows, 128)) * STEP).astype(np.float32)).cuda()
    x[0, 0], x[0, 64] = peak * STEP, -peak * STEP

    def edit(kv):
        kv[:rows] = x

    a.call(b, edit=edit)
    codes, scales = a.after
    values = x.double().cpu().numpy()
    p = int(b.pages[0, 0])
    for which in (0, 1):
        want, scale = want_codes(values[:, 64 * which: 64 * which + 64])
        assert scales[p, 0, which] == scale
        page = codes[p, 0, which].reshape(-1)
        got = (page.reshape(4, 16, 16).transpose(1, 0, 2).reshape(16, 64) if which == 0
               else page.reshape(1, 64, 16).transpose(0, 2, 1).reshape(16, 64))
        assert np.array_equal(got[:rows], want)
