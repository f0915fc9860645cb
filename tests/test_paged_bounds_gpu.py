"""max_rows as an upper bound, however far above the rows there are."""
import numpy as np
import pytest

from paged_ref import Batch, attention, random_cache
from test_paged_gpu import Appender, run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,ctx,kv_heads,group,hs", [
    ([1, 1], [40, 300], 1, 300, 16), ([1], [500], 2, 1, 64), ([2, 1], [90, 33], 2, 4, 64), ([70, 1, 3], [90, 200, 3], 3, 2, 128)])
def test_attend_any_row_bound(cuda, rows, ctx, kv_heads, group, hs):
    rng = np.random.default_rng(group)
    batch = Batch(rng, rows, ctx, 32)
    codes, scales = random_cache(rng, batch.n_pages, kv_heads, hs, 32)
    q = rng.standard_normal((batch.n_rows, kv_heads * group, hs)) * 2
    for bound in (batch.n_rows, 2**31 - 1):
        qv, out, lse = run_attention(cuda, q, codes, scales, batch, "f32", hs, hs**-0.5, dev=batch.device(cuda, max_rows=bound))
        want, wlse, tol, ltol = attention(qv, codes, scales, batch, "f32", hs**-0.5)
        assert np.all(np.abs(out - want) <= tol) and np.all(np.abs(lse - wlse) <= ltol)


@pytest.mark.parametrize("rows,ctx", [([1], [20]), ([1, 1], [20, 5]), ([5, 30], [20, 30])])
def test_append_any_row_bound(cuda, rows, ctx):
    rng = np.random.default_rng(len(rows))
    b = Batch(rng, rows, ctx, 16)
    a = Appender(cuda, rng, b.n_pages, 2, 64, 16, "f32", "pairs")
    a.scales.fill_(0.001)
    a.check(b, dev=b.device(cuda, max_rows=2**31 - 1))
