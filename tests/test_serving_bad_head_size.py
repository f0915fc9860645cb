"""A bad head size is refused by the library, not by what Python makes of it first (CPU only)."""
import pytest

from test_serving_refusals import paged, refused, seqs


@pytest.mark.parametrize("head_size", [0, -64, 24])
def test_attention_default_scale(lq, head_size):
    refused(lq, lq.paged_attention, 256, 256, 4, paged(lq, head_size=head_size), seqs(lq), ld_q=1 << 20, ld_out=1 << 20)


def test_rope_table_negative_head_size(lq):
    refused(lq, lq.rope_table, 4, -48)
