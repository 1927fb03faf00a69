"""The sizes that a PagedBlock refuses when it is made, without a GPU: what its operators would refuse at each step."""
import pytest

import perseus_amd as pa
from perseus_amd import attention
from tests.test_clear import NoStream


@pytest.mark.parametrize("bad", [dict(decay=float("inf")), dict(decay=1e39), dict(decay=float("nan")), dict(seqs=65536),
                                 dict(heads=65536, kv_heads=65536, dim=8), dict(heads=32768, kv_heads=32768, dim=256),
                                 dict(kv_heads=4, dim=256, page_rows=1 << 21)])
def test_a_paged_block_refuses_what_its_operators_would(bad):
    ops = pa.Clear(NoStream, workspace=0)
    with pytest.raises(ValueError):
        attention.PagedBlock(**{**dict(ops=ops, heads=4, kv_heads=2, dim=64, seqs=2, pages=8), **bad})
