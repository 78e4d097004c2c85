"""Block tables that the binding of the drafted-token functions takes, on CPU tensors (their device index is -1)."""
import pytest
import torch

from pluto_b200 import PlutoStatusError
from pluto_b200.layers import _draft_calls, gqa_decode, kv_layout


def pool_of(pages, table, batch, dtype=torch.bfloat16):
    k = torch.zeros(pages, 16, 2, 64, dtype=dtype)
    return _draft_calls().draft_pool(k, k, table, None, None, batch, -1)


@pytest.mark.parametrize("batch", [1, 2, 4])
def test_a_table_without_columns_is_refused(engine, batch):
    """It has no address, and must not pass for the absence of a table, where every sequence has a page of its own."""
    table = torch.zeros(batch, 0, dtype=torch.int32)
    assert table.data_ptr() == 0
    with pytest.raises(PlutoStatusError, match="block table"):
        pool_of(2, table, batch)


def test_tables_of_other_shapes(engine):
    for bad in (torch.zeros(2, dtype=torch.int32), torch.zeros(3, 4, dtype=torch.int32), torch.zeros(2, 4, dtype=torch.int64),
                torch.zeros(2, 8, dtype=torch.int32)[:, ::2]):
        with pytest.raises(PlutoStatusError, match="block table"):
            pool_of(8, bad, 2)
    cache, scales = pool_of(8, torch.zeros(2, 4, dtype=torch.int32), 2)
    assert scales is None and len(cache) > 0
    with pytest.raises(PlutoStatusError, match="a page for every sequence"):
        pool_of(1, None, 2)


def test_the_other_paged_functions_refuse_such_a_table_too(engine):
    k, table = torch.zeros(1, 16, 2, 64, dtype=torch.bfloat16), torch.zeros(4, 0, dtype=torch.int32)
    q, lengths = torch.zeros(4, 4, 64, dtype=torch.bfloat16), torch.ones(4, dtype=torch.int32)
    with pytest.raises(PlutoStatusError, match="block table"):
        kv_layout(k, k, table, 16, 2048, 128)
    with pytest.raises(PlutoStatusError, match="block table"):
        gqa_decode(q, k, k, lengths, 16, block_table=table)
