"""The host side of the paged cache where masks and batches are at a limit."""
import pytest
import torch

from quarot_b200.transformers import MultiLayerPagedKVCache4Bit
from quarot_b200.transformers import kv_cache as KV
from oracle import quarot_oracle as O


def test_the_page_table_of_the_cache_stays_in_the_pool():
    cache = MultiLayerPagedKVCache4Bit(2, 16, 32, "cpu", 1, 1, 128)
    cache.length = 30
    got = cache.get_cache_specs_for_flash_infer(torch.ones(2, 90, dtype=torch.int64))
    assert got["kv_indices"].tolist() == [0, 2, 1, 3] and got["kv_indptr"].tolist() == [0, 2, 4]
    assert got["last_page_offset"].tolist() == [16, 16]


@pytest.mark.parametrize("batch,page,width,seed", [(1, 1, 3, 0), (7, 16, 4, 1), (50, 10, 9, 2), (300, 8, 2, 3)])
def test_page_table_in_torch_operations_against_the_oracle(batch, page, width, seed):
    """Fixed ownership; the lengths end at the capacity, slot maps fit exactly or have rows to spare."""
    g = torch.Generator().manual_seed(seed)
    total = torch.randint(0, width * page + 1, (batch,), generator=g, dtype=torch.int32)
    new = torch.minimum(torch.randint(0, 2 * page + 2, (batch,), generator=g, dtype=torch.int32), total)
    total[0] = new[0] = 0
    for tokens in (int(new.sum()), int(new.sum()) + 9):
        got = KV._fixed_page_table(total, new, tokens, page, width)
        want = O.kv_page_table((total - new).tolist(), new.tolist(), tokens, page, None, None, width)
        used = want["kv_indptr"][-1]
        assert got["kv_indices"].tolist() == want["kv_indices"][:used] and got["kv_indices"].dtype is torch.int32
        for key in ("kv_indptr", "last_page_offset", "append_indptr", "slot_map"):
            assert got[key].tolist() == want[key], key
        assert got["kv_indptr"].dtype is got["append_indptr"].dtype is got["last_page_offset"].dtype is torch.int32
        assert got["slot_map"].dtype is torch.int64


def test_page_table_in_torch_operations_leaves_out_what_does_not_fit():
    got = KV._fixed_page_table(torch.tensor([40, 20], dtype=torch.int32), torch.tensor([3, 2], dtype=torch.int32), 5, 16, 2)
    assert got["slot_map"].tolist() == [-1, -1, -1, (2 + 1) * 16 + 2, (2 + 1) * 16 + 3]
    assert got["kv_indptr"].tolist() == [0, 2, 4] and got["last_page_offset"].tolist() == [16, 4]
