"""The host side of the paged cache where masks and batches are at a limit."""
import torch

from quarot_b200.transformers import MultiLayerPagedKVCache4Bit


def test_the_page_table_of_the_cache_stays_in_the_pool():
    cache = MultiLayerPagedKVCache4Bit(2, 16, 32, "cpu", 1, 1, 128)
    cache.length = 30
    got = cache.get_cache_specs_for_flash_infer(torch.ones(2, 90, dtype=torch.int64))
    assert got["kv_indices"].tolist() == [0, 2, 1, 3] and got["kv_indptr"].tolist() == [0, 2, 4]
    assert got["last_page_offset"].tolist() == [16, 16]
