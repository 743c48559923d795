"""Steps of the paged 4-bit cache in which something is hidden, refused, padded or at a limit: masks that hide single
tokens, page tables of many or over-long sequences, calls with ragged bounds.  Attention is held to the oracle's bounds, as
in test_gpu_kv_attend.py; everything else is exact."""
import os
import subprocess
import sys
import threading

import pytest
import torch

from quarot_b200 import _lib
from quarot_b200.transformers import MultiLayerPagedKVCache4Bit
from quarot_b200.transformers import kv_cache as KV
from oracle import quarot_oracle as O
from test_gpu_kv_attend import DEV, _attend, _check, _i32, _oracle, _run_table, _setup, both_kernels, kernel  # noqa: F401
from test_gpu_kv_attend_calls import _need, _raw

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_a_prompt_in_any_strides_is_cached():
    """Keys and values whose head dimension is not contiguous are copied, as a single token's are."""
    T, H, P = 21, 2, 16
    g = torch.Generator().manual_seed(92)
    k, v = (torch.randn(1, T, 128, H, generator=g).half().to(DEV).transpose(2, 3) for _ in range(2))
    pools = []
    for kk, vv in ((k, v), (k.contiguous(), v.contiguous())):
        cache = MultiLayerPagedKVCache4Bit(1, P, 64, DEV, 1, H, 128)
        cache.pages.fill_(0)
        cache.scales.fill_(0)
        assert cache.update(kk, vv, 0, {})[0] is kk
        r = cache.update(kk[:, :3], vv[:, :3], 0, {})
        pools.append((cache.pages, cache.scales, r(kk[:, :3])))
    assert all(torch.equal(a, b) for a, b in zip(*pools)) and bool((pools[0][1] != 0).any())
