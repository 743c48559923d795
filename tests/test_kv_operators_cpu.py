"""Argument checks of the cache operators that are made before anything touches a GPU, and the CPU side of the cache."""
import threading

import pytest
import torch

from quarot_b200 import _lib
from quarot_b200.transformers import MultiLayerPagedKVCache4Bit
from quarot_b200.transformers import kv_cache as KV
from oracle import quarot_oracle as O

P = 1 << 20                                                         # stands for an aligned pointer; nothing reads it


def _call(name, *args):
    """(status, error text) of a C entry, from a thread of its own: the text of the last error is kept per thread."""
    out = []
    t = threading.Thread(target=lambda: out.append((getattr(_lib.lib, name)(*args), _lib.last_error())))
    t.start()
    t.join()
    return out[0]


def _attend(**kw):
    a = dict(o=P, ots=1024, ohs=128, q=P, qts=1024, qhs=128, data=P, param=P, pages=10, indptr=P, indices=P, entries=100, last=P, qo=P, total=8,
             most=8, batch=1, layers=1, layer=0, heads=8, kv_heads=8, page=16, dim=128, window=0, sinks=0, rotate=0, work=None, bytes=0,
             stream=None)
    assert not set(kw) - set(a)
    a.update(kw)
    return _call("qr_kv_attend_i4", *a.values())


@pytest.mark.parametrize("kw,words", [
    (dict(batch=-1), "negative"), (dict(total=-1), "negative"), (dict(most=-1), "negative"), (dict(entries=-1), "negative"),
    (dict(o=None), "null"), (dict(q=None), "null"), (dict(data=None), "null"), (dict(param=None), "null"), (dict(indptr=None), "null"),
    (dict(indices=None), "null"), (dict(last=None), "null"), (dict(dim=64), "head_dim"), (dict(layer=1), "layer"), (dict(layer=-1), "layer"),
    (dict(page=0), "page"), (dict(pages=0), "pages"), (dict(heads=12), "multiple"), (dict(kv_heads=0), "multiple"), (dict(heads=0), "multiple"),
    (dict(pages=1 << 32), "2^32"), (dict(window=-1), "window"), (dict(sinks=-1), "sink"), (dict(qo=None), "one new token"),
    (dict(qo=None, total=1, most=2), "one new token"), (dict(most=9), "max_q_len"), (dict(total=1 << 40, most=1), "rows"), (dict(total=1 << 62, most=1), "rows"),
    (dict(o=P + 4), "aligned"), (dict(q=P + 2), "aligned"), (dict(data=P + 8), "aligned"), (dict(param=P + 2), "aligned"),
    (dict(qts=1022), "aligned"), (dict(ohs=130), "aligned"), (dict(work=P + 8, bytes=64), "aligned")])
def test_attention_entry_refuses(kw, words):
    rc, text = _attend(**kw)
    assert rc != 0 and words in text


def test_empty_calls_do_nothing():
    assert [_attend(**kw)[0] for kw in (dict(batch=0), dict(total=0), dict(most=0))] == [0, 0, 0]
    assert _lib.lib.qr_kv_page_table(None, None, 0, 0, 16, 4, None, None, 0, None, None, None, None, None, None, None, None, None) == 0


@pytest.mark.parametrize("change", [{0: None}, {2: -1}, {2: 8193}, {3: -1}, {4: 0}, {5: 0}, {2: 8192, 5: 1 << 18}, {3: 1 << 31}, {8: 4, 7: None},
                                    {9: None}, {10: None}, {11: None}, {12: None}, {13: None}, {14: None}, {15: None}, {16: None}])
def test_page_table_entry_refuses(change):
    a = [P, P, 4, 8, 16, 4, P, P, 4, P, P, P, P, P, P, P, P, None]
    for i, v in change.items():
        a[i] = v
    rc, text = _call("qr_kv_page_table", *a)
    assert rc != 0 and "qr_kv_page_table" in text


@pytest.mark.parametrize("change", [{0: None}, {1: None}, {3: None}, {4: None}, {7: None}, {2: 0}, {10: -1}, {11: 0}, {12: 5}, {13: 0}, {14: 0},
                                    {15: 64}, {5: 1022}, {4: P + 4}])
def test_append_by_slot_map_entry_refuses(change):
    a = [P, P, 10, P, P, 1024, 128, P, 1024, 128, 4, 2, 1, 8, 16, 128, 0, None]
    for i, v in change.items():
        a[i] = v
    rc, text = _call("qr_kv_append_slots_i4", *a)
    assert rc != 0 and "qr_kv_append_slots_i4" in text


def test_tensors_of_the_cpu_are_refused():
    data, param = torch.zeros(4, 1, 2, 2, 16, 64, dtype=torch.uint8), torch.zeros(4, 1, 2, 2, 16, 2, dtype=torch.float16)
    i = torch.zeros(4, dtype=torch.int32)
    q = torch.zeros(3, 2, 128, dtype=torch.float16)
    with pytest.raises(RuntimeError):
        KV.chunk_attention_i4(q.clone(), q, data, param, i[:2], i, i[:1], i[:2], 0)
    with pytest.raises(RuntimeError):
        KV.batch_decode_i4(q.clone(), q, data, param, i, i, i[:3], 0, window=4)
    with pytest.raises(RuntimeError):
        KV.append_kv_slots_i4(data, param, torch.zeros(3, dtype=torch.int64), q, q, 0)
    with pytest.raises(RuntimeError):
        KV.build_page_table(i, None, 4, 16, max_blocks=2)


@pytest.mark.parametrize("kw", [dict(window_size=0), dict(window_size=-3), dict(window_size=8, sink_tokens=-1), dict(sink_tokens=-1)])
def test_cache_refuses_windows_that_are_none(kw):
    with pytest.raises(ValueError):
        MultiLayerPagedKVCache4Bit(1, 16, 64, "cpu", 1, 2, 128, **kw)


def test_page_table_of_the_cache_with_ragged_masks_on_the_cpu():
    cache = MultiLayerPagedKVCache4Bit(3, 4, 32, "cpu", 1, 2, 128)
    cache.length = 9
    mask = torch.zeros(3, 9, dtype=torch.int64)
    for b, n in enumerate((9, 1, 4)):
        mask[b, :n] = 1
    got = cache.get_cache_specs_for_flash_infer(mask)
    assert got["kv_indptr"].tolist() == [0, 3, 4, 5] and got["kv_indices"].tolist() == [0, 3, 6, 1, 2]
    assert got["last_page_offset"].tolist() == [1, 1, 4]


def test_oracle_page_table_and_attention_agree_with_plain_definitions():
    """One sequence, one head, pages in order: the oracle is the textbook softmax of the dequantised rows."""
    g = torch.Generator().manual_seed(5)
    n, page = 11, 4
    codes = torch.randint(0, 256, (3, 1, 2, 1, page, 64), generator=g, dtype=torch.uint8)
    par = torch.rand(3, 1, 2, 1, page, 2, generator=g).half()
    q = torch.randn(2, 1, 128, generator=g).half()
    o, bound = O.paged_attention(q, codes, par, 0, [0, 3], torch.arange(3, dtype=torch.int32), [n - 2 * page], [0, 2], 0, 0)
    kv = []
    for which in (0, 1):
        c = codes[:, 0, which, 0].reshape(-1, 64)[:n]
        x = torch.stack((c & 15, c >> 4), -1).reshape(n, 128).double()
        pr = par[:, 0, which, 0].reshape(-1, 2)[:n].double()
        kv.append(x * pr[:, :1] - pr[:, 1:])
    for i in range(2):
        m = n - 1 + i
        w = torch.softmax(kv[0][:m] @ q[i, 0].double() / 128 ** 0.5, 0)
        assert torch.allclose(o[i, 0], w @ kv[1][:m], rtol=1e-12, atol=1e-12)
    assert bool((bound > 0).all())
