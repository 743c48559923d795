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


# ------------------------------------------------------------------ masks
def _bytes(cache):
    return cache.pages.cpu(), cache.scales.cpu().view(torch.int16)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("window,sinks,group", [(None, 0, 1), (None, 0, 2), (20, 2, 1), (20, 2, 4)])
def test_a_single_token_that_the_mask_hides_is_not_cached(window, sinks, group, wide):
    """Ragged sequences, an empty one among them; steps of one token that is padding for some of them.  What is cached of
    those stays, their rows give zeros, the others get their token.  A mask may be wider than the tokens so far."""
    B, H, P, L = 4, 2, 16, 2
    cache = MultiLayerPagedKVCache4Bit(B, P, 64, DEV, L, H, 128, window_size=window, sink_tokens=sinks)
    cache.pages.fill_(0xEE)
    cache.scales.fill_(float("nan"))
    g = torch.Generator().manual_seed(91)
    mask = torch.zeros(B, 0, dtype=torch.int64)
    count = [0] * B
    for n, new in enumerate([[30, 16, 0, 5], [1, 0, 0, 1], [0, 0, 1, 1], [0, 0, 0, 0], [1, 1, 1, 1]]):
        length = 33 if n == 0 else 1
        column = torch.zeros(B, length, dtype=torch.int64)
        for b, m in enumerate(new):
            column[b, length - m:] = 1
        mask = torch.cat((mask, column), 1)
        given = torch.nn.functional.pad(mask, (0, 9)) if wide else mask
        k, v = (torch.randn(B, length, H, 128, generator=g).half() for _ in range(2))
        q = (torch.randn(B, length, H * group, 128, generator=g) * 1.5).half()
        shown = [b for b in range(B) if new[b]]
        for layer in range(L):
            before = _bytes(cache)
            r = cache.update((k + layer).half().to(DEV), v.to(DEV), layer, {"attention_mask": given.to(DEV)})
            after = _bytes(cache)
            ours = torch.zeros(before[0].shape[:5], dtype=torch.bool)
            for b, m in enumerate(new):
                for t in range(count[b], count[b] + m):
                    ours[t // P * B + b, layer, :, :, t % P] = True
            assert torch.equal(before[0][~ours], after[0][~ours]) and torch.equal(before[1][~ours], after[1][~ours])
            assert bool((after[1][ours][:, 0] != before[1][ours][:, 0]).all())
            if n == 0:
                continue
            got = r(q.to(DEV)).view(B, H * group, 128).cpu()
            total = [c + m for c, m in zip(count, new)]
            assert all(bool((got[b] == 0).all()) for b in range(B) if not new[b])
            if not shown:
                continue
            pages = [-(-t // P) for t in total]
            ref = O.paged_attention(O.kv_hadamard_fp16(q.view(B, H * group, 128)[shown]), cache.pages.cpu(), cache.scales.cpu(), layer,
                                    torch.tensor([0] + pages).cumsum(0), torch.tensor([j * B + b for b in range(B) for j in range(pages[b])]),
                                    [t - max(p - 1, 0) * P for t, p in zip(total, pages)], torch.tensor([0] + new).cumsum(0), window or 0, sinks)
            _check(got[shown], ref)
        count = [c + m for c, m in zip(count, new)]


@pytest.mark.parametrize("window", [None, 8])
def test_masks_that_hide_everything(window):
    """No sequence has a page: single tokens and chunks give zeros and cache nothing; the next token is the first."""
    B, H, P = 2, 2, 16
    cache = MultiLayerPagedKVCache4Bit(B, P, 64, DEV, 1, H, 128, hadamard_dtype=None, window_size=window)
    cache.pages.fill_(0xEE)
    g = torch.Generator().manual_seed(101)
    mask = torch.zeros(B, 0, dtype=torch.int64, device=DEV)
    for length in (5, 1, 3):
        mask = torch.cat((mask, mask.new_zeros(B, length)), 1)
        k = torch.randn(B, length, H, 128, generator=g).half().to(DEV)
        r = cache.update(k, k, 0, {"attention_mask": mask})
        assert length == 5 or bool((r(k) == 0).all())
    assert bool((cache.pages == 0xEE).all())
    mask = torch.cat((mask, mask.new_ones(B, 1)), 1)
    k = torch.randn(B, 1, H, 128, generator=g).half().to(DEV)
    got = cache.update(k, k, 0, {"attention_mask": mask})(k)
    codes, scale, zero = O.kv_asym_quant_pack(k.cpu().view(B, H, 128))
    value = torch.stack((codes & 15, codes >> 4), -1).view(B, H, 128) * scale.float() - zero.float()
    assert float((got.cpu().view(B, H, 128).float() - value).abs().max()) <= 2.0 ** -11 * float(value.abs().max()) * 1.01


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


def test_the_page_table_of_the_cache_stays_in_the_pool():
    cache = MultiLayerPagedKVCache4Bit(2, 16, 32, DEV, 1, 1, 128)
    cache.length = 30
    got = cache.get_cache_specs_for_flash_infer(torch.ones(2, 90, dtype=torch.int64, device=DEV))
    assert got["kv_indices"].tolist() == [0, 2, 1, 3] and got["kv_indptr"].tolist() == [0, 2, 4]
    assert got["last_page_offset"].tolist() == [16, 16]


def test_a_cache_of_more_sequences_than_the_page_table_kernel_takes():
    """Prompt, single tokens with and without a mask, and a chunk for 9000 sequences."""
    B, H, P = 9000, 1, 8
    g = torch.Generator().manual_seed(93)
    mask = torch.ones(B, 6, dtype=torch.int64)
    mask[::3, :4] = 0
    for masked in (False, True):
        cache = MultiLayerPagedKVCache4Bit(B, P, 16, DEV, 1, H, 128, hadamard_dtype=None)
        seen = mask if masked else torch.ones_like(mask)
        keys = []
        for n, length in enumerate((6, 1, 4)):
            k = torch.randn(B, length, H, 128, generator=g).half()
            if n:
                seen = torch.cat((seen, torch.ones(B, length, dtype=torch.int64)), 1)
            keys.append(k)
            r = cache.update(k.to(DEV), k.to(DEV), 0, {"attention_mask": seen.to(DEV)} if masked else {})
            if n == 0:
                continue
            got = r(k.to(DEV)).cpu()
            every = torch.cat(keys, 1)
            pick = [0, 1, 2, 3, 8191, 8192, 8193, B - 2, B - 1]
            for b in pick:
                mine = every[b][seen[b].bool()]
                m = mine.shape[0]
                pages, par = torch.zeros(2, 1, 2, H, P, 64, dtype=torch.uint8), torch.zeros(2, 1, 2, H, P, 2).half()
                qq, s, z = O.kv_asym_quant_pack(mine)
                for t in range(m):
                    pages[t // P, 0, :, 0, t % P] = qq[t, 0]
                    par[t // P, 0, :, 0, t % P] = torch.cat((s, z), -1)[t, 0]
                used = -(-m // P)
                ref = O.paged_attention(k[b], pages, par, 0, [0, used], torch.arange(used), [m - (used - 1) * P], [0, length])
                _check(got[b], ref)


# ------------------------------------------------------------------ page tables
_FRESH = """
import torch
from quarot_b200.transformers import kv_cache as KV
for width in (3, 400):
    for batch in (3060, 3063, 3064, 3067, 3071, 3075, 4000):
        lens = torch.randint(0, width * 16 - 1, (batch,), generator=torch.Generator().manual_seed(batch)).int()
        t = KV.build_page_table(lens.cuda(), None, batch, 16, max_blocks=width)
        want = torch.cat((torch.zeros(1, dtype=torch.int64), ((lens.long() + 16) // 16).cumsum(0)))
        assert torch.equal(t["kv_indptr"].cpu().long(), want), batch
        assert torch.equal(t["positions"].cpu(), lens) and t["status"].tolist() == [0, 0]
print("fine")
"""


def test_page_tables_around_48_kb_of_shared_memory_in_a_fresh_process():
    """No larger batch has come before: every launch asks for what it needs itself."""
    r = subprocess.run([sys.executable, "-c", _FRESH], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "fine", r.stderr[-2000:]


def test_page_tables_of_different_sizes_from_two_threads():
    errors = []

    def work(batch):
        try:
            lens = torch.full((batch,), 20, dtype=torch.int32, device=DEV)
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(400):
                    t = KV.build_page_table(lens, None, batch, 16, max_blocks=2)
                assert t["kv_indptr"][-1].item() == 2 * batch and t["slot_map"][-1].item() == (2 * batch - 1) * 16 + 4
        except Exception as e:  # noqa: BLE001 - reported below, from the main thread
            errors.append((batch, str(e)))
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(n,)) for n in (8192, 3100, 6000)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors


@pytest.mark.parametrize("form", ["free list", "pages there", "fixed"])
def test_sequences_longer_than_their_row_are_refused_as_they_are(form):
    """Their length is reported as it was, with and without new tokens; the pages listed are those of the row."""
    table, free, width = [[1, 2], [3, 4], [5, 6], [7, -1]], [8, 9], None
    if form == "pages there":
        free = None
    elif form == "fixed":
        table, free, width = None, None, 2
    got = _run_table([100, 33, 32, 5], [0, 2, 0, 4], 6, 16, table, free, width)
    assert got["seq_lens"].tolist() == [100, 33, 32, 9] and got["status"].tolist() == [0, 2]
    assert got["kv_indptr"].tolist() == [0, 2, 4, 6, 7] and got["last_page_offset"].tolist() == [16, 16, 16, 9]
    assert got["slot_map"].tolist()[:2] == [-1, -1] and got["positions"].tolist() == [-1, -1, 5, 6, 7, 8]


@both_kernels
@pytest.mark.parametrize("new", [[2, 3, 1], [70, 90, 80]])
def test_rows_of_a_refused_sequence(new):
    """The free list ends at the second sequence.  Its tokens are not cached; its rows, which stand among the others in q,
    give zeros where the positions are passed on, and the other sequences do not notice."""
    page, H, G, W = 16, 2, 2, 12
    lens = [30, 31, 4]
    g = torch.Generator().manual_seed(94)
    need = [-(-(n + m) // page) - -(-n // page) for n, m in zip(lens, new)]
    bt = torch.zeros(3, W, dtype=torch.int32, device=DEV)
    free = torch.randperm(40, generator=g).to(torch.int32).to(DEV)
    data = torch.zeros((40, 1, 2, H, page, 64), dtype=torch.uint8, device=DEV)
    param = torch.full((40, 1, 2, H, page, 2), float("nan"), dtype=torch.float16, device=DEV)
    first = KV.build_page_table(torch.zeros(3, dtype=torch.int32, device=DEV), _i32(lens).to(DEV), sum(lens), page, bt, free)
    k = torch.randn(sum(lens), H, 128, generator=g).half().to(DEV)
    KV.append_kv_slots_i4(data, param, first["slot_map"], k, -k, 0)
    used = sum(-(-n // page) for n in lens)
    left = free[used:used + need[0] + need[1] - 1].clone()
    t = KV.build_page_table(first["seq_lens"], _i32(new).to(DEV), sum(new), page, bt, left)
    # the third needs no page if it stays in its last one, and none is left for it otherwise
    fits = [True, False, need[2] == 0]
    assert t["status"].tolist()[1] == fits.count(False)
    assert t["seq_lens"].tolist() == [n + m * f for n, m, f in zip(lens, new, fits)]
    k = torch.randn(sum(new), H, 128, generator=g).half().to(DEV)
    q = torch.randn(sum(new), H * G, 128, generator=g).half()
    KV.append_kv_slots_i4(data, param, t["slot_map"], k, k, 0)
    o = torch.full(q.shape, float("nan"), dtype=torch.float16, device=DEV)
    KV.chunk_attention_i4(o, q.to(DEV), data, param, t["kv_indptr"], t["kv_indices"], t["last_page_offset"], t["append_indptr"], 0,
                          max_q_len=max(new), positions=t["positions"])
    ref = O.paged_attention(q, data.cpu(), param.cpu(), 0, t["kv_indptr"].cpu(), t["kv_indices"].cpu(), t["last_page_offset"].cpu(),
                            t["append_indptr"].cpu())
    shown = torch.repeat_interleave(torch.tensor(fits), torch.tensor(new))
    _check(o.cpu()[shown], (ref[0][shown], ref[1][shown]))
    assert bool((o.cpu()[~shown] == 0).all())
    assert (t["positions"].cpu() < 0).tolist() == (~shown).tolist()


@pytest.mark.parametrize("window,group", [(None, 1), (None, 2), (20, 1)])
def test_single_tokens_of_a_refused_sequence(window, group):
    s = _setup([40, 17, 33], [1, 1, 1], 2, group, 16, seed=95)
    positions = _i32([39, -1, 32]).to(DEV)
    o = torch.full(s["q"].shape, float("nan"), dtype=torch.float16, device=DEV)
    args = (s["pages"].to(DEV), s["params"].to(DEV), s["indptr"].to(DEV), s["indices"].to(DEV), s["last"].to(DEV), s["layer"])
    KV.batch_decode_i4(o, s["q"].to(DEV), *args, window=window, positions=positions)
    ref = _oracle(s, window or 0)
    _check(o.cpu()[[0, 2]], (ref[0][[0, 2]], ref[1][[0, 2]]))
    assert bool((o[1] == 0).all())
    for bad in (positions[:2], positions.long(), positions.cpu()):
        with pytest.raises(RuntimeError):
            KV.batch_decode_i4(o, s["q"].to(DEV), *args, window=window, positions=bad)


# ------------------------------------------------------------------ workspace
@pytest.mark.parametrize("lens,new,heads,group", [
    ([300] * 64, [1] * 63 + [200], 1, 4), ([600] + [40] * 63, [512] + [1] * 63, 1, 4), ([900] * 20, [300] + [2] * 19, 2, 4),
    ([1000] * 16, [100] + [1] * 15, 2, 8), ([512] + [300] * 63, [512] + [1] * 63, 2, 8), ([300] * 150, [100] + [1] * 149, 8, 1),
    ([2000, 30], [90, 1], 1, 1), ([4000], [128], 2, 2), ([200] * 100, [100] + [1] * 99, 2, 8)])
def test_the_workspace_that_is_asked_for_is_the_one_that_is_used(lens, new, heads, group):
    """The query and the call make the same plan: bytes are written exactly where some were asked for, and not with one byte
    less."""
    s = _setup(lens, new, heads, group, 16, seed=96)
    need = _need(s, max(new))
    work = torch.empty(max(need, 1 << 25), dtype=torch.uint8, device=DEV)
    o = torch.empty_like(s["q"], device=DEV)
    for size, used in ((need, need > 0), (work.numel(), need > 0), (need - 1, False)):
        if size < 0:
            continue
        work.fill_(0xA5)
        assert _raw(s, o, max(new), work[:size]) == 0
        assert bool((work[:max(size, 1)] != 0xA5).any()) == used
        assert bool((work[need:] == 0xA5).all())


def test_the_tcgen05_kernel_uses_the_workspace_that_it_asks_for(request):
    _lib.set_tuning("kv_attend", 2)
    request.addfinalizer(lambda: _lib.set_tuning("kv_attend", 0))
    s = _setup([3000, 100], [40, 70], 1, 4, 16, seed=97)
    need = _need(s, 70)
    assert need > 0
    o = torch.empty_like(s["q"], device=DEV)
    for size in (need, need - 1):
        work = torch.full((need,), 0xA5, dtype=torch.uint8, device=DEV)
        assert _raw(s, o, 70, work[:size]) == 0
        assert bool((work != 0xA5).any()) == (size == need)


# ------------------------------------------------------------------ long contexts
@both_kernels
@pytest.mark.parametrize("lens,new,group,window,sinks", [([70001], [3], 2, 0, 0), ([40000, 66000], [2, 1], 3, 0, 0), ([70001], [9], 1, 65000, 5)])
def test_contexts_of_many_thousand_tokens(lens, new, group, window, sinks):
    s = _setup(lens, new, 1, group, 64, seed=98)
    _check(_attend(s, window, sinks, max_q=max(new)), _oracle(s, window, sinks))


@both_kernels
def test_a_first_token_that_dominates_a_long_context():
    """Its key is the query's direction: all other tokens share what the softmax leaves them."""
    s = _setup([20000], [2], 1, 2, 16, seed=99)
    q = torch.randn(1, 1, 128, generator=torch.Generator().manual_seed(100)).half()
    s["q"] = (q * torch.tensor([1.0, 0.75, 0.5, 0.25]).view(2, 2, 1)).half()
    codes, scale, zero = O.kv_asym_quant_pack(q)
    first = int(s["indices"][0])
    s["pages"][first, 1, 0, :, 0] = codes[0]
    s["params"][first, 1, 0, :, 0] = torch.cat((scale, zero), -1)[0]
    for window, sinks in ((0, 0), (5000, 4)):
        _check(_attend(s, window, sinks, max_q=2), _oracle(s, window, sinks))
