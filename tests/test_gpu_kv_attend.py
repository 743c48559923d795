"""Attention of chunks, of single tokens with a window, and of grouped query heads over the paged 4-bit cache, the page
table from request lengths and the append by slot map, on the GPU against the fp64 oracle.  The tolerance of every element
is the oracle's bound, derived there from the roundings of the evaluation."""
import numpy as np
import pytest
import torch

from quarot_b200 import _lib
from quarot_b200.transformers import MultiLayerPagedKVCache4Bit
from quarot_b200.transformers import kv_cache as KV
from oracle import quarot_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(params=["mma.sync", "tcgen05"])
def kernel(request):
    """Both attention kernels serve every call; which one does is a matter of time."""
    _lib.set_tuning("kv_attend", 1 if request.param == "mma.sync" else 2)
    yield request.param
    _lib.set_tuning("kv_attend", 0)


both_kernels = pytest.mark.usefixtures("kernel")


def _i32(v):
    return torch.tensor(v, dtype=torch.int32)


def _setup(lens, new, kv_heads, group, page, seed, spare=2, scale=1.0, layers=2, layer=1):
    """A cache filled through the oracle's quantiser, pages in random order, everything else of the pool garbage."""
    g = torch.Generator().manual_seed(seed)
    cnt = [-(-n // page) for n in lens]
    total = sum(cnt) + spare
    pages = torch.randint(0, 256, (total, layers, 2, kv_heads, page, 64), generator=g, dtype=torch.uint8)
    params = torch.full((total, layers, 2, kv_heads, page, 2), float("nan"), dtype=torch.float16)
    order = torch.randperm(total, generator=g).tolist()
    indices, indptr, last = [], [0], []
    for n, c in zip(lens, cnt):
        mine = [order.pop() for _ in range(c)]
        for which in (0, 1):
            size = torch.exp(0.5 * torch.randn(n, kv_heads, 1, generator=g))
            x = (torch.randn(n, kv_heads, 128, generator=g) * size * scale).half()
            qq, s, z = O.kv_asym_quant_pack(x)
            for j, pg in enumerate(mine):
                m = min(page, n - j * page)
                pages[pg, layer, which, :, :m] = qq[j * page:j * page + m].permute(1, 0, 2)
                params[pg, layer, which, :, :m] = torch.cat((s, z), -1)[j * page:j * page + m].permute(1, 0, 2)
        indices += mine
        indptr.append(len(indices))
        last.append(n - max(c - 1, 0) * page)
    rows = np.cumsum([0] + list(new)).tolist()
    q = (torch.randn(rows[-1], kv_heads * group, 128, generator=g) * 1.5).half()
    return dict(q=q, pages=pages, params=params, indptr=_i32(indptr), indices=_i32(indices), last=_i32(last), rows=_i32(rows), layer=layer)


def _table(s):
    return dict(kv_data=s["pages"].to(DEV), kv_param=s["params"].to(DEV), kv_indptr=s["indptr"].to(DEV),
                kv_indices=s["indices"].to(DEV), last_page_offset=s["last"].to(DEV))


def _attend(s, window=0, sinks=0, rotate=False, decode=False, max_q=None, o=None, q=None):
    q = s["q"].to(DEV) if q is None else q
    o = torch.full(q.shape, float("nan"), dtype=torch.float16, device=DEV) if o is None else o
    if decode:
        KV.batch_decode_i4(o, q, **_table(s), layer_idx=s["layer"], hadamard_q=rotate, window=window or None, sink_tokens=sinks)
    else:
        KV.chunk_attention_i4(o, q, **_table(s), qo_indptr=s["rows"].to(DEV), layer_idx=s["layer"], max_q_len=max_q,
                              hadamard_q=rotate, window=window or None, sink_tokens=sinks)
    torch.cuda.synchronize()
    assert _lib.kernel_status() == 0
    return o


def _oracle(s, window=0, sinks=0, rotate=False):
    q = O.kv_hadamard_fp16(s["q"]) if rotate else s["q"]
    return O.paged_attention(q, s["pages"], s["params"], s["layer"], s["indptr"], s["indices"], s["last"], s["rows"], window, sinks)


def _check(got, ref):
    o, bound = ref
    got = got.cpu().double()
    assert torch.isfinite(got).all()
    over = (got - o).abs() - bound
    assert float(over.max()) <= 0, "off by %g beyond the bound at %s" % (float(over.max()), np.unravel_index(int(over.argmax()), over.shape))


# (cached tokens, new tokens) per sequence, KV heads, group, page size, window, sinks, rotated
CASES = [
    ([1], [1], 1, 1, 16, 0, 0, True),
    ([5], [5], 2, 1, 1, 0, 0, False),
    ([45, 33, 32, 31], [3, 1, 32, 2], 2, 1, 16, 0, 0, True),
    ([130, 7, 200], [2, 7, 1], 1, 8, 16, 0, 0, True),
    ([77, 300], [9, 4], 2, 3, 10, 0, 0, False),
    ([513], [64], 1, 1, 16, 0, 0, True),
    ([260, 129], [130, 128], 1, 2, 64, 0, 0, False),
    ([400], [400], 1, 1, 7, 0, 0, False),
    ([700, 90], [33, 90], 1, 7, 16, 0, 0, True),
    ([700], [40], 2, 4, 16, 100, 4, True),
    ([700, 64], [300, 64], 1, 2, 16, 64, 33, False),
    ([500], [200], 1, 1, 16, 1, 0, False),
    ([500], [200], 1, 1, 16, 1, 1, False),
    ([333, 40], [50, 40], 1, 4, 10, 32, 5, False),
    ([600], [150], 1, 2, 16, 450, 16, True),
    ([600], [5], 1, 8, 16, 10000, 4, False),
    ([900], [700], 1, 1, 100, 200, 0, False),
]


@both_kernels
@pytest.mark.parametrize("lens,new,heads,group,page,window,sinks,rotate", CASES)
def test_chunk_attention_against_the_oracle(lens, new, heads, group, page, window, sinks, rotate):
    s = _setup(lens, new, heads, group, page, seed=sum(lens) + group)
    ref = _oracle(s, window, sinks, rotate)
    _check(_attend(s, window, sinks, rotate, max_q=max(new)), ref)
    _check(_attend(s, window, sinks, rotate), ref)             # without a bound on the chunk lengths


@both_kernels
@pytest.mark.parametrize("lens,heads,group,page,window,sinks,rotate", [
    ([1, 2, 31, 32, 33], 2, 4, 16, 0, 0, True), ([700, 1200, 64], 2, 8, 16, 0, 0, False), ([700, 1200, 64], 2, 1, 16, 500, 4, True),
    ([2000], 1, 16, 16, 0, 0, True), ([2000], 1, 24, 64, 1024, 4, True), ([40, 1], 1, 40, 5, 0, 0, False), ([900, 33], 3, 5, 16, 1, 0, False),
    ([900, 33], 3, 5, 16, 1, 2, False), ([3000, 100, 1], 2, 4, 10, 1000, 40, True), ([300], 4, 1, 16, 301, 0, False),
    ([64, 96, 128], 1, 1, 32, 32, 32, False)])
def test_single_tokens_with_window_and_shared_heads(lens, heads, group, page, window, sinks, rotate):
    s = _setup(lens, [1] * len(lens), heads, group, page, seed=sum(lens))
    ref = _oracle(s, window, sinks, rotate)
    _check(_attend(s, window, sinks, rotate, decode=True), ref)
    _check(_attend(s, window, sinks, rotate, max_q=1), ref)


@both_kernels
def test_values_of_very_different_sizes_and_constant_rows():
    """Tokens whose rows are constant (the smallest scale the quantiser writes, a zero point a million times as large),
    tiny or large stand next to ordinary ones and get their weight and their value."""
    s = _setup([200, 40], [20, 3], 1, 4, 16, seed=5)
    g = torch.Generator().manual_seed(6)
    for t in range(0, 200, 3):
        pg, slot = int(s["indices"][t // 16]), t % 16
        row = [torch.full((1, 1, 128), 5.0), torch.randn(1, 1, 128, generator=g) * 3e-4, torch.randn(1, 1, 128, generator=g) * 200][(t // 3) % 3]
        qq, sc, z = O.kv_asym_quant_pack(row.half())
        for which in (0, 1):
            if which == 0 and (t // 3) % 3 == 2:
                continue                                        # large values, not large keys: those would take all weight
            s["pages"][pg, 1, which, :, slot] = qq[0]
            s["params"][pg, 1, which, :, slot] = torch.cat((sc, z), -1)[0]
    ref = _oracle(s)
    _check(_attend(s, max_q=20), ref)


@both_kernels
@pytest.mark.parametrize("new", [[3, 2], [150, 40]])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 4)])
def test_hidden_infinities_and_nan_do_not_reach_a_row(new, window, sinks):
    """Cached tokens with infinite or NaN parameters poison exactly the rows that see them."""
    s = _setup([200, 120], new, 1, 2, 16, seed=11)
    clean = _oracle(s, window, sinks)
    bad = {0: (60, 199), 1: (119, 30)}
    hit = torch.zeros(s["q"].shape[0], dtype=torch.bool)
    for b, ts in bad.items():
        for i, t in enumerate(ts):
            pg = int(s["indices"][int(s["indptr"][b]) + t // 16])
            s["params"][pg, 1, i % 2, :, t % 16] = float("nan") if b else float("inf")
            n = [200, 120][b]
            for r in range(new[b]):
                pos = n - new[b] + r
                if t <= pos and (not window or t > pos - window or t < sinks):
                    hit[int(s["rows"][b]) + r] = True
    got = _attend(s, window, sinks, max_q=max(new)).cpu()
    assert not torch.isfinite(got[hit]).any()
    assert bool((~hit).any()) == bool(torch.isfinite(got).any())
    keep = ~hit
    if bool(keep.any()):
        _check(got[keep], (clean[0][keep], clean[1][keep]))


@both_kernels
@pytest.mark.parametrize("new", [[2, 0, 3], [200, 0, 90]])
def test_empty_sequences_and_rows_behind_the_last_one(new):
    """Sequences without new tokens, without cached tokens, rows of q beyond the last sequence, and a sequence with more
    rows than cached tokens (its first rows see nothing and give zeros)."""
    s = _setup([60, 17, new[2]], new, 2, 2, 16, seed=3)
    s["last"][0] = 12                                             # four pages: 48 + 12 = 60
    extra = torch.randn(7, 4, 128).half()
    s["q"] = torch.cat((s["q"], extra))
    got = _attend(s, max_q=max(new))
    n = int(s["rows"][-1])
    assert torch.isnan(got[n:]).all()
    ref = _oracle(s)
    _check(got[:n], (ref[0][:n], ref[1][:n]))
    if new[0] > 60:
        assert bool((got[:new[0] - 60] == 0).all())
    empty = _setup([0, 5], [3, 2], 1, 1, 16, seed=4)
    got = _attend(empty, max_q=3).cpu()
    assert bool((got[:3] == 0).all())
    ref = _oracle(empty)
    _check(got[3:], (ref[0][3:], ref[1][3:]))
    s["rows"] = _i32([0, 1, 1, 100000])                           # the last sequence's rows lie beyond q: left out
    got = _attend(s, max_q=max(new)).cpu()
    assert torch.isnan(got[1:]).all() and torch.isfinite(got[0]).all()


@both_kernels
@pytest.mark.parametrize("new", [[3], [140]])
def test_strided_queries_and_outputs(new):
    """q as a column slice of a fused projection, o heads-first, both as [tokens, heads, 128] views; q itself as output."""
    s = _setup([300], new, 2, 4, 16, seed=8)
    ref = _oracle(s)
    n = new[0]
    fused = torch.zeros(n, 8 * 128 + 4 * 128, dtype=torch.float16, device=DEV)
    fused[:, 128:128 + 1024] = s["q"].view(n, -1).to(DEV)
    qv = fused[:, 128:128 + 1024].view(n, 8, 128)
    ov = torch.full((8, n, 128), float("nan"), dtype=torch.float16, device=DEV).transpose(0, 1)
    _check(_attend(s, max_q=n, q=qv, o=ov), ref)
    own = s["q"].to(DEV).clone()
    _check(_attend(s, max_q=n, q=own, o=own), ref)


@both_kernels
def test_offsets_beyond_32_bits():
    """A pool of more than 2^32 bytes whose last pages are used."""
    free = torch.cuda.mem_get_info()[0]
    pages = (1 << 32) // (2 * 8 * 64 * 64) + 64
    if free < 3 * pages * 2 * 8 * 64 * 64:
        pytest.skip("needs about 13 GB")
    small = _setup([500, 130], [60, 1], 8, 2, 64, seed=21, layers=1, layer=0)
    ref = _oracle(small)
    data = torch.zeros((pages, 1, 2, 8, 64, 64), dtype=torch.uint8, device=DEV)
    param = torch.zeros((pages, 1, 2, 8, 64, 2), dtype=torch.float16, device=DEV)
    n = small["pages"].shape[0]
    data[-n:], param[-n:] = small["pages"].to(DEV), small["params"].to(DEV)
    for max_q in (60, None):
        o = torch.empty(61, 16, 128, dtype=torch.float16, device=DEV)
        KV.chunk_attention_i4(o, small["q"].to(DEV), data, param, small["indptr"].to(DEV), (small["indices"] + pages - n).to(DEV),
                              small["last"].to(DEV), small["rows"].to(DEV), 0, max_q_len=max_q)
        _check(o, ref)
    k = torch.randn(3, 8, 128, device=DEV).half()
    slots = torch.tensor([pages * 64 - 1, pages * 64, -1], dtype=torch.int64, device=DEV)
    KV.append_kv_slots_i4(data, param, slots, k, k, 0, hadamard_k=False)
    qq, sc, z = O.kv_asym_quant_pack(k.cpu())
    assert torch.equal(data[-1, 0, 1, :, 63].cpu(), qq[0]) and torch.equal(param[-1, 0, 0, :, 63].cpu(), torch.cat((sc, z), -1)[0])


@both_kernels
def test_another_stream_and_repeated_calls_give_the_same_bits():
    s = _setup([900, 300], [260, 4], 2, 4, 16, seed=31)
    first = _attend(s, max_q=260)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = _attend(s, max_q=260)
    side.synchronize()
    assert torch.equal(first, again) and torch.equal(first, _attend(s, max_q=260))


# ------------------------------------------------------------------ page table
def _run_table(lens, new, tokens, page, table=None, free=None, max_blocks=None):
    dev = lambda v, t=torch.int32: None if v is None else torch.tensor(v, dtype=t, device=DEV)  # noqa: E731
    bt = dev(table)
    got = KV.build_page_table(dev(lens), dev(new), tokens, page, bt, dev(free), max_blocks)
    want_table = [list(r) for r in table] if table is not None else None
    want = O.kv_page_table(lens, new if new is not None else [1] * len(lens), tokens, page, want_table, free, max_blocks)
    assert set(got) == set(want)
    for k in want:
        assert got[k].tolist() == want[k], k
    if table is not None:
        assert bt.tolist() == want_table
    return got


@pytest.mark.parametrize("batch,page,width,free,seed", [(1, 16, 4, 10, 0), (3, 1, 40, 100, 1), (5, 16, 8, 0, 2), (40, 10, 30, 25, 3),
                                                        (200, 16, 64, 4000, 4), (2500, 8, 12, 3000, 5), (8192, 7, 3, 9000, 6)])
def test_page_table_against_the_oracle(batch, page, width, free, seed):
    """Ragged lengths, empty sequences, full rows, free lists that run out in the middle of the batch, padded slot maps."""
    rng = np.random.RandomState(seed)
    lens = rng.randint(0, width * page + 1, batch).tolist()
    new = np.where(rng.rand(batch) < 0.3, 0, rng.randint(1, 2 * page + 2, batch)).tolist()
    pool = rng.permutation(batch * width + free)
    table = pool[:batch * width].reshape(batch, width).tolist()
    spare = pool[batch * width:].tolist()
    for tokens in (sum(new), sum(new) + 13, max(sum(new) // 2, 0)):
        _run_table(lens, new, tokens, page, table, spare)
    _run_table(lens, new, sum(new), page, table)                     # the table holds the pages already
    _run_table(lens, new, sum(new), page, None, None, width)         # fixed ownership
    _run_table(lens, None, batch, page, table, spare)                # one token each


def test_page_table_refuses_and_survives_bad_lengths():
    _run_table([-5, 100, 7], [3, 2, -4], 5, 16, [[1, 2], [3, 4], [5, 6]], [9, 8])
    out = KV.build_page_table(torch.zeros(0, dtype=torch.int32, device=DEV), None, 3, 16, max_blocks=4)
    assert out["kv_indptr"].tolist() == [0] and out["slot_map"].tolist() == [-1] * 3
    lens = torch.tensor([1, 2], dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError):
        KV.build_page_table(lens, None, 2, 16)
    with pytest.raises(RuntimeError):
        KV.build_page_table(lens, None, 2, 0, max_blocks=2)
    with pytest.raises(RuntimeError):
        KV.build_page_table(lens, None, -1, 16, max_blocks=2)
    with pytest.raises(RuntimeError):
        KV.build_page_table(lens.long(), None, 2, 16, max_blocks=2)
    with pytest.raises(RuntimeError):
        KV.build_page_table(lens, None, 2, 16, torch.zeros(3, 2, dtype=torch.int32, device=DEV))
    with pytest.raises(RuntimeError):
        KV.build_page_table(lens, lens[:1], 2, 16, max_blocks=2)
    with pytest.raises(RuntimeError):
        KV.build_page_table(torch.zeros(8193, dtype=torch.int32, device=DEV), None, 8193, 16, max_blocks=2)


def test_attention_and_append_refusals():
    s = _setup([40], [4], 2, 2, 16, seed=1)
    t = _table(s)
    q, rows = s["q"].to(DEV), s["rows"].to(DEV)
    ok = dict(t, qo_indptr=rows, layer_idx=1, max_q_len=4)
    o = torch.empty_like(q)
    bad = [dict(ok, layer_idx=2), dict(ok, window=0), dict(ok, sink_tokens=-1), dict(ok, qo_indptr=None), dict(ok, max_q_len=0),
           dict(ok, qo_indptr=rows.long()), dict(ok, kv_indptr=t["kv_indptr"][:1]), dict(ok, kv_param=t["kv_param"].float()),
           dict(ok, kv_data=t["kv_data"][..., :32].contiguous()), dict(ok, kv_indices=t["kv_indices"].cpu())]
    for kw in bad:
        with pytest.raises(RuntimeError):
            KV.chunk_attention_i4(o, q, **kw)
    for qq, oo in ((q[:, :3], o[:, :3]), (q.float(), o), (q, o[:2]), (q, o[:1].expand(4, 4, 128)), (q[:, :, :64], o[:, :, :64]),
                   (q.transpose(1, 2).contiguous().transpose(1, 2), o), (q.cpu(), o), (q, o.bfloat16())):
        with pytest.raises(RuntimeError):
            KV.chunk_attention_i4(oo, qq, **ok)
    with pytest.raises(RuntimeError):
        KV.batch_decode_i4(o, q, **t, layer_idx=1, window=8)              # four queries, one sequence
    k = torch.zeros(4, 2, 128, dtype=torch.float16, device=DEV)
    slots = torch.full((4,), -1, dtype=torch.int64, device=DEV)
    for sl, kk in ((slots.int(), k), (slots[:3], k), (slots, k[:, :1]), (slots, k.float())):
        with pytest.raises(RuntimeError):
            KV.append_kv_slots_i4(t["kv_data"], t["kv_param"], sl, kk, kk, 1)
    before = t["kv_data"].clone()
    KV.append_kv_slots_i4(t["kv_data"], t["kv_param"], slots, k, k, 1)    # all left out
    assert torch.equal(before, t["kv_data"])


@pytest.mark.parametrize("hadamard", [False, True])
def test_append_by_slot_map_writes_the_bytes_of_the_append_by_table(hadamard):
    """Fixed ownership, ragged prompt: both appends give the same pool; k and v as column slices of one projection."""
    lens, new, page, H = [20, 0, 33], [13, 5, 40], 16, 3
    W = 8
    table = KV.build_page_table(_i32(lens).to(DEV), _i32(new).to(DEV), sum(new), page, max_blocks=W)
    g = torch.Generator().manual_seed(2)
    fused = torch.randn(sum(new), 2 * H * 128 + 64, generator=g).half().to(DEV)
    k, v = fused[:, 64:64 + H * 128].view(-1, H, 128), fused[:, 64 + H * 128:].view(-1, H, 128)
    pools = []
    for by_slots in (True, False):
        data = torch.zeros((3 * W, 2, 2, H, page, 64), dtype=torch.uint8, device=DEV)
        param = torch.zeros((3 * W, 2, 2, H, page, 2), dtype=torch.float16, device=DEV)
        if by_slots:
            KV.append_kv_slots_i4(data, param, table["slot_map"], k, v, 1, hadamard_k=hadamard)
        else:
            KV.append_kv_i4(data, param, table["kv_indptr"], table["kv_indices"], table["last_page_offset"], k.contiguous(), v.contiguous(),
                            1, seqlen_indptr=table["append_indptr"], hadamard_k=hadamard)
        pools.append((data, param))
    assert torch.equal(pools[0][0], pools[1][0]) and torch.equal(pools[0][1], pools[1][1])
    assert int(pools[0][1].abs().sum() > 0)


# ------------------------------------------------------------------ together
def test_serving_steps_in_a_captured_graph():
    """Page table, append and windowed attention of a decode step in one graph: replayed with new lengths and inputs it
    gives what the eager calls give."""
    B, H, G, page, W = 5, 2, 4, 16, 12
    g = torch.Generator().manual_seed(77)
    data = torch.zeros((B * W + 4, 1, 2, H, page, 64), dtype=torch.uint8, device=DEV)
    param = torch.ones((B * W + 4, 1, 2, H, page, 2), dtype=torch.float16, device=DEV)
    free = torch.randperm(B * W + 4, generator=g).to(torch.int32).to(DEV)
    # prompts through the eager path
    lens = [30, 16, 1, 63, 15]
    bt = torch.zeros((B, W), dtype=torch.int32, device=DEV)
    first = KV.build_page_table(torch.zeros(B, dtype=torch.int32, device=DEV), _i32(lens).to(DEV), sum(lens), page, bt, free)
    assert first["status"].tolist()[1] == 0 and first["seq_lens"].tolist() == lens
    used = int(first["status"][0])
    k = torch.randn(sum(lens), H, 128, generator=g).half().to(DEV)
    KV.append_kv_slots_i4(data, param, first["slot_map"], k, -k, 0)
    seq, pool = first["seq_lens"].clone(), free[used:].clone()
    kn, qn = torch.zeros(B, H, 128, dtype=torch.float16, device=DEV), torch.zeros(B, H * G, 128, dtype=torch.float16, device=DEV)
    o = torch.zeros_like(qn)

    def step():
        t = KV.build_page_table(seq, None, B, page, bt, pool)
        KV.append_kv_slots_i4(data, param, t["slot_map"], kn, kn, 0)
        KV.batch_decode_i4(o, qn, data, param, t["kv_indptr"], t["kv_indices"], t["last_page_offset"], 0, hadamard_q=True, window=20, sink_tokens=2)
        return t

    step()                                                          # warm-up (its page entries are written again below)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t = step()
    for i in range(3):
        kn.copy_(torch.randn(B, H, 128, generator=g).half())
        qn.copy_(torch.randn(B, H * G, 128, generator=g).half())
        graph.replay()
        torch.cuda.synchronize()
        got = o.clone()
        ref = O.paged_attention(O.kv_hadamard_fp16(qn.cpu()), data.cpu(), param.cpu(), 0, t["kv_indptr"].cpu(), t["kv_indices"].cpu(),
                                t["last_page_offset"].cpu(), list(range(B + 1)), 20, 2)
        _check(got, ref)
        step()
        assert torch.equal(o, got)
        taken = int(t["status"][0])                                 # the user's program moves on
        seq.copy_(t["seq_lens"].clone())
        pool.copy_(torch.cat((pool[taken:], pool[:taken])).clone())


@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 3)])
def test_cache_prompt_chunks_and_tokens(window, sinks):
    """The cache class: a left-padded prompt whose sequences differ by several pages, a chunk with padding of its own, a full
    chunk, single tokens; grouped query heads; every output against the oracle on the pool."""
    B, H, G, P, L = 3, 2, 4, 16, 2
    cache = MultiLayerPagedKVCache4Bit(B, P, 256, DEV, L, H, 128, window_size=window, sink_tokens=sinks)
    cache.pages.fill_(0xEE)
    cache.scales.fill_(float("nan"))
    g = torch.Generator().manual_seed(9)
    mask = torch.zeros(B, 0, dtype=torch.int64)
    steps = [(70, [70, 20, 3]), (50, [50, 17, 50]), (40, None), (1, None), (1, None)]
    for n, (length, real) in enumerate(steps):
        new = torch.ones(B, length, dtype=torch.int64)
        if real is not None:
            for b, r in enumerate(real):
                new[b, :length - r] = 0
        mask = torch.cat((mask, new), 1)
        k, v = (torch.randn(B, length, H, 128, generator=g).half() for _ in range(2))
        q = torch.randn(B, length, H * G, 128, generator=g).half()
        for layer in range(L):
            r = cache.update((k + layer).half().to(DEV), v.to(DEV), layer, {"attention_mask": mask.to(DEV)})
            if n == 0:
                continue
            got = r(q.to(DEV))
            assert got.shape == q.shape
            specs = cache.get_cache_specs_for_flash_infer(mask.to(DEV))
            keep = new.bool().flatten()
            rows = [0] + torch.cumsum(new.sum(1), 0).tolist()
            qq = O.kv_hadamard_fp16(q.reshape(B * length, H * G, 128)[keep])
            ref = O.paged_attention(qq, cache.pages.cpu(), cache.scales.cpu(), layer, specs["kv_indptr"].cpu(), specs["kv_indices"].cpu(),
                                    specs["last_page_offset"].cpu(), rows, window or 0, sinks)
            flat = got.reshape(B * length, H * G, 128)
            _check(flat[keep.to(DEV)], ref)
            assert bool((flat[~keep.to(DEV)] == 0).all())
    assert cache.get_seq_length() == 162
    # without a mask: equal lengths, a chunk straight after the prompt
    cache = MultiLayerPagedKVCache4Bit(2, P, 128, DEV, 1, H, 128, hadamard_dtype=None, window_size=window, sink_tokens=sinks)
    k, v = (torch.randn(2, 30, H, 128, generator=g).half().to(DEV) for _ in range(2))
    cache.update(k, v, 0, {})
    k, v, q = (torch.randn(2, 45, h, 128, generator=g).half().to(DEV) for h in (H, H, H))
    got = cache.update(k, v, 0)(q)
    specs = cache.get_cache_specs_for_flash_infer(None)
    ref = O.paged_attention(q.cpu().reshape(90, H, 128), cache.pages.cpu(), cache.scales.cpu(), 0, specs["kv_indptr"].cpu(),
                            specs["kv_indices"].cpu(), specs["last_page_offset"].cpu(), [0, 45, 90], window or 0, sinks)
    _check(got.reshape(90, H, 128), ref)
