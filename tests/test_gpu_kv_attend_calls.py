"""How the chunk attention is called: without and with its workspace, in captured graphs, on two streams at once, with
degenerate tables and windows.  Tolerances are the oracle's bounds, as in test_gpu_kv_attend.py."""
import ctypes

import pytest
import torch

from quarot_b200 import _lib
from quarot_b200.transformers import kv_cache as KV
from oracle import quarot_oracle as O
from test_gpu_kv_attend import DEV, _attend, _check, _oracle, _setup, _table, both_kernels, kernel  # noqa: F401

pytestmark = pytest.mark.gpu


def _raw(s, o, max_q, work, window=0, sinks=0, rotate=0):
    """The C entry with an explicit workspace (a tensor, or None)."""
    t, q, rows = _table(s), s["q"].to(DEV), s["rows"].to(DEV)
    pages, layers, _, heads, page, _ = t["kv_data"].shape
    rc = _lib.lib.qr_kv_attend_i4(
        o.data_ptr(), o.stride(0), o.stride(1), q.data_ptr(), q.stride(0), q.stride(1), t["kv_data"].data_ptr(), t["kv_param"].data_ptr(),
        pages, t["kv_indptr"].data_ptr(), t["kv_indices"].data_ptr(), t["kv_indices"].numel(), t["last_page_offset"].data_ptr(), rows.data_ptr(), q.shape[0], max_q,
        len(s["last"]), layers, s["layer"], q.shape[1], heads, page, 128, window, sinks, rotate,
        None if work is None else work.data_ptr(), 0 if work is None else work.numel(), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert _lib.kernel_status() == 0
    return rc


def _need(s, max_q, window=0, sinks=0):
    _, _, _, heads, page, _ = s["pages"].shape
    return _lib.lib.qr_kv_attend_workspace_bytes(s["indices"].numel(), page, s["q"].shape[0], max_q, len(s["last"]), s["q"].shape[1], heads, window, sinks)


# few tiles over long sequences; more sequences than SMs, of which the last few share the SMs (some of their CTAs see nothing)
@pytest.mark.parametrize("lens,new,heads,group,window,pays", [
    ([2500], [100], 1, 1, 0, True),
    ([3000, 100], [40, 70], 1, 4, 2600, True),
    ([60 + 13 * i % 150 for i in range(76)], [20 + i % 3 for i in range(76)], 2, 4, 0, False),
    ([800 + 13 * i % 150 for i in range(76)], [11 + i % 3 for i in range(76)], 2, 7, 0, True),
])
def test_with_and_without_a_workspace(lens, new, heads, group, window, pays, request):
    _lib.set_tuning("kv_attend", 2)
    request.addfinalizer(lambda: _lib.set_tuning("kv_attend", 0))
    s = _setup(lens, new, heads, group, 16, seed=51)
    # the oracle looks at the first KV head
    ref = _oracle(dict(s, q=s["q"][:, :group], pages=s["pages"][:, :, :, :1], params=s["params"][:, :, :, :1]), window)
    most = max(new)
    need = _need(s, most, window)
    assert (need > 0) == pays
    guard = torch.full((need + 256,), 0xA5, dtype=torch.uint8, device=DEV)
    first = None
    for work in (None, guard[:need], guard[:max(need - 1, 0)]):     # a workspace that is too small is not used
        o = torch.full_like(s["q"], float("nan"), device=DEV)
        assert _raw(s, o, most, work, window) == 0
        _check(o[:, :group], ref)
        assert bool((guard[need:] == 0xA5).all())
        if work is None:
            first = o
    assert torch.equal(first, o)
    assert torch.equal(_attend(s, window, max_q=most), _attend(s, window, max_q=most))


@pytest.mark.parametrize("tokens,rows,tc", [(300, 100, False), (300, 1000, False), (60000, 100, True), (6000, 1024, True), (60000, 64, False)])
def test_the_kernel_is_chosen_by_rows_and_length(tokens, rows, tc):
    """One sequence, one group of eight heads on each of eight KV heads: only the tcgen05 kernel has a workspace."""
    need = _lib.lib.qr_kv_attend_workspace_bytes(-(-tokens // 16), 16, rows // 8, rows // 8, 1, 64, 8, 0, 0)
    assert (need > 0) == tc


def test_workspace_size_of_calls_that_need_none():
    f = _lib.lib.qr_kv_attend_workspace_bytes
    assert f(1000, 16, 4, 4, 1, 8, 8, 0, 0) == 0                      # few rows
    for bad in ((-1, 16, 512, 512, 1, 8, 8, 0, 0), (10, 0, 512, 512, 1, 8, 8, 0, 0), (10, 16, 512, 513, 1, 8, 8, 0, 0),
                (10, 16, 512, 512, 1, 9, 8, 0, 0), (10, 16, 512, 512, 1, 8, 0, 0, 0), (10, 16, 512, 512, 1, 8, 8, -1, 0)):
        assert f(*bad) == 0


@both_kernels
@pytest.mark.parametrize("new,group", [([3, 2], 4), ([150, 20], 2)])
def test_captured_and_replayed_with_new_lengths_and_queries(new, group):
    """The lengths are read on the device: the captured call follows the table that it finds at replay."""
    s = _setup([700, 260], new, 2, group, 16, seed=52)
    t = _table(s)
    q, rows, o = s["q"].to(DEV), s["rows"].to(DEV), torch.empty_like(s["q"], device=DEV)

    def call():
        KV.chunk_attention_i4(o, q, **t, qo_indptr=rows, layer_idx=s["layer"], max_q_len=max(new), hadamard_q=True, window=300, sink_tokens=3)

    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        call()
    gen = torch.Generator().manual_seed(53)
    for cut in (0, 5, 17):
        short = dict(s, q=torch.randn(s["q"].shape, generator=gen).half(), last=s["last"].clone())
        # sequence 0 ends `cut` tokens earlier
        whole = 700 - cut
        keep = -(-whole // 16)
        first = int(s["indptr"][1])
        short["indices"] = torch.cat((s["indices"][:keep], s["indices"][first:], s["indices"][keep:first]))
        short["indptr"] = torch.tensor([0, keep, keep + int(s["indptr"][2]) - first], dtype=torch.int32)
        short["last"][0] = whole - (keep - 1) * 16
        q.copy_(short["q"])
        for k, name in (("kv_indptr", "indptr"), ("kv_indices", "indices"), ("last_page_offset", "last")):
            t[k].copy_(short[name])
        o.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert _lib.kernel_status() == 0
        got = o.clone()
        _check(got, _oracle(short, 300, 3, rotate=True))
        call()
        torch.cuda.synchronize()
        assert torch.equal(got, o)


@both_kernels
def test_two_calls_at_once_on_two_streams():
    """Each call has its own shares and its own result; the kernels of both are in flight together."""
    sets = [_setup([2000], [100], 1, 2, 16, seed=54), _setup([1500, 200], [90, 100], 1, 2, 16, seed=55)]
    alone = [_attend(s, max_q=100) for s in sets]
    tables = [(_table(s), s["q"].to(DEV), s["rows"].to(DEV), s["layer"]) for s in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[], []]
    torch.cuda.synchronize()
    for _ in range(10):
        for i, (t, q, rows, layer) in enumerate(tables):
            with torch.cuda.stream(streams[i]):
                o = torch.empty_like(q)
                KV.chunk_attention_i4(o, q, **t, qo_indptr=rows, layer_idx=layer, max_q_len=100)
                outs[i].append(o)
    torch.cuda.synchronize()
    assert _lib.kernel_status() == 0
    for i in range(2):
        assert all(torch.equal(o, alone[i]) for o in outs[i])


@both_kernels
@pytest.mark.parametrize("new", [[9], [90]])
@pytest.mark.parametrize("window", [0, 3, 0x7fffffff])
def test_more_new_tokens_than_cached_ones(new, window):
    """The first rows stand before the sequence: they see nothing, the others see what their positions allow."""
    s = _setup([7], new, 2, 2, 16, seed=56)
    got = _attend(s, window, max_q=new[0])
    _check(got, _oracle(s, window))
    assert bool((got[:new[0] - 7] == 0).all()) and bool((got[new[0] - 7:] != 0).any(-1).all())


@both_kernels
@pytest.mark.parametrize("new", [[2], [80]])
def test_a_last_page_that_says_too_much_ends_with_the_listed_pages(new):
    s = _setup([96], new, 1, 2, 16, seed=57)
    ref = _attend(s, max_q=new[0])
    s["last"] = s["last"] + 1000
    assert torch.equal(ref, _attend(s, max_q=new[0]))


@both_kernels
@pytest.mark.parametrize("new", [[4], [70]])
def test_one_page_listed_several_times(new):
    s = _setup([160], new, 1, 2, 16, seed=58)
    s["indices"] = s["indices"][:1].expand(10).contiguous()
    s["last"] = torch.tensor([16], dtype=torch.int32)
    _check(_attend(s, max_q=new[0]), _oracle(s))


@both_kernels
@pytest.mark.parametrize("new", [[2, 3], [100, 40]])
def test_a_close_or_a_wide_bound_of_the_new_tokens(new):
    s = _setup([400, 300], new, 2, 2, 16, seed=59)
    ref = _oracle(s)
    for most in (max(new), max(new) + 1, sum(new), None):
        _check(_attend(s, max_q=most), ref)


@both_kernels
@pytest.mark.parametrize("new", [[3, 40], [90, 100]])
def test_rows_whose_scores_grow_beyond_the_first_reference(new):
    """Keys that grow along the sequence: the weights' reference moves many times, in every row at other places."""
    s = _setup([900, 500], new, 1, 4, 16, seed=60)
    for b in range(2):
        mine = s["indices"][int(s["indptr"][b]):int(s["indptr"][b + 1])].long()
        grow = torch.exp2(torch.linspace(-6, 3, len(mine))).view(-1, 1, 1, 1)
        pr = s["params"][mine]
        pr[:, s["layer"], 0] = (pr[:, s["layer"], 0].float() * grow).half()
        s["params"][mine] = pr
    for window, sinks in ((0, 0), (250, 4)):
        _check(_attend(s, window, sinks, max_q=max(new)), _oracle(s, window, sinks))


@both_kernels
@pytest.mark.parametrize("size", [2.0 ** -24, 2.0 ** -14, 60000.0])
def test_queries_of_extreme_sizes(size):
    """Tiny, subnormal and huge queries next to ordinary ones: the codes' powers of two are taken back without loss."""
    s = _setup([80, 200], [3, 70], 1, 2, 16, seed=61, scale=1e-3)
    q = s["q"].float() / 8
    q[::2] = (q[::2] * size).clamp(-65504, 65504)
    s["q"] = q.half()
    _check(_attend(s, max_q=70), _oracle(s))
    few = _setup([80], [3], 1, 2, 16, seed=62, scale=1e-3)
    q = few["q"].float() / 8
    q[::2] = (q[::2] * size).clamp(-65504, 65504)
    few["q"] = q.half()
    _check(_attend(few, max_q=3), _oracle(few))


def test_refusals_of_the_c_entry_that_need_a_device():
    s = _setup([200], [100], 1, 1, 16, seed=63)
    o = torch.empty_like(s["q"], device=DEV)
    work = torch.empty(64, dtype=torch.uint8, device=DEV)[8:]
    assert _raw(s, o, 100, work) != 0 and b"16-byte aligned" in ctypes.c_char_p(_lib.lib.qr_last_error()).value


@both_kernels
@pytest.mark.parametrize("batch,heads,group,new", [(33, 32, 1, 1), (64, 16, 4, 3), (65, 16, 1, 2), (40, 16, 1, 70)])
def test_more_sequences_than_one_round_in_any_order_of_lengths(batch, heads, group, new):
    """Sequences are served by length then (up to 64 of them), equal and empty ones among them."""
    g = torch.Generator().manual_seed(64)
    lens = (torch.randint(1, 6, (batch,), generator=g) ** 3 + new).tolist()
    news = [new] * batch
    lens[1], news[1] = 0, 0
    s = _setup(lens, news, heads, group, 16, seed=65)
    few = dict(s)                                                   # the oracle looks at four KV heads
    pick = [0, 1, heads // 2, heads - 1]
    few["pages"], few["params"] = s["pages"][:, :, :, pick], s["params"][:, :, :, pick]
    cols = [h * group + e for h in pick for e in range(group)]
    few["q"] = s["q"][:, cols]
    _check(_attend(s, max_q=new)[:, cols], _oracle(few))


@both_kernels
@pytest.mark.parametrize("new", [[2, 1], [80, 3]])
def test_no_sequence_has_a_page(new):
    s = _setup([0, 0], new, 1, 2, 16, seed=66)
    assert s["indices"].numel() == 0
    assert bool((_attend(s, max_q=max(new)) == 0).all())
