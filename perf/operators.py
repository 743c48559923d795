"""Cases for the paged 4-bit KV cache operators: page tables and slot maps built from request lengths, attention of a
chunk of new tokens over the cached pages, and attention with a sliding window and sink tokens.

`run` computes them in elementary torch operations (32 bits, rounded once) while `own` is false and through the public
entry points of quarot_b200.transformers.kv_cache while it is true; `exact` is the definition in 64 bits.

Cache layout: pages [pages, layers, 2 (k | v), heads, page_size, 64] uint8, two unsigned 4-bit codes per byte (element 2j
in the low nibble), parameters [pages, layers, 2, heads, page_size, 2] fp16 = (scale, zero), value = code * scale - zero.
Sequence b owns the pages kv_indices[kv_indptr[b] .. kv_indptr[b + 1]), the last one with last_page_offset[b] tokens.
"""
import math
import random

import torch

own = False

D = 128                       # head dimension of the cache
DEV = "cuda"


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of a small batch: every sequence appends one token, few cross into a new page
        dict(name="table_decode_16", op="table", batch=16, page=16, kv_len=2048, new=1, ragged=True),
        # a step of continuous batching: decoding sequences and prompt chunks of up to 512 tokens side by side
        dict(name="table_mixed_256", op="table", batch=256, page=16, kv_len=8192, new=512, ragged=True),
        # a large pool of long sequences, one token each, odd page size
        dict(name="table_pool_2048", op="table", batch=2048, page=10, kv_len=16384, new=1, ragged=True),
        # LLaMA-2-7B heads: the second 512-token piece of a prompt that is fed in chunks, keys and queries rotated
        dict(name="chunk_512_7b", op="attend", batch=1, q_heads=32, kv_heads=32, page=16, q_len=512, kv_len=2560,
             window=0, sinks=0, rotate=True, ragged=False),
        # LLaMA-2-70B heads (eight query heads per KV head): a long chunk over a long context
        dict(name="chunk_2048_70b", op="attend", batch=1, q_heads=64, kv_heads=8, page=16, q_len=2048, kv_len=10240,
             window=0, sinks=0, rotate=True, ragged=False),
        # continuous batching: chunks of 1 to 700 tokens over caches of different lengths in one call
        dict(name="chunk_ragged_8", op="attend", batch=8, q_heads=32, kv_heads=8, page=16, q_len=700, kv_len=5003,
             window=0, sinks=0, rotate=False, ragged=True),
        # a few drafted tokens per sequence checked in one call: bound by reading the cache
        dict(name="chunk_drafts_32x4", op="attend", batch=32, q_heads=64, kv_heads=8, page=16, q_len=4, kv_len=4100,
             window=0, sinks=0, rotate=True, ragged=True),
        # one short chunk at the end of a very long context: few rows, the token axis has to be split
        dict(name="chunk_128_long", op="attend", batch=1, q_heads=32, kv_heads=8, page=64, q_len=128, kv_len=65536,
             window=0, sinks=0, rotate=False, ragged=False),
        # a single sequence decoding with a window: the smallest call, where latency counts
        dict(name="window_decode_1", op="attend", batch=1, q_heads=32, kv_heads=8, page=16, q_len=1, kv_len=8191,
             window=1024, sinks=4, rotate=True, ragged=False),
        # serving batch decoding with a window of 4096 tokens: streams the window out of the cache
        dict(name="window_decode_64", op="attend", batch=64, q_heads=32, kv_heads=8, page=16, q_len=1, kv_len=12000,
             window=4096, sinks=4, rotate=True, ragged=True),
        # the same without shared heads, an odd window and page size
        dict(name="window_decode_mha", op="attend", batch=16, q_heads=32, kv_heads=32, page=10, q_len=1, kv_len=4999,
             window=2001, sinks=5, rotate=False, ragged=True),
        # a prompt chunk with a window over a long cache: most of the cache is not visible
        dict(name="window_chunk_2048", op="attend", batch=1, q_heads=32, kv_heads=8, page=16, q_len=2048, kv_len=32768,
             window=4096, sinks=4, rotate=True, ragged=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    page = rng.choice([1, 8, 10, 16, 16, 32, 64, 100])
    if rng.random() < 0.25:
        return dict(op="table", batch=_log(rng, 1, 1500), page=max(page, 8), kv_len=_log(rng, 1, 12000),
                    new=rng.choice([1, 1, _log(rng, 2, 300)]), ragged=rng.random() < 0.8)
    kv_heads = rng.choice([1, 2, 4, 8, 8, 32])
    group = 1 if kv_heads == 32 else rng.choice([1, 2, 3, 4, 7, 8, 8])
    kind = rng.random()
    if kind < 0.35:                                  # single tokens
        batch, q_len = _log(rng, 1, 64), 1
        kv_len = _log(rng, 1, 16000)
    elif kind < 0.55:                                # a few tokens each
        batch, q_len = _log(rng, 1, 32), _log(rng, 2, 16)
        kv_len = q_len + _log(rng, 1, 6000)
    else:                                            # chunks
        batch, q_len = _log(rng, 1, 6), _log(rng, 17, 1200)
        kv_len = q_len + _log(rng, 1, 8000)
    window = rng.choice([0, 0, _log(rng, 1, 5000), _log(rng, 100, 5000)])
    return dict(op="attend", batch=batch, q_heads=kv_heads * group, kv_heads=kv_heads, page=page, q_len=q_len,
                kv_len=kv_len, window=window, sinks=rng.choice([0, 1, 4, 5, 33]) if window else 0,
                rotate=rng.random() < 0.5, ragged=batch > 1 and rng.random() < 0.8)


def _lengths(case):
    """(cached tokens without / with the new ones, new tokens) per sequence: by the case alone, so that `work` knows them."""
    rng = random.Random("%(op)s %(batch)d %(kv_len)d %(page)d" % case)
    new_most = case["new"] if case["op"] == "table" else case["q_len"]
    total, new = [], []
    for b in range(case["batch"]):
        if case["ragged"] and b:
            n = rng.randint(1, new_most)
            if case["op"] == "table" and rng.random() < 0.5:
                n = 1                                # a sequence that decodes next to the chunks
            total.append(rng.randint(max(n, case["kv_len"] // 3), max(n, case["kv_len"])))
        else:
            n = new_most
            total.append(max(n, case["kv_len"]))
        new.append(n)
    return [t - n for t, n in zip(total, new)], total, new


def _visible(total, new, window, sinks):
    """(tokens that some row of the sequence sees, (row, token) pairs) for the last `new` of `total` tokens."""
    pairs = 0
    first = total - new                               # position of the first row
    if not window:
        pairs = new * (first + 1) + new * (new - 1) // 2
        return total, pairs
    for p in range(first, total):
        lo = max(0, p - window + 1)
        pairs += p - lo + 1 + min(sinks, lo)
    lo = max(0, first - window + 1)
    return total - lo + min(sinks, lo), pairs


def work(case):
    old, total, new = _lengths(case)
    if case["op"] == "table":
        pages = [-(-t // case["page"]) for t in total]
        # lengths in, the used part of the block table in; indptr / offsets / lengths, indices (whole), slots and positions out
        cap = case["batch"] * _blocks(case)
        return {"bytes": 8 * case["batch"] + 4 * sum(pages) + 4 * (4 * case["batch"] + 2) + 4 * cap + 12 * sum(new), "flops": 0}
    tokens = pairs = 0
    for t, n in zip(total, new):
        a, b = _visible(t, n, case["window"], case["sinks"])
        tokens, pairs = tokens + a, pairs + b
    rows = sum(new)
    return {"bytes": tokens * case["kv_heads"] * 2 * (D // 2 + 4) + 4 * rows * case["q_heads"] * D,
            "flops": 4 * D * case["q_heads"] * pairs}


# ------------------------------------------------------------------ inputs
def _blocks(case):
    return -(-max(_lengths(case)[1]) // case["page"]) + 1


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _table_state(case, seed):
    """A serving loop's page pool: block table with the pages that the sequences hold, the free pages in the order in which
    they are handed out, and the lengths on the device."""
    old, total, new = _lengths(case)
    ps, B, W = case["page"], case["batch"], _blocks(case)
    g = _gen(seed)
    pool = torch.randperm(B * W, generator=g, device=DEV).to(torch.int32)
    old_t = torch.tensor(old, dtype=torch.int32, device=DEV)
    held = (old_t.long() + ps - 1) // ps
    start = torch.cumsum(held, 0) - held
    col = torch.arange(W, device=DEV)
    flat = (start[:, None] + col).clamp(max=B * W - 1)
    table = torch.where(col < held[:, None], pool[flat], torch.full_like(pool[flat], -1)).contiguous()
    return dict(case=case, seq_lens=old_t, new_lens=torch.tensor(new, dtype=torch.int32, device=DEV), new_tokens=sum(new),
                block_table=table, free_pages=pool[sum(-(-t // ps) for t in old):].clone(), page=ps)


def _quantise(x):
    """Per-(token, head) codes of x [.., 128] fp16 as the cache holds them: scale = max((max - min), 1e-5) / 15, zero = -min,
    every step in fp16."""
    hi, lo = x.amax(-1, keepdim=True), x.amin(-1, keepdim=True)
    scale = (hi - lo).clamp(min=1e-5) / 15
    q = torch.clamp(torch.round((x - lo) / scale), 0, 15).to(torch.uint8)
    return q[..., 0::2] | (q[..., 1::2] << 4), torch.cat((scale, -lo), -1)


def _attend_state(case, seed):
    """A filled cache with its page table, and the new queries: keys and values of roughly normal channels whose size
    varies from token to token, quantised as the cache does it; pages in random order; layer 1 of 2."""
    old, total, new = _lengths(case)
    ps, B, H, G = case["page"], case["batch"], case["kv_heads"], case["q_heads"] // case["kv_heads"]
    g = _gen(seed)
    pages = [-(-t // ps) for t in total]
    n = sum(pages)
    spare = 3
    data = torch.empty((n + spare, 2, 2, H, ps, D // 2), dtype=torch.uint8, device=DEV)
    param = torch.empty((n + spare, 2, 2, H, ps, 2), dtype=torch.float16, device=DEV)
    data[:, 0] = 0x5A                                  # the other layer of the cache
    param[:, 0] = 1.0
    step = max(1, (1 << 27) // (2 * H * ps * D))       # pages at a time
    for a in range(0, n + spare, step):
        m = min(step, n + spare - a)
        size = torch.exp(0.4 * torch.randn((m, 2, H, ps, 1), generator=g, device=DEV))
        x = (torch.randn((m, 2, H, ps, D), generator=g, device=DEV) * size).half()
        data[a:a + m, 1], param[a:a + m, 1] = _quantise(x)
    indptr = [0]
    for c in pages:
        indptr.append(indptr[-1] + c)
    rows = [0]
    for c in new:
        rows.append(rows[-1] + c)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    q = (torch.randn((rows[-1], H * G, D), generator=g, device=DEV) * 1.5).half()
    return dict(case=case, q=q, kv_data=data, kv_param=param, kv_indptr=i32(indptr),
                kv_indices=torch.randperm(n + spare, generator=g, device=DEV)[:n].to(torch.int32),
                last_page_offset=i32([t - (c - 1) * ps for t, c in zip(total, pages)]), qo_indptr=i32(rows),
                layer=1, max_q=max(new), max_kv=max(total))


def prepare(case, seed):
    return _table_state(case, seed) if case["op"] == "table" else _attend_state(case, seed)


# ------------------------------------------------------------------ the plain forms
def _table_plain(s):
    old, new, ps, table, free = s["seq_lens"].long(), s["new_lens"].long(), s["page"], s["block_table"], s["free_pages"]
    B, W = table.shape
    N = s["new_tokens"]
    held = (old + ps - 1) // ps
    want = (old + new + ps - 1) // ps
    need = torch.where(want <= W, want - held, torch.zeros_like(held))
    ends = torch.cumsum(need, 0)
    fits = (want <= W) & ((need == 0) | (ends <= free.numel()))
    after = torch.where(fits, old + new, old)
    pages = torch.where(fits, want, held)
    col = torch.arange(W, device=table.device)
    fresh = (col >= held[:, None]) & (col < pages[:, None])
    if free.numel():
        at = ((ends - need)[:, None] + col - held[:, None]).clamp(0, free.numel() - 1)
        table.copy_(torch.where(fresh, free[at], table))
    zero = torch.zeros(1, dtype=torch.long, device=table.device)
    indptr = torch.cat((zero, torch.cumsum(pages, 0)))
    rows = torch.cat((zero, torch.cumsum(new, 0)))
    i = torch.arange(B * W, device=table.device)
    b = torch.searchsorted(indptr, i, right=True).clamp(max=B) - 1
    indices = torch.where(i < indptr[-1], table[b, (i - indptr[b]).clamp(max=W - 1)], torch.full_like(i, -1, dtype=torch.int32))
    i = torch.arange(N, device=table.device)
    b = (torch.searchsorted(rows, i, right=True) - 1).clamp(max=B - 1)
    pos = old[b] + i - rows[b]
    good = (i < rows[-1]) & fits[b]
    page = table[b, (pos // ps).clamp(max=W - 1)].long()
    slots = torch.where(good, page * ps + pos % ps, torch.full_like(pos, -1))
    pos = torch.where(good, pos, torch.full_like(pos, -1))
    taken = torch.where(fits, need, torch.zeros_like(need)).sum()
    return dict(kv_indptr=indptr.int(), kv_indices=indices, last_page_offset=(after - (pages - 1).clamp(min=0) * ps).int(),
                append_indptr=rows.int(), slot_map=slots, positions=pos.int(), seq_lens=after.int(),
                status=torch.stack((taken, (~fits).sum())).int(), block_table=table)


def _rotate(q):
    """Walsh-Hadamard transform over the last axis, scale 1 / sqrt(128); the rotated query is an fp16 tensor."""
    x = q.reshape(-1, D)
    h = 1
    while h < D:
        x = x.view(-1, D // (2 * h), 2, h)
        x = torch.stack((x[:, :, 0] + x[:, :, 1], x[:, :, 0] - x[:, :, 1]), 2).reshape(-1, D)
        h *= 2
    return (x * D ** -0.5).half().to(q.dtype).view(q.shape)


def _attend_plain(s):
    case, dev = s["case"], s["q"].device
    ps, H, window, sinks = case["page"], case["kv_heads"], case["window"], case["sinks"]
    q = s["q"].float()
    if case["rotate"]:
        q = _rotate(q)
    G = q.shape[1] // H
    indptr, rows = s["kv_indptr"].long(), s["qo_indptr"].long()
    pages, new = indptr[1:] - indptr[:-1], rows[1:] - rows[:-1]
    total = (pages - 1) * ps + s["last_page_offset"].long()
    B, Q = new.shape[0], s["max_q"]
    # positions that any row of the sequence may see: all of them, or the sinks and the window of its rows
    if window and sinks + window + Q - 1 < s["max_kv"]:
        base = (total - new - window + 1).clamp(min=sinks)
        t = torch.cat((torch.arange(sinks, device=dev).expand(B, sinks), base[:, None] + torch.arange(window + Q - 1, device=dev)), 1)
    else:
        t = torch.arange(s["max_kv"], device=dev).expand(B, -1)
    at = t.minimum(total[:, None] - 1)
    page = s["kv_indices"].long()[indptr[:-1, None] + at // ps]
    slot = at % ps

    def values(which):
        codes = s["kv_data"][page, s["layer"], which, :, slot]
        par = s["kv_param"][page, s["layer"], which, :, slot].float()
        codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
        return (codes * par[..., :1] - par[..., 1:]).permute(0, 2, 1, 3)          # [B, H, T, D]

    i = torch.arange(Q, device=dev)
    row = (rows[:-1, None] + i).clamp(max=q.shape[0] - 1)
    qp = q[row].view(B, Q, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, Q * G, D)
    sc = (qp @ values(0).transpose(-1, -2)) * D ** -0.5
    pos = (total - new)[:, None] + i
    see = (t[:, None, :] <= pos[:, :, None]) & (i[:, None] < new[:, None, None])
    if window:
        see &= (t[:, None, :] > pos[:, :, None] - window) | (t[:, None, :] < sinks)
    see = see.repeat_interleave(G, 1)[:, None]
    sc.masked_fill_(~see, float("-inf"))
    top = sc.amax(-1, keepdim=True)
    sc = torch.exp(sc.sub_(torch.where(top == float("-inf"), torch.zeros_like(top), top)))
    out = (sc @ values(1)) / sc.sum(-1, keepdim=True).clamp(min=1e-30)
    out = out.view(B, H, Q, G, D).permute(0, 2, 1, 3, 4).reshape(B, Q, H * G, D)
    b = torch.searchsorted(rows, torch.arange(q.shape[0], device=dev), right=True) - 1
    return out[b, torch.arange(q.shape[0], device=dev) - rows[b]].half()


# ------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    if not own:
        return _table_plain(s) if case["op"] == "table" else _attend_plain(s)
    from quarot_b200.transformers import kv_cache as KV
    if case["op"] == "table":
        return dict(KV.build_page_table(s["seq_lens"], s["new_lens"], s["new_tokens"], s["page"], s["block_table"],
                                        s["free_pages"]), block_table=s["block_table"])
    o = torch.empty_like(s["q"])
    table = (s["kv_data"], s["kv_param"], s["kv_indptr"], s["kv_indices"], s["last_page_offset"])
    window = case["window"] or None
    if s["max_q"] == 1:
        KV.batch_decode_i4(o, s["q"], *table, layer_idx=s["layer"], hadamard_q=case["rotate"], window=window,
                           sink_tokens=case["sinks"])
    else:
        KV.chunk_attention_i4(o, s["q"], *table, qo_indptr=s["qo_indptr"], layer_idx=s["layer"], max_q_len=s["max_q"],
                              hadamard_q=case["rotate"], window=window, sink_tokens=case["sinks"])
    return o


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    """Row by row of the definition, one sequence and KV head at a time; page tables are whole numbers and have no rounding."""
    if case["op"] == "table" or work(case)["flops"] > 1.5e12:
        return None
    s = _attend_state(case, seed)
    ps, H, G = case["page"], case["kv_heads"], case["q_heads"] // case["kv_heads"]
    q = s["q"].double()
    if case["rotate"]:
        order = torch.arange(D, device=DEV)
        bits = order[:, None] & order
        odd = sum((bits >> k) & 1 for k in range(7)) % 2
        q = (q @ (1.0 - 2.0 * odd.double()) / math.sqrt(D)).half().double()
    out = torch.zeros_like(q)
    indptr, rows, last = s["kv_indptr"].tolist(), s["qo_indptr"].tolist(), s["last_page_offset"].tolist()
    for b in range(case["batch"]):
        mine = s["kv_indices"][indptr[b]:indptr[b + 1]].long()
        n = (len(mine) - 1) * ps + last[b]
        m = rows[b + 1] - rows[b]
        p = torch.arange(n - m, n, device=DEV)[:, None]
        t = torch.arange(n, device=DEV)[None, :]
        hidden = t > p
        if case["window"]:
            hidden |= (t <= p - case["window"]) & (t >= case["sinks"])
        for h in range(H):
            kv = []
            for which in (0, 1):
                codes = s["kv_data"][mine, s["layer"], which, h].reshape(-1, D // 2)[:n]
                par = s["kv_param"][mine, s["layer"], which, h].reshape(-1, 2)[:n].double()
                x = torch.empty((n, D), dtype=torch.float64, device=DEV)
                x[:, 0::2] = (codes % 16).double()
                x[:, 1::2] = (codes // 16).double()
                kv.append(x * par[:, :1] - par[:, 1:])
            for e in range(h * G, (h + 1) * G):
                w = (q[rows[b]:rows[b + 1], e] @ kv[0].T / math.sqrt(D)).masked_fill(hidden, float("-inf"))
                out[rows[b]:rows[b + 1], e] = torch.softmax(w, -1) @ kv[1]
    return out
