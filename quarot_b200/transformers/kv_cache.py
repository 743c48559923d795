"""Paged 4-bit KV cache behind the upstream name (quarot/transformers/kv_cache.py:130-289).

Same constructor, same `update()` contract and the same memory layout as upstream -- pages
[pages, layers, 2, heads, page_size, head_dim / 2] uint8 with per-(token, head) fp16 (scale, zero) pairs beside them
-- so a model written against `quarot.transformers.MultiLayerPagedKVCache4Bit` runs unchanged.  Underneath, fused
CUDA kernels replace upstream's chain: `qr_kv_append_i4` (Hadamard of the keys over the head dimension, asymmetric
int4 quantisation, packing and the write into the page slot, for prompt and single-token appends alike) and
`qr_kv_decode_i4` (Hadamard of the query, then single-token attention straight from the packed pages).

Beyond upstream: `build_page_table` (page table and slot map from request lengths, on the GPU), `append_kv_slots_i4` (the
append that takes that slot map), `chunk_attention_i4` (causal attention of several new tokens per sequence, ragged, with
grouped query heads), and a sliding window with sink tokens for chunks and single tokens.  The cache class uses them for
prompts and chunks, for sequences of different page counts and with `window_size` / `sink_tokens`.

Not built: `disable_quant=True` (the fp16 variant of the cache) raises NotImplementedError.
"""
import functools
import math

import torch

from .. import _lib, _ops
from ..functional.quantization import get_minq_maxq

_lib_c = _lib.lib


def asym_quantize_and_pack_i4(x: torch.Tensor):
    """Per-(token, head) asymmetric int4 codes of x over its last axis, two per byte, with (scale, zero) -- the format of
    the cache, in torch (quarot/transformers/kv_cache.py:10-24).  The CUDA append kernel produces the same bytes."""
    _, maxq = get_minq_maxq(bits=4, sym=False)
    xmax = torch.amax(x, dim=-1, keepdim=True)
    xmin = torch.amin(x, dim=-1, keepdim=True)
    scale = (xmax - xmin).clamp(min=1e-5) / maxq
    zero = -xmin
    q = torch.clamp(torch.round((x + zero) / scale), 0, maxq).to(dtype=torch.uint8)
    return q[..., 0::2] | (q[..., 1::2] << 4), scale, zero


def unpack_i4_and_asym_dequantize(q, scale, zero):
    """Inverse of the above: code * scale - zero (quarot/transformers/kv_cache.py:26-30)."""
    assert q.dtype == torch.uint8
    codes = torch.stack((q & 0x0f, (q >> 4) & 0x0f), dim=-1).view(*q.shape[:-1], q.shape[-1] * 2)
    return codes * scale - zero


def matmul_had_cuda(X, dtype):
    """Walsh-Hadamard transform over the last axis with scale 1/sqrt(n), computed in `dtype` and returned in X's dtype
    (quarot/transformers/kv_cache.py:32-35); one kernel with fp32 arithmetic inside."""
    return _ops.hadamard(X.to(dtype).contiguous(), None, 1).to(X.dtype).view(X.shape)


def _stream(dev):
    return torch.cuda.current_stream(dev).cuda_stream


def append_kv_i4(kv_data, kv_param, kv_indptr, kv_indices, last_page_offset, k, v, layer_idx, seqlen_indptr=None,
                 hadamard_k=True):
    """Quantise the new keys / values k, v (fp16 [tokens, heads, head_dim]) and write them into their page slots.  The
    page table must already describe the sequences WITH the new tokens.  seqlen_indptr [batch + 1] gives the new tokens
    per sequence (a prompt); without it every sequence appends one token.  Stands in for upstream's
    asym_quantize_and_pack_i4 + init_kv_i4 / append_kv_i4 (quarot/transformers/kv_cache.py:38-62)."""
    tokens, heads, head_dim = k.shape
    assert v.shape == k.shape and k.dtype == v.dtype == torch.float16
    assert k.is_contiguous() and v.is_contiguous() and kv_data.is_contiguous() and kv_param.is_contiguous()
    dev = kv_data.device
    with torch.cuda.device(dev):
        _lib.check(_lib_c.qr_kv_append_i4(
            kv_data.data_ptr(), kv_param.data_ptr(), kv_indptr.data_ptr(),
            kv_indices.data_ptr() or kv_indptr.data_ptr(),         # no page at all: not read
            last_page_offset.data_ptr(), k.data_ptr(), v.data_ptr(), seqlen_indptr.data_ptr() if seqlen_indptr is not None else None,
            tokens, last_page_offset.shape[0], kv_data.shape[1], int(layer_idx), heads, kv_data.shape[4], head_dim,
            1 if hadamard_k else 0, _stream(dev)), "append_kv_i4")


def _launch(op, dev, fn, *args):
    """fn(*args, stream) on the current stream of dev.  The calls below are short next to what a device context and a
    stream object cost to make, so the context is entered only where dev is not the current device."""
    if torch.cuda.current_device() == dev.index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    if rc:
        _lib.check(rc, op)


def _check_i32(op, dev, name, t, n):
    if t is None:
        return None
    if t.dtype is not torch.int32 or t.device != dev or not t.is_contiguous():
        raise RuntimeError("%s: %s must be a contiguous int32 tensor on %s" % (op, name, dev))
    if n and t.numel() < n:
        raise RuntimeError("%s: %s has %d entries, %d are needed" % (op, name, t.numel(), n))
    return t.data_ptr()


def _check_pages(op, kv_data, kv_param, layer_idx):
    """Checks of the page pool [pages, layers, 2, heads, page_size, 64] and its parameters; its device and sizes."""
    dev = kv_data.device
    if dev.type != "cuda" or kv_param.device != dev or not kv_data.is_contiguous() or not kv_param.is_contiguous():
        raise RuntimeError("%s: the pages and their parameters must be contiguous tensors on one CUDA device" % op)
    if kv_data.dtype is not torch.uint8 or kv_param.dtype is not torch.float16:
        raise RuntimeError("%s: the pages are uint8 and their parameters fp16" % op)
    shape = kv_data.shape
    if len(shape) != 6 or shape[2] != 2 or kv_param.shape != shape[:5] + (2,):
        raise RuntimeError("%s: pages %s and parameters %s do not belong together" % (op, tuple(shape), tuple(kv_param.shape)))
    if shape[5] != 64:
        raise RuntimeError("%s: head_dim must be 128" % op)
    if not 0 <= layer_idx < shape[1]:
        raise RuntimeError("%s: layer %d of %d" % (op, layer_idx, shape[1]))
    return dev, shape


def _check_rows(op, dev, name, t):
    """[tokens, heads, 128] fp16 on dev, last axis contiguous; address, strides of the other two, shape."""
    shape = t.shape
    if t.dtype is not torch.float16 or t.device != dev or len(shape) != 3 or shape[2] != 128:
        raise RuntimeError("%s: %s must be fp16 [tokens, heads, 128] on %s" % (op, name, dev))
    ts, hs, ds = t.stride()
    ts, hs = ts if shape[0] > 1 else 0, hs if shape[1] > 1 else 0
    at = t.data_ptr()
    if (ds != 1 or ts % 4 or hs % 4 or at % 8) and t.numel():
        raise RuntimeError("%s: %s needs a contiguous last axis, 8-byte alignment and strides that are multiples of 4" % (op, name))
    return at, ts, hs, shape


def build_page_table(seq_lens, new_lens, new_tokens, page_size, block_table=None, free_pages=None, max_blocks=None):
    """Page table and slot map of one step from request lengths, in one launch and without reading anything back.

    seq_lens int32 [batch]: cached tokens before the step; new_lens int32 [batch]: tokens the step adds (None: one each);
    new_tokens: rows of the slot map, at least the sum of new_lens (the batch size is right for None).  block_table int32
    [batch, max_blocks] holds the pages of the sequences; pages that a sequence needs beyond those it holds are taken from
    free_pages (int32, in order) and written into it.  Without free_pages the block table already holds them; without
    block_table page j of sequence b is j * batch + b (the cache below), at most max_blocks per sequence.

    Returns a dict: kv_indptr [batch + 1], kv_indices [batch * max_blocks] (-1 behind the last page), last_page_offset
    [batch] -- the sequences WITH the new tokens -- append_indptr [batch + 1], slot_map int64 [new_tokens], positions
    int32 [new_tokens], seq_lens [batch] after the step, status int32 [2] = (free pages taken, sequences refused).  A
    sequence that does not fit (free list, block table or slot map too short) is refused: it keeps its length and its
    tokens get slot and position -1, which append_kv_slots_i4 skips; append_indptr, which lays out the rows of k, v and q,
    counts them all the same, and the attention is told by `positions` which of its rows they are.  So is one that is longer than its row of the block
    table already, new tokens or not; the row's pages are listed for it.
    """
    op = "build_page_table"
    if seq_lens.dim() != 1 or not seq_lens.is_cuda:
        raise RuntimeError("%s: seq_lens must be a one-dimensional CUDA tensor" % op)
    dev, batch, new_tokens, page_size = seq_lens.device, seq_lens.shape[0], int(new_tokens), int(page_size)
    if block_table is not None:
        if block_table.dim() != 2 or block_table.shape[0] != batch or (max_blocks not in (None, block_table.shape[1])):
            raise RuntimeError("%s: block_table must be [batch, max_blocks]" % op)
        max_blocks = block_table.shape[1]
    elif free_pages is not None or max_blocks is None:
        raise RuntimeError("%s: without a block_table there is no free list, and max_blocks is needed" % op)
    max_blocks = int(max_blocks)
    if new_tokens < 0 or page_size < 1 or max_blocks < 1:
        raise RuntimeError("%s: bad number of new tokens, page size or blocks per sequence" % op)
    seq_p, new_p = _check_i32(op, dev, "seq_lens", seq_lens, batch), _check_i32(op, dev, "new_lens", new_lens, batch)
    table_p, free_p = _check_i32(op, dev, "block_table", block_table, 0), _check_i32(op, dev, "free_pages", free_pages, 0)
    # one allocation for all outputs; the slot map (64-bit) and kv_indices come first, on 16-byte boundaries
    cap, gap = batch * max_blocks, 2 if new_tokens & 1 else 0
    sizes = [2 * new_tokens, cap, batch + 1, batch, batch + 1, new_tokens, batch, 2]
    if gap:
        sizes.insert(1, gap)
    buf = torch.empty(sum(sizes), dtype=torch.int32, device=dev)
    if batch:
        at = buf.data_ptr()
        indices = at + 8 * new_tokens + 4 * gap
        indptr = indices + 4 * cap
        last = indptr + 4 * (batch + 1)
        append = last + 4 * batch
        positions = append + 4 * (batch + 1)
        after = positions + 4 * new_tokens
        _launch(op, dev, _lib_c.qr_kv_page_table, seq_p, new_p, batch, new_tokens, page_size, max_blocks, table_p, free_p or None,
                -1 if free_pages is None else free_pages.numel(), indptr, indices, last, append, at, positions, after,
                after + 4 * batch)
    else:
        buf.zero_()[:2 * new_tokens].fill_(-1)
    parts = buf.split_with_sizes(sizes)
    slots, (indices, indptr, last, append, positions, after, status) = parts[0], parts[-7:]
    if not batch:
        positions.fill_(-1)
    return {"kv_indptr": indptr, "kv_indices": indices, "last_page_offset": last, "append_indptr": append,
            "slot_map": slots.view(torch.int64), "positions": positions, "seq_lens": after, "status": status}


def _as_rows(x):
    """x [tokens, heads, 128] as the slot append takes it: copied where the head dimension is not contiguous or the rows do
    not begin on 8 bytes."""
    ts, hs, ds = x.stride()
    return x if ds == 1 and ts % 4 == 0 and hs % 4 == 0 and x.data_ptr() % 8 == 0 else x.clone(memory_format=torch.contiguous_format)


def append_kv_slots_i4(kv_data, kv_param, slot_map, k, v, layer_idx, hadamard_k=True):
    """append_kv_i4 with the page slots from a slot map (build_page_table): slot_map int64 [tokens], k and v fp16 [tokens,
    heads, 128] (strided views are fine).  Tokens whose slot lies outside the pool, -1 among others, are left out; the other
    slots have to differ."""
    op = "append_kv_slots_i4"
    layer_idx = int(layer_idx)
    dev, (pages, layers, _, heads, page_size, _) = _check_pages(op, kv_data, kv_param, layer_idx)
    k_p, kt, kh, shape = _check_rows(op, dev, "k", k)
    v_p, vt, vh, v_shape = _check_rows(op, dev, "v", v)
    tokens = shape[0]
    if shape != v_shape or shape[1] != heads:
        raise RuntimeError("%s: k %s and v %s over %d heads" % (op, tuple(shape), tuple(v_shape), heads))
    if slot_map.dtype is not torch.int64 or slot_map.device != dev or not slot_map.is_contiguous() or slot_map.numel() != tokens:
        raise RuntimeError("%s: slot_map must be contiguous int64 on %s with one entry per token" % (op, dev))
    _launch(op, dev, _lib_c.qr_kv_append_slots_i4, kv_data.data_ptr(), kv_param.data_ptr(), pages, slot_map.data_ptr(), k_p, kt, kh,
            v_p, vt, vh, tokens, layers, layer_idx, heads, page_size, 128, 1 if hadamard_k else 0)


def _attend_i4(op, o, q, kv_data, kv_param, kv_indptr, kv_indices, last_page_offset, qo_indptr, max_q_len, layer_idx, hadamard_q,
               window, sink_tokens):
    layer_idx = int(layer_idx)
    dev, (pages, layers, _, kv_heads, page_size, _) = _check_pages(op, kv_data, kv_param, layer_idx)
    q_p, qt, qh, shape = _check_rows(op, dev, "q", q)
    o_p, ot, oh, o_shape = _check_rows(op, dev, "o", o)
    if o_shape != shape:
        raise RuntimeError("%s: o %s, q %s" % (op, tuple(o_shape), tuple(shape)))
    tokens, heads, _ = shape
    if not ((heads < 2 or oh >= 128) and (tokens < 2 or ot >= 128) and
            (heads < 2 or tokens < 2 or ot >= oh * heads or oh >= ot * tokens)):
        raise RuntimeError("%s: the rows of o overlap" % op)
    if heads == 0 or heads % kv_heads:
        raise RuntimeError("%s: %d query heads over %d KV heads" % (op, heads, kv_heads))
    if window is not None and window < 1 or sink_tokens < 0:
        raise RuntimeError("%s: window must be positive (None: no window), sink_tokens not negative" % op)
    batch = last_page_offset.shape[0]
    window, sink_tokens = min(int(window), 0x7fffffff) if window else 0, min(int(sink_tokens), 0x7fffffff)
    indptr = _check_i32(op, dev, "kv_indptr", kv_indptr, batch + 1)
    indices, entries = _check_i32(op, dev, "kv_indices", kv_indices, 0), kv_indices.numel()      # none at all: not read
    # the shares of CTAs that meet in memory; decode-sized calls have none
    work = None
    if max_q_len * heads > 64 * kv_heads:
        sizes = (entries, page_size, tokens, max_q_len, batch, heads, kv_heads, window, sink_tokens)
        if torch.cuda.current_device() == dev.index:
            nbytes = _lib_c.qr_kv_attend_workspace_bytes(*sizes)
        else:
            with torch.cuda.device(dev):
                nbytes = _lib_c.qr_kv_attend_workspace_bytes(*sizes)
        if nbytes:
            work = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _launch(op, dev, _lib_c.qr_kv_attend_i4, o_p, ot, oh, q_p, qt, qh, kv_data.data_ptr(), kv_param.data_ptr(), pages,
            indptr, indices or indptr, entries,
            _check_i32(op, dev, "last_page_offset", last_page_offset, batch), _check_i32(op, dev, "qo_indptr", qo_indptr, batch + 1),
            tokens, max_q_len, batch, layers, layer_idx, heads, kv_heads, page_size, 128, window, sink_tokens,
            1 if hadamard_q else 0, work.data_ptr() if work is not None else None, work.numel() if work is not None else 0)


def _check_positions(op, q, positions):
    if positions is not None and (positions.dtype is not torch.int32 or positions.device != q.device or positions.shape != q.shape[:1]):
        raise RuntimeError("%s: positions must be int32 on %s with one entry per token" % (op, q.device))


def _clear_refused(o, positions):
    """The rows of tokens that have no place in the cache, by the page table's positions."""
    if positions is not None:
        o.masked_fill_((positions < 0).view(-1, 1, 1), 0)


def chunk_attention_i4(o, q, kv_data, kv_param, kv_indptr, kv_indices, last_page_offset, qo_indptr, layer_idx, max_q_len=None,
                       hadamard_q=False, window=None, sink_tokens=0, positions=None):
    """Causal attention of several new tokens per sequence over the packed pages, which already hold them.

    q, o fp16 [tokens, heads, 128] (strided views are fine), the new tokens of sequence b in rows qo_indptr[b] ..
    qo_indptr[b + 1]; they are the last of its cached tokens.  heads may be a multiple of the cache's heads: query head h
    reads KV head h // (heads // kv_heads).  window: a token sees itself and the window - 1 tokens before it, and the first
    sink_tokens tokens.  max_q_len: an upper bound of the new tokens of any sequence (default: all of q; a close bound
    makes a better grid).  Rows that see nothing give zeros; rows of o that belong to no sequence stay as they are.
    positions int32 [tokens], as build_page_table gives them: rows with -1, those of refused sequences and of padding behind
    the last one, give zeros.  Without it the new tokens of a refused sequence are taken for the last of its old ones."""
    _check_positions("chunk_attention_i4", q, positions)
    max_q_len = q.shape[0] if max_q_len is None else int(max_q_len)
    if qo_indptr is None:
        raise RuntimeError("chunk_attention_i4: qo_indptr is needed")
    if max_q_len < 1 and q.shape[0]:
        raise RuntimeError("chunk_attention_i4: max_q_len must be positive")
    _attend_i4("chunk_attention_i4", o, q, kv_data, kv_param, kv_indptr, kv_indices, last_page_offset, qo_indptr,
               min(max_q_len, q.shape[0]), layer_idx, hadamard_q, window, sink_tokens)
    _clear_refused(o, positions)


def batch_decode_i4(o, q, kv_data, kv_param, kv_indptr, kv_indices, last_page_offset, layer_idx, hadamard_q=False, window=None,
                    sink_tokens=0, positions=None):
    """o[b, h] = softmax(q[b, h] K^T / sqrt(d)) V over the packed pages, one new token per sequence
    (quarot/transformers/kv_cache.py:64-72); with hadamard_q the query is Hadamard-transformed first.  With a window only
    the last `window` tokens and the first sink_tokens are seen; the query may have a multiple of the cache's heads.
    positions as in chunk_attention_i4.  With a window or shared heads the softmax weights have 11 bits, as chunks have them,
    without these they are fp32."""
    shape = q.shape
    _check_positions("batch_decode_i4", q, positions)
    if window is not None or len(shape) == 3 and shape[1] != kv_data.shape[3]:
        if shape[0] != last_page_offset.shape[0]:
            raise RuntimeError("batch_decode_i4: %d queries for %d sequences" % (shape[0], last_page_offset.shape[0]))
        _attend_i4("batch_decode_i4", o, q, kv_data, kv_param, kv_indptr, kv_indices, last_page_offset, None, 1, layer_idx,
                   hadamard_q, window, sink_tokens)
        return _clear_refused(o, positions)
    batch, heads, head_dim = shape
    assert o.shape == shape and q.dtype == o.dtype == torch.float16 and q.is_contiguous() and o.is_contiguous()
    dev = kv_data.device
    with torch.cuda.device(dev):
        _lib.check(_lib_c.qr_kv_decode_i4(
            o.data_ptr(), q.data_ptr(), kv_data.data_ptr(), kv_param.data_ptr(), kv_indptr.data_ptr(),
            kv_indices.data_ptr() or kv_indptr.data_ptr(),         # no page at all: not read
            last_page_offset.data_ptr(), batch, kv_data.shape[1], int(layer_idx), heads, kv_data.shape[4], head_dim,
            1 if hadamard_q else 0, _stream(dev)), "batch_decode_i4")
    _clear_refused(o, positions)


_TABLE_MOST = 8192                              # sequences that build_page_table takes


def _fixed_page_table(seq_lens, new_lens, new_tokens, page_size, max_blocks):
    """What the cache needs of build_page_table without a block_table, in torch operations: on the CPU, and for more
    sequences than the kernel takes.  seq_lens: lengths WITH the new tokens."""
    batch, dev = seq_lens.shape[0], seq_lens.device
    rows = lambda n: torch.nn.functional.pad(torch.cumsum(n, 0, dtype=torch.int32), (1, 0))  # noqa: E731
    held = seq_lens.clamp(min=0, max=max_blocks * page_size)
    page_cnt = (held + page_size - 1) // page_size
    indptr, append = rows(page_cnt), rows(new_lens)
    total = int(indptr[-1])
    b = torch.repeat_interleave(torch.arange(batch, device=dev), page_cnt.long(), output_size=total)
    indices = ((torch.arange(total, device=dev) - indptr[b]) * batch + b).to(torch.int32)
    i = torch.arange(new_tokens, device=dev, dtype=torch.int32)
    b = torch.searchsorted(append[1:], i, right=True).clamp(max=batch - 1)
    pos = (seq_lens - new_lens)[b].long() + i - append[b]
    slots = ((pos // page_size) * batch + b) * page_size + pos % page_size
    return {"kv_indptr": indptr, "kv_indices": indices, "last_page_offset": (held - (page_cnt - 1).clamp(min=0) * page_size).to(torch.int32),
            "append_indptr": append, "slot_map": torch.where((i < append[-1]) & (seq_lens[b] <= max_blocks * page_size), slots, -1)}


_TABLE_KEYS = ("kv_data", "kv_indptr", "kv_indices", "last_page_offset", "kv_param")


class _AttentionStub(object):
    """What `update()` hands back once the prompt is cached: attention of the new tokens against the cache."""

    def __init__(self, cache_page_size, device, n_layers, disable_quant, hadamard_dtype, window_size=None, sink_tokens=0):
        self.cache_page_size = cache_page_size
        self.n_layers = n_layers
        self.disable_quant = disable_quant
        self.hadamard_dtype = hadamard_dtype
        self.window_size = window_size
        self.sink_tokens = sink_tokens

    def forward(self, q, num_kv_heads, attention_kwargs, layer_idx, chunk=None):
        batch_size, q_len, num_qo_heads, head_dim = q.shape
        table = {k: attention_kwargs[k] for k in _TABLE_KEYS}
        if chunk is None:
            assert q_len == 1
            q = q.reshape(batch_size, num_qo_heads, head_dim).contiguous()
            attn_output = torch.empty_like(q)
            batch_decode_i4(attn_output, q, **table, layer_idx=layer_idx, hadamard_q=self.hadamard_dtype is not None,
                            window=self.window_size, sink_tokens=self.sink_tokens)
            return attn_output.unsqueeze(1)
        added, qo_indptr, keep = chunk
        assert q_len == added
        rows = q.reshape(batch_size * q_len, num_qo_heads, head_dim)
        rows = (rows if keep is None else rows[keep]).contiguous()
        attn_output = torch.empty_like(rows)
        chunk_attention_i4(attn_output, rows, **table, qo_indptr=qo_indptr, layer_idx=layer_idx, max_q_len=q_len,
                           hadamard_q=self.hadamard_dtype is not None, window=self.window_size, sink_tokens=self.sink_tokens)
        if keep is not None:                    # padded positions of the chunk give zeros
            full = attn_output.new_zeros((batch_size * q_len, num_qo_heads, head_dim))
            full[keep] = attn_output
            attn_output = full
        return attn_output.view(batch_size, q_len, num_qo_heads, head_dim)


class MultiLayerPagedKVCache4Bit:
    """window_size / sink_tokens: attention of the cached tokens with a sliding window and a few first tokens that stay
    visible (models trained or run that way); the cache itself keeps every token."""

    def __init__(self, batch_size, page_size, max_seq_len, device, n_layers, num_heads, head_dim,
                 disable_quant=False, hadamard_dtype=torch.float16, window_size=None, sink_tokens=0):
        if disable_quant:
            raise NotImplementedError("MultiLayerPagedKVCache4Bit(disable_quant=True): the fp16 variant of the cache is not built")
        if head_dim != 128:
            raise NotImplementedError("MultiLayerPagedKVCache4Bit: head_dim must be 128 (as in the upstream kernels)")
        if window_size is not None and window_size < 1 or sink_tokens < 0:
            raise ValueError("MultiLayerPagedKVCache4Bit: window_size must be positive (None: no window), sink_tokens not negative")
        self.page_size = page_size
        self.batch_size = batch_size
        max_page_cnt = self.page_cnt_from_length(max_seq_len)
        self.disable_quant = disable_quant
        self.pages = torch.empty((max_page_cnt * batch_size, n_layers, 2, num_heads, page_size, head_dim // 2),
                                 dtype=torch.uint8, device=device)
        self.scales = torch.empty((max_page_cnt * batch_size, n_layers, 2, num_heads, page_size, 2),
                                  dtype=torch.float16, device=device)
        self.max_seq_len = max_seq_len
        self._needs_init = [True] * n_layers
        self.length = 0
        self.device = device
        self.hadamard_dtype = hadamard_dtype
        self._stub = _AttentionStub(self.page_size, device, n_layers, disable_quant=self.disable_quant,
                                    hadamard_dtype=self.hadamard_dtype, window_size=window_size, sink_tokens=sink_tokens)

    def page_cnt_from_length(self, length):
        return (length + self.page_size - 1) // self.page_size

    def _ensure_page_cnt_per_batch(self, expected_page_cnt_per_batch):
        if expected_page_cnt_per_batch * self.batch_size <= self.pages.shape[0]:
            return
        raise NotImplementedError

    @property
    def seen_tokens(self):
        return self.length

    def update(self, key_states, value_states, layer_idx, cache_kwargs=None):
        """First call per layer (the prompt): caches the keys / values and returns them unchanged, for the caller's own
        prefill attention.  Later calls: cache one token per sequence, or a chunk of them, and return a callable that maps
        the query [batch, tokens, heads, head_dim] to the attention output against the cache.  cache_kwargs may hold an
        attention_mask [batch, cached + new tokens]; sequences may then differ in length by more than a page, and a new
        token that it hides is not cached and gives zeros."""
        b_sz, added_length, num_heads, head_dim = key_states.shape
        assert b_sz == self.batch_size
        attention_mask = (cache_kwargs or {}).get("attention_mask")
        if layer_idx == 0:
            new_length = self.length + added_length
            self._ensure_page_cnt_per_batch(self.page_cnt_from_length(new_length))
            self.length = new_length
        had = self.hadamard_dtype is not None
        k = key_states.reshape(b_sz * added_length, num_heads, head_dim)
        v = value_states.reshape(b_sz * added_length, num_heads, head_dim)
        shown = None
        if attention_mask is not None:
            if 0 < self.length < attention_mask.shape[-1]:          # wider than the tokens so far: the last of these are the new ones
                attention_mask = attention_mask[:, :self.length]
            shown = attention_mask[:, -added_length:]
        if not self._needs_init[layer_idx] and added_length == 1:
            # a sequence whose token the mask hides is empty in the table of this step: nothing is written, and its row is zero
            specs = self._page_table(attention_mask, only=shown)[0]
            append_kv_i4(specs["kv_data"], specs["kv_param"], specs["kv_indptr"], specs["kv_indices"],
                         specs["last_page_offset"], k.contiguous(), v.contiguous(), layer_idx, hadamard_k=had)
            return functools.partial(self._stub.forward, num_kv_heads=num_heads, attention_kwargs=specs, layer_idx=layer_idx)
        if shown is not None:
            new_lens = shown.sum(dim=-1, dtype=torch.int32)
        else:
            new_lens = torch.full((b_sz,), added_length, dtype=torch.int32, device=self.device)
        specs, table = self._page_table(attention_mask, new_lens, b_sz * added_length)
        slots = table["slot_map"]
        if shown is not None:
            # the map holds the tokens that the mask shows one behind the other; the others are not cached
            at = table["append_indptr"][:-1, None] + torch.cumsum(shown, 1, dtype=torch.int32) - 1
            shown = shown.bool().flatten()
            slots = slots.index_select(0, at.clamp(min=0).flatten()).masked_fill(~shown, -1)
        append_kv_slots_i4(self.pages, self.scales, slots, _as_rows(k), _as_rows(v), layer_idx, hadamard_k=had)
        if self._needs_init[layer_idx]:
            self._needs_init[layer_idx] = False
            return key_states, value_states
        return functools.partial(self._stub.forward, num_kv_heads=num_heads, attention_kwargs=specs, layer_idx=layer_idx,
                                 chunk=(added_length, table["append_indptr"], shown))

    def _page_table(self, attention_mask, new_lens=None, new_tokens=0, only=None):
        """Page table of the cached tokens as the kernels take it (sequence b owns pages b, b + batch, b + 2 batch, ...), and
        with it where a step's tokens go, as build_page_table gives it.  new_lens: how many of the tokens the step adds (None:
        none, they are cached already), new_tokens: rows of the slot map.  only [batch, 1]: sequences with a 0 are left empty."""
        if attention_mask is not None:
            seqlens = attention_mask.sum(dim=-1, dtype=torch.int32)
        else:
            seqlens = torch.full((self.batch_size,), self.length, dtype=torch.int32, device=self.device)
        if only is not None:
            seqlens.masked_fill_(only[:, 0] == 0, 0)
        most = self.length if attention_mask is None else max(self.length, attention_mask.shape[-1])
        # a mask may claim more tokens than the pool holds; what is listed lies in the pool
        blocks = max(min(self.page_cnt_from_length(most), self.pages.shape[0] // self.batch_size), 1)
        if new_lens is None:
            new_lens = torch.zeros_like(seqlens)
        if seqlens.is_cuda and self.batch_size <= _TABLE_MOST:
            table = build_page_table(seqlens - new_lens if new_tokens else seqlens, new_lens, new_tokens, self.page_size, max_blocks=blocks)
        else:
            table = _fixed_page_table(seqlens, new_lens, new_tokens, self.page_size, blocks)
        indptr, indices, last = (table[k] for k in ("kv_indptr", "kv_indices", "last_page_offset"))
        if attention_mask is not None:
            indices = indices[:int(indptr[-1])]
        elif self.length == 0:
            indices = indices[:0]
        specs = {
            "kv_data": self.pages,
            "kv_indptr": indptr,
            "kv_indices": indices,
            "last_page_offset": last,
            "kv_param": self.scales,
        }
        return specs, table

    def get_cache_specs_for_flash_infer(self, attention_mask):
        """Page table of the cache as the kernels take it: sequence b owns pages b, b + batch, b + 2 batch, ..."""
        return self._page_table(attention_mask)[0]

    def get_seq_length(self, layer_idx=0):
        return self.length

    def get_max_length(self):
        return None

    def to_legacy_cache(self):
        return self
