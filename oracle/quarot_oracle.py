"""CPU oracle for the quantized-linear path (TEST INFRASTRUCTURE, not product).

This module restates, in plain CPU torch, the arithmetic that the upstream
QuaRot project performs on the path OnlineHadamard -> Quantizer -> Linear4bit.
It exists only so that tests, the smoke check and the CPU-baseline leg of the
benchmark have something independent to compare the CUDA kernels against.
Nothing in the ``quarot_b200`` package imports it, and it never runs on a GPU.

Pinning: every function below is checked bit-for-bit against outputs of the
upstream torch functions (generated by tests/golden/make_golden.py from an
upstream checkout and committed as tests/golden/*.npz).  The two third-party
CUDA libraries upstream calls on this path (CUTLASS int4 GEMM and
fast-hadamard-transform) are not part of the upstream tree; for them the
published mathematics is used (exact integer matmul; Walsh-Hadamard transform
in natural order) and parity at those two boundaries is "unpinned".

Citations are paths inside the upstream project.
"""
import importlib.util
import math
import os

import numpy as np
import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
_TABLES = None


def _tables():
    """Sign tables, read as data from the packed hex module shipped with the package."""
    global _TABLES
    if _TABLES is None:
        path = os.path.join(_HERE, "..", "quarot_b200", "functional", "_had_tables.py")
        spec = importlib.util.spec_from_file_location("_oracle_had_tables", path)
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        out = {}
        for k, hexs in mod.PACKED.items():
            bits = np.unpackbits(np.frombuffer(bytes.fromhex(hexs), dtype=np.uint8))[: k * k]
            out[k] = torch.from_numpy(1.0 - 2.0 * bits.astype(np.float32)).reshape(k, k)
        _TABLES = out
    return _TABLES


# order in which upstream tests divisibility (quarot/functional/hadamard.py:5-55)
_ORDER_PRIORITY = (172, 156, 140, 108, 60, 52, 36, 28, 40, 20, 12)


def is_pow2(n):
    return n > 0 and (n & (n - 1)) == 0


def get_hadK(n, transpose=False):
    """(table, K) for a transform of size n  (quarot/functional/hadamard.py:5-55)."""
    for k in _ORDER_PRIORITY:
        if n % k == 0:
            assert is_pow2(n // k)
            h = _tables()[k]
            return (h.T if transpose else h), k
    assert is_pow2(n)
    return None, 1


def hadamard(x, transpose=False):
    """y = x (hadK (x) H_{n/K})^T / sqrt(n) over the last axis, in x's dtype.

    Follows matmul_hadU (quarot/functional/hadamard.py:58-79): radix-2
    butterflies on the low log2(n/K) index bits, lowest bit first, then the
    dense K x K factor over the major axis, then one division by sqrt(n).
    """
    n = x.shape[-1]
    hk, k = get_hadK(n, transpose)
    m = n // k
    v = x.reshape(-1, k, m).clone()
    rows = v.shape[0]
    stride = 1
    while stride < m:
        # pair element j with j + stride inside each block of 2*stride
        w = v.view(rows, k, m // (2 * stride), 2, stride)
        a = w[:, :, :, 0, :] + w[:, :, :, 1, :]
        b = w[:, :, :, 0, :] - w[:, :, :, 1, :]
        v = torch.stack((a, b), dim=3).reshape(rows, k, m)
        stride *= 2
    if k > 1:
        v = hk.view(1, k, k).to(v) @ v
    return v.reshape(x.shape) / torch.tensor(n).sqrt()


def quantizer_scales(y, clip=1.0):
    """Per-token scale of Quantizer.forward (quarot/nn/quantization.py:10), flat [rows]."""
    y2 = y.reshape(-1, y.shape[-1])
    return ((torch.max(torch.abs(y2), dim=-1)[0] / 7).to(torch.float16) * clip).to(torch.float16)


def sym_quant_codes(y, scale, maxq=7):
    """Integer codes clamp(round(y / s), -8, 7) (quarot/functional/quantization.py:29-32).

    y fp16 [rows, cols], scale fp16 [rows]; the division and rounding are done
    by torch in fp16 (fp32 divide, round to fp16, then round-half-even).
    With a zero scale torch evaluates x / 0: 0 / 0 = NaN is mapped to code 0 and
    +-inf saturates to 7 / -8 (the upstream CUDA kernel does the same through
    __hdiv and a clamped __half2int_rn, quarot/kernels/quant.cu:36-38).
    """
    s = scale.reshape(-1, 1)
    q = torch.clamp(torch.round(y / s), -(maxq + 1), maxq)
    q = torch.nan_to_num(q, nan=0.0, posinf=float(maxq), neginf=float(-(maxq + 1)))
    return q.to(torch.int8)


def pack_i4(q):
    """Two signed nibbles per byte, even index in the low nibble
    (quarot/functional/quantization.py:42-49)."""
    assert q.dtype in (torch.int8, torch.int16, torch.int32, torch.int64)
    assert int(q.min()) >= -8 and int(q.max()) <= 7
    u = (q.to(torch.int16) & 0xF).to(torch.uint8)
    if u.shape[-1] % 2:
        u = torch.cat((u, torch.zeros_like(u[..., :1])), dim=-1)
    return u[..., 0::2] | (u[..., 1::2] << 4)


def unpack_i4(p):
    """Inverse of pack_i4, sign-extended to int32 (quarot/functional/quantization.py:52-74)."""
    assert p.dtype == torch.uint8
    lo = (p & 0xF).to(torch.int32)
    hi = (p >> 4).to(torch.int32)
    lo = lo - 16 * (lo >= 8).to(torch.int32)
    hi = hi - 16 * (hi >= 8).to(torch.int32)
    return torch.stack((lo, hi), dim=-1).reshape(*p.shape[:-1], p.shape[-1] * 2)


def matmul_i4(a_packed, b_packed, via="float64"):
    """int32 C[M,N] = unpack(A)[M,K] . unpack(B)[N,K]^T, exact
    (the identity stated in quarot/kernels/bindings.cpp:386-390; upstream runs
    it through a CUTLASS int4 GEMM, quarot/kernels/gemm.cu:7-46).

    via="float64": float64 BLAS, exact here because |C| <= 64 K < 2^53 (fast).
    via="int32":   torch's integer matmul on the unpacked int32 tensors, the literal
                   form of the identity (slow; used when timing the CPU baseline).
    """
    a = unpack_i4(a_packed.reshape(-1, a_packed.shape[-1]))
    b = unpack_i4(b_packed.reshape(-1, b_packed.shape[-1]))
    if via == "int32":
        return a @ b.T
    return (a.to(torch.float64) @ b.to(torch.float64).T).to(torch.int32)


def sym_dequant_fp16(acc, scale_row, scale_col):
    """Upstream kernel arithmetic, all in fp16: s_row * s_col * half(acc)
    (quarot/kernels/quant.cu:64-81)."""
    r = scale_row.reshape(-1, 1).to(torch.float16)
    c = scale_col.reshape(1, -1).to(torch.float16)
    return (r * c) * acc.to(torch.float16)


def sym_dequant_fp32(acc, scale_row, scale_col):
    """fp32 statement of the same product: float(acc) * (s_row * s_col).  The product of
    two fp16 scales is exact in fp32, so this is the real product rounded once to fp32
    (the accuracy target for the fused epilogue)."""
    sc = scale_row.reshape(-1, 1).float() * scale_col.reshape(1, -1).float()
    return acc.to(torch.float32) * sc


def linear4bit_forward(x, w_packed, w_scales, hadamard_dim=0, clip=1.0, bias=None):
    """Whole path on CPU: optional online Hadamard (fp16 in/out, fp16 internal as
    OnlineHadamard(force_fp32=False) or see `hadamard`), Quantizer, int4 matmul,
    fp32 dequant.  Returns dict of every intermediate."""
    x2 = x.reshape(-1, x.shape[-1])
    if hadamard_dim:
        y = hadamard(x2.float()).to(torch.float16)
    else:
        y = x2
    s = quantizer_scales(y, clip)
    q = sym_quant_codes(y, s)
    qp = pack_i4(q)
    acc = matmul_i4(qp, w_packed)
    out = sym_dequant_fp32(acc, s, w_scales)
    if bias is not None:
        out = out + bias.float()
    return {"y": y, "scales": s, "codes": q, "packed": qp, "acc": acc, "out": out}


def swiglu_fp16(gate, up):
    """act_fn(gate_proj(x)) * up_proj(x) of the LLaMA MLP that upstream subclasses
    (e2e/quantized_llama/modeling_llama.py:105-119; HF LlamaMLP with act_fn = SiLU) on fp16 tensors:
    SiLU evaluated in fp32 and rounded to fp16, then the product rounded to fp16."""
    act = torch.nn.functional.silu(gate.float()).to(torch.float16)
    return (act.float() * up.float()).to(torch.float16)


def rmsnorm_fp16(x, mean_dim, eps=1e-5):
    """Weight-less RMSNorm of the reference (quarot/nn/normalization.py:15-21): fp32 arithmetic, fp16 result."""
    xf = x.float()
    variance = xf.pow(2).sum(-1, keepdim=True) / mean_dim
    return (xf * torch.rsqrt(variance + eps)).to(x.dtype)



# ------------------------------------------------------------------ paged 4-bit KV cache
def kv_asym_quant_pack(x):
    """Asymmetric per-(token, head) int4 quantisation of keys / values over the head dimension and nibble packing
    (quarot/transformers/kv_cache.py:10-24): scale = clamp(max - min, 1e-5) / 15, zero = -min, code =
    clamp(round((x + zero) / scale), 0, 15); every step is a torch op on fp16 tensors (fp32 arithmetic, rounded to
    fp16 after each op).  Returns (packed uint8 [..., d/2], scale [..., 1], zero [..., 1])."""
    xmax = torch.amax(x, dim=-1, keepdim=True)
    xmin = torch.amin(x, dim=-1, keepdim=True)
    scale = (xmax - xmin).clamp(min=1e-5) / torch.tensor(15)
    zero = -xmin
    q = torch.clamp(torch.round((x + zero) / scale), 0, torch.tensor(15)).to(torch.uint8)
    return q[..., 0::2] | (q[..., 1::2] << 4), scale, zero


def kv_unpack_dequant(q, scale, zero):
    """code * scale - zero in the dtype of scale (quarot/transformers/kv_cache.py:26-30)."""
    assert q.dtype == torch.uint8
    codes = torch.stack((q & 0x0F, (q >> 4) & 0x0F), dim=-1).view(*q.shape[:-1], q.shape[-1] * 2)
    return codes * scale - zero


def kv_hadamard(x):
    """Walsh-Hadamard transform over the head dimension with scale 1/sqrt(n), as matmul_had_cuda applies it to keys
    and queries (quarot/transformers/kv_cache.py:32-35); fp32 here, the caller rounds."""
    return hadamard(x.float())


def paged_kv_dense(pages, params, layer, kv_indptr, kv_indices, last_page_offset, b):
    """Dequantised keys and values of sequence b as fp32 [seq_len, heads, head_dim], gathered from the paged layout
    [page, layer, k|v, head, slot, head_dim/2] (+ [.., slot, 2] = (scale, zero)) of
    quarot/kernels/include/flashinfer/page.cuh:76-103; dequantisation as decode.cuh does it through
    quantization.cuh:60-84: float(code) * scale - zero in fp32."""
    page_size = pages.shape[4]
    first, last = int(kv_indptr[b]), int(kv_indptr[b + 1])
    ks, vs = [], []
    for it in range(first, last):
        pg = int(kv_indices[it])
        valid = int(last_page_offset[b]) if it == last - 1 else page_size
        for which, dst in ((0, ks), (1, vs)):
            data = pages[pg, layer, which, :, :valid]                        # [heads, valid, d/2]
            par = params[pg, layer, which, :, :valid].float()                 # [heads, valid, 2]
            codes = torch.stack((data & 0x0F, (data >> 4) & 0x0F), dim=-1).reshape(*data.shape[:-1], -1).float()
            dst.append((codes * par[..., 0:1] - par[..., 1:2]).permute(1, 0, 2))
    return torch.cat(ks, 0), torch.cat(vs, 0)


def paged_decode_attention(q, pages, params, layer, kv_indptr, kv_indices, last_page_offset):
    """softmax(q K^T / sqrt(d)) V over the paged cache for one new token per sequence (the computation of
    BatchDecodeWithPagedKVCacheKernel, quarot/kernels/include/flashinfer/decode.cuh:492, no rotary embedding), in
    fp32.  q fp16/fp32 [batch, heads, head_dim] -> fp32 [batch, heads, head_dim]."""
    outs = []
    d = q.shape[-1]
    for b in range(q.shape[0]):
        k, v = paged_kv_dense(pages, params, layer, kv_indptr, kv_indices, last_page_offset, b)
        s = torch.einsum("hd,thd->ht", q[b].float(), k) / math.sqrt(d)
        p = torch.softmax(s, dim=-1)
        outs.append(torch.einsum("ht,thd->hd", p, v))
    return torch.stack(outs, 0)


def kv_hadamard_fp16(x):
    """The rotated query as the kernels hold it: Walsh-Hadamard butterflies over 128 values in fp32 with the strides 1, 2,
    4 .. 64, times fp32(1 / sqrt(128)), rounded to fp16.  Sums and differences of fp32 numbers, so it is exact to the bit."""
    y = x.float()
    n, h = x.shape[-1], 1
    while h < n:
        y = y.view(*x.shape[:-1], n // (2 * h), 2, h)
        y = torch.stack((y[..., 0, :] + y[..., 1, :], y[..., 0, :] - y[..., 1, :]), -2).reshape(x.shape)
        h *= 2
    return (y * torch.tensor(0.08838834764831845, dtype=torch.float32)).half()


def kv_page_table(seq_lens, new_lens, new_tokens, page_size, block_table=None, free_pages=None, max_blocks=None):
    """Page table and slot map of a step, sequence by sequence (lists in, dict of lists out; block_table is updated)."""
    batch = len(seq_lens)
    width = len(block_table[0]) if block_table is not None else max_blocks
    pages = lambda n: -(-n // page_size)  # noqa: E731
    out = dict(kv_indptr=[0], kv_indices=[], last_page_offset=[], append_indptr=[0], seq_lens=[],
               slot_map=[-1] * new_tokens, positions=[-1] * new_tokens)
    wanted = taken = refused = 0
    for b in range(batch):
        old, new = min(max(seq_lens[b], 0), width * page_size), max(new_lens[b], 0)
        over = seq_lens[b] > width * page_size                 # longer than its row: refused, all of the row listed
        row = out["append_indptr"][-1]
        out["append_indptr"].append(row + new)
        ok = not over and (new == 0 or (pages(old + new) <= width and row + new <= new_tokens))
        if ok and block_table is not None and free_pages is not None:
            need = pages(old + new) - pages(old)
            first = wanted
            wanted += need
            if need and wanted > len(free_pages):
                ok = False
            else:
                block_table[b][pages(old):pages(old) + need] = free_pages[first:first + need]
                taken += need
        refused += not ok
        after = old + new if ok else old
        mine = [block_table[b][j] if block_table is not None else j * batch + b for j in range(pages(after))]
        out["kv_indices"] += mine
        out["kv_indptr"].append(len(out["kv_indices"]))
        out["seq_lens"].append(seq_lens[b] if over else after)
        out["last_page_offset"].append(after - max(len(mine) - 1, 0) * page_size)
        for i in range(new if ok else 0):
            pos = old + i
            slot = mine[pos // page_size] * page_size + pos % page_size
            out["slot_map"][row + i], out["positions"][row + i] = max(slot, -1), pos
    out["kv_indices"] += [-1] * (batch * width - len(out["kv_indices"]))
    out["status"] = [taken, refused]
    return out


def paged_attention(q, pages, params, layer, kv_indptr, kv_indices, last_page_offset, qo_indptr, window=0, sinks=0):
    """Causal attention of the last new tokens of every sequence over the paged cache, in fp64, row by row of the
    definition; query head h reads KV head h // group, window > 0: only the last `window` tokens and the first `sinks`.

    q [tokens, heads, d] -> (o fp64 [tokens, heads, d], bound fp64): |result - o| <= bound holds for an evaluation that
      * rounds the result to fp16 (2^-11 |o|, 2^-25 below the normal numbers),
      * rounds weights to fp16, relative to the largest of them: 2^-11 for each (2^-25 of the largest where that is more).
        Either the weights p_t s_t (softmax times value scale), and only in front of the product with the codes c - 7.5:
        a change d of weight t moves the result by d (c_t - 7.5).  Or the weights p_t g_t (g_t the scale brought to
        [1, 2), for scales above 2^12 s_t / 2^11), in front of all sums, the denominator among them: with p_t + d_t for p_t,
          sum (p_t + d_t) v_t / sum (p_t + d_t) - o = sum d_t (v_t - o) / (1 + sum d_t),
        |d_t| <= max(2^-11 p_t, 2^-25 max(p g) / g_t); weights cut to 11 bits, p_t (1 - c_t) with 0 <= c_t < 2^-10, are
        (1 - 2^-11) p_t (1 + d_t / p_t) with |d_t| <= 2^-11 (1 + 2^-10) p_t, and the common factor drops out.  What such an
        evaluation rounds once more, below 2^-14 of the largest, meets c - 7.5 with 2^-25 of the largest.  The larger of the two,
      * has scores that are off by at most e_t = 2^-19 (31 |s_t| sum|q| + |z_t| |sum q|) / sqrt(d): products of a query with
        codes 16 + c <= 31 summed in fp32 (128 terms and the corrections, each off by 2^-23 of the sum of magnitudes at
        most), which changes weight t by the factor exp(e_t): sum p_t (exp(e_t) - 1) |v_t - o|, twice for the denominator's
        own change,
      * sums and joins everything else in fp32: 2^-18 of the largest magnitude.
    A row that sees nothing is 0."""
    d, heads = q.shape[-1], q.shape[1]
    page_size, kv_heads = pages.shape[4], pages.shape[3]
    group = heads // kv_heads
    out = torch.zeros(q.shape, dtype=torch.float64)
    bound = torch.zeros(q.shape, dtype=torch.float64)
    for b in range(len(last_page_offset)):
        first, last = int(kv_indptr[b]), int(kv_indptr[b + 1])
        r0, r1 = int(qo_indptr[b]), int(qo_indptr[b + 1])
        n = (last - first - 1) * page_size + int(last_page_offset[b]) if last > first else 0
        if n <= 0 or r1 <= r0:
            continue
        mine = kv_indices[first:last].long()
        pos = torch.arange(n - (r1 - r0), n).view(-1, 1)
        t = torch.arange(n).view(1, -1)
        see = t <= pos
        if window > 0:
            see &= (t > pos - window) | (t < sinks)
        for h in range(kv_heads):
            kv, codes, par = [], [], []
            for which in (0, 1):
                data = pages[mine, layer, which, h].reshape(-1, d // 2)[:n]
                pr = params[mine, layer, which, h].reshape(-1, 2)[:n].double()
                cc = torch.stack((data & 0x0F, data >> 4), -1).reshape(n, d).double()
                codes.append(cc)
                par.append(pr)
                kv.append(cc * pr[:, :1] - pr[:, 1:])
            for e in range(h * group, (h + 1) * group):
                qq = q[r0:r1, e].double()
                for i in range(r1 - r0):
                    vis = see[i]
                    if not bool(vis.any()):
                        continue
                    k, v, s = kv[0][vis], kv[1][vis], par[1][vis, :1]
                    sc = (k @ qq[i]) / math.sqrt(d)
                    p = torch.exp(sc - sc.max())
                    p = p / p.sum()
                    o = p @ v
                    out[r0 + i, e] = o
                    kp = par[0][vis]
                    es = (2.0 ** -19 * (31 * kp[:, 0].abs() * qq[i].abs().sum() + kp[:, 1].abs() * qq[i].sum().abs()) / math.sqrt(d))
                    w = p[:, None] * s
                    off = (codes[1][vis] - 7.5).abs()
                    rounding = torch.maximum(2.0 ** -11 * w, 2.0 ** -25 * w.max())
                    sv = s.clamp(min=2.0 ** -22)
                    size = sv / 2.0 ** torch.floor(torch.log2(sv)).clamp(max=11)
                    dp = torch.maximum(2.0 ** -11 * (1 + 2.0 ** -10) * p[:, None], 2.0 ** -25 * (p[:, None] * size).max() / size)
                    moved = (dp * (v - o).abs()).sum(0) / (1 - dp.sum()) + (2.0 ** -25 * w.max() * off).sum(0)
                    bound[r0 + i, e] = ((2.0 ** -11 * o.abs()).clamp(min=2.0 ** -25) + torch.maximum((rounding * off).sum(0), moved)
                                        + 2 * ((p * torch.expm1(es))[:, None] * (v - o).abs()).sum(0) + 2.0 ** -18 * v.abs().max())
    return out, bound
