// Attention over the paged 4-bit cache for many query rows per KV head (chunks of a prompt): both products on the
// 5th-generation tensor cores.  Same operator, masks and layouts as kv_attend_rows.cu.
//
// One CTA takes up to 256 query rows of one (sequence, KV head) -- row = (new token, query head of the group), so a
// group shares the tokens it reads -- as two tiles of 128, and walks over the visible tokens in blocks of 128:
//   S_i = Q_i (16 + Ck)^T          tcgen05.mma 128 x 128 x 128, Q and the key codes in shared memory
//   P_i = softmax weights          S from tensor memory to registers and back as fp16
//   O_i += P_i (Cv - 8)            P from tensor memory, the value codes, transposed, in shared memory
// The tensor cores see the codes, which are exact in fp16, never dequantised keys or values: scales and zero points
// of a token are folded into its column of S and into its weight, as described in kv_attend_rows.cu:
//   score_t = s_t S_t - (z_t + 16 s_t) sum(q),   w_t = exp2(score_t + log2 s'_t - M),
//   l = sum w / s',   y = sum w (z' / s' - 8),   o = (O - y) / l,
// which leaves the fp16 rounding of w as the only one in front of the result's own.  M follows the running maximum in
// steps: it moves (and O is multiplied through, a rare pass over tensor memory) only where a block's maximum is more than
// 2^8 above it, weights are scaled by 2^6, so they stay below 2^14 and the normal fp16 range reaches down to 2^-20.
//
// Warps: two warpgroups make the softmax of one row tile each, so that one works while the tensor cores are on the other's
// tile (S_0, O_0, S_1, O_1 in that order); four warps unpack the next block; one thread issues the MMAs.  A token's
// five numbers are per COLUMN of S, so a thread that owned a whole row would have to read all of them: S is read
// with the 16x256b shape instead, which gives a lane two neighbouring columns of eight in four rows, the numbers of
// a column pair serve four rows, and a row's maximum is two shuffles away.  Unpacking: keys as they stand (two
// logical instructions per pair of codes; the query follows their order), values transposed by byte permutes over
// eight tokens, so that both operands are K-major 128-byte-swizzled tiles written by conflict-free 16-byte stores.
// Few tiles: a cluster shares the token axis and merges through distributed shared memory.
//
// Registers: 512 threads start with 128 each; the softmax warpgroups go up to 192, the unpacking warps down to 88 and the
// MMA warpgroup to 40 (sum 512 x 128).  All waits are bounded (tc_ptx.cuh).
#include "kv_common.cuh"
#include "tc_ptx.cuh"

#include <math.h>

namespace qr {

constexpr int kAtThreads = 512;
constexpr int kAtRows = 256;
constexpr int kAtTok = 128;
constexpr int kAtTile = 128 * 128 * 2;                    // bytes of one 128 x 128 fp16 operand tile
constexpr int kAtPairFloats = 12;                         // per column pair: ks ks kz kz | lv lv rv rv | zv zv - -
constexpr int kAtParStages = 3;
constexpr uint32_t kAtIdesc = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);   // fp16 x fp16 -> fp32, K-major, 128 x 128

struct AtShared {
  float par[kAtParStages][kAtTok / 2][kAtPairFloats];
  long long row[2][kAtTok];                               // rows of the key block of the tokens, -1: not read
  float qsum[kAtRows];
  int pos[kAtRows];
  float m[kAtRows], l[kAtRows];
  unsigned long long bars[32];
  uint32_t tmem;
  int abort;
};
constexpr size_t kAtSmem = 1024 + 6 * kAtTile + sizeof(AtShared);
static_assert(kAtSmem <= 227 * 1024, "shared memory");

__device__ __forceinline__ void umma_f16_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 da, {%1, %3};\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t}"
      ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(kDescHiKmajorSw128), "r"(kAtIdesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}"
      ::"r"(d), "r"(a_tmem), "r"(b_lo), "r"(kDescHiKmajorSw128), "r"(kAtIdesc), "r"(acc) : "memory");
}
// 16 lanes x 64 columns of tensor memory: lane (g, c) gets columns 8 k + 2 c, + 1 of row g in r[4 k], r[4 k + 1] and of row
// g + 8 in r[4 k + 2], r[4 k + 3].  No wait: tmem_ld_done() below.
__device__ __forceinline__ void tmem_ld_16x256_x8(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st_16x256_x8(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x8.b32 [%32], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
      ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]),
        "r"(taddr) : "memory");
}
// 16 lanes x 32 columns of fp16 pairs (64 matrix columns): r[2 k] is row g, r[2 k + 1] row g + 8, column pair 4 k + c.
__device__ __forceinline__ void tmem_st_16x128_x8(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%16], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
      ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(taddr) : "memory");
}
// Waits for the loads of this thread; the registers pass through, so that no use of them moves above the wait.
template <int N>
__device__ __forceinline__ void tmem_ld_done(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; i += 8)
    asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]));
}
__device__ __forceinline__ void tmem_st_done() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
template <int N> __device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// pairs of fp32
__device__ __forceinline__ uint64_t f2_pack(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_unpack(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
template <int J>
__device__ __forceinline__ uint32_t at_centred_pair(uint32_t w) {     // 16 + c - 24, exact
  const uint32_t x = code_pair<J>(w);
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&x), __float2half2_rn(24.0f));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ void st_shared16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// 16-byte chunk of row r, columns 4 chunk .. + 3, in the fp32 merge area [256][128].
__device__ __forceinline__ uint32_t at_part_off(int r, int chunk) { return (uint32_t)(r * 512 + ((chunk ^ ((r & 7) << 1)) << 4)); }

__device__ __forceinline__ __half* at_out_row(const KvAttendParams& p, const KvTile& w, int head_kv, int r) {
  const int row = w.row0 + r;
  const int tok = fast_div(row, p.group_div), hh = row - tok * p.group;
  return p.o + (w.tok0 + tok) * p.o_ts + (int64_t)(head_kv * p.group + hh) * p.o_hs;
}

__global__ void __launch_bounds__(kAtThreads, 1)
kv_attend_tc_kernel(const KvAttendParams p) {
  extern __shared__ unsigned char s_raw[];
  const uint32_t base = (smem_u32(s_raw) + 1023u) & ~1023u;
  unsigned char* smem = s_raw + (base - smem_u32(s_raw));
  // [Q tile 0, Q tile 1][K 2 stages][V 2 stages][AtShared]; the merge area is Q and K, the fp16 result goes through Q
  const uint32_t s_q = base, s_k = base + 2 * kAtTile, s_v = base + 4 * kAtTile;
  AtShared& sh = *reinterpret_cast<AtShared*>(smem + 6 * kAtTile);
  const uint32_t bars = smem_u32(sh.bars);
  const uint32_t k_full = bars, k_empty = bars + 16, v_full = bars + 32, v_empty = bars + 48, par_full = bars + 64, s_full = bars + 88,
                 p_full = bars + 104, o_full = bars + 120;                          // 2, 2, 2, 2, 3, 2, 2, 2
  volatile int* abort_flag = &sh.abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t crank = 0;
  if (p.splits > 1) crank = kv_cluster_rank();
  const int unit = blockIdx.x / p.splits;
  const int head_kv = unit % p.kv_heads;
  // the last tiles of a sequence see the most tokens: they start first
  const KvTile w = kv_find_tile(p, p.max_tiles - 1 - unit / p.kv_heads, kAtRows, lane);
  if (w.rows == 0) return;                                // the whole cluster has the same tile
  const int tiles = w.rows > 128 ? 2 : 1;
  const int p_min = w.pos0 + fast_div(w.row0, p.group_div), p_max = w.pos0 + fast_div(w.row0 + w.rows - 1, p.group_div);
  const KvBlocks blk = kv_blocks<kAtTok>(p_min, p_max, p.window, p.sinks);
  const int per = (blk.count + p.splits - 1) / p.splits;
  const int begin = (int)crank * per;
  const int n = max(min(begin + per, blk.count) - begin, 0);

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(k_full + 8 * s, 4); mbar_init(k_empty + 8 * s, 1);
      mbar_init(v_full + 8 * s, 4); mbar_init(v_empty + 8 * s, 1);
      mbar_init(s_full + 8 * s, 1); mbar_init(p_full + 8 * s, 4); mbar_init(o_full + 8 * s, 1);
    }
    for (int s = 0; s < kAtParStages; ++s) mbar_init(par_full + 8 * s, 4);
    sh.abort = 0;
    fence_mbar_init();
  }
  if (warp == 12) {
    tmem_alloc(smem_u32(&sh.tmem), 512);
    tmem_relinquish();
  }
  // query rows: 8 dimensions 8 i .. 8 i + 7 lie as 0 4 1 5 2 6 3 7, the order in which a word of key codes comes apart
  for (int r = warp; r < 128 * tiles; r += kAtThreads / 32) {
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    int pos = -1;
    if (r < w.rows) {
      const int row = w.row0 + r;
      const int tok = fast_div(row, p.group_div), hh = row - tok * p.group;
      pos = w.pos0 + tok;
      load4_f16(p.q + (w.tok0 + tok) * p.q_ts + (int64_t)(head_kv * p.group + hh) * p.q_hs + 4 * lane, x);
      if (p.hadamard_q) {
        fwht128_warp(x, lane);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __half2float(__float2half_rn(x[e] * 0.08838834764831845f));
      }
    }
    float sum = x[0] + x[1] + x[2] + x[3];
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    const bool odd = lane & 1;
    const float give0 = odd ? x[0] : x[2], give1 = odd ? x[1] : x[3];
    const float got0 = __shfl_xor_sync(0xffffffffu, give0, 1), got1 = __shfl_xor_sync(0xffffffffu, give1, 1);
    const __half2 h0 = odd ? __floats2half2_rn(got0, x[2]) : __floats2half2_rn(x[0], got0);
    const __half2 h1 = odd ? __floats2half2_rn(got1, x[3]) : __floats2half2_rn(x[1], got1);
    const int rr = r & 127, ch = (lane >> 1) & 7;
    unsigned char* dst = smem + (r >> 7) * kAtTile + (lane >> 4) * (kAtTile / 2) + rr * 128 + ((ch ^ (rr & 7)) << 4) + (odd ? 8 : 0);
    uint2 u;
    u.x = *reinterpret_cast<const uint32_t*>(&h0);
    u.y = *reinterpret_cast<const uint32_t*>(&h1);
    *reinterpret_cast<uint2*>(dst) = u;
    if (lane == 0) { sh.qsum[r] = sum; sh.pos[r] = pos; }
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&sh.tmem);

  if (warp < 8) {
    // ---------------------------------------------------------------- softmax of one row tile
    regs_inc<192>();
    const int i = warp >> 2, g = lane >> 2, c = lane & 3;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;                    // first tensor-memory lane of the warp, << 16
    const uint32_t t_s = tmem + i * 128 + lanes, t_o = tmem + 256 + i * 128 + lanes;
    const int row0 = i * 128 + (warp & 3) * 32;                           // the lane's rows: row0 + g + 8 x, x = 0 .. 3
    float m[4], qs[4];
    uint64_t l2[4], y2[4];
    int ps[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      m[x] = -INFINITY;
      l2[x] = 0; y2[x] = 0;
      qs[x] = i < tiles ? sh.qsum[row0 + g + 8 * x] : 0.0f;
      ps[x] = i < tiles ? sh.pos[row0 + g + 8 * x] : -1;
    }
    bool ok = i < tiles;
    for (int j = 0; ok && j < n; ++j) {
      const int t0 = kv_block_index(blk, begin + j) * kAtTok;
      const bool edge = t0 + kAtTok - 1 > p_min || (p.window > 0 && t0 <= p_max - p.window && t0 + kAtTok - 1 >= p.sinks);
      const int ring = j % kAtParStages;
      ok = mbar_wait(par_full + 8 * ring, (j / kAtParStages) & 1, abort_flag, p.status, 71) &&
           mbar_wait(s_full + 8 * i, j & 1, abort_flag, p.status, 72);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      tc_fence_after();
      uint32_t s[2][64];                                  // [rows 0 - 15 / 16 - 31 of the warp][4 k + ..]
      tmem_ld_16x256_x8(t_s, s[0]);
      tmem_ld_16x256_x8(t_s + (16u << 16), s[1]);
      tmem_ld_16x256_x8(t_s + 64, s[0] + 32);
      tmem_ld_16x256_x8(t_s + 64 + (16u << 16), s[1] + 32);
      tmem_ld_done<64>(s[0]);
      tmem_ld_done<64>(s[1]);
      const float* par = &sh.par[ring][c][0];
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const float4 a = *reinterpret_cast<const float4*>(par + 4 * k * kAtPairFloats);
        const float2 b = *reinterpret_cast<const float2*>(par + 4 * k * kAtPairFloats + 4);
        const uint64_t ks = f2_pack(a.x, a.y), kz = f2_pack(a.z, a.w), lv = f2_pack(b.x, b.y);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          uint32_t* r = s[x >> 1] + 4 * k + 2 * (x & 1);
          uint64_t v = f2_fma(kz, f2_pack(qs[x], qs[x]), lv);
          v = f2_fma(ks, f2_pack(__uint_as_float(r[0]), __uint_as_float(r[1])), v);
          float v0, v1;
          f2_unpack(v, v0, v1);
          if (edge) {
            const int t = t0 + 8 * k + 2 * c;
            const int lo = p.window > 0 ? ps[x] - p.window : -1;
            if (t > ps[x] || (t <= lo && t >= p.sinks)) v0 = -INFINITY;
            if (t + 1 > ps[x] || (t + 1 <= lo && t + 1 >= p.sinks)) v1 = -INFINITY;
          }
          top[x] = fmaxf(top[x], fmaxf(v0, v1));
          r[0] = __float_as_uint(v0);
          r[1] = __float_as_uint(v1);
        }
      }
      bool grows = false;
      float mn[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 1));
        top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 2));
        mn[x] = top[x] > m[x] + 8.0f ? top[x] : m[x];
        grows |= mn[x] != m[x];
      }
      if (__any_sync(0xffffffffu, grows)) {
        float f[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          f[x] = mn[x] != m[x] ? ex2(m[x] - mn[x]) : 1.0f;
          m[x] = mn[x];
          const uint64_t ff = f2_pack(f[x], f[x]);
          l2[x] = f2_fma(l2[x], ff, 0);
          y2[x] = f2_fma(y2[x], ff, 0);
        }
        if (j > 0) {                                      // the products of the blocks before are complete: S follows them
#pragma unroll 1
          for (int q4 = 0; q4 < 4; ++q4) {
            uint32_t o[32];
            const uint32_t at = t_o + (q4 >> 1) * 64 + ((uint32_t)(q4 & 1) << 20);
            tmem_ld_16x256_x8(at, o);
            tmem_ld_done<32>(o);
            const float fa = q4 & 1 ? f[2] : f[0], fb = q4 & 1 ? f[3] : f[1];
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * ((e & 2) ? fb : fa));
            tmem_st_16x256_x8(at, o);
          }
          tmem_st_done();
        }
      }
#pragma unroll
      for (int hcol = 0; hcol < 2; ++hcol) {              // 64 columns at a time
        uint32_t pk[2][16];
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          const int k = 8 * hcol + kk;
          const float2 b = *reinterpret_cast<const float2*>(par + 4 * k * kAtPairFloats + 6);
          const float2 d = *reinterpret_cast<const float2*>(par + 4 * k * kAtPairFloats + 8);
          const uint64_t rv = f2_pack(b.x, b.y), zv = f2_pack(d.x, d.y);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            uint32_t* r = s[x >> 1] + 4 * k + 2 * (x & 1);
            const float off = m[x] == -INFINITY ? 0.0f : 6.0f - m[x];
            float v0, v1;
            f2_unpack(f2_add(f2_pack(__uint_as_float(r[0]), __uint_as_float(r[1])), f2_pack(off, off)), v0, v1);
            const float w0 = ex2(v0), w1 = ex2(v1);
            const uint64_t ww = f2_pack(w0, w1);
            if (edge) {
              // a hidden token leaves the sums alone whatever its parameters hold
              const uint64_t rr = f2_pack(w0 != 0.0f ? b.x : 0.0f, w1 != 0.0f ? b.y : 0.0f);
              const uint64_t zz = f2_pack(w0 != 0.0f ? d.x : 0.0f, w1 != 0.0f ? d.y : 0.0f);
              l2[x] = f2_fma(ww, rr, l2[x]);
              y2[x] = f2_fma(ww, zz, y2[x]);
            } else {
              l2[x] = f2_fma(ww, rv, l2[x]);
              y2[x] = f2_fma(ww, zv, y2[x]);
            }
            const __half2 wh = __floats2half2_rn(w0, w1);
            pk[x >> 1][2 * kk + (x & 1)] = *reinterpret_cast<const uint32_t*>(&wh);
          }
        }
        tmem_st_16x128_x8(t_s + 32 * hcol, pk[0]);        // over S, which is in registers
        tmem_st_16x128_x8(t_s + 32 * hcol + (16u << 16), pk[1]);
      }
      tmem_st_done();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full + 8 * i);
    }
    // sums over the four lanes of a row
    float l[4], y[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      float a, b;
      f2_unpack(l2[x], a, b);
      l[x] = a + b;
      f2_unpack(y2[x], a, b);
      y[x] = a + b;
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], d);
        y[x] += __shfl_xor_sync(0xffffffffu, y[x], d);
      }
    }
    if (ok && n > 0) {
      ok = mbar_wait(o_full + 8 * i, 0, abort_flag, p.status, 73);
      ok = __all_sync(0xffffffffu, ok);
    }
    if (ok) {
      tc_fence_after();
#pragma unroll 1
      for (int q4 = 0; q4 < 4; ++q4) {                    // columns 64 (q4 / 2) .., rows 16 (q4 % 2) ..
        uint32_t o[32];
        if (n > 0) {
          tmem_ld_16x256_x8(t_o + (q4 >> 1) * 64 + ((uint32_t)(q4 & 1) << 20), o);
          tmem_ld_done<32>(o);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float ll = q4 & 1 ? l[2 + h] : l[h], yy = q4 & 1 ? y[2 + h] : y[h];
          const int r = row0 + 16 * (q4 & 1) + 8 * h + g;
          const float inv = p.splits > 1 ? 1.0f : (ll != 0.0f ? 1.0f / ll : 0.0f);      // a row that sees nothing gives zeros
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float a = (__uint_as_float(o[4 * k + 2 * h]) - yy) * inv, b = (__uint_as_float(o[4 * k + 2 * h + 1]) - yy) * inv;
            const int col = 64 * (q4 >> 1) + 8 * k + 2 * c;
            if (p.splits > 1) {
              *reinterpret_cast<float2*>(smem + at_part_off(r, col >> 2) + (col & 2) * 4) = make_float2(a, b);
            } else {
              const __half2 hv = __floats2half2_rn(a, b);
              *reinterpret_cast<__half2*>(smem + r * 256 + (((col >> 3) ^ (r & 7)) << 4) + (col & 7) * 2) = hv;
            }
          }
        }
      }
      if (p.splits > 1) {
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if (c == 0) { sh.m[row0 + g + 8 * x] = m[x]; sh.l[row0 + g + 8 * x] = l[x]; }
      } else {
        __syncwarp();
        for (int rr = 0; rr < 32; ++rr) {                 // a row is 256 contiguous bytes
          const int r = row0 + rr;
          if (r >= w.rows) break;
          const uint2 v = *reinterpret_cast<const uint2*>(smem + r * 256 + (((lane >> 1) ^ (r & 7)) << 4) + (lane & 1) * 8);
          *reinterpret_cast<uint2*>(at_out_row(p, w, head_kv, r) + 4 * lane) = v;
        }
      }
    }
    if (p.splits > 1) {
      kv_cluster_barrier();
      // the CTAs of the cluster deal out the rows
      for (int r = (int)crank + p.splits * warp; r < w.rows; r += p.splits * 8) {
        float mm = -INFINITY;
        for (int x = 0; x < p.splits; ++x) mm = fmaxf(mm, kv_peer_f32(kv_peer_addr(&sh.m[r], x)));
        float ll = 0.0f;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int x = 0; x < p.splits; ++x) {
          const float mx = kv_peer_f32(kv_peer_addr(&sh.m[r], x)), lx = kv_peer_f32(kv_peer_addr(&sh.l[r], x));
          if (mx == -INFINITY && lx == 0.0f) continue;
          const float f = ex2(mx - mm);
          const float4 v = kv_peer_f32x4(kv_peer_addr(smem + at_part_off(r, lane), x));
          ll = fmaf(lx, f, ll);
          acc.x = fmaf(v.x, f, acc.x); acc.y = fmaf(v.y, f, acc.y); acc.z = fmaf(v.z, f, acc.z); acc.w = fmaf(v.w, f, acc.w);
        }
        const float inv = ll != 0.0f ? 1.0f / ll : 0.0f;
        const __half2 h0 = __floats2half2_rn(acc.x * inv, acc.y * inv), h1 = __floats2half2_rn(acc.z * inv, acc.w * inv);
        uint2 out;
        out.x = *reinterpret_cast<const uint32_t*>(&h0);
        out.y = *reinterpret_cast<const uint32_t*>(&h1);
        *reinterpret_cast<uint2*>(at_out_row(p, w, head_kv, r) + 4 * lane) = out;
      }
      kv_cluster_barrier();                                  // nobody leaves while its shared memory may still be read
    }
  } else if (warp < 12) {
    // ---------------------------------------------------------------- unpacking of keys, values and parameters
    regs_dec<88>();
    const int tid = threadIdx.x - 256, pw = warp - 8;
    const int first_page = p.indptr[w.b];
    const int tokens = min(p_max + 1, w.seq_len);
    const size_t page_rows = (size_t)p.layers * 2 * p.kv_heads * p.page_size;
    const size_t row_k = ((size_t)p.layer * 2 * p.kv_heads + head_kv) * p.page_size;
    const size_t v_rows = (size_t)p.kv_heads * p.page_size;               // from a key row to the value row of its token
    const float sm_scale = 0.08838834764831845f * 1.4426950408889634f;    // log2(e) / sqrt(128)
    // keys: row (lane & 7) + 8 (warp + 4 it), 16-byte chunk lane / 8; values: tokens 64 (warp & 1) + 8 (lane & 7) + 0 .. 7,
    // 8 bytes (16 dimensions) at 32 (warp / 2) + 8 (lane / 8)
    const int kr = (lane & 7) + 8 * pw, kc = lane >> 3;
    const int vt = 64 * (pw & 1) + 8 * (lane & 7), vb = 32 * (pw >> 1) + 8 * (lane >> 3);

    auto page_id = [&](int j) -> int {
      const int t = kv_block_index(blk, begin + j) * kAtTok + tid;
      return t < tokens ? __ldg(p.indices + first_page + fast_div(t, p.page_div)) : 0;
    };
    auto put_rows = [&](int j, int id) -> long long {
      const int t = kv_block_index(blk, begin + j) * kAtTok + tid;
      long long row = -1;
      if (t < tokens) {
        const int slot = t - fast_div(t, p.page_div) * p.page_size;
        const size_t page = min((size_t)(uint32_t)id, (size_t)p.num_pages - 1);        // an index outside the pool reads its last page
        row = (long long)(page * page_rows + row_k + slot);
      }
      sh.row[j & 1][tid] = row;
      asm volatile("bar.sync 1, 128;" ::: "memory");
      return row;
    };
    uint4 kw[4];
    uint2 vw[8];
    uint32_t kp = 0, vp = 0;
    auto load_k = [&](int j) {
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        const long long row = sh.row[j & 1][kr + 32 * it];
        kw[it] = row >= 0 ? __ldg(reinterpret_cast<const uint4*>(p.data + row * 64 + 16 * kc)) : make_uint4(0, 0, 0, 0);
      }
    };
    auto load_v = [&](int j) {
#pragma unroll
      for (int it = 0; it < 8; ++it) {
        const long long row = sh.row[j & 1][vt + it];
        vw[it] = row >= 0 ? __ldg(reinterpret_cast<const uint2*>(p.data + (row + (long long)v_rows) * 64 + vb)) : make_uint2(0, 0);
      }
    };
    auto load_par = [&](long long row) {
      kp = 0; vp = 0;
      if (row >= 0) {
        kp = __ldg(reinterpret_cast<const uint32_t*>(p.param + row));
        vp = __ldg(reinterpret_cast<const uint32_t*>(p.param + row + v_rows));
      }
    };
    bool ok = true;
    int id = 0;
    if (n > 0) {
      const long long row = put_rows(0, page_id(0));
      load_par(row);
      load_k(0);
      load_v(0);
      if (n > 1) id = page_id(1);
    }
    for (int j = 0; j < n; ++j) {
      const int stage = j & 1, ring = j % kAtParStages;
      {
        // parameters of token tid; its slot of the ring is free: block j - 3 is through (v_empty of block j - 1 was awaited)
        const float2 k2 = __half22float2(*reinterpret_cast<const __half2*>(&kp));
        float2 v2 = __half22float2(*reinterpret_cast<const __half2*>(&vp));
        // scales of a cache are positive; below 2^-30 the codes of a token cannot move an fp16 result
        if (v2.x < 9.31322575e-10f) v2.x = 9.31322575e-10f;
        const float rv = __fdividef(1.0f, v2.x), ks = k2.x * sm_scale;
        float* q = &sh.par[ring][tid >> 1][tid & 1];
        q[0] = ks;
        q[2] = -fmaf(16.0f, ks, k2.y * sm_scale);
        // x - x: 0, or NaN where key parameters are not finite (the score of such a token may not end up at -infinity)
        q[4] = __log2f(v2.x) + ((k2.x - k2.x) + (k2.y - k2.y));
        q[6] = rv;
        q[8] = fmaf(v2.y, rv, -8.0f);
        __syncwarp();
        if (lane == 0) mbar_arrive(par_full + 8 * ring);
      }
      if (j + 1 < n) {
        const long long row = put_rows(j + 1, id);        // everybody has read the rows of block j - 1
        load_par(row);
        if (j + 2 < n) id = page_id(j + 2);
      }
      if (j >= 2) {
        ok = mbar_wait(k_empty + 8 * stage, ((j >> 1) + 1) & 1, abort_flag, p.status, 74);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; }
      }
      {
        const uint32_t dst = s_k + stage * kAtTile + (kc >> 1) * (kAtTile / 2);
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          const int r = kr + 32 * it;
          const uint32_t ww[4] = {kw[it].x, kw[it].y, kw[it].z, kw[it].w};
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int ch = 4 * (kc & 1) + x;
            st_shared16(dst + r * 128 + ((ch ^ (r & 7)) << 4), code_pair<0>(ww[x]), code_pair<1>(ww[x]), code_pair<2>(ww[x]),
                        code_pair<3>(ww[x]));
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(k_full + 8 * stage);
      if (j + 1 < n) load_k(j + 1);
      if (j >= 2) {
        ok = mbar_wait(v_empty + 8 * stage, ((j >> 1) + 1) & 1, abort_flag, p.status, 75);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; }
      }
      {
        const uint32_t dst = s_v + stage * kAtTile + (pw & 1) * (kAtTile / 2);
#pragma unroll
        for (int half = 0; half < 4; ++half) {            // four dimensions of the lane's sixteen
          const uint32_t sel = (half & 1) ? 0x7632u : 0x5410u;
          uint32_t x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            x[i] = __byte_perm(half < 2 ? vw[2 * i].x : vw[2 * i].y, half < 2 ? vw[2 * i + 1].x : vw[2 * i + 1].y, sel);
          const int d0 = 2 * vb + 4 * half;
          const int tg = lane & 7;
          st_shared16(dst + d0 * 128 + ((tg ^ (d0 & 7)) << 4), at_centred_pair<0>(x[0]), at_centred_pair<0>(x[1]),
                      at_centred_pair<0>(x[2]), at_centred_pair<0>(x[3]));
          st_shared16(dst + (d0 + 1) * 128 + ((tg ^ ((d0 + 1) & 7)) << 4), at_centred_pair<1>(x[0]), at_centred_pair<1>(x[1]),
                      at_centred_pair<1>(x[2]), at_centred_pair<1>(x[3]));
          st_shared16(dst + (d0 + 2) * 128 + ((tg ^ ((d0 + 2) & 7)) << 4), at_centred_pair<2>(x[0]), at_centred_pair<2>(x[1]),
                      at_centred_pair<2>(x[2]), at_centred_pair<2>(x[3]));
          st_shared16(dst + (d0 + 3) * 128 + ((tg ^ ((d0 + 3) & 7)) << 4), at_centred_pair<3>(x[0]), at_centred_pair<3>(x[1]),
                      at_centred_pair<3>(x[2]), at_centred_pair<3>(x[3]));
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(v_full + 8 * stage);
      if (j + 1 < n) load_v(j + 1);
    }
    if (p.splits > 1) { kv_cluster_barrier(); kv_cluster_barrier(); }
  } else {
    // ---------------------------------------------------------------- MMA issue
    regs_dec<40>();
    if (warp == 12) {
      if (lane == 0 && n > 0) {
        bool ok = mbar_wait(k_full, 0, abort_flag, p.status, 76);
        auto scores = [&](int i, int stage) {
          const uint32_t a = desc_lo(s_q + i * kAtTile), b = desc_lo(s_k + stage * kAtTile);
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {
            const uint32_t off = ((ks >> 2) * (kAtTile / 2) + (ks & 3) * 32) >> 4;
            umma_f16_ss(tmem + i * 128, a + off, b + off, ks > 0);
          }
          umma_commit(s_full + 8 * i);
        };
        if (ok) {
          tc_fence_after();
          for (int i = 0; i < tiles; ++i) scores(i, 0);
          umma_commit(k_empty);
        }
        for (int j = 0; ok && j < n; ++j) {
          const int stage = j & 1;
          ok = mbar_wait(v_full + 8 * stage, (j >> 1) & 1, abort_flag, p.status, 77);
          if (ok && j + 1 < n) ok = mbar_wait(k_full + 8 * (stage ^ 1), ((j + 1) >> 1) & 1, abort_flag, p.status, 78);
          for (int i = 0; ok && i < tiles; ++i) {
            ok = mbar_wait(p_full + 8 * i, j & 1, abort_flag, p.status, 79);
            if (!ok) break;
            tc_fence_after();
            const uint32_t b = desc_lo(s_v + stage * kAtTile);
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
              const uint32_t off = ((ks >> 2) * (kAtTile / 2) + (ks & 3) * 32) >> 4;
              umma_f16_ts(tmem + 256 + i * 128, tmem + i * 128 + ks * 8, b + off, j > 0 || ks > 0);
            }
            if (j + 1 < n) scores(i, stage ^ 1);
            else umma_commit(o_full + 8 * i);
          }
          if (ok) {
            if (j + 1 < n) umma_commit(k_empty + 8 * (stage ^ 1));
            umma_commit(v_empty + 8 * stage);
          }
        }
      }
      __syncwarp();
    }
    if (p.splits > 1) { kv_cluster_barrier(); kv_cluster_barrier(); }
  }
  drain_after_abort(abort_flag);
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

int launch_kv_attend_tc(KvAttendParams& p, int64_t max_rows, cudaStream_t st) {
  const int64_t per_seq = (max_rows + kAtRows - 1) / kAtRows;
  const int64_t bound = p.total_q * p.group / kAtRows + p.batch;
  const bool uniform = !p.qo_indptr || p.batch * per_seq <= 2 * bound;
  p.tiles_per_seq = uniform ? (int)per_seq : 0;
  p.max_tiles = (int)(uniform ? p.batch * per_seq : bound);
  const int64_t units = (int64_t)p.max_tiles * p.kv_heads;
  int splits = 1;
  while (splits < 8 && units * splits * 2 <= num_sms()) splits *= 2;
  p.splits = splits;
  if (units * splits > 0x7fffffffll) return fail(QR_EUNSUPPORTED, "qr_kv_attend_i4: too many tiles");
  QR_CUDA(cudaFuncSetAttribute(kv_attend_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kAtSmem));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(units * splits));
  cfg.blockDim = dim3(kAtThreads);
  cfg.dynamicSmemBytes = kAtSmem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = splits > 1 ? 1 : 0;
  QR_CUDA(cudaLaunchKernelEx(&cfg, kv_attend_tc_kernel, (const KvAttendParams)p));
  return QR_OK;
}

}  // namespace qr
