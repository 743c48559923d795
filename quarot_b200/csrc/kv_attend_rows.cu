// Attention over the paged 4-bit cache for few query rows per KV head (decode, drafted tokens, short chunks; any number
// of rows is right, 8 or 16 at a time).  Causal, with an optional sliding window and sink tokens, grouped query heads.
//
// Mathematics.  With key codes c, scale s and zero z per (token, head), the score of row r and token t is
//   s_t <q_r, c_t> - z_t sum(q_r),   and value = s' c' - z'  (s', z' the value parameters).
// The tensor cores see the codes as they stand: four bits masked out of a word are the subnormal fp16 number c 2^-24 (bits
// 0 .. 3) or c 2^-20 (bits 4 .. 7), exact, so that a pair of codes takes one logical instruction and four pairs one shift.
// The powers of two are taken back in the query (brought to 2^10 .. 2^15 by powers of two per row, in which no bit is lost)
// and in the output, where the two kinds lie in different registers.
// Weights: w_t = exp2(score_t + log2 s'_t - M) so that the value scale is inside the weight.  M does not follow the
// maximum: it is set 1 below the first one and moves, in whole steps, only where a weight would pass 2^15, so that sums
// are rarely multiplied through and no maximum is looked for across lanes.  Weights are cut to the 11 bits of fp16 before
// all sums,
//   l = sum w / s'_t  (the softmax denominator),   y = sum w (z'_t / s'_t - 7.5),   o = (sum w~ c' - 7.5 sum w~ - y) / l,
// so that a cut of weight t moves the result by its difference from v_t - o only (a row that looks at one token has
// nothing of it) and their common part not at all.  l and y are fp32 sums of w; w~ (the B operand) differs from w below
// 2^-14 of the largest, by at most 2^-25, and meets the centred codes c' - 7.5 with it (sum w~: one more MMA row of ones):
// next to a token with the weight 1, one below 2^-25 has its share of the softmax and its centre, but not its codes.
//
// Mapping.  A warp takes blocks of 32 tokens.  Scores: S^T = K Q^T with mma.m16n8k16, 16 tokens as M, 8 rows as N; lane
// (g, c) = (lane / 4, lane % 4) reads 16 bytes of each of its token rows (32 codes), and since the order of the 128
// dimensions is free as long as the query follows it, nibbles j and j + 4 of a word are a fragment register as they
// stand.  Weights: S^T leaves the tensor core as (token, row) pairs and movmatrix turns it into the B operand (tokens as
// K).  Values: O^T = V^T w, dimensions as M; a fragment register holds two tokens of one dimension, made by one byte
// permute per four of them.  Which token sits in which fragment row is free too and is chosen so that all reads of the
// shared-memory ring are free of bank conflicts.  Warps keep their own softmax state and are merged through shared
// memory; few (tile, head) pairs: a cluster shares the token axis and is merged through distributed shared memory.
// Every warp has its own ring of cp.async stages, so no barrier runs inside the loop.
// What bounds it: instructions.  64 sequences, window of 4096, 32 heads over 8: 74 us = 3.9 TB/s of the cache (0.59 of the
// copy rate), issue slots 58 %, logical pipe 55 %; 32 x 4 drafted tokens, 64 heads over 8, ragged to 4100 tokens: 73.5 us
// (floor 15.5), 43 % of issue slots with eight warps per SM.  With 16 + c in fp16 instead of subnormal codes 89 and 94 us;
// 32 rows at once, their query fragments read from shared memory, 128 us in the second case.
#include "kv_common.cuh"

#include <math.h>
#include <atomic>

namespace qr {

constexpr int kRwTok = 32;                              // tokens per block
constexpr int kRwStageBytes = kRwTok * (64 + 64 + 4 + 4);
constexpr int kRwORow = kHeadDim + 4;                   // floats per row of the merge buffers
constexpr uint32_t kRwLow = 0x000F000Fu, kRwHigh = 0x00F000F0u;   // codes as they stand in subnormal fp16: c 2^-24 and c 2^-20
constexpr float kRwTop = 15.0f;                         // weights are at most 2^15

// Warps work on two 16-token tiles at once (TA), which hides more latency than further warps would: eight rows take 128
// registers a thread, four CTAs of four warps per SM; sixteen rows 232, two CTAs.  CTAs of four warps balance better than
// larger ones, and smaller ones have too much beside the loop.
template <int NT>
struct RwConfig {
  static constexpr int kWarps = 4;
  static constexpr int kStages = NT == 1 ? 2 : 3;
  static constexpr int kCtas = NT == 1 ? 4 : 2;                  // per SM
  static constexpr int kRing = kWarps * kStages * kRwStageBytes;
};

template <int NT>
struct RwShared {
  static constexpr int kWarps = RwConfig<NT>::kWarps;
  __half q[8 * NT][kHeadDim];                           // rows in fragment order
  float qsum[8 * NT], qmul[8 * NT];                     // sum of the row's elements; the power of two that its products lack
  int pos[8 * NT];                                      // position of the row, -1: not a row
  union {
    struct {                                            // of a warp's block, per token:
      float4 par4[kWarps][kRwTok];                      // s, -z (both times log2(e) / sqrt(d)), log2 s', 1 / s'
      float par1[kWarps][kRwTok];                       // z' / s' - 7.5
    };
    float part_o[8 * NT][kHeadDim];                     // after the loop: the CTA's share
  };
  float m[kWarps][8 * NT], l[kWarps][8 * NT];
  float part_m[8 * NT], part_l[8 * NT];
};

__device__ __forceinline__ void rw_cp16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void rw_cp4(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void rw_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void rw_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
// The 11 leading bits of a weight, those of a normal fp16 number.
__device__ __forceinline__ float rw_cut(float w) { return __uint_as_float(__float_as_uint(w) & 0xffffe000u); }
// Row of a block's stage that holds 64 bytes of codes: 16-byte chunk ch of row r lies at chunk ch ^ rw_swz(r).
__device__ __forceinline__ int rw_swz(int r) { return (r & 2); }
// Token of a 16-token tile in fragment slot s: the four tokens that a V fragment reads at once, and the two of a K
// fragment, differ in the bank halves that their rows start in.
__device__ __forceinline__ int rw_token_even(int c) { return c; }              // slot 2 c
__device__ __forceinline__ int rw_token_odd(int c) { return 4 + (c ^ 1); }     // slot 2 c + 1

__device__ __forceinline__ void rw_store_row(const KvAttendParams& p, const KvTile& w, int head_kv, int r, int d4, float4 v, float inv) {
  const int row = w.row0 + r;
  const int tok = fast_div(row, p.group_div), hh = row - tok * p.group;
  const __half2 h0 = __floats2half2_rn(v.x * inv, v.y * inv), h1 = __floats2half2_rn(v.z * inv, v.w * inv);
  uint2 out;
  out.x = *reinterpret_cast<const uint32_t*>(&h0);
  out.y = *reinterpret_cast<const uint32_t*>(&h1);
  *reinterpret_cast<uint2*>(p.o + (w.tok0 + tok) * p.o_ts + (int64_t)(head_kv * p.group + hh) * p.o_hs + d4) = out;
}

template <int NT>
__global__ void __launch_bounds__(32 * RwConfig<NT>::kWarps, RwConfig<NT>::kCtas)
kv_attend_rows_kernel(const KvAttendParams p) {
  constexpr int R = 8 * NT;
  constexpr int kStages = RwConfig<NT>::kStages;
  constexpr int kWarps = RwConfig<NT>::kWarps;
  constexpr int TA = 2;                                 // 16-token tiles of a block worked on together
  extern __shared__ __align__(128) unsigned char s_dyn[];
  unsigned char* ring = s_dyn;
  RwShared<NT>& sh = *reinterpret_cast<RwShared<NT>*>(s_dyn + RwConfig<NT>::kRing);
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  pdl_wait();
  const int unit = blockIdx.x / p.splits;
  uint32_t crank = 0;
  if (p.splits > 1) crank = kv_cluster_rank();
  const int head_kv = unit % p.kv_heads;
  const KvTile w = kv_find_tile(p, unit / p.kv_heads, R, lane);
  if (w.rows == 0) return;                              // the whole cluster has the same tile

  const int last_row = w.row0 + w.rows - 1;
  const int p_min = w.pos0 + fast_div(w.row0, p.group_div), p_max = w.pos0 + fast_div(last_row, p.group_div);
  const KvBlocks blk = kv_blocks<kRwTok>(p_min, p_max, p.window, p.sinks);
  // the CTAs of a cluster take contiguous ranges of blocks, the warps of a CTA every fourth one
  const int per = (blk.count + p.splits - 1) / p.splits;
  const int begin = (int)crank * per + warp, end = min((int)(crank + 1) * per, blk.count);

  const int32_t* pages = p.indices + w.first;
  const int tokens = min(p_max + 1, w.seq_len);         // tokens from here on are not read
  // a pool has fewer than 2^32 rows of 64 bytes
  const uint32_t page_rows = (uint32_t)p.layers * 2 * p.kv_heads * p.page_size;
  const uint32_t row_k = ((uint32_t)p.layer * 2 * p.kv_heads + head_kv) * p.page_size;
  const uint32_t v_rows = (uint32_t)p.kv_heads * p.page_size;
  const uint64_t v_bytes = (uint64_t)v_rows * 64;
  const uint32_t last_page = (uint32_t)(p.num_pages - 1);
  const uint32_t my_ring = smem_u32(ring) + warp * (kStages * kRwStageBytes);

  // Lane copies chunk c of the rows g + 8 i of a block.  Where pages hold a multiple of 16 tokens the rows i = 0, 1 and
  // 2, 3 lie in one page each, eight slots apart.
  const bool by16 = (p.page_size & 15) == 0;
  auto page_ids = [&](int bi, int (&id)[4]) {
    const int t0 = kv_block_index(blk, bi) * kRwTok + g;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if ((i & 1) && by16) continue;
      id[i] = t0 + 8 * i < tokens ? __ldg(pages + fast_div(t0 + 8 * i, p.page_div)) : 0;
    }
  };
  auto issue = [&](int bi, int stage, const int (&id)[4]) {
    const int t0 = kv_block_index(blk, bi) * kRwTok + g;
    const uint32_t st = my_ring + stage * kRwStageBytes + g * 64 + ((c ^ rw_swz(g)) << 4);
    const uint32_t sp = my_ring + stage * kRwStageBytes + kRwTok * 128 + (c & 1) * (kRwTok * 4) + g * 4;
    const uint8_t* src = nullptr;
    const __half2* num = nullptr;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = t0 + 8 * i;
      const bool ok = t < tokens;
      if ((i & 1) && by16) {
        src += 8 * 64;
        num += 8;
      } else {
        // an index outside the pool reads its last page
        const uint32_t row = min((uint32_t)id[i], last_page) * page_rows + row_k + (t - fast_div(t, p.page_div) * p.page_size);
        src = p.data + (uint64_t)row * 64 + 16 * c;
        num = p.param + (row + (c ? v_rows : 0u));
      }
      rw_cp16(st + 512 * i, src, ok ? 16 : 0);
      rw_cp16(st + 512 * i + kRwTok * 64, src + v_bytes, ok ? 16 : 0);
      if (c < 2) rw_cp4(sp + 32 * i, num, ok ? 4 : 0);
    }
  };
  // the query rows are on their way while the first pages are looked up
  uint2 raw[R / kWarps];
  int pos[R / kWarps];
#pragma unroll
  for (int i = 0; i < R / kWarps; ++i) {
    const int r = warp + i * kWarps;
    raw[i] = make_uint2(0, 0);
    pos[i] = -1;
    if (r < w.rows) {
      const int row = w.row0 + r;
      const int tok = fast_div(row, p.group_div), hh = row - tok * p.group;
      pos[i] = w.pos0 + tok;
      raw[i] = *reinterpret_cast<const uint2*>(p.q + (w.tok0 + tok) * p.q_ts + (int64_t)(head_kv * p.group + hh) * p.q_hs + 4 * lane);
    }
  }
  int id[4];
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    const int bi = begin + s * kWarps;
    if (bi < end) { page_ids(bi, id); issue(bi, s, id); }
    rw_commit();
  }
  if (begin + (kStages - 1) * kWarps < end) page_ids(begin + (kStages - 1) * kWarps, id);

#pragma unroll
  for (int i = 0; i < R / kWarps; ++i) {
    const int r = warp + i * kWarps;
    float x[4];
    half4_to_f32(raw[i], x);
    if (p.hadamard_q) {
      fwht128_warp(x, lane);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = __half2float(__float2half_rn(x[e] * 0.08838834764831845f));
    }
    float sum = x[0] + x[1] + x[2] + x[3], big = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, s);
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, s));
    }
    // a power of two that brings the largest element to 2^10 .. 2^11 (fp16 elements: no bit is lost in [2^-24, 2^11])
    const int eb = big > 0.0f && big <= 65504.0f ? (int)(__float_as_uint(big) >> 23) - 127 : 10;
    const float down = __uint_as_float((uint32_t)(127 + 10 - eb) << 23);
    // dimension d = 32 cc + 8 wi + e sits in register (2 wi + e % 4 / 2, e % 2), half e / 4, of lane column cc
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
      const int d = 4 * lane + e4, e = d & 7;
      sh.q[r][(d >> 5) * 32 + ((d >> 3) & 3) * 8 + (e & 3) * 2 + (e >> 2)] = __float2half_rn(x[e4] * (e & 1 ? down : down * 16.0f));
    }
    if (lane == 0) { sh.qsum[r] = sum; sh.qmul[r] = __uint_as_float((uint32_t)(127 + 10 + eb) << 23); sh.pos[r] = pos[i]; }
  }
  __syncthreads();

  uint32_t qf[NT][16];                                  // query fragments
  float qs[NT][2], qm[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 u = *reinterpret_cast<const uint4*>(&sh.q[8 * n + g][32 * c + 8 * i]);
      qf[n][4 * i] = u.x; qf[n][4 * i + 1] = u.y; qf[n][4 * i + 2] = u.z; qf[n][4 * i + 3] = u.w;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) { qs[n][k] = sh.qsum[8 * n + 2 * c + k]; qm[n][k] = sh.qmul[8 * n + 2 * c + k]; }
  }

  float o[NT][8][4], ws[NT][4], l[NT][2], y[NT][2], m[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][t][e] = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) ws[n][e] = 0.0f;
#pragma unroll
    for (int k = 0; k < 2; ++k) { l[n][k] = 0.0f; y[n][k] = 0.0f; m[n][k] = -INFINITY; }
  }

  int stage = 0;
  const float sm_scale = 0.08838834764831845f * 1.4426950408889634f;   // log2(e) / sqrt(128)
  // slots of a 16-token tile -> tokens, see rw_token_even: rows g, g + 8 of a K fragment; 2 c, 2 c + 1 (+ 8) of a V fragment
  const int tau = (g & 1) ? rw_token_odd(g >> 1) : rw_token_even(g >> 1), ta = rw_token_even(c), tb = rw_token_odd(c);
#pragma unroll 1
  for (int bi = begin; bi < end; bi += kWarps) {
    {
      const int ahead = bi + (kStages - 1) * kWarps;
      if (ahead < end) issue(ahead, stage == 0 ? kStages - 1 : stage - 1, id);
      rw_commit();
      if (ahead + kWarps < end) page_ids(ahead + kWarps, id);
    }
    rw_wait<kStages - 1>();
    __syncwarp();
    const unsigned char* st = ring + warp * (kStages * kRwStageBytes) + stage * kRwStageBytes;
    const int t0 = kv_block_index(blk, bi) * kRwTok;
    const bool edge = t0 + kRwTok - 1 > p_min || (p.window > 0 && t0 <= p_max - p.window && t0 + kRwTok - 1 >= p.sinks);
    {
      // the numbers of token `lane`
      const float2 kp = __half22float2(*reinterpret_cast<const __half2*>(st + kRwTok * 128 + lane * 4));
      float2 vp = __half22float2(*reinterpret_cast<const __half2*>(st + kRwTok * 132 + lane * 4));
      // scales of a cache are positive; below 2^-30 the codes of a token cannot move an fp16 result
      if (vp.x < 9.31322575e-10f) vp.x = 9.31322575e-10f;
      // x - x: 0, or NaN where it is not finite.  Then the weight of the token is NaN in the rows that see it, and its other
      // numbers are 0, so that a weight 0 leaves the sums of the rows that do not see it alone.
      const float bad = ((kp.x - kp.x) + (kp.y - kp.y)) + ((vp.x - vp.x) + (vp.y - vp.y));
      const bool fine = bad == 0.0f;
      const float rv = __fdividef(1.0f, vp.x), ks = kp.x * sm_scale;
      sh.par4[warp][lane] = make_float4(ks, -kp.y * sm_scale, __log2f(vp.x) + bad, fine ? rv : 0.0f);
      sh.par1[warp][lane] = fine ? fmaf(vp.y, rv, -7.5f) : 0.0f;
    }
    __syncwarp();
    float s[TA][NT][4];
    uint4 xk[TA], zk[TA];
#pragma unroll
    for (int a = 0; a < TA; ++a) {
      // fragment rows g and g + 8: tokens tau and 8 + tau of the tile
      const unsigned char* sk = st + (16 * a + tau) * 64 + ((c ^ rw_swz(tau)) << 4);
      xk[a] = *reinterpret_cast<const uint4*>(sk);
      zk[a] = *reinterpret_cast<const uint4*>(sk + 8 * 64);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[a][n][e] = 0.0f;
    }
#pragma unroll
    for (int wi = 0; wi < 4; ++wi)
#pragma unroll
      for (int a = 0; a < TA; ++a) {
        const uint32_t xw = wi == 0 ? xk[a].x : wi == 1 ? xk[a].y : wi == 2 ? xk[a].z : xk[a].w;
        const uint32_t zw = wi == 0 ? zk[a].x : wi == 1 ? zk[a].y : wi == 2 ? zk[a].z : zk[a].w;
        const uint32_t xh = xw >> 8, zh = zw >> 8;
        const uint32_t f0 = xw & kRwLow, f1 = zw & kRwLow, f2 = xw & kRwHigh, f3 = zw & kRwHigh;
        const uint32_t h0 = xh & kRwLow, h1 = zh & kRwLow, h2 = xh & kRwHigh, h3 = zh & kRwHigh;
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_f16(s[a][n], f0, f1, f2, f3, qf[n][4 * wi], qf[n][4 * wi + 1]);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_f16(s[a][n], h0, h1, h2, h3, qf[n][4 * wi + 2], qf[n][4 * wi + 3]);
      }
    float rv[TA][2], zv[TA][2];                         // 1 / s', z' / s' - 7.5 of the lane's tokens
    float e[TA][NT][4];                                 // exponents relative to M
    float top = -INFINITY;
#pragma unroll
    for (int a = 0; a < TA; ++a)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = 16 * a + 8 * h + tau;
        const float4 pr = sh.par4[warp][r];
        rv[a][h] = pr.w;
        zv[a][h] = sh.par1[warp][r];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            s[a][n][2 * h + k] = fmaf(pr.x * qm[n][k], s[a][n][2 * h + k], fmaf(pr.y, qs[n][k], pr.z));
            e[a][n][2 * h + k] = s[a][n][2 * h + k] - m[n][k];          // +infinity before the row has seen a token
            top = fmaxf(top, e[a][n][2 * h + k]);
          }
      }
    if (__builtin_expect(edge, 0)) {
      top = -INFINITY;
#pragma unroll
      for (int a = 0; a < TA; ++a)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int t = t0 + 16 * a + 8 * h + tau;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int pos = sh.pos[8 * n + 2 * c + k];
              if (t > pos || (p.window > 0 && t <= pos - p.window && t >= p.sinks)) s[a][n][2 * h + k] = e[a][n][2 * h + k] = -INFINITY;
              top = fmaxf(top, e[a][n][2 * h + k]);
            }
        }
    }
    if (__builtin_expect(__any_sync(0xffffffffu, top > kRwTop), 0)) {
      // a weight would pass 2^15, or a row sees its first token: M moves, and what has been summed up is multiplied through
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float f[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float up = fmaxf(s[0][n][k], s[0][n][2 + k]);
#pragma unroll
          for (int a = 1; a < TA; ++a) up = fmaxf(up, fmaxf(s[a][n][k], s[a][n][2 + k]));
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, x));
          const bool move = up - m[n][k] > kRwTop;
          const float to = ceilf(up) - 1.0f;
          f[k] = !move ? 1.0f : m[n][k] == -INFINITY ? 0.0f : ex2(m[n][k] - to);
          m[n][k] = move ? to : m[n][k];
          l[n][k] *= f[k];
          y[n][k] *= f[k];
#pragma unroll
          for (int a = 0; a < TA; ++a)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              e[a][n][2 * h + k] = s[a][n][2 * h + k] == -INFINITY ? -INFINITY : s[a][n][2 * h + k] - m[n][k];
        }
#pragma unroll
        for (int t = 0; t < 8; ++t)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[n][t][x] *= f[x & 1];
#pragma unroll
        for (int x = 0; x < 4; ++x) ws[n][x] *= f[x & 1];
      }
    }
    uint32_t pb[TA][NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int a = 0; a < TA; ++a)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float w0 = rw_cut(ex2(e[a][n][2 * h])), w1 = rw_cut(ex2(e[a][n][2 * h + 1]));
          l[n][0] = fmaf(w0, rv[a][h], l[n][0]); y[n][0] = fmaf(w0, zv[a][h], y[n][0]);
          l[n][1] = fmaf(w1, rv[a][h], l[n][1]); y[n][1] = fmaf(w1, zv[a][h], y[n][1]);
          const __half2 wh = __floats2half2_rn(w0, w1);
          pb[a][n][h] = movmatrix_trans(*reinterpret_cast<const uint32_t*>(&wh));
        }
    }
#pragma unroll
    for (int a = 0; a < TA; ++a) {
      // slots 2c, 2c + 1, 2c + 8, 2c + 9: tokens of the tile
      const unsigned char* sv = st + kRwTok * 64 + (16 * a) * 64 + (g & 1) * 8;
      const unsigned char* sa = sv + ta * 64 + (((g >> 1) ^ rw_swz(ta)) << 4);
      const unsigned char* sb = sv + tb * 64 + (((g >> 1) ^ rw_swz(tb)) << 4);
      const uint2 va = *reinterpret_cast<const uint2*>(sa), vb = *reinterpret_cast<const uint2*>(sb);
      const uint2 vc = *reinterpret_cast<const uint2*>(sa + 8 * 64), vd = *reinterpret_cast<const uint2*>(sb + 8 * 64);
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {                    // four dimensions of the lane's sixteen
        const uint32_t sel = (q4 & 1) ? 0x7632u : 0x5410u;
        const uint32_t ab = __byte_perm(q4 < 2 ? va.x : va.y, q4 < 2 ? vb.x : vb.y, sel);
        const uint32_t cd = __byte_perm(q4 < 2 ? vc.x : vc.y, q4 < 2 ? vd.x : vd.y, sel);
        const uint32_t ah = ab >> 8, ch = cd >> 8;
        const uint32_t f0 = ab & kRwLow, f1 = ab & kRwHigh, f2 = cd & kRwLow, f3 = cd & kRwHigh;
        const uint32_t h0 = ah & kRwLow, h1 = ah & kRwHigh, h2 = ch & kRwLow, h3 = ch & kRwHigh;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_f16(o[n][2 * q4], f0, f1, f2, f3, pb[a][n][0], pb[a][n][1]);
          mma_f16(o[n][2 * q4 + 1], h0, h1, h2, h3, pb[a][n][0], pb[a][n][1]);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_f16(ws[n], 0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u, pb[a][n][0], pb[a][n][1]);
    }
    __syncwarp();                                       // the stage is filled again in the next round
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  rw_wait<0>();
  __syncthreads();                                      // the ring becomes the merge buffer

  float* merge = reinterpret_cast<float*>(ring);        // [warp][row][kRwORow]
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) {
        l[n][k] += __shfl_xor_sync(0xffffffffu, l[n][k], x);
        y[n][k] += __shfl_xor_sync(0xffffffffu, y[n][k], x);
      }
      const int r = 8 * n + 2 * c + k;
      const float off = fmaf(7.5f, ws[n][k], y[n][k]);
      float* dst = merge + ((size_t)warp * R + r) * kRwORow + 16 * g;
#pragma unroll
      for (int t = 0; t < 4; ++t)
        *reinterpret_cast<float4*>(dst + 4 * t) = make_float4(fmaf(o[n][2 * t][k], 16777216.0f, -off), fmaf(o[n][2 * t][2 + k], 1048576.0f, -off),
                                                              fmaf(o[n][2 * t + 1][k], 16777216.0f, -off), fmaf(o[n][2 * t + 1][2 + k], 1048576.0f, -off));
      if (g == 0) { sh.m[warp][r] = m[n][k]; sh.l[warp][r] = l[n][k]; }
    }
  __syncthreads();
  for (int r = warp; r < w.rows; r += kWarps) {
    float mm = -INFINITY;
#pragma unroll
    for (int x = 0; x < kWarps; ++x) mm = fmaxf(mm, sh.m[x][r]);
    float ll = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int x = 0; x < kWarps; ++x) {
      if (sh.m[x][r] == -INFINITY && sh.l[x][r] == 0.0f) continue;     // a warp that saw no token of the row
      const float f = ex2(sh.m[x][r] - mm);
      const float4 v = *reinterpret_cast<const float4*>(merge + ((size_t)x * R + r) * kRwORow + 4 * lane);
      ll = fmaf(sh.l[x][r], f, ll);
      acc.x = fmaf(v.x, f, acc.x); acc.y = fmaf(v.y, f, acc.y); acc.z = fmaf(v.z, f, acc.z); acc.w = fmaf(v.w, f, acc.w);
    }
    if (p.splits == 1) {
      rw_store_row(p, w, head_kv, r, 4 * lane, acc, ll != 0.0f ? 1.0f / ll : 0.0f);     // a row that sees nothing gives zeros
    } else {
      *reinterpret_cast<float4*>(&sh.part_o[r][4 * lane]) = acc;
      if (lane == 0) { sh.part_m[r] = mm; sh.part_l[r] = ll; }
    }
  }
  if (p.splits > 1) {
    kv_cluster_barrier();
    // the CTAs of the cluster deal out the rows
    kv_merge_rows<1>(p.splits, (int)crank + p.splits * warp, p.splits * kWarps, w.rows, lane, sh.part_m, sh.part_l,
                     [&](int r) { return &sh.part_o[r][4 * lane]; },
                     [&](int r, float4 v, float inv) { rw_store_row(p, w, head_kv, r, 4 * lane, v, inv); });
    kv_cluster_barrier();
  }
}

namespace {
// Clusters of s CTAs that fit on a device, for s = 1 .. 16.  Two threads that ask first write the same numbers.
struct KvFit {
  std::atomic<int> known, per_sm, fit[17];
};
constexpr int kKvDevices = 32;
KvFit g_kv_fit[kKvKernels][kKvDevices];

int kv_ask_fit(KvFit& k, const void* kernel, int threads, size_t smem) {
  QR_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  QR_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  int per_sm = 0;
  QR_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, smem));
  k.per_sm.store(per_sm, std::memory_order_relaxed);
  k.fit[1].store(per_sm * num_sms(), std::memory_order_relaxed);
  for (int s = 2; s <= 16; ++s) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)s;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)s);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) { cudaGetLastError(); n = 0; }
    k.fit[s].store(n, std::memory_order_relaxed);
  }
  k.known.store(1, std::memory_order_release);
  return QR_OK;
}
}  // namespace

int kv_pick_splits(int which, const void* kernel, int threads, size_t smem, int64_t units, int64_t most, double alone,
                   double joined, int* splits, int* resident, double* cost_out) {
  int dev = 0;
  QR_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= kKvDevices) return fail(QR_EUNSUPPORTED, "qr_kv_attend_i4: device %d (at most %d)", dev, kKvDevices - 1);
  KvFit& k = g_kv_fit[which][dev];
  if (!k.known.load(std::memory_order_acquire)) {
    if (const int rc = kv_ask_fit(k, kernel, threads, smem)) return rc;
  }
  const int per_sm = k.per_sm.load(std::memory_order_relaxed);
  *resident = k.fit[1].load(std::memory_order_relaxed);
  double best = 0.0;
  *splits = 1;
  for (int s = 1; s <= 16 && s <= most; ++s) {
    const int fit = k.fit[s].load(std::memory_order_relaxed);
    if (fit < 1) continue;
    // CTAs that the fullest SM works through, against those that it holds.  Of four, three take three quarters of the time
    // (instructions); of two, one takes 0.6 of it (latency); an SM is not faster with fewer than it could hold in all.
    const int64_t load = (units * per_sm + fit - 1) / fit;
    // Clusters start as a whole: in several rounds of two CTAs per SM that costs some 15 % more.
    // With these two against neither, units x tokens, us: 192 x 1000 31 -> 20, 512 x 4000 132 -> 108; where several rounds of
    // long units run the rule is not borne out: 192 x 16000 170 -> 187, 320 x 16000 270 -> 309.
    double rounds = load <= per_sm ? 1.0 : (double)load / per_sm;
    if (per_sm == 2 && load > 2) rounds = ((double)(load / 2) + 0.6 * (double)(load % 2)) * (s > 1 ? 1.15 : 1.0);
    const double cost = rounds * (1.0 / s + (s > 1 ? joined : alone));
    if (s == 1 || cost < best * 0.98) { best = cost; *splits = s; }
  }
  if (cost_out) *cost_out = best;
  return QR_OK;
}

// Tiles and split of a call; the cost of kv_pick_splits.
template <int NT>
static int plan_rows(KvAttendParams& p, int64_t max_rows, int64_t* units, double* cost) {
  constexpr int R = 8 * NT, kWarps = RwConfig<NT>::kWarps;
  constexpr size_t smem = RwConfig<NT>::kRing + sizeof(RwShared<NT>);
  static_assert(kWarps * R * kRwORow * sizeof(float) <= RwConfig<NT>::kRing, "the merge buffer lies in the ring");
  static_assert(RwConfig<NT>::kCtas * (smem + 1024) <= 228 * 1024, "shared memory");
  // tiles: at most one ragged tile per sequence beyond the full ones; a grid of equal shares per sequence needs no search
  const int64_t per_seq = (max_rows + R - 1) / R;
  const int64_t bound = p.total_q * p.group / R + p.batch;
  // by the sizes alone, which the workspace query has too; without qo_indptr (one token each) it always holds
  const bool uniform = p.batch * per_seq <= 2 * bound;
  const int64_t tiles = uniform ? p.batch * per_seq : bound;
  *units = tiles * p.kv_heads;
  if (*units > 0x7fffffff / 16) return fail(QR_EUNSUPPORTED, "qr_kv_attend_i4: too many tiles");
  p.tiles_per_seq = uniform ? (int)per_seq : 0;
  p.max_tiles = (int)tiles;
  // start, query rows and the join of the warps take about as long as two blocks of a warp, a cluster's join half of one
  // more, two with sixteen rows; a list of pages much longer than what the sequences use must not lead to splits that only
  // pay for such lengths
  const int64_t blocks = visible_blocks(p, max_rows, kRwTok, false), evenly = visible_blocks(p, max_rows, kRwTok, true);
  const double length = (double)(evenly < 256 ? evenly : 256) / kWarps;
  int resident = 0;
  if (const int rc = kv_pick_splits(NT == 1 ? kKvKernelRows8 : kKvKernelRows16, (const void*)kv_attend_rows_kernel<NT>, 32 * kWarps,
                                    smem, *units, (blocks + kWarps - 1) / kWarps, 2.0 / length, (NT == 1 ? 2.5 : 4.0) / length,
                                    &p.splits, &resident, cost)) return rc;
  // more than one round: the longest sequences first (32 of ragged lengths: 87 us -> 75); a window makes them alike
  p.sorted = uniform && p.window <= 0 && p.batch > 1 && p.batch <= 64 && *units * p.splits > resident;
  return QR_OK;
}

int kv_attend_rows_time(const KvAttendParams& p, int64_t max_rows, double* us) {
  KvAttendParams c = p;
  int64_t units = 0;
  double cost = 0.0;
  if (const int rc = plan_rows<2>(c, max_rows, &units, &cost)) return rc;
  *us = 1.0 + cost * (double)visible_blocks(c, max_rows, kRwTok, true) * 0.425;      // 13.3 ns per token of a unit
  return QR_OK;
}

template <int NT>
static int launch_rows(KvAttendParams& p, int64_t max_rows, cudaStream_t st) {
  constexpr int kWarps = RwConfig<NT>::kWarps;
  constexpr size_t smem = RwConfig<NT>::kRing + sizeof(RwShared<NT>);
  int64_t units = 0;
  if (const int rc = plan_rows<NT>(p, max_rows, &units, nullptr)) return rc;
  const int splits = p.splits;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = use_pdl(p.total_q);
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)splits;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(units * splits));
  cfg.blockDim = dim3(32 * kWarps);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = splits > 1 ? 2 : 1;
  QR_CUDA(cudaLaunchKernelEx(&cfg, kv_attend_rows_kernel<NT>, (const KvAttendParams)p));
  return QR_OK;
}

int launch_kv_attend_rows(KvAttendParams& p, int64_t max_rows, cudaStream_t st) {
  if (max_rows <= 8) return launch_rows<1>(p, max_rows, st);
  return launch_rows<2>(p, max_rows, st);
}

// Which kernel: mma.sync, 16 rows at a time, or tcgen05, 256 rows at a time at a cost that hardly depends on the rows and
// with 11 us (18 where CTAs are joined) beside the tokens.  Measured, us in the one and in the other:
//   32 sequences of 8192 tokens, 8 KV heads: 32 rows 194 and 378, 48 rows 289 and 378, 64 rows 382 and 378, 96 rows 569 and 379;
//   one sequence, 8 KV heads, 128 rows: 300 tokens 11 and 23, 4000 tokens 22 and 28, 16000 tokens 55 and 41; 256 rows: 13 and 25,
//   33 and 32, 99 and 47.
// Up to 64 rows the first is never much behind; above, the estimates decide (both within about 15 % of the figures above).
static int kv_pick_kernel(const KvAttendParams& p, int64_t rows, bool* tc, size_t* bytes) {
  *tc = false;
  if (g_tuning.kv_attend == 1 || (g_tuning.kv_attend == 0 && rows <= 64)) return QR_OK;
  double a = 0.0, b = 0.0;
  if (const int rc = kv_attend_tc_time(p, rows, &b, bytes)) return rc;
  // more tiles than the first kernel's grid may have: the second takes them
  *tc = g_tuning.kv_attend == 2 || kv_attend_rows_time(p, rows, &a) != QR_OK || b < a;
  return QR_OK;
}

}  // namespace qr

extern "C" int qr_kv_attend_i4(void* o, int64_t o_token_stride, int64_t o_head_stride, const void* q, int64_t q_token_stride,
                               int64_t q_head_stride, const void* kv_data, const void* kv_param, int64_t num_pages,
                               const int32_t* kv_indptr, const int32_t* kv_indices, int64_t num_indices,
                               const int32_t* last_page_offset, const int32_t* qo_indptr, int64_t total_q, int64_t max_q_len,
                               int batch, int num_layers, int layer, int num_q_heads, int num_kv_heads, int page_size, int head_dim, int window, int sink_tokens,
                               int hadamard_q, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace qr;
  if (batch < 0 || total_q < 0 || max_q_len < 0 || num_indices < 0) return fail(QR_EINVAL, "qr_kv_attend_i4: negative size");
  if (batch == 0 || total_q == 0 || max_q_len == 0) return QR_OK;
  if (!o || !q || !kv_data || !kv_param || !kv_indptr || !kv_indices || !last_page_offset)
    return fail(QR_EINVAL, "qr_kv_attend_i4: null pointer");
  if (head_dim != kHeadDim) return fail(QR_EUNSUPPORTED, "qr_kv_attend_i4: head_dim = %d (only 128)", head_dim);
  if (num_layers < 1 || layer < 0 || layer >= num_layers || page_size < 1 || num_pages < 1)
    return fail(QR_EINVAL, "qr_kv_attend_i4: bad layer / page size / pages");
  if (num_q_heads < 1 || num_kv_heads < 1 || num_q_heads % num_kv_heads)
    return fail(QR_EINVAL, "qr_kv_attend_i4: %d query heads over %d KV heads (a multiple is needed)", num_q_heads, num_kv_heads);
  if (num_pages > 0xffffffffll / (2ll * num_layers * num_kv_heads) / page_size)
    return fail(QR_EUNSUPPORTED, "qr_kv_attend_i4: a pool of 2^32 or more (page, layer, key / value, head, slot) rows");
  if (window < 0 || sink_tokens < 0) return fail(QR_EINVAL, "qr_kv_attend_i4: negative window or sink tokens");
  if (!qo_indptr && (total_q != batch || max_q_len != 1))
    return fail(QR_EINVAL, "qr_kv_attend_i4: without qo_indptr every sequence has one new token");
  if (max_q_len > total_q) return fail(QR_EINVAL, "qr_kv_attend_i4: max_q_len exceeds the number of new tokens");
  const int group = num_q_heads / num_kv_heads;
  if (total_q > 0x3fffffffll / group || (int64_t)batch * max_q_len * group > 0xffffffffffll)
    return fail(QR_EUNSUPPORTED, "qr_kv_attend_i4: too many query rows");
  if (workspace && ((uintptr_t)workspace & 15)) return fail(QR_EALIGN, "qr_kv_attend_i4: workspace must be 16-byte aligned");
  if (((uintptr_t)q & 7) || ((uintptr_t)o & 7) || ((uintptr_t)kv_data & 15) || ((uintptr_t)kv_param & 3) || (q_token_stride & 3) ||
      (q_head_stride & 3) || (o_token_stride & 3) || (o_head_stride & 3))
    return fail(QR_EALIGN, "qr_kv_attend_i4: q and o must be 8-byte aligned with strides that are multiples of 4, the pages 16-byte aligned");
  KvAttendParams p = {};
  p.o = reinterpret_cast<__half*>(o); p.q = reinterpret_cast<const __half*>(q);
  p.data = reinterpret_cast<const uint8_t*>(kv_data); p.param = reinterpret_cast<const __half2*>(kv_param);
  p.indptr = kv_indptr; p.indices = kv_indices; p.last_page_offset = last_page_offset; p.qo_indptr = qo_indptr;
  p.q_ts = q_token_stride; p.q_hs = q_head_stride; p.o_ts = o_token_stride; p.o_hs = o_head_stride;
  p.total_q = total_q; p.batch = batch; p.layers = num_layers; p.layer = layer; p.kv_heads = num_kv_heads; p.group = group;
  p.page_size = page_size; p.num_pages = num_pages; p.num_indices = num_indices < 0x7fffffff ? num_indices : 0x7fffffff;
  p.page_div = make_fastdiv((uint32_t)page_size); p.group_div = make_fastdiv((uint32_t)group);
  p.window = window; p.sinks = window > 0 ? sink_tokens : 0; p.hadamard_q = hadamard_q;
  p.status = kernel_status_ptr();
  const int64_t rows = max_q_len * group;
  bool tc = false;
  size_t bytes = 0;
  if (const int rc = kv_pick_kernel(p, rows, &tc, &bytes)) return rc;
  return tc ? launch_kv_attend_tc(p, rows, workspace, workspace_bytes, (cudaStream_t)stream) : launch_kv_attend_rows(p, rows, (cudaStream_t)stream);
}

extern "C" size_t qr_kv_attend_workspace_bytes(int64_t num_indices, int page_size, int64_t total_q, int64_t max_q_len, int batch,
                                               int num_q_heads, int num_kv_heads, int window, int sink_tokens) {
  using namespace qr;
  if (num_indices < 0 || page_size < 1 || total_q < 1 || total_q > 0x3fffffffll || max_q_len < 1 || batch < 1 || num_kv_heads < 1 || num_q_heads < num_kv_heads ||
      num_q_heads % num_kv_heads || window < 0 || sink_tokens < 0 || max_q_len > total_q)
    return 0;
  KvAttendParams p = {};
  p.num_indices = num_indices < 0x7fffffff ? num_indices : 0x7fffffff;
  p.page_size = page_size; p.total_q = total_q; p.batch = batch; p.kv_heads = num_kv_heads;
  p.group = num_q_heads / num_kv_heads; p.window = window; p.sinks = window > 0 ? sink_tokens : 0;
  bool tc = false;
  size_t bytes = 0;
  return kv_pick_kernel(p, max_q_len * p.group, &tc, &bytes) == QR_OK && tc ? bytes : 0;
}
