// Attention over the paged 4-bit cache for many query rows per KV head (chunks of a prompt): both products on the
// 5th-generation tensor cores.  Same operator, masks and layouts as kv_attend_rows.cu.
//
// One CTA takes up to 256 query rows of one (sequence, KV head) -- row = (new token, query head of the group), so a
// group shares the tokens it reads -- as two tiles of 128, and walks over the visible tokens in blocks of 96:
//   S_i = Q_i (16 + Ck)^T          tcgen05.mma 128 x 48 x 128 twice, Q and the key codes in shared memory
//   P_i = softmax weights          S from tensor memory to registers and back as fp16
//   O_i += P_i Cv                  tcgen05.mma 128 x 144 x 48 twice, P from tensor memory, the value codes in shared memory
// The tensor cores see the codes, which are exact in fp16, never dequantised keys or values: scales and zero points
// of a token are folded into its column of S and into its weight.  With s' = sigma 2^-k, sigma in [1, 2),
//   score_t = s_t S_t - (z_t + 16 s_t) sum(q),   w_t = exp2(score_t + log2 sigma_t - M),   Cv = (c' - 7.5) 2^-k,
//   l = sum w / sigma,   y = sum w (z' / sigma - 7.5 2^-k),   o = (O - y) / l.
// l and y are four more rows of the transposed values (128 .. 131: 2^10 / sigma and z' / sigma - .., each as the sum of two
// fp16 numbers, which is exact to 2^-22), so the same rounded weights are in all sums and the softmax has no sums to make;
// 144 is the next multiple of 16.  The fp16 rounding of w is the only one in front of the result's own, and a rounding d of
// weight t moves the result by d (v_t - o) / l.
// M does not follow the maximum: it is set 1 below the first one and moves, in whole steps, only where a weight would pass
// 2^15 (all rows of the warp that have grown by 2 move then; what is summed up in tensor memory is multiplied through, by
// powers of two, which round nothing).  So weights are made in one pass, without looking for a maximum first, and the
// normal fp16 range reaches down to 2^-14 of the first largest or further.  The fp16 range ends below: a weight under 2^-25
// of the reference's unit is 0 in all sums, so that next to one token that dominates by as much, n such tokens lose up to
// n 2^-25 of the softmax (2^-9 for 65536 of them).
//
// S is made and used in halves of 48 tokens with a buffer each, the weights lie over the half of S they came from: while
// the softmax is on one half, the tensor cores make the products of the other and then its next scores.
//
// Warps: two warpgroups make the softmax of one row tile each, four warps unpack keys and make the numbers of a token, four
// unpack values, two issue the MMAs of a row tile each.  A token's
// numbers are per COLUMN of S, so a thread that owned a whole row would have to read all of them: S is read
// with the 16x256b shape instead, which gives a lane two neighbouring columns of eight in four rows, the numbers of
// a column pair serve four rows, and a row's maximum is two shuffles away.  Unpacking: keys as they stand (two
// logical instructions per pair of codes; the query follows their order), values transposed by byte permutes over
// eight tokens, so that both operands are K-major 128-byte-swizzled tiles written by conflict-free 16-byte stores.
// Few tiles: several CTAs share the token axis of a tile and meet in a workspace, or in a cluster where there is none.
//
// Registers: 20 warps, five per scheduler, start with 96 each; the softmax warps go up to 160, the unpacking warps down to
// 64 and the MMA warpgroup to 32 (per scheduler 2 x 160 + 2 x 64 + 32 = 5 x 96).  All waits are bounded (tc_ptx.cuh).
//
// Measured (2048 tokens x 64 heads over 10240 tokens, 8 KV heads): 830 us, 746 TFLOP/s.  A block of 96 tokens takes 4800
// cycles: in each half the softmax of a warp takes 2300 -- 325 until S has arrived, 750 for scores (a part of them now made
// while S arrives), 760 for weights (exp2 alone would take 384 of a scheduler's special function unit per warp, and there
// are two), 450 waiting -- which is what bounds it; the tensor cores are busy half of the time.  A CTA takes 15000 cycles before its first scores.
#include "kv_common.cuh"
#include "tc_ptx.cuh"

#include <math.h>

namespace qr {

constexpr int kAtThreads = 640;
constexpr int kAtRows = 256;
constexpr int kAtTok = 96, kAtHalf = 48;                  // tokens of a block; columns of a score buffer
constexpr int kAtQTile = 128 * 128 * 2;                   // bytes: 128 rows, two atoms of 64 dimensions
constexpr int kAtKTile = kAtTok * 128 * 2;                // 96 tokens, two atoms of 64 dimensions
constexpr int kAtVRows = 144;                             // 128 dimensions, 4 rows for the sums, filled up to a multiple of 16
constexpr int kAtVAtom = kAtVRows * 128;                  // 64 tokens (of the second atom 32 are used)
constexpr int kAtVTile = 2 * kAtVAtom;
constexpr int kAtPairFloats = 8;                          // per column pair: ks ks kz kz | lv lv - -
constexpr uint32_t kTmem = 0;                             // the CTA owns all 512 columns of tensor memory, from 0 on
constexpr uint32_t kTmemO = kTmem, kTmemS = kTmem + 2 * kAtVRows;     // O_0 O_1 (144 columns each), then S of (tile, half)
constexpr int kAtParStages = 3;
constexpr float kAtTop = 15.0f;                           // weights are at most 2^15
constexpr float kAtMove = 2.0f;                           // where one row has to move, all that have grown by this much do
constexpr uint32_t kAtIdescS = (1u << 4) | ((48u >> 3) << 17) | ((128u >> 4) << 24);    // fp16 x fp16 -> fp32, K-major, 128 x 48
constexpr uint32_t kAtIdescO = (1u << 4) | ((144u >> 3) << 17) | ((128u >> 4) << 24);   // 128 x 144

struct AtShared {
  float par[kAtParStages][kAtTok / 2][kAtPairFloats];
  long long row[2][2][kAtTok];                            // [keys / values][block & 1] rows of the tokens, -1: not read
  __half vscale[2][kAtTok];                               // [block & 1] 2^-k of the tokens' value codes
  float qsum[kAtRows];
  int pos[kAtRows];
  float m[kAtRows], l[kAtRows];
  unsigned long long bars[32];
  uint32_t tmem;
  int abort;
};
constexpr size_t kAtSmem = 1024 + 2 * kAtQTile + 2 * kAtKTile + 2 * kAtVTile + sizeof(AtShared);
static_assert(kAtSmem <= 227 * 1024, "shared memory");

// The MMAs and commits are written for a warp whose lanes all run the issuing loop: addresses and descriptors then stay in
// uniform registers, and only the instruction itself is predicated on the elected lane.
__device__ __forceinline__ void umma_f16_ss(uint32_t lead, uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 q, %0, 0;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "mov.b64 da, {%2, %4};\n\t"
      "mov.b64 db, {%3, %4};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%1], da, db, %5, p;\n\t}"
      ::"r"(lead), "r"(d), "r"(a_lo), "r"(b_lo), "n"(kDescHiKmajorSw128), "n"(kAtIdescS), "r"(acc) : "memory");
}
__device__ __forceinline__ void umma_f16_ts(uint32_t lead, uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 db;\n\t"
      "setp.ne.b32 q, %0, 0;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "mov.b64 db, {%3, %4};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%1], [%2], db, %5, p;\n\t}"
      ::"r"(lead), "r"(d), "r"(a_tmem), "r"(b_lo), "n"(kDescHiKmajorSw128), "n"(kAtIdescO), "r"(acc) : "memory");
}
__device__ __forceinline__ void umma_commit_lead(uint32_t lead, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %0, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n\t}"
      ::"r"(lead), "r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t elect_lane() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r));
  return r;
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
__device__ __forceinline__ void tmem_ld_16x256_x4(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_ld_16x256_x2(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st_16x256_x4(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x4.b32 [%16], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
      ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st_16x256_x2(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.16x256b.x2.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};"
               ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st_16x128_x2(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x2.b32 [%4], {%0, %1, %2, %3};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(taddr) : "memory");
}
// 16 lanes x 16 columns of fp16 pairs (32 matrix columns): r[2 k] is row g, r[2 k + 1] row g + 8, column pair 4 k + c.
__device__ __forceinline__ void tmem_st_16x128_x4(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};"
               ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr) : "memory");
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
__device__ __forceinline__ uint32_t at_centred_pair(uint32_t w, __half2 scale, __half2 bias) {     // (c - 7.5) 2^-k, exact
  const uint32_t x = code_pair<J>(w);
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&x), scale, bias);
  return *reinterpret_cast<const uint32_t*>(&r);
}
// Value parameters of a token.  The weight of a token carries sigma = s' 2^k in [1, 2), its codes 2^-k, so that weights compare
// as the softmax does: with s' itself in them, the weights of tokens with small scales would be rounded at the fp16 numbers'
// lower end next to a token with a large one.  k lies in -11 .. 23, where (c - 7.5) 2^-k is exact (and 23.5 2^11 finite);
// scales above 2^12 then give a sigma of up to 4.3.  The centre z' / sigma - 7.5 2^-k is a value of the row over sigma: in
// the range of fp16 as the row is.
struct AtValue {
  float sigma, down, z, bad;                              // sigma, 2^-k, z' / sigma - 7.5 2^-k, 0 or NaN
};
__device__ __forceinline__ AtValue at_value(uint32_t raw) {
  float2 v = __half22float2(*reinterpret_cast<const __half2*>(&raw));
  AtValue r;
  r.bad = (v.x - v.x) + (v.y - v.y);
  // scales of a cache are positive; below 2^-22 the codes of a token cannot move an fp16 result by more than 2^-18
  if (!(v.x >= 2.384185791015625e-07f)) v.x = 2.384185791015625e-07f;
  if (r.bad != 0.0f) v = make_float2(1.0f, 0.0f);
  const int k = max(127 - (__float_as_int(v.x) >> 23), -11);
  r.down = __int_as_float((127 - k) << 23);
  r.sigma = v.x * __int_as_float((127 + k) << 23);
  r.z = fmaf(-7.5f, r.down, __fdividef(v.y, r.sigma));
  return r;
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

// Tile of rows of a unit.  The last tiles of a sequence see the most tokens: they start first.
__device__ __forceinline__ int at_tile(const KvAttendParams& p, int unit) {
  const int x = unit / p.kv_heads;
  if (!p.sorted) return p.max_tiles - 1 - x;
  const int rank = x / p.tiles_per_seq;
  return rank * p.tiles_per_seq + p.tiles_per_seq - 1 - (x - rank * p.tiles_per_seq);
}

// What a lane of a softmax warp keeps of its four rows (g + 8 x of the warp's 32).
struct AtRows {
  float m[4], qs[4];
};

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// -infinity for the columns of a pair that a row at position pos does not see; t: token of the first
__device__ __forceinline__ void at_hide(float& v0, float& v1, int t, int pos, int window, int sinks) {
  const int lo = window > 0 ? pos - window : -1;
  if (t > pos || (t <= lo && t >= sinks)) v0 = -INFINITY;
  if (t + 1 > pos || (t + 1 <= lo && t + 1 >= sinks)) v1 = -INFINITY;
}

// 48 columns of S of the warp's 32 rows: s[0] rows 0 - 15, s[1] rows 16 - 31, pairs 4 k + 2 (row / 8 & 1) of column group k.
__device__ __forceinline__ void at_fetch(uint32_t (&s)[2][24], uint32_t t_s) {
  tmem_ld_16x256_x4(t_s, s[0]);
  tmem_ld_16x256_x4(t_s + (16u << 16), s[1]);
  tmem_ld_16x256_x2(t_s + 32, s[0] + 16);
  tmem_ld_16x256_x2(t_s + 32 + (16u << 16), s[1] + 16);
}

// What the scores of 48 columns have besides S: u = log2 sigma - (z + 16 s) sum(q) - M, of the four rows of a lane.
__device__ __forceinline__ void at_offsets(uint64_t (&u)[4][6], const float* par, const AtRows& w) {
#pragma unroll
  for (int k = 0; k < 6; ++k) {
    const float2 a = *reinterpret_cast<const float2*>(par + 4 * k * kAtPairFloats + 2);
    const float2 b = *reinterpret_cast<const float2*>(par + 4 * k * kAtPairFloats + 4);
    const uint64_t kz = f2_pack(a.x, a.y), lv = f2_pack(b.x, b.y);
#pragma unroll
    for (int x = 0; x < 4; ++x)                           // +infinity before the row has seen a token: M has to be set
      u[x][k] = f2_add(f2_fma(kz, f2_pack(w.qs[x], w.qs[x]), lv), f2_pack(-w.m[x], -w.m[x]));
  }
}
// The exponents of 48 columns, relative to M, in place of S; the lane's largest is returned.
__device__ __forceinline__ float at_scores(uint32_t (&s)[2][24], const float* par, const uint64_t (&u)[4][6]) {
  float top0 = -INFINITY, top1 = -INFINITY;
#pragma unroll
  for (int k = 0; k < 6; ++k) {
    const float2 a = *reinterpret_cast<const float2*>(par + 4 * k * kAtPairFloats);
    const uint64_t ks = f2_pack(a.x, a.y);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      uint32_t* r = s[x >> 1] + 4 * k + 2 * (x & 1);
      float v0, v1;
      f2_unpack(f2_fma(ks, f2_pack(__uint_as_float(r[0]), __uint_as_float(r[1])), u[x][k]), v0, v1);
      if (x & 1) top1 = max3(top1, v0, v1); else top0 = max3(top0, v0, v1);
      r[0] = __float_as_uint(v0);
      r[1] = __float_as_uint(v1);
    }
  }
  return fmaxf(top0, top1);
}

// Hides what the rows do not see (pos: positions of the warp's rows, t: token of the lane's first column); the largest of
// what is left.
__device__ __forceinline__ float at_mask(uint32_t (&s)[2][24], const int* pos, int t, int window, int sinks) {
  float top = -INFINITY;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const int ps = pos[8 * x];
#pragma unroll
    for (int k = 0; k < 6; ++k) {
      uint32_t* r = s[x >> 1] + 4 * k + 2 * (x & 1);
      float v0 = __uint_as_float(r[0]), v1 = __uint_as_float(r[1]);
      at_hide(v0, v1, t + 8 * k, ps, window, sinks);
      top = max3(top, v0, v1);
      r[0] = __float_as_uint(v0);
      r[1] = __float_as_uint(v1);
    }
  }
  return top;
}

// The weights of 48 columns, as fp16 to tensor memory.
__device__ __forceinline__ void at_weights(const uint32_t (&s)[2][24], uint32_t t_p) {
  uint32_t pk[2][12];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
#pragma unroll
    for (int e = 0; e < 12; ++e) {
      const __half2 wh = __floats2half2_rn(ex2(__uint_as_float(s[x][2 * e])), ex2(__uint_as_float(s[x][2 * e + 1])));
      pk[x][e] = *reinterpret_cast<const uint32_t*>(&wh);
    }
    tmem_st_16x128_x4(t_p + ((uint32_t)x << 20), pk[x]);
    tmem_st_16x128_x2(t_p + 16 + ((uint32_t)x << 20), pk[x] + 8);
  }
}

// The largest exponents of the four rows over 48 columns, relative to nothing.
__device__ __forceinline__ void at_tops(uint32_t (&s)[2][24], const float* par, const AtRows& w, float (&top)[4], bool edge, const int* pos, int t,
                                        int window, int sinks) {
#pragma unroll
  for (int x = 0; x < 4; ++x) top[x] = -INFINITY;
#pragma unroll
  for (int k = 0; k < 6; ++k) {
    const float4 a = *reinterpret_cast<const float4*>(par + 4 * k * kAtPairFloats);
    const float2 b = *reinterpret_cast<const float2*>(par + 4 * k * kAtPairFloats + 4);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const uint32_t* r = s[x >> 1] + 4 * k + 2 * (x & 1);
      float v0 = fmaf(a.x, __uint_as_float(r[0]), fmaf(a.z, w.qs[x], b.x)), v1 = fmaf(a.y, __uint_as_float(r[1]), fmaf(a.w, w.qs[x], b.y));
      if (edge) at_hide(v0, v1, t + 8 * k, pos[8 * x], window, sinks);
      top[x] = max3(top[x], v0, v1);
    }
  }
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 1));
    top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 2));
  }
}

// The largest of the exponents that at_scores left, per row.
__device__ __forceinline__ void at_largest(const uint32_t (&s)[2][24], float (&top)[4]) {
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    top[x] = -INFINITY;
#pragma unroll
    for (int k = 0; k < 6; ++k) {
      const uint32_t* r = s[x >> 1] + 4 * k + 2 * (x & 1);
      top[x] = max3(top[x], __uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 1));
    top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 2));
  }
}

// Multiplies O, the columns of the sums included, by the factors of the four rows, 48 columns at a time.
__device__ __forceinline__ void at_scale_o(uint32_t t_o, const float (&f)[4]) {
  static_assert(kAtVRows % 48 == 0, "columns of O");
#pragma unroll 1
  for (int q = 0; q < kAtVRows / 48; ++q, t_o += 48) {
    uint32_t o[2][24];
    at_fetch(o, t_o);
    tmem_ld_done<24>(o[0]);
    tmem_ld_done<24>(o[1]);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int e = 0; e < 24; ++e) o[h][e] = __float_as_uint(__uint_as_float(o[h][e]) * f[2 * h + ((e >> 1) & 1)]);
      tmem_st_16x256_x4(t_o + ((uint32_t)h << 20), o[h]);
      tmem_st_16x256_x2(t_o + 32 + ((uint32_t)h << 20), o[h] + 16);
    }
  }
  tmem_st_done();
}

// The 32 query rows of a softmax warp: into the Q tile, their sums and positions.  8 dimensions 8 i .. 8 i + 7 lie as
// 0 4 1 5 2 6 3 7, the order in which a word of key codes comes apart.
// (A call: inlined, its registers cost the loop of the softmax 5 %.)
struct AtQuery {
  const __half* q;                                        // first new token of the sequence, first query head of the group
  int64_t ts, hs;                                         // strides of tokens and heads
  FastDiv group_div;
  int group, row0, rows, pos0, hadamard;
};
__device__ __noinline__ void at_load_rows(const AtQuery a, int row0, int lane, unsigned char* tile, float* s_sum, int* s_pos) {
  // all rows on their way at once, each to its place in the two swizzled atoms, in their natural order; two at a time where they are
  // 16-byte aligned
  const bool wide = ((reinterpret_cast<uintptr_t>(a.q) & 15) | (a.ts & 7) | (a.hs & 7)) == 0;
  const int per = wide ? 2 : 1, piece = wide ? lane & 15 : lane, bytes = wide ? 16 : 8;
  {
    int r = row0 + (wide ? lane >> 4 : 0);
    const uint32_t at = smem_u32(tile) + (piece * bytes >> 7) * (kAtQTile / 2) + (piece * bytes & 15), ch = (piece * bytes >> 4) & 7;
    const __half* mine = a.q + piece * (bytes / 2);
#pragma unroll 2
    for (; r < row0 + 32; r += per) {
      const uint32_t dst = at + (r & 127) * 128 + ((ch ^ (r & 7)) << 4);
      const bool on = r < a.rows;
      const int tok = fast_div(a.row0 + r, a.group_div), hh = a.row0 + r - tok * a.group;
      const __half* src = on ? mine + tok * a.ts + hh * a.hs : a.q;
      if (wide) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
      else asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(on ? 8 : 0) : "memory");
      if (piece == 0) s_pos[r] = on ? a.pos0 + tok : -1;
    }
  }
  asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
  __syncwarp();
  // a lane has 64 dimensions of a row, lane ^ 16 the others: one exchange (shuffles are what this would otherwise wait for)
#pragma unroll 1
  for (int r = row0 + (lane & 15); r < row0 + 32; r += 16) {
    unsigned char* mine = tile + (lane >> 4) * (kAtQTile / 2) + (r & 127) * 128;
    float x[64];
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const uint4 raw = *reinterpret_cast<const uint4*>(mine + ((c ^ (r & 7)) << 4));
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
        x[8 * c + 2 * e] = f.x; x[8 * c + 2 * e + 1] = f.y;
      }
    }
    if (a.hadamard) {
#pragma unroll
      for (int h = 1; h < 64; h <<= 1)
#pragma unroll
        for (int e = 0; e < 64; ++e)
          if ((e & h) == 0) {
            const float p = x[e], m = x[e + h];
            x[e] = p + m;
            x[e + h] = p - m;
          }
      const float sg = (lane & 16) ? -1.0f : 1.0f;
#pragma unroll
      for (int e = 0; e < 64; ++e)
        x[e] = __half2float(__float2half_rn(fmaf(x[e], sg, __shfl_xor_sync(0xffffffffu, x[e], 16)) * 0.08838834764831845f));
    }
    float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      uint32_t h[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        part[e] += x[8 * c + e] + x[8 * c + e + 4];
        const __half2 hv = __floats2half2_rn(x[8 * c + e], x[8 * c + e + 4]);
        h[e] = *reinterpret_cast<const uint32_t*>(&hv);
      }
      *reinterpret_cast<uint4*>(mine + ((c ^ (r & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
    }
    float sum = (part[0] + part[1]) + (part[2] + part[3]);
    sum += __shfl_xor_sync(0xffffffffu, sum, 16);
    if (lane < 16) s_sum[r] = sum;
  }
}

__global__ void __launch_bounds__(kAtThreads, 1)
kv_attend_tc_kernel(const __grid_constant__ KvAttendParams p) {
  extern __shared__ unsigned char s_raw[];
  const uint32_t base = (smem_u32(s_raw) + 1023u) & ~1023u;
  unsigned char* smem = s_raw + (base - smem_u32(s_raw));
  // [Q tile 0, Q tile 1][K 2 stages][V 2 stages][AtShared]; the merge area is Q, K and a part of V, the fp16 result of a row
  // tile goes through its Q tile
  const uint32_t s_q = base, s_k = base + 2 * kAtQTile, s_v = s_k + 2 * kAtKTile;
  AtShared& sh = *reinterpret_cast<AtShared*>(smem + 2 * kAtQTile + 2 * kAtKTile + 2 * kAtVTile);
  const uint32_t bars = smem_u32(sh.bars);
  const uint32_t k_full = bars, k_empty = bars + 16, v_full = bars + 32, v_empty = bars + 48, par_full = bars + 64, s_full = bars + 88,
                 p_full = bars + 120, pv_done = bars + 152, o_full = bars + 168, q_full = bars + 184;   // 2 2 2 2 3 [2][2] [2][2] 2 2 2
  volatile int* abort_flag = &sh.abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t crank = 0;
  const int share = blockIdx.x - p.whole;                 // of the units that are split
  const int splits = share < 0 ? 1 : p.splits;
  const int unit = share < 0 ? blockIdx.x : p.whole + share / p.splits;
  const bool joined = splits > 1, clustered = joined && !p.part;
  if (joined) crank = share % p.splits;                   // also the rank within a cluster
  const int head_kv = unit % p.kv_heads;
  const KvTile w = kv_find_tile(p, at_tile(p, unit), kAtRows, lane);
  if (w.rows == 0) return;                                // the whole cluster has the same tile
  const int tiles = w.rows > 128 ? 2 : 1;
  const int p_min = w.pos0 + fast_div(w.row0, p.group_div), p_max = w.pos0 + fast_div(w.row0 + w.rows - 1, p.group_div);
  const KvBlocks blk = kv_blocks<kAtTok>(p_min, p_max, p.window, p.sinks);
  const int per = (blk.count + splits - 1) / splits;
  const int begin = (int)crank * per;
  const int n = max(min(begin + per, blk.count) - begin, 0);

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(k_full + 8 * s, 4); mbar_init(k_empty + 8 * s, tiles);
      mbar_init(v_full + 8 * s, 4); mbar_init(v_empty + 8 * s, tiles);
      mbar_init(s_full + 16 * s, 1); mbar_init(s_full + 16 * s + 8, 1);
      mbar_init(p_full + 16 * s, 4); mbar_init(p_full + 16 * s + 8, 4);
      mbar_init(pv_done + 8 * s, 1); mbar_init(o_full + 8 * s, 1); mbar_init(q_full + 8 * s, 4);
    }
    for (int s = 0; s < kAtParStages; ++s) mbar_init(par_full + 8 * s, 4);
    sh.abort = 0;
    fence_mbar_init();
  }
  if (warp == 16) {
    tmem_alloc(smem_u32(&sh.tmem), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  if (warp < 8) {
    // ---------------------------------------------------------------- softmax: 32 rows of a row tile
    regs_inc<160>();
    const int i = warp >> 2, g = lane >> 2, c = lane & 3;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;                    // first tensor-memory lane of the warp, << 16
    const uint32_t t_s = kTmemS + i * (2 * kAtHalf) + lanes, t_o = kTmemO + i * kAtVRows + lanes;
    const int row0 = i * 128 + (warp & 3) * 32;                           // the lane's rows: row0 + g + 8 x, x = 0 .. 3
    const int* pos = &sh.pos[row0 + g];
    if (i < tiles) {
      const AtQuery a = {p.q + w.tok0 * p.q_ts + (int64_t)(head_kv * p.group) * p.q_hs, p.q_ts, p.q_hs, p.group_div, p.group, w.row0, w.rows,
                         w.pos0, p.hadamard_q};
      at_load_rows(a, row0, lane, smem + i * kAtQTile, sh.qsum, sh.pos);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full + 8 * i);
    }
    AtRows rw;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      rw.m[x] = -INFINITY;
      rw.qs[x] = i < tiles ? sh.qsum[row0 + g + 8 * x] : 0.0f;
    }
    bool ok = i < tiles;
    // One copy of the code for all half blocks, the rare branches out of its way: with the loop unrolled, the warps of a
    // scheduler spent a third of their time on instruction fetches.  The next scores are asked for as soon as the
    // registers of these are free.
    uint32_t s[2][24];
    int ring = 0, ring_phase = 0;
    const float* par = &sh.par[0][c][0];
    if (ok && n > 0) {
      ok = mbar_wait(par_full, 0, abort_flag, p.status, 71) && mbar_wait(s_full + 16 * i, 0, abort_flag, p.status, 72);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      at_fetch(s, t_s);
    }
    int t0 = kv_block_index(blk, begin) * kAtTok;         // first token of the half block
#pragma unroll 1
    for (int h = 0; ok && h < 2 * n; ++h) {
      const bool edge = t0 + kAtHalf - 1 > p_min || (p.window > 0 && t0 <= p_max - p.window && t0 + kAtHalf - 1 >= p.sinks);
      const uint32_t t_sb = t_s + (h & 1) * kAtHalf;
      uint64_t u[4][6];
      at_offsets(u, par, rw);                             // while S is on its way
      tmem_ld_done<24>(s[0]);
      tmem_ld_done<24>(s[1]);
      float top = at_scores(s, par, u);
      if (__builtin_expect(edge, 0)) top = at_mask(s, pos, t0 + 2 * c, p.window, p.sinks);
      if (__builtin_expect(__any_sync(0xffffffffu, top > kAtTop), 0)) {
        // a weight would pass 2^15, or a row sees its first token: M moves, O follows by powers of two (or 0)
        float mn[4], f[4];
        const bool fresh = __any_sync(0xffffffffu, fminf(fminf(rw.m[0], rw.m[1]), fminf(rw.m[2], rw.m[3])) == -INFINITY);
        if (fresh) {                                      // no exponents yet: the scores are looked at once more
          at_fetch(s, t_sb);
          tmem_ld_done<24>(s[0]);
          tmem_ld_done<24>(s[1]);
          at_tops(s, par, rw, mn, edge, pos, t0 + 2 * c, p.window, p.sinks);
        } else {
          at_largest(s, mn);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          if (fresh) {
            const bool move = mn[x] - rw.m[x] > kAtMove;
            const float to = ceilf(mn[x]) - 1.0f;
            f[x] = !move ? 1.0f : rw.m[x] == -INFINITY ? 0.0f : ex2(rw.m[x] - to);
            rw.m[x] = move ? to : rw.m[x];
          } else {
            mn[x] = mn[x] > kAtMove ? ceilf(mn[x]) - 1.0f : 0.0f;
            f[x] = ex2(-mn[x]);
            rw.m[x] += mn[x];
          }
        }
        if (h > 0) {                                      // the products of half h - 1 may still be on their way
          ok = mbar_wait(pv_done + 8 * i, (h - 1) & 1, abort_flag, p.status, 73) && ok;
          __syncwarp();
          tc_fence_after();
          at_scale_o(t_o, f);
        }
        if (fresh) {
          at_offsets(u, par, rw);
          at_scores(s, par, u);
          if (edge) at_mask(s, pos, t0 + 2 * c, p.window, p.sinks);
        } else {
#pragma unroll
          for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int k = 0; k < 6; ++k)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                uint32_t& v = s[x >> 1][4 * k + 2 * (x & 1) + e];
                v = __float_as_uint(__uint_as_float(v) - mn[x]);
              }
        }
      }
      at_weights(s, t_sb);                                // in place of S, which is in registers
      tmem_st_done();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full + 16 * i + 8 * (h & 1));
      if (h + 1 == 2 * n) break;
      t0 += kAtHalf;
      par += kAtHalf / 2 * kAtPairFloats;
      if (h & 1) {                                        // the block is done
        if (++ring == kAtParStages) { ring = 0; ring_phase ^= 1; }
        par = &sh.par[ring][c][0];
        t0 = kv_block_index(blk, begin + ((h + 1) >> 1)) * kAtTok;
        ok = mbar_wait(par_full + 8 * ring, ring_phase, abort_flag, p.status, 71) && ok;
      }
      ok = mbar_wait(s_full + 16 * i + 8 * ((h + 1) & 1), ((h + 1) >> 1) & 1, abort_flag, p.status, 72) && ok;
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      at_fetch(s, t_s + ((h + 1) & 1) * kAtHalf);
    }
    ok = __all_sync(0xffffffffu, ok);
    if (ok && n > 0) {
      ok = mbar_wait(o_full + 8 * i, 0, abort_flag, p.status, 80);
      ok = __all_sync(0xffffffffu, ok);
    }
    // the merge area of one row tile lies over operands of the other, whose MMAs may still be running
    __syncwarp();
    if (clustered) asm volatile("bar.sync 3, 256;" ::: "memory");
    if (ok) {
      tc_fence_after();
      // the sums: columns 128, 129 (2^10 w / sigma, in two parts) in lane c = 0, 130, 131 (w (z' / sigma - ..)) in lane c = 1
      float l[4], y[4];
#pragma unroll
      for (int q2 = 0; q2 < 2; ++q2) {
        uint32_t o[8];
        if (n > 0) {
          tmem_ld_16x256_x2(t_o + 128 + ((uint32_t)q2 << 20), o);
          tmem_ld_done<8>(o);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = 0;
        }
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const float sum = __uint_as_float(o[2 * hh]) + __uint_as_float(o[2 * hh + 1]);
          l[2 * q2 + hh] = __shfl_sync(0xffffffffu, sum, lane & ~3) * 0.0009765625f;
          y[2 * q2 + hh] = __shfl_sync(0xffffffffu, sum, (lane & ~3) + 1);
        }
      }
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
        for (int hh = 0; hh < 2; ++hh) {
          const float ll = q4 & 1 ? l[2 + hh] : l[hh], yy = q4 & 1 ? y[2 + hh] : y[hh];
          const int r = row0 + 16 * (q4 & 1) + 8 * hh + g;
          const float inv = joined ? 1.0f : (ll != 0.0f ? 1.0f / ll : 0.0f);      // a row that sees nothing gives zeros
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float e0 = (__uint_as_float(o[4 * k + 2 * hh]) - yy) * inv, e1 = (__uint_as_float(o[4 * k + 2 * hh + 1]) - yy) * inv;
            const int col = 64 * (q4 >> 1) + 8 * k + 2 * c;
            if (clustered) {
              *reinterpret_cast<float2*>(smem + at_part_off(r, col >> 2) + (col & 2) * 4) = make_float2(e0, e1);
            } else if (joined) {
              if (n > 0) *reinterpret_cast<float2*>(p.part + ((size_t)share * kAtRows + r) * kHeadDim + col) = make_float2(e0, e1);
            } else {
              const __half2 hv = __floats2half2_rn(e0, e1);
              *reinterpret_cast<__half2*>(smem + r * 256 + (((col >> 3) ^ (r & 7)) << 4) + (col & 7) * 2) = hv;
            }
          }
        }
      }
      if (joined) {
        float* m_out = clustered ? sh.m : p.part + (size_t)(gridDim.x - p.whole) * kAtRows * kHeadDim + (size_t)share * (2 * kAtRows);
        float* l_out = clustered ? sh.l : m_out + kAtRows;
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if (c == 0) { m_out[row0 + g + 8 * x] = rw.m[x]; l_out[row0 + g + 8 * x] = l[x]; }
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
    if (clustered) {
      kv_cluster_barrier();
      // the CTAs of the cluster deal out the rows
      kv_merge_rows<4>(p.splits, (int)crank + p.splits * warp, p.splits * 8, w.rows, lane, sh.m, sh.l,
                       [&](int r) { return smem + at_part_off(r, lane); },
                       [&](int r, float4 v, float inv) {
                         const __half2 h0 = __floats2half2_rn(v.x * inv, v.y * inv), h1 = __floats2half2_rn(v.z * inv, v.w * inv);
                         uint2 out;
                         out.x = *reinterpret_cast<const uint32_t*>(&h0);
                         out.y = *reinterpret_cast<const uint32_t*>(&h1);
                         *reinterpret_cast<uint2*>(at_out_row(p, w, head_kv, r) + 4 * lane) = out;
                       });
      kv_cluster_barrier();                               // nobody leaves while its shared memory may still be read
    }
  } else if (warp < 16) {
    // ---------------------------------------------------------------- unpacking: warps 8 - 11 keys and parameters, 12 - 15 values
    regs_dec<64>();
    const int tid = threadIdx.x & 127, pw = warp & 3;
    const int what = warp >= 12;
    const int first_page = w.first;
    const int tokens = min(p_max + 1, w.seq_len);
    const size_t page_rows = (size_t)p.layers * 2 * p.kv_heads * p.page_size;
    const size_t row_k = ((size_t)p.layer * 2 * p.kv_heads + head_kv) * p.page_size;
    const size_t v_rows = (size_t)p.kv_heads * p.page_size;               // from a key row to the value row of its token
    const size_t row_0 = row_k + (what ? v_rows : 0);
    auto page_id = [&](int j) -> int {
      const int t = kv_block_index(blk, begin + j) * kAtTok + tid;
      return tid < kAtTok && t < tokens ? __ldg(p.indices + first_page + fast_div(t, p.page_div)) : 0;
    };
    auto put_rows = [&](int j, int id) -> long long {
      const int t = kv_block_index(blk, begin + j) * kAtTok + tid;
      long long row = -1;
      if (tid < kAtTok && t < tokens) {
        const int slot = t - fast_div(t, p.page_div) * p.page_size;
        const size_t page = min((size_t)(uint32_t)id, (size_t)p.num_pages - 1);        // an index outside the pool reads its last page
        row = (long long)(page * page_rows + row_0 + slot);
      }
      if (tid < kAtTok) sh.row[what][j & 1][tid] = row;
      __syncwarp();
      asm volatile("bar.sync %0, 128;" ::"r"(1 + what) : "memory");
      return row;
    };
    // a wait that ran out of time sets the abort flag: the others end at once, and what is written then is read by nobody
    int id = 0;
    if (!what) {
      // row (lane & 7) + 8 (warp + 4 it), 16-byte chunk lane / 8
      const float sm_scale = 0.08838834764831845f * 1.4426950408889634f;  // log2(e) / sqrt(128)
      const int kr = (lane & 7) + 8 * pw, kc = lane >> 3;
      uint4 kw[3];
      uint32_t kp = 0, vp = 0;
      auto load = [&](int j, long long mine) {
#pragma unroll
        for (int it = 0; it < 3; ++it) {
          const long long row = sh.row[0][j & 1][kr + 32 * it];
          kw[it] = row >= 0 ? __ldg(reinterpret_cast<const uint4*>(p.data + row * 64 + 16 * kc)) : make_uint4(0, 0, 0, 0);
        }
        kp = 0; vp = 0;
        if (mine >= 0) {
          kp = __ldg(reinterpret_cast<const uint32_t*>(p.param + mine));
          vp = __ldg(reinterpret_cast<const uint32_t*>(p.param + mine + v_rows));
        }
      };
      if (n > 0) {
        load(0, put_rows(0, page_id(0)));
        if (n > 1) id = page_id(1);
      }
      for (int j = 0; j < n; ++j) {
        const int stage = j & 1, ring = j % kAtParStages;
        long long mine = -1;
        if (j + 1 < n) {
          mine = put_rows(j + 1, id);                     // everybody has read the rows of block j - 1
          if (j + 2 < n) id = page_id(j + 2);
        }
        if (j >= 2) {
          mbar_wait(k_empty + 8 * stage, ((j >> 1) + 1) & 1, abort_flag, p.status, 74);
          __syncwarp();
        }
        if (tid < kAtTok) {
          // parameters of token tid; the slot of the ring is free: the scores of block j - 2 were issued after the weights of
          // block j - 3 had been made
          const float2 k2 = __half22float2(*reinterpret_cast<const __half2*>(&kp));
          const AtValue v = at_value(vp);
          const float ks = k2.x * sm_scale;
          float* q = &sh.par[ring][tid >> 1][tid & 1];
          q[0] = ks;
          q[2] = -fmaf(16.0f, ks, k2.y * sm_scale);
          // x - x: 0, or NaN where it is not finite: the weight of such a token is NaN in the rows that see it
          q[4] = __log2f(v.sigma) + ((k2.x - k2.x) + (k2.y - k2.y) + v.bad);
        }
        const uint32_t dst = s_k + stage * kAtKTile + (kc >> 1) * (kAtKTile / 2);
#pragma unroll 1
        for (int r = kr; r < kAtTok; r += 32) {           // the words of the next round move up: see the note on code size
          const uint32_t ww[4] = {kw[0].x, kw[0].y, kw[0].z, kw[0].w};
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int ch = 4 * (kc & 1) + x;
            st_shared16(dst + r * 128 + ((ch ^ (r & 7)) << 4), code_pair<0>(ww[x]), code_pair<1>(ww[x]), code_pair<2>(ww[x]),
                        code_pair<3>(ww[x]));
          }
          kw[0] = kw[1]; kw[1] = kw[2];
        }
        if (j + 1 < n) load(j + 1, mine);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(par_full + 8 * ring);
          mbar_arrive(k_full + 8 * stage);
        }
      }
    } else {
      // warps 0, 1: tokens 8 (lane & 7) + 0 .. 7 of the first atom, 8 bytes (16 dimensions) at 32 warp + 8 (lane / 8); warp 2:
      // tokens 64 + 8 (lane & 3) + 0 .. 7, 8 bytes at 8 (lane / 4); thread t < 96: the rows of the sums for token t
      const int tg = pw < 2 ? lane & 7 : lane & 3;
      const int vt = pw < 2 ? 8 * tg : 64 + 8 * tg, vb = pw < 2 ? 32 * pw + 8 * (lane >> 3) : 8 * (lane >> 2);
      uint2 vw[8];
      uint32_t vp = 0;
      auto load = [&](int j) {
#pragma unroll
        for (int it = 0; it < 8; ++it) {
          const long long row = pw < 3 ? sh.row[1][j & 1][vt + it] : -1;
          vw[it] = row >= 0 ? __ldg(reinterpret_cast<const uint2*>(p.data + row * 64 + vb)) : make_uint2(0, 0);
        }
      };
      auto load_par = [&](long long mine) { vp = mine >= 0 ? __ldg(reinterpret_cast<const uint32_t*>(p.param + mine)) : 0u; };
      long long mine = -1;
      if (n > 0) {
        mine = put_rows(0, page_id(0));
        load_par(mine);
        load(0);
        if (n > 1) id = page_id(1);
      }
      for (int j = 0; j < n; ++j) {
        const int stage = j & 1;
        const AtValue v = at_value(vp);
        if (tid < kAtTok) sh.vscale[stage][tid] = __float2half_rn(v.down);
        if (j + 1 < n) {
          mine = put_rows(j + 1, id);                     // its barrier orders the scales as well
          load_par(mine);
          if (j + 2 < n) id = page_id(j + 2);
        } else {
          __syncwarp();
          asm volatile("bar.sync 2, 128;" ::: "memory");
        }
        if (j >= 2) {
          mbar_wait(v_empty + 8 * stage, ((j >> 1) + 1) & 1, abort_flag, p.status, 75);
          __syncwarp();
        }
        const uint32_t tile = s_v + stage * kAtVTile;
        if (tid < kAtTok) {
          // rows 128 .. 131: 2^10 / sigma and z' / sigma - .., each as the sum of two fp16 numbers; 0 where the token is bad
          const float rv = v.bad == 0.0f ? __fdividef(1024.0f, v.sigma) : 0.0f, zv = v.bad == 0.0f ? v.z : 0.0f;
          const __half rh = __float2half_rn(rv), zh = __float2half_rn(zv);
          const __half part[4] = {rh, __float2half_rn(rv - __half2float(rh)), zh, __float2half_rn(zv - __half2float(zh))};
          unsigned char* at = smem + (tile - base) + (tid >> 6) * kAtVAtom + 128 * 128 + (tid & 7) * 2;
#pragma unroll
          for (int e = 0; e < 4; ++e)                     // row 128 + e: its number mod 8 is e
            *reinterpret_cast<__half*>(at + e * 128 + (((((uint32_t)tid & 63) >> 3) ^ e) << 4)) = part[e];
        }
        if (pw < 3) {
          const uint32_t dst = tile + (pw < 2 ? 0 : kAtVAtom);
          __half2 sc[4], bi[4];
          const uint4 raw = *reinterpret_cast<const uint4*>(&sh.vscale[stage][vt]);
          const uint32_t rs[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            sc[i] = *reinterpret_cast<const __half2*>(&rs[i]);
            bi[i] = __hmul2(sc[i], __float2half2_rn(-23.5f));
          }
#pragma unroll 1
          for (int d0 = 2 * vb; d0 < 2 * vb + 16; d0 += 8) {  // eight dimensions: one word of each token
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              uint32_t x[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) x[i] = __byte_perm(vw[2 * i].x, vw[2 * i + 1].x, half ? 0x7632u : 0x5410u);
              const uint32_t at = dst + (d0 + 4 * half) * 128;              // d0 is a multiple of 8
              st_shared16(at + ((tg ^ (4 * half)) << 4), at_centred_pair<0>(x[0], sc[0], bi[0]), at_centred_pair<0>(x[1], sc[1], bi[1]),
                          at_centred_pair<0>(x[2], sc[2], bi[2]), at_centred_pair<0>(x[3], sc[3], bi[3]));
              st_shared16(at + 128 + ((tg ^ (4 * half + 1)) << 4), at_centred_pair<1>(x[0], sc[0], bi[0]), at_centred_pair<1>(x[1], sc[1], bi[1]),
                          at_centred_pair<1>(x[2], sc[2], bi[2]), at_centred_pair<1>(x[3], sc[3], bi[3]));
              st_shared16(at + 256 + ((tg ^ (4 * half + 2)) << 4), at_centred_pair<2>(x[0], sc[0], bi[0]), at_centred_pair<2>(x[1], sc[1], bi[1]),
                          at_centred_pair<2>(x[2], sc[2], bi[2]), at_centred_pair<2>(x[3], sc[3], bi[3]));
              st_shared16(at + 384 + ((tg ^ (4 * half + 3)) << 4), at_centred_pair<3>(x[0], sc[0], bi[0]), at_centred_pair<3>(x[1], sc[1], bi[1]),
                          at_centred_pair<3>(x[2], sc[2], bi[2]), at_centred_pair<3>(x[3], sc[3], bi[3]));
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) vw[i].x = vw[i].y;
          }
        }
        if (j + 1 < n) load(j + 1);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(v_full + 8 * stage);
      }
    }
    if (clustered) { kv_cluster_barrier(); kv_cluster_barrier(); }
  } else {
    // ---------------------------------------------------------------- MMA issue
    regs_dec<32>();
    const int i = warp - 16;                              // a warp per row tile: they do not wait for each other
    if (i < tiles && n > 0) {
      const uint32_t lead = elect_lane();
      const uint32_t t_s = kTmemS + i * (2 * kAtHalf), t_o = kTmemO + i * kAtVRows;
      const uint32_t q = desc_lo(s_q) + i * (kAtQTile >> 4);
      bool ok = mbar_wait(q_full + 8 * i, 0, abort_flag, p.status, 74) && mbar_wait(k_full, 0, abort_flag, p.status, 76);
      // scores of a half of the block in K stage `stage`
      auto scores = [&](int buf, int stage) {
        const uint32_t b = desc_lo(s_k) + stage * (kAtKTile >> 4) + buf * (kAtHalf * 128 >> 4), d = t_s + buf * kAtHalf;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks)
          umma_f16_ss(lead, d, q + (ks >> 2) * (kAtQTile / 2 >> 4) + (ks & 3) * 2, b + (ks >> 2) * (kAtKTile / 2 >> 4) + (ks & 3) * 2, ks > 0);
        umma_commit_lead(lead, s_full + 16 * i + 8 * buf);
      };
      if (ok) {
        tc_fence_after();
#pragma unroll 1
        for (int buf = 0; buf < 2; ++buf) scores(buf, 0);
        umma_commit_lead(lead, k_empty);
      }
#pragma unroll 1
      for (int j = 0; ok && j < n; ++j) {
        const int stage = j & 1;
        const bool more = j + 1 < n;
        ok = mbar_wait(v_full + 8 * stage, (j >> 1) & 1, abort_flag, p.status, 77);
        if (ok && more) ok = mbar_wait(k_full + 8 * (stage ^ 1), ((j + 1) >> 1) & 1, abort_flag, p.status, 78);
#pragma unroll 1
        for (int buf = 0; ok && buf < 2; ++buf) {
          ok = mbar_wait(p_full + 16 * i + 8 * buf, j & 1, abort_flag, p.status, 79);
          if (!ok) break;
          tc_fence_after();
          // 16 tokens at 48 buf + 16 ks: the first four steps lie in the first atom
          const uint32_t b = desc_lo(s_v) + stage * (kAtVTile >> 4), b0 = b + buf * 6, b1 = buf ? b + (kAtVAtom >> 4) : b + 2;
          const uint32_t first = buf | j;
          umma_f16_ts(lead, t_o, t_s + buf * kAtHalf, b0, first);
          umma_f16_ts(lead, t_o, t_s + buf * kAtHalf + 8, b1, 1u);
          umma_f16_ts(lead, t_o, t_s + buf * kAtHalf + 16, b1 + 2, 1u);
          // scores of half h imply the products of half h - 2: the softmax is at most one phase of pv_done behind
          umma_commit_lead(lead, (more || !buf ? pv_done : o_full) + 8 * i);
          if (more) scores(buf, stage ^ 1);                 // over the weights, which the products before it have read
        }
        if (ok) {
          if (more) umma_commit_lead(lead, k_empty + 8 * (stage ^ 1));
          umma_commit_lead(lead, v_empty + 8 * stage);
        }
      }
      __syncwarp();
    }
    if (clustered) { kv_cluster_barrier(); kv_cluster_barrier(); }
  }
  drain_after_abort(abort_flag);
  tc_fence_before();
  __syncthreads();
  if (warp == 16) {
    tc_fence_after();
    tmem_dealloc(kTmem, 512);
  }
}

// Shares of the CTAs of a unit that went to global memory joined into the result: a warp per row.
__global__ void __launch_bounds__(256) kv_attend_join_kernel(const KvAttendParams p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x / (kAtRows / 8), unit = p.whole + split, r = (blockIdx.x % (kAtRows / 8)) * 8 + warp;
  const int head_kv = unit % p.kv_heads;
  const KvTile w = kv_find_tile(p, at_tile(p, unit), kAtRows, lane);
  if (r >= w.rows) return;
  const int cta = split * p.splits;
  const float* stat = p.part + (size_t)(gridDim.x / (kAtRows / 8)) * p.splits * kAtRows * kHeadDim + (size_t)cta * (2 * kAtRows) + r;
  const float* part = p.part + ((size_t)cta * kAtRows + r) * kHeadDim + 4 * lane;
  float f = lane < p.splits ? stat[lane * (2 * kAtRows)] : -INFINITY;
  const float l = lane < p.splits ? stat[lane * (2 * kAtRows) + kAtRows] : 0.0f;
  float mm = f;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, d));
  f = f == -INFINITY && l == 0.0f ? 0.0f : ex2(f - mm);   // a share that saw no token of the row
  float ll = l * f;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, d);
  const float inv = ll != 0.0f ? 1.0f / ll : 0.0f;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int x = 0; x < p.splits; ++x) {
    const float fx = __shfl_sync(0xffffffffu, f, x);
    if (fx == 0.0f) continue;                             // may not have been written
    const float4 v = *reinterpret_cast<const float4*>(part + (size_t)x * (kAtRows * kHeadDim));
    acc.x = fmaf(v.x, fx, acc.x); acc.y = fmaf(v.y, fx, acc.y); acc.z = fmaf(v.z, fx, acc.z); acc.w = fmaf(v.w, fx, acc.w);
  }
  const __half2 h0 = __floats2half2_rn(acc.x * inv, acc.y * inv), h1 = __floats2half2_rn(acc.z * inv, acc.w * inv);
  uint2 out;
  out.x = *reinterpret_cast<const uint32_t*>(&h0);
  out.y = *reinterpret_cast<const uint32_t*>(&h1);
  *reinterpret_cast<uint2*>(at_out_row(p, w, head_kv, r) + 4 * lane) = out;
}

// How the work is cut: tiles, CTAs per tile and, where these are to meet in global memory, the bytes for it.
struct AtPlan {
  int64_t units;
  int whole, splits;                                      // with memory to meet in
  size_t bytes;                                           // 0: of no use
  double cost;                                            // of the better way, in parts of a unit and SM
};
static int at_plan(KvAttendParams& p, int64_t max_rows, AtPlan* plan) {
  const int64_t per_seq = (max_rows + kAtRows - 1) / kAtRows;
  const int64_t bound = p.total_q * p.group / kAtRows + p.batch;
  const bool uniform = p.batch * per_seq <= 2 * bound;
  const int64_t tiles = uniform ? p.batch * per_seq : bound;
  plan->units = tiles * p.kv_heads;
  plan->bytes = 0;
  if (plan->units > 0x7fffffff / 16) return fail(QR_EUNSUPPORTED, "qr_kv_attend_i4: too many tiles");
  p.tiles_per_seq = uniform ? (int)per_seq : 0;
  p.max_tiles = (int)tiles;
  // beside its blocks a CTA has about four blocks' time, and three more where there are others to join
  const int64_t blocks = visible_blocks(p, max_rows, kAtTok, false);
  const double length = (double)visible_blocks(p, max_rows, kAtTok, true), alone = 4.0 / length, joined = 7.0 / length;
  double cost = 0.0;
  int resident = 0;
  if (const int rc = kv_pick_splits(kKvKernelTc, (const void*)kv_attend_tc_kernel, kAtThreads, kAtSmem, plan->units, blocks, alone, joined,
                                    &p.splits, &resident, &cost)) return rc;
  p.sorted = uniform && p.window <= 0 && p.batch > 1 && p.batch <= 64 && plan->units > resident;
  plan->cost = cost;
  // Clusters lie within a GPC and leave SMs over (16 units get 6 CTAs each from them, 9 without), and they split all units
  // alike.  Here full rounds of units have an SM each, what is left over shares all SMs.  At the same split a second kernel
  // that joins is no slower than the cluster (32 units in four: 40.1 and 42.0 us) unless there are but two (64 units: 59 and 60).
  const int64_t sms = num_sms(), rounds = plan->units / sms, rest = plan->units % sms;
  int64_t s = rest ? sms / rest : 1;
  if (s > blocks) s = blocks;
  if (s > 32) s = 32;
  const double here = rounds * (1.0 + alone) + 1.0 / s + joined;
  if (s > 1 && (here < 0.999 * cost || (s > 2 && here <= cost))) {
    plan->whole = (int)(rounds * sms);
    plan->splits = (int)s;
    plan->bytes = (size_t)(rest * s) * kAtRows * (kHeadDim + 2) * sizeof(float);
    plan->cost = here;
  }
  return QR_OK;
}

int kv_attend_tc_time(const KvAttendParams& p, int64_t max_rows, double* us, size_t* bytes) {
  KvAttendParams c = p;
  AtPlan plan = {};
  if (const int rc = at_plan(c, max_rows, &plan)) return rc;
  *us = 3.0 + plan.cost * (double)visible_blocks(c, max_rows, kAtTok, true) * (max_rows <= 128 ? 2.3 : 2.6);
  *bytes = plan.bytes;
  return QR_OK;
}

int launch_kv_attend_tc(KvAttendParams& p, int64_t max_rows, void* workspace, size_t workspace_bytes, cudaStream_t st) {
  AtPlan plan = {};
  if (const int rc = at_plan(p, max_rows, &plan)) return rc;
  if (plan.bytes > 0 && workspace && workspace_bytes >= plan.bytes) {
    p.part = reinterpret_cast<float*>(workspace);
    p.whole = plan.whole;
    p.splits = plan.splits;
  }
  const int64_t split = plan.units - p.whole;             // units that p.splits CTAs share
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(p.whole + split * p.splits));
  cfg.blockDim = dim3(kAtThreads);
  cfg.dynamicSmemBytes = kAtSmem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = p.splits > 1 && !p.part ? 1 : 0;
  QR_CUDA(cudaLaunchKernelEx(&cfg, kv_attend_tc_kernel, (const KvAttendParams)p));
  if (p.part) {
    kv_attend_join_kernel<<<(unsigned)(split * (kAtRows / 8)), 256, 0, st>>>(p);
    QR_LAUNCH_CHECK("kv_attend_join_kernel");
  }
  return QR_OK;
}

}  // namespace qr
