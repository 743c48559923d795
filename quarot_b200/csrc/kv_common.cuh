// What the kernels of the paged 4-bit KV cache share: the 128-long Walsh-Hadamard transform of a warp, exact division
// by the page size, the parameters of the chunk / window attention kernels and the walk over the visible tokens.
#pragma once
#include "common.cuh"

namespace qr {

constexpr int kHeadDim = 128;

#ifdef __CUDACC__
// Walsh-Hadamard transform of 128 values held four per lane (element index = 4 lane + e), unscaled.
__device__ __forceinline__ void fwht128_warp(float (&x)[4], int lane) {
  {
    const float a = x[0] + x[1], b = x[0] - x[1], c = x[2] + x[3], d = x[2] - x[3];
    x[0] = a + c; x[1] = b + d; x[2] = a - c; x[3] = b - d;
  }
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const float sg = (lane & s) ? -1.0f : 1.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float o = __shfl_xor_sync(0xffffffffu, x[e], s);
      x[e] = fmaf(x[e], sg, o);
    }
  }
}

__device__ __forceinline__ void half4_to_f32(uint2 u, float (&x)[4]) {
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
  x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
}
__device__ __forceinline__ void load4_f16(const __half* p, float (&x)[4]) { half4_to_f32(*reinterpret_cast<const uint2*>(p), x); }
#endif

#ifdef __CUDACC__
// Nibbles J and J + 4 of a word (or of two 16-bit halves) as the fp16 pair (16 + c_J, 16 + c_{J+4}): a code in the upper
// mantissa bits of 16.0.
template <int J>
__device__ __forceinline__ uint32_t code_pair(uint32_t w) {
  const uint32_t x = J == 0 ? w << 6 : J == 1 ? w << 2 : J == 2 ? w >> 2 : w >> 6;
  uint32_t r;
  // (x & mask) | bias as one instruction; with both constants as immediates it would be two
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(0x03C003C0u), "r"(0x4C004C00u));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Clusters that share a token axis.
__device__ __forceinline__ uint32_t kv_cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void kv_cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the place of `local` in the shared memory of CTA `rank` of the cluster, and loads from there
__device__ __forceinline__ uint32_t kv_peer_addr(const void* local, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(local)), "r"(rank));
  return r;
}
__device__ __forceinline__ float kv_peer_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 kv_peer_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
#endif

// Division of 0 <= n < 2^31 by a fixed d >= 1 as one wide multiplication: with s = ceil(log2 d) and
// m = ceil(2^(31+s) / d) <= 2^32 - 1 (2^31 for d = 1), m d - 2^(31+s) < d <= 2^s, hence floor(n m / 2^(31+s)) = floor(n / d),
// the upper half of 2 n times m shifted by s.
struct FastDiv {
  uint32_t d, m;
  int s;
};
static inline FastDiv make_fastdiv(uint32_t d) {
  FastDiv f;
  f.d = d;
  f.s = ilog2(d);
  f.m = (uint32_t)((((uint64_t)1 << (31 + f.s)) + d - 1) / d);
  return f;
}
#ifdef __CUDACC__
__device__ __forceinline__ int fast_div(int n, const FastDiv& f) {
  return (int)(__umulhi((uint32_t)n << 1, f.m) >> f.s);
}
#endif

// Attention of new tokens over the cache (qr_kv_attend_i4).
struct KvAttendParams {
  __half* o;                    // new token x head x 128, strides below
  const __half* q;
  const uint8_t* data;
  const __half2* param;
  const int32_t* indptr;
  const int32_t* indices;
  const int32_t* last_page_offset;
  const int32_t* qo_indptr;     // [batch + 1], or null: one new token per sequence
  int64_t q_ts, q_hs, o_ts, o_hs;   // strides in elements between tokens and between heads
  int64_t total_q;
  int batch, layers, layer, kv_heads, group, page_size;
  int64_t num_pages, num_indices;   // pages of the pool, entries of indices
  FastDiv page_div, group_div;
  int window, sinks;            // window 0: none
  int hadamard_q;
  int splits;                   // CTAs (one cluster, or joined through `part`) that share the tokens of a tile of rows
  float* part;                  // tcgen05 kernel: shares of the CTAs in global memory, or NULL
  int whole;                    // with `part`: units before this one have a CTA each
  int tiles_per_seq;            // > 0: tile index = sequence * tiles_per_seq + tile; 0: found by a search in qo_indptr
  int max_tiles;                // tiles that the grid holds per KV head
  int sorted;                   // tiles_per_seq > 0, at most 64 sequences: the longest sequences come first
  int* status;
};

// Blocks of T tokens that a tile of rows sees: at most (`all` entries of the page list), or as many as each of the
// sequences has where they share the list evenly.
static inline int64_t visible_blocks(const KvAttendParams& p, int64_t max_rows, int T, bool evenly) {
  const int64_t pages = evenly ? (p.num_indices + p.batch - 1) / p.batch : p.num_indices;
  const int64_t all = (pages * p.page_size + T - 1) / T;
  if (p.window <= 0) return all > 0 ? all : 1;
  const int64_t seen = ((int64_t)p.window + max_rows / p.group + T - 1) / T + 1 + ((int64_t)p.sinks + T - 1) / T;
  return seen < all ? seen : all > 0 ? all : 1;
}

#ifdef __CUDACC__
// Splitting the token axis of a unit of work (a tile of rows of one KV head) over a cluster of s = 1 .. 16 CTAs.  The cost of
// s, in parts of a unit, is (rounds of CTAs that an SM goes through) * (1 / s + what a CTA costs beside its share of the
// tokens); `most` is the number of parts that there are.
// `resident`: CTAs that the device holds at once.  `alone` and `joined`: that cost without and with other CTAs to
// join.  How many clusters fit is asked once per kernel, device and size (clusters lie within a GPC, whose SMs they do not
// divide evenly: 15 clusters of 8 fit, 16 do not); the kernel's attributes are set then too.
enum { kKvKernelRows8, kKvKernelRows16, kKvKernelTc, kKvKernels };
int kv_pick_splits(int which, const void* kernel, int threads, size_t smem, int64_t units, int64_t most, double alone,
                   double joined, int* splits, int* resident, double* cost = nullptr);

// fp32 shares [rows][128] (addr(r): the lane's four columns of row r) of the CTAs of a cluster joined into one row, U rows
// at a time.  Lane x looks at the statistics of CTA x; the first two shares are asked for before that.
template <int U, class Addr, class Store>
__device__ __forceinline__ void kv_merge_rows(int splits, int first, int step, int rows, int lane, const float* s_m, const float* s_l,
                                              Addr addr, Store store) {
#pragma unroll 1
  for (int r0 = first; r0 < rows; r0 += U * step) {
    float f[U], inv[U];
    float4 acc[U], v[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * step < rows ? r0 + u * step : r0;
      f[u] = lane < splits ? kv_peer_f32(kv_peer_addr(s_m + r, lane)) : -INFINITY;
      inv[u] = lane < splits ? kv_peer_f32(kv_peer_addr(s_l + r, lane)) : 0.0f;
#pragma unroll
      for (int x = 0; x < 2; ++x) v[u][x] = kv_peer_f32x4(kv_peer_addr(addr(r), x));
      acc[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float mm = f[u];
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, d));
      // a share that saw no token of the row has l = 0 (its statistics say nothing); NaN stays NaN
      f[u] = f[u] == -INFINITY && inv[u] == 0.0f ? 0.0f : ex2(f[u] - mm);
      float ll = inv[u] * f[u];
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, d);
      inv[u] = ll != 0.0f ? 1.0f / ll : 0.0f;             // a row that sees nothing gives zeros
    }
#pragma unroll 1
    for (int x0 = 0; x0 < splits; x0 += 2) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float fx = __shfl_sync(0xffffffffu, f[u], x0 + x);        // 0 beyond the last share
          if (fx != 0.0f) {
            acc[u].x = fmaf(v[u][x].x, fx, acc[u].x); acc[u].y = fmaf(v[u][x].y, fx, acc[u].y);
            acc[u].z = fmaf(v[u][x].z, fx, acc[u].z); acc[u].w = fmaf(v[u][x].w, fx, acc[u].w);
          }
        }
      }
      if (x0 + 2 < splits) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            v[u][x] = kv_peer_f32x4(kv_peer_addr(addr(r0 + u * step < rows ? r0 + u * step : r0), x0 + 2 + x < splits ? x0 + 2 + x : 0));
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      inv[u] = __shfl_sync(0xffffffffu, inv[u], 0);
      if (r0 + u * step < rows) store(r0 + u * step, acc[u], inv[u]);
    }
  }
}

// The tile of query rows that a CTA works on.  Row r of a sequence is (new token r / group, head r % group of the KV head).
struct KvTile {
  int b, row0, rows;            // sequence, first row, rows (0: nothing to do)
  int first;                    // the sequence's first entry of the page list
  int64_t tok0;                 // first new token of the sequence in q and o
  int seq_len, pos0;            // cached tokens with the new ones; position of new token 0
};

constexpr int kKvMostTokens = 0x7fff0000;
// Sequence and tile of rows behind tile index `tile`, by all lanes of a warp.
__device__ __forceinline__ KvTile kv_find_tile(const KvAttendParams& p, int tile, int tile_rows, int lane) {
  KvTile w;
  w.rows = 0; w.b = 0; w.first = 0; w.row0 = 0; w.tok0 = 0; w.seq_len = 0; w.pos0 = 0;
  int j = -1, b = 0;
  int qo0, qo1, first, behind, last;
  if (p.sorted) {
    // a lane looks at two sequences and counts the longer ones; the sequence with as many as the tile asks for is the tile's
    const int rank = tile / p.tiles_per_seq;
    j = tile - rank * p.tiles_per_seq;
    int v[2][5], len[2], ahead[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int bb = min(lane + 32 * k, p.batch - 1);
      v[k][0] = p.qo_indptr ? __ldg(p.qo_indptr + bb) : bb;
      v[k][1] = p.qo_indptr ? __ldg(p.qo_indptr + bb + 1) : bb + 1;
      v[k][2] = __ldg(p.indptr + bb); v[k][3] = __ldg(p.indptr + bb + 1); v[k][4] = __ldg(p.last_page_offset + bb);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const long long seq = ((long long)v[k][3] - v[k][2] - 1) * p.page_size + v[k][4];
      // clamped: any order is right
      len[k] = lane + 32 * k >= p.batch ? -1 : (int)(seq < 0 ? 0 : seq < 0x7fffffffll ? seq : 0x7fffffffll);
    }
#pragma unroll 8
    for (int x = 0; x < 32; ++x) {
      const int l0 = __shfl_sync(0xffffffffu, len[0], x), l1 = __shfl_sync(0xffffffffu, len[1], x);
      ahead[0] += (l0 > len[0] || (l0 == len[0] && x < lane)) + (l1 > len[0]);
      ahead[1] += (l0 >= len[1]) + (l1 > len[1] || (l1 == len[1] && x < lane));
    }
    const uint32_t hit0 = __ballot_sync(0xffffffffu, ahead[0] == rank), hit1 = __ballot_sync(0xffffffffu, ahead[1] == rank);
    const int src = __ffs(hit0 ? hit0 : hit1) - 1;
    b = hit0 ? src : src + 32;
    qo0 = __shfl_sync(0xffffffffu, hit0 ? v[0][0] : v[1][0], src);
    qo1 = __shfl_sync(0xffffffffu, hit0 ? v[0][1] : v[1][1], src);
    first = __shfl_sync(0xffffffffu, hit0 ? v[0][2] : v[1][2], src);
    behind = __shfl_sync(0xffffffffu, hit0 ? v[0][3] : v[1][3], src);
    last = __shfl_sync(0xffffffffu, hit0 ? v[0][4] : v[1][4], src);
  } else {
    if (p.tiles_per_seq > 0) {
      b = tile / p.tiles_per_seq;
      j = tile - b * p.tiles_per_seq;
    } else {
      int base = 0;
      for (int b0 = 0; b0 < p.batch; b0 += 32) {
        const int bb = b0 + lane;
        int n = 0;
        if (bb < p.batch) {
          const long long rows = (long long)(p.qo_indptr[bb + 1] - p.qo_indptr[bb]) * p.group;
          n = rows > 0 ? (int)((rows + tile_rows - 1) / tile_rows) : 0;
        }
        int end = n;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, end, s);
          if (lane >= s) end += up;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, base + end > tile);
        if (hit) {
          const int src = __ffs(hit) - 1;
          b = b0 + src;
          j = tile - base - (__shfl_sync(0xffffffffu, end, src) - __shfl_sync(0xffffffffu, n, src));
          break;
        }
        base += __shfl_sync(0xffffffffu, end, 31);
      }
      if (j < 0) return w;
    }
    if (b >= p.batch) return w;
    // one round trip for all of them
    qo0 = p.qo_indptr ? __ldg(p.qo_indptr + b) : b;
    qo1 = p.qo_indptr ? __ldg(p.qo_indptr + b + 1) : b + 1;
    first = __ldg(p.indptr + b); behind = __ldg(p.indptr + b + 1); last = __ldg(p.last_page_offset + b);
  }
  const long long tok0 = qo0, len = (long long)qo1 - qo0;
  if (tok0 < 0 || tok0 + len > p.total_q) return w;       // rows beyond q are not touched
  const long long rows = len * p.group, row0 = (long long)j * tile_rows;
  if (row0 >= rows) return w;
  // not beyond the pages that are listed, whatever kv_indptr and the last page's offset say
  const long long pages = first < 0 ? 0 : (behind < p.num_indices ? behind : p.num_indices) - first;
  const long long listed = pages * p.page_size;
  long long seq = listed - p.page_size + last;
  if (seq > listed) seq = listed;
  if (seq > kKvMostTokens) return w;                      // tokens are counted in 32 bits
  w.first = first;
  w.b = b;
  w.row0 = (int)row0;
  w.rows = (int)(rows - row0 < tile_rows ? rows - row0 : tile_rows);
  w.tok0 = tok0;
  w.seq_len = seq > 0 ? (int)seq : 0;
  w.pos0 = (int)(seq > 0 ? seq - len : -len);
  return w;
}

// Blocks of T tokens that the rows at positions p_min .. p_max see: first .. first + body - 1, and with a window that does
// not reach the sinks the blocks 0 .. count - body - 1 that hold these.  Where rows see only parts of the first block (a
// window begins in it) it comes after the others, and the sinks last: the reference of a row's weights is set by the tokens
// that it sees first, and moves the less the more of them there are.
struct KvBlocks {
  int first, body, turn, count;
};
template <int T>
__device__ __forceinline__ KvBlocks kv_blocks(int p_min, int p_max, int window, int sinks) {
  KvBlocks k;
  const int end = p_max >= 0 ? p_max / T + 1 : 0;
  // p_min < 0: a row before the sequence (more new tokens than cached ones), which sees nothing
  const int lo = window > 0 ? max(0, max(p_min, 0) - window + 1) : 0;
  k.first = min(lo / T, end);
  int head = (max(min(sinks, p_max + 1), 0) + T - 1) / T;
  if (window <= 0 || head >= k.first) { head = 0; k.first = 0; }
  k.body = end - k.first;
  k.turn = k.first > 0 && k.body > 1 ? 1 : 0;
  k.count = head + k.body;
  return k;
}
__device__ __forceinline__ int kv_block_index(const KvBlocks& k, int i) {
  return i < k.body - k.turn ? k.first + k.turn + i : i < k.body ? k.first : i - k.body;
}
#endif

int launch_kv_attend_rows(KvAttendParams& p, int64_t max_rows, cudaStream_t st);
int launch_kv_attend_tc(KvAttendParams& p, int64_t max_rows, void* workspace, size_t workspace_bytes, cudaStream_t st);
// Estimates of the two kernels' times; bytes: workspace that the tcgen05 kernel can use.
int kv_attend_rows_time(const KvAttendParams& p, int64_t max_rows, double* us);
int kv_attend_tc_time(const KvAttendParams& p, int64_t max_rows, double* us, size_t* bytes);

}  // namespace qr
