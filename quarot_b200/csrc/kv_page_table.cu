// Page table and slot map of the paged KV cache from request lengths (qr_kv_page_table).
//
// With P(n) = ceil(n / page_size), sequence b holds P(old_b) pages and wants P(old_b + new_b).  The pages it lacks come
// off a list of free pages in the order of the sequences: sequence b takes free[N_b .. N_b + need_b), N_b the prefix sum
// of need.  Everything the cache kernels read follows from three prefix sums over the batch: indptr (of the pages), the
// rows of the new tokens (of new) and N.  A sequence that does not fit -- its row of the block table, the free list or
// the slot map ends before it -- keeps its old length and its new tokens get slot -1, so that no consumer writes
// anywhere for them; one that is longer than its row already does not fit either, and the row's pages are listed for it.  Since N only grows, the sequences that the free list serves are a prefix of those that need pages.
//
// The call writes a few megabytes at most, so it is one launch without a second pass: every CTA makes the three prefix
// sums of the whole batch itself (512 threads x 4 sequences per round, the sums of up to 8192 sequences in shared
// memory) and then takes its share of the flat list of outputs; an entry finds its sequence by a binary search in
// shared memory, 128 to 512 entries of kv_indices per search.  A new page is read from the free list by everyone, never from
// the block table, whose new entries are written in the same launch: no CTA waits for another.
// Measured: 16 requests 5.7 us, 2048 requests with 9 MB of table entries 11.9 us (3.4 us at the copy rate): latency of chained
// reads and scans (programmatic dependent launch takes off 0.5 us); a call from Python takes 18 us, a dozen torch operations
// for the same 600 us.
#include "kv_common.cuh"

namespace qr {

constexpr int kPtThreads = 512;
constexpr int kPtPer = 4;              // sequences per thread and round
constexpr int kPtMaxBatch = 8192;

struct PageTableParams {
  const int32_t* seq_lens;
  const int32_t* new_lens;             // or null: one token each
  int32_t* block_table;                // [batch, max_blocks], or null: page j of sequence b is j * batch + b
  const int32_t* free_pages;
  int64_t num_free, new_tokens;        // num_free < 0: the block table holds the pages of the new tokens already
  int batch, max_blocks, page_size;
  FastDiv page_div;
  int32_t* kv_indptr;
  int32_t* kv_indices;
  int32_t* last_page_offset;
  int32_t* append_indptr;
  int64_t* slot_map;
  int32_t* positions;
  int32_t* seq_lens_out;
  int32_t* status;
};

// Exclusive prefix sum over the block of one value per thread; `total` is the sum of all.
__device__ __forceinline__ long long pt_block_scan(long long v, long long* s_warp, long long* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  long long inc = v;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, inc, s);
    if (lane >= s) inc += up;
  }
  if (lane == 31) s_warp[warp] = inc;
  __syncthreads();
  long long before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPtThreads / 32; ++w) {
    const long long x = s_warp[w];
    if (w < warp) before += x;
    all += x;
  }
  __syncthreads();
  *total = all;
  return before + inc - v;
}

// The last b of 0 .. n - 1 with s[b] <= i (s non-decreasing, s[0] = 0 <= i < s[n]).
__device__ __forceinline__ int pt_find(const int* s, int n, int i) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s[mid] <= i) lo = mid; else hi = mid;
  }
  return lo;
}

// R: rounds of 128 entries of kv_indices that a warp takes at a time (4 where there is enough for every warp, 1 otherwise)
template <int R>
__global__ void __launch_bounds__(kPtThreads)
kv_page_table_kernel(const PageTableParams p) {
  pdl_launch_dependents();
  extern __shared__ int s_pt[];
  __shared__ long long s_warp[kPtThreads / 32];
  int* s_pages = s_pt;                          // [batch + 1] prefix sum of the pages
  int* s_rows = s_pages + p.batch + 1;          // [batch + 1] prefix sum of the new tokens
  int* s_held = s_rows + p.batch + 1;           // [batch] pages held before the call
  int* s_free = s_held + p.batch;               // [batch] first entry of the free list, -1: the sequence was refused
  const int tid = threadIdx.x;
  const int W = p.max_blocks;
  const bool take = p.block_table && p.num_free >= 0;
  pdl_wait();
  long long base_rows = 0, base_need = 0, base_pages = 0, taken = 0, refused = 0;
  for (int b0 = 0; b0 < p.batch; b0 += kPtThreads * kPtPer) {
    const int first = b0 + tid * kPtPer;
    int old[kPtPer], add[kPtPer], held[kPtPer], need[kPtPer];
    bool fits[kPtPer], over[kPtPer];
    long long sum = 0, total;
#pragma unroll
    for (int k = 0; k < kPtPer; ++k) {
      const int b = first + k;
      const long long cap = (long long)W * p.page_size;
      const int most = cap < 0x7fffffffll ? (int)cap : 0x7fffffff;
      const int len = b < p.batch ? max(p.seq_lens[b], 0) : 0;
      over[k] = len > most;                     // longer than its row: refused, and the row's pages are listed
      old[k] = min(len, most);
      add[k] = b < p.batch ? (p.new_lens ? max(p.new_lens[b], 0) : 1) : 0;
      sum += add[k];
    }
    long long rows = base_rows + pt_block_scan(sum, s_warp, &total);
    base_rows += total;
    sum = 0;
#pragma unroll
    for (int k = 0; k < kPtPer; ++k) {
      const long long after = (long long)old[k] + add[k];
      held[k] = old[k] > 0 ? fast_div(old[k] - 1, p.page_div) + 1 : 0;
      // lengths stay below 2^31 - 1: positions and lengths are 32-bit
      const int want = after > 0 && after < 0x7fffffffll ? fast_div((int)after - 1, p.page_div) + 1 : 0;
      const int b = first + k;
      if (b < p.batch) s_rows[b] = (int)min(rows, 0x7fffffffll);
      rows += add[k];
      fits[k] = !over[k] && (add[k] == 0 || (after < 0x7fffffffll && want <= W && rows <= p.new_tokens));
      need[k] = fits[k] && take ? want - held[k] : 0;
      // where the pages are there already the sequence just has more of them
      if (fits[k] && !take) held[k] = want;
      sum += need[k];
    }
    long long start = base_need + pt_block_scan(sum, s_warp, &total);
    base_need += total;
    sum = 0;
#pragma unroll
    for (int k = 0; k < kPtPer; ++k) {
      const int b = first + k;
      if (need[k] > 0 && start + need[k] > p.num_free) fits[k] = false;
      if (b < p.batch) {
        s_held[b] = held[k];
        s_free[b] = fits[k] ? (int)(start < 0x7fffffffll ? start : 0x7fffffffll) : -1;
      }
      start += need[k];
      if (!fits[k]) need[k] = 0;
      sum += held[k] + need[k];
    }
    long long pages = base_pages + pt_block_scan(sum, s_warp, &total);
    base_pages += total;
    long long mine_taken = 0, mine_refused = 0;
#pragma unroll
    for (int k = 0; k < kPtPer; ++k) {
      const int b = first + k;
      if (b < p.batch) {
        s_pages[b] = (int)pages;
        const int n = held[k] + need[k];
        pages += n;
        mine_taken += need[k];
        mine_refused += fits[k] ? 0 : 1;
        if (blockIdx.x == 0) {
          const int after = fits[k] ? old[k] + add[k] : old[k];
          p.seq_lens_out[b] = over[k] ? p.seq_lens[b] : after;
          p.last_page_offset[b] = after - (n > 1 ? (n - 1) * p.page_size : 0);
        }
      }
    }
    if (blockIdx.x == 0) {
      pt_block_scan((mine_taken << 32) + mine_refused, s_warp, &total);
      taken += total >> 32;
      refused += total & 0xffffffffll;
    }
  }
  if (tid == 0) {
    s_pages[p.batch] = (int)base_pages;
    s_rows[p.batch] = (int)min(base_rows, 0x7fffffffll);
    if (blockIdx.x == 0) {
      p.status[0] = (int)taken;
      p.status[1] = (int)refused;
    }
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int b = tid; b <= p.batch; b += kPtThreads) {
      p.kv_indptr[b] = s_pages[b];
      p.append_indptr[b] = s_rows[b];
    }
  }
  // page j of sequence b
  auto page_of = [&](int b, int j, bool* fresh) -> int {
    *fresh = false;
    if (!p.block_table) return j * p.batch + b;
    if (j < s_held[b]) return p.block_table[(size_t)b * W + j];
    *fresh = true;
    return p.free_pages[(size_t)s_free[b] + (j - s_held[b])];
  };
  // kv_indices: a warp takes 128 R entries, looks their first sequence up once and walks on from there
  const int stride = gridDim.x * kPtThreads, at = blockIdx.x * kPtThreads + tid;
  const int lane = tid & 31;
  const long long cap = (long long)p.batch * W;
  const int pages = (int)base_pages;
  const bool vec = (reinterpret_cast<uintptr_t>(p.kv_indices) & 15) == 0;
  for (long long seg = at >> 5; seg * (128 * R) < cap; seg += stride >> 5) {
    const long long i_seg = seg * (128 * R);
    const int b_seg = i_seg < pages ? pt_find(s_pages, p.batch, (int)i_seg) : 0;
    int v[R][4];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long i0 = i_seg + 128 * r + 4 * lane;
#pragma unroll
      for (int k = 0; k < 4; ++k) v[r][k] = -1;
      if (i0 < pages) {
        int b = b_seg;
        while (s_pages[b + 1] <= (int)i0) ++b;
        int j = (int)i0 - s_pages[b];
        if (!p.block_table || j + 4 > s_held[b] || i0 + 4 > pages) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int i = (int)i0 + k;
            if (i < pages) {
              while (s_pages[b + 1] <= i) ++b;
              bool fresh;
              j = i - s_pages[b];
              v[r][k] = page_of(b, j, &fresh);
              if (fresh) p.block_table[(size_t)b * W + j] = v[r][k];
            }
          }
        } else {
          const int32_t* src = p.block_table + (size_t)b * W + j;
#pragma unroll
          for (int k = 0; k < 4; ++k) v[r][k] = src[k];
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long i0 = i_seg + 128 * r + 4 * lane;
      if (vec && i0 + 4 <= cap) {
        *reinterpret_cast<int4*>(p.kv_indices + i0) = make_int4(v[r][0], v[r][1], v[r][2], v[r][3]);
      } else {
        for (int k = 0; k < 4 && i0 + k < cap; ++k) p.kv_indices[i0 + k] = v[r][k];
      }
    }
  }
  const int rows = s_rows[p.batch];
  for (long long i = at; i < p.new_tokens; i += stride) {
    long long slot = -1;
    int pos = -1;
    if (i < rows) {
      const int b = pt_find(s_rows, p.batch, (int)i);
      if (s_free[b] >= 0) {
        const long long cap_b = (long long)W * p.page_size;
        pos = min(max(p.seq_lens[b], 0), (int)min(cap_b, 0x7fffffffll)) + (int)i - s_rows[b];
        const int j = fast_div(pos, p.page_div);
        bool fresh;
        slot = (long long)page_of(b, j, &fresh) * p.page_size + (pos - j * p.page_size);
        if (slot < 0) slot = -1;
      }
    }
    p.slot_map[i] = slot;
    p.positions[i] = pos;
  }
}

}  // namespace qr

extern "C" int qr_kv_page_table(const int32_t* seq_lens, const int32_t* new_lens, int batch, int64_t new_tokens, int page_size,
                                int max_blocks, int32_t* block_table, const int32_t* free_pages, int64_t num_free,
                                int32_t* kv_indptr, int32_t* kv_indices, int32_t* last_page_offset, int32_t* append_indptr,
                                int64_t* slot_map, int32_t* positions, int32_t* seq_lens_out, int32_t* status, void* stream) {
  using namespace qr;
  if (batch < 0 || new_tokens < 0) return fail(QR_EINVAL, "qr_kv_page_table: negative size");
  if (page_size < 1 || max_blocks < 1) return fail(QR_EINVAL, "qr_kv_page_table: page size and blocks per sequence must be positive");
  if (batch == 0) return QR_OK;
  if (batch > kPtMaxBatch) return fail(QR_EUNSUPPORTED, "qr_kv_page_table: %d sequences (at most %d)", batch, kPtMaxBatch);
  if ((int64_t)batch * max_blocks > 0x7ffffff0ll) return fail(QR_EUNSUPPORTED, "qr_kv_page_table: batch x blocks per sequence exceeds 32 bits");
  if (new_tokens > 0x7ffffff0ll) return fail(QR_EUNSUPPORTED, "qr_kv_page_table: too many new tokens");
  if (!seq_lens || !kv_indptr || !kv_indices || !last_page_offset || !append_indptr || !seq_lens_out || !status ||
      (new_tokens > 0 && (!slot_map || !positions)) || (num_free > 0 && !free_pages))
    return fail(QR_EINVAL, "qr_kv_page_table: null pointer");
  PageTableParams p;
  p.seq_lens = seq_lens; p.new_lens = new_lens; p.block_table = block_table; p.free_pages = free_pages;
  p.num_free = num_free; p.new_tokens = new_tokens; p.batch = batch; p.max_blocks = max_blocks; p.page_size = page_size;
  p.page_div = make_fastdiv((uint32_t)page_size);
  p.kv_indptr = kv_indptr; p.kv_indices = kv_indices; p.last_page_offset = last_page_offset; p.append_indptr = append_indptr;
  p.slot_map = slot_map; p.positions = positions; p.seq_lens_out = seq_lens_out; p.status = status;
  const size_t smem = (size_t)(4 * batch + 2) * sizeof(int);
  // one CTA per 2048 page entries or 512 tokens, at most one per SM: each of them makes the prefix sums for itself
  const int64_t cap = (int64_t)batch * max_blocks;
  const int64_t want = (cap + 4 * kPtThreads - 1) / (4 * kPtThreads) + (new_tokens + kPtThreads - 1) / kPtThreads;
  const int grid = (int)(want < num_sms() ? (want > 0 ? want : 1) : num_sms());
  auto kern = cap > 512ll * (kPtThreads / 32) * num_sms() ? kv_page_table_kernel<4> : kv_page_table_kernel<1>;
  // More than 48 KB, the kernel's own shared memory counted, has to be asked for.  Always the most that a call can need: the
  // limit belongs to the kernel, and another thread's smaller batch must not lower it between this line and the launch.
  constexpr int kMost = (4 * kPtMaxBatch + 2) * (int)sizeof(int);
  if (smem > 40 * 1024) QR_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost));
  QR_CUDA(launch_kernel(kern, dim3(grid), dim3(kPtThreads), smem, (cudaStream_t)stream, g_tuning.pdl != 0, p));
  return QR_OK;
}
