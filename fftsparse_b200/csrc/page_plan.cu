// page_plan.cu -- one serving step's page bookkeeping, built on the GPU from request lengths.
//
// For request r with c_r cached and n_r new tokens and pages of ps tokens:
//   have_r = ceil(c_r / ps), last_r = ceil((c_r + n_r) / ps), need_r = last_r - have_r
//   start_r = sum of need over the requests before r        (its first entry of the free list)
//   table[r][have_r + i] = free[start_r + i], i < need_r
//   token t of request r: pos = c_r + (t - cu_q[r]), slot = table[r][pos / ps] * ps + pos % ps, -1 if that is no int32
// A request is served if its pages fit the table row, its tokens fit num_tokens and its pages fit the
// free list (start_r + need_r <= n_free, or it needs none).  An unserved request gets kv_len 0 and slots
// -1; one that fails the first two conditions asks for no pages, so the later requests' do not move.
//
// Every CTA scans all requests itself (8 bytes each, from L2) instead of waiting for another CTA's
// prefix, then fills its own share of the tokens and of the new table entries: one launch, no
// workspace, no order between CTAs.  The tokens of a CTA find their request by a binary search in
// the chunk's prefix in shared memory.  Nothing a CTA reads is written by another one: tokens read
// table entries below have_r, the new entries lie at or above it, and a token in a new page takes its
// page from the free list.  Latency bound: 4.2 us for 64 requests of one token, 7.4 us for 1024 of 1 to
// 256 (256 threads 3.5 and 9.6, 1024 threads 6.6 and 7.5; 1024 tokens per CTA 4.3 and 8.0).

#include "ffts_common.cuh"

namespace ffts {
namespace plan {

constexpr int kThreads = 512;       // also the requests scanned at a time
constexpr int kTokensPerCta = 512;

struct Params {
  const int32_t *cached, *fresh;  // [R]
  int R;
  int32_t *table;                 // [R, width], row stride table_ld
  int64_t table_ld;
  int width;
  const int32_t *free_pages;      // [n_free]
  int n_free;
  int ps_shift;
  int T;
  int32_t *cu_q, *kv_lens, *positions, *slots, *info;
};

// Inclusive sum over the block; *total receives the block's sum.  Sums are 64-bit: lengths are the
// caller's data and their total is not known to fit 32 bits.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t *warp_sums, int64_t *total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();  // the previous scan's sums have been read
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    const int64_t s = warp_sums[w];
    if (w < warp) before += s;
    all += s;
  }
  *total = all;
  return v + before;
}

// First i in [0, n) with a[i] > x (a non-decreasing); n if none.
__device__ __forceinline__ int upper(const int64_t *a, int n, int64_t x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] > x) hi = mid; else lo = mid + 1;
  }
  return lo;
}

__global__ void __launch_bounds__(kThreads) page_plan_kernel(const __grid_constant__ Params p) {
  __shared__ int64_t s_end[kThreads];     // tokens up to and with the request
  __shared__ int64_t s_pages[kThreads];   // pages asked for up to and with the request
  __shared__ int64_t warp_sums[kThreads / 32];
  __shared__ int s_cached[kThreads];
  __shared__ int s_need[kThreads];
  __shared__ uint8_t s_served[kThreads];
  __shared__ int s_unserved, s_taken;
  const int tid = threadIdx.x;
  const int ps = 1 << p.ps_shift;
  const int64_t t_lo = int64_t(blockIdx.x) * kTokensPerCta;
  const int64_t t_hi = min(int64_t(p.T), t_lo + kTokensPerCta);
  if (tid == 0) {
    s_unserved = 0;
    s_taken = 0;
    if (blockIdx.x == 0) p.cu_q[0] = 0;
  }
  int64_t tok_base = 0, page_base = 0;
  for (int r0 = 0; r0 < p.R; r0 += kThreads) {
    const int nr = min(kThreads, p.R - r0);
    const int r = r0 + tid;
    int c = 0, n = 0;
    if (tid < nr) {
      c = max(0, p.cached[r]);
      n = max(0, p.fresh[r]);
    }
    int64_t toks, pages;
    const int64_t end = tok_base + block_scan(n, warp_sums, &toks);
    const int have = int((int64_t(c) + ps - 1) >> p.ps_shift);
    const int64_t last = (int64_t(c) + n + ps - 1) >> p.ps_shift;
    const bool fits = last <= p.width && end <= p.T;
    const int need = fits ? int(last - have) : 0;
    const int64_t upto = page_base + block_scan(need, warp_sums, &pages);
    const bool served = fits && (need == 0 || upto <= p.n_free);
    s_end[tid] = end;
    s_pages[tid] = upto;
    s_cached[tid] = c;
    s_need[tid] = need;
    s_served[tid] = served;
    if (blockIdx.x == 0 && tid < nr) {
      p.cu_q[r + 1] = int(min(end, int64_t(p.T)));
      p.kv_lens[r] = served ? int(int64_t(c) + n) : 0;
      if (!served) atomicAdd(&s_unserved, 1);
      if (served && need > 0) atomicMax(&s_taken, int(upto));
    }
    __syncthreads();
    // this CTA's tokens of the chunk's requests
    const int64_t a = max(t_lo, tok_base), b = min(t_hi, tok_base + toks);
    for (int64_t t = a + tid; t < b; t += kThreads) {
      const int i = upper(s_end, nr, t);  // t < s_end[nr - 1], so i < nr
      const int64_t first = i > 0 ? s_end[i - 1] : tok_base;
      const int pos = int(s_cached[i] + (t - first));
      int slot = -1;
      if (s_served[i]) {
        const int have_i = int((int64_t(s_cached[i]) + ps - 1) >> p.ps_shift);
        const int col = pos >> p.ps_shift;
        const int page = col < have_i
                             ? p.table[int64_t(r0 + i) * p.table_ld + FFTS_INDEX(col, p.width)]
                             : p.free_pages[FFTS_INDEX(int(s_pages[i] - s_need[i]) + col - have_i, p.n_free)];
        // a number of no pool (negative, or its slots pass 31 bits) gives no slot, not another page's
        if (uint32_t(page) < (0x80000000u >> p.ps_shift)) slot = int(uint32_t(page) << p.ps_shift) + (pos & (ps - 1));
      }
      p.positions[t] = pos;
      p.slots[t] = slot;
    }
    // the chunk's new table entries, spread over all CTAs
    const int64_t f_hi = min(page_base + pages, int64_t(p.n_free));
    for (int64_t f = page_base + int64_t(blockIdx.x) * kThreads + tid; f < f_hi; f += int64_t(gridDim.x) * kThreads) {
      const int i = upper(s_pages, nr, f);  // f < s_pages[nr - 1]
      if (!s_served[i]) continue;
      const int have_i = int((int64_t(s_cached[i]) + ps - 1) >> p.ps_shift);
      const int col = have_i + int(f - (s_pages[i] - s_need[i]));
      if (FFTS_IN_RANGE(col, p.width)) p.table[int64_t(r0 + i) * p.table_ld + col] = p.free_pages[f];
    }
    tok_base += toks;
    page_base += pages;
  }
  // rows behind the last request's tokens: no position, no slot
  for (int64_t t = max(t_lo, tok_base) + tid; t < t_hi; t += kThreads) {
    p.positions[t] = 0;
    p.slots[t] = -1;
  }
  if (blockIdx.x == 0) {
    __syncthreads();
    if (tid == 0) {
      p.info[0] = s_taken;
      p.info[1] = s_unserved;
    }
  }
}

}  // namespace plan

int page_plan(const ffts_page_plan_args &a, cudaStream_t stream) {
  using namespace plan;
  FFTS_REQUIRE(a.R >= 0 && a.num_tokens >= 0 && a.width >= 0 && a.n_free >= 0, "page_plan: negative size");
  FFTS_REQUIRE(a.R < (int64_t(1) << 30) && a.num_tokens <= (int64_t(1) << 30) && a.n_free < (int64_t(1) << 31),
               "page_plan: more than 2^30 requests or tokens, or 2^31 free pages");
  FFTS_REQUIRE(a.page_size >= 1 && a.page_size <= 4096 && (a.page_size & (a.page_size - 1)) == 0,
               "page_plan: page_size must be a power of two up to 4096 (got %lld)", (long long)a.page_size);
  FFTS_REQUIRE(a.width <= (int64_t(1) << 30) / a.page_size, "page_plan: a table row spans more than 2^30 tokens");
  FFTS_REQUIRE(a.table_ld >= a.width, "page_plan: table rows overlap (row stride %lld, width %lld)",
               (long long)a.table_ld, (long long)a.width);
  FFTS_REQUIRE(a.cu_q && a.info && (a.R == 0 || (a.cached_lens && a.new_lens && a.kv_lens && (a.width == 0 || a.table))) &&
                   (a.num_tokens == 0 || (a.positions && a.slots)) && (a.n_free == 0 || a.free_pages),
               "page_plan: NULL argument");
  const int64_t T = a.num_tokens;
  Params p{};
  p.cached = a.cached_lens;
  p.fresh = a.new_lens;
  p.R = int(a.R);
  p.table = a.table;
  p.table_ld = a.table_ld;
  p.width = int(a.width);
  p.free_pages = a.free_pages;
  p.n_free = int(a.n_free);
  p.ps_shift = ilog2_ceil(a.page_size);
  p.T = int(T);
  p.cu_q = a.cu_q;
  p.kv_lens = a.kv_lens;
  p.positions = a.positions;
  p.slots = a.slots;
  p.info = a.info;
  const unsigned grid = unsigned(T > kTokensPerCta ? ceil_div(T, kTokensPerCta) : 1);
  page_plan_kernel<<<grid, kThreads, 0, stream>>>(p);
  FFTS_CUDA(cudaGetLastError());
  return FFTS_OK;
}

}  // namespace ffts
