// paged_common.cuh -- what the two paged attention kernels share: the schedule (q tiles, the line of work and its
// shares), the walk along a share, and the element types.  The kernels differ in the size of their tiles:
// paged_attn.cu has 128 rows x 64 keys and two CTAs per SM, paged_chunk.cu 256 rows x 128 keys and one.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>

#include "ffts_common.cuh"
#include "tc_sm100.cuh"

namespace ffts {
namespace paged {

using namespace ::ffts::tc;

constexpr int kMinShare = 4;      // length of a share, at least
constexpr int kOverhead = 2;      // length of a (q tile, head) besides its key tiles
constexpr int kSchedThreads = 1024;
constexpr int kOwnTiles = 1024;   // up to so many q tiles every CTA builds the schedule itself
constexpr int kMaxCtas = 512;

constexpr int kErrProducer = 10, kErrMma = 11, kErrSoftmax = 12, kErrSmemAlign = 13;

// One q tile: tokens [tok0, tok0 + ntok) of request r, the first at position pos0.
struct __align__(16) Tile {
  int tok0, pos0, ntok, r;
};

// A (q tile, head) that several shares cut: rows nrows from token tok0 and head head0 on; its partials lie in
// first_slot and in the first slots of the shares behind it up to s1.  nrows 0: none.
struct Cut {
  int tok0, nrows, head0, s1, first_slot;
};

struct Params {
  int T, R, H, Hkv, G, tpt;   // tpt: tokens per q tile
  const int32_t *table;       // [R, width]
  int64_t table_ld;
  int width, n_pages, ps_shift;
  const int32_t *cu_q, *kv_lens;
  int window, sinks;          // window 0: none
  uint16_t *out;
  int64_t os_t, os_h;
  float scale_log2;
  int own_schedule;           // every CTA has its own copy of tiles and cum
  Tile *tiles;                // [max_tiles]
  long long *cum;             // [max_tiles + 1]: length (of one head) before q tile x
  int *header;                // [0]: q tiles
  Cut *cuts;                  // [ctas]: the (q tile, head) that share c begins and others go on with
  float *part;                // [2 * ctas][D / 4][rows] float4
  float2 *part_ml;            // [2 * ctas][rows]: m (log2 units) and l
  int max_tiles, ctas;
  int rows;                   // of a q tile: 128 or 256
  int *status;
  long long wait_cycles, drain_cycles;
};

// The key tiles of BN keys that a q tile visits: [0, st), then [wt0, ...); n of them in all (at least one, which
// may be all masked).  Keys >= hi, and keys < lo that are not sinks, are seen by no row.
struct Keys {
  int hi, lo, st, wt0, n;
};

template <int BN>
__device__ __forceinline__ Keys keys_of(int pos0, int ntok, int window, int sinks) {
  Keys g;
  g.hi = max(0, pos0 + ntok);
  g.lo = window > 0 ? max(0, pos0 - window + 1) : 0;
  const int nt = (g.hi + BN - 1) / BN;
  g.wt0 = g.lo / BN;
  g.st = min((min(sinks, g.hi) + BN - 1) / BN, g.wt0);
  g.n = max(1, g.st + nt - g.wt0);
  return g;
}

// The j-th of them.
__device__ __forceinline__ int key_tile(const Keys &g, int j) { return j < g.st ? j : j - g.st + g.wt0; }

__device__ __forceinline__ long long share_of(const Params &p, long long length) {
  const long long per = (length + p.ctas - 1) / p.ctas;
  return per < kMinShare ? kMinShare : per;
}

// ---------------------------------------------------------------- schedule
// The q tiles of all requests and the line's running sum, by one CTA of NT threads; scratch in its shared memory.
template <int NT>
struct SchedScratch {
  long long warp_sums[32];
  long long tiles[NT];  // q tiles up to and with the request
  int q0[NT], len[NT], kv[NT];
};

template <int NT>
__device__ __forceinline__ long long sched_scan(long long v, long long *warp_sums, long long *total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();  // the previous scan's sums have been read
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  long long s = lane < NT / 32 ? warp_sums[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += u;
  }
  const long long before = __shfl_sync(0xffffffffu, s, max(warp - 1, 0));
  *total = __shfl_sync(0xffffffffu, s, 31);
  return v + (warp > 0 ? before : 0);
}

// tiles [max_tiles], cum [max_tiles + 1]; returns the number of q tiles, *length the line of one head.
template <int BN, int NT>
__device__ int build_schedule(const Params &p, Tile *tiles, long long *cum, SchedScratch<NT> &sc, long long *length) {
  const int tid = threadIdx.x;
  const long long cap = (long long)p.width << p.ps_shift;  // keys a table row can hold
  long long tile_base = 0, line = 0;
  if (tid == 0) cum[0] = 0;
  for (int r0 = 0; r0 < p.R; r0 += NT) {
    const int nr = min(NT, p.R - r0);
    int q0 = 0, len = 0, kv = 0;
    if (tid < nr) {
      // lengths are device data: kept inside q and the table whatever they hold
      q0 = min(max(p.cu_q[r0 + tid], 0), p.T);
      len = min(max(p.cu_q[r0 + tid + 1], q0), p.T) - q0;
      kv = int(min((long long)max(p.kv_lens[r0 + tid], 0), cap));
    }
    long long total;
    const long long upto = sched_scan<NT>((len + p.tpt - 1) / p.tpt, sc.warp_sums, &total);
    sc.tiles[tid] = upto;
    sc.q0[tid] = q0;
    sc.len[tid] = len;
    sc.kv[tid] = kv;
    __syncthreads();
    const long long fit = min(total, (long long)p.max_tiles - tile_base);
    for (long long x0 = 0; x0 < fit; x0 += NT) {
      const long long x = x0 + tid;
      int n = 0;
      if (x < fit) {
        int lo = 0, hi = nr;  // the first request whose tiles reach past x
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (sc.tiles[mid] > x) hi = mid; else lo = mid + 1;
        }
        const int i = int(x - (lo > 0 ? sc.tiles[lo - 1] : 0)) * p.tpt;
        Tile t;
        t.tok0 = sc.q0[lo] + i;
        t.pos0 = sc.kv[lo] - sc.len[lo] + i;
        t.ntok = min(p.tpt, sc.len[lo] - i);
        t.r = r0 + lo;
        n = keys_of<BN>(t.pos0, t.ntok, p.window, p.sinks).n + kOverhead;
        if (FFTS_IN_RANGE(tile_base + x, p.max_tiles)) tiles[tile_base + x] = t;
      }
      long long sum;
      const long long upto_x = sched_scan<NT>(n, sc.warp_sums, &sum);
      if (x < fit && FFTS_IN_RANGE(tile_base + x, p.max_tiles)) cum[tile_base + x + 1] = line + upto_x;
      line += sum;
    }
    tile_base += max(fit, 0ll);
    __syncthreads();  // the chunk's arrays have been read
  }
  *length = line;
  return int(tile_base);
}

template <int BN>
__global__ void __launch_bounds__(kSchedThreads) schedule_kernel(const __grid_constant__ Params p) {
  __shared__ SchedScratch<kSchedThreads> sc;
  long long length;
  const int n = build_schedule<BN, kSchedThreads>(p, p.tiles, p.cum, sc, &length);
  if (threadIdx.x == 0) p.header[0] = n;
}

// Walks the share [u, u1) of the line segment by segment; the same in every lane.
template <int BN>
struct Walk {
  const Params &p;
  const Tile *tiles;
  const long long *cum;
  long long u, u1;
  long long base, next;  // the line before q tile x and behind it, all heads
  int x;
  Tile t;
  Keys g;
  int h, j0, j1;         // the segment: head and key tiles [j0, j1) of the g.n
  long long begin;       // where its (q tile, head) begins
  __device__ __forceinline__ Walk(const Params &prm, const Tile *t_, const long long *c_) : p(prm), tiles(t_), cum(c_) {}

  // Finds the q tile at u0 (whole warp; u0 < length).
  __device__ __forceinline__ void seek(long long u0, long long end, int ntiles) {
    u = u0;
    u1 = end;
    int lo = 0, n = ntiles;  // x is in [lo, lo + n): cum[lo] * Hkv <= u0
    const int lane = threadIdx.x & 31;
    while (n > 1) {
      const int step = (n + 31) / 32;
      const int i = lane * step;
      const bool below = i < n && cum[lo + i] * p.Hkv <= u0;
      const int last = 31 - __clz(__ballot_sync(0xffffffffu, below));
      const int off = last * step;
      lo += off;
      n = min(step, n - off);
    }
    x = lo;
    load();
  }
  __device__ __forceinline__ void load() {
    t = tiles[FFTS_INDEX(x, p.max_tiles)];
    base = cum[x] * p.Hkv;
    next = cum[x + 1] * p.Hkv;
    g = keys_of<BN>(t.pos0, t.ntok, p.window, p.sinks);
  }
  // The next segment with key tiles; false behind the share's end.
  __device__ __forceinline__ bool segment() {
    while (u < u1) {
      if (u >= next) {
        ++x;
        load();
      }
      const int len = g.n + kOverhead;
      const long long rem = u - base;
      h = int(rem / len);
      const int at = int(rem - (long long)h * len);
      const int to = int(min((long long)len, at + (u1 - u)));
      begin = u - at;
      u += to - at;
      j0 = max(0, at - kOverhead);
      j1 = max(0, to - kOverhead);
      if (j1 > j0) return true;
    }
    return false;
  }
};

__device__ __forceinline__ uint64_t below(int k) { return k <= 0 ? 0ull : (k >= 64 ? ~0ull : (1ull << k) - 1ull); }

template <typename E>
struct Num;
template <>
struct Num<__nv_bfloat16> {
  static constexpr uint32_t fmt = 1;
  static constexpr CUtensorMapDataType map = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  // P <= 2^64 against the reference max: bf16 and the fp32 O have the exponents for it
  static constexpr float rescale = 64.0f, pmax = 18446744073709551616.0f;
  static constexpr int degree = 3;  // of paged_chunk.cu's exponential, 2^-13.7 off where P is rounded by 2^-8
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&r);
  }
};
template <>
struct Num<__half> {
  static constexpr uint32_t fmt = 0;
  static constexpr CUtensorMapDataType map = CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  // fp16 ends at 65504: P <= 2^8 after a rescale, 2^14 (a tile's row sum) before the next one; the row's
  // top has P >= 1, so what is lost below 2^-24 is that far under it
  static constexpr float rescale = 8.0f, pmax = 16384.0f;
  static constexpr int degree = 4;  // 2^-18.5, P 2^-11
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 r = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&r);
  }
};

constexpr uint32_t idesc(uint32_t fmt, bool b_mn_major, int n) {
  return (1u << 4) | (fmt << 7) | (fmt << 10) | (b_mn_major ? (1u << 16) : 0u) | (uint32_t(n >> 3) << 17) |
         (uint32_t(128 >> 4) << 24);
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

// The kernel of paged_chunk.cu: p with tiles of 256 rows, K and V maps with boxes of up to 128 keys.
int launch_chunk(const Params &p, bool half, int D, const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv,
                 cudaStream_t stream);

}  // namespace paged
}  // namespace ffts
