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

constexpr int kMinShare = 4;      // length of a share, at least (2 and 3: the same time for one request's decode step)
constexpr int kSchedThreads = 1024;
constexpr int kOwnTiles = 1024;   // up to so many q tiles every CTA builds the schedule itself
constexpr int kMaxCtas = 512;

constexpr int kErrProducer = 10, kErrMma = 11, kErrSoftmax = 12, kErrSmemAlign = 13;

// One q tile: tokens [tok0, tok0 + ntok) of request r, the first at position pos0.
struct __align__(16) Tile {
  int tok0, pos0, ntok, r;
};

// A (q tile, head) that several shares cut: rows nrows from token tok0 (at position pos0) and head head0 on; its
// partials lie in first_slot and in the first slots of the shares behind it up to s1.  nrows 0: none.
struct Cut {
  int tok0, pos0, nrows, head0, s1, first_slot;
};

struct Params {
  int T, R, Hkv, G, tpt;      // tpt: tokens per q tile
  const int32_t *table;       // [R, width]
  int64_t table_ld;
  int width, ps_shift;
  const int32_t *cu_q, *kv_lens;
  int window, sinks;          // window 0: none
  const uint16_t *q;
  int64_t qs_t, qs_h;
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
  uint32_t *notes;            // [ctas][rows][2][4]: channels of a row's o that are +inf, and -inf (NaN: both)
  int max_tiles, ctas;
  int rows;                   // of a q tile: 128 or 256
  int overhead;               // length of a (q tile, head) besides its key tiles
  int *status;
  long long wait_cycles, drain_cycles;
};

// The key tiles of BN keys that a q tile visits: [0, st), then [wt0, ...); n of them in all (at least one, which
// may be all masked).  Keys >= hi, and keys < lo that are not sinks, are seen by no row.
struct Keys {
  int hi, lo, st, wt0, n;
};

template <int BN>
__host__ __device__ __forceinline__ Keys keys_of(int pos0, int ntok, int window, int sinks) {
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
__host__ __device__ __forceinline__ int key_tile(const Keys &g, int j) { return j < g.st ? j : j - g.st + g.wt0; }

// Whether some of the keys [c0, c0 + BN) are seen by no row of the q tile.
template <int BN>
__host__ __device__ __forceinline__ bool has_unseen(const Keys &g, int sinks, int c0) {
  return c0 + BN > g.hi || (c0 < g.lo && c0 + BN > sinks);
}
// Whether the rows of a q tile may differ in what they see of them.
template <int BN>
__host__ __device__ __forceinline__ bool rows_differ(int pos0, int ntok, int window, int sinks, int c0) {
  return ntok > 1 && (c0 + BN > pos0 + 1 || (window > 0 && c0 < pos0 + ntok - window && c0 + BN > sinks));
}

__host__ __device__ __forceinline__ long long share_of(const Params &p, long long length) {
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
        n = keys_of<BN>(t.pos0, t.ntok, p.window, p.sinks).n + p.overhead;
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

// Walks a share segment by segment; the same in every lane.  Positions are kept relative to the share, in 64 bits, and
// to the q tile, in 32: the host refuses a q tile whose heads' line passes 2^31.
template <int BN>
struct Walk {
  const Params &p;
  const Tile *tiles;
  const long long *cum;
  long long left, done;  // of the share: what is ahead, what lies behind
  int rem, all;          // in q tile x: position and length, all heads
  int x;
  Tile t;
  Keys g;
  // The segment: head and key tiles [j0, j1) of the g.n.  The line runs through a (q tile, head)'s key tiles from
  // the last ones to the first: a share that begins inside one takes keys from the start on, a share that
  // ends inside one ends with the last.  So the shares, which run side by side, are at the same keys at their
  // beginnings and at their ends, and find each other's tiles in L2.
  int h, j0, j1;
  bool opens;            // the (q tile, head) begins in this share
  // A whole one begins where the share would be after so many key tiles, for the same reason, and goes round.
  int turn;
  unsigned seen;
  long long begin;       // where its (q tile, head) begins, relative to the share (may be negative)
  __host__ __device__ __forceinline__ Walk(const Params &prm, const Tile *t_, const long long *c_)
      : p(prm), tiles(t_), cum(c_) {}

  // Finds the q tile at u0 (whole warp; u0 < length).
  __device__ __forceinline__ void seek(long long u0, long long u1, int ntiles) {
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
    start(u0, u1, lo);
  }
  // u0 lies in q tile at.
  __host__ __device__ __forceinline__ void start(long long u0, long long u1, int at) {
    left = u1 - u0;
    done = 0;
    seen = 0;
    x = at;
    rem = int(u0 - cum[x] * p.Hkv);
    load();
  }
  __host__ __device__ __forceinline__ void load() {
    t = tiles[FFTS_INDEX(x, p.max_tiles)];
    g = keys_of<BN>(t.pos0, t.ntok, p.window, p.sinks);
    all = (g.n + p.overhead) * p.Hkv;
  }
  // The key tile at step j of [j0, j1).
  __host__ __device__ __forceinline__ int key(int j) const { return key_tile(g, j + turn < j1 ? j + turn : j + turn - g.n); }
  // The next segment with key tiles; false behind the share's end.
  __host__ __device__ __forceinline__ bool segment() {
    while (left > 0) {
      if (rem >= all) {
        rem = 0;
        ++x;
        load();
      }
      const int len = g.n + p.overhead;
      h = rem / len;
      const int at = rem - h * len;
      const int to = int(min((long long)len, at + left));
      begin = done - at;
      rem += to - at;
      done += to - at;
      left -= to - at;
      const int o0 = max(0, at - p.overhead), o1 = max(0, to - p.overhead);
      if (o1 == o0) continue;
      opens = o0 == 0;
      j0 = g.n - o1;
      j1 = g.n - o0;
      turn = j1 - j0 == g.n ? int(seen % unsigned(g.n)) : 0;
      seen += unsigned(j1 - j0);
      return true;
    }
    return false;
  }
  // The share that ends the segment's (q tile, head), from where this one begins and the length of all.
  __host__ __device__ __forceinline__ int last_share(long long u0, long long per) const {
    return int((u0 + begin + p.overhead + g.n - 1) / per);
  }
};

__device__ __forceinline__ uint64_t below(int k) { return k <= 0 ? 0ull : (k >= 64 ? ~0ull : (1ull << k) - 1ull); }

// sum_keys: the tensor core cuts every product p v off at 2^-25 of the sum it is added to (so it measured: behind a
// key of weight 1, products of 2^-25 count and those of 0.53 of that do not), while the divisor is summed exactly.
// Behind one heavy key many light ones would be lost, 131072 of them 2^-8 of the result.  So O is parked after so
// many keys and starts again from zero, which bounds the loss by one rounding of the result; what is parked is
// added up in fp32.  2048 tokens over 131072, 32 / 8 heads: fp16 4.37 ms without, 4.46 with, 4.52 with half as
// many keys to a sum; bf16 4.22 all three (since then, with registers split otherwise, 4.23 and 4.02).
template <typename E>
struct Num;
template <>
struct Num<__nv_bfloat16> {
  static constexpr uint32_t fmt = 1;
  static constexpr CUtensorMapDataType map = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  // P <= 2^64 against the reference max: bf16 and the fp32 O have the exponents for it
  static constexpr float rescale = 64.0f, pmax = 18446744073709551616.0f, bias = 0.0f, chunk_rescale = 64.0f;
  static constexpr int sum_keys = 131072;
  static constexpr uint32_t exponent = 0x7f80;
  // 0 * each half of w added to acc: NaN once one of them is not finite
  static __device__ __forceinline__ void probe(uint32_t w, uint32_t &acc) {
    asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(w), "r"(0u));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&r);
  }
};
template <>
struct Num<__half> {
  static constexpr uint32_t fmt = 0;
  static constexpr CUtensorMapDataType map = CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  // fp16 ends at 65504, and its smallest step is 2^-24: P is off by up to 2^-25, and the errors of many small ones add
  // up (the divisor sums them unrounded).  So the reference maximum stands at 2^bias: an error is 2^-32 of the
  // row's top at most.  What outgrows the reference by 2^rescale resets it.  The smaller tiles exponentiate before they
  // look, and look when 64 keys sum to more than pmax, which takes one that has (2^9.99 < 65504 / 64); the larger
  // tiles look first, and rescale seldom (at 2^2.99: 2048 tokens over 32768 1112 -> 1150 us).
  static constexpr float rescale = 2.99f, pmax = 65504.0f, bias = 7.0f, chunk_rescale = 8.0f;
  static constexpr int sum_keys = 16384;
  static constexpr uint32_t exponent = 0x7c00;
  static __device__ __forceinline__ void probe(uint32_t w, uint32_t &acc) {
    asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(w), "r"(0u));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 r = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&r);
  }
};

constexpr uint32_t idesc(uint32_t fmt, bool b_mn_major, int n, int m = 128) {
  return (1u << 4) | (fmt << 7) | (fmt << 10) | (b_mn_major ? (1u << 16) : 0u) | (uint32_t(n >> 3) << 17) |
         (uint32_t(m >> 4) << 24);
}

// True in one thread of the (converged) warp.  The compiler knows that no other thread is in the branch behind it, so
// the operands of the MMAs there go straight to uniform registers; behind lane == 0 each one takes a
// loop over the threads that might be active (30 to 40 instructions per MMA).
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}

// tcgen05.mma with descriptors as their low words (the address and the leading offset, which an advance along the tile
// leaves alone) and a common high word: one 32-bit addition per operand instead of 64-bit ones.
__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi,
                                        uint32_t idesc_, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %2};\n\tmov.b64 b, {%3, %4};\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc_), "r"(uint32_t(accumulate))
      : "memory");
}
// A from TMEM.
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi, uint32_t idesc_,
                                        bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc_), "r"(uint32_t(accumulate))
      : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float *v) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const float *v) {
  uint32_t r[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(v[i]);
  tmem_st16u(taddr, r);
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

// Launches a kernel that may start while the one before it in the stream drains (it begins with griddepcontrol.wait).
template <typename... Ts>
static int launch_early(void (*kernel)(Ts...), dim3 grid, int threads, int smem, cudaStream_t stream,
                        const std::remove_cv_t<Ts> &...args) {
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(unsigned(threads));
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.stream = stream;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  FFTS_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
  return FFTS_OK;
}

// The weight of a partial with maximum m (log2 units) in a sum scaled to top; NaN stays NaN in what it multiplies.
__device__ __forceinline__ float weight(float m, float top) { return m == -INFINITY ? 0.0f : exp2f(m - top); }

// 32 channels of a row's O, from channel 32 c on, to a slot of the partials (rows side by side).
template <int ROWS>
__device__ __forceinline__ void park(const float *o, float4 *pd, int c) {
#pragma unroll
  for (int q = 0; q < 8; ++q) pd[(c * 8 + q) * ROWS] = make_float4(o[q * 4], o[q * 4 + 1], o[q * 4 + 2], o[q * 4 + 3]);
}
// o += f * what the slot holds of them.
template <int ROWS>
__device__ __forceinline__ void unpark(float *o, const float4 *pd, int c, float f) {
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const float4 old = pd[(c * 8 + q) * ROWS];
    o[q * 4] = fmaf(f, old.x, o[q * 4]);
    o[q * 4 + 1] = fmaf(f, old.y, o[q * 4 + 1]);
    o[q * 4 + 2] = fmaf(f, old.z, o[q * 4 + 2]);
    o[q * 4 + 3] = fmaf(f, old.w, o[q * 4 + 3]);
  }
}
// Adds a row's O in TMEM to what the slot holds (again), or puts it there; m: what it is scaled to, at least the
// slot's.  Not inlined: inside the softmax loop its registers cost 5% (2048 tokens over 32768 1085 -> 1145 us).
template <int D, int ROWS>
__device__ __noinline__ void park_o(const Params &p, int slot, int row, bool live, bool again, float m,
                                    uint32_t o_addr) {
  float4 *pd = reinterpret_cast<float4 *>(p.part) + int64_t(slot) * (ROWS * D / 4) + row;
  float2 *pml = p.part_ml + int64_t(slot) * ROWS + row;
  const float f = again && live ? weight(pml->x, m) : 0.0f;
#pragma unroll 1
  for (int c = 0; c < D / 32; ++c) {
    float o[32];
    __syncwarp();
    tmem_ld32(o_addr + c * 32, o);
    tmem_wait_ld();
    if (again && live) unpark<ROWS>(o, pd, c, f);
    if (live) park<ROWS>(o, pd, c);
  }
  if (live) pml->x = m;
}

// ---------------------------------------------------------------- values that must not count
// The tensor core multiplies all keys of a V tile, and a P of 0 does not make up for NaN or infinity.  Keys that no row
// of the q tile sees are zeroed in shared memory (pages hold anything behind a request's last key).  In tiles that
// rows differ in (the last ones of a q tile, and those at the ends of its window) elements that are not finite are noted for
// the rows that see them, and zeroed; the rows' results get them back at the segment's end.
//
// A row's notes to its result, in the output or (float) in the partials, whose pieces of four channels lie ROWS pieces
// apart.
template <typename E, int D, int ROWS, typename T>
__device__ __noinline__ void put_back(const Params &p, int row, T *o) {
  if (!FFTS_IN_RANGE(row, p.rows)) return;
  const uint32_t *at = p.notes + (int64_t(blockIdx.x) * p.rows + row) * 8;
#pragma unroll 1
  for (int c = 0; c < D; ++c) {
    const bool up = (at[c >> 5] >> (c & 31)) & 1u, down = (at[4 + (c >> 5)] >> (c & 31)) & 1u;
    if (!up && !down) continue;
    const float x = (up ? INFINITY : 0.0f) - (down ? INFINITY : 0.0f);  // both: NaN
    if constexpr (std::is_same<T, float>::value)
      o[(c >> 2) * ROWS * 4 + (c & 3)] += x;
    else
      o[c] = E(float(o[c]) + x);
  }
}

// The kernel of paged_chunk.cu: p with tiles of 256 rows, K and V maps with boxes of up to 128 keys.
int launch_chunk(const Params &p, bool half, int D, const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv,
                 cudaStream_t stream);

}  // namespace paged
}  // namespace ffts
