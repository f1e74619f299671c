// paged_attn.cu -- causal attention of new tokens over a paged KV cache on sm_100a (tcgen05 + TMEM + TMA).
//
// Request r has q_len = cu_q[r+1] - cu_q[r] new tokens (rows of q) at the end of its kv_len cached ones;
// token i sits at pos = kv_len - q_len + i and sees key c iff c <= pos and (no window, or c > pos - W, or
// c < S): o = softmax(scale q k^T) v over the keys it sees, zeros if there are none.  q_len 1 is decoding,
// longer ones are the chunks of a prompt; a batch may mix them.
//
// Work.  The G = H / Hkv query heads of a KV head share one 128-row tile with as many tokens as fit
// (128 / G, row = token * G + head), so a key tile is loaded once for all of them.  A q tile visits the
// 64-key tiles that any of its rows can see (the sinks' and the window's), in an order that brings shares that run side
// by side to the same keys (Walk in paged_common.cuh).  All (q tile, KV head)s form one line, each as long as its key tiles plus kOverhead for loading Q and storing the result, and
// the line is cut into equal shares: CTA c of the persistent grid takes [c * per, (c + 1) * per).  So one
// decode request and a batch of ragged chunks alike load every SM equally, and nothing about the lengths is
// needed on the host.  A share that begins or ends between two key tiles of a (q tile, head) leaves fp32
// partial sums, which are joined in the order of the shares.
//   schedule         q tiles of every request and the running sum of their lengths: up to kOwnTiles q
//                    tiles by every CTA of attn_kernel for itself, beyond by schedule_kernel (one CTA)
//   attn_kernel      two CTAs per SM, each walking its share
//   join_kernel      the (q tile, head)s that several shares cut (a kernel of its own: inside attn_kernel
//                    its registers made the softmax loop spill, 1.15 -> 1.89 ms at 2048 tokens over 32768)
//
// attn_kernel's roles (192 threads):
//   warp 4      producer: page numbers one tile ahead, Q per segment, K tiles into a three-stage ring, V
//               into a two-stage ring; every lane issues its own TMA boxes (a page is one box per 64
//               channels).  A page no row sees gets page number -1: TMA fills zeros, nothing is read.
//   warp 5      MMA issuer (one thread): S = Q K^T into a double-buffered TMEM accumulator, O += P V with
//               P from TMEM.
//   warps 0-3   softmax: thread r owns row r; S(n) is read, masked and exponentiated against a running
//               reference maximum (O and l rescaled only when a score outgrows it by 2^Num<E>::rescale) while
//               the tensor core computes S(n+1).  V rows behind a request's last key, or of no key a
//               row sees, are zeroed in shared memory first: pages hold anything there, and 0 * NaN
//               would reach the sum.  V tiles that rows differ in are looked through for NaN and infinities.
// Every mbarrier wait is bounded (a status code instead of a hang).
//
// Decoding is bound by HBM, or by the power cap before it: 64 requests of 512 to 16384 keys, 32 / 8 heads, pages
// of 16: 155 us at 1.9 GHz (6.3 TB/s, 0.96 of the measured copy), 161 to 167 us a step in a long loop; 2 x 131072
// keys 164 us (1.0) and 173.  Chunks are bound by the tensor core and the softmax around it: a key tile takes
// about 1600 clocks in each of an SM's two CTAs, 640 of them its products (a 64-key S reads 48 KB of shared
// memory, 384 clocks for 256 of products).

#include <cudaTypedefs.h>

#include <algorithm>

#include "paged_common.cuh"

namespace ffts {
namespace paged {

constexpr int kBM = 128;      // rows of a q tile
constexpr int kBN = 64;       // keys of a key tile
constexpr int kThreads = 192;
constexpr int kKStages = 3, kVStages = 2;
constexpr int kTmemCols = 256;  // S0, S1 (64 columns each), O (D): two CTAs fill an SM's 512
constexpr uint32_t kTmemO = 128;
// 2, 3 and 4: 16 ragged chunks 67, 59, 57 us, 64 decoding requests 155.4, 155.8, 157.4 us
constexpr int kOverhead = 3;
constexpr int kFewRows = 32;    // of a q tile: loaded one by one
// With so few rows the products are of 64 rows, whose first 16 lie in the same TMEM lanes 0-15 as those of 128
// rows: half the power of products that are mostly of zeros (64 requests' step 169 -> 164 us under the power cap,
// 2 x 131072 keys 180 -> 172).
constexpr int kSmallRows = 16;
constexpr int64_t kLongRows = 1024, kLongKeys = 4096;  // of a request on average, of a tile
constexpr double kWaitSeconds = 2.0, kDrainSeconds = 4.0;

template <int D>
struct Layout {
  static constexpr int halves = D / 64;             // 64-channel swizzle boxes per row
  static constexpr int q_half = kBM * 128;          // bytes of one half of a tile
  static constexpr int kv_half = kBN * 128;
  static constexpr int q_bytes = halves * q_half, kv_bytes = halves * kv_half;
  static constexpr int q = 0;
  static constexpr int k = q + q_bytes;
  static constexpr int v = k + kKStages * kv_bytes;
  static constexpr int bars = v + kVStages * kv_bytes;
  static constexpr int nbars = 2 + 2 * kKStages + kVStages + 2 + 2 + 2 + 1;
  static constexpr int tmem_slot = bars + nbars * 8;
  static constexpr int abort = tmem_slot + 8;
  static constexpr int odd = (abort + 8 + 15) / 16 * 16;  // OddTile [2]
  static constexpr int noted = odd + 32;                   // the segment of the rows' notes, counted from 1
  static constexpr int bytes = noted + 8;
  static_assert(2 * (bytes + 1024) <= 228 * 1024, "two CTAs must fit in an SM's shared memory");
};

// barriers; one per buffer, since the softmax can run a tile ahead of the MMA issuer
constexpr int BQF = 0;                  // Q loaded
constexpr int BQE = 1;                  // the segment's S products have read Q
constexpr int BKF = 2;                  // K stage loaded    [kKStages]
constexpr int BKE = BKF + kKStages;     // K stage free      [kKStages]
constexpr int BVF = BKE + kKStages;     // V stage loaded    [kVStages]
constexpr int BSF = BVF + kVStages;     // S(n) in buffer n % 2 [2]
constexpr int BPV = BSF + 2;            // PV(n) complete, frees V stage n % 2 [2]
constexpr int BPF = BPV + 2;            // P(n) written (128 arrivals) [2]
constexpr int BDRAIN = BPF + 2;

// A V tile with elements that are not finite, where rows differ in what they see of it: the softmax threads that find
// some say so before they hand P over, and the MMA issuer sees to them before it uses the tile.  Looking costs ragged
// chunks 77 -> 81 us (as many for a meeting of the softmax warps on top: 85; looked through by the producer 95; by a
// warp of its own, with fewer registers for each, 82, and decoding 165 -> 172).
struct __align__(16) OddTile {
  int seg, pos0, ntok, c0;  // segment, counted from 1; 0: none
};

// Whether the thread's part of a V tile (key, one half) has such elements.
template <typename E>
__device__ __noinline__ bool has_odd(const uint8_t *row) {
  uint32_t acc[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) {  // in another order in each lane: no bank conflicts
    const uint4 w = *reinterpret_cast<const uint4 *>(row + (((i ^ threadIdx.x) & 7) << 4));
    Num<E>::probe(w.x, acc[0]);
    Num<E>::probe(w.y, acc[1]);
    Num<E>::probe(w.z, acc[2]);
    Num<E>::probe(w.w, acc[3]);
  }
  return ((acc[0] | acc[1] | acc[2] | acc[3]) & 0x7fff7fffu) != 0;
}

// Notes the elements for the rows that see them and zeroes them (one thread; the rows of earlier segments have put
// theirs back when P of this one is there).
template <typename E, int D>
__device__ __noinline__ void note_odd(const Params &p, uint8_t *v, const OddTile &o, volatile int *notes_seg) {
  constexpr uint32_t top = Num<E>::exponent;
  uint32_t *notes = p.notes + int64_t(blockIdx.x) * p.rows * 8;
  const bool again = *notes_seg == o.seg;
  constexpr int kKeys = 16;  // at a time: their words lie in local memory, which is set aside for every thread of the GPU
  for (int step = 0; step < 4 * (kBN / kKeys); ++step) {
    const int ch = step / (kBN / kKeys), k0 = step % (kBN / kKeys) * kKeys;  // 32 channels of these keys
    uint32_t up[kKeys], down[kKeys];
    for (int k = 0; k < kKeys; ++k) {
      up[k] = down[k] = 0;
      const int key = k0 + k;
      for (int i = 0; ch < D / 32 && i < 16; ++i) {
        uint32_t *at = reinterpret_cast<uint32_t *>(v + ((ch >> 1) * kBN + key) * 128 + (((ch & 1) * 64 + i * 4) ^ ((key & 7) << 4)));
        uint32_t w = *at;
        for (int e = 0; e < 2; ++e) {
          const uint32_t x = (w >> (16 * e)) & 0xffffu;
          if ((x & top) != top) continue;
          const bool nan = (x & 0x7fffu) != top;
          up[k] |= uint32_t(nan || !(x & 0x8000u)) << (2 * i + e);
          down[k] |= uint32_t(nan || (x & 0x8000u)) << (2 * i + e);
          w &= ~(0xffffu << (16 * e));
        }
        *at = w;
      }
    }
    const bool more = again || k0 > 0;
    for (int t = 0; t < o.ntok; ++t) {
      const int pos = o.pos0 + t;
      uint32_t u = 0, d = 0;
      for (int k = 0; k < kKeys; ++k) {
        const int c = o.c0 + k0 + k;
        if (c > pos || (p.window > 0 && c <= pos - p.window && c >= p.sinks)) continue;
        u |= up[k];
        d |= down[k];
      }
      for (int row = t * p.G; row < (t + 1) * p.G; ++row) {
        if (!FFTS_IN_RANGE(row, p.rows)) continue;
        notes[row * 8 + ch] = more ? notes[row * 8 + ch] | u : u;
        notes[row * 8 + 4 + ch] = more ? notes[row * 8 + 4 + ch] | d : d;
      }
    }
  }
  *notes_seg = o.seg;
  __threadfence_block();
  fence_proxy_async();
}

template <typename E, int D>
__global__ void __launch_bounds__(kThreads, 2)
    attn_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ Params p) {
  using Lay = Layout<D>;
  constexpr int kSum = Num<E>::sum_keys / kBN;  // key tiles after which O is parked
  extern __shared__ __align__(16) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {  // SWIZZLE_128B tiles need 1024-byte alignment
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (threadIdx.x == 0) {
      *reinterpret_cast<volatile int *>(p.status) = kErrSmemAlign;
      p.cuts[blockIdx.x].nrows = 0;
    }
    return;
  }
  const uint32_t sbase = smem_u32(smem);
  auto bar = [&](int i) { return sbase + Lay::bars + 8u * uint32_t(i); };
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + Lay::abort);
  volatile OddTile *odd = reinterpret_cast<volatile OddTile *>(smem + Lay::odd);
  volatile int *notes_seg = reinterpret_cast<volatile int *>(smem + Lay::noted);
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + Lay::tmem_slot);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int qrows = p.tpt * p.G;  // rows a Q load fills

  if (threadIdx.x == 0) {
    *abort_flag = *notes_seg = odd[0].seg = odd[1].seg = 0;
    for (int i = 0; i < Lay::nbars; ++i) mbar_init(bar(i), (i == BPF || i == BPF + 1) ? 128u : 1u);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 4 && lane == 0) {
    prefetch_map(&tm_q);
    prefetch_map(&tm_k);
    prefetch_map(&tm_v);
  }
  // launched while the kernel before drains: nothing in global memory is touched before this
  asm volatile("griddepcontrol.wait;" ::: "memory");
  Tile *tiles = p.tiles;
  long long *cum = p.cum;
  int ntiles;
  long long length;
  if (p.own_schedule) {
    tiles += int64_t(blockIdx.x) * p.max_tiles;
    cum += int64_t(blockIdx.x) * (p.max_tiles + 1);
    // the scratch lies where the K ring will be
    ntiles = build_schedule<kBN, kThreads>(p, tiles, cum, *reinterpret_cast<SchedScratch<kThreads> *>(smem + Lay::k), &length);
  } else {
    ntiles = p.header[0];
    length = cum[FFTS_INDEX(ntiles, p.max_tiles + 1)];
  }
  length *= p.Hkv;
  const long long per = share_of(p, length);
  const long long u0 = per * blockIdx.x, u1 = min(length, u0 + per);
  if (u0 >= u1) {  // uniform in the CTA, before any allocation
    if (threadIdx.x == 0) p.cuts[blockIdx.x].nrows = 0;
    return;
  }
  // rows of Q that no load fills stay zeros
  for (int i = threadIdx.x; i < Lay::q_bytes / 16; i += kThreads)
    *reinterpret_cast<uint4 *>(smem + Lay::q + i * 16) = make_uint4(0, 0, 0, 0);
  fence_proxy_async();  // TMA writes over the scratch, the MMAs read the zeros
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tm_o = tmem + kTmemO;

  Walk<kBN> w(p, tiles, cum);
  w.seek(u0, u1, ntiles);

  if (warp == 4) {
    // ============================================================ producer (whole warp)
    const int ps = 1 << p.ps_shift;
    const int box = min(ps, kBN);              // rows of one box
    const int boxes = (kBN / box) * Lay::halves;
    const int my_box = lane / Lay::halves, my_half = lane % Lay::halves;
    const uint32_t my_dst = uint32_t(my_half * Lay::kv_half + my_box * box * 128);
    // the lane's box of one key tile
    struct Load {
      int page, row, h;
    };
    int j = 0, j1 = 0;
    bool fresh = false;  // the fetched tile is its segment's first
    auto fetch = [&](Load &l) -> bool {
      fresh = j >= j1;
      if (fresh) {
        if (!w.segment()) return false;
        j = w.j0;
        j1 = w.j1;
      }
      const int c = w.key(j) * kBN + my_box * box;  // first key of the box
      ++j;
      l.page = -1;
      l.row = c & (ps - 1);
      l.h = w.h;
      if (lane < boxes && c < w.g.hi && (c + box > w.g.lo || c < p.sinks))
        l.page = p.table[int64_t(w.t.r) * p.table_ld + FFTS_INDEX(c >> p.ps_shift, p.width)];
      return true;
    };
    bool ok = true;
    int nk = 0, nv = 0, nq = 0;  // loads issued
    int filled = 0;              // rows of Q that are not zeros
    auto load = [&](const Load &l, bool is_k) {
      const int n = is_k ? nk : nv;
      const int stages = is_k ? kKStages : kVStages, s = n % stages;
      const int full = (is_k ? BKF : BVF) + s, empty = (is_k ? BKE : BPV) + s;
      ok = ok && __all_sync(0xffffffffu, mbar_wait(bar(empty), ((n / stages) & 1) ^ 1, abort_flag, p.wait_cycles));
      if (!ok) return;
      if (lane == 0) mbar_arrive_tx(bar(full), Lay::kv_bytes);
      __syncwarp();
      const uint32_t dst = sbase + (is_k ? Lay::k : Lay::v) + s * Lay::kv_bytes + my_dst;
      if (lane < boxes) tma_load_4d(dst, is_k ? &tm_k : &tm_v, bar(full), my_half * 64, l.row, l.h, l.page);
      if (is_k) ++nk; else ++nv;
    };
    Load cur{}, prev{};
    bool more = fetch(cur);
    while (more && ok) {
      const bool cur_fresh = fresh;
      const int tok0 = w.t.tok0, qh = w.h * p.G, rows = w.t.ntok * p.G;
      // K(n), V(n - 1); a new segment's Q waits for the last S of the one before, so V(n - 1) goes first
      if (cur_fresh && nk > 0) load(prev, false);
      load(cur, true);
      if (cur_fresh && ok) {
        ok = __all_sync(0xffffffffu, mbar_wait(bar(BQE), (nq & 1) ^ 1, abort_flag, p.wait_cycles));
        if (ok && rows <= kFewRows) {
          // Decoding: the few rows themselves, and zeros behind them.  A box would bring the rows of other
          // requests along, whose products cost power: 64 requests' step ran at 1016 W, 1.43 GHz and 179 us.
          constexpr int kVecs = D / 8;
          for (int i = lane; i < rows * kVecs; i += 32) {
            const int r = i / kVecs, c = i % kVecs;
            const int tok = FFTS_INDEX(tok0 + r / p.G, p.T);
            *reinterpret_cast<uint4 *>(smem + Lay::q + (c >> 3) * Lay::q_half + r * 128 + (((c & 7) ^ (r & 7)) << 4)) =
                *reinterpret_cast<const uint4 *>(p.q + int64_t(tok) * p.qs_t + int64_t(qh + r % p.G) * p.qs_h + c * 8);
          }
          for (int i = rows * kVecs + lane; i < filled * kVecs; i += 32) {
            const int r = i / kVecs, c = i % kVecs;
            *reinterpret_cast<uint4 *>(smem + Lay::q + (c >> 3) * Lay::q_half + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          filled = rows;
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(BQF));
        } else if (ok) {
          if (lane == 0) {
            mbar_arrive_tx(bar(BQF), uint32_t(qrows * D * 2));
            for (int hf = 0; hf < Lay::halves; ++hf)
              tma_load_3d(sbase + Lay::q + hf * Lay::q_half, &tm_q, bar(BQF), hf * 64, qh, tok0);
          }
          filled = qrows;
        }
        if (ok) ++nq;
      }
      Load next = cur;
      more = fetch(next);  // its page numbers arrive while the stages fill
      if (!cur_fresh && nk > 1) load(prev, false);
      prev = cur;
      cur = next;
    }
    if (ok && nk > 0) load(prev, false);
    if (!ok) {
      if (lane == 0) {
        *abort_flag = 1;
        *reinterpret_cast<volatile int *>(p.status) = kErrProducer;
        // wait (bounded, ignoring the abort flag) for the copies in flight
        volatile int never = 0;
        if (nq > 0) mbar_wait(bar(BQF), (nq - 1) & 1, &never, p.drain_cycles);
        for (int n = max(0, nk - kKStages); n < nk; ++n)
          mbar_wait(bar(BKF + n % kKStages), (n / kKStages) & 1, &never, p.drain_cycles);
        for (int n = max(0, nv - kVStages); n < nv; ++n)
          mbar_wait(bar(BVF + n % kVStages), (n / kVStages) & 1, &never, p.drain_cycles);
      }
      __syncwarp();
    }
  } else if (warp == 5) {
    // ============================================================ MMA issuer (one thread)
    if (elect_one()) {
      constexpr uint32_t idS = idesc(Num<E>::fmt, false, kBN), idPV = idesc(Num<E>::fmt, true, D);
      constexpr uint32_t idS64 = idesc(Num<E>::fmt, false, kBN, 64), idPV64 = idesc(Num<E>::fmt, true, D, 64);
      const uint64_t dk_ = smem_desc(sbase, 16, 1024), dv_ = smem_desc(sbase, Lay::kv_half, 1024);
      const uint32_t dk_hi = uint32_t(dk_ >> 32), dv_hi = uint32_t(dv_ >> 32);
      const uint32_t dq = uint32_t(dk_) + (Lay::q >> 4), dk0 = uint32_t(dk_) + (Lay::k >> 4),
                     dv0 = uint32_t(dv_) + (Lay::v >> 4);
      bool ok = true;
      // S runs up to two tiles ahead of PV.  s_left: S tiles left in the walked segment; the PV side
      // needs only to know which tiles begin a sum and which have few rows (bit n % 32 of firsts and smalls).
      int s = 0, seg = 0, s_left = 0;
      uint32_t firsts = 0, smalls = 0;
      bool small = false;
      bool more = w.segment();
      for (int n = 0; ok && (more || n < s); ++n) {
        while (more && s < n + 2) {
          const bool first = s_left == 0;
          if (first) {
            // a new segment's Q is not there yet: PV tiles that are due go first
            if (s > n && !mbar_try(bar(BQF), seg & 1)) break;
            ok = mbar_wait(bar(BQF), seg & 1, abort_flag, p.wait_cycles);
            if (!ok) break;
            s_left = w.j1 - w.j0;
            small = w.t.ntok * p.G <= kSmallRows;
            ++seg;
          }
          const bool fresh = (w.j1 - w.j0 - s_left) % kSum == 0;  // O starts from zero
          const int ks = s % kKStages;
          ok = mbar_wait(bar(BKF + ks), (s / kKStages) & 1, abort_flag, p.wait_cycles);
          if (!ok) break;
          fence_after();
          const uint32_t dk = dk0 + ((ks * Lay::kv_bytes) >> 4);
          const uint32_t td = tmem + (s & 1) * kBN;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t qoff = ((kk >> 2) * Lay::q_half + (kk & 3) * 32) >> 4;
            const uint32_t koff = ((kk >> 2) * Lay::kv_half + (kk & 3) * 32) >> 4;
            umma_ss(td, dq + qoff, dk_hi, dk + koff, dk_hi, small ? idS64 : idS, kk > 0);
          }
          umma_commit(bar(BSF + (s & 1)));
          umma_commit(bar(BKE + ks));
          smalls = (smalls & ~(1u << (s & 31))) | (uint32_t(small) << (s & 31));
          if (--s_left == 0) {
            umma_commit(bar(BQE));
            more = w.segment();
          }
          firsts = (firsts & ~(1u << (s & 31))) | (uint32_t(fresh) << (s & 31));
          ++s;
        }
        if (!ok) break;
        const int b = n & 1;
        ok = mbar_wait(bar(BVF + b), (n >> 1) & 1, abort_flag, p.wait_cycles) &&
             mbar_wait(bar(BPF + b), (n >> 1) & 1, abort_flag, p.wait_cycles);
        if (!ok) break;
        fence_after();
        if (odd[b].seg) {
          const OddTile o{odd[b].seg, odd[b].pos0, odd[b].ntok, odd[b].c0};
          odd[b].seg = 0;
          note_odd<E, D>(p, smem + Lay::v + b * Lay::kv_bytes, o, notes_seg);
        }
        const bool first = (firsts >> (n & 31)) & 1u;
        const uint32_t dv = dv0 + ((b * Lay::kv_bytes) >> 4);
        const uint32_t pt = tmem + b * kBN;  // P(n): pairs in the first 32 columns of S buffer n % 2
#pragma unroll
        for (int kk = 0; kk < kBN / 16; ++kk)
          umma_ts(tm_o, pt + kk * 8, dv + ((kk * 2048) >> 4), dv_hi, (smalls >> (n & 31)) & 1u ? idPV64 : idPV,
                  !first || kk > 0);
        umma_commit(bar(BPV + b));
      }
      if (!ok) {
        *abort_flag = 1;
        *reinterpret_cast<volatile int *>(p.status) = kErrMma;
      }
      // wait (bounded) until every MMA this thread issued has completed
      umma_commit(bar(BDRAIN));
      volatile int never = 0;
      mbar_wait(bar(BDRAIN), 0, &never, p.drain_cycles);
    }
  } else {
    // ============================================================ softmax (warps 0-3)
    const int r = threadIdx.x;
    const int tl = r / p.G, hg = r - tl * p.G;  // the row's token in the tile and head in the group
    const uint32_t lane_off = uint32_t(warp * 32) << 16;
    const float2 sc2 = make_float2(p.scale_log2, p.scale_log2);
    bool ok = true, first_seg = true, noted = false;
    int n = 0;
    for (int seg = 1; ok && w.segment(); ++seg) {
      const Keys g = w.g;
      const int nrows = w.t.ntok * p.G;
      const bool active = warp * 32 < nrows, live = r < nrows;
      // rows of no token take the last token's mask; nobody reads them
      const int pos = w.t.pos0 + min(tl, w.t.ntok - 1);
      // and their P is 0, by an offset of -inf
      float m_ref = live ? -INFINITY : 0.0f, l_run = 0.0f;
      for (int j = w.j0, stop = j; ok && j < w.j1;) {
        if (j == stop) stop = min(w.j1, j + kSum);
        for (; j < stop; ++j, ++n) {
          const int b = n & 1;
          const uint32_t parity = (n >> 1) & 1;
          if (!__all_sync(0xffffffffu, mbar_wait(bar(BSF + b), parity, abort_flag, p.wait_cycles))) { ok = false; break; }
          fence_after();
          const int c0 = w.key(j) * kBN;
          if (has_unseen<kBN>(g, p.sinks, c0)) {
            // V rows that no row sees
            if (!__all_sync(0xffffffffu, mbar_wait(bar(BVF + b), parity, abort_flag, p.wait_cycles))) { ok = false; break; }
            const int key = c0 + (r & 63);
            if (r < 64 * Lay::halves && (key >= g.hi || (key < g.lo && key >= p.sinks))) {
              uint8_t *vr = smem + Lay::v + b * Lay::kv_bytes + (r >> 6) * Lay::kv_half + (r & 63) * 128;
#pragma unroll
              for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4 *>(vr + i * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async();
          }
          if (active) {
            uint64_t mask = below(pos + 1 - c0);
            if (p.window > 0) mask &= ~below(pos - p.window + 1 - c0) | below(p.sinks - c0);
            const bool edge = __any_sync(0xffffffffu, mask != ~0ull);
            const uint32_t s_addr = tmem + b * kBN + lane_off;
            float x[kBN];
            tmem_ld32(s_addr, x);
            tmem_wait_ld();
            tmem_ld32(s_addr + 32, x + 32);  // lands while the first half is processed
            if (edge) {
#pragma unroll
              for (int c = 0; c < 32; ++c)
                if (!((uint32_t(mask) >> c) & 1u)) x[c] = -INFINITY;
            }
            // P = exp2(s * scale - m_ref) as pairs over the first 32 columns of this S buffer (columns
            // already read).  The common path takes m_ref as it stands and keeps the result when every
            // P of the row is small enough (by the tile's row sum); a row's first tile with a key, or one
            // that outgrows m_ref, takes the max path: new m_ref, O and l rescaled, P again.
            float2 rs2[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
            float alpha = 1.0f;
            bool fast = !__any_sync(0xffffffffu, m_ref == -INFINITY);
            auto exp_half = [&](int cc, float2 off2) {
              uint32_t pk[16];
#pragma unroll
              for (int e = 0; e < 32; e += 2) {
                const int c = cc * 32 + e;
                const float2 a = __ffma2_rn(make_float2(x[c], x[c + 1]), sc2, off2);
                float2 ex;
                ex.x = fast_exp2(a.x);
                ex.y = fast_exp2(a.y);
                rs2[(e >> 1) & 1] = __fadd2_rn(rs2[(e >> 1) & 1], ex);
                pk[e >> 1] = Num<E>::pack(ex.x, ex.y);
              }
              tmem_st16u(s_addr + cc * 16, pk);
            };
            auto mask_high = [&]() {
              if (edge) {
#pragma unroll
                for (int c = 0; c < 32; ++c)
                  if (!((uint32_t(mask >> 32) >> c) & 1u)) x[32 + c] = -INFINITY;
              }
            };
            if (fast) {
              const float moff = live ? m_ref * p.scale_log2 - Num<E>::bias : INFINITY;
              exp_half(0, make_float2(-moff, -moff));
              tmem_wait_ld();
              mask_high();
              exp_half(1, make_float2(-moff, -moff));
              const float tsum = (rs2[0].x + rs2[0].y) + (rs2[1].x + rs2[1].y);
              if (__any_sync(0xffffffffu, !(tsum <= Num<E>::pmax))) {
                fast = false;
                tmem_wait_st();  // the max path below rewrites P
                rs2[0] = rs2[1] = make_float2(0.0f, 0.0f);
              }
            } else {
              tmem_wait_ld();
              mask_high();
            }
            if (!fast) {
              float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
              for (int c = 0; c < kBN; c += 2) mx4[(c >> 1) & 3] = max3f(mx4[(c >> 1) & 3], x[c], x[c + 1]);
              const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
              if (mx > m_ref && (m_ref == -INFINITY || (mx - m_ref) * p.scale_log2 > Num<E>::rescale)) {
                alpha = m_ref == -INFINITY ? 0.0f : fast_exp2((m_ref - mx) * p.scale_log2);
                m_ref = mx;
              }
              const float moff = live ? (m_ref == -INFINITY ? 0.0f : m_ref) * p.scale_log2 - Num<E>::bias : INFINITY;
              exp_half(0, make_float2(-moff, -moff));
              exp_half(1, make_float2(-moff, -moff));
            }
            const float2 rsum = __fadd2_rn(rs2[0], rs2[1]);
            l_run = l_run * alpha + (rsum.x + rsum.y);
            tmem_wait_st();
            if (j > w.j0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
              // O must hold PV(n-1) before it is rescaled; its barrier's next phase needs P(n+1)
              if (!__all_sync(0xffffffffu,
                              mbar_wait(bar(BPV + (n - 1) % 2), ((n - 1) >> 1) & 1, abort_flag, p.wait_cycles))) {
                ok = false;
                break;
              }
              fence_after();
#pragma unroll 1
              for (int c = 0; c < D / 32; ++c) {
                float o[32];
                tmem_ld32(tm_o + lane_off + c * 32, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                  const float2 v = __fmul2_rn(make_float2(o[e], o[e + 1]), make_float2(alpha, alpha));
                  o[e] = v.x;
                  o[e + 1] = v.y;
                }
                tmem_st32(tm_o + lane_off + c * 32, o);
              }
              tmem_wait_st();
            }
          }
          if (rows_differ<kBN>(w.t.pos0, w.t.ntok, p.window, p.sinks, c0)) break;
          fence_before();
          mbar_arrive(bar(BPF + b));
        }
        if (ok && j < stop) {  // the same for a tile that rows differ in; outside of the loop, which has no registers to give
          const int b = n & 1, key = w.key(j) * kBN + (r & 63);
          ok = __all_sync(0xffffffffu, mbar_wait(bar(BVF + b), (n >> 1) & 1, abort_flag, p.wait_cycles));
          if (!ok) break;
          if (r < 64 * Lay::halves && key < g.hi && (key >= g.lo || key < p.sinks) &&
              has_odd<E>(smem + Lay::v + b * Lay::kv_bytes + (r >> 6) * Lay::kv_half + (r & 63) * 128)) {
            odd[b].pos0 = w.t.pos0;
            odd[b].ntok = w.t.ntok;
            odd[b].c0 = w.key(j) * kBN;
            odd[b].seg = seg;
          }
          fence_before();
          mbar_arrive(bar(BPF + b));
          ++j;
          ++n;
        }
        if (ok && j == stop && j < w.j1) {
          // PV(n - 1), whose barrier's next phase needs P(n + 1)
          ok = __all_sync(0xffffffffu, mbar_wait(bar(BPV + (n - 1) % 2), ((n - 1) >> 1) & 1, abort_flag, p.wait_cycles));
          if (!ok) break;
          fence_after();
          const int slot = 2 * int(blockIdx.x) + (first_seg ? 0 : 1);
          if (active && FFTS_IN_RANGE(slot, 2 * p.ctas))
            park_o<D, kBM>(p, slot, r, live, j - w.j0 > kSum, m_ref * p.scale_log2, tm_o + lane_off);
        }
      }
      if (!ok) break;
      // O is final once the segment's last PV is complete (its barrier's next phase needs our P)
      if (!__all_sync(0xffffffffu, mbar_wait(bar(BPV + (n - 1) % 2), ((n - 1) >> 1) & 1, abort_flag, p.wait_cycles))) {
        ok = false;
        break;
      }
      fence_after();
      const int slot = 2 * int(blockIdx.x) + (first_seg ? 0 : 1);
      if (active) {
        const bool whole = w.j0 == 0 && w.j1 == g.n;
        // (l sums the weights before their rounding to E: sums of the rounded ones, which would give a constant v back
        // exactly, took ragged chunks from 79 to 84 us and windowed ones from 60 to 69, and brought single rows of random
        // values 4% nearer to 64 bits in the median)
        // a row without a key (pos < 0) is zeros; NaN in l, or no key above -inf (l == 0), is NaN as in the formula
        const bool sees = pos >= 0;
        const float inv_l = 1.0f / l_run;
        uint16_t *dst = p.out + int64_t(w.t.tok0 + tl) * p.os_t + int64_t(w.h * p.G + hg) * p.os_h;
        float4 *pd = reinterpret_cast<float4 *>(p.part) + int64_t(slot) * (kBM * D / 4) + r;
        float2 *pml = p.part_ml + int64_t(slot) * kBM + r;
        const bool parked = w.j1 - w.j0 > kSum && live && FFTS_IN_RANGE(slot, 2 * p.ctas);
        const float f = parked ? weight(pml->x, m_ref * p.scale_log2) : 0.0f;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          float o[32];
          __syncwarp();
          tmem_ld32(tm_o + lane_off + c * 32, o);
          tmem_wait_ld();
          if (parked) unpark<kBM>(o, pd, c, f);
          if (live && whole && FFTS_IN_RANGE(w.t.tok0 + tl, p.T)) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint32_t v[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                v[e] = Num<E>::pack(sees ? o[q * 8 + 2 * e] * inv_l : 0.0f, sees ? o[q * 8 + 2 * e + 1] * inv_l : 0.0f);
              *reinterpret_cast<uint4 *>(dst + c * 32 + q * 8) = make_uint4(v[0], v[1], v[2], v[3]);
            }
          }
          if (live && !whole && FFTS_IN_RANGE(slot, 2 * p.ctas)) park<kBM>(o, pd, c);
        }
        if (live && !whole && FFTS_IN_RANGE(slot, 2 * p.ctas)) *pml = make_float2(m_ref * p.scale_log2, l_run);
        if (live && *notes_seg == seg) {
          if (whole && FFTS_IN_RANGE(w.t.tok0 + tl, p.T)) put_back<E, D, kBM>(p, r, reinterpret_cast<E *>(dst));
          if (!whole && FFTS_IN_RANGE(slot, 2 * p.ctas)) put_back<E, D, kBM>(p, r, reinterpret_cast<float *>(pd));
        }
      }
      // the share that opens a (q tile, head) and does not end it leaves a note for the join
      if (w.opens && w.j1 - w.j0 < g.n && r == 0 && FFTS_IN_RANGE(blockIdx.x, p.ctas)) {
        Cut cut;
        cut.tok0 = w.t.tok0;
        cut.pos0 = w.t.pos0;
        cut.nrows = nrows;
        cut.head0 = w.h * p.G;
        cut.s1 = w.last_share(u0, per);
        cut.first_slot = 2 * int(blockIdx.x) + (first_seg ? 0 : 1);
        p.cuts[blockIdx.x] = cut;
        noted = true;
      }
      first_seg = false;
    }
    if (r == 0 && !noted) p.cuts[blockIdx.x].nrows = 0;
    if (!ok) {
      *abort_flag = 1;
      *reinterpret_cast<volatile int *>(p.status) = kErrSoftmax;
    }
  }

  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 5) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
}

// ---------------------------------------------------------------- join
// Blocks (s0, y): the (q tile, head) that share s0 begins and others go on with, the pieces of many rows by turns.
// For each row o = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s over the shares s, with M taken along as they are
// read.  A partial is stored 16-byte piece by piece over the rows ([D / 4][rows]), so neighbouring threads, on
// neighbouring rows, read and write whole sectors.  The time is that of the rounds through L2: a thread has four
// pieces in flight, and where a tile has few rows (decoding), groups of threads take the shares in turn and meet
// in shared memory, in the order of the groups.
constexpr int kJoinThreads = 512;
// 1, 2 and 4 blocks: 16.5, 11.5, 11.2 us after ragged chunks, 4.5, 4.4, 5.7 us after 64 decoding requests
constexpr int kJoinBlocks = 2;

// (m, l, o) of some shares, o a piece of a row; m = -inf: no score above -inf among them (l is 0, or NaN if one was).
struct Part {
  float m, l;
  float4 o;
  __device__ __forceinline__ void scale(float f) {
    l *= f;
    o.x *= f;
    o.y *= f;
    o.z *= f;
    o.w *= f;
  }
  __device__ __forceinline__ void add(float f, float ll, const float4 &v) {
    l = fmaf(f, ll, l);
    o.x = fmaf(f, v.x, o.x);
    o.y = fmaf(f, v.y, o.y);
    o.z = fmaf(f, v.z, o.z);
    o.w = fmaf(f, v.w, o.w);
  }
};

template <typename E, int D>
__global__ void __launch_bounds__(kJoinThreads, 2) join_kernel(const __grid_constant__ Params p) {
  __shared__ Part met[kJoinThreads];
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched early: attn_kernel's stores are visible from here
  const int s0 = int(blockIdx.x), tid = int(threadIdx.x);
  const Cut cut = p.cuts[s0];
  if (cut.nrows == 0) return;
  int rows = 1;
  while (rows < cut.nrows) rows <<= 1;
  const int items = rows * (D / 4);  // (piece, row), rows side by side
  const float4 *part = reinterpret_cast<const float4 *>(p.part);
  auto store = [&](int r, int piece, const Part &t) {
    const int tl = r / p.G, hg = r - tl * p.G;
    if (!FFTS_IN_RANGE(cut.tok0 + tl, p.T)) return;
    const float inv_l = 1.0f / t.l;
    uint2 o = make_uint2(0u, 0u);
    if (cut.pos0 + tl >= 0)  // the row sees a key
      o = make_uint2(Num<E>::pack(t.o.x * inv_l, t.o.y * inv_l), Num<E>::pack(t.o.z * inv_l, t.o.w * inv_l));
    *reinterpret_cast<uint2 *>(p.out + int64_t(cut.tok0 + tl) * p.os_t + int64_t(cut.head0 + hg) * p.os_h + piece * 4) = o;
  };
  // pieces piece + i * step (i < JP) of row r over shares s, s + by, ..., JS at a time; indices in 32 bits: at
  // most 1024 slots of 256 rows of 32 pieces
  auto gather = [&](auto js, auto jp, Part *t, int r, int piece, int step, int s, int by) {
    constexpr int JS = decltype(js)::value, JP = decltype(jp)::value;
    for (; s <= cut.s1; s += JS * by) {
      float2 ml[JS];
      float4 v[JS][JP];
#pragma unroll
      for (int k = 0; k < JS; ++k) {
        ml[k] = make_float2(-INFINITY, 0.0f);
        const int sk = s + k * by;
        if (sk > cut.s1) continue;
        const uint32_t at = uint32_t(FFTS_INDEX(sk == s0 ? cut.first_slot : 2 * sk, 2 * p.ctas));
        ml[k] = __ldcg(&p.part_ml[at * p.rows + r]);
#pragma unroll
        for (int i = 0; i < JP; ++i)
          if (piece + i * step < D / 4) v[k][i] = __ldcg(part + ((at * (D / 4) + piece + i * step) * p.rows + r));
      }
      float top = t[0].m;
#pragma unroll
      for (int k = 0; k < JS; ++k) top = fmaxf(top, ml[k].x);
      const float old = weight(t[0].m, top);
#pragma unroll
      for (int i = 0; i < JP; ++i) {
        t[i].m = top;
        t[i].scale(old);
      }
#pragma unroll
      for (int k = 0; k < JS; ++k) {
        if (ml[k].x == -INFINITY && ml[k].y == 0.0f) continue;  // no share, or none of its keys counts (NaN does)
        const float f = exp2f(ml[k].x - top);
#pragma unroll
        for (int i = 0; i < JP; ++i)
          if (piece + i * step < D / 4) t[i].add(f, ml[k].y, v[k][i]);
      }
    }
  };
  const Part none{-INFINITY, 0.0f, make_float4(0.0f, 0.0f, 0.0f, 0.0f)};
  if (items >= kJoinThreads) {
    const int step = kJoinBlocks * (kJoinThreads / rows);  // pieces the blocks cover at a time
    const int r = tid % rows;
    if (r >= cut.nrows) return;
    constexpr int JP = 2;
    for (int piece = int(blockIdx.y) + kJoinBlocks * (tid / rows); piece < D / 4; piece += JP * step) {
      Part t[JP];
#pragma unroll
      for (int i = 0; i < JP; ++i) t[i] = none;
      gather(std::integral_constant<int, 2>{}, std::integral_constant<int, JP>{}, t, r, piece, step, s0, 1);
#pragma unroll
      for (int i = 0; i < JP; ++i)
        if (piece + i * step < D / 4) store(r, piece + i * step, t[i]);
    }
    return;
  }
  if (blockIdx.y > 0) return;
  const int groups = kJoinThreads / items, g = tid / items, r = tid % rows, piece = tid % items / rows;
  Part t = none;
  if (r < cut.nrows)
    gather(std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{}, &t, r, piece, 1, s0 + g, groups);
  met[tid] = t;
  __syncthreads();
  if (g > 0 || r >= cut.nrows) return;
  float top = -INFINITY;
  for (int k = 0; k < groups; ++k) top = fmaxf(top, met[k * items + tid].m);
  Part sum = none;
  for (int k = 0; k < groups; ++k) {
    const Part &q = met[k * items + tid];
    sum.add(weight(q.m, top), q.l, q.o);
  }
  store(r, piece, sum);
}

// ---------------------------------------------------------------- host side
static PFN_cuTensorMapEncodeTiled_v12000 get_encode() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void *ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    return static_cast<PFN_cuTensorMapEncodeTiled_v12000>(nullptr);
  }();
  return fn;
}

static int encode(CUtensorMap *map, CUtensorMapDataType type, int rank, const void *base, const cuuint64_t *dims,
                  const cuuint64_t *strides, const cuuint32_t *box) {
  auto enc = get_encode();
  if (!enc) {
    set_error(FFTS_E_CUDA, "cuTensorMapEncodeTiled is unavailable");
    return FFTS_E_CUDA;
  }
  const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
  const CUresult r = enc(map, type, rank, const_cast<void *>(base), dims, strides, box, ones,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error(FFTS_E_INVALID, "paged_attn: cuTensorMapEncodeTiled failed (%d)", int(r));
    return FFTS_E_INVALID;
  }
  return FFTS_OK;
}

__device__ int g_status_sink;

// Workspace: cum, tiles, header, cuts, notes, partial (m, l), partial O; every part a multiple of 16 bytes.
struct Space {
  int64_t max_tiles, cum, tiles, header, cuts, notes, ml, part, bytes;
  Space(int64_t T, int64_t R, int64_t G, int64_t D) {
    const int64_t tpt = kBM / G;  // of the smaller tiles; the larger ones are fewer
    max_tiles = T / tpt + std::min(R, T);  // sum of ceil(len / tpt)
    const int64_t copies = max_tiles <= kOwnTiles ? kMaxCtas : 1;
    cum = 0;
    tiles = cum + (copies * (max_tiles + 1) + 1) / 2 * 16;
    header = tiles + copies * max_tiles * 16;
    cuts = header + 16;
    notes = cuts + kMaxCtas * int64_t(sizeof(Cut));
    ml = notes + int64_t(kMaxCtas) * kBM * 32;
    part = ml + int64_t(2 * kMaxCtas) * kBM * 8;
    bytes = part + int64_t(2 * kMaxCtas) * kBM * D * 4;
  }
};

template <typename E, int D>
static int launch(const Params &p, bool chunks, const ffts_paged_attn_args &a, cudaStream_t stream) {
  const int64_t *qs = a.q_strides, *ks = a.kp_strides, *vs = a.vp_strides;
  CUtensorMap mq, mk, mv;
  const cuuint64_t qd[3] = {D, cuuint64_t(a.H), cuuint64_t(a.T)};
  const cuuint64_t qst[2] = {cuuint64_t(qs[1]) * 2, cuuint64_t(qs[0]) * 2};
  const cuuint32_t qbox[3] = {64, cuuint32_t(p.G), cuuint32_t(kBM / p.G)};
  int rc = encode(&mq, Num<E>::map, 3, a.q, qd, qst, qbox);
  if (rc) return rc;
  const cuuint64_t ps = 1ull << p.ps_shift;
  const cuuint64_t kd[4] = {D, ps, cuuint64_t(a.Hkv), cuuint64_t(a.n_pages)};
  const cuuint32_t kbox[4] = {64, cuuint32_t(std::min<cuuint64_t>(ps, chunks ? 2 * kBN : kBN)), 1, 1};
  const cuuint64_t kst[3] = {cuuint64_t(ks[2]) * 2, cuuint64_t(ks[1]) * 2, cuuint64_t(ks[0]) * 2};
  const cuuint64_t vst[3] = {cuuint64_t(vs[2]) * 2, cuuint64_t(vs[1]) * 2, cuuint64_t(vs[0]) * 2};
  rc = encode(&mk, Num<E>::map, 4, a.k_pages, kd, kst, kbox);
  if (!rc) rc = encode(&mv, Num<E>::map, 4, a.v_pages, kd, vst, kbox);
  if (rc) return rc;
  if (chunks) {
    rc = launch_chunk(p, Num<E>::fmt == 0, D, mq, mk, mv, stream);
    if (rc) return rc;
  } else {
    rc = ensure_func_smem(reinterpret_cast<const void *>(&attn_kernel<E, D>), Layout<D>::bytes,
                          int(cudaSharedmemCarveoutMaxShared));
    if (rc) return rc;
    if (!p.own_schedule) {
      schedule_kernel<kBN><<<1, kSchedThreads, 0, stream>>>(p);
      FFTS_CUDA(cudaGetLastError());
    }
    rc = launch_early(attn_kernel<E, D>, dim3(unsigned(p.ctas)), kThreads, Layout<D>::bytes, stream, mq, mk, mv, p);
    if (rc) return rc;
  }
  return launch_early(join_kernel<E, D>, dim3(unsigned(p.ctas), kJoinBlocks), kJoinThreads, 0, stream, p);
}

}  // namespace paged

int64_t paged_workspace_bytes(int64_t T, int64_t R, int64_t H, int64_t Hkv, int64_t D) {
  if (T <= 0 || R <= 0 || H <= 0 || Hkv <= 0 || D <= 0 || H % Hkv || H / Hkv > paged::kBM) return 0;
  return paged::Space(T, R, H / Hkv, D).bytes;
}

int paged_attn(const ffts_paged_attn_args &a, cudaStream_t stream) {
  using namespace paged;
  const int64_t T = a.T, R = a.R, H = a.H, Hkv = a.Hkv, D = a.D, page_size = a.page_size, width = a.width;
  FFTS_REQUIRE(a.dtype == FFTS_DTYPE_BF16 || a.dtype == FFTS_DTYPE_F16, "paged_attn: dtype must be bf16 or fp16");
  FFTS_REQUIRE(D == 64 || D == 128, "paged_attn: head_dim must be 64 or 128 (got %lld)", (long long)D);
  FFTS_REQUIRE(T >= 0 && R >= 0 && H >= 1 && Hkv >= 1 && H % Hkv == 0 && H / Hkv <= kBM,
               "paged_attn: bad shape (T %lld, R %lld, H %lld, Hkv %lld; at most %d query heads per KV head)",
               (long long)T, (long long)R, (long long)H, (long long)Hkv, kBM);
  FFTS_REQUIRE(page_size >= 16 && page_size <= 256 && (page_size & (page_size - 1)) == 0,
               "paged_attn: page_size must be 16, 32, 64, 128 or 256 (got %lld)", (long long)page_size);
  FFTS_REQUIRE(T <= (int64_t(1) << 30) && R <= (int64_t(1) << 30) && H <= 65536 && a.n_pages < (int64_t(1) << 31) &&
                   width >= 0 && width <= (int64_t(1) << 30) / page_size,
               "paged_attn: shape too large (a table row spans at most 2^30 tokens)");
  FFTS_REQUIRE(Hkv * (ceil_div(width * page_size, kBN) + kOverhead) < (int64_t(1) << 31),
               "paged_attn: %lld KV heads over a table row of %lld tokens are too many", (long long)Hkv,
               (long long)(width * page_size));
  FFTS_REQUIRE(a.window >= 0 && a.sinks >= 0, "paged_attn: window and sinks must not be negative");
  FFTS_REQUIRE(a.scale > 0.0f && a.scale < 3.0e38f, "paged_attn: scale must be positive and finite");
  if (T == 0 || R == 0) return FFTS_OK;
  FFTS_REQUIRE(a.q && a.k_pages && a.v_pages && a.cu_q && a.kv_lens && a.out && a.workspace && (width == 0 || a.table) &&
                   a.n_pages >= 1,
               "paged_attn: NULL argument or empty pool");
  FFTS_REQUIRE(a.table_ld >= width || R == 1, "paged_attn: table rows overlap");
  for (const void *x : {a.q, a.k_pages, a.v_pages, static_cast<const void *>(a.out), static_cast<const void *>(a.workspace)})
    FFTS_REQUIRE((reinterpret_cast<uintptr_t>(x) & 15) == 0, "paged_attn: tensors must be 16-byte aligned");
  const int64_t *qs = a.q_strides, *os = a.out_strides;
  FFTS_REQUIRE(qs[0] > 0 && qs[1] > 0 && qs[0] % 8 == 0 && qs[1] % 8 == 0 && os[0] % 8 == 0 && os[1] % 8 == 0,
               "paged_attn: q and out strides must be multiples of 8 elements (16 bytes), q's positive");
  const int64_t out_sizes[2] = {T, H};
  FFTS_REQUIRE(rows_apart(out_sizes, os, 2, D), "paged_attn: rows of out overlap");
  for (const int64_t *st : {a.kp_strides, a.vp_strides})
    for (int i = 0; i < 3; ++i)
      FFTS_REQUIRE(st[i] > 0 && st[i] % 8 == 0 && st[i] < (int64_t(1) << 38),
                   "paged_attn: page strides must be positive multiples of 8 elements (16 bytes)");
  FFTS_REQUIRE(a.workspace_bytes >= paged_workspace_bytes(T, R, H, Hkv, D), "paged_attn: workspace too small");
  const int64_t G = H / Hkv;
  const Space sp(T, R, G, D);
  FFTS_REQUIRE(sp.max_tiles < (int64_t(1) << 31) - 1, "paged_attn: too many q tiles");
  uint8_t *base = static_cast<uint8_t *>(a.workspace);
  Params p{};
  p.T = int(T); p.R = int(R); p.Hkv = int(Hkv); p.G = int(G); p.tpt = int(kBM / G);
  p.table = a.table;
  p.table_ld = a.table_ld;
  p.width = int(width);
  p.ps_shift = ilog2_ceil(page_size);
  p.cu_q = a.cu_q;
  p.kv_lens = a.kv_lens;
  p.window = int(std::min<int64_t>(a.window, int64_t(1) << 30));
  p.sinks = a.window > 0 ? int(std::min<int64_t>(a.sinks, int64_t(1) << 30)) : 0;
  p.q = static_cast<const uint16_t *>(a.q);
  p.qs_t = qs[0];
  p.qs_h = qs[1];
  p.out = static_cast<uint16_t *>(a.out);
  p.os_t = os[0];
  p.os_h = os[1];
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.max_tiles = int(sp.max_tiles);
  p.own_schedule = sp.max_tiles <= kOwnTiles;
  p.cum = reinterpret_cast<long long *>(base + sp.cum);
  p.tiles = reinterpret_cast<Tile *>(base + sp.tiles);
  p.header = reinterpret_cast<int *>(base + sp.header);
  p.cuts = reinterpret_cast<Cut *>(base + sp.cuts);
  p.notes = reinterpret_cast<uint32_t *>(base + sp.notes);
  p.part_ml = reinterpret_cast<float2 *>(base + sp.ml);
  p.part = reinterpret_cast<float *>(base + sp.part);
  int sms = 0;
  int rc = device_sm_count(&sms);
  if (!rc) rc = device_wait_cycles(kWaitSeconds, &p.wait_cycles);
  if (!rc) rc = device_wait_cycles(kDrainSeconds, &p.drain_cycles);
  if (rc) return rc;
  // The larger tiles of paged_chunk.cu: where requests fill several of them on average and the keys that a tile sees,
  // as far as the table and the window bound them, are enough to pay for filling and draining one pipeline per SM
  // instead of two. In long loops under the power cap, against the tiles of paged_attn.cu (32 / 8 heads): 2048
  // tokens over nothing 58 and 63 us, over 4096 177 and 197, over 32768 1.05 and 1.21 ms; 512 over 8192 88 and 92; 16
  // ragged chunks of 780 rows on average 80 and 79; window 1024 at D = 64 61 and 60.
  // The average hides a long chunk among many decoding requests (and counts requests without tokens, and padding): 2048
  // tokens over 32768 beside 63 decoding ones take the smaller tiles, 1.33 ms instead of 1.26, 8192 5.8 instead of 5.0.
  int64_t span = width * page_size;
  if (p.window > 0) span = std::min(span, int64_t(p.window) + p.sinks);
  const bool chunks = T * G >= kLongRows * R && span >= kLongKeys;
  p.ctas = std::min(chunks ? sms : 2 * sms, kMaxCtas / (chunks ? 2 : 1));
  p.rows = chunks ? 2 * kBM : kBM;
  if (chunks) p.tpt *= 2;
  p.overhead = kOverhead;
  if (a.status) {
    p.status = a.status;
  } else {
    void *sink = nullptr;
    FFTS_CUDA(cudaGetSymbolAddress(&sink, g_status_sink));
    p.status = static_cast<int *>(sink);
  }
  if (a.dtype == FFTS_DTYPE_BF16)
    return D == 128 ? launch<__nv_bfloat16, 128>(p, chunks, a, stream) : launch<__nv_bfloat16, 64>(p, chunks, a, stream);
  return D == 128 ? launch<__half, 128>(p, chunks, a, stream) : launch<__half, 64>(p, chunks, a, stream);
}

}  // namespace ffts
