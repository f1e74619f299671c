// paged_chunk.cu -- the paged attention of paged_attn.cu for batches of longer chunks: tiles of 256 rows x 128 keys.
//
// Same schedule, shares and partials as paged_attn.cu.  Where a batch brings rows enough, what bounds it is
// the tensor core, the exponentials and the traffic of K and V, and larger tiles ease all three:
//   - A 64-key S = Q K^T reads 48 KB of shared memory for 256 clocks of products (the 128-row Q each
//     time), more than the 128 bytes a clock that it gets; with 128 keys it is 64 KB for 512.
//   - Two 128-row halves A and B of a q tile share every K and V tile, so half as many bytes are loaded per product.
//   - The halves take turns: while A's softmax works on its S, the tensor core runs B's products.  With S, P and O of
//     both halves the SM's 512 TMEM columns are full: one CTA per SM.
//
// Roles (384 threads; registers are split for the softmax warps, which hold a row's 128 scores):
//   warps 0-3 / 4-7  softmax of half A / B: thread r owns row r; P goes over the S columns already read.
//   warp 8           producer: Q of each half, then K(0), V(0), K(1), ... through one five-stage ring.
//   warp 10          keeper of V tiles with keys that not all rows see (paged_common.cuh).
//   warp 11          none (registers are split by warpgroup)
//   warp 9           MMA issuer (one thread): S_A, S_B, then per key tile n: PV_A(n), S_A(n + 1), PV_B(n), S_B(n + 1).
//                    The product of a half's first 64 keys starts while the exponentials of the others are computed.
// A commit tracks all earlier products of the issuing thread, so S_X(n + 1) being there means that PV_X(n) is
// complete: O may be rescaled then, and only a segment's end waits for its last PV.
// Every wait is bounded.
//
// 2048 tokens of 32 / 8 heads over 32768 cached: 0.93 ms, 1.21 PFLOP/s (0.74 of the measured bf16 burst), 1.05 to
// 1.09 ms once the power cap holds the clock.  A key tile of both halves takes about 3300 clocks, 2048 of them
// products: a half's softmax (about 1850 clocks: scores read and looked through 450, exponentials 1400) and its
// two products follow one another, and the other half's fill the gap only in part.

#include <algorithm>

#include "paged_common.cuh"

namespace ffts {
namespace paged {

constexpr int cBM = 128;       // rows of a half
constexpr int cBN = 128;       // keys of a key tile
constexpr int cThreads = 384;   // three warpgroups
// After the split; launched with 168 each, 2 * 200 + 104 <= 3 * 168.  Neither side has enough: 216 bytes are spilled
// (bf16; 208 and 80: 264), 144 of them by the softmax warps, whose row of scores alone takes 128.
constexpr int cRegsSoftmax = 200, cRegsOther = 104;
constexpr int cStages = 5;
constexpr int cTmemCols = 512;

template <int D>
struct ChunkLayout {
  static constexpr int halves = D / 64;         // 64-channel swizzle boxes per row
  static constexpr int box = 128 * 128;         // bytes of one box of 128 rows (or keys)
  static constexpr int tile = halves * box;     // one half's Q, a K tile or a V tile
  static constexpr int q = 0;
  static constexpr int kv = q + 2 * tile;
  static constexpr int bars = kv + cStages * tile;
  static constexpr int nbars = 3 * cStages + 2 + 2 + 2 + 4 + 2 + 1;
  static constexpr int tmem_slot = bars + nbars * 8;
  static constexpr int abort = tmem_slot + 8;
  static constexpr int notes = abort + 8;
  static constexpr int bytes = notes + 40;
  static_assert(bytes <= 227 * 1024, "one CTA must fit in an SM's shared memory");
};

constexpr int CKF = 0;              // ring stage loaded [cStages]
constexpr int CKE = CKF + cStages;  // ring stage free   [cStages]
constexpr int CVX = CKE + cStages;  // ring stage loaded with V, for the keeper [cStages]
constexpr int CQF = CVX + cStages;  // Q of half x loaded
constexpr int CQE = CQF + 2;        // the segment's S products have read it
constexpr int CSF = CQE + 2;        // S of half x
constexpr int CPF = CSF + 2;        // P of half x written for the first and last 64 keys (128 arrivals) [2 x + part]
constexpr int COF = CPF + 4;        // O of half x final
constexpr int CDRAIN = COF + 2;

// The keeper.  V tiles with keys that not all rows see pass through its hands before the MMA issuer gets them: their copies
// complete a barrier of the keeper's, and its arrival the one that the issuer waits for.
struct Notes {
  volatile int *segment;  // the segment of the notes, counted from 1
  volatile int *done;     // segments that each softmax warp has finished (one without rows runs ahead of the others)
  int warps;
};

// The keys of a V tile in shared memory (BN rows of 128 bytes for each 64 channels, swizzled), from c0 on (whole warp).
// False: the wait for the softmax ran out.
template <typename E, int D, int BN>
__device__ __forceinline__ bool keep_values(const Params &p, uint8_t *v, const Tile &t, const Keys &g, int c0, int seg,
                                            const Notes &notes, volatile int *abort_flag) {
  constexpr uint32_t top = Num<E>::exponent;
  const int lane = threadIdx.x & 31;
  if (has_unseen<BN>(g, p.sinks, c0)) {
#pragma unroll 4
    for (int i = lane; i < BN * D / 8; i += 32) {
      const int c = c0 + (i >> 3) % BN;
      if (c >= g.hi || (c < g.lo && c >= p.sinks)) *reinterpret_cast<uint4 *>(v + i * 16) = make_uint4(0, 0, 0, 0);
    }
    __syncwarp();
  }
  if (rows_differ<BN>(t.pos0, t.ntok, p.window, p.sinks, c0)) {
    uint32_t acc[4] = {0, 0, 0, 0};
#pragma unroll 8
    for (int i = lane; i < BN * D / 8; i += 32) {
      const uint4 w = *reinterpret_cast<const uint4 *>(v + i * 16);
      Num<E>::probe(w.x, acc[0]);
      Num<E>::probe(w.y, acc[1]);
      Num<E>::probe(w.z, acc[2]);
      Num<E>::probe(w.w, acc[3]);
    }
    if (__any_sync(0xffffffffu, ((acc[0] | acc[1] | acc[2] | acc[3]) & 0x7fff7fffu) != 0)) {
      const int nrows = min(t.ntok * p.G, p.rows);
      uint32_t *at = p.notes + int64_t(blockIdx.x) * p.rows * 8;
      if (*notes.segment != seg + 1) {  // the segments before may still need theirs
        const long long t0 = clock64();
        while (__any_sync(0xffffffffu, lane < notes.warps && notes.done[lane] < seg))
          if (__any_sync(0xffffffffu, *abort_flag || clock64() - t0 > p.wait_cycles)) return false;
        for (int i = lane; i < nrows * 8; i += 32) at[i] = 0;
        __syncwarp();
        *notes.segment = seg + 1;
      }
#pragma unroll 1
      for (int i = 0; i < BN * (D / 32); ++i) {
        const int key = i % BN, c = c0 + key, ch = i / BN;  // channel 32 ch + lane
        uint16_t *el = reinterpret_cast<uint16_t *>(v + ((ch >> 1) * BN + key) * 128 + (((ch & 1) * 64 + lane * 2) ^ ((key & 7) << 4)));
        const uint32_t x = *el;
        const bool odd = (x & top) == top, nan = odd && (x & 0x7fffu) != top;
        const uint32_t up = __ballot_sync(0xffffffffu, nan || (odd && !(x & 0x8000u)));
        const uint32_t down = __ballot_sync(0xffffffffu, nan || (odd && (x & 0x8000u)));
        if (!(up | down)) continue;
        if (odd) *el = 0;
        for (int row = lane; row < nrows; row += 32) {
          const int pos = t.pos0 + row / p.G;
          if (c > pos || (p.window > 0 && c <= pos - p.window && c >= p.sinks)) continue;
          at[row * 8 + ch] |= up;
          at[row * 8 + 4 + ch] |= down;
        }
      }
      __threadfence_block();
    }
  }
  fence_proxy_async();
  __syncwarp();
  return true;
}

template <typename E, int D>
__global__ void __launch_bounds__(cThreads, 1)
    chunk_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ Params p) {
  using Lay = ChunkLayout<D>;
  constexpr int kSum = Num<E>::sum_keys / cBN;  // key tiles after which O is parked
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
  volatile int *words = reinterpret_cast<volatile int *>(smem + Lay::notes);
  const Notes notes{words, words + 1, 8};
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + Lay::tmem_slot);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tph = cBM / p.G;        // tokens of a half
  const int qrows = tph * p.G;      // rows of it that a Q load fills

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < 1 + notes.warps; ++i) words[i] = 0;
    for (int i = 0; i < Lay::nbars; ++i) mbar_init(bar(i), (i >= CPF && i < CPF + 4) ? 128u : 1u);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8 && lane == 0) {
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
    // the scratch lies where the ring will be
    ntiles = build_schedule<cBN, cThreads>(p, tiles, cum, *reinterpret_cast<SchedScratch<cThreads> *>(smem + Lay::kv), &length);
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
  // rows no Q load fills: zeros, so that they stay finite
  for (int i = threadIdx.x; i < 2 * (cBM - qrows) * 8 * Lay::halves; i += cThreads) {
    const int at = i >> 3, hf = at % Lay::halves, row = qrows + (at / Lay::halves) % (cBM - qrows);
    const int x = at / Lay::halves / (cBM - qrows);
    *reinterpret_cast<uint4 *>(smem + Lay::q + x * Lay::tile + hf * Lay::box + row * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async();  // TMA writes over the scratch, the MMAs read the zeros
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(cTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;  // S_A, S_B (128 columns each), O_A, O_B

  Walk<cBN> w(p, tiles, cum);
  w.seek(u0, u1, ntiles);

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(cRegsOther));
    if (warp == 8) {
      // ============================================================ producer (whole warp)
      const int ps = 1 << p.ps_shift;
      const int box = min(ps, cBN);              // keys of one box
      const int boxes = (cBN / box) * Lay::halves;
      const int my_box = lane / Lay::halves, my_half = lane % Lay::halves;
      const uint32_t my_dst = uint32_t(my_half * Lay::box + my_box * box * 128);
      // kept: its V goes to the keeper
      struct Load {
        int page, row, h;
        bool kept;
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
        const int c0 = w.key(j) * cBN, c = c0 + my_box * box;  // first key of the tile, of the box
        ++j;
        l.kept = has_unseen<cBN>(w.g, p.sinks, c0) || rows_differ<cBN>(w.t.pos0, w.t.ntok, p.window, p.sinks, c0);
        l.page = -1;
        l.row = c & (ps - 1);
        l.h = w.h;
        if (lane < boxes && c < w.g.hi && (c + box > w.g.lo || c < p.sinks))
          l.page = p.table[int64_t(w.t.r) * p.table_ld + FFTS_INDEX(c >> p.ps_shift, p.width)];
        return true;
      };
      bool ok = true;
      int nl = 0, nq[2] = {0, 0};  // loads issued
      uint32_t kept = 0, odd = 0;  // load n is one for the keeper: bit n % 32; their number in each stage, modulo 2
      auto load = [&](const Load &l, const CUtensorMap *map, bool for_keeper) {
        const int s = nl % cStages;
        ok = ok && __all_sync(0xffffffffu, mbar_wait(bar(CKE + s), ((nl / cStages) & 1) ^ 1, abort_flag, p.wait_cycles));
        if (!ok) return;
        const uint32_t full = bar((for_keeper ? CVX : CKF) + s);
        if (lane == 0) mbar_arrive_tx(full, Lay::tile);
        __syncwarp();
        if (lane < boxes) tma_load_4d(sbase + Lay::kv + s * Lay::tile + my_dst, map, full, my_half * 64, l.row, l.h, l.page);
        kept = (kept & ~(1u << (nl & 31))) | (uint32_t(for_keeper) << (nl & 31));
        odd ^= uint32_t(for_keeper) << s;
        ++nl;
      };
      auto load_q = [&](int x, int tok0, int qh) {
        ok = ok && __all_sync(0xffffffffu, mbar_wait(bar(CQE + x), (nq[x] & 1) ^ 1, abort_flag, p.wait_cycles));
        if (!ok) return;
        if (lane == 0) {
          mbar_arrive_tx(bar(CQF + x), uint32_t(qrows * D * 2));
          for (int hf = 0; hf < Lay::halves; ++hf)
            tma_load_3d(sbase + Lay::q + x * Lay::tile + hf * Lay::box, &tm_q, bar(CQF + x), hf * 64, qh, tok0 + x * tph);
        }
        ++nq[x];
      };
      Load cur{};
      bool more = fetch(cur);
      while (more && ok) {
        // the ring's order is the MMA issuer's: K(n), V(n).  Q waits for the last S of the segment before,
        // whose K and V are all on their way by then.
        const int tok0 = w.t.tok0, qh = w.h * p.G;
        const bool first = fresh, two = w.t.ntok > tph;
        load(cur, &tm_k, false);
        if (first) {
          load_q(0, tok0, qh);
          if (two) load_q(1, tok0, qh);
        }
        Load next = cur;
        more = fetch(next);  // its page numbers arrive while the stages fill
        load(cur, &tm_v, cur.kept);
        cur = next;
      }
      if (!ok) {
        if (lane == 0) {
          *abort_flag = 1;
          *reinterpret_cast<volatile int *>(p.status) = kErrProducer;
          // wait (bounded, ignoring the abort flag) for the copies in flight
          volatile int never = 0;
          for (int x = 0; x < 2; ++x)
            if (nq[x] > 0) mbar_wait(bar(CQF + x), (nq[x] - 1) & 1, &never, p.drain_cycles);
          for (int n = max(0, nl - cStages); n < nl; ++n) {
            const int s = n % cStages;
            if ((kept >> (n & 31)) & 1u) mbar_wait(bar(CVX + s), ((odd >> s) & 1u) ^ 1, &never, p.drain_cycles);
            else mbar_wait(bar(CKF + s), (n / cStages) & 1, &never, p.drain_cycles);
          }
        }
        __syncwarp();
      }
    } else if (warp == 9) {
      // ============================================================ MMA issuer (one thread)
      if (elect_one()) {
        constexpr uint32_t idS = idesc(Num<E>::fmt, false, cBN), idPV = idesc(Num<E>::fmt, true, D);
        const uint64_t dk_ = smem_desc(sbase, 16, 1024), dv_ = smem_desc(sbase, Lay::box, 1024);
        const uint32_t dk_hi = uint32_t(dk_ >> 32), dv_hi = uint32_t(dv_ >> 32);
        const uint32_t dq_lo = uint32_t(dk_) + (Lay::q >> 4), dk_lo = uint32_t(dk_) + (Lay::kv >> 4),
                       dv_lo = uint32_t(dv_) + (Lay::kv >> 4);
        bool ok = true;
        int nl = 0;                  // ring loads consumed up to the current K
        int np[2] = {0, 0}, nseg[2] = {0, 0};
        auto full = [&](int n) { return mbar_wait(bar(CKF + n % cStages), (n / cStages) & 1, abort_flag, p.wait_cycles); };
        auto issue_s = [&](int x, int stage) {
          fence_after();
          const uint32_t dq = dq_lo + ((x * Lay::tile) >> 4), dk = dk_lo + ((stage * Lay::tile) >> 4);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = ((kk >> 2) * Lay::box + (kk & 3) * 32) >> 4;
            umma_ss(tmem + x * cBN, dq + off, dk_hi, dk + off, dk_hi, idS, kk > 0);
          }
          umma_commit(bar(CSF + x));
        };
        auto issue_pv = [&](int x, int stage, int part, bool first) {
          fence_after();
          const uint32_t dv = dv_lo + ((stage * Lay::tile) >> 4) + part * ((4 * 2048) >> 4);
#pragma unroll
          for (int kk = 0; kk < cBN / 32; ++kk)
            umma_ts(tmem + 256 + x * 128, tmem + x * cBN + part * 32 + kk * 8, dv + ((kk * 2048) >> 4), dv_hi, idPV,
                    !first || kk > 0);
        };
        // S of half x for the key tile whose K is load kn; a segment's first one needs its Q, its last one frees it
        auto next_s = [&](int x, int kn, bool first, bool last) {
          ok = full(kn) && (!first || mbar_wait(bar(CQF + x), nseg[x] & 1, abort_flag, p.wait_cycles));
          if (!ok) return;
          nseg[x] += first;
          issue_s(x, kn % cStages);
          if (last) umma_commit(bar(CQE + x));
        };
        int n1 = 0, halves = 0;  // the segment's key tiles and halves
        auto segment = [&]() {
          const bool more = w.segment();
          n1 = more ? w.j1 - w.j0 : 0;
          halves = more ? (w.t.ntok > tph ? 2 : 1) : 0;
        };
        segment();
        for (int x = 0; x < halves && ok; ++x) next_s(x, 0, true, n1 == 1);
        if (ok && halves > 0) umma_commit(bar(CKE));
        for (int n = 0; halves > 0 && ok;) {
          // PV of key tile n and S of the one behind it, which may be the next segment's first: then a half's S
          // goes ahead of the other half's PV only if its Q is there
          const int now = halves, kv = nl + 1, kn = nl + 2;
          const bool first = n % kSum == 0, end = n + 1 == n1;  // first: O starts from zero
          if (end) segment();
          n = end ? 0 : n + 1;
          const bool last = n + 1 == n1;
          bool due = false;
          for (int x = 0; x < 2 && ok; ++x) {
            if (x < now) {
              ok = full(kv) && mbar_wait(bar(CPF + 2 * x), np[x] & 1, abort_flag, p.wait_cycles);
              if (!ok) break;
              issue_pv(x, kv % cStages, 0, first);
              ok = mbar_wait(bar(CPF + 2 * x + 1), np[x] & 1, abort_flag, p.wait_cycles);
              if (!ok) break;
              ++np[x];
              issue_pv(x, kv % cStages, 1, false);
              if (end) umma_commit(bar(COF + x));
            }
            if (x >= halves) continue;
            if (x == 0 && end && now == 2 &&
                !(mbar_try(bar(CQF), nseg[0] & 1) && mbar_try(bar(CKF + kn % cStages), (kn / cStages) & 1)))
              due = true;
            else
              next_s(x, kn, end, last);
          }
          if (ok && due) next_s(0, kn, end, last);
          if (!ok) break;
          umma_commit(bar(CKE + kv % cStages));
          if (halves > 0) umma_commit(bar(CKE + kn % cStages));
          nl += 2;
        }
        if (!ok) {
          *abort_flag = 1;
          *reinterpret_cast<volatile int *>(p.status) = kErrMma;
        }
        // wait (bounded) until every MMA this thread issued has completed
        umma_commit(bar(CDRAIN));
        volatile int never = 0;
        mbar_wait(bar(CDRAIN), 0, &never, p.drain_cycles);
      }
    } else if (warp == 10) {
      // ============================================================ keeper (whole warp)
      bool ok = true;
      int n = 0;         // V tiles
      uint32_t odd = 0;  // tiles kept in each stage, modulo 2
      for (int seg = 0; ok && w.segment(); ++seg) {
        for (int j = w.j0; ok && j < w.j1; ++j, ++n) {
          const int c0 = w.key(j) * cBN, s = (2 * n + 1) % cStages;
          if (!has_unseen<cBN>(w.g, p.sinks, c0) && !rows_differ<cBN>(w.t.pos0, w.t.ntok, p.window, p.sinks, c0)) continue;
          ok = __all_sync(0xffffffffu, mbar_wait(bar(CVX + s), (odd >> s) & 1u, abort_flag, p.wait_cycles));
          odd ^= 1u << s;
          ok = ok && keep_values<E, D, cBN>(p, smem + Lay::kv + s * Lay::tile, w.t, w.g, c0, seg, notes, abort_flag);
          if (ok && lane == 0) mbar_arrive(bar(CKF + s));
        }
      }
      if (!ok && lane == 0) {
        *abort_flag = 1;
        *reinterpret_cast<volatile int *>(p.status) = kErrProducer;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(cRegsSoftmax));
    // ============================================================ softmax (warps 0-3: half A, 4-7: half B)
    const int x = warp >> 2;
    const int r = threadIdx.x & 127;
    const int tl = x * tph + min(r / p.G, tph - 1), hg = r % p.G;  // the row's token in the tile and head in the group
    const int row = x * qrows + r;                                 // the tile's rows without the halves' gaps
    const uint32_t lane_off = uint32_t((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + x * cBN + lane_off, o_addr = tmem + 256 + x * 128 + lane_off;
    const float2 sc2 = make_float2(p.scale_log2, p.scale_log2);
    bool ok = true, first_seg = true, noted = false;
    int n = 0, nseg = 0;  // S tiles and segments of this half
    for (int seg = 0; ok && w.segment(); ++seg) {
      const Keys g = w.g;
      const int nrows = w.t.ntok * p.G;
      const bool mine = w.t.ntok > x * tph;                      // this half has rows
      const bool active = x * qrows + (warp & 3) * 32 < nrows && mine;  // this warp has
      // rows of no token take the last token's mask; nobody reads them
      const int pos = w.t.pos0 + min(tl, w.t.ntok - 1);
      float m_ref = -INFINITY, l_run = 0.0f;
      for (int j = w.j0, stop; mine && ok && j < w.j1;) {
        stop = min(w.j1, j + kSum);
        for (; j < stop; ++j, ++n) {
          if (!__all_sync(0xffffffffu, mbar_wait(bar(CSF + x), n & 1, abort_flag, p.wait_cycles))) { ok = false; break; }
          fence_after();
          const int c0 = w.key(j) * cBN;
          if (active) {
            // whole: the row sees all keys of the tile
            const int lim = pos + 1 - c0, from = p.window > 0 ? pos - p.window + 1 - c0 : 0, sink = p.sinks - c0;
            const bool edge = __any_sync(0xffffffffu, lim < cBN || (from > 0 && sink < cBN));
            float xs[cBN];
            auto mask_chunk = [&](int c) {  // 32 columns; from and sink only matter with a window
              const uint64_t m = (below(lim - 32 * c) & (p.window > 0 ? ~below(from - 32 * c) | below(sink - 32 * c) : ~0ull));
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!((uint32_t(m) >> e) & 1u)) xs[c * 32 + e] = -INFINITY;
            };
            float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            tmem_ld32(s_addr, xs);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              tmem_wait_ld();
              if (c < 3) tmem_ld32(s_addr + 32 * (c + 1), xs + 32 * (c + 1));  // lands while this chunk is looked through
              if (edge) mask_chunk(c);
#pragma unroll
              for (int e = 0; e < 32; e += 2) mx4[(e >> 1) & 3] = max3f(mx4[(e >> 1) & 3], xs[c * 32 + e], xs[c * 32 + e + 1]);
            }
            const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
            // P and O stay scaled to m_ref until a score outgrows it by 2^rescale
            float alpha = 1.0f;
            if (mx > m_ref && (m_ref == -INFINITY || (mx - m_ref) * p.scale_log2 > Num<E>::chunk_rescale)) {
              alpha = m_ref == -INFINITY ? 0.0f : fast_exp2((m_ref - mx) * p.scale_log2);
              m_ref = mx;
            }
            if (j > w.j0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
              // O holds PV(n - 1): S(n) was issued after it and is there
#pragma unroll 1
              for (int c = 0; c < D / 16; ++c) {
                float o[16];
                tmem_ld16(o_addr + c * 16, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] *= alpha;
                tmem_st16(o_addr + c * 16, o);
              }
              tmem_wait_st();
            }
            const float moff = (m_ref == -INFINITY ? 0.0f : m_ref) * p.scale_log2 - Num<E>::bias;
            const float2 off2 = make_float2(-moff, -moff);
            float2 rs2[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
            auto exp_chunk = [&](int c) {
              uint32_t pk[16];
#pragma unroll
              for (int e = 0; e < 32; e += 2) {
                const float2 a = __ffma2_rn(make_float2(xs[c * 32 + e], xs[c * 32 + e + 1]), sc2, off2);
                float2 ex;
                ex.x = fast_exp2(a.x);
                ex.y = fast_exp2(a.y);
                rs2[(e >> 1) & 1] = __fadd2_rn(rs2[(e >> 1) & 1], ex);
                pk[e >> 1] = Num<E>::pack(ex.x, ex.y);
              }
              tmem_st16u(s_addr + c * 16, pk);
            };
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              exp_chunk(c);
              if (c == 1) {  // the first 64 keys' product can start
                tmem_wait_st();
                fence_before();
                mbar_arrive(bar(CPF + 2 * x));
              }
            }
            const float2 rsum = __fadd2_rn(rs2[0], rs2[1]);
            l_run = l_run * alpha + (rsum.x + rsum.y);
            tmem_wait_st();
          } else {
            fence_before();
            mbar_arrive(bar(CPF + 2 * x));
          }
          fence_before();
          mbar_arrive(bar(CPF + 2 * x + 1));
        }
        if (ok && j < w.j1) {
          // O holds PV(n - 1) once S(n) is there, which was issued after it
          ok = __all_sync(0xffffffffu, mbar_wait(bar(CSF + x), n & 1, abort_flag, p.wait_cycles));
          if (!ok) break;
          fence_after();
          const int slot = 2 * int(blockIdx.x) + (first_seg ? 0 : 1);
          if (active && FFTS_IN_RANGE(slot, 2 * p.ctas))
            park_o<D, 2 * cBM>(p, slot, row, r < qrows && row < nrows, j - w.j0 > kSum, m_ref * p.scale_log2, o_addr);
        }
      }
      if (!ok) break;
      if (mine) {
        if (!__all_sync(0xffffffffu, mbar_wait(bar(COF + x), nseg & 1, abort_flag, p.wait_cycles))) { ok = false; break; }
        ++nseg;
        fence_after();
      }
      const int slot = 2 * int(blockIdx.x) + (first_seg ? 0 : 1);
      if (active) {
        const bool live = r < qrows && row < nrows;
        const bool whole = w.j0 == 0 && w.j1 == g.n;
        const bool sees = pos >= 0;  // a row without a key is zeros; NaN in l, or l == 0, is NaN as in the formula
        const float inv_l = 1.0f / l_run;
        uint16_t *dst = p.out + int64_t(w.t.tok0 + tl) * p.os_t + int64_t(w.h * p.G + hg) * p.os_h;
        float4 *pd = reinterpret_cast<float4 *>(p.part) + int64_t(slot) * (2 * cBM * D / 4) + row;
        float2 *pml = p.part_ml + int64_t(slot) * (2 * cBM) + row;
        const bool parked = w.j1 - w.j0 > kSum && live && FFTS_IN_RANGE(slot, 2 * p.ctas);
        const float f = parked ? weight(pml->x, m_ref * p.scale_log2) : 0.0f;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          float o[32];
          __syncwarp();
          tmem_ld32(o_addr + c * 32, o);
          tmem_wait_ld();
          if (parked) unpark<(2 * cBM)>(o, pd, c, f);
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
          if (live && !whole && FFTS_IN_RANGE(slot, 2 * p.ctas)) park<(2 * cBM)>(o, pd, c);
        }
        if (live && !whole && FFTS_IN_RANGE(slot, 2 * p.ctas)) *pml = make_float2(m_ref * p.scale_log2, l_run);
        if (live && *notes.segment == seg + 1) {
          if (whole && FFTS_IN_RANGE(w.t.tok0 + tl, p.T)) put_back<E, D, 2 * cBM>(p, row, reinterpret_cast<E *>(dst));
          if (!whole && FFTS_IN_RANGE(slot, 2 * p.ctas)) put_back<E, D, 2 * cBM>(p, row, reinterpret_cast<float *>(pd));
        }
      }
      __syncwarp();
      if (lane == 0) notes.done[warp] = seg + 1;
      // the share that opens a (q tile, head) and does not end it leaves a note for the join
      if (w.opens && w.j1 - w.j0 < g.n && threadIdx.x == 0 && FFTS_IN_RANGE(blockIdx.x, p.ctas)) {
        Cut cut;
        cut.tok0 = w.t.tok0;
        cut.pos0 = w.t.pos0;
        cut.nrows = nrows;
        cut.head0 = w.h * p.G;
        cut.s1 = w.last_share(u0, per);
        cut.first_slot = slot;
        p.cuts[blockIdx.x] = cut;
        noted = true;
      }
      first_seg = false;
    }
    if (threadIdx.x == 0 && !noted) p.cuts[blockIdx.x].nrows = 0;
    if (!ok) {
      *abort_flag = 1;
      *reinterpret_cast<volatile int *>(p.status) = kErrSoftmax;
    }
  }

  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cTmemCols));
}

template <typename E, int D>
static int launch(const Params &p, const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv,
                  cudaStream_t stream) {
  const int rc = ensure_func_smem(reinterpret_cast<const void *>(&chunk_kernel<E, D>), ChunkLayout<D>::bytes,
                                  int(cudaSharedmemCarveoutMaxShared));
  if (rc) return rc;
  if (!p.own_schedule) {
    schedule_kernel<cBN><<<1, kSchedThreads, 0, stream>>>(p);
    FFTS_CUDA(cudaGetLastError());
  }
  return launch_early(chunk_kernel<E, D>, dim3(unsigned(p.ctas)), cThreads, ChunkLayout<D>::bytes, stream, mq, mk, mv, p);
}

int launch_chunk(const Params &p, bool half, int D, const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv,
                 cudaStream_t stream) {
  if (half) return D == 128 ? launch<__half, 128>(p, mq, mk, mv, stream) : launch<__half, 64>(p, mq, mk, mv, stream);
  return D == 128 ? launch<__nv_bfloat16, 128>(p, mq, mk, mv, stream)
                  : launch<__nv_bfloat16, 64>(p, mq, mk, mv, stream);
}

}  // namespace paged
}  // namespace ffts
