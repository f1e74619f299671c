// rope_append.cu -- rotary positions of new tokens' q and k, and the append of k and v to a paged cache, one pass.
//
// Pair i of a head, i < rd / 2, is (x[i], x[i + rd/2]) in the half layout and (x[2i], x[2i + 1]) in the
// interleaved one; channels from rd on are copied.  With angle a = pos * inv_freq[i]:
//   (x, y) -> (x c - y s, y c + x s),  c = amplitude * cos a,  s = amplitude * sin a.
// The angle is formed in 64 bits and reduced to a fraction of a turn there: at position 2^20 an fp32 angle
// is off by up to 2^-5 rad, the 64-bit turn count by less than 1e-9.  cos and sin of the remaining fraction, the
// products and sums are fp32; the result is rounded once to the tensors' type.
//
// HBM bound: every element is read once and written once (q to q_out, k and v to their slot's page
// row).  A thread keeps one unit of a head -- 16 bytes, or the two 16-byte halves of 8 pairs in the half
// layout -- and walks the CTA's tokens four at a time, so 4 to 8 loads are in flight per thread.  The
// angles of a token are computed once per CTA into shared memory and serve all of its heads.  The sources are read
// as streams (17.8 -> 16.5 us at 5001 tokens): what the attention reads next are the outputs.

#include <cuda_fp16.h>

#include "ffts_common.cuh"

namespace ffts {
namespace ropeapp {

// 256: 141.8 us where 128 take 135.8 (32768 tokens, 32 / 8 heads), 19.5 and 17.8 (5001 tokens, 28 / 4)
constexpr int kThreads = 128;
constexpr int kMaxTokens = 8;   // tokens per CTA (4 and 16: 160 and 135 us, 22.0 and 19.1)
constexpr int kMaxPairs = 64;   // rd / 2, D <= 128

struct Params {
  const uint16_t *q, *k, *v;      // [T, heads, D] with strides (t, h), 16-bit elements; q may be null
  int64_t qs_t, qs_h, ks_t, ks_h, vs_t, vs_h;
  uint16_t *q_out;                // [T, H, D] with strides
  int64_t os_t, os_h;
  uint16_t *kp, *vp;              // [P, Hkv, ps, D] with strides (page, head, row)
  int64_t kp_p, kp_h, kp_r, vp_p, vp_h, vp_r;
  const int32_t *positions, *slots;
  const float *inv_freq;
  float amplitude;
  int T, H, Hkv, D, rd, interleaved, tokens;  // tokens: per CTA
  int64_t n_slots;                // P * ps
  int ps_shift;
};

template <typename E>
__device__ __forceinline__ float2 unpack(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
template <typename E>
__device__ __forceinline__ uint32_t pack(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&r);
}
template <>
__device__ __forceinline__ uint32_t pack<__half>(float a, float b) {
  const __half2 r = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&r);
}

// 8 pairs of the half layout: a holds the first elements, b the second ones
template <typename E>
__device__ __forceinline__ void rotate_half8(uint4 &a, uint4 &b, const float2 *cs) {
  uint32_t *aw = reinterpret_cast<uint32_t *>(&a), *bw = reinterpret_cast<uint32_t *>(&b);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = unpack<E>(aw[i]), y = unpack<E>(bw[i]);
    const float2 c0 = cs[2 * i], c1 = cs[2 * i + 1];
    aw[i] = pack<E>(x.x * c0.x - y.x * c0.y, x.y * c1.x - y.y * c1.y);
    bw[i] = pack<E>(y.x * c0.x + x.x * c0.y, y.y * c1.x + x.y * c1.y);
  }
}

// 4 pairs of the interleaved layout
template <typename E>
__device__ __forceinline__ void rotate_pairs4(uint4 &a, const float2 *cs) {
  uint32_t *aw = reinterpret_cast<uint32_t *>(&a);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = unpack<E>(aw[i]);
    aw[i] = pack<E>(x.x * cs[i].x - x.y * cs[i].y, x.y * cs[i].x + x.x * cs[i].y);
  }
}

template <typename E>
__global__ void __launch_bounds__(kThreads) rope_append_kernel(const __grid_constant__ Params p) {
  __shared__ __align__(16) float2 cs[kMaxTokens][kMaxPairs];
  __shared__ int s_slot[kMaxTokens];
  const int tid = threadIdx.x;
  const int t0 = blockIdx.x * p.tokens;
  const int nt = min(p.tokens, p.T - t0);
  const int half = p.rd >> 1;
  for (int i = tid; i < nt * half; i += kThreads) {
    const int t = i / half, f = i - t * half;
    const double turns = double(p.positions[t0 + t]) * double(p.inv_freq[f]) * 0.15915494309189533577;  // 1 / (2 pi)
    float s, c;
    sincospif(2.0f * float(turns - rint(turns)), &s, &c);
    cs[t][f] = make_float2(c * p.amplitude, s * p.amplitude);
  }
  if (tid < nt) s_slot[tid] = p.slots[t0 + tid];
  __syncthreads();

  // The thread's unit: tensor, head and channel.  A q or k head has rot rotated units, then its copied
  // vectors; a v head has D / 8 copied vectors.
  const int rot = p.interleaved ? p.rd >> 3 : p.rd >> 4;
  const int per_head = rot + ((p.D - p.rd) >> 3);
  const int vecs = p.D >> 3;
  const int hq = p.q ? p.H : 0;
  int u = blockIdx.y * kThreads + tid;
  const uint16_t *src;
  int64_t ss;
  uint16_t *dst;
  int64_t ds_t = 0, d_p = 0, d_r = 0;
  bool paged = true;
  int kind;  // 0 copy, 1 half layout, 2 interleaved
  int ch, pair = 0;
  if (u < (hq + p.Hkv) * per_head) {
    const int h = u / per_head, i = u - h * per_head;
    kind = i < rot ? (p.interleaved ? 2 : 1) : 0;
    ch = i < rot ? i * 8 : p.rd + (i - rot) * 8;
    pair = p.interleaved ? i * 4 : i * 8;
    if (h < hq) {
      src = p.q + h * p.qs_h + ch;
      ss = p.qs_t;
      dst = p.q_out + h * p.os_h + ch;
      ds_t = p.os_t;
      paged = false;
    } else {
      src = p.k + (h - hq) * p.ks_h + ch;
      ss = p.ks_t;
      dst = p.kp + (h - hq) * p.kp_h + ch;
      d_p = p.kp_p;
      d_r = p.kp_r;
    }
  } else {
    u -= (hq + p.Hkv) * per_head;
    const int h = u / vecs;
    if (h >= p.Hkv) return;
    kind = 0;
    ch = (u - h * vecs) * 8;
    src = p.v + h * p.vs_h + ch;
    ss = p.vs_t;
    dst = p.vp + h * p.vp_h + ch;
    d_p = p.vp_p;
    d_r = p.vp_r;
  }
  for (int t = 0; t < nt; t += 4) {
    uint4 a[4], b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (t + j < nt) {
        const uint16_t *s = src + int64_t(t0 + t + j) * ss;
        a[j] = __ldcs(reinterpret_cast<const uint4 *>(s));
        if (kind == 1) b[j] = __ldcs(reinterpret_cast<const uint4 *>(s + half));
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (t + j >= nt) break;
      uint16_t *d = dst;
      if (paged) {
        const int64_t slot = s_slot[t + j];
        if (slot < 0 || slot >= p.n_slots) continue;  // a token without a place in the cache
        d += (slot >> p.ps_shift) * d_p + (slot & ((1 << p.ps_shift) - 1)) * d_r;
      } else {
        d += int64_t(t0 + t + j) * ds_t;
      }
      if (kind == 1) {
        rotate_half8<E>(a[j], b[j], &cs[t + j][FFTS_INDEX(pair, kMaxPairs)]);
        *reinterpret_cast<uint4 *>(d + half) = b[j];
      } else if (kind == 2) {
        rotate_pairs4<E>(a[j], &cs[t + j][FFTS_INDEX(pair, kMaxPairs)]);
      }
      *reinterpret_cast<uint4 *>(d) = a[j];
    }
  }
}

}  // namespace ropeapp

int rope_append(const ffts_rope_append_args &a, cudaStream_t stream) {
  using namespace ropeapp;
  const int64_t T = a.T, H = a.H, Hkv = a.Hkv, D = a.D;
  FFTS_REQUIRE(T >= 0 && Hkv >= 1 && a.n_pages >= 0 && (a.q == nullptr || H >= 1), "rope_append: bad shape");
  FFTS_REQUIRE(a.dtype == FFTS_DTYPE_BF16 || a.dtype == FFTS_DTYPE_F16, "rope_append: dtype must be bf16 or fp16");
  FFTS_REQUIRE(D == 64 || D == 128, "rope_append: head_dim must be 64 or 128 (got %lld)", (long long)D);
  FFTS_REQUIRE(a.rotary_dim >= 0 && a.rotary_dim <= D && a.rotary_dim % 16 == 0,
               "rope_append: the rotated part must be a multiple of 16 channels up to head_dim (got %lld)",
               (long long)a.rotary_dim);
  FFTS_REQUIRE(a.page_size >= 1 && a.page_size <= 4096 && (a.page_size & (a.page_size - 1)) == 0,
               "rope_append: page_size must be a power of two up to 4096 (got %lld)", (long long)a.page_size);
  FFTS_REQUIRE(T <= (int64_t(1) << 30) && H <= 65536 && Hkv <= 65536 && a.n_pages < (int64_t(1) << 31) / a.page_size,
               "rope_append: shape too large (the pool holds less than 2^31 tokens)");
  if (T == 0) return FFTS_OK;
  FFTS_REQUIRE(a.k && a.v && a.positions && a.slots && (a.n_pages == 0 || (a.k_pages && a.v_pages)) &&
                   (a.q == nullptr || a.q_out) && (a.rotary_dim == 0 || a.inv_freq),
               "rope_append: NULL argument");
  for (const void *x : {a.q, a.k, a.v, static_cast<const void *>(a.q_out), static_cast<const void *>(a.k_pages),
                        static_cast<const void *>(a.v_pages)})
    FFTS_REQUIRE((reinterpret_cast<uintptr_t>(x) & 15) == 0, "rope_append: tensors must be 16-byte aligned");
  for (const int64_t *st : {a.q ? a.q_strides : a.k_strides, a.k_strides, a.v_strides, a.q ? a.out_strides : a.k_strides})
    FFTS_REQUIRE(st[0] % 8 == 0 && st[1] % 8 == 0, "rope_append: strides must be multiples of 8 elements (16 bytes)");
  for (const int64_t *st : {a.kp_strides, a.vp_strides})
    FFTS_REQUIRE(st[0] % 8 == 0 && st[1] % 8 == 0 && st[2] % 8 == 0,
                 "rope_append: page strides must be multiples of 8 elements (16 bytes)");
  const int64_t out_sizes[2] = {T, H}, pool_sizes[3] = {a.n_pages, Hkv, a.page_size};
  FFTS_REQUIRE(!a.q || rows_apart(out_sizes, a.out_strides, 2, D), "rope_append: rows of the rotated q overlap");
  FFTS_REQUIRE(rows_apart(pool_sizes, a.kp_strides, 3, D) && rows_apart(pool_sizes, a.vp_strides, 3, D),
               "rope_append: rows of the pages overlap");
  Params p{};
  p.q = static_cast<const uint16_t *>(a.q);
  p.k = static_cast<const uint16_t *>(a.k);
  p.v = static_cast<const uint16_t *>(a.v);
  p.qs_t = a.q_strides[0]; p.qs_h = a.q_strides[1];
  p.ks_t = a.k_strides[0]; p.ks_h = a.k_strides[1];
  p.vs_t = a.v_strides[0]; p.vs_h = a.v_strides[1];
  p.q_out = static_cast<uint16_t *>(a.q_out);
  p.os_t = a.out_strides[0]; p.os_h = a.out_strides[1];
  p.kp = static_cast<uint16_t *>(a.k_pages);
  p.vp = static_cast<uint16_t *>(a.v_pages);
  p.kp_p = a.kp_strides[0]; p.kp_h = a.kp_strides[1]; p.kp_r = a.kp_strides[2];
  p.vp_p = a.vp_strides[0]; p.vp_h = a.vp_strides[1]; p.vp_r = a.vp_strides[2];
  p.positions = a.positions;
  p.slots = a.slots;
  p.inv_freq = a.inv_freq;
  p.amplitude = a.amplitude;
  p.T = int(T); p.H = int(H); p.Hkv = int(Hkv); p.D = int(D); p.rd = int(a.rotary_dim);
  p.interleaved = a.interleaved ? 1 : 0;
  p.n_slots = a.n_pages * a.page_size;
  p.ps_shift = ilog2_ceil(a.page_size);
  int sms = 0;
  const int rc = device_sm_count(&sms);
  if (rc) return rc;
  const int64_t rot = a.interleaved ? a.rotary_dim / 8 : a.rotary_dim / 16;
  const int64_t units = ((a.q ? H : 0) + Hkv) * (rot + (D - a.rotary_dim) / 8) + Hkv * (D / 8);
  const int64_t chunks = ceil_div(units, kThreads);
  // tokens per CTA: as many as keep two CTAs per SM
  p.tokens = 1;
  while (p.tokens < kMaxTokens && ceil_div(T, 2 * p.tokens) * chunks >= 2 * sms) p.tokens *= 2;
  FFTS_REQUIRE(chunks <= 65535, "rope_append: too many heads");
  const dim3 grid(unsigned(ceil_div(T, p.tokens)), unsigned(chunks));
  if (a.dtype == FFTS_DTYPE_BF16)
    rope_append_kernel<__nv_bfloat16><<<grid, kThreads, 0, stream>>>(p);
  else
    rope_append_kernel<__half><<<grid, kThreads, 0, stream>>>(p);
  FFTS_CUDA(cudaGetLastError());
  return FFTS_OK;
}

}  // namespace ffts
