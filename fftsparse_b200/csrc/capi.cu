// capi.cu -- the extern "C" boundary of libfftsparse_b200.so.
//
// Each export validates its arguments, enqueues kernels on the caller's stream
// and returns FFTS_OK or a negative FFTS_E* code; the message of the last
// failure on the calling thread is kept for ffts_last_error_string().

#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <map>
#include <mutex>
#include <string>
#include <vector>

#include <nvtx3/nvToolsExt.h>

#include "ffts_common.cuh"

namespace ffts {

static thread_local std::string g_last_error;

#ifdef FFTS_BOUNDS_CHECK
namespace oob {
struct Entry {
  const char *file;
  Reader read;
};
static std::vector<Entry> &registry() {
  static std::vector<Entry> r;  // filled by static initialisers, read after load
  return r;
}
void register_reader(const char *file, Reader fn) { registry().push_back({file, fn}); }
}  // namespace oob
#endif

void set_error(int code, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_last_error = std::string(buf) + " (code " + std::to_string(code) + ")";
}

int cuda_status(cudaError_t e, const char *what) {
  set_error(FFTS_E_CUDA, "%s failed: %s", what, cudaGetErrorString(e));
  return FFTS_E_CUDA;
}

int ensure_func_smem(const void *func, int bytes, int carveout) {
  static std::mutex mu;
  static std::map<std::pair<const void *, int>, int> done;  // (function, device) -> limit set
  int dev = 0;
  FFTS_CUDA(cudaGetDevice(&dev));
  std::lock_guard<std::mutex> lock(mu);
  auto it = done.find({func, dev});
  if (it != done.end() && it->second >= bytes) return FFTS_OK;
  FFTS_CUDA(cudaFuncSetAttribute(func, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (carveout >= 0) FFTS_CUDA(cudaFuncSetAttribute(func, cudaFuncAttributePreferredSharedMemoryCarveout, carveout));
  done[{func, dev}] = bytes;
  return FFTS_OK;
}

namespace {
struct DeviceProps {
  int sms = 0;
  int clock_khz = 0;
};

int device_props(DeviceProps *out) {
  static std::mutex mu;
  static std::map<int, DeviceProps> cache;
  int dev = 0;
  FFTS_CUDA(cudaGetDevice(&dev));
  std::lock_guard<std::mutex> lock(mu);
  auto it = cache.find(dev);
  if (it == cache.end()) {
    DeviceProps p;
    FFTS_CUDA(cudaDeviceGetAttribute(&p.sms, cudaDevAttrMultiProcessorCount, dev));
    FFTS_CUDA(cudaDeviceGetAttribute(&p.clock_khz, cudaDevAttrClockRate, dev));
    if (p.sms <= 0) p.sms = 1;
    if (p.clock_khz <= 0) p.clock_khz = 2000000;  // an unreported clock: assume 2 GHz
    it = cache.emplace(dev, p).first;
  }
  *out = it->second;
  return FFTS_OK;
}
}  // namespace

int device_sm_count(int *out) {
  DeviceProps p;
  const int rc = device_props(&p);
  if (rc == FFTS_OK) *out = p.sms;
  return rc;
}

int device_wait_cycles(double seconds, long long *out) {
  DeviceProps p;
  const int rc = device_props(&p);
  if (rc == FFTS_OK) *out = static_cast<long long>(seconds * 1e3 * double(p.clock_khz));
  return rc;
}

int launch_pool(const void *x, int dtype, int64_t B, int64_t H, int64_t L, int64_t D, int64_t sb,
                int64_t sh, int64_t sl, int bs, void *out, cudaStream_t stream);
int launch_rope_pool(const void *q_src, int64_t q_ld, const void *k_src, int64_t k_ld, const void *v_src,
                     int64_t v_ld, int64_t L, int64_t Hq, int64_t Hkv, int64_t D, const void *cos, const void *sin,
                     int64_t cs_ld, int bs, void *q_out, void *k_out, void *v_out, void *q_pooled, void *k_pooled,
                     cudaStream_t stream);
int qkv_rope_pool(const void *x, int64_t B, int64_t L, int64_t K, int64_t x_ld, int64_t x_sb, const void *w,
                  int64_t w_ld, const void *bias, int64_t Hq, int64_t Hkv, int64_t D, const void *cos,
                  const void *sin, int64_t cs_ld, int bs, void *q_out, void *k_out, void *v_out, void *q_pooled,
                  void *k_pooled, void *raw, int64_t raw_ld, void *workspace, int64_t ws_bytes, int32_t *status,
                  cudaStream_t stream);
int64_t qkv_workspace_bytes(int64_t L);
int64_t decode_workspace_bytes(int64_t B, int64_t H, int64_t Hkv, int64_t splits);
int decode_attn(const void *q, int64_t qs_b, int64_t qs_h, const void *k, const int64_t *ks, const void *v,
                const int64_t *vs, int64_t B, int64_t H, int64_t Hkv, int64_t Lk, int64_t D, int64_t splits,
                void *ws, int64_t ws_bytes, void *out, int64_t os_b, int64_t os_h, const void *bias,
                int bias_dtype, int64_t bias_sb, cudaStream_t stream);
int page_plan(const ffts_page_plan_args &a, cudaStream_t stream);
int rope_append(const ffts_rope_append_args &a, cudaStream_t stream);
int64_t paged_workspace_bytes(int64_t T, int64_t R, int64_t H, int64_t Hkv, int64_t D);
int paged_attn(const ffts_paged_attn_args &a, cudaStream_t stream);
int64_t mask_workspace_bytes(int64_t B, int64_t H, int64_t N, int64_t D);
int block_mask(const void *qb, const void *kb, int dtype, int64_t B, int64_t H, int64_t Hkv, int64_t D,
               const ffts_mask_params *params, uint32_t *bits, int32_t *row_count, float *corr,
               float *csum, uint8_t *is_stripe, float *svar, void *workspace, int64_t ws_bytes,
               cudaStream_t stream);
int unpack_mask(const uint32_t *bits, int64_t B, int64_t H, int64_t N, uint8_t *out, cudaStream_t stream);
int mask_row_ptr(const int32_t *row_count, int64_t rows, int64_t *row_ptr, cudaStream_t stream);
int mask_col_idx(const uint32_t *bits, int64_t rows, int64_t N, const int64_t *row_ptr, int32_t *col_idx,
                 int64_t capacity, int32_t *status, cudaStream_t stream);
int ensure_tables();
int sparse_attn_fwd(const void *q, const void *k, const void *v, int64_t B, int64_t H, int64_t Hkv,
                    int64_t L, int64_t D, const int64_t *qs, const int64_t *ks, const int64_t *vs,
                    const uint32_t *bits, int bs, int causal, void *out, const int64_t *os,
                    int64_t row_lo, int64_t row_hi, void *const *peer_out, int n_peers, int32_t *status,
                    cudaStream_t stream);

// One NVTX range per compute entry point (visible in nsys / ncu range filters;
// a call into the NVTX stubs when no tool is attached).
namespace {
struct NvtxRange {
  explicit NvtxRange(const char *name) { nvtxRangePushA(name); }
  ~NvtxRange() { nvtxRangePop(); }
};
}  // namespace
#define FFTS_ENTRY(name)        \
  g_last_error.clear();         \
  NvtxRange ffts_nvtx_range_(name)

static int check_device() {
  int dev = 0;
  FFTS_CUDA(cudaGetDevice(&dev));
  int major = 0;
  FFTS_CUDA(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev));
  if (major != 10) {
    set_error(FFTS_E_DEVICE, "device %d has compute capability %d.x; this library targets sm_100a", dev, major);
    return FFTS_E_DEVICE;
  }
  return FFTS_OK;
}

}  // namespace ffts

using namespace ffts;

extern "C" {

int32_t ffts_version(void) { return 100; }

const char *ffts_last_error_string(void) { return g_last_error.c_str(); }

int32_t ffts_init(int32_t device) {
  g_last_error.clear();
  int prev = 0;
  FFTS_CUDA(cudaGetDevice(&prev));
  if (device != prev) FFTS_CUDA(cudaSetDevice(device));
  int rc = check_device();
  if (rc == FFTS_OK) rc = ensure_tables();
  if (device != prev) cudaSetDevice(prev);
  return rc;
}

int32_t ffts_pool(const void *x, int32_t dtype, int64_t B, int64_t H, int64_t L, int64_t D,
                  int64_t stride_b, int64_t stride_h, int64_t stride_l, int32_t block_size, void *out,
                  void *stream) {
  FFTS_ENTRY("ffts_pool");
  FFTS_REQUIRE(x != nullptr && out != nullptr, "ffts_pool: NULL pointer");
  int rc = check_device();
  if (rc) return rc;
  return launch_pool(x, dtype, B, H, L, D, stride_b, stride_h, stride_l, block_size, out,
                     static_cast<cudaStream_t>(stream));
}

int32_t ffts_rope_pool(const void *q_src, int64_t q_ld, const void *k_src, int64_t k_ld, const void *v_src,
                       int64_t v_ld, int64_t L, int64_t Hq, int64_t Hkv, int64_t D, const void *cos,
                       const void *sin, int64_t cs_ld, int32_t block_size, void *q_out, void *k_out, void *v_out,
                       void *q_pooled, void *k_pooled, void *stream) {
  FFTS_ENTRY("ffts_rope_pool");
  int rc = check_device();
  if (rc) return rc;
  return launch_rope_pool(q_src, q_ld, k_src, k_ld, v_src, v_ld, L, Hq, Hkv, D, cos, sin, cs_ld, block_size,
                          q_out, k_out, v_out, q_pooled, k_pooled, static_cast<cudaStream_t>(stream));
}

int32_t ffts_qkv_rope_pool(const void *x, int64_t B, int64_t L, int64_t hidden, int64_t x_stride_l,
                           int64_t x_stride_b, const void *w, int64_t w_ld, const void *bias, int64_t Hq,
                           int64_t Hkv, int64_t D, const void *cos, const void *sin, int64_t cs_ld,
                           int32_t block_size, void *q_out, void *k_out, void *v_out, void *q_pooled,
                           void *k_pooled, void *proj_out, int64_t proj_ld, void *workspace,
                           int64_t workspace_bytes, int32_t *status, void *stream) {
  FFTS_ENTRY("ffts_qkv_rope_pool");
  int rc = check_device();
  if (rc) return rc;
  return qkv_rope_pool(x, B, L, hidden, x_stride_l, x_stride_b, w, w_ld, bias, Hq, Hkv, D, cos, sin, cs_ld,
                       block_size, q_out, k_out, v_out, q_pooled, k_pooled, proj_out, proj_ld, workspace,
                       workspace_bytes, status, static_cast<cudaStream_t>(stream));
}

int64_t ffts_qkv_workspace_bytes(int64_t L) { return qkv_workspace_bytes(L); }

int64_t ffts_decode_workspace_bytes(int64_t B, int64_t H, int64_t Hkv, int64_t splits) {
  return decode_workspace_bytes(B, H, Hkv, splits);
}

int32_t ffts_decode_attn(const void *q, int64_t q_stride_b, int64_t q_stride_h, const void *k_cache,
                         const int64_t *k_strides, const void *v_cache, const int64_t *v_strides, int64_t B,
                         int64_t H, int64_t Hkv, int64_t Lk, int64_t D, int64_t splits, void *workspace,
                         int64_t workspace_bytes, void *out, int64_t out_stride_b, int64_t out_stride_h,
                         const void *mask, int32_t mask_dtype, int64_t mask_stride_b, void *stream) {
  FFTS_ENTRY("ffts_decode_attn");
  int rc = check_device();
  if (rc) return rc;
  return decode_attn(q, q_stride_b, q_stride_h, k_cache, k_strides, v_cache, v_strides, B, H, Hkv, Lk, D, splits,
                     workspace, workspace_bytes, out, out_stride_b, out_stride_h, mask, mask_dtype, mask_stride_b,
                     static_cast<cudaStream_t>(stream));
}

int32_t ffts_page_plan(const ffts_page_plan_args *args, void *stream) {
  FFTS_ENTRY("ffts_page_plan");
  FFTS_REQUIRE(args && args->struct_bytes == int64_t(sizeof(*args)), "page_plan: NULL or foreign argument block");
  int rc = check_device();
  if (rc) return rc;
  return page_plan(*args, static_cast<cudaStream_t>(stream));
}

int32_t ffts_rope_append(const ffts_rope_append_args *args, void *stream) {
  FFTS_ENTRY("ffts_rope_append");
  FFTS_REQUIRE(args && args->struct_bytes == int64_t(sizeof(*args)), "rope_append: NULL or foreign argument block");
  int rc = check_device();
  if (rc) return rc;
  return rope_append(*args, static_cast<cudaStream_t>(stream));
}

int64_t ffts_paged_workspace_bytes(int64_t T, int64_t R, int64_t H, int64_t Hkv, int64_t D) {
  return paged_workspace_bytes(T, R, H, Hkv, D);
}

int32_t ffts_paged_attn(const ffts_paged_attn_args *args, void *stream) {
  FFTS_ENTRY("ffts_paged_attn");
  FFTS_REQUIRE(args && args->struct_bytes == int64_t(sizeof(*args)), "paged_attn: NULL or foreign argument block");
  int rc = check_device();
  if (rc) return rc;
  return paged_attn(*args, static_cast<cudaStream_t>(stream));
}

int64_t ffts_mask_workspace_bytes(int64_t B, int64_t H, int64_t N, int64_t D) {
  if (B <= 0 || H <= 0 || N <= 0 || D <= 0) return 0;
  return mask_workspace_bytes(B, H, N, D);
}

int32_t ffts_block_mask(const void *qb, const void *kb, int32_t dtype, int64_t B, int64_t H, int64_t Hkv,
                        int64_t D, const ffts_mask_params *params, uint32_t *mask_bits, int32_t *row_count,
                        float *corr, float *corr_sum, uint8_t *is_stripe, float *stripe_var, void *workspace,
                        int64_t workspace_bytes, void *stream) {
  FFTS_ENTRY("ffts_block_mask");
  int rc = check_device();
  if (rc) return rc;
  return block_mask(qb, kb, dtype, B, H, Hkv, D, params, mask_bits, row_count, corr, corr_sum, is_stripe,
                    stripe_var, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

int32_t ffts_unpack_mask(const uint32_t *mask_bits, int64_t B, int64_t H, int64_t N, uint8_t *out,
                         void *stream) {
  FFTS_ENTRY("ffts_unpack_mask");
  return unpack_mask(mask_bits, B, H, N, out, static_cast<cudaStream_t>(stream));
}

int32_t ffts_mask_row_ptr(const int32_t *row_count, int64_t rows, int64_t *row_ptr, void *stream) {
  FFTS_ENTRY("ffts_mask_row_ptr");
  int rc = check_device();
  if (rc) return rc;
  return mask_row_ptr(row_count, rows, row_ptr, static_cast<cudaStream_t>(stream));
}

int32_t ffts_mask_col_idx(const uint32_t *mask_bits, int64_t rows, int64_t N, const int64_t *row_ptr,
                          int32_t *col_idx, int64_t capacity, int32_t *status, void *stream) {
  FFTS_ENTRY("ffts_mask_col_idx");
  int rc = check_device();
  if (rc) return rc;
  return mask_col_idx(mask_bits, rows, N, row_ptr, col_idx, capacity, status, static_cast<cudaStream_t>(stream));
}

int32_t ffts_sparse_attn_fwd(const void *q, const void *k, const void *v, int64_t B, int64_t H, int64_t Hkv,
                             int64_t L, int64_t D, const int64_t *q_strides, const int64_t *k_strides,
                             const int64_t *v_strides, const uint32_t *mask_bits, int32_t block_size,
                             int32_t causal, void *out, const int64_t *out_strides, int32_t *status,
                             void *stream) {
  FFTS_ENTRY("ffts_sparse_attn_fwd");
  int rc = check_device();
  if (rc) return rc;
  return sparse_attn_fwd(q, k, v, B, H, Hkv, L, D, q_strides, k_strides, v_strides, mask_bits, block_size,
                         causal, out, out_strides, 0, L, nullptr, 0, status, static_cast<cudaStream_t>(stream));
}

int32_t ffts_sparse_attn_fwd_rows(const void *q, const void *k, const void *v, int64_t B, int64_t H, int64_t Hkv,
                                  int64_t L, int64_t D, const int64_t *q_strides, const int64_t *k_strides,
                                  const int64_t *v_strides, const uint32_t *mask_bits, int32_t block_size,
                                  int32_t causal, int64_t row_lo, int64_t row_hi, void *out,
                                  const int64_t *out_strides, int32_t *status, void *stream) {
  FFTS_ENTRY("ffts_sparse_attn_fwd_rows");
  int rc = check_device();
  if (rc) return rc;
  return sparse_attn_fwd(q, k, v, B, H, Hkv, L, D, q_strides, k_strides, v_strides, mask_bits, block_size,
                         causal, out, out_strides, row_lo, row_hi, nullptr, 0, status,
                         static_cast<cudaStream_t>(stream));
}

int32_t ffts_sparse_attn_fwd_push(const void *q, const void *k, const void *v, int64_t B, int64_t H, int64_t Hkv,
                                  int64_t L, int64_t D, const int64_t *q_strides, const int64_t *k_strides,
                                  const int64_t *v_strides, const uint32_t *mask_bits, int32_t block_size,
                                  int32_t causal, int64_t row_lo, int64_t row_hi, void *out,
                                  const int64_t *out_strides, void *const *peer_out, int32_t n_peers,
                                  int32_t *status, void *stream) {
  FFTS_ENTRY("ffts_sparse_attn_fwd_push");
  int rc = check_device();
  if (rc) return rc;
  return sparse_attn_fwd(q, k, v, B, H, Hkv, L, D, q_strides, k_strides, v_strides, mask_bits, block_size,
                         causal, out, out_strides, row_lo, row_hi, peer_out, n_peers, status,
                         static_cast<cudaStream_t>(stream));
}

int32_t ffts_bounds_check_enabled(void) {
#ifdef FFTS_BOUNDS_CHECK
  return 1;
#else
  return 0;
#endif
}

int32_t ffts_bounds_report(ffts_bounds_record *records, int32_t max_records, int32_t clear) {
  g_last_error.clear();
  FFTS_REQUIRE(max_records >= 0 && (records != nullptr || max_records == 0),
               "ffts_bounds_report: NULL records with max_records > 0");
#ifdef FFTS_BOUNDS_CHECK
  int found = 0;
  for (const oob::Entry &e : oob::registry()) {
    unsigned long long first = 0;
    unsigned int count = 0;
    const int rc = e.read(clear, &first, &count);
    if (rc) return cuda_status(cudaError_t(rc), "ffts_bounds_report: reading the records");
    if (count == 0 && first == 0) continue;
    if (found < max_records) {
      ffts_bounds_record &r = records[found];
      const char *base = strrchr(e.file, '/');
      base = base ? base + 1 : e.file;
      snprintf(r.file, sizeof(r.file), "%s", base);
      r.line = int32_t((first >> 32) & 0x7fffffff);
      r.count = count;
      r.block = int64_t(first & 0xffffffffull);
    }
    ++found;
  }
  return found;
#else
  (void)records;
  (void)clear;
  return 0;
#endif
}

}  // extern "C"
