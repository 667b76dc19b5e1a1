// C-ABI of the 8-bit floating-point operators (include/krasis_b200.h).
#include <algorithm>
#include <cstdarg>
#include <cstdio>

#include "../../include/krasis_b200.h"
#include "fp8.cuh"

using namespace kb2;

extern "C" int kb2_set_error_(int code, const char* msg);

static int failf(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return kb2_set_error_(code, buf);
}
#define CUDA_TRY(expr)                                                                          \
  do {                                                                                          \
    cudaError_t _e = (expr);                                                                    \
    if (_e != cudaSuccess) return failf(KB2_ERR_CUDA, "%s: %s", #expr, cudaGetErrorString(_e)); \
  } while (0)

static bool off16(const void* p) { return ((uintptr_t)p & 15) != 0; }
static size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }
// rows of scales lie on 16 bytes
static long long scale_ld(long long rows) { return (rows + 3) & ~3ll; }

static int check_sizes(const char* what, long long M, long long N, long long K) {
  if (M < 0 || N <= 0 || K <= 0 || K % 16) return failf(KB2_ERR_VALUE, "%s: need M >= 0, N > 0, K %% 16 == 0 (M=%lld N=%lld K=%lld)", what, M, N, K);
  if (M > INT32_MAX / 2 || N > 65535ll * kFp8Block || K > 65535ll * kFp8Block) return failf(KB2_ERR_VALUE, "%s: M=%lld N=%lld K=%lld is too large", what, M, N, K);
  return KB2_OK;
}

// The parts of a workspace.
struct Carve {
  uint8_t* at;
  size_t used = 0;
  explicit Carve(void* p) : at((uint8_t*)p) {}
  template <typename T> T* take(size_t n) {
    T* r = reinterpret_cast<T*>(at + used);
    used += up16(n * sizeof(T));
    return r;
  }
};

extern "C" {

KB2_API int kb2_fp8_quantize_rows(const void* x_dev, int32_t x_f32, int64_t ldx, int32_t M, int32_t K, void* codes_dev, float* scales_dev, int64_t ld_scales,
                                  int32_t device, void* stream) {
  if (const int rc = check_sizes("fp8_quantize_rows", M, 1, K)) return rc;
  if (M == 0) return KB2_OK;
  if (!x_dev || !codes_dev || !scales_dev) return failf(KB2_ERR_VALUE, "null argument");
  if (off16(codes_dev) || ldx < 0 || ld_scales < M) return failf(KB2_ERR_VALUE, "fp8_quantize_rows: codes on 16 bytes, ldx >= 0, ld_scales >= M");
  OnDevice on(device);
  CUDA_TRY(on.err);
  CUDA_TRY(launch_fp8_rows(x_dev, x_f32 != 0, ldx, M, K, codes_dev, scales_dev, ld_scales, nullptr, 0, (cudaStream_t)stream));
  return KB2_OK;
}

KB2_API int kb2_fp8_quantize_blocks(const void* w_dev, int32_t w_f32, int32_t groups, int32_t N, int32_t K, void* codes_dev, float* scales_dev, int32_t device,
                                    void* stream) {
  if (const int rc = check_sizes("fp8_quantize_blocks", groups, N, K)) return rc;
  if (groups == 0) return KB2_OK;
  if (!w_dev || !codes_dev || !scales_dev) return failf(KB2_ERR_VALUE, "null argument");
  if (off16(codes_dev) || groups > 65535) return failf(KB2_ERR_VALUE, "fp8_quantize_blocks: codes on 16 bytes, at most 65535 matrices");
  OnDevice on(device);
  CUDA_TRY(on.err);
  CUDA_TRY(launch_fp8_blocks(w_dev, w_f32 != 0, groups, N, K, codes_dev, scales_dev, (cudaStream_t)stream));
  return KB2_OK;
}

KB2_API int kb2_fp8_linear_rows(const void* codes_dev, const float* scales_dev, int64_t ld_scales, const void* w_dev, const float* w_scales_dev, const float* bias_dev,
                                void* out_dev, int32_t out_f32, int32_t M, int32_t N, int32_t K, int32_t device, void* stream) {
  if (const int rc = check_sizes("fp8_linear", M, N, K)) return rc;
  if (M == 0) return KB2_OK;
  if (!codes_dev || !scales_dev || !w_dev || !w_scales_dev || !out_dev) return failf(KB2_ERR_VALUE, "null argument");
  if (off16(codes_dev) || off16(scales_dev) || off16(w_dev) || off16(out_dev) || ld_scales < M || ld_scales % 4)
    return failf(KB2_ERR_VALUE, "fp8_linear: codes, scales, weights and out on 16 bytes, ld_scales >= M and a multiple of 4");
  OnDevice on(device);
  CUDA_TRY(on.err);
  Fp8Product p;
  p.x = codes_dev; p.xs = scales_dev; p.ldxs = ld_scales; p.w = w_dev; p.ws = w_scales_dev; p.bias = bias_dev;
  p.out = out_dev; p.out_f32 = out_f32 != 0;
  p.M = M; p.N = N; p.K = K;
  CUDA_TRY(launch_fp8_product(p, current_sms(), (cudaStream_t)stream));
  return KB2_OK;
}

KB2_API size_t kb2_fp8_linear_workspace(int32_t M, int32_t K) {
  return M <= 0 || K <= 0 ? 0 : up16((size_t)M * K) + (size_t)scale_ld(M) * fp8_blocks(K) * 4;
}

KB2_API int kb2_fp8_linear(const void* x_dev, int32_t x_f32, int64_t ldx, const void* w_dev, const float* w_scales_dev, const float* bias_dev, void* out_dev,
                           int32_t out_f32, int32_t M, int32_t N, int32_t K, void* work_dev, size_t work_bytes, int32_t device, void* stream) {
  if (const int rc = check_sizes("fp8_linear", M, N, K)) return rc;
  if (M == 0) return KB2_OK;
  if (!work_dev || off16(work_dev) || work_bytes < kb2_fp8_linear_workspace(M, K))
    return failf(KB2_ERR_VALUE, "fp8_linear: a workspace of %zu bytes on 16, %zu needed", work_bytes, kb2_fp8_linear_workspace(M, K));
  if (!w_dev || !w_scales_dev || !out_dev || off16(w_dev) || off16(out_dev)) return failf(KB2_ERR_VALUE, "fp8_linear: weights, scales and out on 16 bytes");
  Carve c(work_dev);
  uint8_t* codes = c.take<uint8_t>((size_t)M * K);
  float* scales = c.take<float>((size_t)scale_ld(M) * fp8_blocks(K));
  if (const int rc = kb2_fp8_quantize_rows(x_dev, x_f32, ldx, M, K, codes, scales, scale_ld(M), device, stream)) return rc;
  return kb2_fp8_linear_rows(codes, scales, scale_ld(M), w_dev, w_scales_dev, bias_dev, out_dev, out_f32, M, N, K, device, stream);
}

// ---- routed experts
struct ExpertsWork {
  uint8_t *xc, *ac;
  float *xs, *as;
  float* y;                                        // the experts' rows
  ChunkDesc* chunks;
  int *n_chunks, *counts, *slot_of;
  int max_chunks;
  long long ldx;
  size_t bytes;
};
static ExpertsWork experts_work(void* work, int T, int top, int E, int W, int F) {
  ExpertsWork k{};
  Carve c(work);
  const size_t slots = (size_t)T * top;
  k.ldx = scale_ld((long long)slots);
  k.max_chunks = (int)std::min<size_t>(slots, slots / kFp8Run + E);
  k.xc = c.take<uint8_t>(slots * W);
  k.xs = c.take<float>((size_t)k.ldx * fp8_blocks(W));
  k.ac = c.take<uint8_t>(slots * F);
  k.as = c.take<float>((size_t)k.ldx * fp8_blocks(F));
  k.y = c.take<float>(slots * W);
  k.chunks = c.take<ChunkDesc>(k.max_chunks);
  k.n_chunks = c.take<int>(1);
  k.counts = c.take<int>(fp8_bin_counts((int)slots, E));
  k.slot_of = c.take<int>(slots);
  k.bytes = c.used;
  return k;
}

static int experts_sizes(long long T, int top, int E, int W, int F) {
  if (T < 0 || top <= 0 || E <= 0 || E > 1024 || W <= 0 || W % 16 || F <= 0 || F % kFp8Block || W > 65535 * 128 || F > 65535 * 64)
    return failf(KB2_ERR_VALUE, "fp8_experts: need T >= 0, top > 0, 1 to 1024 experts, W %% 16 == 0, F %% 128 == 0 (T=%lld top=%d E=%d W=%d F=%d)", T, top, E, W, F);
  if ((long long)E * std::max(2 * F, W) > INT32_MAX / 2) return failf(KB2_ERR_VALUE, "fp8_experts: E=%d W=%d F=%d is too large", E, W, F);
  if (T * top > INT32_MAX / 4) return failf(KB2_ERR_VALUE, "fp8_experts: %lld tokens of %d choices are too many", T, top);
  return KB2_OK;
}

KB2_API size_t kb2_fp8_experts_workspace(int32_t T, int32_t top, int32_t E, int32_t W, int32_t F, int32_t) {
  return experts_sizes(T, top, E, W, F) || T == 0 ? 0 : experts_work(nullptr, T, top, E, W, F).bytes;
}

KB2_API int kb2_fp8_experts(const void* h_dev, int32_t h_f32, int64_t ldh, const int32_t* ids_dev, const float* weights_dev, const void* w1_dev, const float* s1_dev,
                            const void* w2_dev, const float* s2_dev, void* out_dev, int32_t out_f32, int32_t T, int32_t top, int32_t E, int32_t W, int32_t F,
                            void* work_dev, size_t work_bytes, int32_t device, void* stream) {
  if (const int rc = experts_sizes(T, top, E, W, F)) return rc;
  if (T == 0) return KB2_OK;
  if (!h_dev || !ids_dev || !weights_dev || !w1_dev || !s1_dev || !w2_dev || !s2_dev || !out_dev) return failf(KB2_ERR_VALUE, "null argument");
  if (off16(w1_dev) || off16(w2_dev) || off16(out_dev) || ldh < 0) return failf(KB2_ERR_VALUE, "fp8_experts: weights and out on 16 bytes, ldh >= 0");
  const ExpertsWork k = experts_work(work_dev, T, top, E, W, F);
  if (!work_dev || off16(work_dev) || work_bytes < k.bytes) return failf(KB2_ERR_VALUE, "fp8_experts: a workspace of %zu bytes on 16, %zu needed", work_bytes, k.bytes);
  OnDevice on(device);
  CUDA_TRY(on.err);
  cudaStream_t s = (cudaStream_t)stream;
  const int slots = T * top;
  CUDA_TRY(launch_fp8_bin(ids_dev, T, top, E, k.counts, k.chunks, k.n_chunks, k.slot_of, h_dev, h_f32 != 0, ldh, W, k.xc, k.xs, k.ldx, s));
  Fp8Product p;
  p.x = k.xc; p.xs = k.xs; p.ldxs = k.ldx; p.w = w1_dev; p.ws = s1_dev; p.out = k.ac;
  p.M = slots; p.N = 2 * F; p.K = W; p.groups = E;
  p.chunks = k.chunks; p.n_chunks = k.n_chunks; p.max_chunks = k.max_chunks;
  CUDA_TRY(launch_fp8_gated(p, k.as, k.ldx, current_sms(), s));
  p.x = k.ac; p.xs = k.as; p.w = w2_dev; p.ws = s2_dev; p.out = k.y; p.out_f32 = true;
  p.N = W; p.K = F;
  CUDA_TRY(launch_fp8_tiles(p, 1, current_sms(), s));
  CUDA_TRY(launch_fp8_combine(k.y, k.slot_of, weights_dev, T, top, W, out_dev, out_f32 != 0, s));
  return KB2_OK;
}

}  // extern "C"
