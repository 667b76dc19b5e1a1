// Making 8-bit operands: rows of activations (a scale per 128 numbers) and matrices of weights (a scale per 128 x 128).
#include "fp8.cuh"
#include "prof.cuh"

namespace kb2 {

// Sixteen lanes have a block of 128, eight numbers each; a thread block has 16 rows x kRowsAhead blocks, all of a thread's loads on their way at once, its row's slots among them.
// 8191 x 4096 fp32 (169 MB): 24 us, 7.0 TB/s.  Into the slots of ten experts each, 8192 x 2048 bf16 (207 MB): 40 us, 5.2 TB/s (44 with the slots read one after the other).
constexpr int kRowsAhead = 4;
template <bool F32, bool VEC, bool SLOTS>
__global__ void __launch_bounds__(256) fp8_rows_kernel(const void* x, long long ldx, int M, int K, void* codes, float* scales, long long lds, const int* slot_of, int top) {
  pdl_wait();
  const int lane = threadIdx.x & 15, m = blockIdx.x * 16 + (threadIdx.x >> 4), b0 = blockIdx.y * kRowsAhead;
  Fp8Eight<F32> v[kRowsAhead];
#pragma unroll
  for (int i = 0; i < kRowsAhead; ++i) {
    const int k = (b0 + i) * kFp8Block + lane * 8;
    v[i].template load<VEC>(x, m * ldx + k, m < M ? K - k : 0);
  }
  int slots = SLOTS && m < M && lane < top ? slot_of[(long long)m * top + lane] : -1;         // sixteen of them, one a lane
  float inv[kRowsAhead], scale[kRowsAhead];
#pragma unroll
  for (int i = 0; i < kRowsAhead; ++i) {
    uint32_t a = v[i].largest();
#pragma unroll
    for (int o = 8; o; o >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
    const Fp8Scale s = fp8_scale(a);
    inv[i] = s.inv;
    scale[i] = s.scale;
  }
  if constexpr (SLOTS) {
    uint2 c[kRowsAhead];
#pragma unroll
    for (int i = 0; i < kRowsAhead; ++i) c[i] = v[i].codes(inv[i]);
    for (int j = 0; j < top; ++j) {
      if (j > 0 && (j & 15) == 0) slots = m < M && j + lane < top ? slot_of[(long long)m * top + j + lane] : -1;
      const int slot = __shfl_sync(0xffffffffu, slots, j & 15, 16);
      if (slot < 0) continue;
#pragma unroll
      for (int i = 0; i < kRowsAhead; ++i) {
        const int k = (b0 + i) * kFp8Block + lane * 8;
        if (k < K) *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(codes) + (long long)slot * K + k) = c[i];
        if (lane == 0 && (b0 + i) * kFp8Block < K) scales[(b0 + i) * lds + slot] = scale[i];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kRowsAhead; ++i) {
      const int k = (b0 + i) * kFp8Block + lane * 8;
      if (m >= M || (b0 + i) * kFp8Block >= K) continue;
      if (k < K) v[i].store(codes, (long long)m * K + k, inv[i]);
      if (lane == 0) scales[(b0 + i) * lds + m] = scale[i];
    }
  }
}

// A thread block has one block of 128 x 128: sixteen lanes a row, eight rows a thread, all on their way at once and kept as they are.
template <bool F32, bool VEC>
__global__ void __launch_bounds__(256) fp8_blocks_kernel(const void* w, int N, int K, void* codes, float* scales) {
  pdl_wait();
  __shared__ uint32_t s_max[8];
  const int lane = threadIdx.x & 15, row0 = blockIdx.y * kFp8Block + (threadIdx.x >> 4), k = blockIdx.x * kFp8Block + lane * 8;
  const long long base = (long long)blockIdx.z * N * K + k;
  Fp8Eight<F32> v[8];
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = row0 + i * 16;
    v[i].template load<VEC>(w, base + (long long)n * K, n < N ? K - k : 0);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, v[i].largest());
  a = __reduce_max_sync(0xffffffffu, a);
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = a;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, s_max[i]);
  const Fp8Scale s = fp8_scale(a);
  if (threadIdx.x == 0) scales[((long long)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x] = s.scale;
  if (k >= K) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = row0 + i * 16;
    if (n < N) v[i].store(codes, base + (long long)n * K, s.inv);
  }
}

static bool on16(const void* p) { return ((uintptr_t)p & 15) == 0; }

cudaError_t launch_fp8_rows(const void* x, bool f32, long long ldx, int M, int K, void* codes, float* scales, long long ld_scales, const int* slot_of, int top,
                            cudaStream_t s) {
  KernelSpan ks(K_FP8_QUANTIZE, s);
  const dim3 grid((M + 15) / 16, (fp8_blocks(K) + kRowsAhead - 1) / kRowsAhead);
  const bool vec = on16(x) && ldx % (f32 ? 4 : 8) == 0;
  const auto kernel = slot_of ? f32 ? vec ? fp8_rows_kernel<true, true, true> : fp8_rows_kernel<true, false, true>
                                    : vec ? fp8_rows_kernel<false, true, true> : fp8_rows_kernel<false, false, true>
                              : f32 ? vec ? fp8_rows_kernel<true, true, false> : fp8_rows_kernel<true, false, false>
                                    : vec ? fp8_rows_kernel<false, true, false> : fp8_rows_kernel<false, false, false>;
  return launch_pdl(kernel, grid, 256, 0, s, x, ldx, M, K, codes, scales, ld_scales, slot_of, top);
}

cudaError_t launch_fp8_blocks(const void* w, bool f32, int groups, int N, int K, void* codes, float* scales, cudaStream_t s) {
  KernelSpan ks(K_FP8_QUANTIZE, s);
  const dim3 grid(fp8_blocks(K), fp8_blocks(N), groups);
  const bool vec = on16(w);
  const auto kernel = f32 ? vec ? fp8_blocks_kernel<true, true> : fp8_blocks_kernel<true, false> : vec ? fp8_blocks_kernel<false, true> : fp8_blocks_kernel<false, false>;
  return launch_pdl(kernel, grid, 256, 0, s, w, N, K, codes, scales);
}

}  // namespace kb2
