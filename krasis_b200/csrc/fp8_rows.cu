// Making 8-bit operands: rows of activations (a scale per 128 numbers) and matrices of weights (a scale per 128 x 128).
#include "fp8.cuh"
#include "prof.cuh"

namespace kb2 {

// Eight numbers, `have` of them there.
template <bool F32, bool VEC>
__device__ __forceinline__ void load8(const void* p, long long at, int have, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = 0.f;
  if (have <= 0) return;
  if constexpr (VEC) {                             // all eight: their number is a multiple of 16
    if constexpr (F32) {
      const float4 a = __ldcs(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + at)), b = __ldcs(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + at) + 1);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 a = __ldcs(reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(p) + at));
      const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(u[i] << 16);
        v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < have) v[i] = F32 ? reinterpret_cast<const float*>(p)[at + i] : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[at + i]);
  }
}
__device__ __forceinline__ uint32_t largest8(const float (&v)[8]) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, __float_as_uint(v[i]) & 0x7FFFFFFFu);      // as whole numbers infinities and NaN are the largest
  return a;
}
// K is a multiple of 16 and the codes lie on 16 bytes: eight of them are there whole or not at all.
__device__ __forceinline__ void store8(void* codes, long long at, const float (&v)[8], float inv) {
  *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(codes) + at) = make_uint2(fp8_codes4(v[0], v[1], v[2], v[3], inv), fp8_codes4(v[4], v[5], v[6], v[7], inv));
}

// Sixteen lanes have a block of 128, eight numbers each; a thread block has 16 rows x kRowsAhead blocks, all of a thread's loads on their way at once.
constexpr int kRowsAhead = 4;
template <bool F32, bool VEC>
__global__ void __launch_bounds__(256) fp8_rows_kernel(const void* x, long long ldx, int M, int K, void* codes, float* scales, long long lds) {
  pdl_wait();
  const int lane = threadIdx.x & 15, m = blockIdx.x * 16 + (threadIdx.x >> 4), b0 = blockIdx.y * kRowsAhead;
  float v[kRowsAhead][8];
#pragma unroll
  for (int i = 0; i < kRowsAhead; ++i) {
    const int k = (b0 + i) * kFp8Block + lane * 8;
    load8<F32, VEC>(x, m * ldx + k, m < M ? K - k : 0, v[i]);
  }
#pragma unroll
  for (int i = 0; i < kRowsAhead; ++i) {
    const int k = (b0 + i) * kFp8Block + lane * 8;
    uint32_t a = largest8(v[i]);
#pragma unroll
    for (int o = 8; o; o >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
    const Fp8Scale s = fp8_scale(a);
    if (m >= M || (b0 + i) * kFp8Block >= K) continue;
    if (k < K) store8(codes, (long long)m * K + k, v[i], s.inv);
    if (lane == 0) scales[(b0 + i) * lds + m] = s.scale;
  }
}

// A thread block has one block of 128 x 128: sixteen lanes a row, eight rows a thread.
template <bool F32, bool VEC>
__global__ void __launch_bounds__(256) fp8_blocks_kernel(const void* w, int N, int K, void* codes, float* scales) {
  pdl_wait();
  __shared__ uint32_t s_max[8];
  const int lane = threadIdx.x & 15, row0 = blockIdx.y * kFp8Block + (threadIdx.x >> 4), k = blockIdx.x * kFp8Block + lane * 8;
  const long long base = (long long)blockIdx.z * N * K + k;
  float v[8][8];
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = row0 + i * 16;
    load8<F32, VEC>(w, base + (long long)n * K, n < N ? K - k : 0, v[i]);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, largest8(v[i]));
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
    if (n < N) store8(codes, base + (long long)n * K, v[i], s.inv);
  }
}

static bool on16(const void* p) { return ((uintptr_t)p & 15) == 0; }

cudaError_t launch_fp8_rows(const void* x, bool f32, long long ldx, int M, int K, void* codes, float* scales, long long ld_scales, cudaStream_t s) {
  KernelSpan ks(K_FP8_QUANTIZE, s);
  const dim3 grid((M + 15) / 16, (fp8_blocks(K) + kRowsAhead - 1) / kRowsAhead);
  const bool vec = on16(x) && ldx % (f32 ? 4 : 8) == 0;
  const auto go = [&](auto kernel) { return launch_pdl(kernel, grid, 256, 0, s, x, ldx, M, K, codes, scales, ld_scales); };
  return f32 ? vec ? go(fp8_rows_kernel<true, true>) : go(fp8_rows_kernel<true, false>) : vec ? go(fp8_rows_kernel<false, true>) : go(fp8_rows_kernel<false, false>);
}

cudaError_t launch_fp8_blocks(const void* w, bool f32, int groups, int N, int K, void* codes, float* scales, cudaStream_t s) {
  KernelSpan ks(K_FP8_QUANTIZE, s);
  const dim3 grid(fp8_blocks(K), fp8_blocks(N), groups);
  const auto go = [&](auto kernel) { return launch_pdl(kernel, grid, 256, 0, s, w, N, K, codes, scales); };
  return f32 ? on16(w) ? go(fp8_blocks_kernel<true, true>) : go(fp8_blocks_kernel<true, false>)
             : on16(w) ? go(fp8_blocks_kernel<false, true>) : go(fp8_blocks_kernel<false, false>);
}

}  // namespace kb2
