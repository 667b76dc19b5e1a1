// Routed experts on 8-bit operands (fp8.cuh): what lies behind their two products.
#include "fp8.cuh"
#include "prof.cuh"
#include "ptx.cuh"

namespace kb2 {

// out[t] = sum_j weights[t][j] y[slot_of[t][j]] in the order of j; entries without a slot bring nothing.  A thread has 16 bytes of a row, four rows on their way at once.
// W is a multiple of 16, so a row is whole pieces.
template <bool F32>
__global__ void __launch_bounds__(128) fp8_combine_kernel(const void* y, const int* slot_of, const float* weights, int top, int W, void* out) {
  constexpr int kVec = F32 ? 4 : 8;
  pdl_enter_global(y, slot_of, weights, out);
  const int v = blockIdx.y * 128 + threadIdx.x, pieces = W / kVec;
  if (v >= pieces) return;
  const long long e0 = (long long)blockIdx.x * top;
  float sum[kVec] = {};
  for (int j0 = 0; j0 < top; j0 += 4) {
    uint4 x[4];
    float w[4];
    int slot[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) slot[j] = j0 + j < top ? slot_of[e0 + j0 + j] : -1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (slot[j] < 0) continue;
      x[j] = reinterpret_cast<const uint4*>(y)[(long long)slot[j] * pieces + v];
      w[j] = weights[e0 + j0 + j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (slot[j] < 0) continue;
      const uint32_t u[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (F32) {
          sum[i] = fmaf(w[j], __uint_as_float(u[i]), sum[i]);
        } else {
          sum[2 * i] = fmaf(w[j], __uint_as_float(u[i] << 16), sum[2 * i]);
          sum[2 * i + 1] = fmaf(w[j], __uint_as_float(u[i] & 0xFFFF0000u), sum[2 * i + 1]);
        }
      }
    }
  }
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = F32 ? __float_as_uint(sum[i]) : bf16x2_bits_rn(sum[(2 * i + 1) % kVec], sum[2 * i % kVec]);
  reinterpret_cast<uint4*>(out)[(long long)blockIdx.x * pieces + v] = make_uint4(o[0], o[1], o[2], o[3]);
}

cudaError_t launch_fp8_combine(const void* y, bool f32, const int* slot_of, const float* weights, int T, int top, int W, void* out, cudaStream_t s) {
  KernelSpan ks(K_COMBINE, s);
  const dim3 grid(T, (W / (f32 ? 4 : 8) + 127) / 128);
  return f32 ? launch_pdl(fp8_combine_kernel<true>, grid, 128, 0, s, y, slot_of, weights, top, W, out)
             : launch_pdl(fp8_combine_kernel<false>, grid, 128, 0, s, y, slot_of, weights, top, W, out);
}

}  // namespace kb2
