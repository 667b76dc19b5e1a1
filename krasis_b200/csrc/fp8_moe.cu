// Routed experts on 8-bit operands (fp8.cuh): what lies ahead of and behind their two products.
#include "fp8.cuh"
#include "prof.cuh"

namespace kb2 {

// Rows in the experts' order: codes and scales of token slot / top, copied from the tokens' own.
__global__ void __launch_bounds__(256) fp8_gather_kernel(const uint8_t* codes, const float* scales, long long lds, const int* token_of, const int* slots, int K,
                                                         uint8_t* out, float* out_scales, long long ldo) {
  pdl_wait();
  const int slot = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (slot >= slots[0]) return;
  const int t = token_of[slot];
  for (int k = lane * 16; k < K; k += 512) *reinterpret_cast<uint4*>(out + (long long)slot * K + k) = *reinterpret_cast<const uint4*>(codes + (long long)t * K + k);
  for (int b = lane; b < fp8_blocks(K); b += 32) out_scales[b * ldo + slot] = scales[b * lds + t];
}

// out[t] = sum_j weights[t][j] y[slot_of[t][j]] in the order of j; entries without a slot bring nothing.
template <bool F32>
__global__ void __launch_bounds__(256) fp8_combine_kernel(const void* y, const int* slot_of, const float* weights, int top, int W, void* out) {
  pdl_wait();
  const int w = blockIdx.y * 256 + threadIdx.x;
  if (w >= W) return;
  float sum = 0.f;
  for (int j = 0; j < top; ++j) {
    const long long e = (long long)blockIdx.x * top + j;
    const int slot = slot_of[e];
    if (slot < 0) continue;
    const long long at = (long long)slot * W + w;
    sum = fmaf(weights[e], F32 ? reinterpret_cast<const float*>(y)[at] : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(y)[at]), sum);
  }
  const long long at = (long long)blockIdx.x * W + w;
  if constexpr (F32) reinterpret_cast<float*>(out)[at] = sum;
  else reinterpret_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(sum);
}

cudaError_t launch_fp8_gather(const void* codes, const float* scales, long long lds, const int* token_of, const int* slots, int max_slots, int K, void* out,
                              float* out_scales, long long ldo, cudaStream_t s) {
  KernelSpan ks(K_FP8_QUANTIZE, s);
  return launch_pdl(fp8_gather_kernel, (max_slots + 7) / 8, 256, 0, s, (const uint8_t*)codes, scales, lds, token_of, slots, K, (uint8_t*)out, out_scales, ldo);
}
cudaError_t launch_fp8_combine(const void* y, bool f32, const int* slot_of, const float* weights, int T, int top, int W, void* out, cudaStream_t s) {
  KernelSpan ks(K_COMBINE, s);
  const dim3 grid(T, (W + 255) / 256);
  return f32 ? launch_pdl(fp8_combine_kernel<true>, grid, 256, 0, s, y, slot_of, weights, top, W, out)
             : launch_pdl(fp8_combine_kernel<false>, grid, 256, 0, s, y, slot_of, weights, top, W, out);
}

}  // namespace kb2
