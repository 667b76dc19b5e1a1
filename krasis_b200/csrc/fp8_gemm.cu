// Products of 8-bit floating-point operands with a scale per block of 128 (fp8.cuh): out[m][n] = sum_b xs[m][b] ws[n / 128][b] sum_{k in block b} x[m][k] w[n][k].
// A block's 128 products are summed in fp32, then multiplied by the two scales and added up.
#include "fp8.cuh"
#include "prof.cuh"

namespace kb2 {

constexpr int kFTile = 64, kFStep = 32;

// 64 x 64 results of a thread block, 4 x 4 of a thread.
__global__ void __launch_bounds__(256) fp8_product_kernel(const Fp8Product p) {
  pdl_wait();
  __shared__ __align__(16) float xs[kFStep][kFTile + 4], ws[kFStep][kFTile + 4];
  int row0 = 0, rows = p.M, group = 0;
  if (p.chunks) {
    if ((int)blockIdx.z >= p.n_chunks[0]) return;
    const ChunkDesc c = p.chunks[blockIdx.z];
    row0 = c.slot_begin;
    rows = c.n_tok;
    group = c.expert;
  }
  const int m0 = blockIdx.y * kFTile, n0 = blockIdx.x * kFTile, tx = threadIdx.x & 15, ty = threadIdx.x >> 4, nb = fp8_blocks(p.K);
  if (m0 >= rows) return;
  const uint8_t* x = reinterpret_cast<const uint8_t*>(p.x) + (long long)row0 * p.K;
  const uint8_t* w = reinterpret_cast<const uint8_t*>(p.w) + (long long)group * p.N * p.K;
  const auto number = [](uint8_t c) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3))); };
  float acc[4][4] = {};
  for (int b = 0; b < nb; ++b) {
    float part[4][4] = {};
    for (int k0 = b * kFp8Block; k0 < min(p.K, (b + 1) * kFp8Block); k0 += kFStep) {
      for (int i = threadIdx.x; i < kFTile * kFStep; i += 256) {
        const int r = i / kFStep, k = i % kFStep;
        xs[k][r] = m0 + r < rows && k0 + k < p.K ? number(x[(long long)(m0 + r) * p.K + k0 + k]) : 0.f;
        ws[k][r] = n0 + r < p.N && k0 + k < p.K ? number(w[(long long)(n0 + r) * p.K + k0 + k]) : 0.f;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kFStep; ++k) {
        const float4 a = *reinterpret_cast<const float4*>(&xs[k][ty * 4]), c = *reinterpret_cast<const float4*>(&ws[k][tx * 4]);
        const float av[4] = {a.x, a.y, a.z, a.w}, cv[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) part[i][j] = fmaf(av[i], cv[j], part[i][j]);
      }
      __syncthreads();
    }
    const float sw = p.ws[((long long)group * fp8_blocks(p.N) + n0 / kFp8Block) * nb + b];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int m = m0 + ty * 4 + i;
      const float s = m < rows ? p.xs[b * p.ldxs + row0 + m] * sw : 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(part[i][j], s, acc[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
      if (m >= rows || n >= p.N) continue;
      const float v = acc[i][j] + (p.bias ? p.bias[n] : 0.f);
      const long long at = (long long)(row0 + m) * p.N + n;
      if (p.out_f32) reinterpret_cast<float*>(p.out)[at] = v;
      else reinterpret_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
    }
}

cudaError_t launch_fp8_product(const Fp8Product& p, int num_sms, cudaStream_t s) {
  KernelSpan ks(K_FP8_PRODUCT, s);
  const int most = p.chunks ? kMaxChunkTokens : p.M;
  return launch_pdl(fp8_product_kernel, dim3((p.N + kFTile - 1) / kFTile, (most + kFTile - 1) / kFTile, p.chunks ? p.max_chunks : 1), 256, 0, s, p);
}

}  // namespace kb2
