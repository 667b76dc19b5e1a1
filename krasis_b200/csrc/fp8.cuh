// 8-bit floating-point operands with a scale per block of 128, shared by fp8_rows.cu (making them), fp8_gemm.cu (products) and capi_fp8.cu.
//
// A block is 128 numbers of a row (activations) or 128 x 128 numbers of a matrix (weights); the last ones of a row or column may be cut short.  With a = max |x| over
// the block: scale 2^k, k the least whole number >= -126 with a <= 448 2^k, codes e4m3(x / scale), ties to even.  A power of two costs a floating format nothing and
// makes x / scale exact.  a = 0: scale 0, codes 0.  A number that is not finite: scale NaN, codes 0.  The products take any fp32 scales.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "moe_common.cuh"
#include "ptx.cuh"

namespace kb2 {

constexpr int kFp8Block = 128;
constexpr int kFp8Run = 128;      // the most rows of a run
__host__ __device__ constexpr int fp8_blocks(int n) { return (n + kFp8Block - 1) / kFp8Block; }

// What the bits of a block's largest magnitude say: its scale, and the reciprocal that numbers are multiplied by (0 where the codes are zeros).
struct Fp8Scale {
  float scale, inv;
};
__device__ __forceinline__ Fp8Scale fp8_scale(uint32_t a) {
  const int e = (int)(a >> 23) - 127, k = max(e - 8 + ((a & 0x7FFFFFu) > 0x600000u ? 1 : 0), -126);      // 448 = 1.75 2^8
  Fp8Scale s;
  s.scale = __uint_as_float((uint32_t)(k + 127) << 23);
  s.inv = __uint_as_float((uint32_t)(127 - k) << 23);
  if (a == 0) s.scale = s.inv = 0.f;
  if (a >= 0x7F800000u) {
    s.scale = __uint_as_float(0x7FC00000u);
    s.inv = 0.f;
  }
  return s;
}
// Four numbers -> four codes.  inv 0: zeros, whatever the numbers are.
__device__ __forceinline__ uint32_t fp8_codes4(float a, float b, float c, float d, float inv) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a * inv, b * inv), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c * inv, d * inv), __NV_SATFINITE, __NV_E4M3);
  return inv == 0.f ? 0u : lo | hi << 16;
}

// Eight neighbouring numbers as they are in memory.
template <bool F32>
struct Fp8Eight {
  uint32_t u[F32 ? 8 : 4];
  // `have` of them are there
  template <bool VEC>
  __device__ __forceinline__ void load(const void* p, long long at, int have) {
#pragma unroll
    for (int i = 0; i < (F32 ? 8 : 4); ++i) u[i] = 0;
    if (have <= 0) return;
    if constexpr (VEC) {                           // all eight: their number is a multiple of 16
      const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(p) + at * (F32 ? 4 : 2));
#pragma unroll
      for (int i = 0; i < (F32 ? 2 : 1); ++i) {
        const uint4 a = __ldcs(q + i);
        u[4 * i] = a.x; u[4 * i + 1] = a.y; u[4 * i + 2] = a.z; u[4 * i + 3] = a.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i >= have) continue;
        if constexpr (F32) u[i] = reinterpret_cast<const uint32_t*>(p)[at + i];
        else u[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[at + i] << (i & 1) * 16;
      }
    }
  }
  __device__ __forceinline__ float number(int i) const {
    if constexpr (F32) return __uint_as_float(u[i]);
    else return __uint_as_float(i & 1 ? u[i / 2] & 0xFFFF0000u : u[i / 2] << 16);
  }
  // the bits of the largest magnitude: as whole numbers infinities and NaN are the largest
  __device__ __forceinline__ uint32_t largest() const {
    if constexpr (F32) {
      uint32_t a = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) a = max(a, u[i] & 0x7FFFFFFFu);
      return a;
    } else {
      const uint32_t a = __vmaxu2(__vmaxu2(u[0] & 0x7FFF7FFFu, u[1] & 0x7FFF7FFFu), __vmaxu2(u[2] & 0x7FFF7FFFu, u[3] & 0x7FFF7FFFu));
      return max(a << 16, a & 0xFFFF0000u);
    }
  }
  __device__ __forceinline__ uint2 codes(float inv) const {
    return make_uint2(fp8_codes4(number(0), number(1), number(2), number(3), inv), fp8_codes4(number(4), number(5), number(6), number(7), inv));
  }
  // K is a multiple of 16 and the codes lie on 16 bytes: eight of them are there whole or not at all.
  __device__ __forceinline__ void store(void* to, long long at, float inv) const { *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(to) + at) = codes(inv); }
};

template <int N>
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
// c += a b for two numbers at once, where it stands among loads and waits
__device__ __forceinline__ void fma2_here(uint64_t& c, uint64_t a, uint64_t b) { asm volatile("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c) : "l"(a), "l"(b)); }
// out[m] = sum over the blocks of scales x codes of row m times those of w, per matrix of `groups` ones.  x [.][K] codes with scales xs[b * ldxs + row],
// w [groups][N][K] with scales ws [groups][blocks of N][blocks of K].
struct Fp8Product {
  const void* x = nullptr;
  const float* xs = nullptr;
  long long ldxs = 0;
  const void* w = nullptr;
  const float* ws = nullptr;
  const float* bias = nullptr;      // [N], one matrix only
  void* out = nullptr;              // [M][N], bf16 or fp32
  bool out_f32 = false;
  int M = 0, N = 0, K = 0;
  int groups = 1;
  // runs of up to kFp8Run rows that share a matrix (null: all M rows, one matrix), at most max_chunks of them
  const ChunkDesc* chunks = nullptr;
  const int* n_chunks = nullptr;
  int max_chunks = 0;
};

// Rows of activations.  With slot_of [M][top] a row goes to each of its slots (negative: none) instead of its own place, codes and scales.
cudaError_t launch_fp8_rows(const void* x, bool f32, long long ldx, int M, int K, void* codes, float* scales, long long ld_scales, const int* slot_of, int top, cudaStream_t s);
// Routed experts: the slots of the choices ids [T][top] (-1: outside the E experts), the runs of each expert's rows, and the tokens' quantised rows in their slots; counts:
// fp8_bin_counts numbers.
int fp8_bin_counts(int n, int E);
cudaError_t launch_fp8_bin(const int* ids, int T, int top, int E, int* counts, ChunkDesc* runs, int* n_runs, int* slot_of, const void* x, bool f32, long long ldx, int K, void* codes,
                           float* scales, long long lds, cudaStream_t s);
// out[t] = sum_j weights[t][j] y[slot_of[t][j]], bf16 or fp32
cudaError_t launch_fp8_combine(const float* y, const int* slot_of, const float* weights, int T, int top, int W, void* out, bool f32, cudaStream_t s);
cudaError_t launch_fp8_blocks(const void* w, bool f32, int groups, int N, int K, void* codes, float* scales, cudaStream_t s);
// One matrix, all M rows, on pairs of CTAs with tiles of 256 x 256.
cudaError_t launch_fp8_pairs(const Fp8Product& p, int num_sms, cudaStream_t s);
// Runs (one matrix: tiles of kFp8Run rows) on single CTAs; split: CTAs that share a tile of one matrix along K.
cudaError_t launch_fp8_tiles(const Fp8Product& p, int split, int num_sms, cudaStream_t s);
// How many clusters of so many (1, 2, 4, 8) CTAs there can be at once.
int fp8_clusters(int split);
// Runs times matrices [gate: N / 2 | up: N / 2]: silu(gate) up in fp32, quantised by rows: codes [M][N / 2] in p.out, out_scales[b * ld + row].  N % 256 == 0.
cudaError_t launch_fp8_gated(const Fp8Product& p, float* out_scales, long long ld_out_scales, int num_sms, cudaStream_t s);
// One matrix, whichever of the two is estimated to be faster.
cudaError_t launch_fp8_product(const Fp8Product& p, int num_sms, cudaStream_t s);

}  // namespace kb2
