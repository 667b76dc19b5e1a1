// What the kernels of the 8-bit cache's attention on tcgen05 share: descriptors, pairs of fp32 numbers, units of scales.
#pragma once
#include "seq_kv_attn.cuh"

namespace kb2seq {
namespace {
using namespace kb2;

__device__ __forceinline__ uint32_t idesc_f16(uint32_t n, bool mn) {       // A and B fp16, accumulator fp32, 128 rows; mn: B lies with its columns side by side
  return (1u << 4) | ((uint32_t)mn << 16) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}
// rows of 64 numbers (128 bytes) one key apart, chunks of 64 columns `chunk` bytes apart
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr, uint32_t chunk) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)(chunk >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float m;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
  return p;
}
__device__ __forceinline__ float2 pair_get(uint64_t p) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
  return f;
}
__device__ __forceinline__ uint64_t pair_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t p;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(p) : "l"(a), "l"(b), "l"(c));
  return p;
}
__device__ __forceinline__ uint64_t pair_mul(uint64_t a, uint64_t b) {
  uint64_t p;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(p) : "l"(a), "l"(b));
  return p;
}
__device__ __forceinline__ uint64_t pair_add(uint64_t a, uint64_t b) {
  uint64_t p;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(p) : "l"(a), "l"(b));
  return p;
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
      "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// 2^-7 of the least power of two above a scale (its bits), and one over it: codes of 448 times 2^7 stay within fp16, and a scale keeps its bits down to 2^-21 of the
// tile's largest.
__device__ __forceinline__ void scale_unit(uint32_t bits, float* p, float* inv) {
  const uint32_t e = min(max(bits >> 23, 8u), 252u) - 6;
  *p = __uint_as_float(e << 23);
  *inv = __uint_as_float((254 - e) << 23);
}

}  // namespace
}  // namespace kb2seq
