// The 8-bit key / value cache of ragged-batch serving: rows are quantised as they are written, read back, attended to and moved.
//
// A row is one token's key (or value) of one head, x[n], with a = max |x|:
//   e4m3  scale 2^k, k the least whole number >= -126 with a <= 448 2^k.  A power of two costs a floating format nothing and makes x / scale exact;
//   int8  scale a times 1 / 127, each rounded to fp32 (a product, where a quotient would cost ten instructions); the code is the whole number next to the exact quotient, ties to even.
// a = 0: scale 0.  A row with a number that is not finite gets a NaN for its scale and zeros for codes: whoever sees the row gets NaN, and nobody else,
// as a product with the codes stays finite where the row is masked.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "ptx.cuh"
#include "seq_kv.cuh"

namespace kb2seq {

// ------------------------------------------------------------------------------------------------ writing
// Four numbers of a row -> four codes.
template <int FMT>
__device__ __forceinline__ uint32_t kv_codes4(const float (&x)[4], float s, float inv, float up) {
  if constexpr (FMT == KV_E4M3) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[0] * inv, x[1] * inv), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[2] * inv, x[3] * inv), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
  } else {
    uint32_t c[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float y = x[e] * up;
      float n = rintf(y * inv);                        // within one of the answer; what is left over says which it is
      const float r = fmaf(-n, s, y), far = 2.f * fabsf(r);
      if (far > s || (far == s && (((int)n) & 1))) n += copysignf(1.f, r);
      n = fminf(fmaxf(n, -127.f), 127.f);
      c[e] = (uint32_t)(int)n & 0xFFu;
    }
    return c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
  }
}

// One warp per row; lane l holds the numbers 4 l .. 4 l + 3 and 128 + 4 l ...
template <int FMT, bool F32>
__global__ void __launch_bounds__(256) kv_write_kernel(KvLayer c, KvStep t, const void* __restrict__ k, long long ldk, long long hk, const void* __restrict__ v,
                                                        long long ldv, long long hv) {
  kb2::pdl_wait();
  const long long at = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const bool val = at & 1;
  const long long row = at >> 1;
  const int tok = (int)(row / c.G), g = (int)(row - (long long)tok * c.G);
  if (tok >= t.T || tok >= t.cu[t.S]) return;          // rows behind the last sequence
  const int n = val ? c.dv : c.d;
  const long long from = val ? tok * ldv + g * hv : tok * ldk + g * hk;
  const void* src = val ? v : k;
  float x[2][4];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int e = i * 128 + lane * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[i][j] = e < n ? (F32 ? ((const float*)src)[from + e + j] : __bfloat162float(((const bf16*)src)[from + e + j])) : 0.f;
      top = max(top, __float_as_uint(x[i][j]) & 0x7FFFFFFFu);
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  const long long r0 = kv_row(c, t, t.seq_of[tok], t.rows[tok]);
  if (r0 < 0) return;
  const long long r = r0 + ((long long)g << c.lps);
  const float a = __uint_as_float(top);
  float s, inv, up = 1.f;
  if constexpr (FMT == KV_E4M3) {
    const int e = max((int)(top >> 23) - 126 - 9 + ((top & 0x7FFFFFu) > 0x600000u), -126);      // a <= 448 2^e, 448 = 1.75 2^8
    s = __uint_as_float((uint32_t)(e + 127) << 23);
    inv = __uint_as_float((uint32_t)(127 - e) << 23);
  } else {
    s = a * (1.f / 127.f);
    if (a < 1e-20f) up = 1.8446744073709552e19f;       // 2^64 on both: the reciprocal of a smallest scale does not exist
    inv = 1.f / (s * up);
  }
  const bool bad = top >= 0x7F800000u;
  if (bad) s = __uint_as_float(0x7FFFFFFFu);
  else if (top == 0 || s == 0.f) s = 0.f;
  const bool none = bad || s == 0.f;
  uint8_t* codes = (val ? c.v : c.k) + r * n;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int e = i * 128 + lane * 4;
    if (e < n) *reinterpret_cast<uint32_t*>(codes + e) = none ? 0u : kv_codes4<FMT>(x[i], s * up, inv, up);
  }
  if (lane == 0) (val ? c.vs : c.ks)[r] = s;
}

// ------------------------------------------------------------------------------------------------ reading back
template <int FMT>
__device__ __forceinline__ void kv_unpack4(uint32_t w, float (&f)[4]) {
  if constexpr (FMT == KV_E4M3) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const __half2_raw x = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * h)), __NV_E4M3);
      const float2 y = __half22float2(__half2(x));
      f[2 * h] = y.x;
      f[2 * h + 1] = y.y;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = (float)(int)(int8_t)(w >> (8 * e));
  }
}

// Rows first .. first + count - 1 of sequence s -> [count][G][d] and [count][G][dv]; a thread has 16 codes.
template <int FMT, bool F32>
__global__ void __launch_bounds__(256) kv_read_kernel(KvLayer c, KvStep t, int s, int first, int count, void* __restrict__ ko, void* __restrict__ vo) {
  kb2::pdl_wait();
  const int kd = c.d >> 4, w = kd + (c.dv >> 4);
  const long long total = (long long)count * c.G * w;
  for (long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < total; at += (long long)gridDim.x * 256) {
    const long long rg = at / w;
    const int x = (int)(at - rg * w), i = (int)(rg / c.G), g = (int)(rg - (long long)i * c.G);
    const long long r0 = kv_row(c, t, s, first + i);
    const bool val = x >= kd;
    const int n = val ? c.dv : c.d, e = (val ? x - kd : x) * 16;
    uint4 q = make_uint4(0, 0, 0, 0);
    float sc = 0.f;
    if (r0 >= 0) {
      const long long r = r0 + ((long long)g << c.lps);
      q = *reinterpret_cast<const uint4*>((val ? c.v : c.k) + r * n + e);
      sc = (val ? c.vs : c.ks)[r];
    }
    float f[16];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float y[4];
      kv_unpack4<FMT>(j == 0 ? q.x : j == 1 ? q.y : j == 2 ? q.z : q.w, y);
#pragma unroll
      for (int l = 0; l < 4; ++l) f[4 * j + l] = y[l] * sc;
    }
    const long long to = rg * n + e;
    if constexpr (F32) {
      float4* o = reinterpret_cast<float4*>((float*)(val ? vo : ko) + to);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
    } else {
      uint4* o = reinterpret_cast<uint4*>((bf16*)(val ? vo : ko) + to);
#pragma unroll
      for (int j = 0; j < 2; ++j)
        o[j] = make_uint4(kb2::bf16x2_bits_rn(f[8 * j + 1], f[8 * j]), kb2::bf16x2_bits_rn(f[8 * j + 3], f[8 * j + 2]),
                          kb2::bf16x2_bits_rn(f[8 * j + 5], f[8 * j + 4]), kb2::bf16x2_bits_rn(f[8 * j + 7], f[8 * j + 6]));
    }
  }
}

// ------------------------------------------------------------------------------------------------ the accepted path
// Block (sequence, layer): row base + path[i] -> row base + i.  A path rises, so path[i] >= i: what a thread writes at i no later step reads, and a thread
// keeps its 16 bytes of every row, so it has read whatever it overwrites.
constexpr int kKeepMost = 512;
__global__ void __launch_bounds__(256) kv_keep_kernel(KvLayer c, long long layer_k, long long layer_v, long long layer_s, KvStep t, const int* __restrict__ path, int P) {
  __shared__ long long rows[2][kKeepMost];
  __shared__ int moved;
  kb2::pdl_wait();
  const int s = blockIdx.x, base_tok = t.cu[s], n = t.cu[s + 1] - base_tok;
  if (n <= 0) return;
  const int base = t.rows[base_tok];
  if (threadIdx.x == 0) moved = P;
  __syncthreads();
  for (int i = threadIdx.x; i < P; i += 256) {
    const int from = path[(long long)s * P + i], ahead = i ? path[(long long)s * P + i - 1] : -1;
    const bool good = from > ahead && from >= i && from < n;
    const long long a = good ? kv_row(c, t, s, base + from) : -1, b = good ? kv_row(c, t, s, base + i) : -1;
    rows[0][i] = a;
    rows[1][i] = b;
    if (a < 0 || b < 0) atomicMin(&moved, i);          // the path ends here
  }
  __syncthreads();
  const int m = moved, kd = c.d >> 4, w = kd + (c.dv >> 4);
  const long long layer = blockIdx.y;
  uint8_t *k = c.k + layer * layer_k, *v = c.v + layer * layer_v;
  float *ks = c.ks + layer * layer_s, *vs = c.vs + layer * layer_s;
  for (int x = threadIdx.x; x < c.G * w; x += 256) {
    const int g = x / w, e = x - g * w;
    const bool val = e >= kd;
    const long long n16 = val ? c.dv : c.d, off = ((long long)g << c.lps) * n16 + (val ? e - kd : e) * 16;
    uint8_t* p = val ? v : k;
    for (int i0 = 0; i0 < m; i0 += 8) {
      uint4 b[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i0 + i < m) b[i] = *reinterpret_cast<const uint4*>(p + rows[0][i0 + i] * n16 + off);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i0 + i < m) *reinterpret_cast<uint4*>(p + rows[1][i0 + i] * n16 + off) = b[i];
    }
  }
  for (int x = threadIdx.x; x < 2 * c.G; x += 256) {
    float* p = (x & 1) ? vs : ks;
    const long long off = (long long)(x >> 1) << c.lps;
    for (int i = 0; i < m; ++i) p[rows[1][i] + off] = p[rows[0][i] + off];
  }
}
}  // namespace kb2seq

using namespace kb2seq;

extern "C" {

KB2SEQ_API int kb2_seq_kv_write(const kb2_seq_kv_cache* cache, int layer, const kb2_seq_kv_step* step, const void* k, long long ldk, long long hk, const void* v,
                                long long ldv, long long hv, int dt, void* stream) {
  KvLayer c;
  KvStep t;
  if (int e = kv_args("kv_write", cache, layer, step, &c, &t)) return e;
  if (!k || !v || bad_dt(dt)) return failf(KB2SEQ_ERR_VALUE, "kv_write: bad argument");
  if (t.T == 0) return KB2SEQ_OK;
  OnDevice on(step->device);
  SEQ_CUDA(on.err);
  const long long blocks = ((long long)t.T * c.G * 2 + 7) / 8;
  if (blocks > 0x7FFFFFFFll) return failf(KB2SEQ_ERR_VALUE, "kv_write: too many rows");
  auto kern = cache->fmt == KV_E4M3 ? (dt ? kv_write_kernel<KV_E4M3, false> : kv_write_kernel<KV_E4M3, true>)
                                    : (dt ? kv_write_kernel<KV_INT8, false> : kv_write_kernel<KV_INT8, true>);
  kb2::launch_pdl(kern, (unsigned)blocks, 256, 0, (cudaStream_t)stream, c, t, k, ldk, hk, v, ldv, hv);
  SEQ_LAUNCHED();
  return KB2SEQ_OK;
}

KB2SEQ_API int kb2_seq_kv_read(const kb2_seq_kv_cache* cache, int layer, const kb2_seq_kv_step* step, int s, int first, int count, void* k, void* v, int dt,
                               void* stream) {
  KvLayer c;
  KvStep t;
  if (int e = kv_args("kv_read", cache, layer, step, &c, &t)) return e;
  if (bad_dt(dt) || s < 0 || s >= t.S || first < 0 || count < 0 || (count && (!k || !v || (((uintptr_t)k | (uintptr_t)v) & 15))))
    return failf(KB2SEQ_ERR_VALUE, "kv_read: bad argument");
  if ((long long)first + count > (long long)step->layout[4 * s + 3] << c.lps)
    return failf(KB2SEQ_ERR_RANGE, "kv_read: %d pages of %d rows do not hold rows %d .. %lld", step->layout[4 * s + 3], cache->page_size, first, (long long)first + count - 1);
  if (count == 0) return KB2SEQ_OK;
  OnDevice on(step->device);
  SEQ_CUDA(on.err);
  const long long total = (long long)count * c.G * ((c.d + c.dv) / 16);
  const unsigned blocks = (unsigned)std::min((total + 255) / 256, kb2::current_sms() * 16ll);
  auto kern = cache->fmt == KV_E4M3 ? (dt ? kv_read_kernel<KV_E4M3, false> : kv_read_kernel<KV_E4M3, true>)
                                    : (dt ? kv_read_kernel<KV_INT8, false> : kv_read_kernel<KV_INT8, true>);
  kb2::launch_pdl(kern, blocks, 256, 0, (cudaStream_t)stream, c, t, s, first, count, k, v);
  SEQ_LAUNCHED();
  return KB2SEQ_OK;
}

KB2SEQ_API int kb2_seq_kv_keep(const kb2_seq_kv_cache* cache, const kb2_seq_kv_step* step, const int* path, int P, void* stream) {
  KvLayer c;
  KvStep t;
  if (int e = kv_args("kv_keep", cache, 0, step, &c, &t)) return e;
  if (P < 0 || P > kKeepMost || (P && !path)) return failf(KB2SEQ_ERR_VALUE, "kv_keep: a path of at most %d rows", kKeepMost);
  if (P == 0 || t.T == 0) return KB2SEQ_OK;
  if (cache->layers > 65535) return failf(KB2SEQ_ERR_VALUE, "kv_keep: too many layers");
  OnDevice on(step->device);
  SEQ_CUDA(on.err);
  const long long rows = ((long long)c.pages * c.G) << c.lps;
  kb2::launch_pdl(kv_keep_kernel, dim3(t.S, cache->layers), 256, 0, (cudaStream_t)stream, c, rows * c.d, rows * c.dv, rows, t, path, P);
  SEQ_LAUNCHED();
  return KB2SEQ_OK;
}

}  // extern "C"
