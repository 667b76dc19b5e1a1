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
__device__ __forceinline__ uint32_t kv_codes4(const float* x, float s, float inv, float up) {
  if constexpr (FMT == KV_E4M3) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[0] * inv, x[1] * inv), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[2] * inv, x[3] * inv), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
  } else {
    // x / s to a whole number: 1.5 2^23 leaves no room for a fraction, and the lowest byte of what comes is the code.  The reciprocal's rounding moves a quotient of at most
    // 127 by 2^-16 or less, so only one that lies that near to the middle of two codes can have gone the other way: what is left over, x - code s, says so.
    float t[4], far = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      t[e] = fmaf(x[e], inv, 12582912.f);
      far = fmaxf(far, fabsf(fmaf(-(t[e] - 12582912.f), s, x[e])));
    }
    if (2.f * far >= s * 0.9999f || up != 1.f) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float y = x[e] * up, u = s * up, w = fmaf(y, 1.f / u, 12582912.f), r = fmaf(-(w - 12582912.f), u, y), off = 2.f * fabsf(r);
        int k = __float_as_int(w) - 0x4B400000;
        if (off > u || (off == u && (k & 1))) k += r > 0.f ? 1 : -1;
        t[e] = __int_as_float(0x4B400000 + min(max(k, -127), 127));
      }
    }
    return __byte_perm(__byte_perm(__float_as_uint(t[0]), __float_as_uint(t[1]), 0x0040), __byte_perm(__float_as_uint(t[2]), __float_as_uint(t[3]), 0x0040), 0x5410);
  }
}

// A lane has eight numbers of a row, so a row has n / 8 lanes (of a power of two of them), and a warp 32 / lanes rows at a time; kWriteRows times that are asked for at once.
// What bounds it: 8192 tokens of 4 + 4 heads of 128 in bf16 (25 MB, 3.9 us at the copy rate) take 12.6 us as int8, 9.1 without making the codes: two rounds of loads a thread
// (rows and tables, then the page list) and the codes' arithmetic.  Four rows a thread 13.3, one 12.7.  VEC: every eight numbers lie on 16 bytes.
constexpr int kWriteRows = 2;
template <int FMT, bool F32, bool VEC>
__global__ void __launch_bounds__(256) kv_write_kernel(KvLayer c, KvStep t, const void* __restrict__ k, long long ldk, long long hk, const void* __restrict__ v,
                                                        long long ldv, long long hv) {
  kb2::pdl_enter(k, v);
  const bool val = blockIdx.y;
  const int n = val ? c.dv : c.d, lanes = n <= 64 ? 8 : n <= 128 ? 16 : 32, rows = 256 / lanes, e = (threadIdx.x & (lanes - 1)) * 8;
  const void* src = val ? v : k;
  const long long ld = val ? ldv : ldk, hs = val ? hv : hk;
  const unsigned total = (unsigned)t.T * c.G;
  const int end = t.cu[t.S];                                               // behind the last sequence nothing is written; what lies there may be read
  const unsigned first = blockIdx.x * (rows * kWriteRows) + threadIdx.x / lanes;
  float x[kWriteRows][8];
  int seq[kWriteRows], pos[kWriteRows], head[kWriteRows], token[kWriteRows];
#pragma unroll
  for (int i = 0; i < kWriteRows; ++i) {
    const unsigned row = first + i * rows;
    seq[i] = pos[i] = head[i] = 0;
    token[i] = 0x7FFFFFFF;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[i][j] = 0.f;
    if (row >= total) continue;
    const int tok = (int)(row / (unsigned)c.G), g = head[i] = (int)(row - (unsigned)tok * c.G);
    token[i] = tok;
    seq[i] = t.seq_of[tok];
    pos[i] = t.rows[tok];
    if (e >= n) continue;
    const long long from = (long long)tok * ld + g * hs + e;
    if constexpr (F32) {
      const float* p = (const float*)src + from;
      if constexpr (VEC) {
        const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
        x[i][0] = a.x; x[i][1] = a.y; x[i][2] = a.z; x[i][3] = a.w;
        x[i][4] = b.x; x[i][5] = b.y; x[i][6] = b.z; x[i][7] = b.w;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[i][j] = p[j];
      }
    } else {
      const bf16* p = (const bf16*)src + from;
      if constexpr (VEC) {
        unpack8(*reinterpret_cast<const uint4*>(p), x[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[i][j] = __bfloat162float(p[j]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kWriteRows; ++i) {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[i][j]) & 0x7FFFFFFFu);
    for (int o = lanes / 2; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (token[i] >= end) continue;
    const long long r0 = kv_row(c, t, seq[i], pos[i]);
    if (r0 < 0) continue;
    const long long r = r0 + ((long long)head[i] << c.lps);
    const float a = __uint_as_float(top);
    float s, inv, up = 1.f;
    if constexpr (FMT == KV_E4M3) {
      const int b = max((int)(top >> 23) - 126 - 9 + ((top & 0x7FFFFFu) > 0x600000u), -126);      // a <= 448 2^b, 448 = 1.75 2^8
      s = __uint_as_float((uint32_t)(b + 127) << 23);
      inv = __uint_as_float((uint32_t)(127 - b) << 23);
    } else {
      s = a * (1.f / 127.f);
      if (a < 1e-20f) up = 1.8446744073709552e19f;     // 2^64 on both: the reciprocal of a smallest scale does not exist
      inv = __fdividef(1.f, s);
    }
    const bool bad = top >= 0x7F800000u, none = bad || top == 0 || s == 0.f;
    if (none) s = bad ? __uint_as_float(0x7FFFFFFFu) : 0.f;
    if (e < n) {
      const uint32_t lo = none ? 0u : kv_codes4<FMT>(x[i], s, inv, up), hi = none ? 0u : kv_codes4<FMT>(x[i] + 4, s, inv, up);
      *reinterpret_cast<uint2*>((val ? c.v : c.k) + r * n + e) = make_uint2(lo, hi);
    }
    if (e == 0) (val ? c.vs : c.ks)[r] = s;
  }
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

// Rows first .. first + count - 1 of sequence s -> [count][G][d] and [count][G][dv]; a thread has 16 codes, AHEAD times.
// What bounds it: bytes, two thirds of them written (40001 rows of 4 + 4 heads of 128 to bf16: 124 MB in 24.5 us, 5.1 TB/s).
template <int FMT, bool F32, int AHEAD>
__global__ void __launch_bounds__(256) kv_read_kernel(KvLayer c, KvStep t, int s, int first, int count, void* __restrict__ ko, void* __restrict__ vo) {
  kb2::pdl_enter(ko, vo);
  const int kd = c.d >> 4, w = kd + (c.dv >> 4);
  const unsigned total = (unsigned)count * c.G * w, at = blockIdx.x * (256 * AHEAD) + threadIdx.x;
  uint4 q[AHEAD];
  float sc[AHEAD];
  long long to[AHEAD];
  bool val[AHEAD];
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) {
    const unsigned x = at + j * 256;
    to[j] = -1;
    q[j] = make_uint4(0, 0, 0, 0);
    sc[j] = 0.f;
    if (x >= total) continue;
    const unsigned rg = x / (unsigned)w;
    const int y = (int)(x - rg * w), i = (int)(rg / (unsigned)c.G), g = (int)(rg - (unsigned)i * c.G);
    const long long r0 = kv_row(c, t, s, first + i);
    val[j] = y >= kd;
    const int n = val[j] ? c.dv : c.d, e = (val[j] ? y - kd : y) * 16;
    to[j] = (long long)rg * n + e;
    if (r0 >= 0) {
      const long long r = r0 + ((long long)g << c.lps);
      q[j] = ld_stream16((val[j] ? c.v : c.k) + r * n + e);
      sc[j] = (val[j] ? c.vs : c.ks)[r];
    }
  }
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) {
    if (to[j] < 0) continue;
    float f[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float y[4];
      kv_unpack4<FMT>(i == 0 ? q[j].x : i == 1 ? q[j].y : i == 2 ? q[j].z : q[j].w, y);
#pragma unroll
      for (int l = 0; l < 4; ++l) f[4 * i + l] = y[l] * sc[j];
    }
    if constexpr (F32) {
      float4* o = reinterpret_cast<float4*>((float*)(val[j] ? vo : ko) + to[j]);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
    } else {
      uint4* o = reinterpret_cast<uint4*>((bf16*)(val[j] ? vo : ko) + to[j]);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        o[i] = make_uint4(kb2::bf16x2_bits_rn(f[8 * i + 1], f[8 * i]), kb2::bf16x2_bits_rn(f[8 * i + 3], f[8 * i + 2]), kb2::bf16x2_bits_rn(f[8 * i + 5], f[8 * i + 4]),
                          kb2::bf16x2_bits_rn(f[8 * i + 7], f[8 * i + 6]));
    }
  }
}

// ------------------------------------------------------------------------------------------------ the accepted path
// Block (sequence, kKeepLayers layers): row base + path[i] -> row base + i.  A path rises, so path[i] >= i: what a thread writes at i no later step reads, and a thread
// keeps its 16 bytes of every row (eight rows on their way at once), so it has read whatever it overwrites.  What bounds it: the chain of tables ahead of the rows, so
// a block has work for all its threads (64 paths of 8 in 48 layers: a layer a block 22 us, four 15.5, eight 14; 7.9 at the copy rate).
constexpr int kKeepMost = 512, kKeepLayers = 8;
__global__ void __launch_bounds__(256) kv_keep_kernel(KvLayer c, int layers, KvStep t, const int* __restrict__ path, int P) {
  __shared__ long long rows[2][kKeepMost];
  __shared__ int moved;
  kb2::pdl_enter(path);
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
  const int m = moved, kd = c.d >> 4, w = kd + (c.dv >> 4), of = c.G * (w + 2), l0 = blockIdx.y * kKeepLayers, ln = min(kKeepLayers, layers - l0);
  const long long all = ((long long)c.pages * c.G) << c.lps;               // rows of a layer
  for (int x = threadIdx.x; x < of * ln; x += 256) {
    const int layer = l0 + x / of, y = x % of, g = y / (w + 2), e = y - g * (w + 2);
    const long long head = layer * all + ((long long)g << c.lps);
    if (e < w) {
      const bool val = e >= kd;
      const long long n16 = val ? c.dv : c.d;
      uint8_t* p = (val ? c.v : c.k) + head * n16 + (val ? e - kd : e) * 16;
      for (int i0 = 0; i0 < m; i0 += 8) {
        uint4 b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i0 + i < m) b[i] = *reinterpret_cast<const uint4*>(p + rows[0][i0 + i] * n16);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i0 + i < m) *reinterpret_cast<uint4*>(p + rows[1][i0 + i] * n16) = b[i];
      }
    } else {
      float* p = (e > w ? c.vs : c.ks) + head;
      for (int i0 = 0; i0 < m; i0 += 8) {
        float b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i0 + i < m) b[i] = p[rows[0][i0 + i]];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i0 + i < m) p[rows[1][i0 + i]] = b[i];
      }
    }
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
  if (bad_dt(dt) || (t.T > 0 && (!k || !v))) return failf(KB2SEQ_ERR_VALUE, "kv_write: bad argument");
  if (t.T == 0) return KB2SEQ_OK;
  OnDevice on(step->device);
  SEQ_CUDA(on.err);
  const int most = std::max(c.d, c.dv), rows = 256 / (most <= 64 ? 8 : most <= 128 ? 16 : 32) * kWriteRows;      // the wider of the two: the other's last blocks have none
  const long long blocks = ((long long)t.T * c.G + rows - 1) / rows;
  if ((long long)t.T * c.G > 0x7FFFFFFFll - 4096) return failf(KB2SEQ_ERR_VALUE, "kv_write: too many rows");
  const long long unit = dt ? 8 : 4;
  const bool vec = !(((uintptr_t)k | (uintptr_t)v) & 15) && ldk % unit == 0 && ldv % unit == 0 && hk % unit == 0 && hv % unit == 0;
  auto kern = cache->fmt == KV_E4M3 ? (dt ? (vec ? kv_write_kernel<KV_E4M3, false, true> : kv_write_kernel<KV_E4M3, false, false>)
                                          : (vec ? kv_write_kernel<KV_E4M3, true, true> : kv_write_kernel<KV_E4M3, true, false>))
                                    : (dt ? (vec ? kv_write_kernel<KV_INT8, false, true> : kv_write_kernel<KV_INT8, false, false>)
                                          : (vec ? kv_write_kernel<KV_INT8, true, true> : kv_write_kernel<KV_INT8, true, false>));
  kb2::launch_pdl(kern, dim3((unsigned)blocks, 2), 256, 0, (cudaStream_t)stream, c, t, k, ldk, hk, v, ldv, hv);
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
  if (total > 0x7FFFFFFFll - 4096) return failf(KB2SEQ_ERR_VALUE, "kv_read: too many rows");
  const bool ahead = total > kb2::current_sms() * 2048ll;                  // more than the GPU has threads: four pieces each are on their way at once
  const unsigned blocks = (unsigned)((total + (ahead ? 1023 : 255)) / (ahead ? 1024 : 256));
  auto kern = cache->fmt == KV_E4M3 ? (dt ? (ahead ? kv_read_kernel<KV_E4M3, false, 4> : kv_read_kernel<KV_E4M3, false, 1>)
                                          : (ahead ? kv_read_kernel<KV_E4M3, true, 4> : kv_read_kernel<KV_E4M3, true, 1>))
                                    : (dt ? (ahead ? kv_read_kernel<KV_INT8, false, 4> : kv_read_kernel<KV_INT8, false, 1>)
                                          : (ahead ? kv_read_kernel<KV_INT8, true, 4> : kv_read_kernel<KV_INT8, true, 1>));
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
  if (cache->layers > 65535 * kKeepLayers) return failf(KB2SEQ_ERR_VALUE, "kv_keep: too many layers");
  OnDevice on(step->device);
  SEQ_CUDA(on.err);
  kb2::launch_pdl(kv_keep_kernel, dim3(t.S, (cache->layers + kKeepLayers - 1) / kKeepLayers), 256, 0, (cudaStream_t)stream, c, cache->layers, t, path, P);
  SEQ_LAUNCHED();
  return KB2SEQ_OK;
}

}  // extern "C"
