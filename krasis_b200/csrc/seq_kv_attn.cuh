// Attention over the 8-bit cache: what its three kernels and their join share.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "ptx.cuh"
#include "seq_kv.cuh"

namespace kb2seq {

constexpr float kLog2e = 1.4426950408889634f;

struct KvAttn {                              // what a call says beside the cache and the tables
  const void* q;
  long long ldq, hq;
  int dtq, H, window, first;
  bool vec;                                  // four numbers of a query at a time lie on whole addresses
  float scale;
  const float* sinks;
  void* out;
  int dt_out;
  int rows, per_seq;                         // rows (tokens times heads per kv head) a tile; per_seq: the tiles of each sequence where the step's bring as many tokens each, else 0
  int piece, pieces;                         // groups of 16 keys a piece; the most pieces of a tile
  // Partial results, an output of dv numbers and its maximum and sum each: of the rows (token, head) that are cut alone.  Sequences that are cut lie one behind the other, in
  // each its rows, in each row its pieces (KvParts).
  float *part_o, *part_ml;                   // [parts][dv] and [parts][2]
  int parts;
  bool cluster;                              // a tile's pieces are the blocks of a cluster, which joins them itself
  bool linear;                               // all tiles' keys in a row are cut evenly, wherever the ends lie: `pieces` is then the most that a tile may have,
  int2* counts;                              // and this, [tiles][G], how many it has and the chunk of its first.  A piece's results lie at number chunk + tile G + head, which
                                             // no two share (from piece to piece the chunk or the tile moves on), `rows` to each
};
struct KvParts {                             // of a sequence
  int first, pieces;                         // where they begin; of each row (one: nothing is cut)
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// bytes 0, 1 and bytes 2, 3 of a word of codes as pairs of fp16
template <int FMT>
__device__ __forceinline__ void codes_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (FMT == KV_E4M3) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
  } else {
    const uint32_t u = w ^ 0x80808080u;                      // 0 .. 255 for -128 .. 127: 0x6400 + u is the fp16 number 1024 + u
    const __half2 off = __half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));      // 1152
    uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), off), y = __hsub2(*reinterpret_cast<__half2*>(&b), off);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  }
}
__device__ __forceinline__ uint32_t f16_pair(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 f16_get(uint32_t p) { return __half22float2(*reinterpret_cast<const __half2*>(&p)); }
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// Whether token `tok` at position `pos` of a sequence (first token c0, n of them) sees its row j.
__device__ __forceinline__ bool kv_sees(const KvStep& t, const KvAttn& a, const KvSpan& span, int c0, int n, int tok, int pos, int j) {
  int spot = j;
  if (j >= span.base) {
    const int i = j - span.base;
    if (i >= n || !(t.bits[(long long)tok * t.words + (i >> 5)] >> (i & 31) & 1u)) return false;
    spot = t.positions[c0 + i];
  }
  return spot <= pos && (pos - spot < a.window || spot < a.first);
}
// The least and the most position of the tokens t0 .. t1: the first and the last of a portion; of a tree the least is any that is no more.  The most matters under a window.
__device__ __forceinline__ void kv_reach(const KvStep& t, const KvAttn& a, const KvSpan& span, int t0, int t1, int* least, int* most) {
  const bool tree = span.base < kKvNoWindow;
  *least = tree ? span.base : span.p0;
  *most = *least;
  if (a.window >= kKvNoWindow) return;
  *most = span.p1;
  if (tree) {
    for (int x = t0; x < t1; ++x) *most = max(*most, t.positions[x]);
  }
}

// Into how many pieces (at most) of how many groups the keys of a sequence's tiles are cut, by what its tokens see together.  Tiles on the tensor cores have them all alike.
__device__ __forceinline__ int kv_cut(const KvLayer& c, const KvStep& t, const KvAttn& a, int s, int* length) {
  const int c0 = t.cu[s], c1 = t.cu[s + 1];
  const int groups = c1 > c0 ? kv_span(c, t, s, c0, c1 - 1, a.window, a.first).groups() : 0;
  const int n = max(min((groups + a.piece - 1) / a.piece, a.pieces), 1);
  *length = a.rows <= 16 ? a.piece : (max((groups + n - 1) / n, 1) + 3) / 4 * 4;      // whole tiles of 64 keys
  return n;
}
// Where the parts of sequence `seq` begin, which is one of few rows.  One warp.
__device__ __forceinline__ int kv_parts_ahead(const KvLayer& c, const KvStep& t, const KvAttn& a, const KvKinds& kinds, int seq) {
  int ahead = 0, length;
  for (int s = threadIdx.x & 31; s < seq; s += 32) {
    const int n = kinds.on_tiles(s) ? 1 : kv_cut(c, t, a, s, &length);
    if (n > 1) ahead += (t.cu[s + 1] - t.cu[s]) * a.H * n;
  }
  return __reduce_add_sync(0xffffffffu, ahead);
}
// The (sequence, tile, piece) number `at`, the pieces of one sequence behind those of the one before, a piece's tiles together (they read the same keys), and the sequence's
// parts.  One warp; false behind the last.
__device__ __forceinline__ bool kv_find_piece(const KvLayer& c, const KvStep& t, const KvAttn& a, const KvKinds& kinds, int per, int at, int* seq, int* tile, int* piece,
                                              int* length, KvParts* parts) {
  const int lane = threadIdx.x & 31;
  int before = 0, ahead = 0;
  for (int s0 = 0; s0 < t.S; s0 += 32) {
    const int s = s0 + lane;
    int tiles = 0, len = 1, n = 0, cut = 1, take = 0;
    if (s < t.S) {
      const int tokens = t.cu[s + 1] - t.cu[s], have = tokens * per;
      tiles = have > 0 && kinds.on_tiles(s) ? (have + a.rows - 1) / a.rows : 0;
      if (tiles && a.pieces > 1) cut = kv_cut(c, t, a, s, &len);
      n = tiles * cut;
      if (cut > 1) take = tokens * a.H * cut;
    }
    int upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + upto > at);
    if (hit) {
      const int l = __ffs(hit) - 1, of = __shfl_sync(0xffffffffu, tiles, l), i = at - before - __shfl_sync(0xffffffffu, upto - n, l);
      *length = __shfl_sync(0xffffffffu, len, l);
      *seq = s0 + l;
      *piece = i / of;
      *tile = i - *piece * of;
      *parts = {ahead + __reduce_add_sync(0xffffffffu, lane < l ? take : 0), __shfl_sync(0xffffffffu, cut, l)};
      return true;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
    ahead += __reduce_add_sync(0xffffffffu, take);
  }
  return false;
}

// 2^e that brings a row's largest magnitude (its bits: top) below 2^15, and 2^-e.  Of a row of smallest numbers or one that is not finite both stay within fp32.
__device__ __forceinline__ void kv_row_scale(uint32_t top, float* up, float* down) {
  const int e = min(max(141 - (int)(top >> 23), -113), 100);
  *up = __uint_as_float((uint32_t)(127 + e) << 23);
  *down = __uint_as_float((uint32_t)(127 - e) << 23);
}

// Four numbers of the queries from `from` on, of which `left` are the row's (none or all four).  vec: addresses are whole in them.
__device__ __forceinline__ void query4(const KvAttn& a, long long from, int left, float (&x)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = 0.f;
  if (left <= 0) return;
  if (a.dtq) {
    const bf16* p = (const bf16*)a.q + from;
    if (a.vec) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      x[0] = __uint_as_float(v.x << 16);
      x[1] = __uint_as_float(v.x & 0xFFFF0000u);
      x[2] = __uint_as_float(v.y << 16);
      x[3] = __uint_as_float(v.y & 0xFFFF0000u);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = __bfloat162float(p[j]);
    }
  } else {
    const float* p = (const float*)a.q + from;
    if (a.vec) {
      const float4 v = *reinterpret_cast<const float4*>(p);
      x[0] = v.x;
      x[1] = v.y;
      x[2] = v.z;
      x[3] = v.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = p[j];
    }
  }
}

// Tiles on the tensor cores: 256 rows (seq_kv_pair.cu), 128 where tensor memory has no room for two outputs (seq_kv_tile.cu).
int kv_pair_attend(int fmt, const KvLayer& c, const KvStep& t, const KvAttn& a, const KvKinds& kinds, int tiles, cudaStream_t stream);
int kv_tile_attend(int fmt, const KvLayer& c, const KvStep& t, const KvAttn& a, const KvKinds& kinds, int tiles, cudaStream_t stream);
inline bool kv_pairs(int d, int dv) { return d <= 192 && dv <= 128; }

}  // namespace kb2seq
