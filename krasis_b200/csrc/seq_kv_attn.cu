// Attention over the 8-bit cache (seq_kv.cu) for few query rows per key / value head: decoded tokens, short portions, small trees.
//
//   o = sum_j w_j v_j / (sum_j w_j + exp(sink)),  w_j = exp(scale q . k_j - max),  over the rows j that a token sees
//
// The H / G query heads of a kv head read the same rows, so a tile is 8 or 16 (token, head) pairs of one sequence and kv head, and a warp takes 16 keys at a time
// through mma.m16n8k16 in fp16, in which every code of both formats is exact: S = Q K^T with the queries as rows, then O^T = V^T P^T with the value columns as rows,
// so that S's accumulators are P's fragments where they stand, without a shuffle.  Dimensions and keys may be summed in any order, so a lane takes 16 neighbouring
// bytes of a key row and 8 or 16 of a value row for its fragments: everything a lane multiplies it has copied itself (cp.async into its own slots), no warp waits for
// another, and no byte is read from shared memory twice.
// What bounds it: the cache's bytes.  16 keys of 128 + 128 dimensions are 4.2 KB a warp and iteration; 3 stages x 16 warps an SM keep 200 KB on the way.  64 requests of 500 to
// 60000 rows, 64 / 4 heads of 128, int8 (862 MB, 131 us at the copy rate): 219 us, the copies alone 170 or so; 64 of 12000, 32 / 4 heads (811 MB) 182, the copies alone 162.
// What is left beside them is arithmetic on codes (a conversion is a half-rate instruction for two codes), which 16 query rows cannot hide behind four warps a scheduler; heads of
// 128 with 16 rows take all 128 registers of two blocks an SM and spill 60 bytes.
// Tried and left out: int8 keys as whole numbers (mma.s8 on queries of 15 bits: no conversion, no faster), the next keys' scores beside these keys' products (no faster).
//
// Rounding.  q: a row is scaled by a power of two to the top of fp16's range, bf16 numbers keep their 8 bits, fp32 ones are rounded to 11 (PARTS 1) or split into two
// fp16 numbers with 22 together (PARTS 2, for fp32 results).  Scores, maxima and sums are fp32; the key's scale multiplies the fp32 score.  The weight times the value's
// scale is rounded to fp16, relative to a reference R of its own that follows the largest such product (2^6 to 2^15 of it), so that small scales or weights do not
// fall out of fp16's range: 11 bits, or 22 with PARTS 2, down to 2^-30 of the largest.  R is never less than kLeastRef: where all values so far were zero, or weigh nothing
// beside a zero one, the next product that counts is above fp16's range and asks for a new R.
#include <cmath>

#include "seq_kv_attn.cuh"

namespace kb2seq {
namespace {

constexpr int kSWarps = 8, kSStages = 3, kSMostGroups = 768, kMostPieces = 1024, kMostTiles = 768, kClusterMost = 8;
constexpr float kLeastRef = 1e-37f;
constexpr int kPieceCost = 40;               // what a piece costs beside its keys, in groups of 16 (11 us against 0.25 a group, with two blocks on an SM)

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ void sts4(uint32_t a, uint32_t v) { asm volatile("st.shared.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory"); }
__device__ __forceinline__ void cp_async8(uint32_t to, const void* from, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(in ? 8 : 0) : "memory");
}
// DU, VU: units of 64 of d and dv.
template <int DU, int VU, int NQ, int PARTS>
struct StreamShape {
  static constexpr int MT = 8 * NQ;
  static constexpr int VB = VU % 2 ? 8 : 16, VC = VU * 8 / VB;            // a lane's bytes of a value row: VC times VB
  static constexpr int kK = 2 * DU * 512, kV = 4 * VU * 256, kStage = kK + kV + 128;
  static constexpr bool kQShared = NQ == 2 || DU * 8 * PARTS > 32;      // registers of the queries; spilled ones cost more than those read again
  static constexpr int kQ = DU * 4 * PARTS * 2 * NQ * 128;
  static constexpr int kRow = VU * 64 + 8;                                // numbers from row to row of a warp's share at the end: 32 bytes apart in the banks
  static constexpr int kRing = kSWarps * kSStages * kStage, kShare = MT * (VU * 64 + 4) * 4, kRed = kSWarps * MT * kRow * 4 + kShare;      // kShare: what a block has for the others of its cluster
  static constexpr int kOffRow = kRing > kRed ? kRing : kRed, kOffStat = kOffRow + kSMostGroups * 4, kOffTok = kOffStat + kSWarps * MT * 4 * 4, kOffQ = kOffTok + MT * 16,
                       kOffScan = kOffQ + kQ, kOffParts = kOffScan + (kMostTiles + 4) * 4;
  static constexpr int kTotal = kOffParts + 16;
  static constexpr int kBlocks = 2 * (kTotal + 1024) <= 227 * 1024 ? 2 : 1;
  static_assert(kTotal <= 227 * 1024 && kOffQ % 16 == 0 && kStage % 16 == 0, "shared memory");
};

// Four numbers at this place in the shared memory of block `rank` of the cluster.
__device__ __forceinline__ float4 lds_of(const float* p, int rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(kb2::cluster_addr(p, rank)));
  return v;
}
// Eight columns of a row: finished (part < 0), or as a partial result with its maximum and sum.
__device__ __forceinline__ void store8(const KvLayer& c, const KvAttn& a, const float (&acc)[8], float top, float sum, long long row, int hd, int dim, int part) {
  float y[8];
  float by = 1.f;
  if (part >= a.parts) return;
  if (part < 0) {
    if (a.sinks != nullptr && top != -INFINITY) sum += ex2(fmaf(a.sinks[hd], kLog2e, -top));
    by = sum == 0.f ? 0.f : 1.f / sum;
  } else if (dim == 0) {
    *reinterpret_cast<float2*>(a.part_ml + 2ll * part) = make_float2(top, sum);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = acc[e] * by;
  if (part < 0 && a.dt_out) {
    *reinterpret_cast<uint4*>((bf16*)a.out + row * c.dv + dim) =
        make_uint4(kb2::bf16x2_bits_rn(y[1], y[0]), kb2::bf16x2_bits_rn(y[3], y[2]), kb2::bf16x2_bits_rn(y[5], y[4]), kb2::bf16x2_bits_rn(y[7], y[6]));
  } else {
    float4* to = reinterpret_cast<float4*>(part < 0 ? (float*)a.out + row * c.dv + dim : a.part_o + (long long)part * c.dv + dim);
    to[0] = make_float4(y[0], y[1], y[2], y[3]);
    to[1] = make_float4(y[4], y[5], y[6], y[7]);
  }
}

// FULL: d and dv are whole units, and every copy's address is one of two a lane has plus a constant.
template <int FMT, int DU, int VU, int NQ, int PARTS, bool FULL>
__global__ void __launch_bounds__(kSWarps * 32, (StreamShape<DU, VU, NQ, PARTS>::kBlocks)) kv_stream_kernel(KvLayer c, KvStep t, KvAttn a, const __grid_constant__ KvKinds kinds) {
  using L = StreamShape<DU, VU, NQ, PARTS>;
  constexpr int MT = L::MT, VB = L::VB, VC = L::VC, MV = VU * 4;         // MV: 16-row tiles of O^T
  extern __shared__ __align__(16) uint8_t smem[];
  kb2::pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, t4 = lane & 3;
  const int per = a.H / c.G;

  // Many keys and few tiles: the groups of all tiles and heads in a row, each tile's behind its kPieceCost, are cut into chunks of one length, one for each block that fits
  // the GPU at once, wherever a chunk's ends lie in a tile.  (Pieces of tiles: requests of 500 to 60000 rows left a quarter of the blocks idle.)
  int* prefix = reinterpret_cast<int*>(smem + L::kOffScan);                // of the tiles' costs
  const int tiles = a.per_seq * t.S;
  long long chunk = 0, all = 0, at_cost = 0, to_cost = 0, next_chunk = blockIdx.x;
  if (a.linear) {
    int before = 0, most = 0;
    int* part = reinterpret_cast<int*>(smem + L::kOffStat);
    for (int b = 0; b < tiles; b += kSWarps * 32) {
      const int x = b + threadIdx.x, q = x / a.per_seq, from = (x - q * a.per_seq) * MT;
      int cost = 0;
      if (x < tiles) {
        const int f = t.cu[q], have = (int)min((long long)(t.cu[q + 1] - f) * per - from, (long long)MT);
        if (have > 0) cost = kv_span(c, t, q, f + from / per, f + (from + have - 1) / per, a.window, a.first).groups() + kPieceCost;
      }
      most = max(most, cost);
      int upto = cost;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      __syncthreads();
      if (lane == 31) part[warp] = upto;
      __syncthreads();
      int ahead = before, whole = before;
      for (int w = 0; w < kSWarps; ++w) {
        ahead += w < warp ? part[w] : 0;
        whole += part[w];
      }
      if (x < tiles) prefix[x] = ahead + upto - cost;
      before = whole;
    }
    most = __reduce_max_sync(0xffffffffu, most);
    __syncthreads();
    if (lane == 0) part[warp] = most;
    if (threadIdx.x == 0) prefix[tiles] = before;
    __syncthreads();
    for (int w = 0; w < kSWarps; ++w) most = max(most, part[w]);
    all = (long long)before * c.G;
    // no tile has more than a.pieces pieces, and no piece more groups than there is room for
    chunk = min(max(max((all + gridDim.x - 1) / gridDim.x, (long long)(most + a.pieces - 2) / (a.pieces - 1)), 8ll), (long long)kSMostGroups);
    __syncthreads();
  }

  for (bool once = true;; once = false) {
  int s, tile, head, u0 = 0, u1 = 0, np = 0, z = blockIdx.z, number = 0;
  if (a.linear) {
    if (!once) __syncthreads();              // the last piece's shares have been read
    if (at_cost >= to_cost) {
      at_cost = next_chunk * chunk;
      if (at_cost >= all) return;
      to_cost = min(at_cost + chunk, all);
      next_chunk += gridDim.x;
    }
    int lo = 0, hi = tiles;                  // the last tile that begins at or before this cost (of those without any, the one behind them)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((long long)prefix[mid] * c.G <= at_cost) lo = mid;
      else hi = mid;
    }
    number = lo;
    const int cost = prefix[lo + 1] - prefix[lo];
    const long long begin = (long long)prefix[lo] * c.G, mine = begin + (at_cost - begin) / cost * cost, stop = min(mine + cost, to_cost);
    head = (int)((at_cost - begin) / cost);
    u0 = (int)max(at_cost - mine - kPieceCost, 0ll);
    u1 = (int)max(stop - mine - kPieceCost, 0ll);
    const bool start = at_cost == mine;
    at_cost = stop;
    const int groups = cost - kPieceCost;
    if (groups == 0 ? !start : u1 == u0) continue;
    const long long first = (mine + kPieceCost) / chunk;
    np = groups == 0 ? 1 : (int)((mine + kPieceCost + groups - 1) / chunk - first) + 1;
    z = groups == 0 ? 0 : (int)(next_chunk - gridDim.x - first);
    s = number / a.per_seq;
    tile = number - s * a.per_seq;
    if (z == 0 && threadIdx.x == 0) a.counts[number * c.G + head] = make_int2(np, (int)first);
  } else {
    if (!once) return;
    head = blockIdx.y;
    if (a.per_seq) {
      s = blockIdx.x / a.per_seq;
      tile = blockIdx.x - s * a.per_seq;
    } else if (!kv_find_tile(t, kinds, per, MT, blockIdx.x, &s, &tile)) {
      return;
    }
  }
  const int c0 = t.cu[s], n = t.cu[s + 1] - c0, r0 = tile * MT, nr = (int)min((long long)n * per - r0, (long long)MT);
  if (nr <= 0) return;
  const int t0 = c0 + r0 / per, t1 = c0 + (r0 + nr - 1) / per;

  // queries: row r of the tile is head `r0 + r` mod per of a token.  kT threads have eight numbers each of a row (those of a row are neighbours in a warp); asked for first, as
  // everything else waits for the tables
  constexpr int kT = kSWarps * 32 / MT, kEach = (DU * 8 + kT - 1) / kT;
  const int qr = threadIdx.x / kT, qx = threadIdx.x % kT;
  float x[kEach][8];
  {
    const bool in = qr < nr;
    const int rr = r0 + (in ? qr : 0), tk = c0 + rr / per, hd = head * per + rr % per;
    const long long from = tk * a.ldq + hd * a.hq;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int e = (qx + i * kT) * 8;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        float y[4];
        query4(a, from + e + 4 * b, in ? c.d - e : 0, y);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[i][4 * b + j] = y[j];
      }
    }
    if (qx == 0) *reinterpret_cast<int2*>(smem + L::kOffTok + qr * 16) = make_int2(tk, in ? t.positions[tk] : -1);
  }
  const KvSpan span = kv_span(c, t, s, t0, t1, a.window, a.first);
  if (!a.linear) {
    const int total = span.groups();
    np = a.cluster ? a.pieces : min((total + a.piece - 1) / a.piece, a.pieces);
    if (z > 0 && z >= np) return;
    u0 = min(z * a.piece, total);
    u1 = min(total, u0 + a.piece);           // z = 0 of nothing to see: no group
  }

  // where the piece's groups lie: a row of this head in units of 16, or -1
  int* rows = reinterpret_cast<int*>(smem + L::kOffRow);
  for (int i = threadIdx.x; i < u1 - u0; i += kSWarps * 32) {
    const long long r = kv_row(c, t, s, span.group(u0 + i) * kKvGroup);
    rows[i] = r < 0 ? -1 : (int)((r + ((long long)head << c.lps)) / kKvGroup);
  }
  // the queries as fragments: of a lane's 16 numbers of a unit, four products with four each
  {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[i][j]) & 0x7FFFFFFFu);
#pragma unroll
    for (int o = kT / 2; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    float up, down;
    kv_row_scale(top, &up, &down);
    if (qx == 0) *reinterpret_cast<float*>(smem + L::kOffTok + qr * 16 + 8) = a.scale * kLog2e * down;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int e = (qx + i * kT) * 8;
      if (e >= DU * 64) continue;
      const int at = (e >> 6) * 4 + ((e & 15) >> 2), to = (qr & 7) * 4 + ((e & 63) >> 4);        // product, lane
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const float y0 = x[i][4 * k + 2 * b] * up, y1 = x[i][4 * k + 2 * b + 1] * up;
          uint32_t p[PARTS];
          p[0] = f16_pair(y0, y1);
          if constexpr (PARTS == 2) {
            const float2 f = f16_get(p[0]);
            p[1] = f16_pair(y0 - f.x, y1 - f.y);
          }
#pragma unroll
          for (int o = 0; o < PARTS; ++o) sts4(kb2::smem_u32(smem) + L::kOffQ + ((((at + k) * PARTS + o) * 32 + to) * 2 * NQ + b * NQ + (qr >> 3)) * 4, p[o]);
        }
    }
  }
  __syncthreads();

  const uint32_t ring = kb2::smem_u32(smem) + warp * (kSStages * L::kStage);
  const int d = FULL ? 64 * DU : c.d, dv = FULL ? 64 * VU : c.dv;
  const uint8_t *k_lane = c.k + (4 * (g8 >> 1) + (g8 & 1)) * d + 16 * t4, *v_lane = c.v + 4 * t4 * dv + VB * g8;
  const float* s_lane = (lane < 4 ? c.ks : c.vs) + 4 * (lane & 3);
  const auto issue = [&](int u, int st) {
    if (u < u1) {
      const int r16 = rows[u - u0];
      if (r16 >= 0) {
        const uint32_t to = ring + st * L::kStage;
        const uint8_t *k = k_lane + (long long)r16 * (kKvGroup * d), *v = v_lane + (long long)r16 * (kKvGroup * dv);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < DU; ++i) {
            const bool in = FULL || 64 * i + 16 * t4 < d;
            cp_async16_stream(to + ((j * DU + i) * 32 + lane) * 16, k + 2 * j * d + (in ? 64 * i : -16 * t4), in);
          }
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int i = 0; i < VC; ++i) {
            const bool in = FULL || (8 * i + g8) * VB < dv;
            const uint32_t at = to + L::kK + ((x * VC + i) * 32 + lane) * VB;
            const uint8_t* from = v + x * dv + (in ? 8 * i * VB : -VB * g8);
            if constexpr (VB == 16) cp_async16_stream(at, from, in);
            else cp_async8(at, from, in);
          }
        if (lane < 8) cp_async16_stream(to + L::kK + L::kV + lane * 16, s_lane + (long long)r16 * kKvGroup, true);
      }
    }
    kb2::cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kSStages; ++i) issue(u0 + warp + i * kSWarps, i);

  // where this piece's results go, those of row 0 of the tile (an even cut) or of the sequence, and how far apart rows are; looked up while the first keys are on their way
  KvParts* mine = reinterpret_cast<KvParts*>(smem + L::kOffParts);
  if (warp == 0 && !a.cluster) {
    KvParts parts{-1, 1};
    int length;
    if (np > 1 && a.linear) parts.first = ((int)next_chunk - gridDim.x + number * c.G + head) * MT;
    else if (np > 1) parts = {kv_parts_ahead(c, t, a, kinds, s) + z, nr == n * per ? np : kv_cut(c, t, a, s, &length)};
    if (lane == 0) *mine = parts;
  }

  constexpr int QR = L::kQShared ? 1 : DU * 4;
  uint32_t qf[QR][PARTS][2 * NQ];
  if constexpr (!L::kQShared) {
#pragma unroll
    for (int i = 0; i < DU * 4; ++i)
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
        const uint2 v = lds8(kb2::smem_u32(smem) + L::kOffQ + ((i * PARTS + p) * 32 + lane) * 8);
        qf[i][p][0] = v.x;
        qf[i][p][1] = v.y;
      }
  }
  float rf[NQ];
  int pos[NQ], tok[NQ];
  float m[NQ], l[NQ], ref[NQ], inv[NQ];
#pragma unroll
  for (int h = 0; h < NQ; ++h) {
    const int4 v = *reinterpret_cast<const int4*>(smem + L::kOffTok + (g8 + 8 * h) * 16);
    tok[h] = v.x;
    pos[h] = v.y;
    rf[h] = __int_as_float(v.z);
    m[h] = -INFINITY;
    l[h] = 0.f;
    ref[h] = kLeastRef;
    inv[h] = 1.f / kLeastRef;
  }
  int pmin, pmax;
  kv_reach(t, a, span, t0, t1, &pmin, &pmax);

  float o[MV][NQ][4];
#pragma unroll
  for (int i = 0; i < MV; ++i)
#pragma unroll
    for (int h = 0; h < NQ; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][h][e] = 0.f;

  const auto sees = [&](int j, int h) { return g8 + 8 * h < nr && kv_sees(t, a, span, c0, n, tok[h], pos[h], j); };      // row h of the lane, position j

  int st = 0;
  for (int u = u0 + warp; u < u1; u += kSWarps) {
    kb2::cp_async_wait<kSStages - 1>();
    __syncwarp();
    const uint32_t at = ring + st * L::kStage;
    if (rows[u - u0] >= 0) {
      const int key0 = span.group(u) * kKvGroup;
      float sc[2][4] = {};
#pragma unroll
      for (int i = 0; i < DU; ++i) {
        const uint4 k0 = lds16(at + (i * 32 + lane) * 16), k1 = lds16(at + ((DU + i) * 32 + lane) * 16);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t b[2][2];
          codes_f16<FMT>(word(k0, k), b[0][0], b[0][1]);
          codes_f16<FMT>(word(k1, k), b[1][0], b[1][1]);
#pragma unroll
          for (int p = 0; p < PARTS; ++p) {
            uint32_t x[2 * NQ];              // [dimensions 0, 1 | 8, 9 of the product][row]
            if constexpr (L::kQShared) {
              const uint32_t qa = kb2::smem_u32(smem) + L::kOffQ + (((i * 4 + k) * PARTS + p) * 32 + lane) * 8 * NQ;
              if constexpr (NQ == 2) {
                const uint4 v = lds16(qa);
                x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
              } else {
                const uint2 v = lds8(qa);
                x[0] = v.x; x[1] = v.y;
              }
            } else {
#pragma unroll
              for (int e = 0; e < 2 * NQ; ++e) x[e] = qf[i * 4 + k][p][e];
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) mma_f16(sc[j], x[0], NQ == 2 ? x[1] : 0u, x[NQ], NQ == 2 ? x[NQ + 1] : 0u, b[j][0], b[j][1]);
          }
        }
      }
      const uint4 kq = lds16(at + L::kK + L::kV + t4 * 16), vq = lds16(at + L::kK + L::kV + 64 + t4 * 16);
      // all rows of the tile see all 16 keys
      const bool all = key0 + kKvGroup <= span.base && key0 + kKvGroup - 1 <= pmin && (pmax - key0 < a.window || key0 + kKvGroup <= a.first);
      float y[NQ][4], p[NQ][4];              // scores in powers of two, weights
      uint32_t w[NQ][PARTS][2];
#pragma unroll
      for (int h = 0; h < NQ; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) y[h][e] = sc[e >> 1][2 * h + (e & 1)] * (__uint_as_float(word(kq, e)) * rf[h]);
      if (!all) {
#pragma unroll
        for (int h = 0; h < NQ; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!sees(key0 + 4 * t4 + e, h)) y[h][e] = -INFINITY;
      }
      const auto weigh = [&](int h) {        // against the row's maximum and reference: the largest of the lane's scores and products over them
        float top = -INFINITY, big = 0.f;
        const float from = m[h] == -INFINITY ? 0.f : m[h];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float z = y[h][e] - from;
          p[h][e] = ex2(z);
          top = fmaxf(top, z);
        }
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = p[h][e] * __uint_as_float(word(vq, e)) * inv[h];          // the scale not times 1 / R first: that may be infinite, and the weight zero
          if (!all && y[h][e] == -INFINITY) x[e] = 0.f;                    // a row that nobody sees may hold anything
          big = fmaxf(big, x[e]);
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          w[h][0][b] = f16_pair(x[2 * b], x[2 * b + 1]);
          if constexpr (PARTS == 2) {
            const float2 f = f16_get(w[h][0][b]);
            w[h][PARTS - 1][b] = f16_pair(x[2 * b] - f.x, x[2 * b + 1] - f.y);
          }
        }
        return top > 8.f || big > 32768.f;   // a weight above 2^8, a product above fp16's range
      };
      bool again = false;
#pragma unroll
      for (int h = 0; h < NQ; ++h) again |= weigh(h) || m[h] == -INFINITY;
      if (__any_sync(0xffffffffu, again)) {  // seldom after the first keys: maxima and references anew
        float grow[NQ];
#pragma unroll
        for (int h = 0; h < NQ; ++h) {
          float top = fmaxf(fmaxf(y[h][0], y[h][1]), fmaxf(y[h][2], y[h][3]));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const float mn = fmaxf(m[h], top), from = mn == -INFINITY ? 0.f : mn, back = ex2(m[h] - from);
          m[h] = mn;
          l[h] *= back;
          ref[h] *= back;
          float big = 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (y[h][e] != -INFINITY) big = fmaxf(big, ex2(y[h][e] - from) * __uint_as_float(word(vq, e)));
          big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
          big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
          const float r = fmaxf(big > ref[h] * 32768.f ? big * 0.015625f : ref[h], kLeastRef);
          grow[h] = ref[h] / r;
          ref[h] = r;
          inv[h] = 1.f / r;
          weigh(h);
        }
#pragma unroll
        for (int h = 0; h < NQ; ++h) {       // the columns of O^T that a lane holds are the rows 2 t4, 2 t4 + 1 of the queries
          const float f0 = __shfl_sync(0xffffffffu, grow[h], 8 * t4), f1 = __shfl_sync(0xffffffffu, grow[h], 8 * t4 + 4);
#pragma unroll
          for (int i = 0; i < MV; ++i) {
            o[i][h][0] *= f0;
            o[i][h][1] *= f1;
            o[i][h][2] *= f0;
            o[i][h][3] *= f1;
          }
        }
      }
#pragma unroll
      for (int h = 0; h < NQ; ++h) l[h] += (p[h][0] + p[h][1]) + (p[h][2] + p[h][3]);
#pragma unroll
      for (int i = 0; i < VC; ++i) {
        uint32_t v[4][VB / 4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t va = at + L::kK + ((k * VC + i) * 32 + lane) * VB;
          if constexpr (VB == 16) {
            const uint4 q = lds16(va);
            v[k][0] = q.x; v[k][1] = q.y; v[k][2] = q.z; v[k][VB / 4 - 1] = q.w;
          } else {
            const uint2 q = lds8(va);
            v[k][0] = q.x; v[k][1] = q.y;
          }
        }
#pragma unroll
        for (int x = 0; x < VB / 4; ++x)
#pragma unroll
          for (int b = 0; b < 2; ++b) {      // bytes 2 b, 2 b + 1 of the word: rows g8 and g8 + 8 of a tile of O^T
            uint32_t a0, a1, a2, a3;
            codes_f16<FMT>(__byte_perm(v[0][x], v[1][x], b ? 0x7362 : 0x5140), a0, a1);
            codes_f16<FMT>(__byte_perm(v[2][x], v[3][x], b ? 0x7362 : 0x5140), a2, a3);
#pragma unroll
            for (int h = 0; h < NQ; ++h)
#pragma unroll
              for (int p = 0; p < PARTS; ++p) mma_f16(o[i * (VB / 2) + 2 * x + b][h], a0, a1, a2, a3, w[h][p][0], w[h][p][1]);
          }
      }
    }
    __syncwarp();
    issue(u + kSStages * kSWarps, st);
    st = st + 1 == kSStages ? 0 : st + 1;
  }
  kb2::cp_async_wait<0>();

  // the warps' shares, joined in their order
  float4* stat = reinterpret_cast<float4*>(smem + L::kOffStat);            // [warp][row]: maximum, sum, reference
#pragma unroll
  for (int h = 0; h < NQ; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    if (t4 == 0) stat[warp * MT + g8 + 8 * h] = make_float4(m[h], l[h], ref[h], 0.f);
  }
  __syncthreads();                           // the rings are free from here on
  float* red = reinterpret_cast<float*>(smem);                             // [warp][row][tile of O^T][g8][2]
#pragma unroll
  for (int h = 0; h < NQ; ++h)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int q = 8 * h + 2 * t4 + e;
#pragma unroll
      for (int i = 0; i < MV; ++i) *reinterpret_cast<float2*>(red + (warp * MT + q) * L::kRow + (i * 8 + g8) * 2) = make_float2(o[i][h][e], o[i][h][2 + e]);
    }
  __syncthreads();
  // a thread takes eight columns of a row
  constexpr int kCols = VU * 8;
  for (int i = threadIdx.x; i < MT * kCols; i += kSWarps * 32) {
    const int q = i / kCols, dim = (i - q * kCols) * 8;
    // the eight columns are the pairs of four tiles of O^T, of one lane each
    const int from = VB == 16 ? ((dim >> 7) * 8 + (dim >> 3 & 1) * 4) * 16 + ((dim & 127) >> 4) * 2 : (dim >> 6) * 64 + ((dim & 63) >> 3) * 2;
    if (q >= nr || dim >= c.dv) continue;
    float top = -INFINITY, sum = 0.f, acc[8] = {};
#pragma unroll
    for (int w = 0; w < kSWarps; ++w) top = fmaxf(top, stat[w * MT + q].x);
#pragma unroll
    for (int w = 0; w < kSWarps; ++w) {
      const float4 x = stat[w * MT + q];
      const float g = x.x == -INFINITY ? 0.f : ex2(x.x - top), f = x.z * g;
      sum += x.x == -INFINITY ? x.y : x.y * g;                             // a sum without a maximum is 0, or NaN from a row that holds one
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 v = *reinterpret_cast<const float2*>(red + (w * MT + q) * L::kRow + from + 16 * e);
        acc[2 * e] = fmaf(v.x, f, acc[2 * e]);
        acc[2 * e + 1] = fmaf(v.y, f, acc[2 * e + 1]);
      }
    }
    if (a.cluster) {                         // the tile's pieces are the blocks of a cluster: they meet in shared memory
      float* share = red + kSWarps * MT * L::kRow + q * (VU * 64 + 4);
      *reinterpret_cast<float4*>(share + dim) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      *reinterpret_cast<float4*>(share + dim + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
      if (dim == 0) *reinterpret_cast<float4*>(share + VU * 64) = make_float4(top, sum, 0.f, 0.f);
      continue;
    }
    const int hd = head * per + (r0 + q) % per;
    const int row = (r0 + q) / per * a.H + hd;                             // of the sequence
    const KvParts parts = *mine;
    store8(c, a, acc, top, sum, (long long)c0 * a.H + row, hd, dim, parts.first < 0 ? -1 : parts.first + (a.linear ? q : row * parts.pieces));
  }
  if (a.cluster) {
    kb2::cluster_sync_all();
    const int rank = (int)kb2::cluster_rank(), i = threadIdx.x * np + rank, q = i / kCols, dim = (i - q * kCols) * 8;
    if (q < nr && dim < c.dv) {
      const float* share = red + kSWarps * MT * L::kRow + q * (VU * 64 + 4);
      float top = -INFINITY, sum = 0.f, acc[8] = {};
      float4 ml[kClusterMost], v[kClusterMost][2];                         // all asked for at once: one after another they took half of a small call's time
#pragma unroll
      for (int b = 0; b < kClusterMost; ++b) {
        const int of = min(b, np - 1);
        ml[b] = lds_of(share + VU * 64, of);
        v[b][0] = lds_of(share + dim, of);
        v[b][1] = lds_of(share + dim + 4, of);
      }
#pragma unroll
      for (int b = 0; b < kClusterMost; ++b) top = fmaxf(top, ml[b].x);
#pragma unroll
      for (int b = 0; b < kClusterMost; ++b) {
        if (b >= np) continue;
        const float f = ml[b].x == -INFINITY ? 1.f : ex2(ml[b].x - top);   // a piece without a maximum holds zeros, or NaN
        sum += ml[b].y * f;
        acc[0] = fmaf(v[b][0].x, f, acc[0]);
        acc[1] = fmaf(v[b][0].y, f, acc[1]);
        acc[2] = fmaf(v[b][0].z, f, acc[2]);
        acc[3] = fmaf(v[b][0].w, f, acc[3]);
        acc[4] = fmaf(v[b][1].x, f, acc[4]);
        acc[5] = fmaf(v[b][1].y, f, acc[5]);
        acc[6] = fmaf(v[b][1].z, f, acc[6]);
        acc[7] = fmaf(v[b][1].w, f, acc[7]);
      }
      store8(c, a, acc, top, sum, (long long)(c0 + (r0 + q) / per) * a.H + head * per + (r0 + q) % per, head * per + (r0 + q) % per, dim, -1);
    }
    kb2::cluster_sync_all();                 // nobody leaves while its share is read
  }
  }
}

// The pieces of a row (token, head), joined in a fixed order; rows that one piece finished are left alone.  x, y: sequences of few rows, and those on tiles.  W warps a row take the pieces in
// turn, four of a warp's on their way at once (one at a time 64 pieces took 27 us).  One request of 30000 rows, 16 / 2 heads: four warps a row 17 us in all, one 38 at the time;
// 62000 rows of few pieces: four warps 50 us more than one.  `rows`: of the sequences that are cut, one behind the other.
template <int W>
__global__ void __launch_bounds__(128) kv_join_kernel(KvLayer c, KvStep t, KvAttn x, KvAttn y, const __grid_constant__ KvKinds kinds, int rows) {
  __shared__ float weights[W > 1 ? kMostPieces : 4 * 32];
  __shared__ __align__(16) float share[3][256];
  __shared__ float total[4];
  kb2::pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wr = warp % W, at = wr * 32 + lane;
  int at_row = (int)(blockIdx.x * (4 / W) + warp / W);
  float* weight = weights + (W > 1 ? 0 : warp * 32);
  const auto meet = [&] {
    if (W > 1) __syncthreads();
    else __syncwarp();
  };
  if (at_row >= rows) return;
  int s = -1, length = 1;
  KvParts parts{};
  if (x.linear) {                            // all sequences are
    const int tok = at_row / x.H;
    if (tok >= t.cu[t.S]) return;
    s = t.seq_of[tok];
    at_row -= t.cu[s] * x.H;
  } else {
    int before = 0, ahead[2] = {};           // parts of sequences of few rows, of those on tiles
    for (int s0 = 0; s0 < t.S; s0 += 32) {
      const int q = s0 + lane;
      const bool tiles = q < t.S && kinds.on_tiles(q);
      const KvAttn& z = tiles ? y : x;
      int cut = 1, len = 1;
      if (q < t.S && z.pieces > 1 && !z.cluster) cut = kv_cut(c, t, z, q, &len);
      const int n = cut > 1 ? (t.cu[q + 1] - t.cu[q]) * x.H : 0;
      int upto = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + upto > at_row);
      const int l = hit ? __ffs(hit) - 1 : 32;
      const bool kind = __shfl_sync(0xffffffffu, tiles, l & 31);
#pragma unroll
      for (int k = 0; k < 2; ++k) ahead[k] += __reduce_add_sync(0xffffffffu, lane < l && tiles == (k == 1) ? n * cut : 0);
      if (hit) {
        s = s0 + l;
        parts = {kind ? ahead[1] : ahead[0], __shfl_sync(0xffffffffu, cut, l)};
        length = __shfl_sync(0xffffffffu, len, l);
        at_row -= before + __shfl_sync(0xffffffffu, upto - n, l);
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (s < 0) return;
  }
  const int per = x.H / c.G, c0 = t.cu[s], n = t.cu[s + 1] - c0, tok = c0 + at_row / x.H, hd = at_row % x.H;
  const long long row = (long long)tok * x.H + hd;
  const KvAttn& a = kinds.on_tiles(s) ? y : x;
  const int in_seq = (tok - c0) * per + hd % per, r0 = in_seq / a.rows * a.rows, nr = (int)min((long long)n * per - r0, (long long)a.rows);
  const KvSpan span = kv_span(c, t, s, c0 + r0 / per, c0 + (r0 + nr - 1) / per, a.window, a.first);
  int np = min((span.groups() + length - 1) / length, a.pieces), step = 1, p0 = parts.first + at_row * parts.pieces;
  if (a.linear) {
    const int number = (s * a.per_seq + r0 / a.rows) * c.G + hd / per;
    const int2 v = a.counts[number];
    np = v.x;
    step = a.rows;
    p0 = (v.y + number) * step + in_seq - r0;
  }
  if (np <= 1 || p0 < 0 || p0 + (long long)(np - 1) * step >= a.parts) return;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + p0;
  float top = -INFINITY, sum = 0.f;
  for (int i = at; i < np; i += 32 * W) top = fmaxf(top, ml[i * step].x);
  top = warp_max(top);
  if (W > 1) {
    if (lane == 0) total[warp] = top;
    meet();
    top = fmaxf(fmaxf(total[0], total[1]), fmaxf(total[2], total[3]));
    meet();
  }
  for (int i = at; i < np; i += 32 * W) {
    const float2 v = ml[i * step];
    const bool none = v.x == -INFINITY;      // a piece without a maximum holds zeros, or NaN
    weight[i] = none ? 1.f : ex2(v.x - top);
    sum += none ? v.y : v.y * weight[i];
  }
  sum = warp_sum(sum);
  if (W > 1 && lane == 0) total[warp] = sum;
  meet();
  if (W > 1) sum = (total[0] + total[1]) + (total[2] + total[3]);
  float acc[2][4] = {};
  for (int i0 = wr; i0 < np; i0 += 4 * W) {
    float4 v[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        v[i][h] = i0 + W * i < np && h * 128 + lane * 4 < c.dv ? *reinterpret_cast<const float4*>(a.part_o + (long long)(p0 + (i0 + W * i) * step) * c.dv + h * 128 + lane * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float f = i0 + W * i < np ? weight[i0 + W * i] : 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        acc[h][0] = fmaf(v[i][h].x, f, acc[h][0]);
        acc[h][1] = fmaf(v[i][h].y, f, acc[h][1]);
        acc[h][2] = fmaf(v[i][h].z, f, acc[h][2]);
        acc[h][3] = fmaf(v[i][h].w, f, acc[h][3]);
      }
    }
  }
  if (W > 1 && warp) {
#pragma unroll
    for (int h = 0; h < 2; ++h) *reinterpret_cast<float4*>(&share[warp - 1][h * 128 + lane * 4]) = make_float4(acc[h][0], acc[h][1], acc[h][2], acc[h][3]);
  }
  meet();
  if (wr) return;
  if (a.sinks != nullptr && top != -INFINITY) sum += ex2(fmaf(a.sinks[hd], kLog2e, -top));
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int e = h * 128 + lane * 4;
    if (e >= c.dv) continue;
#pragma unroll
    for (int w = 0; w < W - 1; ++w) {
      const float4 v = *reinterpret_cast<const float4*>(&share[w][e]);
      acc[h][0] += v.x;
      acc[h][1] += v.y;
      acc[h][2] += v.z;
      acc[h][3] += v.w;
    }
    if (a.dt_out) {
      *reinterpret_cast<uint2*>((bf16*)a.out + row * c.dv + e) = make_uint2(kb2::bf16x2_bits_rn(acc[h][1] * inv, acc[h][0] * inv), kb2::bf16x2_bits_rn(acc[h][3] * inv, acc[h][2] * inv));
    } else {
      *reinterpret_cast<float4*>((float*)a.out + row * c.dv + e) = make_float4(acc[h][0] * inv, acc[h][1] * inv, acc[h][2] * inv, acc[h][3] * inv);
    }
  }
}

// ------------------------------------------------------------------------------------------------ host
// Rows per kv head (a sequence's tokens times the heads that share one) from which a sequence may run on the tensor cores' tiles.  Fewer are faster on the kernel for few rows
// (us there / on tiles, 16 / 2 heads of 128, int8: 24 rows after 2000 keys 13 / 20, eight sequences of 32 rows after 16000 51 / 62, of 48 after 30000 106 / 120); more are where
// there is enough to do to make up for the tiles' longer start (64 rows after 2000 13 / 23, eight of 64 after 30000 133 / 123; 128 rows after 2000 18 / 25, after 30000 49 / 34).
// One rule for all heads, made for those of 128; for others both kernels cost more a group.  Of 48 to 512 rows, one sequence or eight, after 2000, 8000 and 30000 keys it loses at
// most 14 % of the better kernel's time on heads of 128, 34 % on 192 / 128 (256 rows after 8000: 47 / 35), 27 % on 128 / 256 and 21 % on 256.
constexpr int kTileFrom = 48;
constexpr long long kWideWaves = 2;          // pieces for each SM, of such sequences (sixteen trees of 57 to 64 tokens: 2 530 us, 3 548, 4 571, 6 638)
// How the sequences of one kind are cut: into tiles of rows, and the keys that a tile sees (in groups of 16) into pieces.
struct KvPlan {
  int rows, tiles, per_seq, piece, pieces, blocks;                         // blocks: of the even cut (0 for pieces of tiles); of tiles on the tensor cores, pieces and all
  bool cluster;                              // the pieces of a tile are a cluster, which joins them itself
  long long parts, joined;                   // partial results; rows (token, head) of the sequences that are cut
  size_t floats;                             // workspace
  void size(int G, int dv, bool wide) {      // what lies behind begins on 16 bytes too
    floats = ((size_t)parts * (dv + 2) + (blocks && !wide ? 2 * (size_t)tiles * G : 0) + 3) / 4 * 4;
  }
};
// The most groups of 16 that the tokens start .. start + n - 1 see.
inline long long groups_seen(long long start, long long n, int window, int first) {
  const long long lo = window < kKvNoWindow ? std::max(0ll, start - window + 1) : 0;
  return (start + n - lo + 30) / 16 + (std::min<long long>(first, lo) + 15) / 16;
}
KvPlan kv_plan(const kb2_seq_kv_cache* cache, const kb2_seq_kv_step* step, int H, int window, int first, const KvKinds& kinds, bool wide) {
  KvPlan p{};
  const int per = H / cache->G;
  long long top = 0, work = 0, rows = 0;
  bool same = true;
  for (int s = 0; s < step->S; ++s) {
    const long long r = (long long)step->layout[4 * s + 1] * per;
    if (kinds.on_tiles(s) == wide) rows = std::max(rows, r);
  }
  p.rows = wide ? (kv_pairs(cache->d, cache->dv) ? 256 : 128) : rows <= 8 ? 8 : 16;
  const auto tiles = [&](int s) {            // of a sequence of this kind
    const long long r = (long long)step->layout[4 * s + 1] * per;
    return kinds.on_tiles(s) == wide ? (r + p.rows - 1) / p.rows : 0ll;
  };
  const auto seen = [&](int s) {             // captured launches are run again with later positions: what the page lists hold
    const int* l = step->layout + 4 * s;
    const long long end = step->replayed ? (long long)step->max_pages * cache->page_size : (long long)l[2] + l[1];
    return groups_seen(end - l[1], l[1], window, first);
  };
  for (int s = 0; s < step->S; ++s) {
    same = same && step->layout[4 * s + 1] == step->layout[1];
    const long long n = tiles(s);
    if (n == 0) continue;
    p.tiles += (int)n;
    top = std::max(top, seen(s));
    work += seen(s) * n;
  }
  if (p.tiles == 0) return p;
  p.per_seq = same ? p.tiles / step->S : 0;
  const auto cut = [&](int s, long long n) { // into n pieces
    const long long rows = n > 1 ? (long long)step->layout[4 * s + 1] * H : 0;
    p.joined += rows;
    p.parts += rows * n;
  };
  long long piece;
  if (wide) {                                // one block an SM; a piece of at least four tiles of keys
    const long long want = kWideWaves * kb2::current_sms();
    piece = std::max((work * cache->G + want - 1) / want, std::max(16ll, (top + 63) / 64));
    if ((long long)p.tiles * cache->G >= 2ll * kb2::current_sms() && same) piece = top;
    p.piece = (int)std::max(piece, 8ll);
    p.pieces = (int)std::max(1ll, (top + p.piece - 1) / p.piece);
    for (int s = 0; s < step->S; ++s) {
      const long long n = tiles(s) ? std::max(1ll, (seen(s) + p.piece - 1) / p.piece) : 0;
      p.blocks += (int)(tiles(s) * n);
      cut(s, n);
    }
    p.size(cache->G, cache->dv, wide);
    return p;
  } else {
    // Blocks of one length in whole waves, as the last wave takes as long as the others: the length whose waves, with what a block costs beside its keys (some 16 groups), end
    // first.  A mixed fp32 step on heads of 256: 73 -> 61 us.
    const long long slots = (long long)kb2::current_sms() * (cache->d <= 128 && cache->dv <= 128 ? 2 : 1);
    const long long even = (work + (long long)p.tiles * kPieceCost) * cache->G / slots;
    if (p.per_seq && p.tiles <= kMostTiles && work * cache->G >= slots * kPieceCost) {
      p.blocks = (int)slots;
      // a captured step's keys may come to lie in one sequence: the kernel makes its pieces no more than this
      p.pieces = (int)(step->replayed ? std::max(34ll, (top + kPieceCost) / kSMostGroups + 2) : (top + kPieceCost) / std::min<long long>(std::max(even, 8ll), kSMostGroups) + 2);
    }
    // Few keys: up to eight blocks a tile meet in shared memory, without a second launch and a workspace (four requests of 1028 visible rows: 9.0 us, with a join 9.8; 11.0 against 15 with what the host does, as measured then);
    // more than that, a warp would have too many keys one after another (6144 a tile).
    if (!p.blocks && top > kSWarps && top <= 48 * kClusterMost && (long long)p.tiles * cache->G * kClusterMost <= slots) {
      p.cluster = true;
      p.pieces = (int)std::min<long long>(kClusterMost, (top + kSWarps - 1) / kSWarps);
      p.piece = (int)((top + p.pieces - 1) / p.pieces);
      if (p.piece <= kSMostGroups) return p;
      p.cluster = false;
    }
    long long best = 0, cost = 0;
    for (int waves = 1; waves <= 4; ++waves) {
      long long len = std::max<long long>((work * cache->G + waves * slots - 1) / (waves * slots), (top + 63) / 64);
      for (int tries = 0; tries < 8; ++tries) {
        len = std::max<long long>((len + kSWarps - 1) / kSWarps * kSWarps, kSWarps);
        if (len >= kSMostGroups) break;
        long long blocks = 0;
        for (int s = 0; s < step->S; ++s) blocks += seen(s) ? tiles(s) * ((seen(s) + len - 1) / len) : 0;
        if (blocks * cache->G <= waves * slots) break;
        len += std::max<long long>(len / 16, 1);
      }
      len = std::min<long long>(len, kSMostGroups);
      if (best == 0 || waves * (len + 16) < cost) {
        best = len;
        cost = waves * (len + 16);
      }
      if (len == kSWarps) break;
    }
    piece = best;
  }
  p.piece = (int)std::max(piece, 8ll);
  if (p.blocks) {                            // a chunk for each block, or each kSMostGroups groups where that is more; a piece ends a chunk or a tile of a head
    const long long all = (work + (long long)p.tiles * kPieceCost) * cache->G;
    p.parts = (std::max<long long>(p.blocks, (all + kSMostGroups - 1) / kSMostGroups) + (long long)p.tiles * cache->G) * p.rows;
    p.joined = (long long)step->T * H;
  } else {
    p.pieces = (int)std::max(1ll, (top + p.piece - 1) / p.piece);
    for (int s = 0; s < step->S; ++s) cut(s, tiles(s) ? (seen(s) + p.piece - 1) / p.piece : 0);
  }
  p.size(cache->G, cache->dv, wide);
  return p;
}
struct KvPlans {
  KvPlan few, many;
  KvKinds kinds;
  size_t bytes() const { return (few.floats + many.floats) * 4; }
};
KvPlans kv_plans(const kb2_seq_kv_cache* cache, const kb2_seq_kv_step* step, int H, int window, int first, int dt_out) {
  int split = 0x7FFFFFFF;                    // fp32 results carry 22 bits: the tiles have 11
  KvPlans p{};
  if (dt_out && step->tiles_from > 0) {
    split = step->tiles_from - 1;
  } else if (dt_out) {
    long long few = 0, many = 0;             // groups of 16 keys times tiles, either way
    const int per = H / cache->G, rows = kv_pairs(cache->d, cache->dv) ? 256 : 128;
    for (int s = 0; s < step->S; ++s) {
      const int* l = step->layout + 4 * s;
      const long long r = (long long)l[1] * per, end = step->replayed ? (long long)step->max_pages * cache->page_size : (long long)l[2] + l[1];
      if (r < kTileFrom) continue;
      const long long g = groups_seen(end - l[1], l[1], window, first) * cache->G;
      few += (r + 15) / 16 * g;
      many += (r + rows - 1) / rows * g;
    }
    // 0.27 us a group on one of two blocks an SM, 0.3 on the one of the tiles, and 8 us
    const long long sms = kb2::current_sms();
    if (few * 27 > 2 * (many * 30 + 800 * sms)) split = kTileFrom - 1;
  }
  // more than `split` rows: on tiles.  Of steps with more sequences than there are bits, neighbours are if all of them that have tokens do.
  KvKinds& kinds = p.kinds;
  int wide = 0, all = 0;
  if (split < 0x7FFFFFFF) {
    while ((step->S - 1) >> kinds.shift >= kKvKindBits) ++kinds.shift;
    for (int s0 = 0; s0 < step->S; s0 += 1 << kinds.shift) {
      int n = 0, on = 0;
      for (int s = s0; s < std::min(s0 + (1 << kinds.shift), step->S); ++s) {
        const long long r = (long long)step->layout[4 * s + 1] * (H / cache->G);
        n += r > 0;
        on += r > split;
      }
      all += n;
      if (on == 0 || on < n) continue;
      wide += on;
      kinds.on[s0 >> kinds.shift >> 5] |= 1u << (s0 >> kinds.shift & 31);
    }
    kinds.every = wide == 0 ? 0 : wide == all ? 1 : 2;
  }
  if (kinds.every != 1) p.few = kv_plan(cache, step, H, window, first, kinds, false);
  if (kinds.every) p.many = kv_plan(cache, step, H, window, first, kinds, true);
  return p;
}
inline KvAttn with_plan(KvAttn a, const KvPlan& p, float* work, int dv) {
  a.rows = p.rows;
  a.per_seq = p.per_seq;
  a.piece = p.piece;
  a.pieces = p.pieces;
  a.part_o = work;
  a.part_ml = work + (size_t)p.parts * dv;
  a.parts = (int)p.parts;
  a.linear = p.blocks > 0 && p.rows <= 16;
  a.cluster = p.cluster;
  a.counts = reinterpret_cast<int2*>(a.part_ml + 2 * (size_t)p.parts);
  return a;
}

template <int FMT, int DU, int VU, int NQ, int PARTS, bool FULL>
int stream_launch(const KvLayer& c, const KvStep& t, const KvAttn& a, const KvPlan& p, const KvKinds& kinds, cudaStream_t st) {
  using L = StreamShape<DU, VU, NQ, PARTS>;
  SEQ_CUDA((kb2::allow_smem<kv_stream_kernel<FMT, DU, VU, NQ, PARTS, FULL>>(L::kTotal)));
  auto kern = kv_stream_kernel<FMT, DU, VU, NQ, PARTS, FULL>;
  kb2::launch_pdl_clusters(kern, p.blocks ? dim3(p.blocks) : dim3(p.tiles, c.G, p.pieces), kSWarps * 32, L::kTotal, st, dim3(1, 1, p.cluster ? p.pieces : 1), c, t, a, kinds);
  SEQ_LAUNCHED();
  return KB2SEQ_OK;
}
template <int FMT, int DU, int VU, bool FULL>
int stream_rows(const KvLayer& c, const KvStep& t, const KvAttn& a, const KvPlan& p, const KvKinds& kinds, cudaStream_t st) {
  if (p.rows == 8) return a.dt_out ? stream_launch<FMT, DU, VU, 1, 1, FULL>(c, t, a, p, kinds, st) : stream_launch<FMT, DU, VU, 1, 2, FULL>(c, t, a, p, kinds, st);
  return a.dt_out ? stream_launch<FMT, DU, VU, 2, 1, FULL>(c, t, a, p, kinds, st) : stream_launch<FMT, DU, VU, 2, 2, FULL>(c, t, a, p, kinds, st);
}
template <int FMT>
int stream_sizes(const KvLayer& c, const KvStep& t, const KvAttn& a, const KvPlan& p, const KvKinds& kinds, cudaStream_t st) {
  const auto is = [&](int d, int dv) { return c.d == d && c.dv == dv; };
  if (is(64, 64)) return stream_rows<FMT, 1, 1, true>(c, t, a, p, kinds, st);
  if (is(128, 128)) return stream_rows<FMT, 2, 2, true>(c, t, a, p, kinds, st);
  if (is(192, 128)) return stream_rows<FMT, 3, 2, true>(c, t, a, p, kinds, st);
  if (is(128, 256)) return stream_rows<FMT, 2, 4, true>(c, t, a, p, kinds, st);
  if (is(256, 256)) return stream_rows<FMT, 4, 4, true>(c, t, a, p, kinds, st);
  return c.d <= 128 && c.dv <= 128 ? stream_rows<FMT, 2, 2, false>(c, t, a, p, kinds, st) : stream_rows<FMT, 4, 4, false>(c, t, a, p, kinds, st);
}
}  // namespace
}  // namespace kb2seq

using namespace kb2seq;

extern "C" {

KB2SEQ_API size_t kb2_seq_kv_attn_workspace(const kb2_seq_kv_cache* cache, const kb2_seq_kv_step* step, int H, int window, int first, int dt_out) {
  if (!cache || !step || !step->layout || step->T < 1 || cache->G < 1 || H < cache->G || bad_dt(dt_out)) return 0;
  OnDevice on(step->device);
  return kv_plans(cache, step, H, window > 0 ? std::min(window, kKvNoWindow) : kKvNoWindow, first, dt_out).bytes();
}

KB2SEQ_API int kb2_seq_kv_attn(const kb2_seq_kv_cache* cache, int layer, const kb2_seq_kv_step* step, const void* q, int dt_q, long long ldq, long long hq, int H,
                               float scale, int window, int first, const float* sinks, void* out, int dt_out, void* work, size_t work_bytes, void* stream) {
  KvLayer c;
  KvStep t;
  if (int e = kv_args("kv_attn", cache, layer, step, &c, &t)) return e;
  if ((t.T > 0 && (!q || !out)) || ((uintptr_t)out & 15) || bad_dt(dt_q) || bad_dt(dt_out) || H < c.G || H % c.G || window < 0 || first < 0 || !std::isfinite(scale))
    return failf(KB2SEQ_ERR_VALUE, "kv_attn: bad argument");
  if (c.G > 65535 || (long long)t.T * H > 0x7FFFFFFFll / 2) return failf(KB2SEQ_ERR_VALUE, "kv_attn: too many heads or tokens");
  if (t.T == 0) return KB2SEQ_OK;
  OnDevice on(step->device);                 // ahead of the plan, which goes by the device's size
  const int win = window > 0 ? std::min(window, kKvNoWindow) : kKvNoWindow;
  const KvPlans p = kv_plans(cache, step, H, win, first, dt_out);
  if (work_bytes < p.bytes() || (p.bytes() && (!work || ((uintptr_t)work & 15))))
    return failf(KB2SEQ_ERR_VALUE, "kv_attn: workspace of %zu bytes, %zu needed", work_bytes, p.bytes());
  if (std::max(p.few.pieces, p.many.pieces) > kMostPieces) return failf(KB2SEQ_ERR_VALUE, "kv_attn: too many rows in a sequence");
  if (std::max(p.few.parts, p.many.parts) > 0x7FFFFFFFll) return failf(KB2SEQ_ERR_VALUE, "kv_attn: too many rows that are cut");
  SEQ_CUDA(on.err);
  KvAttn a{};
  a.q = q;
  a.ldq = ldq;
  a.hq = hq;
  a.dtq = dt_q;
  a.vec = ((uintptr_t)q & (dt_q ? 7 : 15)) == 0 && ldq % 4 == 0 && hq % 4 == 0;
  a.H = H;
  a.window = win;
  a.first = first;
  a.scale = scale;
  a.sinks = sinks;
  a.out = out;
  a.dt_out = dt_out;
  const KvAttn few = with_plan(a, p.few, (float*)work, c.dv), many = with_plan(a, p.many, (float*)work + p.few.floats, c.dv);
  const cudaStream_t st = (cudaStream_t)stream;
  if (p.many.tiles) {
    if (int e = (kv_pairs(c.d, c.dv) ? kv_pair_attend : kv_tile_attend)(cache->fmt, c, t, many, p.kinds, p.many.blocks, st)) return e;
  }
  if (p.few.tiles) {
    if (int e = cache->fmt == KV_E4M3 ? stream_sizes<KV_E4M3>(c, t, few, p.few, p.kinds, st) : stream_sizes<KV_INT8>(c, t, few, p.few, p.kinds, st)) return e;
  }
  const long long rows = p.few.joined + p.many.joined;
  if (rows == 0) return KB2SEQ_OK;
  const int most = std::max(p.few.cluster ? 1 : p.few.pieces, p.many.pieces);
  const bool wide = rows <= 4096 || (most > 8 && rows <= 16384) || most > 32;
  auto join = wide ? kv_join_kernel<4> : kv_join_kernel<1>;
  kb2::launch_pdl(join, (unsigned)(wide ? rows : (rows + 3) / 4), 128, 0, st, c, t, few, many, p.kinds, (int)rows);
  SEQ_LAUNCHED();
  return KB2SEQ_OK;
}

}  // extern "C"
