// Attention over the 8-bit cache for many query rows per key / value head (portions of prompts, trees of drafted tokens) on tcgen05, where a head has more than 192 (keys) or
// 128 (values) numbers: tensor memory has room for one output of 128 rows there (seq_kv_pair.cu has two).
//
// A tile is 128 (token, head) rows of one sequence and kv head: the H / G heads that share keys fill it together, so a key tile is decoded once for all of them.  Roles of
// a CTA of 16 warps:
//   warp  1      brings codes and scales from the pages into a ring of three half tiles (bulk copies of 16 rows)
//   warps 12-15  decode: codes as fp16 into the swizzled operand tiles.  A row's scale over a power of two near the tile's largest one is multiplied in there (one packed
//                product for two codes; exact for scales that are powers of two), the power joins the softmax's factor
//   warp  0      tcgen05.mma: S = Q K^T, O += P V (P from tensor memory)
//   warps 4-11   softmax, two threads a row
// S and P have two buffers each; 64 keys a tile (tensor memory: 3 x 64 + 256 columns).
// What bounds it: a tile of keys is decoded for 128 rows, half as many as in seq_kv_pair.cu, and no pipe is near its limit (tensor 18 %, issue slots 30 %).  A portion of 2048
// tokens after 3000: 16 / 2 heads of 256 440 us (135 GFLOP, 0.19 of the measured cuBLAS rate), 32 / 4 heads of 128 / 256 411 (203 GFLOP, 0.30).
//
// Rounding, for bf16 results: queries, decoded numbers and weights times their tile's value scale are fp16 (11 bits).  Weights are rounded relative to a reference R per row
// that follows the largest weight times unit (2^6 to 2^15 of it); maxima, weights and their sum are fp32.  Weights below 2^-20 of the row's largest lose bits, whatever that one's value.
// A row whose scale is NaN gets NaN keys and zero values: scores that nobody sees are replaced, and those that see it carry the NaN into the sum.
#include "seq_kv_tc.cuh"

namespace kb2seq {
namespace {
using namespace kb2;

constexpr int kThreads = 512, kRows = 128, FK = 64, GT = FK / kKvGroup, NR = FK / 32;      // keys of a tile, their groups, a decoding thread's rows

template <int NC, int NV>                    // chunks of 64 of d and dv
struct TileShape {
  static constexpr int VS = NC + NV > 6 ? 1 : 2;                           // buffers of values
  static constexpr int kQ = NC * 128 * 128, kK = NC * FK * 128, kV = NV * FK * 128;
  static constexpr int kSlots = 3, kCodes = FK * 64 * (NC > NV ? NC : NV), kSlot = kCodes + FK * 8;       // codes as they come | scales of keys | of values
  static constexpr int kOffQ = 0, kOffK = kQ, kOffV = kOffK + 2 * kK, kOffSlot = kOffV + VS * kV, kOffBar = kOffSlot + kSlots * kSlot, kOffParts = kOffBar + 176, kOffRef = kOffParts + 16,
                       kOffHave = kOffRef + 4 * 8, kOffGone = kOffHave + kSlots * 4, kOffTmem = kOffGone + 4 * 4, kOffX = kOffTmem + 4, kOffRow = kOffX + 2 * 2 * 128 * 4;
  static constexpr int kTotal = kOffRow + 128 * 4;
  static_assert(kTotal <= 227 * 1024 && 3 * FK + 64 * NV <= 512 && kSlot % 128 == 0 && kOffRef % 8 == 0 && kOffX % 16 == 0, "memory");
};

// Codes of a tile from `from` (rows of `width` bytes) into the operand at `to`.  A thread has the rows ct / 4 and ct / 4 + 32 and 16 bytes of each chunk of 64 of those, f times
// the codes where see.  Odd rows take their chunks in another order: eight lanes that are served together then read 128 neighbouring bytes or two rows' halves, and the stores
// of 16 bytes meet 8 rows' swizzles, two of them in eight lanes: no bank twice either way.
template <int FMT, int CH>
__device__ __forceinline__ void decode(uint8_t* to, const uint8_t* from, int width, int ct, const float (&f)[NR], const bool (&see)[NR]) {
  static_assert(CH % 2 == 0, "odd rows begin with the second chunk of two");
  const int q = ct & 3;
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int row = (ct >> 2) + 32 * i;
    const uint32_t m = f16_pair(f[i], f[i]);
#pragma unroll
    for (int h0 = 0; h0 < CH; ++h0) {
      const int h = h0 ^ (row & 1), e0 = h * 64 + q * 16;
      const uint4 v = see[i] && e0 < width ? *reinterpret_cast<const uint4*>(from + row * width + e0) : make_uint4(0, 0, 0, 0);
      uint32_t y[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        codes_f16<FMT>(word(v, e), y[2 * e], y[2 * e + 1]);
        y[2 * e] = hmul2(y[2 * e], m);
        y[2 * e + 1] = hmul2(y[2 * e + 1], m);
      }
      uint8_t* p = to + h * (32 * NR * 128) + row * 128;
      *reinterpret_cast<uint4*>(p + (((2 * q) ^ (row & 7)) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
      *reinterpret_cast<uint4*>(p + (((2 * q + 1) ^ (row & 7)) << 4)) = make_uint4(y[4], y[5], y[6], y[7]);
    }
  }
  fence_proxy_async_smem();
  __syncwarp();
}

// This thread's arrival once its copies so far (cp.async) are there.
__device__ __forceinline__ void arrive_behind_copies(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

template <int FMT, int NC, int NV>
__global__ void __launch_bounds__(kThreads, 1) kv_tile_kernel(KvLayer c, KvStep t, KvAttn a, const __grid_constant__ KvKinds kinds) {
  using L = TileShape<NC, NV>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
  uint64_t *k_full = bars, *k_empty = bars + 2, *v_full = bars + 4, *v_empty = bars + 6, *s_full = bars + 8, *s_cons = bars + 10, *p_full = bars + 12, *pv_done = bars + 14,
           *c_full = bars + 16, *c_empty = bars + 19;
  float2* refs = reinterpret_cast<float2*>(smem + L::kOffRef);             // [4] tile's units: keys, values
  uint32_t* have = reinterpret_cast<uint32_t*>(smem + L::kOffHave);        // [3] a slot's groups that are there, a bit each
  uint32_t* gone = reinterpret_cast<uint32_t*>(smem + L::kOffGone);        // [4] a tile's groups that are not
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(smem + L::kOffTmem);
  KvParts* seq_parts = reinterpret_cast<KvParts*>(smem + L::kOffParts);    // where the piece's partial results lie, those of the sequence's row 0; -1: there are none, the tile has one piece
  float* rows_down = reinterpret_cast<float*>(smem + L::kOffRow);          // [128] what the queries' own scaling is undone with
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 4);
      mbar_init(&v_full[i], 4);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&pv_done[i], 1);
      mbar_init(&s_cons[i], 8);
      mbar_init(&p_full[i], 8);
    }
    for (int i = 0; i < 3; ++i) {
      mbar_init(&c_full[i], 33);                // the bytes of the bulk copies, and the lanes that copy scales
      mbar_init(&c_empty[i], 4);
    }
    fence_mbar_init();
  }
  if (warp == 2) tmem_alloc(tmem_at, 512);
  pdl_wait();

  // which tile, and what its rows see: the same in every warp
  const int per = a.H / c.G, head = blockIdx.y;
  int s = 0, tile = 0, z = 0, length = 0x7FFFFFFF;
  bool in = true;
  KvParts parts{};
  if (a.per_seq && a.pieces == 1) {
    s = blockIdx.x / a.per_seq;
    tile = blockIdx.x - s * a.per_seq;
  } else {
    in = kv_find_piece(c, t, a, kinds, per, blockIdx.x, &s, &tile, &z, &length, &parts);
  }
  const int c0 = t.cu[s], n = t.cu[s + 1] - c0, r0 = tile * kRows, nr = in ? (int)min((long long)n * per - r0, (long long)kRows) : 0;
  int u0 = 0, u1 = 0, np = 0, t0 = c0, t1 = c0;
  KvSpan span{};
  if (nr > 0) {
    t0 = c0 + r0 / per;
    t1 = c0 + (r0 + nr - 1) / per;
    span = kv_span(c, t, s, t0, t1, a.window, a.first);
    np = a.pieces == 1 ? 1 : min((span.groups() + length - 1) / length, a.pieces);
    u0 = a.pieces == 1 ? 0 : z * length;
    u1 = a.pieces == 1 ? span.groups() : min(span.groups(), u0 + length);
  }
  if (threadIdx.x == 0) *seq_parts = {np <= 1 ? -1 : parts.first + z, parts.pieces};
  const bool work = nr > 0 && (z == 0 || z < np);   // piece 0 of a tile that sees nothing writes its zeros
  const int n_tiles = work ? max(0, (u1 - u0 + GT - 1) / GT) : 0;

  // queries, 8 rows a warp: scaled by a power of two, rounded to fp16, in the operand's layout (rows of 64 numbers, 16-byte pieces swizzled by the row)
  if (work) {
    const float sign = a.scale < 0.f ? -1.f : a.scale == 0.f ? 0.f : 1.f;  // factors on scores are positive: a row's maximum is its largest raw score's
#pragma unroll 2
    for (int i = 0; i < 8; ++i) {
      const int r = warp * 8 + i, rr = r0 + r;
      const bool row = r < nr;
      const long long from = row ? (c0 + rr / per) * a.ldq + (head * per + rr % per) * a.hq : 0;
      float x[2][4];
      uint32_t top = 0;
#pragma unroll
      for (int b = 0; b < (NC + 1) / 2; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int e = b * 128 + lane * 4 + j;
          x[b][j] = row && e < c.d ? (a.dtq ? __bfloat162float(((const bf16*)a.q)[from + e]) : ((const float*)a.q)[from + e]) : 0.f;
          top = max(top, __float_as_uint(x[b][j]) & 0x7FFFFFFFu);
        }
      top = __reduce_max_sync(0xffffffffu, top);
      float up, down;
      kv_row_scale(top, &up, &down);
      up *= sign;
#pragma unroll
      for (int b = 0; b < (NC + 1) / 2; ++b) {
        const int e = b * 128 + lane * 4;
        if (e < NC * 64)
          *reinterpret_cast<uint2*>(smem + L::kOffQ + (e >> 6) * (128 * 128) + r * 128 + ((((e & 63) >> 3) ^ (r & 7)) << 4) + (e & 4) * 2) =
              make_uint2(f16_pair(x[b][0] * up, x[b][1] * up), f16_pair(x[b][2] * up, x[b][3] * up));
      }
      if (lane == 0) rows_down[r] = sign == 0.f ? 1.f : fabsf(a.scale) * kLog2e * down;
    }
  }
  fence_proxy_async_smem();
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_at;
  constexpr uint32_t kColS = 0, kColP = 2 * FK, kColO = 3 * FK;

  if (n_tiles == 0) {
    if (work && warp >= 4 && warp < 12) {                                  // nothing to see (no piece shares this tile): zeros
      for (int i = (warp - 4) * 32 + lane; i < nr * c.dv; i += 256) {
        const int r = i / c.dv, rr = r0 + r;
        ((bf16*)a.out)[((long long)(c0 + rr / per) * a.H + head * per + rr % per) * c.dv + i - r * c.dv] = __float2bfloat16_rn(0.f);
      }
    }
  } else if (warp >= 12) {
    // ------------------------------------------------------------ decode: K(0), then K(it + 1) and V(it) in turn
    const int ct = threadIdx.x - 384;
    bool see[NR], see_v[NR];
    float fk[NR], fv[NR], fv_next[NR];
    int job = 0;
    const auto keys = [&](int it) {
      const int b = it & 1, slot = job % L::kSlots;
      const uint8_t* from = smem + L::kOffSlot + slot * L::kSlot;
      const float *ks = reinterpret_cast<const float*>(from + L::kCodes), *vs = ks + FK;
      mbar_wait(&c_full[slot], job / L::kSlots & 1);
      const uint32_t groups = have[slot];
      const auto seen = [&](int row) {       // by any row of the tile
        const int j = span.group(u0 + it * GT + row / 16) * kKvGroup + (row & 15);
        return (groups >> (row / 16) & 1u) && j < span.hi && (j >= span.lo || j < a.first);
      };
      uint32_t kt = 0, vt = 0;               // the tile's largest scales
#pragma unroll
      for (int i = 0; i < FK / 32; ++i) {
        const int row = i * 32 + lane;
        if (seen(row)) {
          const uint32_t x = __float_as_uint(ks[row]), y = __float_as_uint(vs[row]);
          if (x < 0x7F800000u) kt = max(kt, x);
          if (y < 0x7F800000u) vt = max(vt, y);
        }
      }
      float kp, ki, vp, vi;
      scale_unit(__reduce_max_sync(0xffffffffu, kt), &kp, &ki);
      vt = __reduce_max_sync(0xffffffffu, vt);
      scale_unit(vt, &vp, &vi);
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const int row = (ct >> 2) + 32 * i;
        see[i] = seen(row);
        const float x = see[i] ? ks[row] : 0.f, y = see[i] ? vs[row] : 0.f;
        fk[i] = y != y ? y : x * ki;         // a row that is no number: its keys say so
        fv_next[i] = y != y ? 0.f : y * vi;
      }
      mbar_wait(&k_empty[b], (it >> 1 & 1) ^ 1);
      decode<FMT, NC>(smem + L::kOffK + b * L::kK, from, c.d, ct, fk, see);
      if (ct == 0) {
        refs[it & 3] = make_float2(kp, vt ? vp : 0.f);
        gone[it & 3] = ~groups & ((1u << GT) - 1);
      }
      if (lane == 0) {
        mbar_arrive(&k_full[b]);
        mbar_arrive(&c_empty[slot]);
      }
      ++job;
    };
    keys(0);
    for (int it = 0; it < n_tiles; ++it) {
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        fv[i] = fv_next[i];
        see_v[i] = see[i];
      }
      if (it + 1 < n_tiles) keys(it + 1);
      const int b = it % L::VS, slot = job % L::kSlots;
      mbar_wait(&c_full[slot], job / L::kSlots & 1);
      mbar_wait(&v_empty[b], (it / L::VS & 1) ^ 1);
      decode<FMT, NV>(smem + L::kOffV + b * L::kV, smem + L::kOffSlot + slot * L::kSlot, c.dv, ct, fv, see_v);
      if (lane == 0) {
        mbar_arrive(&v_full[b]);
        mbar_arrive(&c_empty[slot]);
      }
      ++job;
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ codes and scales from the pages, in the decoders' order.  A run of groups that one page holds is one run of
    // bytes in each pool, and one bulk copy (heads of 128, 4096 tokens: one a group 1083 us, one a run 989); scales go 16 bytes a lane.
    const auto at_row = [&](int it) {        // lane's group of a tile
      const int u = u0 + it * GT + lane;
      const long long r = lane < GT && it < n_tiles && u < u1 ? kv_row(c, t, s, span.group(u) * kKvGroup) : -1;
      return r < 0 ? -1ll : r + ((long long)head << c.lps);
    };
    int job = 0;
    const auto fetch = [&](long long r, bool val) {
      const int slot = job % L::kSlots;
      uint8_t* to = smem + L::kOffSlot + slot * L::kSlot;
      const long long before = __shfl_up_sync(0xffffffffu, r, 1), mine = __shfl_sync(0xffffffffu, r, lane / 4);      // the lane's scales are its group's: row 4 lane of the tile
      const uint32_t there = __ballot_sync(0xffffffffu, r >= 0);
      const uint32_t lead = __ballot_sync(0xffffffffu, r >= 0 && !(lane && before >= 0 && r == before + kKvGroup)) | ~there;      // a run ends where another or a gap begins
      const int run = lane < 31 ? __ffs(lead >> (lane + 1)) : 0;           // lanes behind the last group are gaps
      mbar_wait(&c_empty[slot], (job / L::kSlots & 1) ^ 1);
      if (lane == 0) {
        have[slot] = there;
        mbar_arrive_expect_tx(&c_full[slot], __popc(there) * kKvGroup * (val ? c.dv : c.d));
      }
      __syncwarp();
      if (r >= 0 && (lead >> lane & 1u)) {
        const int n = kKvGroup * (val ? c.dv : c.d);
        bulk_g2s(to + lane * n, val ? c.v + r * c.dv : c.k + r * c.d, run * n, &c_full[slot]);
      }
      if (!val && lane * 4 < FK && mine >= 0) {
        cp_async16_stream(smem_u32(to + L::kCodes) + lane * 16, c.ks + mine + (lane & 3) * 4, true);
        cp_async16_stream(smem_u32(to + L::kCodes) + FK * 4 + lane * 16, c.vs + mine + (lane & 3) * 4, true);
      }
      arrive_behind_copies(&c_full[slot]);
      ++job;
    };
    long long cur = at_row(0), next = at_row(1);
    fetch(cur, false);
    for (int it = 0; it < n_tiles; ++it) {
      const long long later = at_row(it + 2);
      if (it + 1 < n_tiles) fetch(next, false);
      fetch(cur, true);
      cur = next;
      next = later;
    }
  } else if (warp == 0) {
    // ------------------------------------------------------------ tensor cores
    const uint32_t id_s = idesc_f16(FK, false), id_o = idesc_f16(64 * NV, true);
    const uint32_t q_at = smem_u32(smem + L::kOffQ);
    const auto scores = [&](int it) {
      const int b = it & 1;
      mbar_wait(&k_full[b], it >> 1 & 1);
      if (it >= 2) mbar_wait(&s_cons[b], (it >> 1 & 1) ^ 1);
      tc_fence_after_sync();
      const uint32_t k_at = smem_u32(smem + L::kOffK + b * L::kK);
      if (elect_one()) {
#pragma unroll
        for (int h = 0; h < NC; ++h) {
          const uint64_t ad = umma_desc_k_sw128(q_at + h * (128 * 128)), bd = umma_desc_k_sw128(k_at + h * (FK * 128));
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_bf16(tmem + kColS + b * FK, ad + 2 * k, bd + 2 * k, id_s, h > 0 || k > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[b]);
        umma_commit(&k_empty[b]);
      }
      __syncwarp();
    };
    scores(0);
    if (n_tiles > 1) scores(1);
    for (int it = 0; it < n_tiles; ++it) {
      const int b = it & 1;
      if (it + 2 < n_tiles) scores(it + 2);
      const int vb = it % L::VS;
      mbar_wait(&v_full[vb], it / L::VS & 1);
      mbar_wait(&p_full[b], it >> 1 & 1);
      tc_fence_after_sync();
      const uint32_t v_at = smem_u32(smem + L::kOffV + vb * L::kV);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < FK / 16; ++k)
          umma_bf16_ts(tmem + kColO, tmem + kColP + b * (FK / 2) + 8 * k, desc_mn(v_at + k * 2048, FK * 128), id_o, it > 0 || k > 0 ? 1u : 0u);
        umma_commit(&pv_done[b]);
        umma_commit(&v_empty[vb]);
      }
      __syncwarp();
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ softmax: warp w has the rows of quarter w & 3; warps 4-7 the first 32 of every 64 keys and half of the
    // output columns, warps 8-11 the others.  The two threads of a row exchange their maxima through shared memory.
    const int quarter = warp & 3, hf = (warp - 4) >> 2, row = quarter * 32 + lane, rr = r0 + row;
    const bool live = row < nr;
    const int tok = live ? c0 + rr / per : t0, pos = live ? t.positions[tok] : -1;
    int least, most;
    {                                        // of the warp's rows
      const int ra = min(r0 + quarter * 32, r0 + nr - 1), rb = min(r0 + quarter * 32 + 31, r0 + nr - 1);
      KvSpan own = span;
      own.p0 = t.positions[c0 + ra / per];
      own.p1 = t.positions[c0 + rb / per];
      kv_reach(t, a, own, c0 + ra / per, c0 + rb / per, &least, &most);
    }
    const uint32_t lane_at = tmem + ((uint32_t)(quarter * 32) << 16);
    float* xchg = reinterpret_cast<float*>(smem + L::kOffX);
    const float down = rows_down[row];
    constexpr int OH = 32 * NV;
    float m = -INFINITY, l = 0.f, ref = 0.f;
    const auto tell = [&](uint64_t* bar) {
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    const auto pv_wait = [&](int it) {
      mbar_wait(&pv_done[it & 1], it >> 1 & 1);
      tc_fence_after_sync();
    };
    for (int it = 0; it < n_tiles; ++it) {
      const int b = it & 1;
      mbar_wait(&s_full[b], it >> 1 & 1);
      tc_fence_after_sync();
      const float2 p2 = refs[it & 3];        // written ahead of the keys; the tile after next writes none before this one's scores are taken
      const uint32_t away = gone[it & 3];
      float x[32];
      {
        uint32_t r[2][16];
        tmem_ld16(lane_at + kColS + b * FK + hf * 32, r[0]);
        tmem_ld16(lane_at + kColS + b * FK + hf * 32 + 16, r[1]);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j) x[j] = __uint_as_float(r[j / 16][j % 16]);
      }
      tell(&s_cons[b]);
      const int ua = u0 + it * GT, ub = min(ua + GT, u1) - 1;              // groups of the tile
      const int pa = span.group(ua) * kKvGroup, pb = span.group(ub) * kKvGroup + kKvGroup - 1;
      const bool all = away == 0 && ub == ua + GT - 1 && pb < span.base && pb <= least && (pb < a.first || (ua >= span.na && most - pa < a.window));
      if (!all) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const int u = ua + hf * 2 + g, j0 = span.group(u) * kKvGroup;
          uint32_t see = 0;
          if (u < u1 && live && !(away >> (u - ua) & 1u)) {
#pragma unroll 1
            for (int j = 0; j < 16; ++j) see |= (uint32_t)kv_sees(t, a, span, c0, n, tok, pos, j0 + j) << j;
          }
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (!(see >> j & 1u)) x[16 * g + j] = -INFINITY;
        }
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < 32; j += 2) mx[j >> 1 & 3] = max3(mx[j >> 1 & 3], x[j], x[j + 1]);
      float mt = max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]);
      float* xb = xchg + b * 256;
      xb[hf * 128 + row] = mt;
      __syncwarp();
      named_bar_sync(1 + quarter, 64);
      const float fac = fminf(fmaxf(down * p2.x, 1e-37f), 1e37f);
      mt = fmaxf(mt, xb[(hf ^ 1) * 128 + row]) * fac;
      const float mn = fmaxf(m, mt), from = mn == -INFINITY ? 0.f : mn, back = ex2(m - from);
      m = mn;
      l *= back;
      ref *= back;
      const float big = ex2(mt - from) * p2.y;                             // the tile's largest weight times scale
      float grow = 1.f;
      bool again = false;
      const float least = fmaxf(p2.y * 7.8886091e-31f, 1e-37f);            // 2^-100 of the unit: 1 / ref times it stays within fp32
      if (big > 1e-37f && (big > ref * 32768.f || ref < least)) {
        const float r = fmaxf(big * 0.015625f, least);
        grow = ref / r;
        again = it > 0;                      // a reference that has shrunk to nothing as well: what O holds is then far below
        ref = r;
      }
      const float f = ref >= least ? p2.y * __frcp_rn(ref) : 0.f;
      const uint64_t fac2 = pair_of(fac, fac), neg2 = pair_of(-from, -from), f2 = pair_of(f, f);
      uint64_t sum[2] = {0, 0};
      uint32_t pk[16];
#pragma unroll
      for (int j = 0; j < 32; j += 2) {
        const float2 e = pair_get(pair_fma(pair_of(x[j], x[j + 1]), fac2, neg2));
        const uint64_t p = pair_of(ex2(e.x), ex2(e.y));
        sum[j >> 1 & 1] = pair_add(sum[j >> 1 & 1], p);
        const float2 y = pair_get(pair_mul(p, f2));
        pk[j / 2] = f16_pair(y.x, y.y);
      }
      const float2 s2 = pair_get(pair_add(sum[0], sum[1]));
      l += s2.x + s2.y;
      if (it >= 2) pv_wait(it - 2);          // PV(it - 2) has read this P buffer
      if (__any_sync(0xffffffffu, again)) {
        pv_wait(it - 1);                     // O holds every product so far 
        const float sc = again ? grow : 1.f;
#pragma unroll 2
        for (int o = hf * OH; o < (hf + 1) * OH; o += 16) {
          uint32_t r[16];
          tmem_ld16(lane_at + kColO + o, r);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * sc);
          tmem_st16(lane_at + kColO + o, r);
        }
      }
      tmem_st16(lane_at + kColP + b * (FK / 2) + hf * 16, pk);
      tmem_st_wait();
      tell(&p_full[b]);
    }
    float* xb = xchg + (n_tiles & 1) * 256;  // the buffer that the last tile did not use
    xb[hf * 128 + row] = l;
    __syncwarp();
    named_bar_sync(1 + quarter, 64);
    l += xb[(hf ^ 1) * 128 + row];
    if (n_tiles >= 2) pv_wait(n_tiles - 2);
    pv_wait(n_tiles - 1);
    const int hd = head * per + rr % per;
    const bool whole = seq_parts->first < 0;
    const long long orow = (long long)tok * a.H + hd;
    const int part = whole ? 0 : seq_parts->first + ((tok - c0) * a.H + hd) * seq_parts->pieces;
    const bool kept = live && (whole || (unsigned)part < (unsigned)a.parts);
    if (whole && live && a.sinks != nullptr && m != -INFINITY) l += ex2(fmaf(a.sinks[hd], kLog2e, -m));
    const float by = whole ? (l == 0.f ? 0.f : ref / l) : ref;
    if (!whole && kept && hf == 0) {
      a.part_ml[2ll * part] = m;
      a.part_ml[2ll * part + 1] = l;
    }
#pragma unroll 2
    for (int o = hf * OH; o < (hf + 1) * OH; o += 16) {
      uint32_t r[16];
      __syncwarp();                          // the warp reads tensor memory together
      tmem_ld16(lane_at + kColO + o, r);
      tmem_ld_wait();
      if (!kept || o >= c.dv) continue;
      float y[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) y[j] = __uint_as_float(r[j]) * by + (l != l ? l : 0.f);         // a sum that is NaN has a zero for its reference, maybe
      if (whole) {
        uint4* to = reinterpret_cast<uint4*>((bf16*)a.out + orow * c.dv + o);
#pragma unroll
        for (int j = 0; j < 2; ++j)
          to[j] = make_uint4(bf16x2_bits_rn(y[8 * j + 1], y[8 * j]), bf16x2_bits_rn(y[8 * j + 3], y[8 * j + 2]), bf16x2_bits_rn(y[8 * j + 5], y[8 * j + 4]),
                             bf16x2_bits_rn(y[8 * j + 7], y[8 * j + 6]));
      } else {
        float4* to = reinterpret_cast<float4*>(a.part_o + (long long)part * c.dv + o);
#pragma unroll
        for (int j = 0; j < 4; ++j) to[j] = make_float4(y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3]);
      }
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 2) tmem_dealloc(tmem, 512);
}

template <int FMT, int NC, int NV>
int launch(const KvLayer& c, const KvStep& t, const KvAttn& a, const KvKinds& kinds, int tiles, cudaStream_t st) {
  using L = TileShape<NC, NV>;
  SEQ_CUDA((kb2::allow_smem<kv_tile_kernel<FMT, NC, NV>>(L::kTotal)));
  auto kern = kv_tile_kernel<FMT, NC, NV>;
  kb2::launch_pdl(kern, dim3(tiles, c.G), kThreads, L::kTotal, st, c, t, a, kinds);
  SEQ_LAUNCHED();
  return KB2SEQ_OK;
}
template <int FMT>
int sizes(const KvLayer& c, const KvStep& t, const KvAttn& a, const KvKinds& kinds, int tiles, cudaStream_t st) {
  return c.d <= 128 ? launch<FMT, 2, 4>(c, t, a, kinds, tiles, st) : launch<FMT, 4, 4>(c, t, a, kinds, tiles, st);
}
}  // namespace

int kv_tile_attend(int fmt, const KvLayer& c, const KvStep& t, const KvAttn& a, const KvKinds& kinds, int tiles, cudaStream_t stream) {
  return fmt == KV_E4M3 ? sizes<KV_E4M3>(c, t, a, kinds, tiles, stream) : sizes<KV_INT8>(c, t, a, kinds, tiles, stream);
}

}  // namespace kb2seq
