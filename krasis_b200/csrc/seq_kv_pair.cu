// Attention over the 8-bit cache for many query rows per key / value head on tcgen05, heads of up to 192 (keys) and 128 (values): two tiles of 128 (token, head) rows of one
// sequence and kv head share every key tile that is decoded.  The H / G heads that share keys fill the rows together.  Roles of a CTA of 16 warps:
//   warp  1      plans 128 keys at a time: looks up their groups in the page list, reads their scales, and leaves for each row the factors that its codes are multiplied with
//   warps 12-15  decode 64 keys at a time: codes from the pages into registers, two tiles ahead, as fp16 (code times factor, one packed product for two) into the operands
//   warps 0, 3   tcgen05.mma for a row tile each: S = Q K^T and O += P V (P from tensor memory, in S's place)
//   warps 4-7, 8-11  softmax of the first and of the second row tile, a thread a row
// Where a sequence has no more than 128 rows left both softmax groups have the same rows and take the key tiles in turn; they are joined at the end.
// Key tiles of 64 with two buffers of scores per row tile, so that the next scores are made while a tile's are worked on; four buffers of keys and of values.
// Tensor memory: S 2 x 2 x 64 | O 2 x 64 NV.
//
// What bounds it: the tensor pipe.  A product of 128 x 64 x 16 with both operands in shared memory takes 75 cycles (64 x 16 of K and 128 x 16 of Q are read each time), one of
// 128 x 128 x 16 with P in tensor memory 76, so 128 keys and 256 rows take 3616; their 32768 exponentials take 2048 (16 a cycle).  A portion of 4096 tokens after 5001, window
// 4096, 64 / 4 heads of 128: 621 us, 4510 cycles for those 128 keys, 552 GFLOP at 0.54 of the measured cuBLAS rate.  On the way there: one row tile a CTA with 128 keys a tile
// 989, two 722, softmax groups in turn 679, tiles of 64 keys with two buffers of scores 688 with one warp for the tensor cores, which spends 300 cycles between two batches of
// products while the pipe takes two ahead, and 606 with two; groups of pages that are not there, looked for in each tile, cost most of the rest.
// Heads of 192 spill 264 bytes a thread (a portion of 2048 after 3000, 64 / 4 heads of 192 / 128: 440 us, 338 GFLOP at 0.46 of that rate), those of 64 24.
//
// Rounding, for bf16 results: queries, decoded numbers and weights times their tile's value unit are fp16 (11 bits).  A row's factor is its scale over a unit, a power of two
// near the tile's largest scale (exact for scales that are powers of two); the units join the softmax's factors.  Weights are rounded relative to a reference R per row that
// follows the largest weight times unit (2^6 to 2^15 of it); maxima, weights and their sum are fp32.  The largest weight's own value may be zero (the kernel for few rows goes by
// each row's scale): weights below 2^-20 of the row's largest lose bits all the same.
// A row whose scale is NaN gets NaN keys and zero values: scores that nobody sees are replaced, and those that see it carry the NaN into the sum.
#include "seq_kv_tc.cuh"

namespace kb2seq {
namespace {

constexpr int kThreads = 512, FK = 64, GT = FK / kKvGroup, kBufs = 4;      // keys of a tile, their groups; operand buffers
constexpr int kBarShare = 1;                 // named barrier of both softmax groups
constexpr int kPlans = 4, kUnits = 8;        // pairs of tiles that are planned ahead; units are read later than the rest

template <int NC, int NV>                    // chunks of 64 of d and dv
struct PairShape {
  static constexpr int kQ = NC * 128 * 128, kK = NC * FK * 128, kV = NV * FK * 128, kKeys = NC > 2 ? 2 : kBufs;      // kKeys: buffers of keys
  static constexpr int kOffQ = 0, kOffK = 2 * kQ, kOffV = kOffK + kKeys * kK, kOffFac = kOffV + kBufs * kV, kOffGroup = kOffFac + kPlans * 512,
                       kOffBar = kOffGroup + kPlans * 32, kOffParts = kOffBar + 304, kOffUnit = kOffParts + 16, kOffTmem = kOffUnit + kUnits * 16, kOffRow = kOffTmem + 16, kTotal = kOffRow + 256 * 4;
  static_assert(kTotal <= 227 * 1024 && 4 * FK + 128 * NV <= 512, "memory");
  static_assert(128 * (64 * NV + 1) * 4 + 128 * 12 <= 2 * kQ + kKeys * kK + kBufs * kV, "the second group's share at the end");
};

// A thread's 16 bytes of each chunk of 64 of the rows ct / 4 + 32 i.
template <int NR, int CH>
__device__ __forceinline__ void pair_load(const uint8_t* pool, int width, int ct, const int* groups, uint4 (&x)[NR * CH]) {
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int row = (ct >> 2) + 32 * i, r16 = groups[row >> 4];
    const uint8_t* from = pool + ((long long)r16 * kKvGroup + (row & 15)) * width + (ct & 3) * 16;
#pragma unroll
    for (int h = 0; h < CH; ++h) x[i * CH + h] = r16 >= 0 && h * 64 + (ct & 3) * 16 < width ? ld_stream16(from + h * 64) : make_uint4(0, 0, 0, 0);
  }
}
// The same as fp16 in the operand at `to`, times the rows' factors.  The stores of 16 bytes a lane meet 8 rows' swizzles, two of them in eight lanes: no bank twice.
template <int FMT, int NR, int CH>
__device__ __forceinline__ void pair_store(uint8_t* to, int ct, const uint32_t (&f)[NR], const uint4 (&x)[NR * CH]) {
  const int q = ct & 3;
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int row = (ct >> 2) + 32 * i;
#pragma unroll
    for (int h = 0; h < CH; ++h) {
      uint32_t y[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        codes_f16<FMT>(word(x[i * CH + h], e), y[2 * e], y[2 * e + 1]);
        y[2 * e] = hmul2(y[2 * e], f[i]);
        y[2 * e + 1] = hmul2(y[2 * e + 1], f[i]);
      }
      uint8_t* p = to + h * (32 * NR * 128) + row * 128;
      *reinterpret_cast<uint4*>(p + (((2 * q) ^ (row & 7)) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
      *reinterpret_cast<uint4*>(p + (((2 * q + 1) ^ (row & 7)) << 4)) = make_uint4(y[4], y[5], y[6], y[7]);
    }
  }
  fence_proxy_async_smem();
  __syncwarp();
}

template <int FMT, int NC, int NV>
__global__ void __launch_bounds__(kThreads, 1) kv_pair_kernel(KvLayer c, KvStep t, KvAttn a, const __grid_constant__ KvKinds kinds) {
  using L = PairShape<NC, NV>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
  // by buffer: k_full .. v_empty; by row tile and buffer of scores: s_full, p_full, pv_done; by plan: plan_full, plan_empty
  uint64_t *k_full = bars, *k_empty = bars + 4, *v_full = bars + 8, *v_empty = bars + 12, *s_full = bars + 16, *p_full = bars + 20, *pv_done = bars + 24, *plan_full = bars + 28,
           *plan_empty = bars + 28 + kPlans, *q_full = bars + 28 + 2 * kPlans;
  uint32_t* factors = reinterpret_cast<uint32_t*>(smem + L::kOffFac);      // [kPlans][128] fp16: of the row's key codes, of its value codes
  int* groups = reinterpret_cast<int*>(smem + L::kOffGroup);               // [kPlans][8] where the groups lie (rows / 16), -1: nowhere
  float4* units = reinterpret_cast<float4*>(smem + L::kOffUnit);           // [kUnits] of keys, of values; four bits a group: whether it lies nowhere
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(smem + L::kOffTmem);
  KvParts* seq_parts = reinterpret_cast<KvParts*>(smem + L::kOffParts);    // where the piece's partial results lie, those of the sequence's row 0; -1: there are none, the tile has one piece
  float* rows_down = reinterpret_cast<float*>(smem + L::kOffRow);          // [256] what the queries' own scaling is undone with
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
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
  const int c0 = t.cu[s], n = t.cu[s + 1] - c0, r0 = tile * 256, nr = in ? (int)min((long long)n * per - r0, 256ll) : 0;
  int u0 = 0, u1 = 0, np = 0, t0 = c0;
  KvSpan span{};
  if (nr > 0) {
    t0 = c0 + r0 / per;
    span = kv_span(c, t, s, t0, c0 + (r0 + nr - 1) / per, a.window, a.first);
    np = a.pieces == 1 ? 1 : min((span.groups() + length - 1) / length, a.pieces);
    u0 = a.pieces == 1 ? 0 : z * length;
    u1 = a.pieces == 1 ? span.groups() : min(span.groups(), u0 + length);
  }
  if (threadIdx.x == 0) *seq_parts = {np <= 1 ? -1 : parts.first + z, parts.pieces};
  const bool work = nr > 0 && (z == 0 || z < np);   // piece 0 of a tile that sees nothing writes its zeros
  const int n_tiles = work ? max(0, (u1 - u0 + GT - 1) / GT) : 0;
  const bool two = nr > 128;                 // two row tiles; else one whose key tiles go to both groups in turn
  if (threadIdx.x == 0) {
    for (int i = 0; i < 4; ++i) {
      mbar_init(&k_full[i], 4);
      mbar_init(&v_full[i], 4);
      mbar_init(&k_empty[i], two ? 2 : 1);
      mbar_init(&v_empty[i], two ? 2 : 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&pv_done[i], 1);
    }
    for (int i = 0; i < kPlans; ++i) {
      mbar_init(&plan_full[i], 1);
      mbar_init(&plan_empty[i], 4);
    }
    mbar_init(q_full, 8);
    fence_mbar_init();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_at;
  constexpr uint32_t kColO = 4 * FK;

  if (n_tiles == 0) {
    if (work && warp >= 4 && warp < 12) {                                  // nothing to see (no piece shares this tile): zeros
      for (int i = (warp - 4) * 32 + lane; i < nr * c.dv; i += 256) {
        const int r = i / c.dv, rr = r0 + r;
        ((bf16*)a.out)[((long long)(c0 + rr / per) * a.H + head * per + rr % per) * c.dv + i - r * c.dv] = __float2bfloat16_rn(0.f);
      }
    }
  } else if (warp >= 12) {
    // ------------------------------------------------------------ decode
    const int ct = threadIdx.x - 384;
    constexpr int NR = FK / 32;
    uint4 xk[2][NR * NC], xv[2][NR * NV];
    const auto fetch = [&](int it, auto& k, auto& v) {
      if (it >= n_tiles) return;
      const int p = it >> 1, slot = p % kPlans;
      mbar_wait(&plan_full[slot], p / kPlans & 1);
      const int* g = groups + slot * 8 + (it & 1) * GT;
      pair_load<NR, NC>(c.k, c.d, ct, g, k);
      pair_load<NR, NV>(c.v, c.dv, ct, g, v);
    };
    const auto work_on = [&](int it, auto& k, auto& v) {
      if (it >= n_tiles) return;
      const int kb = it % L::kKeys, vb = it % kBufs, slot = (it >> 1) % kPlans;
      uint32_t f[NR], fk[NR], fv[NR];
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        f[i] = factors[slot * 128 + (it & 1) * FK + (ct >> 2) + 32 * i];
        fk[i] = __byte_perm(f[i], 0, 0x1010);
        fv[i] = __byte_perm(f[i], 0, 0x3232);
      }
      mbar_wait(&k_empty[kb], (it / L::kKeys & 1) ^ 1);
      pair_store<FMT, NR, NC>(smem + L::kOffK + kb * L::kK, ct, fk, k);
      if (lane == 0) mbar_arrive(&k_full[kb]);
      mbar_wait(&v_empty[vb], (it / kBufs & 1) ^ 1);
      pair_store<FMT, NR, NV>(smem + L::kOffV + vb * L::kV, ct, fv, v);
      if (lane == 0) {
        mbar_arrive(&v_full[vb]);
        if ((it & 1) || it + 1 == n_tiles) mbar_arrive(&plan_empty[slot]);
      }
    };
    fetch(0, xk[0], xv[0]);
    fetch(1, xk[1], xv[1]);
    for (int it = 0; it < n_tiles; it += 2) {
      work_on(it, xk[0], xv[0]);
      fetch(it + 2, xk[0], xv[0]);
      work_on(it + 1, xk[1], xv[1]);
      fetch(it + 3, xk[1], xv[1]);
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ softmax: group w has row tile w (or the key tiles w, w + 2 ... of the one there is), a thread a row
    const int grp = (warp - 4) >> 2, quarter = warp & 3, row = (two ? grp * 128 : 0) + quarter * 32 + lane, rr = r0 + row;
    const bool live = row < nr;
    const int tok = live ? c0 + rr / per : t0, pos = live ? t.positions[tok] : -1;
    int least, most;
    {                                        // of the warp's rows
      const int w0 = row - lane, ra = min(r0 + w0, r0 + nr - 1), rb = min(r0 + w0 + 31, r0 + nr - 1);
      KvSpan own = span;
      own.p0 = t.positions[c0 + ra / per];
      own.p1 = t.positions[c0 + rb / per];
      kv_reach(t, a, own, c0 + ra / per, c0 + rb / per, &least, &most);
    }
    const uint32_t lane_at = tmem + ((uint32_t)(quarter * 32) << 16), s_at = lane_at + grp * (2 * FK), o_at = lane_at + kColO + grp * (64 * NV);
    // queries, a warp a row: scaled by a power of two, rounded to fp16, in the operand's layout (rows of 64 numbers, 16-byte pieces swizzled by the row).  A warp brings
    // its own rows; where both groups have the same, the first half of its group's 32.
    const int own = two ? 32 : 16, first_row = (two ? grp * 128 : 0) + quarter * 32 + (two ? 0 : grp * 16);
    const float sign = a.scale < 0.f ? -1.f : a.scale == 0.f ? 0.f : 1.f;  // factors on scores are positive: a row's maximum is its largest raw score's
    for (int i0 = 0; i0 < own; i0 += 16) {
      float x[16][(NC + 1) / 2][4];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = first_row + i0 + i, q = r0 + r, e = lane * 4;
        const long long from = r < nr ? (c0 + q / per) * a.ldq + (head * per + q % per) * a.hq : 0;
#pragma unroll
        for (int b = 0; b < (NC + 1) / 2; ++b) query4(a, from + b * 128 + e, r < nr ? c.d - b * 128 - e : 0, x[i][b]);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = first_row + i0 + i;
        uint32_t top = 0;
#pragma unroll
        for (int b = 0; b < (NC + 1) / 2; ++b)
#pragma unroll
          for (int j = 0; j < 4; ++j) top = max(top, __float_as_uint(x[i][b][j]) & 0x7FFFFFFFu);
        top = __reduce_max_sync(0xffffffffu, top);
        float up, undo;
        kv_row_scale(top, &up, &undo);
        up *= sign;
#pragma unroll
        for (int b = 0; b < (NC + 1) / 2; ++b) {
          const int e = b * 128 + lane * 4;
          if (e < NC * 64)
            *reinterpret_cast<uint2*>(smem + L::kOffQ + (r >> 7) * L::kQ + (e >> 6) * (128 * 128) + (r & 127) * 128 + ((((e & 63) >> 3) ^ (r & 7)) << 4) + (e & 4) * 2) =
                make_uint2(f16_pair(x[i][b][0] * up, x[i][b][1] * up), f16_pair(x[i][b][2] * up, x[i][b][3] * up));
        }
        if (lane == 0) rows_down[r] = sign == 0.f ? 1.f : fabsf(a.scale) * kLog2e * undo;
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(q_full);
    if (!two) named_bar_sync(kBarShare, 256);
    const float down = rows_down[row];
    float m = -INFINITY, l = 0.f, ref = 0.f, inv_ref = 0.f;
    int k = 0;                               // tiles of this group so far
    for (int it = two ? 0 : grp; it < n_tiles; it += two ? 1 : 2, ++k) {
      const int b = grp * 2 + (k & 1), turn = k >> 1 & 1;
      const uint32_t x_at = s_at + (k & 1) * FK;
      mbar_wait(&s_full[b], turn);
      tc_fence_after_sync();
      const float4 unit = units[(it >> 1) % kUnits];
      const uint32_t gone = __float_as_uint(unit.z) >> (it & 1) * 16 & 0xFFFFu;
      float x[FK];
      {
        uint32_t r[FK / 16][16];
#pragma unroll
        for (int i = 0; i < FK / 16; ++i) tmem_ld16(x_at + 16 * i, r[i]);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < FK; ++j) x[j] = __uint_as_float(r[j / 16][j % 16]);
      }
      const int ua = u0 + it * GT, ub = min(ua + GT, u1) - 1;              // groups of the tile
      const int pa = span.group(ua) * kKvGroup, pb = span.group(ub) * kKvGroup + kKvGroup - 1;
      const bool all = gone == 0 && ub == ua + GT - 1 && pb < span.base && pb <= least && (pb < a.first || (ua >= span.na && most - pa < a.window));
      if (!all) {
#pragma unroll
        for (int g = 0; g < GT; ++g) {
          const int u = ua + g, j0 = span.group(u) * kKvGroup;
          uint32_t see = 0;
          if (u < u1 && live && !(gone >> 4 * g & 1u)) {
            if (j0 + kKvGroup <= span.base) {                              // the positions of a group that are no further than the row's, and near enough or among the first
              see = pos < j0 ? 0u : pos - j0 >= 15 ? 0xFFFFu : (2u << (pos - j0)) - 1;
              const int far = pos - a.window - j0 + 1;                     // these of the group lie ahead of the window
              if (far > 0) see &= (far >= 16 ? 0u : 0xFFFFu << far) | (a.first <= j0 ? 0u : a.first - j0 >= 16 ? 0xFFFFu : (1u << (a.first - j0)) - 1);
            } else {
#pragma unroll 1
              for (int j = 0; j < 16; ++j) see |= (uint32_t)kv_sees(t, a, span, c0, n, tok, pos, j0 + j) << j;
            }
          }
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (!(see >> j & 1u)) x[16 * g + j] = -INFINITY;
        }
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < FK; j += 2) mx[j >> 1 & 3] = max3(mx[j >> 1 & 3], x[j], x[j + 1]);
      const float fac = fminf(fmaxf(down * unit.x, 1e-37f), 1e37f);
      const float mt = max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]) * fac;
      // a new maximum, or values whose unit may take a weight beyond fp16: seldom after the first tiles
      if (__any_sync(0xffffffffu, mt > m || unit.y > (inv_ref == 0.f ? 0.f : ref * 32768.f))) {
        const float mn = fmaxf(m, mt), from = mn == -INFINITY ? 0.f : mn, back = ex2(m - from);
        m = mn;
        l *= back;
        ref *= back;
        const float big = ex2(mt - from) * unit.y;                         // the tile's largest weight times unit
        float grow = 1.f;
        const float least = fmaxf(unit.y * 7.8886091e-31f, 1e-37f);        // 2^-100 of the unit: 1 / ref times it stays within fp32
        if (big > 1e-37f && (big > ref * 32768.f || ref < least)) {
          const float r = fmaxf(big * 0.015625f, least);
          grow = ref / r;
          ref = r;
        }
        inv_ref = ref >= least ? 1.f / ref : 0.f;                          // no reference: what the tile's weights come to is nothing
        if (k > 0 && __any_sync(0xffffffffu, grow != 1.f)) {
          mbar_wait(&pv_done[grp * 2 + ((k - 1) & 1)], (k - 1) >> 1 & 1);  // O holds every product so far
          tc_fence_after_sync();
#pragma unroll 2
          for (int o = 0; o < 64 * NV; o += 16) {
            uint32_t r[16];
            tmem_ld16(o_at + o, r);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * grow);
            tmem_st16(o_at + o, r);
          }
        }
      }
      const float from = m == -INFINITY ? 0.f : m, f = unit.y * inv_ref;
      const uint64_t fac2 = pair_of(fac, fac), neg2 = pair_of(-from, -from), f2 = pair_of(f, f);
      uint64_t sum[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < FK / 32; ++i) {
        uint32_t pk[16];
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          const float2 e = pair_get(pair_fma(pair_of(x[32 * i + j], x[32 * i + j + 1]), fac2, neg2));
          const uint64_t p = pair_of(ex2(e.x), ex2(e.y));
          sum[j >> 1 & 1] = pair_add(sum[j >> 1 & 1], p);
          const float2 y = pair_get(pair_mul(p, f2));
          pk[j / 2] = f16_pair(y.x, y.y);
        }
        tmem_st16(x_at + 16 * i, pk);
      }
      const float2 s2 = pair_get(pair_add(sum[0], sum[1]));
      l += s2.x + s2.y;
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[b]);
    }
    if (k > 0) {
      mbar_wait(&pv_done[grp * 2 + ((k - 1) & 1)], (k - 1) >> 1 & 1);      // products end in their order
      tc_fence_after_sync();
    }
    const int hd = head * per + rr % per;
    const bool whole = seq_parts->first < 0;
    const long long orow = (long long)tok * a.H + hd;
    const int part = whole ? 0 : seq_parts->first + ((tok - c0) * a.H + hd) * seq_parts->pieces;
    const bool kept = live && (whole || (unsigned)part < (unsigned)a.parts);
    float ref1 = 0.f;
    constexpr int kPad = 64 * NV + 1;        // numbers a row, an odd number: a row a thread meets every bank once
    float* share = reinterpret_cast<float*>(smem + L::kOffQ) + (quarter * 32 + lane) * kPad;
    float* stat = reinterpret_cast<float*>(smem + L::kOffQ) + 128 * kPad + (quarter * 32 + lane) * 3;
    if (!two) {                              // the second group's share goes through the operands' memory, which no product reads any more once both groups are here
      named_bar_sync(kBarShare, 256);
      if (grp == 1) {
        for (int o = 0; o < 64 * NV; o += 16) {
          uint32_t r[16];
          if (k > 0) {
            tmem_ld16(o_at + o, r);
            tmem_ld_wait();
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) share[o + j] = k > 0 ? __uint_as_float(r[j]) : 0.f;
        }
        stat[0] = m;
        stat[1] = l;
        stat[2] = ref;
      }
      named_bar_sync(kBarShare, 256);
      if (grp == 0) {
        const float m1 = stat[0], mn = fmaxf(m, m1), from = mn == -INFINITY ? 0.f : mn, back = ex2(m - from), back1 = ex2(m1 - from);
        l = l * back + stat[1] * back1 + (stat[1] != stat[1] ? stat[1] : 0.f);
        ref *= back;
        ref1 = stat[2] * back1;
        m = mn;
      }
    }
    if (two || grp == 0) {
      if (whole && live && a.sinks != nullptr && m != -INFINITY) l += ex2(fmaf(a.sinks[hd], kLog2e, -m));
      const float inv = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f, by = ref * inv, by1 = ref1 * inv, none = l != l ? l : 0.f;      // a NaN may have a reference of 0
      if (!whole && kept) {
        a.part_ml[2ll * part] = m;
        a.part_ml[2ll * part + 1] = l;
      }
#pragma unroll 2
      for (int o = 0; o < 64 * NV; o += 16) {
        uint32_t r[16];
        __syncwarp();                          // the warp reads tensor memory together
        tmem_ld16(o_at + o, r);
        tmem_ld_wait();
        if (!kept || o >= c.dv) continue;
        float y[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) y[j] = __uint_as_float(r[j]) * by + none;
        if (!two) {
#pragma unroll
          for (int j = 0; j < 16; ++j) y[j] = fmaf(share[o + j], by1, y[j]);
        }
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
  } else {
    if (warp == 1) {
      // ---------------------------------------------------------- plans: lane l has the rows 4 l .. 4 l + 3 of two tiles
      const auto at_row = [&](int p) {
        const int u = u0 + p * (2 * GT) + lane / 4;
        const long long r = u < u1 ? kv_row(c, t, s, span.group(u) * kKvGroup) : -1;
        return r < 0 ? -1ll : r + ((long long)head << c.lps);
      };
      long long r = at_row(0);
      for (int p = 0; p < (n_tiles + 1) / 2; ++p) {
        float ks[4] = {}, vs[4] = {};
        if (r >= 0) {
          const float4 x = *reinterpret_cast<const float4*>(c.ks + r + (lane & 3) * 4), y = *reinterpret_cast<const float4*>(c.vs + r + (lane & 3) * 4);
          ks[0] = x.x; ks[1] = x.y; ks[2] = x.z; ks[3] = x.w;
          vs[0] = y.x; vs[1] = y.y; vs[2] = y.z; vs[3] = y.w;
        }
        const long long next = at_row(p + 1);
        uint32_t kt = 0, vt = 0;             // the largest scales of rows that any row of the tile sees
        const int j0 = span.group(u0 + p * (2 * GT) + lane / 4) * kKvGroup + (lane & 3) * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (!(j0 + e < span.hi && (j0 + e >= span.lo || j0 + e < a.first))) ks[e] = vs[e] = 0.f;
          const uint32_t x = __float_as_uint(ks[e]), y = __float_as_uint(vs[e]);
          if (x < 0x7F800000u) kt = max(kt, x);
          if (y < 0x7F800000u) vt = max(vt, y);
        }
        float kp, ki, vp, vi;
        scale_unit(__reduce_max_sync(0xffffffffu, kt), &kp, &ki);
        vt = __reduce_max_sync(0xffffffffu, vt);
        scale_unit(vt, &vp, &vi);
        uint32_t f[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool none = vs[e] != vs[e];  // a row that is no number: its keys say so
          f[e] = f16_pair(none ? vs[e] : ks[e] * ki, none ? 0.f : vs[e] * vi);
        }
        const int slot = p % kPlans;
        mbar_wait(&plan_empty[slot], (p / kPlans & 1) ^ 1);
        *reinterpret_cast<uint4*>(factors + slot * 128 + lane * 4) = make_uint4(f[0], f[1], f[2], f[3]);
        if ((lane & 3) == 0) groups[slot * 8 + lane / 4] = r < 0 ? -1 : (int)(r / kKvGroup);
        const uint32_t gone = __ballot_sync(0xffffffffu, r < 0);
        if (lane == 0) units[p % kUnits] = make_float4(kp, vt ? vp : 0.f, __uint_as_float(gone), 0.f);
        __syncwarp();
        if (lane == 0) mbar_arrive(&plan_full[slot]);
        r = next;
      }
    } else if (warp == 0 || warp == 3) {
      // ---------------------------------------------------------- tensor cores.  A warp for each row tile: the tensor cores take few products ahead (two or so), so what a warp does
      // between its batches (waits, commits: some 300 cycles) is hidden by the other's.  S(k + 2) lies where P(k) did and waits for the second product of k.
      const int g = warp == 3;
      const uint32_t id_s = idesc_f16(FK, false), id_o = idesc_f16(64 * NV, true);
      const uint32_t q_at = smem_u32(smem + L::kOffQ), k_at = smem_u32(smem + L::kOffK), v_at = smem_u32(smem + L::kOffV);
      const auto scores = [&](int k) {                              // S = Q K^T of the group's tile k
        const int it = two ? k : 2 * k + g, b = it % L::kKeys, x = g * 2 + (k & 1);
        if (it >= n_tiles) return;
        mbar_wait(&k_full[b], it / L::kKeys & 1);
        if (k >= 2) mbar_wait(&pv_done[x], ((k - 2) >> 1) & 1);
        tc_fence_after_sync();
        if (elect_one()) {
#pragma unroll
          for (int h = 0; h < NC; ++h) {
            const uint64_t ad = umma_desc_k_sw128(q_at + (two ? g : 0) * L::kQ + h * (128 * 128)), bd = umma_desc_k_sw128(k_at + b * L::kK + h * (FK * 128));
#pragma unroll
            for (int i = 0; i < 4; ++i) umma_bf16(tmem + x * FK, ad + 2 * i, bd + 2 * i, id_s, h > 0 || i > 0 ? 1u : 0u);
          }
          umma_commit(&s_full[x]);
          umma_commit(&k_empty[b]);
        }
        __syncwarp();
      };
      const auto output = [&](int k) {                              // O += P V
        const int it = two ? k : 2 * k + g, b = it % kBufs, x = g * 2 + (k & 1);
        if (it >= n_tiles) return;
        mbar_wait(&v_full[b], it / kBufs & 1);
        mbar_wait(&p_full[x], k >> 1 & 1);
        tc_fence_after_sync();
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < FK / 16; ++i)
            umma_bf16_ts(tmem + kColO + g * (64 * NV), tmem + x * FK + 8 * i, desc_mn(v_at + b * L::kV + i * 2048, FK * 128), id_o, k > 0 || i > 0 ? 1u : 0u);
          umma_commit(&pv_done[x]);
          umma_commit(&v_empty[b]);
        }
        __syncwarp();
      };
      mbar_wait(q_full, 0);
      scores(0);
      scores(1);
      for (int k = 0; (two ? k : 2 * k + g) < n_tiles; ++k) {
        output(k);
        scores(k + 2);
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
  using L = PairShape<NC, NV>;
  SEQ_CUDA((kb2::allow_smem<kv_pair_kernel<FMT, NC, NV>>(L::kTotal)));
  auto kern = kv_pair_kernel<FMT, NC, NV>;
  kb2::launch_pdl(kern, dim3(tiles, c.G), kThreads, L::kTotal, st, c, t, a, kinds);
  SEQ_LAUNCHED();
  return KB2SEQ_OK;
}
template <int FMT>
int sizes(const KvLayer& c, const KvStep& t, const KvAttn& a, const KvKinds& kinds, int tiles, cudaStream_t st) {
  if (c.d <= 64 && c.dv <= 64) return launch<FMT, 1, 1>(c, t, a, kinds, tiles, st);
  return c.d <= 128 ? launch<FMT, 2, 2>(c, t, a, kinds, tiles, st) : launch<FMT, 3, 2>(c, t, a, kinds, tiles, st);
}
}  // namespace

int kv_pair_attend(int fmt, const KvLayer& c, const KvStep& t, const KvAttn& a, const KvKinds& kinds, int tiles, cudaStream_t stream) {
  return fmt == KV_E4M3 ? sizes<KV_E4M3>(c, t, a, kinds, tiles, stream) : sizes<KV_INT8>(c, t, a, kinds, tiles, stream);
}

}  // namespace kb2seq
