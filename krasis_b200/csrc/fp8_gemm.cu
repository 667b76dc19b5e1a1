// Products of 8-bit floating-point operands with a scale per block of 128 (fp8.cuh): out[m][n] = sum_b xs[m][b] ws[n / 128][b] sum_{k in block b} x[m][k] w[n][k], of one matrix or of
// runs of rows that have a matrix each (routed experts).
//
// The scales are any fp32 numbers, by which the tensor cores' accumulators cannot be rescaled on the way (the products that scale their operands take powers of two alone), so each
// block of 128 products per result is a sum of its own in tensor memory (two of them in turn), which sixteen warps multiply by its
// scales and add up in registers, 64 sums a thread, while the next one runs.  The rows of x are the M side: a thread has one row, so one scale of it per block, and 64 columns of one
// block of weights.  With the weights there a column's scale came from shared memory, 512 bytes of a warp's loads for every 16 numbers: 1024 cycles a block of 128
// rows (8192 x 10 rows of 512 experts: 325 us a product, 225 so).  A tile is 256 weight rows, and
//   one CTA has 128 rows of x: runs, and matrices whose tiles fill the SMs better so.  Few rows cost the same 512 cycles of MMAs a block, less than its 32 KB of weights take from
//     memory (1380 cycles at the copy rate): 64 experts of 3 x 1408 x 2048 and 2334 rows take 66 + 40 us for 57 + 32 of weights, rows and results at that rate, 512 of 3 x 512 x 2048 and
//     81920 rows 270 + 215 for 197 + 191 (results in fp32).  Pairs for such runs: 285 us a product against 211; at 8192 rows an expert 161 against 162;
//   a pair of CTAs has 256, each half of the weights, so that a block's 32 KB of loads feed 512 cycles of its MMAs: many rows.  M 8192, N 12288, K 2048: 187 us, 2210 TFLOP/s; N 4096,
//     K 4096: 117 us, 2345 of the 3341 that twice the bf16 rate is.  The tensor pipe is busy 61 % of the time, the issue slots 56 %;
//   a cluster of 2 to 8 shares 128 rows along K, where tiles are fewer than SMs; the CTAs' sums meet in shared memory and are added in the order of the ranks.
// Gated units: 32 rows of gate and of up in turn, so that a thread has both numbers of 32 units, and the four warps of its row all 128 of a scale.
#include <cuda.h>

#include <atomic>

#include "fp8.cuh"
#include "prof.cuh"

namespace kb2 {

cudaError_t make_tmap_u8_rows(void* out_tmap, const void* base, long long rows, long long cols, int box_rows);

constexpr int kTRows = kFp8Run, kTBox = 32, kTABytes = kTRows * 128, kTWBytes = 256 * 128;
// One CTA, a cluster that shares a tile along K, or a pair of CTAs that multiplies as one.
enum Fp8Ctas { kAlone, kSplit, kPair };
__host__ __device__ constexpr int tile_stage(int ctas) { return kTABytes + kTWBytes / (ctas == kPair ? 2 : 1); }
constexpr int kTWarps = 16, kTThreads = 32 * (kTWarps + 4);
// The scales of kTGroup blocks are handed over at once, two groups are at hand: products for each row, for the first and the second 128 columns.
constexpr int kTGroup = 4, kTScales = 2 * kTGroup;
constexpr int kTOut = 32 * 128;                    // a warp's results on their way out
__host__ __device__ constexpr int tile_stages(bool glu, int ctas) { return glu || ctas == kPair ? 4 : 3; }      // gated units have nothing on its way out in shared memory
constexpr int kTOffOut = 3 * tile_stage(kAlone), kTOffScale = kTOffOut + kTWarps * kTOut, kTOffMax = kTOffScale + kTScales * 2 * kTRows * 4, kTOffBar = kTOffMax + 2 * 4 * kTRows * 4, kTSmem = kTOffBar + 512;
constexpr int kTPart = 260;                        // numbers from row to row of the sums that a cluster joins
static_assert(4 * tile_stage(kAlone) <= kTOffScale && 4 * tile_stage(kPair) <= kTOffOut && kTRows * kTPart * 4 <= kTOffOut && kTSmem <= 227 * 1024 && kTSmem >= 512 * 430 - 1024, "stages, results and scales; what a CTA of a cluster takes for 512 columns (tmem_smem)");

// silu(g) u with one approximate power of two and one approximate reciprocal: off by 2^-21 of it, and for g below zero by |g| 2^-24 more, which is less than the rounding of g moves it.
// Below g = -87.3 the reciprocal of 1 + e^-g, less than 2^-126, is flushed and the unit is 0 instead of 1e-36 u or less.
__device__ __forceinline__ float gated(float g, float u) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return g * r * u;
}

struct TileArgs {
  Fp8Product p;
  int w_tiles;                                     // tiles of 256 weight rows (gated: 128 of either half)
  int split;                                       // CTAs of a cluster that share a tile along K
  // gated units: out is codes [M][N / 2] with scales
  float* out_scales;
  long long ld_out_scales;
};

template <bool kGlu, bool kOutF32, int kCtas>
__global__ void __launch_bounds__(kTThreads, 1)
    fp8_tile_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_out, const TileArgs a) {
  constexpr int kTStages = tile_stages(kGlu, kCtas), kTStage = tile_stage(kCtas);
  constexpr int kRun = kCtas == kPair ? 2 * kTRows : kTRows;            // the most rows of a run
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kTOffBar);         // a pair's: of the first CTA, for both CTAs' loads
  uint64_t* empty = full + kTStages;
  uint64_t* acc_full = empty + kTStages;           // [2]
  uint64_t* acc_empty = acc_full + 2;              // [2], a pair's: of the first CTA
  uint64_t* s_full = acc_empty + 2;                // [2]
  uint64_t* s_empty = s_full + 2;
  uint32_t* tmem_ptr_smem = reinterpret_cast<uint32_t*>(s_empty + 2);
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const Fp8Product& p = a.p;
  if (threadIdx.x == 32) {
    if (smem_u32(smem) & 1023u) __trap();
    for (int i = 0; i < kTStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], (kCtas == kPair ? 2 : 1) * kTWarps);
      mbar_init(&s_full[i], 2);
      mbar_init(&s_empty[i], kTWarps);
    }
    fence_mbar_init();
  }
  if (threadIdx.x == 64) {
    prefetch_tmap(&tmap_x);
    prefetch_tmap(&tmap_w);
    prefetch_tmap(&tmap_out);
  }
  if (warp == 0) {
    if constexpr (kCtas == kPair) tmem_alloc_pair(tmem_ptr_smem, 512);
    else tmem_alloc(tmem_ptr_smem, 512);
  }
  tc_fence_before_sync();
  __syncthreads();
  if constexpr (kCtas == kPair) cluster_sync_all();      // the other CTA's barriers are there
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_ptr_smem;
  pdl_wait();
  const int blocks = fp8_blocks(p.K), total = (p.chunks ? p.n_chunks[0] : (p.M + kRun - 1) / kRun) * a.w_tiles;
  // with a split, one tile and some of its blocks of K; else every gridDim.x-th tile
  const int rank = kCtas != kAlone ? (int)cluster_rank() : 0, first = kCtas == kSplit ? (int)blockIdx.x / a.split : kCtas == kPair ? (int)blockIdx.x >> 1 : (int)blockIdx.x,
            step = kCtas == kSplit ? total : kCtas == kPair ? (int)gridDim.x >> 1 : (int)gridDim.x;
  const int kb0 = kCtas == kSplit ? blocks * rank / a.split : 0, nb = kCtas == kSplit ? blocks * (rank + 1) / a.split - kb0 : blocks;
  struct Item {
    int row0, rows, group, wt;
    int boxes;                                     // of a pair's rows in all
  };
  // weight tiles first, so that CTAs that run at once share the rows of x.  Everyone asks for the next item when it starts on one.
  const auto item = [&](int t) {
    Item i;
    const int u = t / a.w_tiles;
    i.wt = t - u * a.w_tiles;
    if (p.chunks) {
      const int4 c = t < total ? *reinterpret_cast<const int4*>(p.chunks + u) : make_int4(0, 0, 0, 0);
      i.row0 = c.y;
      i.rows = c.z;
      i.group = c.x;
    } else {
      i.row0 = u * kRun;
      i.rows = t < total ? min(kRun, p.M - i.row0) : 0;
      i.group = 0;
    }
    if constexpr (kCtas == kPair) {                // half of the rows each, in boxes
      const int half = min(i.rows, ((i.rows + 1) / 2 + kTBox - 1) & ~(kTBox - 1));
      i.boxes = (half + kTBox - 1) / kTBox + (i.rows - half + kTBox - 1) / kTBox;
      i.row0 += rank * half;
      i.rows = rank ? i.rows - half : half;
    }
    return i;
  };

  if (warp >= 4) {
    more_registers<112>();
    const int q = warp & 3, h = (warp - 4) >> 2, row = q * 32 + lane;     // of the run
    const uint32_t from = tmem_base + ((uint32_t)(q * 32) << 16) + h * 64;
    int b = 0;
    uint32_t aphase = 0, slot = 0, sphase = 0, tile = 0;
    Item next = item(first);
    for (int t = first; t < total; t += step, ++tile) {
      const Item i = next;
      next = item(t + step);
      const bool mine = __any_sync(0xffffffffu, row < i.rows);
      uint64_t acc[32];                            // two columns in each
#pragma unroll
      for (int j = 0; j < 32; ++j) acc[j] = 0;
      for (int kb = 0; kb < nb; ++kb) {
        if ((slot & (kTGroup - 1)) == 0) mbar_wait(&s_full[slot / kTGroup], sphase);
        const uint32_t* sc = reinterpret_cast<const uint32_t*>(smem + kTOffScale) + slot * 2 * kTRows + q * 32 + lane;
        const uint32_t s0 = sc[kGlu ? 0 : (h >> 1) * kTRows], s1 = kGlu ? sc[kTRows] : s0;
        const uint64_t two[2] = {pack2(s0, s0), pack2(s1, s1)};
        mbar_wait(&acc_full[b], aphase);
        tc_fence_after_sync();
        const auto read = [&]() {                  // this block's sums are in registers
          tc_fence_before_sync();
          __syncwarp();
          if (lane != 0) return;
          if constexpr (kCtas == kPair) mbar_arrive_cluster_relaxed(cluster_addr(&acc_empty[b], 0));
          else mbar_arrive(&acc_empty[b]);
        };
        if (mine) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t v[32];
            tmem_ld32(from + b * 256 + c * 32, v);
            tmem_ld_wait();
            if (c) read();
#pragma unroll
            for (int j = 0; j < 16; ++j) fma2_here(acc[c * 16 + j], pack2(v[2 * j], v[2 * j + 1]), two[c]);
          }
        } else {
          read();
        }
        ++slot;
        if ((slot & (kTGroup - 1)) == 0) {
          if (lane == 0) mbar_arrive(&s_empty[slot / kTGroup - 1]);
          if (slot == kTScales) { slot = 0; sphase ^= 1; }
        }
        b ^= 1;
        aphase ^= b == 0;
      }
      if constexpr (kGlu) {
        // columns 0 to 31 are gate, the others up of units 32 h on of the tile's 128
        uint32_t* most = reinterpret_cast<uint32_t*>(smem + kTOffMax) + (tile & 1) * 4 * kTRows + row;
        uint32_t m = 0;
        if (mine) {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float g0, g1, u0, u1;
            unpack2(acc[j], g0, g1);
            unpack2(acc[16 + j], u0, u1);
            const uint32_t v0 = __float_as_uint(gated(g0, u0)), v1 = __float_as_uint(gated(g1, u1));
            acc[j] = pack2(v0, v1);
            m = max(m, max(v0 & 0x7FFFFFFFu, v1 & 0x7FFFFFFFu));
          }
        }
        most[h * kTRows] = m;
        named_bar_sync(1 + q, 128);                // the four warps of these rows; the tile after next writes here again, behind the next one's barrier
        if (row < i.rows) {
          const Fp8Scale f = fp8_scale(max(max(most[0], most[kTRows]), max(most[2 * kTRows], most[3 * kTRows])));
          const long long at = i.row0 + row;
          if (h == 0) a.out_scales[i.wt * a.ld_out_scales + at] = f.scale;
          uint32_t w[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float v0, v1, v2, v3;
            unpack2(acc[2 * j], v0, v1);
            unpack2(acc[2 * j + 1], v2, v3);
            w[j] = fp8_codes4(v0, v1, v2, v3, f.inv);
          }
          uint4* to = reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(p.out) + at * (p.N / 2) + i.wt * 128 + h * 32);
          to[0] = make_uint4(w[0], w[1], w[2], w[3]);
          to[1] = make_uint4(w[4], w[5], w[6], w[7]);
        }
      } else if constexpr (kCtas == kSplit) {
        // the ring is free: all of this CTA's products are done
        if (mine) {
          float* part = reinterpret_cast<float*>(smem) + row * kTPart + h * 64;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float v[4];
            unpack2(acc[2 * j], v[0], v[1]);
            unpack2(acc[2 * j + 1], v[2], v[3]);
            *reinterpret_cast<float4*>(part + 4 * j) = make_float4(v[0], v[1], v[2], v[3]);
          }
        }
      } else if (mine) {
        // 32 rows x 128 bytes at a time go out from shared memory by one copy, while the next tile's blocks are added: all SMs end their tiles at the same time, and a tile's
        // stores by the lanes took 3500 cycles (16 bytes of a row by each lane, row by row, 12000).  A run's last rows, as the next run's follow them, and rows that are not on
        // 16 bytes are the lanes'.
        constexpr int kCols = kOutF32 ? 32 : 64, kVec = kOutF32 ? 4 : 8;
        uint8_t* st = smem + kTOffOut + (warp - 4) * kTOut;
        const int row0 = i.row0 + q * 32, have = i.rows - q * 32;
        const bool on16 = p.N % kVec == 0;
#pragma unroll
        for (int c = 0; c < 64 / kCols; ++c) {
          const int n0 = i.wt * 256 + h * 64 + c * kCols;
          if (n0 >= p.N) break;
          if (lane == 0) bulk_wait_group_read0();
          __syncwarp();
#pragma unroll
          for (int j = 0; j < kCols; j += kVec) {
            float v[kVec];
#pragma unroll
            for (int k = 0; k < kVec; k += 2) unpack2(acc[(c * kCols + j + k) / 2], v[k], v[k + 1]);
            if (p.bias != nullptr)
#pragma unroll
              for (int k = 0; k < kVec; ++k) v[k] += n0 + j + k < p.N ? p.bias[n0 + j + k] : 0.f;
            uint4 x;
            if constexpr (kOutF32) x = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
            else x = make_uint4(bf16x2_bits_rn(v[1], v[0]), bf16x2_bits_rn(v[3], v[2]), bf16x2_bits_rn(v[5], v[4]), bf16x2_bits_rn(v[7], v[6]));
            *reinterpret_cast<uint4*>(st + lane * 128 + (j / kVec ^ (lane & 7)) * 16) = x;       // the order that the copy reads them in
          }
          if (on16 && have >= 32) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&tmap_out, n0 * (kOutF32 ? 4 : 2), row0, st);
              bulk_commit_group();
            }
            continue;
          }
          __syncwarp();
          const int n = n0 + (lane & 7) * kVec;
          for (int r = lane >> 3; r < min(have, 32); r += 4) {
            if (n >= p.N) continue;
            const uint4 x = *reinterpret_cast<const uint4*>(st + r * 128 + ((lane & 7) ^ (r & 7)) * 16);
            const long long to = (long long)(row0 + r) * p.N + n;
            if (on16) {
              *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(p.out) + to * (16 / kVec)) = x;
            } else if (p.N % (kVec / 2) == 0) {
              uint2* at = reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(p.out) + to * (16 / kVec));
              at[0] = make_uint2(x.x, x.y);
              if (n + kVec / 2 < p.N) at[1] = make_uint2(x.z, x.w);
            } else {
              const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
              for (int y = 0; y < kVec; ++y) {
                if (n + y >= p.N) continue;
                if constexpr (kOutF32) reinterpret_cast<float*>(p.out)[to + y] = __uint_as_float(u[y]);
                else reinterpret_cast<__nv_bfloat16*>(p.out)[to + y] = __ushort_as_bfloat16((unsigned short)(u[y >> 1] >> (y & 1) * 16));
              }
            }
          }
        }
      }
    }
    if (!kGlu && kCtas != kSplit && lane == 0) bulk_wait_group0();
    if constexpr (kCtas == kSplit) {
      __syncwarp();
      cluster_sync_all();                          // every CTA's sums are there
      const Item i = item(first);
      for (int x = rank + (warp - 4 >> 1) * a.split; x < i.rows; x += kTWarps / 2 * a.split) {       // two warps a row, four columns a lane
        const int c = (warp & 1) * 128 + lane * 4, n = i.wt * 256 + c;
        if (n >= p.N) continue;
        float s[4] = {};
        for (int r = 0; r < a.split; ++r) {
          float4 v;
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                       : "r"(cluster_addr(reinterpret_cast<float*>(smem) + x * kTPart + c, r))
                       : "memory");
          s[0] += v.x;
          s[1] += v.y;
          s[2] += v.z;
          s[3] += v.w;
        }
        if (p.bias != nullptr)
#pragma unroll
          for (int k = 0; k < 4; ++k) s[k] += n + k < p.N ? p.bias[n + k] : 0.f;
        const long long at = (long long)(i.row0 + x) * p.N + n;
        if constexpr (kOutF32) {
          float* to = reinterpret_cast<float*>(p.out) + at;
          if ((p.N & 3) == 0) *reinterpret_cast<float4*>(to) = make_float4(s[0], s[1], s[2], s[3]);
          else
            for (int k = 0; k < 4; ++k)
              if (n + k < p.N) to[k] = s[k];
        } else {
          __nv_bfloat16* to = reinterpret_cast<__nv_bfloat16*>(p.out) + at;
          if ((p.N & 3) == 0) *reinterpret_cast<uint2*>(to) = make_uint2(bf16x2_bits_rn(s[1], s[0]), bf16x2_bits_rn(s[3], s[2]));
          else
            for (int k = 0; k < 4; ++k)
              if (n + k < p.N) to[k] = __float2bfloat16_rn(s[k]);
        }
      }
      __syncwarp();
      cluster_sync_all();                          // nobody's sums go while a peer still reads them
    }
  } else if (fewer_registers<32>(), warp == 0) {
    int stage = 0;
    uint32_t phase = 0;
    Item next = item(first);
    for (int t = first; t < total; t += step) {
      const Item i = next;
      next = item(t + step);
      const int rows = (i.rows + kTBox - 1) & ~(kTBox - 1);    // in boxes; what lies behind them in a stage is multiplied, too, and looked at by nobody
      const int w0 = i.group * p.N + i.wt * (kGlu ? 128 : 256);
      for (int kb = 0; kb < nb; ++kb) {
        mbar_wait(&empty[stage], phase ^ 1);
        uint8_t* at = smem + stage * kTStage;
        if (elect_one()) {
          const int k = (kb0 + kb) * 128;
          if constexpr (kCtas == kPair) {          // this CTA's rows and its half of the weights
            const uint32_t bar = cluster_addr(&full[stage], 0);
            if (rank == 0) mbar_arrive_expect_tx(&full[stage], kTWBytes + i.boxes * kTBox * 128);
            tma_load_2d_pair(at + kTABytes, &tmap_w, k, w0 + rank * 128, bar);
            for (int r = 0; r < rows; r += kTBox) tma_load_2d_pair(at + r * 128, &tmap_x, k, i.row0 + r, bar);
          } else {
            mbar_arrive_expect_tx(&full[stage], kTWBytes + rows * 128);
            if constexpr (kGlu) {                  // 32 rows of gate and of up in turn
              for (int r = 0; r < 128; r += 32) {
                tma_load_2d(at + kTABytes + r * 256, &tmap_w, k, w0 + r, &full[stage]);
                tma_load_2d(at + kTABytes + r * 256 + 4096, &tmap_w, k, w0 + p.N / 2 + r, &full[stage]);
              }
            } else {
              tma_load_2d(at + kTABytes, &tmap_w, k, w0, &full[stage]);
            }
            for (int r = 0; r < rows; r += kTBox) tma_load_2d(at + r * 128, &tmap_x, k, i.row0 + r, &full[stage]);
          }
        }
        __syncwarp();
        if (++stage == kTStages) { stage = 0; phase ^= 1; }
      }
    }
    for (int i = 0; i < kTStages; ++i) {           // the last reports of freed stages have arrived, too
      mbar_wait(&empty[stage], phase ^ 1);
      if (++stage == kTStages) { stage = 0; phase ^= 1; }
    }
  } else if (warp == 1) {
    int stage = 0, b = 0;
    uint32_t phase = 0, aphase = 0;
    const uint32_t idesc = umma_idesc_e4m3(kRun, 256);
    for (int t = first; t < total && (kCtas != kPair || rank == 0); t += step) {
      for (int kb = 0; kb < nb; ++kb) {
        mbar_wait(&full[stage], phase);
        mbar_wait(&acc_empty[b], aphase ^ 1);
        tc_fence_after_sync();
        const uint32_t addr = smem_u32(smem + stage * kTStage);
        const uint64_t ad = umma_desc_k_sw128(addr), bd = umma_desc_k_sw128(addr + kTABytes);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if constexpr (kCtas == kPair) umma_f8_pair(tmem_base + b * 256, ad + 2 * k, bd + 2 * k, idesc, k > 0 ? 1u : 0u);
            else umma_f8(tmem_base + b * 256, ad + 2 * k, bd + 2 * k, idesc, k > 0 ? 1u : 0u);
          }
          if constexpr (kCtas == kPair) {
            umma_commit_pair(&acc_full[b]);
            umma_commit_pair(&empty[stage]);
          } else {
            umma_commit(&acc_full[b]);
            umma_commit(&empty[stage]);
          }
        }
        __syncwarp();
        if (++stage == kTStages) { stage = 0; phase ^= 1; }
        b ^= 1;
        aphase ^= b == 0;
      }
    }
  } else {
    // The scales, by two warps in turn: the rows' times the weights'.  Each has two blocks' on their way at once, as that takes longer than a block's products.
    const int w_blocks = fp8_blocks(p.N);
    struct Scales {
      float x[4], w[2];
    };
    int t = first, kb = warp - 2;
    const auto settle = [&]() {
      while (kb >= nb && t < total) {
        kb -= nb;
        t += step;
      }
    };
    settle();
    Item i = item(t);
    const auto ask = [&](Scales& s) {
      const int n = kGlu ? i.wt : i.wt * 2, n1 = kGlu ? i.wt + w_blocks / 2 : min(n + 1, w_blocks - 1);
      const float *w = p.ws + (long long)i.group * w_blocks * blocks + kb0 + kb, *x = p.xs + (kb0 + kb) * p.ldxs + i.row0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = j * 32 + lane;
        s.x[j] = row < i.rows ? x[row] : 0.f;
      }
      s.w[0] = w[(long long)n * blocks];
      s.w[1] = w[(long long)n1 * blocks];
      const int was = t;
      kb += 2;
      settle();
      if (t != was) i = item(t);
    };
    uint32_t slot = warp - 2, phase = 0;
    const auto put = [&](const Scales& s) {
      if ((slot & (kTGroup - 1)) < 2) mbar_wait(&s_empty[slot / kTGroup], phase ^ 1);
      float* to = reinterpret_cast<float*>(smem + kTOffScale) + slot * 2 * kTRows + lane;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        to[j * 32] = s.x[j] * s.w[0];
        to[kTRows + j * 32] = s.x[j] * s.w[1];
      }
      __syncwarp();
      if ((slot & (kTGroup - 1)) >= kTGroup - 2 && lane == 0) mbar_arrive(&s_full[slot / kTGroup]);
      slot += 2;
      if (slot >= kTScales) { slot -= kTScales; phase ^= 1; }
    };
    const int all = total > first ? (total - first + step - 1) / step * nb : 0, mine = (all - (warp - 2) + 1) / 2;
    Scales s0{}, s1{};
    if (mine > 0) ask(s0);
    if (mine > 1) ask(s1);
    for (int n = 0; n < mine; n += 2) {
      put(s0);
      if (n + 2 < mine) ask(s0);
      if (n + 1 < mine) put(s1);
      if (n + 3 < mine) ask(s1);
    }
    if (all % kTGroup > 0 && all % kTGroup < kTGroup - 3 + warp) {         // the last group is short: of either warp's two blocks, one or both are missing
      if (all % kTGroup == 1 && warp == 3) mbar_wait(&s_empty[slot / kTGroup], phase ^ 1);
      if (lane == 0) mbar_arrive(&s_full[slot / kTGroup]);
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  if (kCtas == kSplit && warp < 4) {                        // as the others do (above); nothing that takes registers stands behind the roles
    cluster_sync_all();
    cluster_sync_all();
  }
  __syncthreads();
  if constexpr (kCtas == kPair) cluster_sync_all();      // nobody leaves while the other may still report to its barriers
  tc_fence_after_sync();
  if (warp == 0) {
    if constexpr (kCtas == kPair) tmem_dealloc_pair(tmem_base, 512);
    else tmem_dealloc(tmem_base, 512);
  }
}

template <bool kGlu, bool kOutF32, int kCtas>
static cudaError_t launch_tile(const TileArgs& a, int num_sms, cudaStream_t s) {
  const Fp8Product& p = a.p;
  const int wide = kOutF32 ? 4 : 2, kRun = kCtas == kPair ? 2 * kTRows : kTRows;
  alignas(64) CUtensorMap tx, tw, to;
  cudaError_t e = make_tmap_u8_rows(&tx, p.x, p.M, p.K, kTBox);
  if (e == cudaSuccess) e = make_tmap_u8_rows(&tw, p.w, (long long)p.groups * p.N, p.K, kGlu ? 32 : kCtas == kPair ? 128 : 256);
  to = tw;
  if (e == cudaSuccess && !kGlu && kCtas != kSplit && p.N * (long long)wide % 16 == 0) e = make_tmap_u8_rows(&to, p.out, p.M, (long long)p.N * wide, 32);      // as bytes
  if (e == cudaSuccess) e = allow_smem<fp8_tile_kernel<kGlu, kOutF32, kCtas>>(kTSmem);
  if (e != cudaSuccess) return e;
  const long long total = (long long)a.w_tiles * (p.chunks ? p.max_chunks : (p.M + kRun - 1) / kRun);
  const int at_once = kCtas == kPair ? num_sms / 2 : num_sms;
  const unsigned grid = kCtas == kSplit ? (unsigned)(total * a.split) : (unsigned)(total < at_once ? total : at_once) * (kCtas == kPair ? 2 : 1);
  return launch_pdl_clusters(fp8_tile_kernel<kGlu, kOutF32, kCtas>, grid, kTThreads, kTSmem, s, dim3(kCtas == kSplit ? a.split : kCtas == kPair ? 2 : 1, 1, 1), tx, tw, to, a);
}

int fp8_clusters(int split) {
  static std::atomic<int> known[64][4];            // by device, for clusters of 1, 2, 4 and 8
  int dev = 0, n = 0, at = 0;
  while ((2 << at) <= split) ++at;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  if ((n = known[dev][at].load(std::memory_order_relaxed)) > 0) return n;
  const auto kernel = fp8_tile_kernel<false, false, kSplit>;
  if (allow_smem<fp8_tile_kernel<false, false, kSplit>>(kTSmem) != cudaSuccess) return 0;
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = split;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(split);
  cfg.blockDim = dim3(kTThreads);
  cfg.dynamicSmemBytes = kTSmem;
  cfg.attrs = &cluster;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    return 0;
  }
  known[dev][at].store(n, std::memory_order_relaxed);
  return n;
}

cudaError_t launch_fp8_tiles(const Fp8Product& p, int split, int num_sms, cudaStream_t s) {
  KernelSpan ks(K_FP8_PRODUCT, s);
  const TileArgs a{p, (p.N + 255) / 256, split, nullptr, 0};
  if (split > 1) return p.out_f32 ? launch_tile<false, true, kSplit>(a, num_sms, s) : launch_tile<false, false, kSplit>(a, num_sms, s);
  return p.out_f32 ? launch_tile<false, true, kAlone>(a, num_sms, s) : launch_tile<false, false, kAlone>(a, num_sms, s);
}
cudaError_t launch_fp8_pairs(const Fp8Product& p, int num_sms, cudaStream_t s) {
  KernelSpan ks(K_FP8_PRODUCT, s);
  const TileArgs a{p, (p.N + 255) / 256, 1, nullptr, 0};
  return p.out_f32 ? launch_tile<false, true, kPair>(a, num_sms, s) : launch_tile<false, false, kPair>(a, num_sms, s);
}
cudaError_t launch_fp8_gated(const Fp8Product& p, float* out_scales, long long ld_out_scales, int num_sms, cudaStream_t s) {
  KernelSpan ks(K_FP8_PRODUCT, s);
  const TileArgs a{p, p.N / 256, 1, out_scales, ld_out_scales};
  return launch_tile<true, false, kAlone>(a, num_sms, s);
}

// Which kernel, by estimates fitted to times of 7 matrices (N 1024 to 16384, K 512 to 8192) with 4 to 4200 rows, us beside what all forms share: a round of tiles takes 0.39 a block of K on
// pairs of CTAs and 0.43 on single ones (half as large), and 1.0 / 0.7 for its ends; a cluster's joining its sums 3 and 0.02 a row.  us in all on both sides of the lines: N 2048, K 8192,
// M 4200 pairs 63.6 / tiles 69.7, N 16384, K 1024, M 520 24.6 / 22.6, N 7168, K 4096, M 520 36.9 / 26.7; N 2048, K 8192, M 333 tiles 36.9, two along K 28.7, four 22.7; N 1024, K 2048,
// M 100 16.4 / 16.4 / 15.2.
cudaError_t launch_fp8_product(const Fp8Product& p, int num_sms, cudaStream_t s) {
  const int nb = fp8_blocks(p.K);
  const long long w_tiles = (p.N + 255) / 256, tiles = w_tiles * ((p.M + kFp8Run - 1) / kFp8Run), pairs = w_tiles * ((p.M + 2 * kFp8Run - 1) / (2 * kFp8Run));
  const auto rounds = [](long long n, int at_once) { return (float)((n + at_once - 1) / at_once); };
  float least = rounds(pairs, num_sms / 2) * (nb * 0.39f + 1.f);
  int split = 0;
  for (int n = 1; n <= 8 && n <= nb; n *= 2) {
    if (n > 1 && tiles > fp8_clusters(n)) break;             // a cluster's CTAs that have to wait for SMs are another round
    const float time = rounds(tiles, n > 1 ? (int)tiles : num_sms) * ((float)((nb + n - 1) / n) * 0.43f + 0.7f) + (n > 1 ? 3.f + 0.02f * (p.M < kFp8Run ? p.M : kFp8Run) : 0.f);
    if (time < least) {
      least = time;
      split = n;
    }
  }
  return split ? launch_fp8_tiles(p, split, num_sms, s) : launch_fp8_pairs(p, num_sms, s);
}

}  // namespace kb2
