// Products of 8-bit floating-point operands with a scale per block of 128 (fp8.cuh): out[m][n] = sum_b xs[m][b] ws[n / 128][b] sum_{k in block b} x[m][k] w[n][k].
//
// The tensor cores' accumulators cannot be rescaled on the way, so each block of 128 products per result is a sum of its own in tensor memory (two of them in turn),
// which the other warps multiply by its scales and add up in registers while the next one runs.
#include <cuda.h>

#include "fp8.cuh"
#include "prof.cuh"
#include "ptx.cuh"

namespace kb2 {

cudaError_t make_tmap_u8_rows(void* out_tmap, const void* base, long long rows, long long cols, int box_rows);

// ---- many rows: pairs of CTAs, 256 rows of x x 256 weight rows
// A CTA has 128 rows of x (the M side) and half the weight rows, 32 KB for 512 cycles of MMAs per block of K.  Sixteen warps hold the tile's sums, 64 a thread: a thread has one
// row of x, so one scale of it per block, and 64 columns of one block of weights, so one of those.  With the weights on the M side a column's scale came from shared memory, 256
// broadcast loads per block beside the MMAs' own reads, and a block took 1070 cycles of eight warps (M 8192, N 4096, K 4096: 150 us).
constexpr int kFRows = 128, kFBox = 32, kFABytes = kFRows * 128, kFStage = 2 * kFABytes;
constexpr int kFThreads = 640, kFWarps = 16;
// The scales of kFGroup blocks are handed over at once, two groups are at hand: products for each row, for the first and the second 128 columns.
constexpr int kFGroup = 4, kFScales = 2 * kFGroup;
constexpr int kFOut = 32 * 128;                    // a warp's results on their way out
constexpr int kFStages = 4, kFTile = 2 * kFRows;
constexpr int kFOffOut = kFStages * kFStage, kFOffScale = kFOffOut + kFWarps * kFOut, kFOffBar = kFOffScale + kFScales * 2 * kFRows * 4, kFUsed = kFOffBar + 512,
              kFSmem = kFUsed > 512 * 430 - 1024 ? kFUsed : 512 * 430 - 1024;
static_assert(kFSmem <= 227 * 1024, "what a CTA of a cluster takes for 512 columns (tmem_smem)");

struct PairArgs {
  Fp8Product p;
  int w_tiles;                                     // tiles of 256 weight rows
};

template <bool kOutF32>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kFThreads, 1)
    fp8_pair_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_out, const PairArgs a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kFOffBar);       // of the first CTA: both CTAs' loads
  uint64_t* empty = full + kFStages;
  uint64_t* acc_full = empty + kFStages;       // [2]
  uint64_t* acc_empty = acc_full + 2;              // [2], of the first CTA: both CTAs' read-outs
  uint64_t* s_full = acc_empty + 2;                // [2]
  uint64_t* s_empty = s_full + 2;
  uint32_t* tmem_ptr_smem = reinterpret_cast<uint32_t*>(s_empty + 2);
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const Fp8Product& p = a.p;
  if (threadIdx.x == 32) {
    if (smem_u32(smem) & 1023u) __trap();
    for (int i = 0; i < kFStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 2 * kFWarps);
      mbar_init(&s_full[i], 2);
      mbar_init(&s_empty[i], kFWarps);
    }
    fence_mbar_init();
  }
  if (threadIdx.x == 64) {
    prefetch_tmap(&tmap_x);
    prefetch_tmap(&tmap_w);
    prefetch_tmap(&tmap_out);
  }
  if (warp == 0) tmem_alloc_pair(tmem_ptr_smem, 512);
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();                              // the other CTA's barriers are there
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_ptr_smem;
  pdl_wait();
  const int nb = fp8_blocks(p.K), total = (p.M + kFTile - 1) / kFTile * a.w_tiles;
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;
  struct Item {
    int row0, rows, wt;
  };
  // weight tiles first, so that pairs that run at once share the rows of x
  const auto item = [&](int t) {
    Item i;
    const int u = t / a.w_tiles;
    i.wt = t - u * a.w_tiles;
    i.row0 = u * kFTile;
    i.rows = min(kFTile, p.M - i.row0);
    return i;
  };

  if (warp >= 4) {
    more_registers<112>();
    const int q = warp & 3, h = (warp - 4) >> 2, row = rank * kFRows + q * 32 + lane;     // of the tile
    const uint32_t from = tmem_base + ((uint32_t)(q * 32) << 16) + h * 64;
    int b = 0;
    uint32_t aphase = 0, slot = 0, sphase = 0;
    for (int t = first; t < total; t += step) {
      const Item i = item(t);
      const bool mine = __any_sync(0xffffffffu, row < i.rows);
      uint64_t acc[32];                            // two columns in each
#pragma unroll
      for (int j = 0; j < 32; ++j) acc[j] = 0;
      for (int kb = 0; kb < nb; ++kb) {
        if ((slot & (kFGroup - 1)) == 0) mbar_wait(&s_full[slot / kFGroup], sphase);
        const uint32_t* sc = reinterpret_cast<const uint32_t*>(smem + kFOffScale) + slot * 2 * kFRows + q * 32 + lane;
        const uint32_t s0 = sc[(h >> 1) * kFRows];
        const uint64_t two = pack2(s0, s0);
        mbar_wait(&acc_full[b], aphase);
        tc_fence_after_sync();
        const auto read = [&]() {                  // this block's sums are in registers
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster_relaxed(cluster_addr(&acc_empty[b], 0));
        };
        if (mine) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t v[32];
            tmem_ld32(from + b * 256 + c * 32, v);
            tmem_ld_wait();
            if (c) read();
#pragma unroll
            for (int j = 0; j < 16; ++j) fma2_here(acc[c * 16 + j], pack2(v[2 * j], v[2 * j + 1]), two);
          }
        } else {
          read();
        }
        ++slot;
        if ((slot & (kFGroup - 1)) == 0) {
          if (lane == 0) mbar_arrive(&s_empty[slot / kFGroup - 1]);
          if (slot == kFScales) { slot = 0; sphase ^= 1; }
        }
        b ^= 1;
        aphase ^= b == 0;
      }
      if (mine) {
        // 32 rows x 128 bytes at a time go out from shared memory by one copy, while the next tile's blocks are added: all SMs end their tiles at the same time, and a tile's
        // stores by the lanes took 3500 cycles (16 bytes of a row by each lane, row by row, 12000).  The last rows, and rows that are not on 16 bytes, are the lanes'.
        constexpr int kCols = kOutF32 ? 32 : 64, kVec = kOutF32 ? 4 : 8;
        uint8_t* st = smem + kFOffOut + (warp - 4) * kFOut;
        const int row0 = i.row0 + rank * kFRows + q * 32, have = i.rows - (int)(rank * kFRows + q * 32);
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
    if (lane == 0) bulk_wait_group0();
  } else if (fewer_registers<32>(), warp == 0) {
    int stage = 0;
    uint32_t phase = 0;
    for (int t = first; t < total; t += step) {
      const Item i = item(t);
      // boxes of rows that are there; what lies behind them in a stage is multiplied, too, and looked at by nobody
      const int boxes0 = (min(i.rows, kFRows) + kFBox - 1) / kFBox, boxes1 = (max(i.rows - kFRows, 0) + kFBox - 1) / kFBox, boxes = rank ? boxes1 : boxes0;
      const uint32_t bytes = 2 * kFABytes + (boxes0 + boxes1) * kFBox * 128;
      for (int kb = 0; kb < nb; ++kb) {
        mbar_wait(&empty[stage], phase ^ 1);
        uint8_t* at = smem + stage * kFStage;
        if (elect_one()) {
          const uint32_t bar = cluster_addr(&full[stage], 0);
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], bytes);
          tma_load_2d_pair(at + kFABytes, &tmap_w, kb * 128, i.wt * 256 + rank * 128, bar);
          for (int r = 0; r < boxes; ++r) tma_load_2d_pair(at + r * kFBox * 128, &tmap_x, kb * 128, i.row0 + rank * kFRows + r * kFBox, bar);
        }
        __syncwarp();
        if (++stage == kFStages) { stage = 0; phase ^= 1; }
      }
    }
    for (int i = 0; i < kFStages; ++i) {           // the last reports of freed stages have arrived, too
      mbar_wait(&empty[stage], phase ^ 1);
      if (++stage == kFStages) { stage = 0; phase ^= 1; }
    }
  } else if (warp == 1 && rank == 0) {
    int stage = 0, b = 0;
    uint32_t phase = 0, aphase = 0;
    const uint32_t idesc = umma_idesc_e4m3(256, 256);
    for (int t = first; t < total; t += step) {
      for (int kb = 0; kb < nb; ++kb) {
        mbar_wait(&full[stage], phase);
        mbar_wait(&acc_empty[b], aphase ^ 1);
        tc_fence_after_sync();
        const uint32_t addr = smem_u32(smem + stage * kFStage);
        const uint64_t ad = umma_desc_k_sw128(addr), bd = umma_desc_k_sw128(addr + kFABytes);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_f8_pair(tmem_base + b * 256, ad + 2 * k, bd + 2 * k, idesc, k > 0 ? 1u : 0u);
          umma_commit_pair(&acc_full[b]);
          umma_commit_pair(&empty[stage]);
        }
        __syncwarp();
        if (++stage == kFStages) { stage = 0; phase ^= 1; }
        b ^= 1;
        aphase ^= b == 0;
      }
    }
  } else if (warp >= 2) {
    // The scales, by two warps in turn: this CTA's rows times the weights'.  Each has two blocks' on their way at once, as that takes longer than a block's products.
    const int w_blocks = fp8_blocks(p.N);
    struct Scales {
      float x[4], w[2];
    };
    int t = first, kb = warp - 2;
    const auto settle = [&]() {
      while (kb >= nb) {
        kb -= nb;
        t += step;
      }
    };
    settle();
    Item i = item(t);
    const auto ask = [&](Scales& s) {
      const int n = i.wt * 2, n1 = min(n + 1, w_blocks - 1);
      const float *w = p.ws + kb, *x = p.xs + kb * p.ldxs + i.row0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = rank * kFRows + j * 32 + lane;
        s.x[j] = row < i.rows ? x[row] : 0.f;
      }
      s.w[0] = w[(long long)n * nb];
      s.w[1] = w[(long long)n1 * nb];
      const int was = t;
      kb += 2;
      settle();
      if (t != was) i = item(t);
    };
    uint32_t slot = warp - 2, phase = 0;
    const auto put = [&](const Scales& s) {
      if ((slot & (kFGroup - 1)) < 2) mbar_wait(&s_empty[slot / kFGroup], phase ^ 1);
      float* to = reinterpret_cast<float*>(smem + kFOffScale) + slot * 2 * kFRows + lane;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        to[j * 32] = s.x[j] * s.w[0];
        to[kFRows + j * 32] = s.x[j] * s.w[1];
      }
      __syncwarp();
      if ((slot & (kFGroup - 1)) >= kFGroup - 2 && lane == 0) mbar_arrive(&s_full[slot / kFGroup]);
      slot += 2;
      if (slot >= kFScales) { slot -= kFScales; phase ^= 1; }
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
    if (all % kFGroup > 0 && all % kFGroup < kFGroup - 3 + warp) {         // the last group is short: of either warp's two blocks, one or both are missing
      if (all % kFGroup == 1 && warp == 3) mbar_wait(&s_empty[slot / kFGroup], phase ^ 1);
      if (lane == 0) mbar_arrive(&s_full[slot / kFGroup]);
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();                              // nobody leaves while the other may still report to its barriers
  tc_fence_after_sync();
  if (warp == 0) tmem_dealloc_pair(tmem_base, 512);
}

template <bool kOutF32>
static cudaError_t launch_pair(const Fp8Product& p, int num_sms, cudaStream_t s) {
  const PairArgs a{p, (p.N + 255) / 256};
  const int wide = kOutF32 ? 4 : 2;
  alignas(64) CUtensorMap tx, tw, to;
  cudaError_t e = make_tmap_u8_rows(&tx, p.x, p.M, p.K, kFBox);
  if (e == cudaSuccess) e = make_tmap_u8_rows(&tw, p.w, p.N, p.K, kFRows);
  to = tw;
  if (e == cudaSuccess && p.N * (long long)wide % 16 == 0) e = make_tmap_u8_rows(&to, p.out, p.M, (long long)p.N * wide, 32);      // as bytes
  if (e == cudaSuccess) e = allow_smem<fp8_pair_kernel<kOutF32>>(kFSmem);
  if (e != cudaSuccess) return e;
  const long long total = (long long)a.w_tiles * ((p.M + kFTile - 1) / kFTile);
  const int pairs = (int)(total < num_sms / 2 ? total : num_sms / 2);
  return launch_pdl(fp8_pair_kernel<kOutF32>, 2 * pairs, kFThreads, kFSmem, s, tx, tw, to, a);
}

cudaError_t launch_fp8_pairs(const Fp8Product& p, int num_sms, cudaStream_t s) {
  KernelSpan ks(K_FP8_PRODUCT, s);
  return p.out_f32 ? launch_pair<true>(p, num_sms, s) : launch_pair<false>(p, num_sms, s);
}

// Which kernel, by estimates fitted to times of 7 matrices (N 1024 to 16384, K 512 to 8192) with 4 to 4200 rows, us beside what all forms share: a round of tiles takes 0.39 a block of K on
// pairs of CTAs and 0.43 on single ones (half as large), and 1.0 / 0.7 for its ends; a cluster's joining its sums 3 and 0.02 a row.  us in all on both sides of the lines: N 2048, K 8192,
// M 4200 pairs 63.6 / tiles 69.7, N 16384, K 1024, M 520 24.6 / 22.6, N 7168, K 4096, M 520 36.9 / 26.7; N 2048, K 8192, M 333 tiles 36.9, two along K 28.7, four 22.7; N 1024, K 2048,
// M 100 16.4 / 16.4 / 15.2.
cudaError_t launch_fp8_product(const Fp8Product& p, int num_sms, cudaStream_t s) {
  const int nb = fp8_blocks(p.K);
  const long long w_tiles = (p.N + 255) / 256, tiles = w_tiles * ((p.M + kFp8Run - 1) / kFp8Run), pairs = w_tiles * ((p.M + kFTile - 1) / kFTile);
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
