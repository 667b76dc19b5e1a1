// Products of 8-bit floating-point operands with a scale per block of 128 (fp8.cuh): out[m][n] = sum_b xs[m][b] ws[n / 128][b] sum_{k in block b} x[m][k] w[n][k].
//
// The tensor cores' accumulators cannot be rescaled on the way, so each block of 128 products per result is a sum of its own in tensor memory (two of them in turn),
// which the other warps multiply by its scales and add up in registers while the next one runs.
#include <cuda.h>

#include "fp8.cuh"
#include "prof.cuh"
#include "ptx.cuh"
#include "seq_act.cuh"

namespace kb2 {

template <int N>
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
// a b + c for two numbers at once
__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// the larger of the number at a place of either CTA's shared memory and v
__device__ __forceinline__ void max_cluster(uint32_t addr, uint32_t v) { asm volatile("red.shared::cluster.max.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
// mbar_wait for what the other CTA has written and told
__device__ __forceinline__ void mbar_wait_cluster(uint64_t* bar, uint32_t parity) {
  mbar_wait(bar, parity);
  asm volatile("fence.acq_rel.cluster;" ::: "memory");
}
cudaError_t make_tmap_u8_rows(void* out_tmap, const void* base, long long rows, long long cols, int box_rows);
cudaError_t make_tmap_u8_gate_up(void* out_tmap, const void* base, long long groups, long long F, long long cols);

// ---- many rows: pairs of CTAs, 256 weight rows x up to 256 rows of x
// The weights are the M side of the instruction: a CTA has 128 of them, of one block of 128 (one scale), and half the rows of x, 32 KB for 512 cycles of MMAs.  The N side,
// rows of x, goes in steps of 32, so runs of rows (an expert's) need little padding.  Eight warps hold the tile's sums, 128 a thread: one weight row and
// half the rows of x, whose scales come four at a time from shared memory.
constexpr int kFStages = 6, kFRows = 128, kFBox = 16, kFABytes = kFRows * 128, kFStage = 2 * kFABytes;
constexpr int kFMost = kFp8Run;                       // rows of x per tile
constexpr int kFScales = 4;                        // blocks whose scales are at hand: those with gate's, and from kFUp on with up's (other banks)
constexpr int kFUp = kFMost + 8, kFSlot = 2 * kFMost + 16;
constexpr int kFThreads = 384, kFWarps = 8;
constexpr int kFStageOut = 2304;                   // a warp's results on their way out
constexpr int kFOffOut = kFStages * kFStage, kFOffScale = kFOffOut + kFWarps * kFStageOut, kFOffMax = kFOffScale + kFScales * kFSlot * 4,
              kFOffInv = kFOffMax + 2 * kFMost * 4, kFOffBar = kFOffInv + kFMost * 4, kFSmem = kFOffBar + 256;
static_assert(kFSmem >= 512 * 430 - 1024 && kFSmem <= 227 * 1024, "what a CTA of a cluster takes for 512 columns (tmem_smem)");

struct PairArgs {
  Fp8Product p;
  int w_tiles, row_tile;                           // tiles of 256 weight rows (gated: 128 of either half); rows of x per tile (one matrix)
  // gated units: out is codes [M][N / 2] with scales
  float* out_scales;
  long long ld_out_scales;
};

template <bool kGlu, bool kOutF32>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kFThreads, 1)
    fp8_pair_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const PairArgs a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kFOffBar);       // of the first CTA: both CTAs' loads
  uint64_t* empty = full + kFStages;
  uint64_t* acc_full = empty + kFStages;           // [2]
  uint64_t* acc_empty = acc_full + 2;              // [2], of the first CTA: both CTAs' read-outs
  uint64_t* s_full = acc_empty + 2;                // [kFScales]
  uint64_t* s_empty = s_full + kFScales;
  uint64_t* max_full = s_empty + kFScales;         // [2]
  uint32_t* tmem_ptr_smem = reinterpret_cast<uint32_t*>(max_full + 2);
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
      mbar_init(&max_full[i], 2 * kFWarps);
    }
    for (int i = 0; i < kFScales; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], kFWarps);
    }
    fence_mbar_init();
  }
  if (threadIdx.x == 64) {
    prefetch_tmap(&tmap_x);
    prefetch_tmap(&tmap_w);
  }
  if (kGlu)
    for (int i = threadIdx.x; i < 2 * kFMost; i += kFThreads) reinterpret_cast<uint32_t*>(smem + kFOffMax)[i] = 0;
  if (warp == 0) tmem_alloc_pair(tmem_ptr_smem, 512);
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();                              // the other CTA's barriers are there
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_ptr_smem;
  pdl_wait();
  const int F = p.N / 2, nb = fp8_blocks(p.K);
  const int units = p.chunks ? p.n_chunks[0] : (p.M + a.row_tile - 1) / a.row_tile, total = units * a.w_tiles;
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;
  struct Item {
    int row0, rows, group, wt;
    __device__ int nt() const { return __shfl_sync(0xffffffffu, (rows + 31) & ~31, 0); }
  };
  // weight tiles first, so that pairs that run at once share the rows of x.  Everyone asks for the next item when it starts on one.
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
      i.row0 = u * a.row_tile;
      i.rows = min(a.row_tile, p.M - i.row0);
      i.group = 0;
    }
    return i;
  };

  if (warp >= 4) {
    more_registers<216>();
    const int q = warp & 3, h = (warp - 4) >> 2;
    const uint32_t lanes = tmem_base + ((uint32_t)(q * 32) << 16);
    uint8_t* out_at = smem + kFOffOut + (warp - 4) * kFStageOut;
    const int up = kGlu && lane >= 16 ? kFUp : 0;
    int b = 0;
    uint32_t aphase = 0, slot = 0, sphase = 0, tile = 0;
    Item next = item(first);
    for (int t = first; t < total; t += step, ++tile) {
      const Item i = next;
      next = item(t + step);
      const int nt = i.nt(), c0 = h * (nt / 2), cols = nt / 2, steps = (cols + 31) / 32;
      uint64_t acc[4][16];                         // of this thread's weight row: 32 columns, two in each
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[s][j] = 0;
      for (int kb = 0; kb < nb; ++kb) {
        const float* sc = reinterpret_cast<const float*>(smem + kFOffScale) + slot * kFSlot + up + c0;
        mbar_wait(&s_full[slot], sphase);
        mbar_wait(&acc_full[b], aphase);
        tc_fence_after_sync();
        const uint32_t from = lanes + b * 256 + c0;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          if (s >= steps) break;
          uint32_t v[32];
          tmem_ld32(from + s * 32, v);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint4 g = *reinterpret_cast<const uint4*>(sc + s * 32 + j * 4);
            acc[s][2 * j] = fma2(pack2(v[4 * j], v[4 * j + 1]), pack2(g.x, g.y), acc[s][2 * j]);
            acc[s][2 * j + 1] = fma2(pack2(v[4 * j + 2], v[4 * j + 3]), pack2(g.z, g.w), acc[s][2 * j + 1]);
          }
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive_cluster_relaxed(cluster_addr(&acc_empty[b], 0));
          mbar_arrive(&s_empty[slot]);
        }
        if (++slot == kFScales) { slot = 0; sphase ^= 1; }
        b ^= 1;
        aphase ^= b == 0;
      }
      if constexpr (kGlu) {
        // a warp's rows are 16 of gate and the same 16 of up: lane f takes the even columns of unit f, lane 16 + f the odd ones
        uint32_t* most = reinterpret_cast<uint32_t*>(smem + kFOffMax) + (tile & 1) * kFMost;
        uint32_t* other = reinterpret_cast<uint32_t*>(smem + kFOffMax) + (~tile & 1) * kFMost;
        float* inv = reinterpret_cast<float*>(smem + kFOffInv);
        const bool odd = lane >= 16;
        named_bar_sync(1, 32 * kFWarps);           // everyone has read the last tile's maxima
        if (warp == 4)
          for (int c = lane; c < kFMost; c += 32) other[c] = 0;
        const uint32_t peer = cluster_addr(most, rank ^ 1);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          if (s >= steps) break;
          uint32_t m[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float even, odd_;
            unpack2(acc[s][j], even, odd_);
            const float got = __shfl_xor_sync(0xffffffffu, odd ? even : odd_, 16);
            const float v = kb2act::silu(odd ? got : even) * (odd ? odd_ : got);
            acc[s][j] = __float_as_uint(v);
            m[j] = __float_as_uint(v) & 0x7FFFFFFFu;
          }
          // over the 16 units: halves of the columns change sides until a lane has one of them
#pragma unroll
          for (int o = 8; o; o >>= 1)
#pragma unroll
            for (int j = 0; j < o; ++j) {
              const bool high = lane & o;
              m[j] = max(high ? m[j + o] : m[j], __shfl_xor_sync(0xffffffffu, high ? m[j] : m[j + o], o));
            }
          const int c = s * 32 + (lane & 15) * 2 + odd;
          if (c < cols) {
            atomicMax(&most[c0 + c], m[0]);
            max_cluster(peer + (c0 + c) * 4, m[0]);
          }
        }
        __syncwarp();
        if (lane == 0) {
          mbar_arrive_cluster(cluster_addr(&max_full[tile & 1], rank));
          mbar_arrive_cluster(cluster_addr(&max_full[tile & 1], rank ^ 1));
        }
        mbar_wait_cluster(&max_full[tile & 1], tile >> 1 & 1);
        {                                          // a column a thread; even columns of 32 lie ahead of odd ones, as the lanes want them
          const int c = threadIdx.x - 128;
          const Fp8Scale f = fp8_scale(most[c]);
          const int half = c >= nt / 2 ? nt / 2 : 0, in = c - half;
          if (c < nt) inv[(half ? kFMost / 2 : 0) + (in & ~31) + (in & 1) * 16 + (in >> 1 & 15)] = f.inv;
          if (rank == 0 && c < i.rows) a.out_scales[i.wt * a.ld_out_scales + i.row0 + c] = f.scale;
        }
        named_bar_sync(1, 32 * kFWarps);
        uint8_t* codes = reinterpret_cast<uint8_t*>(p.out) + (long long)i.row0 * F + i.wt * 128 + rank * 64 + q * 16 + (lane & 12);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          if (s >= steps) break;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float4 n = *reinterpret_cast<const float4*>(inv + h * (kFMost / 2) + s * 32 + odd * 16 + k * 4);
            const float f[4] = {n.x, n.y, n.z, n.w};
            float v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = f[j] == 0.f ? 0.f : __uint_as_float((uint32_t)acc[s][4 * k + j]) * f[j];
            // codes of four columns of this lane's unit -> those of four units of one column
            uint32_t w = fp8_codes4(v[0], v[1], v[2], v[3], 1.f);
            const uint32_t x = __shfl_xor_sync(0xffffffffu, w, 2);
            w = lane & 2 ? __byte_perm(x, w, 0x7632) : __byte_perm(w, x, 0x5410);
            const uint32_t y = __shfl_xor_sync(0xffffffffu, w, 1);
            w = lane & 1 ? __byte_perm(y, w, 0x7351) : __byte_perm(w, y, 0x6240);
            const int m = c0 + s * 32 + (k * 4 + (lane & 2) + (lane & 1)) * 2 + odd;
            if (m < min(i.rows, c0 + cols)) *reinterpret_cast<uint32_t*>(codes + (long long)m * F) = w;
          }
        }
      } else {
        const int n0 = i.wt * 256 + rank * 128 + q * 32;
        const float bias = p.bias != nullptr && n0 + lane < p.N ? p.bias[n0 + lane] : 0.f;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          if (s >= steps) break;
          const int m0 = c0 + s * 32, have = min(i.rows, c0 + cols) - m0;
          uint32_t* st = reinterpret_cast<uint32_t*>(out_at);
          if constexpr (kOutF32) {                 // [16 columns][36]
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              __syncwarp();
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                float v0, v1;
                unpack2(acc[s][half * 8 + j], v0, v1);
                st[(2 * j) * 36 + lane] = __float_as_uint(v0 + bias);
                st[(2 * j + 1) * 36 + lane] = __float_as_uint(v1 + bias);
              }
              __syncwarp();
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const int c = k * 4 + (lane >> 3), m = half * 16 + c, n = n0 + (lane & 7) * 4;
                if (m >= have || n >= p.N) continue;
                const float4 x = *reinterpret_cast<const float4*>(st + c * 36 + (lane & 7) * 4);
                float* to = reinterpret_cast<float*>(p.out) + (long long)(i.row0 + m0 + m) * p.N + n;
                if ((p.N & 3) == 0) *reinterpret_cast<float4*>(to) = x;
                else {
                  to[0] = x.x;
                  if (n + 1 < p.N) to[1] = x.y;
                  if (n + 2 < p.N) to[2] = x.z;
                  if (n + 3 < p.N) to[3] = x.w;
                }
              }
            }
          } else {                                 // [16 pairs of columns][36]
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              float v0, v1;
              unpack2(acc[s][j], v0, v1);
              st[j * 36 + lane] = bf16x2_bits_rn(v1 + bias, v0 + bias);
            }
            __syncwarp();
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int c = k * 4 + (lane >> 3), n = n0 + (lane & 7) * 4;
              const uint4 x = *reinterpret_cast<const uint4*>(st + c * 36 + (lane & 7) * 4);
              if (n >= p.N) continue;
              __nv_bfloat16* to = reinterpret_cast<__nv_bfloat16*>(p.out) + (long long)(i.row0 + m0 + 2 * c) * p.N + n;
#pragma unroll
              for (int o = 0; o < 2; ++o, to += p.N) {
                if (2 * c + o >= have) continue;
                const uint32_t lo = __byte_perm(x.x, x.y, o ? 0x7632 : 0x5410), hi = __byte_perm(x.z, x.w, o ? 0x7632 : 0x5410);
                if ((p.N & 3) == 0) *reinterpret_cast<uint2*>(to) = make_uint2(lo, hi);
                else {
                  to[0] = __ushort_as_bfloat16((unsigned short)lo);
                  if (n + 1 < p.N) to[1] = __ushort_as_bfloat16((unsigned short)(lo >> 16));
                  if (n + 2 < p.N) to[2] = __ushort_as_bfloat16((unsigned short)hi);
                  if (n + 3 < p.N) to[3] = __ushort_as_bfloat16((unsigned short)(hi >> 16));
                }
              }
            }
          }
        }
      }
    }
  } else if (fewer_registers<64>(), warp == 0) {
    int stage = 0;
    uint32_t phase = 0;
    Item next = item(first);
    for (int t = first; t < total; t += step) {
      const Item i = next;
      next = item(t + step);
      const int nt = i.nt(), x0 = i.row0 + rank * (nt / 2);
      const uint32_t bytes = 2 * kFABytes + nt * 128;
      for (int kb = 0; kb < nb; ++kb) {
        mbar_wait(&empty[stage], phase ^ 1);
        uint8_t* at = smem + stage * kFStage;
        if (elect_one()) {
          const uint32_t bar = cluster_addr(&full[stage], 0);
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], bytes);
          if constexpr (kGlu) tma_load_5d_pair(at, &tmap_w, kb * 128, 0, 0, (i.wt * 128 + (int)rank * 64) / 16, i.group, bar);
          else tma_load_2d_pair(at, &tmap_w, kb * 128, i.group * p.N + i.wt * 256 + rank * 128, bar);
          for (int r = 0; r < nt / 2; r += kFBox) tma_load_2d_pair(at + kFABytes + r * 128, &tmap_x, kb * 128, x0 + r, bar);
        }
        __syncwarp();
        if (++stage == kFStages) { stage = 0; phase ^= 1; }
      }
    }
    for (int i = 0; i < kFStages; ++i) {           // the last reports of freed stages have arrived, too
      mbar_wait(&empty[stage], phase ^ 1);
      if (++stage == kFStages) { stage = 0; phase ^= 1; }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      int stage = 0, b = 0;
      uint32_t phase = 0, aphase = 0;
      Item next = item(first);
      for (int t = first; t < total; t += step) {
        const uint32_t idesc = umma_idesc_e4m3(256, next.nt());
        next = item(t + step);
        for (int kb = 0; kb < nb; ++kb) {
          mbar_wait(&acc_empty[b], aphase ^ 1);
          mbar_wait(&full[stage], phase);
          tc_fence_after_sync();
          const uint32_t addr = smem_u32(smem + stage * kFStage);
          const uint64_t ad = umma_desc_k_sw128(addr), bd = umma_desc_k_sw128(addr + kFABytes);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 4; ++k) umma_f8_pair(tmem_base + b * 256, ad + 2 * k, bd + 2 * k, idesc, k > 0 ? 1u : 0u);
            umma_commit_pair(&empty[stage]);
            umma_commit_pair(&acc_full[b]);
          }
          __syncwarp();
          if (++stage == kFStages) { stage = 0; phase ^= 1; }
          b ^= 1;
          aphase ^= b == 0;
        }
      }
    }
  } else if (warp < 4) {
    // the scales of a block: those of the rows of x times the weights', by two warps in turn.  A block's are asked for while the one before it goes out: their way from L2
    // takes longer than a block's products.
    struct Scales {
      float g, u, v[kFMost / 32];
    };
    const auto ask = [&](const Item& i, int kb) {
      const int blocks = fp8_blocks(p.N), n0 = kGlu ? i.wt : min(i.wt * 2 + (int)rank, blocks - 1);
      const float *ws = p.ws + ((long long)i.group * blocks + n0) * nb + kb, *xs = p.xs + kb * p.ldxs + i.row0;
      Scales r;
      r.g = ws[0];
      r.u = kGlu ? ws[(long long)(F / kFp8Block) * nb] : 0.f;
#pragma unroll
      for (int j = 0; j < kFMost / 32; ++j) r.v[j] = j * 32 + lane < i.rows ? xs[j * 32 + lane] : 0.f;
      return r;
    };
    int t = first, kb = warp - 2;
    while (kb >= nb) { kb -= nb; t += step; }
    uint32_t slot = warp - 2, phase = 0;
    Item i = item(t);
    Scales now{};
    if (t < total) now = ask(i, kb);
    while (t < total) {
      const int rows = i.rows, before = t;
      for (kb += 2; kb >= nb; kb -= nb) t += step;
      if (t != before) i = item(t);
      Scales next{};
      if (t < total) next = ask(i, kb);
      mbar_wait(&s_empty[slot], phase ^ 1);
      float* to = reinterpret_cast<float*>(smem + kFOffScale) + slot * kFSlot;
#pragma unroll
      for (int j = 0; j < kFMost / 32; ++j)
        if (j * 32 < rows) {
          to[j * 32 + lane] = now.v[j] * now.g;
          if (kGlu) to[kFUp + j * 32 + lane] = now.v[j] * now.u;
        }
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_full[slot]);
      slot += 2;
      if (slot >= kFScales) { slot -= kFScales; phase ^= 1; }
      now = next;
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();                              // nobody leaves while the other may still report to its barriers
  tc_fence_after_sync();
  if (warp == 0) tmem_dealloc_pair(tmem_base, 512);
}

// Rows of x per tile of one matrix: what takes the fewest rounds of the chip's pairs, weighed by a block's time, which is that of 256 weight rows on their way (as much as
// 96 rows of x in MMAs) at least.
static int pair_rows(int M, int w_tiles, int pairs) {
  int best = kFMost;
  long long least = -1;
  for (int nt = kFMost; nt >= 32; nt -= 32) {
    const long long rounds = ((long long)((M + nt - 1) / nt) * w_tiles + pairs - 1) / pairs, time = rounds * (nt > 96 ? nt : 96);
    if (least < 0 || time < least) {
      least = time;
      best = nt;
    }
  }
  return best;
}

template <bool kGlu, bool kOutF32>
static cudaError_t launch_pair(const PairArgs& a, int num_sms, cudaStream_t s) {
  const Fp8Product& p = a.p;
  alignas(64) CUtensorMap tx, tw;
  cudaError_t e = make_tmap_u8_rows(&tx, p.x, p.M, p.K, kFBox);
  if (e == cudaSuccess) e = kGlu ? make_tmap_u8_gate_up(&tw, p.w, p.groups, p.N / 2, p.K) : make_tmap_u8_rows(&tw, p.w, (long long)p.groups * p.N, p.K, kFRows);
  if (e == cudaSuccess) e = allow_smem<fp8_pair_kernel<kGlu, kOutF32>>(kFSmem);
  if (e != cudaSuccess) return e;
  const long long total = (long long)a.w_tiles * (p.chunks ? p.max_chunks : (p.M + a.row_tile - 1) / a.row_tile);
  const int pairs = (int)(total < num_sms / 2 ? total : num_sms / 2);
  return launch_pdl(fp8_pair_kernel<kGlu, kOutF32>, 2 * pairs, kFThreads, kFSmem, s, tx, tw, a);
}

cudaError_t launch_fp8_product(const Fp8Product& p, int num_sms, cudaStream_t s) {
  KernelSpan ks(K_FP8_PRODUCT, s);
  PairArgs a{p, (p.N + 255) / 256, 0, nullptr, 0};
  if (!p.chunks) a.row_tile = pair_rows(p.M, a.w_tiles, num_sms / 2);
  return p.out_f32 ? launch_pair<false, true>(a, num_sms, s) : launch_pair<false, false>(a, num_sms, s);
}

cudaError_t launch_fp8_gated(const Fp8Product& p, float* out_scales, long long ld_out_scales, int num_sms, cudaStream_t s) {
  KernelSpan ks(K_FP8_PRODUCT, s);
  const PairArgs a{p, p.N / 256, 0, out_scales, ld_out_scales};
  return launch_pair<true, false>(a, num_sms, s);
}

}  // namespace kb2
