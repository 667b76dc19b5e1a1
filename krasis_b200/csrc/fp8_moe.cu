// Routed experts on 8-bit operands (fp8.cuh): what lies ahead of and behind their two products.
#include "fp8.cuh"
#include "prof.cuh"
#include "ptx.cuh"

namespace kb2 {

// Which rows of the experts' order the choices take, for many of them: three launches, counters of each 4096 choices for themselves, so that no counter of the whole step is fought for (81920 choices of 512
// experts: 15.5 us for the last launch with such; 4.5, 8 and 5 for the three).  Within 4096 choices an expert's rows are in any order, which no result depends on.
constexpr int kBinChoices = 4096;
// The rows of expert e from `row` on as n runs of about the same size, a multiple of 16.
__device__ __forceinline__ void write_runs(ChunkDesc* runs, int e, int row, int rows, int n) {
  const int per = n ? ((rows + n - 1) / n + 15) & ~15 : 0;
  for (int i = 0; i < n; ++i) {
    ChunkDesc d;
    d.expert = e;
    d.slot_begin = row + i * per;
    d.n_tok = min(per, rows - i * per);
    d.pad_ = 0;
    runs[i] = d;
  }
}
__global__ void __launch_bounds__(1024) fp8_count_kernel(const int* ids, int n, int E, int* counts) {
  pdl_wait();
  __shared__ int s_count[1024];
  s_count[threadIdx.x] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kBinChoices / 1024; ++r) {
    const int i = blockIdx.x * kBinChoices + r * 1024 + threadIdx.x, e = i < n ? ids[i] : -1;
    if ((unsigned)e < (unsigned)E) atomicAdd(&s_count[e], 1);
  }
  __syncthreads();
  if ((int)threadIdx.x < E) counts[(long long)blockIdx.x * E + threadIdx.x] = s_count[threadIdx.x];
}
// Every block's counters become its first row of each expert; the runs of at most kFp8Run rows.
__global__ void __launch_bounds__(1024) fp8_runs_kernel(int* counts, int blocks, int E, ChunkDesc* runs, int* n_runs) {
  pdl_wait();
  __shared__ int s_warp[2][32];
  const int e = threadIdx.x, lane = e & 31, warp = e >> 5;
  int rows = 0;
  if (e < E) {
#pragma unroll 8
    for (int b = 0; b < blocks; ++b) rows += counts[(long long)b * E + e];
  }
  const int n = (rows + kFp8Run - 1) / kFp8Run;
  int row = rows, run = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, row, o), c = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) {
      row += a;
      run += c;
    }
  }
  if (lane == 31) {
    s_warp[0][warp] = row;
    s_warp[1][warp] = run;
  }
  __syncthreads();
  row -= rows;
  run -= n;
  for (int w = 0; w < warp; ++w) {
    row += s_warp[0][w];
    run += s_warp[1][w];
  }
  if (e == 1023) *n_runs = run + n;
  write_runs(runs + run, e, row, rows, n);
  if (e < E)
    for (int b = 0; b < blocks; ++b) {
      int* at = counts + (long long)b * E + e;
      const int c = *at;
      *at = row;
      row += c;
    }
}
__global__ void __launch_bounds__(1024) fp8_place_kernel(const int* ids, int n, int E, const int* firsts, int* slot_of) {
  pdl_wait();
  __shared__ int s_next[1024];
  if ((int)threadIdx.x < E) s_next[threadIdx.x] = firsts[(long long)blockIdx.x * E + threadIdx.x];
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kBinChoices / 1024; ++r) {
    const int i = blockIdx.x * kBinChoices + r * 1024 + threadIdx.x;
    if (i >= n) continue;
    const int e = ids[i];
    slot_of[i] = (unsigned)e < (unsigned)E ? atomicAdd(&s_next[e], 1) : -1;
  }
}

// Up to kBinRows choices: their places and their quantised rows in one launch.  Every block counts all choices in shared memory and adds the counters up by itself, so blocks need
// nothing from one another; a warp finds its choice's place among its expert's by counting the equal ones before it, and quantises its token's row into it, sixteen lanes a
// block of 128.  A token's row is read once a choice, from L2.  40 choices of rows of 2048: 7.5 us, 10.6 in two launches.
constexpr int kBinRows = 4096, kBinAhead = 4;
template <bool F32, bool VEC>
__global__ void __launch_bounds__(256) fp8_bin_rows_kernel(const int* ids, int n, int top, int E, ChunkDesc* runs, int* n_runs, int* slot_of, const void* x, long long ldx, int K,
                                                            uint8_t* codes, float* scales, long long lds) {
  pdl_wait();
  __shared__ short s_id[kBinRows];
  __shared__ int s_count[1024], s_first[1024], s_warp[2][8];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
#pragma unroll
  for (int i = 0; i < 4; ++i) s_count[i * 256 + t] = 0;
  __syncthreads();
  for (int i = t; i < n; i += 256) {
    const int e = ids[i];
    const bool mine = (unsigned)e < (unsigned)E;
    s_id[i] = mine ? (short)e : (short)-1;
    if (mine) atomicAdd(&s_count[e], 1);
  }
  __syncthreads();
  // first row and first run of each expert, four experts a thread
  int c[4], r[4], rows = 0, n_of = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    c[i] = s_count[t * 4 + i];
    r[i] = (c[i] + kFp8Run - 1) / kFp8Run;
    rows += c[i];
    n_of += r[i];
  }
  int row = rows, run = n_of;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, row, o), b = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) {
      row += a;
      run += b;
    }
  }
  if (lane == 31) {
    s_warp[0][warp] = row;
    s_warp[1][warp] = run;
  }
  __syncthreads();
  row -= rows;
  run -= n_of;
  for (int w = 0; w < warp; ++w) {
    row += s_warp[0][w];
    run += s_warp[1][w];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s_first[t * 4 + i] = row;
    if (blockIdx.x == 0) write_runs(runs + run, t * 4 + i, row, c[i], r[i]);
    row += c[i];
    run += r[i];
  }
  if (blockIdx.x == 0 && t == 255) *n_runs = run;
  __syncthreads();
  const int i = blockIdx.x * 8 + warp;
  if (i >= n) return;
  const int e = s_id[i];
  if (e < 0) {
    if (lane == 0) slot_of[i] = -1;
    return;
  }
  int before = 0;
  for (int j = lane; j < i; j += 32) before += s_id[j] == e;
  const int slot = s_first[e] + __reduce_add_sync(0xffffffffu, before);
  if (lane == 0) slot_of[i] = slot;
  const int l = lane & 15, blocks = fp8_blocks(K);
  const long long from = (long long)(i / top) * ldx, to = (long long)slot * K;
  for (int b0 = 0; b0 < blocks; b0 += 2 * kBinAhead) {
    Fp8Eight<F32> v[kBinAhead];
#pragma unroll
    for (int a = 0; a < kBinAhead; ++a) {
      const int k = (b0 + 2 * a + (lane >> 4)) * kFp8Block + l * 8;
      v[a].template load<VEC>(x, from + k, K - k);
    }
#pragma unroll
    for (int a = 0; a < kBinAhead; ++a) {
      const int b = b0 + 2 * a + (lane >> 4), k = b * kFp8Block + l * 8;
      uint32_t m = v[a].largest();
#pragma unroll
      for (int o = 8; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      const Fp8Scale f = fp8_scale(m);
      if (k < K) v[a].store(codes, to + k, f.inv);
      if (l == 0 && b < blocks) scales[b * lds + slot] = f.scale;
    }
  }
}

// out[t] = sum_j weights[t][j] y[slot_of[t][j]] in the order of j; entries without a slot bring nothing.  The experts' rows come in fp32, so that a bf16 result is rounded once (rows
// rounded to bf16 ahead of the sum halve what is read and put a result 0.0023 of it off, against 0.0017 by the last rounding alone).  A thread has 16 bytes of a row, four rows on their
// way at once.  W is a multiple of 16, so a row is whole pieces.
template <bool F32>
__global__ void __launch_bounds__(128) fp8_combine_kernel(const float* y, const int* slot_of, const float* weights, int top, int W, void* out) {
  pdl_enter_global(y, slot_of, weights, out);
  const int v = blockIdx.y * 128 + threadIdx.x, pieces = W / 4;
  if (v >= pieces) return;
  const long long e0 = (long long)blockIdx.x * top;
  float sum[4] = {};
  for (int j0 = 0; j0 < top; j0 += 4) {
    float4 x[4];
    float w[4];
    int slot[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) slot[j] = j0 + j < top ? slot_of[e0 + j0 + j] : -1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (slot[j] < 0) continue;
      x[j] = reinterpret_cast<const float4*>(y)[(long long)slot[j] * pieces + v];
      w[j] = weights[e0 + j0 + j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (slot[j] < 0) continue;
      sum[0] = fmaf(w[j], x[j].x, sum[0]);
      sum[1] = fmaf(w[j], x[j].y, sum[1]);
      sum[2] = fmaf(w[j], x[j].z, sum[2]);
      sum[3] = fmaf(w[j], x[j].w, sum[3]);
    }
  }
  const long long at = (long long)blockIdx.x * pieces + v;
  if constexpr (F32) reinterpret_cast<float4*>(out)[at] = make_float4(sum[0], sum[1], sum[2], sum[3]);
  else reinterpret_cast<uint2*>(out)[at] = make_uint2(bf16x2_bits_rn(sum[1], sum[0]), bf16x2_bits_rn(sum[3], sum[2]));
}

int fp8_bin_counts(int n, int E) { return n <= kBinRows ? 0 : (n + kBinChoices - 1) / kBinChoices * E; }

cudaError_t launch_fp8_bin(const int* ids, int T, int top, int E, int* counts, ChunkDesc* runs, int* n_runs, int* slot_of, const void* x, bool f32, long long ldx, int K, void* codes,
                           float* scales, long long lds, cudaStream_t s) {
  const int n = T * top, blocks = (n + kBinChoices - 1) / kBinChoices;
  if (n <= kBinRows) {
    KernelSpan ks(K_BINNING, s);
    const bool vec = ((uintptr_t)x & 15) == 0 && ldx % (f32 ? 4 : 8) == 0;
    const auto kernel = f32 ? vec ? fp8_bin_rows_kernel<true, true> : fp8_bin_rows_kernel<true, false> : vec ? fp8_bin_rows_kernel<false, true> : fp8_bin_rows_kernel<false, false>;
    return launch_pdl(kernel, (n + 7) / 8, 256, 0, s, ids, n, top, E, runs, n_runs, slot_of, x, ldx, K, (uint8_t*)codes, scales, lds);
  }
  cudaError_t e;
  {
    KernelSpan ks(K_BINNING, s, 3);
    e = launch_pdl(fp8_count_kernel, blocks, 1024, 0, s, ids, n, E, counts);
    if (e == cudaSuccess) e = launch_pdl(fp8_runs_kernel, 1, 1024, 0, s, counts, blocks, E, runs, n_runs);
    if (e == cudaSuccess) e = launch_pdl(fp8_place_kernel, blocks, 1024, 0, s, ids, n, E, (const int*)counts, slot_of);
  }
  return e == cudaSuccess ? launch_fp8_rows(x, f32, ldx, T, K, codes, scales, lds, slot_of, top, s) : e;
}
cudaError_t launch_fp8_combine(const float* y, const int* slot_of, const float* weights, int T, int top, int W, void* out, bool f32, cudaStream_t s) {
  KernelSpan ks(K_COMBINE, s);
  const dim3 grid(T, (W / 4 + 127) / 128);
  return launch_pdl(f32 ? fp8_combine_kernel<true> : fp8_combine_kernel<false>, grid, 128, 0, s, y, slot_of, weights, top, W, out);
}

}  // namespace kb2
