// Log probabilities of given tokens, entropy and the largest alternatives of rows of logits, in one pass over them.
//
// With a running maximum m: s = sum exp(z - m), u = sum exp(z - m) (z - m); where m rises by d, s <- s exp(-d) and u <- (u - d s) exp(-d).  At the end lse = m + log s, logprob =
// z[token] - lse, entropy = log s - u / s.
// Bound: the rows' way from memory.  A block of sixteen warps has a row; where there are fewer rows than SMs, a cluster of up to eight blocks shares it and its first block
// joins what they found, read through distributed shared memory.  Of the largest numbers every warp keeps a list of its own: what passes the least of the numbers that can still be among
// the `top` goes to the list's end, and when it is full a sort of it leaves `top` of them.
#include "ptx.cuh"
#include "seq_common.cuh"

namespace kb2seq {

constexpr int kLpWarps = 16, kLpThreads = 32 * kLpWarps, kLpTop = 64, kLpList = 128, kLpMostCtas = 8, kLpPieces = 4;

// A number's place among a row's: larger numbers first, then lower indices; -0 and +0 are equal.  0: no number.
__device__ __forceinline__ unsigned long long logp_key(float z, uint32_t i) {
  const uint32_t b = __float_as_uint(z + 0.f), up = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (unsigned long long)up << 32 | (uint32_t)~i;
}
__device__ __forceinline__ float logp_number(unsigned long long key) {
  const uint32_t up = (uint32_t)(key >> 32);
  return __uint_as_float(up & 0x80000000u ? up & 0x7FFFFFFFu : ~up);
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// e^d for d <= 0: an approximate power of two, off by 2^-22 beside the rounding of d / ln 2
__device__ __forceinline__ float exp_neg(float d) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d * 1.4426950408889634f));
  return r;
}

struct LogpArgs {
  const void* z;
  long long ldz;
  int V, top;
  const long long* tokens;
  float *logprob, *entropy, *best;
  int* ids;
};
struct LogpSums {
  float m, s, u;
  // numbers with the maximum `most`
  __device__ __forceinline__ void raise(float most) {
    if (most > m) {
      if (m > -INFINITY) {
        const float d = m - most, f = exp_neg(d);
        u = d > -200.f ? f * fmaf(d, s, u) : 0.f;
        s *= f;
      }
      m = most;
    }
  }
  __device__ __forceinline__ void join(const LogpSums& o) {
    LogpSums b = o;
    raise(b.m);
    b.raise(m);
    s += b.s;
    u += b.u;
  }
};

// 128 keys of a warp, four a lane, sorted so that the largest come first (a bitonic network; place p is the lane p % 32's key p / 32).
__device__ __forceinline__ void sort_list(unsigned long long* list, int n, int lane) {
  unsigned long long k[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) k[i] = i * 32 + lane < n ? list[i * 32 + lane] : 0ull;
#pragma unroll
  for (int size = 2; size <= 128; size <<= 1)
#pragma unroll
    for (int half = size >> 1; half; half >>= 1) {
      if (half >= 32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = i ^ half / 32;
          if (j > i) {
            const bool down = ((i * 32 + lane) & size) == 0;      // the larger one ahead
            const unsigned long long a = k[i], b = k[j];
            k[i] = down == (a > b) ? a : b;
            k[j] = down == (a > b) ? b : a;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const unsigned long long o = __shfl_xor_sync(0xffffffffu, k[i], half);
          const bool ahead = (lane & half) == 0, down = ((i * 32 + lane) & size) == 0;
          k[i] = (ahead == down) == (k[i] > o) ? k[i] : o;
        }
      }
    }
#pragma unroll
  for (int i = 0; i < 4; ++i) list[i * 32 + lane] = k[i];
  __syncwarp();
}

// The `top` largest of n keys (zeros are none) at `from`, to `to` in their order; `threads` threads.
__device__ __forceinline__ void choose(const unsigned long long* from, int n, unsigned long long* to, int top) {
  for (int i = threadIdx.x; i < n; i += kLpThreads) {
    const unsigned long long k = from[i];
    if (k == 0) continue;
    int ahead = 0;
    for (int j = 0; j < n; ++j) ahead += from[j] > k;
    if (ahead < top) to[ahead] = k;
  }
}

// What a thread knows of its numbers, and its warp of the largest ones.
template <int kVec, int kHave>
struct LogpState {
  LogpSums sum;
  bool bad;
  int lane, top, listed;                           // keys in the warp's list
  unsigned long long least;                        // only larger ones can still be among the `top`
  unsigned long long* list;

  __device__ __forceinline__ void prune() {
    __syncwarp();
    sort_list(list, listed, lane);
    listed = min(listed, top);
    if (listed == top) least = max(least, list[top - 1]);
    __syncwarp();
  }
  // where the j-th of a thread's numbers stands in the row
  static __device__ __forceinline__ uint32_t place(uint32_t first, int j) { return first + j / kVec * 32 * kVec + j % kVec; }
  // The first `count` of the numbers, those that stand ahead of `end`, go to the list's end: of every lane the largest left over at a time.
  __device__ __forceinline__ void offer(float (&v)[kHave], uint32_t first, int count, uint32_t end) {
    for (;;) {
      unsigned long long k = 0;
      int which = -1;
#pragma unroll
      for (int j = 0; j < kHave; ++j) {
        const unsigned long long n = logp_key(v[j], place(first, j));
        if (v[j] == v[j] && j < count && place(first, j) < end && n > k) {
          k = n;
          which = j;
        }
      }
      const bool in = k > least;
      const uint32_t who = __ballot_sync(0xffffffffu, in);
      if (who == 0) return;
      if (listed + __popc(who) > kLpList) {
        prune();
        continue;
      }
      if (in) list[listed + __popc(who & ((1u << lane) - 1))] = k;
      listed += __popc(who);
#pragma unroll
      for (int j = 0; j < kHave; ++j)
        if (in && j == which) v[j] = NAN;          // taken
    }
  }
  __device__ __forceinline__ void feed(float (&v)[kHave], uint32_t first, int count, uint32_t end) {
    float most = v[0];
#pragma unroll
    for (int j = 1; j < kHave; ++j) most = max_nan(most, v[j]);
    bad |= !(most < INFINITY);
    sum.raise(most);
    if (sum.m > -INFINITY) {
#pragma unroll
      for (int j = 0; j < kHave; ++j) {
        const float d = fmaxf(v[j] - sum.m, -200.f), e = exp_neg(d);
        sum.s += e;
        sum.u = fmaf(e, d, sum.u);
      }
    }
    if (top > 0 && __any_sync(0xffffffffu, logp_key(most, 0) > least)) {
      if (least == 0 && listed == 0 && top <= 32) {
        // the first numbers: of the lanes' largest ones the top-th bounds what can be among the largest
        const unsigned long long k = most == most ? logp_key(most, 0xFFFFFFFFu) : 0ull;
        int ahead = 0;
        for (int j = 0; j < 32; ++j) {
          const unsigned long long o = __shfl_sync(0xffffffffu, k, j);
          ahead += o > k || (o == k && j < lane);
        }
        const uint32_t who = __ballot_sync(0xffffffffu, ahead == top - 1);
        const unsigned long long bound = __shfl_sync(0xffffffffu, k, __ffs(who) - 1);
        if (bound > 0) least = bound - 1;          // with an index behind all others: equal numbers pass
      }
      offer(v, first, count, end);
    }
  }
};

template <bool BF16>
__global__ void __launch_bounds__(kLpThreads, 2) token_logprobs_kernel(const LogpArgs a) {
  constexpr int kVec = BF16 ? 8 : 4, kPieces = BF16 ? kLpPieces / 2 : kLpPieces, kHave = kVec * kPieces;      // sixteen numbers a thread at a time
  __shared__ unsigned long long s_list[kLpWarps][kLpList], s_all[kLpMostCtas][kLpTop];
  __shared__ LogpSums s_sums[kLpWarps], s_cta[kLpMostCtas];
  __shared__ int s_bad[kLpMostCtas];
  kb2::pdl_wait();
  uint32_t ctas, rank;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int t = blockIdx.x / ctas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, top = a.top;
  const long long row = t * a.ldz;
  const char* z = reinterpret_cast<const char*>(a.z) + row * (BF16 ? 2 : 4);
  const auto number = [&](int i) { return BF16 ? __bfloat162float(reinterpret_cast<const bf16*>(z)[i]) : reinterpret_cast<const float*>(z)[i]; };

  // numbers ahead of the first 16-byte boundary, pieces of 16 bytes, numbers behind them
  const int head = min(a.V, (int)((16 - ((uintptr_t)z & 15)) & 15) / (BF16 ? 2 : 4)), pieces = (a.V - head) / kVec, tail0 = head + pieces * kVec;
  const int per = (pieces + ctas - 1) / ctas, p0 = min(pieces, (int)rank * per), p1 = min(pieces, p0 + per);
  const uint4* body = reinterpret_cast<const uint4*>(z + head * (BF16 ? 2 : 4));

  LogpState<kVec, kHave> st;
  st.sum = {-INFINITY, 0.f, 0.f};
  st.bad = false;
  st.lane = lane;
  st.top = top;
  st.listed = 0;
  st.least = 0;
  st.list = s_list[warp];
  const auto whole = [&](const uint4 (&x)[kPieces], float (&v)[kHave]) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const uint32_t u[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (BF16) {
          v[i * 8 + 2 * e] = __uint_as_float(u[e] << 16);
          v[i * 8 + 2 * e + 1] = __uint_as_float(u[e] & 0xFFFF0000u);
        } else {
          v[i * 4 + e] = __uint_as_float(u[e]);
        }
      }
    }
  };
  constexpr int kRound = kLpThreads * kPieces;
  constexpr uint32_t kNone = BF16 ? 0xFF80FF80u : 0xFF800000u;                            // -inf
  const auto load = [&](int p, uint4 (&x)[kPieces]) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int q = p + (warp * kPieces + i) * 32 + lane;
      x[i] = q < p1 ? ld_stream16(body + q) : make_uint4(kNone, kNone, kNone, kNone);
    }
  };
  uint4 x[kPieces];
  load(p0, x);
  for (int p = p0; p < p1; p += kRound) {
    float v[kHave];
    whole(x, v);
    if (p + kRound < p1) load(p + kRound, x);
    st.feed(v, head + (p + warp * kPieces * 32 + lane) * kVec, kHave, head + p1 * kVec);
  }
  if (rank == 0 && warp == 0 && (head > 0 || tail0 < a.V)) {
    // up to 15 numbers: one a lane
    float v[kHave];
#pragma unroll
    for (int j = 0; j < kHave; ++j) v[j] = -INFINITY;
    const int i = lane < 16 ? lane : tail0 + lane - 16;
    const bool there = lane < 16 ? lane < head : i < a.V;
    if (there) v[0] = number(i);
    st.feed(v, there ? i : a.V, 1, a.V);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    LogpSums b;
    b.m = __shfl_xor_sync(0xffffffffu, st.sum.m, o);
    b.s = __shfl_xor_sync(0xffffffffu, st.sum.s, o);
    b.u = __shfl_xor_sync(0xffffffffu, st.sum.u, o);
    st.sum.join(b);
  }
  if (top > 0) {
    st.prune();
  }
  if (lane == 0) s_sums[warp] = st.sum;
  bool bad = __syncthreads_or(st.bad);
  // the block's lists one behind the other
  if (top > 0) {
    for (int i = tid; i < kLpTop; i += kLpThreads) s_all[0][i] = 0;
    unsigned long long mine[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int i = r * kLpThreads + tid;
      mine[r] = i < kLpWarps * top ? s_list[i / top][i % top] : 0ull;
    }
    __syncthreads();
    unsigned long long* all = &s_list[0][0];
#pragma unroll
    for (int r = 0; r < 2; ++r)
      if (r * kLpThreads + tid < kLpWarps * top) all[r * kLpThreads + tid] = mine[r];
    __syncthreads();
    choose(all, kLpWarps * top, s_all[0], top);
  }
  if (tid == 0) {
    LogpSums w = s_sums[0];
    for (int i = 1; i < kLpWarps; ++i) w.join(s_sums[i]);
    s_cta[0] = w;
    s_bad[0] = bad;
  }
  if (ctas > 1) {
    kb2::cluster_sync_all();
    if (rank == 0) {
      for (int c = 1 + warp; c < (int)ctas; c += kLpWarps) {
        for (int i = lane; i < top; i += 32) {
          unsigned long long k;
          asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(k) : "r"(kb2::cluster_addr(&s_all[0][i], c)) : "memory");
          s_all[c][i] = k;
        }
        if (lane < 4) {
          uint32_t b;
          const uint32_t from = lane < 3 ? kb2::cluster_addr(reinterpret_cast<const float*>(&s_cta[0]) + lane, c) : kb2::cluster_addr(&s_bad[0], c);
          asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(b) : "r"(from) : "memory");
          if (lane < 3) reinterpret_cast<uint32_t*>(&s_cta[c])[lane] = b;
          else s_bad[c] = (int)b;
        }
      }
    }
    kb2::cluster_sync_all();                       // nobody leaves while the first block reads
    if (rank != 0) return;
    if (top > 0) {
      unsigned long long* all = &s_list[0][0];
      for (int i = tid; i < (int)ctas * top; i += kLpThreads) all[i] = s_all[i / top][i % top];
      __syncthreads();
      choose(all, ctas * top, s_all[0], top);
    }
  }
  __syncthreads();
  LogpSums w = s_cta[0];
  bad = s_bad[0];
  for (int c = 1; c < (int)ctas; ++c) {
    w.join(s_cta[c]);
    bad |= s_bad[c] != 0;
  }
  bad |= w.m == -INFINITY;
  const float lse = logf(w.s);
  if (tid == 0) {
    const long long k = a.tokens[t];
    a.logprob[t] = bad ? NAN : k < 0 || k >= a.V ? -INFINITY : number((int)k) - w.m - lse;
    a.entropy[t] = bad ? NAN : lse - w.u / w.s;
  }
  for (int i = tid; i < top; i += kLpThreads) {
    const unsigned long long k = s_all[0][i];
    a.ids[(long long)t * top + i] = bad ? -1 : (int)~(uint32_t)k;
    a.best[(long long)t * top + i] = bad ? NAN : logp_number(k) - w.m - lse;
  }
}

}  // namespace kb2seq

using namespace kb2seq;

extern "C" {

KB2SEQ_API int kb2_seq_token_logprobs(const void* z, int dt, long long ldz, int T, int V, const long long* tokens, int top, float* logprob, float* entropy, int* ids,
                                      float* best, int device, void* stream) {
  if (bad_dt(dt) || T < 0 || V <= 0 || top < 0 || top > kLpTop || top > V || ldz < 0)
    return failf(KB2SEQ_ERR_VALUE, "token_logprobs: T=%d V=%d top=%d dt=%d: need V > 0, 0 <= top <= min(V, %d)", T, V, top, dt, kLpTop);
  if (T == 0) return KB2SEQ_OK;
  if (!z || !tokens || !logprob || !entropy || (top && (!ids || !best))) return failf(KB2SEQ_ERR_VALUE, "token_logprobs: null argument");
  kb2::OnDevice on(device);
  SEQ_CUDA(on.err);
  // blocks of a row: as many as there are SMs for, each with a round's numbers at least
  const int round = kLpThreads * 16, sms = kb2::current_sms();
  int ctas = 1;
  while (ctas < kLpMostCtas && 2ll * ctas * T <= sms && V > ctas * round) ctas *= 2;
  if (T > INT32_MAX / kLpMostCtas) return failf(KB2SEQ_ERR_VALUE, "token_logprobs: %d rows are too many", T);
  const LogpArgs a{z, ldz, V, top, tokens, logprob, entropy, best, ids};
  const auto go = [&](auto kernel) { return kb2::launch_pdl_clusters(kernel, dim3(T * ctas), dim3(kLpThreads), 0, (cudaStream_t)stream, dim3(ctas, 1, 1), a); };
  SEQ_CUDA(dt ? go(token_logprobs_kernel<true>) : go(token_logprobs_kernel<false>));
  SEQ_LAUNCHED();
  return KB2SEQ_OK;
}

}  // extern "C"
