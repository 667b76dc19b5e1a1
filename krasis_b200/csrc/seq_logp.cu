// Log probabilities of given tokens, entropy and the largest alternatives of rows of logits, in one pass over them.
//
// With c the largest number so far and d = z - c: s = the sum of e^d without one of the largest's, which is 1, and u = the sum of d e^d.  Then log sum exp z = c + log(1 + s), logprob =
// d(token) - log(1 + s) and entropy = log(1 + s) - u / (1 + s).  As the 1 stays out of the sums, the log probability of a token that has nearly all of the weight is as exact as the
// others are beside it (with it inside, 0.05 was off by 2e-7).  Where c rises by x, u <- e^-x (u - x (1 + s)) and s <- e^-x (1 + s).
// Bound: the rows' way from memory.  A block of eight warps has a row (of sixteen, 2048 rows of 32768 and five alternatives took 102 us instead of 80); where more blocks
// could run at once than there are rows, a cluster of up to eight shares it and its first block joins what they found, read through distributed shared memory.
// The largest numbers: after one, four and sixteen rounds the block's numbers so far give a bound that `top` of the row pass (the top-th largest among the eight largest lanes'
// maxima of each warp).  What passes it goes to the end of a list of the warp, of which a sort leaves `top` when it is full and at the end; the warps' lists are merged two by two.
// With a bound of each warp's own, 20 alternatives of 2048 x 151936 logits took 815 us.  Now, fp32: 194 us without alternatives (6.4 TB/s), 212 with one, 240 with 20, 351 with 64.
#include "ptx.cuh"
#include "seq_common.cuh"

namespace kb2seq {

constexpr int kLpWarps = 8, kLpThreads = 32 * kLpWarps, kLpTop = 64, kLpList = 128, kLpMostCtas = 8, kLpPieces = 4, kLpFirst = 8;

typedef unsigned long long Key;
// A number's place among a row's: larger numbers first, then lower indices; -0 and +0 are equal.  0: no number.
__device__ __forceinline__ Key logp_key(float z, uint32_t i) {
  const uint32_t b = __float_as_uint(z + 0.f), up = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (Key)up << 32 | (uint32_t)~i;
}
__device__ __forceinline__ float logp_number(Key key) {
  const uint32_t up = (uint32_t)(key >> 32);
  return __uint_as_float(up & 0x80000000u ? up & 0x7FFFFFFFu : ~up);
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float exp2_fast(float t) {      // off by 2^-22
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;

struct LogpArgs {
  const void* z;
  long long ldz;
  int V, top;
  const long long* tokens;
  float *logprob, *entropy, *best;
  int* ids;
};
// What lies 210 below is e^-210 = 0, infinities too.
__device__ __forceinline__ float below(float z, float c) { return fmaxf(z - c, -210.f); }
struct LogpSums {
  float c, s, u;                                   // c -inf: nothing yet
  // `own`: the 1 that is not in s
  __device__ __forceinline__ void raise(float to, float own) {
    if (c > -INFINITY) {
      const float d = below(c, to), f = exp2_fast(d * kLog2e);
      u = f * fmaf(d, own + s, u);
      s = f * (own + s);
    }
    c = to;
  }
  __device__ __forceinline__ void join(const LogpSums& o) {
    if (o.c == -INFINITY) return;
    LogpSums b = o;
    if (b.c > c) raise(b.c, 1.f);                  // the 1 is the other's
    else b.raise(c, 1.f);
    s += b.s;
    u += b.u;
  }
};
// One step of a bitonic network over N * 32 keys or numbers of a warp, place i * 32 + lane in k[i]: partners `half` apart, blocks of `size` in turn down (the larger ones
// ahead) and up.
template <int N, typename T>
__device__ __forceinline__ void step(T (&k)[N], int size, int half, int lane) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const bool down = ((i * 32 + lane) & size) == 0;
    if (half >= 32) {
      const int other = i | half / 32;
      if (other == i) continue;
      const T x = k[i], y = k[other < N ? other : i];
      k[i] = down ? max(x, y) : min(x, y);
      k[other < N ? other : i] = down ? min(x, y) : max(x, y);
    } else {
      const T o = __shfl_xor_sync(0xffffffffu, k[i], half);
      k[i] = ((lane & half) == 0) == down ? max(k[i], o) : min(k[i], o);
    }
  }
}
// The first n of a list's N * 32 places, the others taken as empty, in their order.
template <int N>
__device__ __forceinline__ void sort_list(Key* list, int n, int lane) {
  Key k[N];
#pragma unroll
  for (int i = 0; i < N; ++i) k[i] = i * 32 + lane < n ? list[i * 32 + lane] : 0ull;
#pragma unroll
  for (int size = 2; size <= N * 32; size <<= 1)
#pragma unroll
    for (int half = size >> 1; half; half >>= 1) step(k, size, half, lane);
#pragma unroll
  for (int i = 0; i < N; ++i) list[i * 32 + lane] = k[i];
}
// The N * 32 largest of two sorted lists, in their order, in the first one's place.
template <int N>
__device__ __forceinline__ void merge_lists(Key* a, const Key* b, int lane) {
  Key k[N];
#pragma unroll
  for (int i = 0; i < N; ++i) k[i] = max(a[i * 32 + lane], b[N * 32 - 1 - (i * 32 + lane)]);
#pragma unroll
  for (int half = N * 16; half; half >>= 1) step(k, N * 64, half, lane);
#pragma unroll
  for (int i = 0; i < N; ++i) a[i * 32 + lane] = k[i];
}

// What a thread knows of its numbers, and its warp of the largest ones.
template <int kVec, int kHave>
struct LogpState {
  LogpSums sum;
  float own;                                       // 1 where the warp's largest number is the lane's
  bool bad;
  int lane, top, listed;                           // keys in the warp's list
  Key least;                                       // only larger ones can still be among the `top`
  float floor;                                     // its number
  Key* list;

  __device__ __forceinline__ void prune() {
    __syncwarp();
    if (listed <= 32 && top <= 32) sort_list<1>(list, listed, lane);      // what is merged is sorted whole: 32 places, or 64 for more alternatives
    else if (listed <= 64) sort_list<2>(list, listed, lane);
    else sort_list<4>(list, listed, lane);
    __syncwarp();
    listed = min(listed, top);
    if (listed == top && list[top - 1] > least) {
      least = list[top - 1];
      floor = logp_number(least);
    }
    __syncwarp();
  }
  // where the j-th of a thread's numbers stands in the row
  static __device__ __forceinline__ uint32_t place(uint32_t first, int j) { return first + j / kVec * 32 * kVec + j % kVec; }
  // Numbers that stand ahead of `end` go to the list's end.
  __device__ __forceinline__ void offer(float (&v)[kHave], uint32_t first, uint32_t end) {
    for (;;) {
      bool full = false;
#pragma unroll
      for (int j = 0; j < kHave; ++j) {
        if (!__any_sync(0xffffffffu, v[j] >= floor && place(first, j) < end)) continue;
        const Key k = v[j] >= floor && place(first, j) < end ? logp_key(v[j], place(first, j)) : 0ull;
        const uint32_t who = __ballot_sync(0xffffffffu, k > least);
        if (listed + __popc(who) > kLpList) {
          full = true;
          continue;
        }
        if (k > least) {
          list[listed + __popc(who & ((1u << lane) - 1))] = k;
          v[j] = NAN;                              // taken
        }
        listed += __popc(who);
      }
      if (!full) return;
      prune();
    }
  }
  // A warp's c is one for all of its lanes, and rises a few times a row; one lane has the 1.  (A c of each lane's own rose in some lane in nearly every round: 254 us instead of 212 for
  // 2048 x 151936 and one alternative.)
  __device__ __forceinline__ void add(const float (&v)[kHave], float most) {
    bad |= !(most < INFINITY);                     // an infinity or a NaN; any other number is taken by its distance to the largest
    if (__any_sync(0xffffffffu, most > sum.c)) {
      float to = most;
#pragma unroll
      for (int o = 16; o; o >>= 1) to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, o));
      sum.raise(to, own);
      const uint32_t who = __ballot_sync(0xffffffffu, most == to);
      own = lane == __ffs(who) - 1 ? 1.f : 0.f;
      bool out = own == 0.f;                       // the first of the owner's largest stays out
#pragma unroll
      for (int j = 0; j < kHave; ++j) {
        const float d = below(v[j], to), e = exp2_fast(d * kLog2e);
        const bool it = !out && v[j] == to;
        out |= it;
        sum.s += it ? 0.f : e;
        sum.u = fmaf(e, d, sum.u);
      }
    } else if (sum.c > -INFINITY) {
#pragma unroll
      for (int j = 0; j < kHave; ++j) {
        const float d = below(v[j], sum.c), e = exp2_fast(d * kLog2e);
        sum.s += e;
        sum.u = fmaf(e, d, sum.u);
      }
    }
  }
  static __device__ __forceinline__ float largest(const float (&v)[kHave]) {
    float most = v[0];
#pragma unroll
    for (int j = 1; j < kHave; ++j) most = max_nan(most, v[j]);
    return most;
  }
  // The bound that the lanes' largest numbers so far give; `firsts` is room for kLpWarps * kLpFirst numbers.  Lanes without numbers have -inf, which bounds nothing.
  __device__ __forceinline__ void bound(float most, float* firsts, int warp) {
    __syncthreads();                               // the last one's have been read
    float k[1] = {most == most ? most : -INFINITY};
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
      for (int half = size >> 1; half; half >>= 1) step(k, size, half, lane);
    if (lane < kLpFirst) firsts[warp * kLpFirst + lane] = k[0];
    __syncthreads();
    float all[2] = {firsts[lane], firsts[32 + lane]};
#pragma unroll
    for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
      for (int half = size >> 1; half; half >>= 1) step(all, size, half, lane);
    const float it = __shfl_sync(0xffffffffu, top > 32 ? all[1] : all[0], (top - 1) & 31);
    if (it > floor) {
      floor = it;
      least = logp_key(it, 0xFFFFFFFFu) - 1;       // equal numbers pass
    }
  }
};
static_assert(kLpWarps * kLpFirst == 64 && kLpTop == 64, "the bound is found among 64 numbers");

template <bool BF16>
__global__ void __launch_bounds__(kLpThreads, 3) token_logprobs_kernel(const LogpArgs a) {
  constexpr int kVec = BF16 ? 8 : 4, kPieces = BF16 ? kLpPieces / 2 : kLpPieces, kHave = kVec * kPieces;      // sixteen numbers a thread at a time
  __shared__ Key s_list[kLpWarps][kLpList], s_all[kLpMostCtas][kLpTop];
  __shared__ float s_first[kLpWarps * kLpFirst];
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
  st.own = 0.f;
  st.bad = false;
  st.lane = lane;
  st.top = top;
  st.listed = 0;
  st.least = 0;
  st.floor = -INFINITY;
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
  if (rank == 0 && warp == 0 && (head > 0 || tail0 < a.V)) {
    // up to 14 numbers: one a lane, and a place of the list for each
    const int i = lane < 16 ? lane : tail0 + lane - 16;
    const bool there = lane < 16 ? lane < head : i < a.V;
    float v[kHave];
#pragma unroll
    for (int j = 0; j < kHave; ++j) v[j] = -INFINITY;
    if (there) v[0] = number(i);
    st.add(v, v[0]);
    const uint32_t who = __ballot_sync(0xffffffffu, there);
    if (top > 0) {
      if (there) st.list[__popc(who & ((1u << lane) - 1))] = logp_key(v[0], i);
      st.listed = __popc(who);
    }
  }
  float best = -INFINITY;
  int next_bound = p0;
  for (int p = p0; p < p1; p += kRound) {
    float v[kHave];
    whole(x, v);
    if (p + kRound < p1) load(p + kRound, x);
    const float most = st.largest(v);
    st.add(v, most);
    if (top > 0) {
      best = fmaxf(best, most);
      if (p >= next_bound) {                       // after one, four and sixteen rounds
        st.bound(best, s_first, warp);
        next_bound = p0 + (4 * ((p - p0) / kRound + 1) - 1) * kRound;
      }
      if (__any_sync(0xffffffffu, most >= st.floor)) st.offer(v, head + (p + warp * kPieces * 32 + lane) * kVec, head + p1 * kVec);
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    st.sum.s += __shfl_xor_sync(0xffffffffu, st.sum.s, o);
    st.sum.u += __shfl_xor_sync(0xffffffffu, st.sum.u, o);
  }
  if (top > 0) st.prune();
  if (lane == 0) s_sums[warp] = st.sum;
  bool bad = __syncthreads_or(st.bad);
  const auto merge = [&](Key* to, const Key* from) {
    if (top <= 32) merge_lists<1>(to, from, lane);
    else merge_lists<2>(to, from, lane);
  };
  if (top > 0) {
    for (int o = 1; o < kLpWarps; o *= 2) {        // two by two
      if (warp % (2 * o) == 0) merge(s_list[warp], s_list[warp + o]);
      __syncthreads();
    }
    if (tid < kLpTop) s_all[0][tid] = s_list[0][tid];
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
        for (int i = lane; i < kLpTop; i += 32) {
          Key k;
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
      for (int o = 1; o < (int)ctas; o *= 2) {
        __syncthreads();
        if (warp % (2 * o) == 0 && warp + o < (int)ctas) merge(s_all[warp], s_all[warp + o]);
      }
    }
  }
  __syncthreads();
  LogpSums w = s_cta[0];
  bad = s_bad[0];
  for (int c = 1; c < (int)ctas; ++c) {
    w.join(s_cta[c]);
    bad |= s_bad[c] != 0;
  }
  bad |= w.c == -INFINITY;
  const float lse = log1pf(w.s);                   // of what is above c
  const auto logprob = [&](float x) { return (x - w.c) - lse; };
  if (tid == 0) {
    const long long k = a.tokens[t];
    a.logprob[t] = bad ? NAN : k < 0 || k >= a.V ? -INFINITY : logprob(number((int)k));
    a.entropy[t] = bad ? NAN : lse - w.u / (1.f + w.s);
  }
  for (int i = tid; i < top; i += kLpThreads) {
    const Key k = s_all[0][i];
    a.ids[(long long)t * top + i] = bad ? -1 : (int)~(uint32_t)k;
    a.best[(long long)t * top + i] = bad ? NAN : logprob(logp_number(k));
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
  // Blocks of a row: as many as run at once, three an SM and some room for clusters, each with two rounds of numbers at least.  us with 1, 2, 4, 8 of them, V 151936 and one alternative:
  // 16 rows 36.9, 26.6, 20.5, 18.5; 100 rows 38.9, 30.7, 26.7, 41.0; 200 rows 43.0, 36.9, 45.1, 65.5; 300 rows 49.2, 57.3, 61.5, 90.1.  V 8000, 100 rows 12.3, 14.4, 15.2, 26.6.
  const int round = kLpThreads * 16, sms = kb2::current_sms();
  int ctas = 1;
  while (ctas < kLpMostCtas && 4 * 2ll * ctas * T <= 11 * sms && V > 2 * ctas * round) ctas *= 2;
  if (T > INT32_MAX / kLpMostCtas) return failf(KB2SEQ_ERR_VALUE, "token_logprobs: %d rows are too many", T);
  const LogpArgs a{z, ldz, V, top, tokens, logprob, entropy, best, ids};
  const auto kernel = dt ? token_logprobs_kernel<true> : token_logprobs_kernel<false>;
  SEQ_CUDA(kb2::launch_pdl_clusters(kernel, dim3(T * ctas), dim3(kLpThreads), 0, (cudaStream_t)stream, dim3(ctas, 1, 1), a));
  SEQ_LAUNCHED();
  return KB2SEQ_OK;
}

}  // extern "C"
