// Log probabilities of given tokens, entropy and the largest alternatives of rows of logits.
#include "seq_common.cuh"

namespace kb2seq {

// A number's place among a row's: larger numbers first, then lower indices; -0 and +0 are equal.
__device__ __forceinline__ unsigned long long logp_key(float z, int i) {
  const uint32_t b = __float_as_uint(z == 0.f ? 0.f : z), up = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (unsigned long long)up << 32 | (uint32_t)~i;
}
__device__ __forceinline__ float logp_number(unsigned long long key) {
  const uint32_t up = (uint32_t)(key >> 32);
  return __uint_as_float(up & 0x80000000u ? up & 0x7FFFFFFFu : ~up);
}

struct LogpArgs {
  const void* z;
  long long ldz;
  int dt, V, top;
  const long long* tokens;
  float *logprob, *entropy, *best;
  int* ids;
};

// A block per row: the maximum, the sums, then `top` rounds that each take the largest key below the last one.
__global__ void __launch_bounds__(256) token_logprobs_kernel(const LogpArgs a) {
  kb2::pdl_wait();
  __shared__ float red[32];
  __shared__ unsigned long long red_key[8];
  const int t = blockIdx.x, tid = threadIdx.x;
  const long long row = t * a.ldz;
  float m = -INFINITY;
  bool bad = false;
  for (int i = tid; i < a.V; i += 256) {
    const float z = ld_dt(a.z, a.dt, row + i);
    bad |= !(z < INFINITY);
    m = fmaxf(m, z);
  }
  m = warp_max(m);
  if ((tid & 31) == 0) red[tid >> 5] = m;
  bad = __syncthreads_or(bad);
  for (int w = 0; w < 8; ++w) m = fmaxf(m, red[w]);
  bad |= m == -INFINITY;
  float s = 0.f, u = 0.f;
  for (int i = tid; i < a.V; i += 256) {
    const float d = ld_dt(a.z, a.dt, row + i) - m, e = expf(d);
    s += e;
    u += e > 0.f ? e * d : 0.f;
  }
  s = block_sum(s, red);
  u = block_sum(u, red);
  const float lse = logf(s);
  if (tid == 0) {
    const long long k = a.tokens[t];
    a.logprob[t] = bad ? NAN : k < 0 || k >= a.V ? -INFINITY : ld_dt(a.z, a.dt, row + k) - m - lse;
    a.entropy[t] = bad ? NAN : lse - u / s;
  }
  unsigned long long last = ~0ull;
  for (int j = 0; j < a.top; ++j) {
    unsigned long long best = 0;
    if (!bad)
      for (int i = tid; i < a.V; i += 256) {
        const unsigned long long k = logp_key(ld_dt(a.z, a.dt, row + i), i);
        if (k < last && k > best) best = k;
      }
    for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    __syncthreads();
    if ((tid & 31) == 0) red_key[tid >> 5] = best;
    __syncthreads();
    for (int w = 0; w < 8; ++w) best = max(best, red_key[w]);
    last = best;
    if (tid == 0) {
      a.ids[(long long)t * a.top + j] = bad ? -1 : (int)~(uint32_t)best;
      a.best[(long long)t * a.top + j] = bad ? NAN : logp_number(best) - m - lse;
    }
  }
}

}  // namespace kb2seq

using namespace kb2seq;

extern "C" {

KB2SEQ_API int kb2_seq_token_logprobs(const void* z, int dt, long long ldz, int T, int V, const long long* tokens, int top, float* logprob, float* entropy, int* ids,
                                      float* best, int device, void* stream) {
  if (bad_dt(dt) || T < 0 || V <= 0 || top < 0 || top > 64 || top > V || ldz < 0)
    return failf(KB2SEQ_ERR_VALUE, "token_logprobs: T=%d V=%d top=%d dt=%d: need V > 0, 0 <= top <= min(V, 64)", T, V, top, dt);
  if (T == 0) return KB2SEQ_OK;
  if (!z || !tokens || !logprob || !entropy || (top && (!ids || !best))) return failf(KB2SEQ_ERR_VALUE, "token_logprobs: null argument");
  const LogpArgs a{z, ldz, dt, V, top, tokens, logprob, entropy, best, ids};
  kb2::OnDevice on(device);
  SEQ_CUDA(on.err);
  SEQ_CUDA(kb2::launch_pdl(token_logprobs_kernel, T, 256, 0, (cudaStream_t)stream, a));
  SEQ_LAUNCHED();
  return KB2SEQ_OK;
}

}  // extern "C"
