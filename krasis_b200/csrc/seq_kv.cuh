// The 8-bit key / value cache of ragged-batch serving: what its kernels share.  Codes [layers][pages][G][page_size][d or dv], a scale per row in fp32 beside them
// ([layers][pages][G][page_size]): the rows of one head in one page lie together, so a tile of keys is one run of bytes.
#pragma once
#include "seq_common.cuh"

namespace kb2seq {

enum { KV_E4M3 = 0, KV_INT8 = 1 };
constexpr int kKvGroup = 16;                 // keys that one page always holds together
constexpr int kKvNoWindow = 1 << 30;

struct KvLayer {                             // one layer's pools
  uint8_t *k, *v;
  float *ks, *vs;
  int pages, lps, G, d, dv;                  // lps: log2 of the page size
};
struct KvStep {
  const int *positions, *seq_of, *cu, *pages, *rows;      // rows: where a token's key and value lie (positions, but for drafted tokens)
  const uint32_t* bits;                                   // drafted tokens: [T][words], bit i of a token: it sees token i of its sequence
  int words, T, S, max_pages;
};

// Row of head 0 in the pools of position j of sequence s; -1 where the page list or the pool ends before it.
__device__ __forceinline__ long long kv_row(const KvLayer& c, const KvStep& t, int s, int j) {
  const int at = j >> c.lps;
  if (j < 0 || at >= t.max_pages) return -1;
  const int page = t.pages[(long long)s * t.max_pages + at];
  if ((unsigned)page >= (unsigned)c.pages) return -1;
  return (((long long)page * c.G) << c.lps) + (j & ((1 << c.lps) - 1));
}

// What the tokens t0 .. t1 of sequence s see at all, in groups of 16 positions: the groups 0 .. na - 1 of the first tokens, then nb groups from b0 on.
struct KvSpan {
  int na, b0, nb, base;                      // base: the first drafted row, or past every position
  int lo, hi;                                // seen are the positions below `first` and lo .. hi - 1
  int p0, p1;                                // positions of the first and the last token
  __device__ __forceinline__ int groups() const { return na + nb; }
  __device__ __forceinline__ int group(int i) const { return i < na ? i : b0 + i - na; }
};
__device__ __forceinline__ KvSpan kv_span(const KvLayer& c, const KvStep& t, int s, int t0, int t1, int window, int first) {
  KvSpan r;
  int lo, hi;
  const int most = t.max_pages << c.lps;     // fits: checked on the host
  r.p0 = t.positions[t0];
  r.p1 = t.positions[t1];
  if (t.bits != nullptr) {                   // a token's position is base + its depth, and its ancestors come before it
    const int c0 = t.cu[s];
    r.base = t.rows[c0];
    lo = r.base;
    hi = r.base + (t1 - c0) + 1;
  } else {
    r.base = 0x7FFFFFFF;
    lo = r.p0;
    hi = r.p1 + 1;
  }
  hi = min(hi, most);
  lo = window < kKvNoWindow ? max(0, lo - window + 1) : 0;
  r.na = (min(min(first, lo), max(hi, 0)) + kKvGroup - 1) / kKvGroup;
  r.b0 = max(lo / kKvGroup, r.na);
  r.lo = lo;
  r.hi = hi;
  r.nb = max(0, (hi + kKvGroup - 1) / kKvGroup - r.b0);
  return r;
}

// Which sequences run on the tensor cores' tiles, as the host's layout has it: the device's table may end early, and a sequence's rows there are then fewer than those that
// it was planned with.  A bit for each 2^shift sequences; every: 0 none, 1 all, 2 by the bits.
constexpr int kKvKindBits = 2048;
struct KvKinds {
  uint32_t on[kKvKindBits / 32];
  int shift, every;
  __host__ __device__ __forceinline__ bool on_tiles(int s) const { return every < 2 ? every : on[s >> shift >> 5] >> (s >> shift & 31) & 1u; }
};

// Tile number `at` of the sequences that are not on the tensor cores' tiles, of `per` rows a token and `rows` a tile.  One warp; false behind the last tile.
__device__ __forceinline__ bool kv_find_tile(const KvStep& t, const KvKinds& kinds, int per, int rows, int at, int* seq, int* tile) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int s0 = 0; s0 < t.S; s0 += 32) {
    const int s = s0 + lane;
    int n = 0;
    if (s < t.S) {
      const int have = (t.cu[s + 1] - t.cu[s]) * per;
      n = have > 0 && !kinds.on_tiles(s) ? (have + rows - 1) / rows : 0;
    }
    int upto = n;                            // tiles up to and with sequence s
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + upto > at);
    if (hit) {
      const int l = __ffs(hit) - 1;
      *seq = s0 + l;
      *tile = at - before - __shfl_sync(0xffffffffu, upto - n, l);
      return true;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return false;
}

// ------------------------------------------------------------------------------------------------ host
// The device of a call for as long as it lasts: the launches go to a stream of that device.
struct OnDevice {
  int was = -1;
  cudaError_t err;
  explicit OnDevice(int dev) {
    int now = -1;
    err = cudaGetDevice(&now);
    if (err == cudaSuccess && now != dev && (err = cudaSetDevice(dev)) == cudaSuccess) was = now;
  }
  ~OnDevice() {
    if (was >= 0) cudaSetDevice(was);
  }
};

// The two structures of the C interface as the kernels take them.
inline int kv_args(const char* name, const kb2_seq_kv_cache* cache, int layer, const kb2_seq_kv_step* step, KvLayer* c, KvStep* t) {
  if (!cache || !step || !cache->k || !cache->v || !cache->k_scale || !cache->v_scale || !step->cu || !step->pages || !step->layout ||
      (step->T > 0 && (!step->positions || !step->seq_of)))                // of no tokens there are none
    return failf(KB2SEQ_ERR_VALUE, "%s: a pointer is missing", name);
  if (((uintptr_t)cache->k | (uintptr_t)cache->v | (uintptr_t)cache->k_scale | (uintptr_t)cache->v_scale) & 15)
    return failf(KB2SEQ_ERR_VALUE, "%s: the pools begin on 16 bytes", name);
  const int ps = cache->page_size;
  if (cache->fmt != KV_E4M3 && cache->fmt != KV_INT8) return failf(KB2SEQ_ERR_VALUE, "%s: format %d", name, cache->fmt);
  if (ps < kKvGroup || ps > 1024 || (ps & (ps - 1))) return failf(KB2SEQ_ERR_VALUE, "%s: pages of %d rows: a power of two from 16 to 1024", name, ps);
  if (cache->layers < 1 || cache->pages < 1 || cache->G < 1 || cache->d < 16 || cache->d > 256 || cache->d % 16 || cache->dv < 16 || cache->dv > 256 || cache->dv % 16)
    return failf(KB2SEQ_ERR_VALUE, "%s: head sizes %d / %d: multiples of 16 up to 256", name, cache->d, cache->dv);
  if (layer < 0 || layer >= cache->layers) return failf(KB2SEQ_ERR_RANGE, "%s: layer %d of %d", name, layer, cache->layers);
  if (step->T < 0 || step->S < 1 || step->max_pages < 1 || step->max_pages > (1 << 30) / ps || (step->bits && (step->words < 1 || !step->rows)))
    return failf(KB2SEQ_ERR_VALUE, "%s: bad tables", name);
  if ((long long)cache->pages * cache->G * (ps / kKvGroup) > 0x7FFFFFFFll) return failf(KB2SEQ_ERR_VALUE, "%s: too many rows in a layer", name);
  for (int s = 0; s < step->S; ++s) {        // ahead of the first launch: the kernels go by the page lists alone
    const int* l = step->layout + 4 * s;
    if (step->bits && l[1] > 32ll * step->words)
      return failf(KB2SEQ_ERR_VALUE, "%s: sequence %d: %d words of bits for %d drafted tokens", name, s, step->words, l[1]);
    if (l[1] > 0 && (long long)l[2] + l[1] > (long long)l[3] * ps)
      return failf(KB2SEQ_ERR_RANGE, "%s: sequence %d: %d pages of %d rows do not hold %lld positions", name, s, l[3], ps, (long long)l[2] + l[1]);
  }
  int lps = 0;
  while (1 << lps < ps) ++lps;
  const long long rows = (((long long)cache->pages * cache->G) << lps) * layer;
  *c = {(uint8_t*)cache->k + rows * cache->d, (uint8_t*)cache->v + rows * cache->dv, cache->k_scale + rows, cache->v_scale + rows, cache->pages, lps, cache->G, cache->d,
        cache->dv};
  *t = {step->positions, step->seq_of, step->cu, step->pages, step->rows ? step->rows : step->positions, step->bits, step->words, step->T, step->S, step->max_pages};
  return KB2SEQ_OK;
}

}  // namespace kb2seq
