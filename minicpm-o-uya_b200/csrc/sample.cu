// sample.cu -- tokens drawn from logits with temperature, top-k, top-p and
// min-p, from given random numbers.
//
// Every cut of the kept prefix and the draw itself is one question: in the
// order of the tokens (logit descending, index ascending), where does a count
// or a sum of weights reach a target?  Sorting a row would answer them all;
// the kernel instead narrows each question to the few tokens that decide it.
//
// One thread-block cluster holds one row in its shared memory, so the logits
// are read from HBM once.  The distance from the largest logit, in base-2
// units of the temperature, gives each token one of 2048 bins; prefix sums
// over the bins' counts (and weights) bound where each target lies.  When all
// that the filters can keep fits one CTA it is gathered there, sorted, and
// every question is answered from running sums; otherwise each question is
// answered alone: its bin is narrowed by further histograms until what is left
// can be sorted, or is one value.
//
// Weights are 2^(-distance) in 64-bit floating point, rounded to multiples of
// 2^-shift of the largest, and added as 64-bit integers: sums do not depend on
// the order, and are off by at most 2^-(shift + 1) per token (shift = 62 -
// log2(vocab), 44 for 152k tokens), where f32 sums would move the borders.
// The work per token, not HBM, is the bound: about 12 64-bit operations, a
// few f32 ones and one or two shared-memory atomics.  A row of 152k tokens
// takes 18 us, most of it the chain of cluster barriers; 32 f32 rows with mixed
// filters 55 to 62 (as long as the row with the most kept tokens), 128 bf16
// rows 124 (0.3 TB/s of logits: four rounds of rows, about 10 us of 64-bit
// arithmetic per 19k tokens and CTA).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <limits.h>
#include <math.h>
#include <stdint.h>

#include "paged.cuh"

namespace mcpo {
namespace {

namespace cg = cooperative_groups;

constexpr int kSmpThreads = 512;     // two CTAs per SM: one row's barriers pass behind another's arithmetic
constexpr int kSmpBins = 2048;
constexpr int kSmpSort = 1024;       // tokens that one CTA sorts: two per thread
constexpr int kSmpSlice = 47 * 1024; // tokens of one CTA at most: their logits fill its shared memory
constexpr int kSmpHalf = 19 * 1024 + 512;  // tokens that leave room for a second CTA
constexpr int kSmpMaxCluster = 16;
constexpr int kSmpMaxVocab = 1 << 19;
constexpr float kBinsPerOctave = 32.0f;  // 2048 bins: 64 octaves
constexpr int kExpTable = 64;
constexpr float kTopPOff = 0.999999f, kGreedyBelow = 1e-6f;
constexpr uint32_t kKeyNegInf = 0x007fffffu, kKeyInf = 0xff800000u;

struct SampleArgs {
  const void* logits;
  long long stride;
  int rows, vocab, slice, shift;
  const float* temperature;
  const int32_t* top_k;
  const float *top_p, *min_p, *uniform;
  int32_t* tokens;
  float* probs;
  int32_t* kept;
};

// Integers in the order of the floats (no NaN, no -0).
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

struct Row {
  float top, c_bins, d_max;  // the largest logit; bins per unit of distance; the distance of the last bin
  double top64, c64;         // -kExpTable * log2(e) / T
  int shift;
  const double* table;       // 2^(-j / kExpTable)

  // weight * 2^shift, rounded.  With t = distance * 64 in base-2 units, t =
  // 64 e + j + r, |r| <= 1/2: 2^(-t / 64) = 2^-e * table[j] * e^(-r ln 2 / 64),
  // the last by its Taylor series to the 5th power (the next term is below
  // 2^-54 of it).
  __device__ __forceinline__ unsigned long long mass(float x) const {
    // from 53 octaves on it is below half a unit for every shift
    const double d = ((double)x - top64) * c64, t = d < (double)(kExpTable * 53) ? d : (double)(kExpTable * 53);
    const double big = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number
    const double kf = t + big;
    const int k = __double2loint(kf);
    const double r = (t - (kf - big)) * (-0.69314718055994530942 / kExpTable);
    double p = fma(r, 1.0 / 120.0, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    const double f = table[k & (kExpTable - 1)];
    const double scaled = __hiloint2double(__double2hiint(f) + (shift - k / kExpTable) * (1 << 20), __double2loint(f));
    return __double_as_longlong(fma(p, scaled, 4503599627370496.0)) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ double weight(float x) const {
    return exp2(((double)x - top64) * (c64 * (-1.0 / kExpTable)));
  }
  // never decreases as x falls: each step is a rounding of a monotone one
  __device__ __forceinline__ int bin(float x) const {
    const float d = fminf(top - x, d_max);
    return __float_as_int(fmaf(d, c_bins, 8388608.0f)) & 0xffff;  // 2^23: to the nearest whole number
  }
};

// A place in the order of the tokens.
struct Place {
  int n;                     // tokens up to and with it
  unsigned long long mass;   // their weights
  uint32_t key;
  int index;                 // -1: not asked for
};

// The bin where a target is reached.
struct Found {
  int bin, cnt;              // its tokens
  int above_cnt;             // those above it, and their weights
  unsigned long long above_mass;
};

struct alignas(16) Shared {
  // this CTA's histogram; after add_up its share of the bins holds the cluster's
  uint32_t cnt[kSmpBins], mass_lo[kSmpBins], mass_hi[kSmpBins];
  unsigned long long list[kSmpSort];   // gathered tokens, key in the upper half, ~index in the lower
  double table[kExpTable];
  unsigned long long red[2][kSmpThreads / 32];
  uint32_t top;
  int valid, word, list_n;
  unsigned long long mark;
  // written by the other CTAs of the cluster
  uint32_t lo[kSmpMaxCluster], hi[kSmpMaxCluster];
  int same[kSmpMaxCluster];
  unsigned long long z[kSmpMaxCluster], tot_c[kSmpMaxCluster], tot_m[kSmpMaxCluster];
  Found found;
  Place place;
};

// Inclusive block scan of (c, m); tc and tm get the block's sums.
__device__ __forceinline__ void scan2(Shared& s, unsigned long long& c, unsigned long long& m, unsigned long long& tc,
                                      unsigned long long& tm) {
  constexpr int kWarps = kSmpThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long cu = __shfl_up_sync(0xffffffffu, c, o), mu = __shfl_up_sync(0xffffffffu, m, o);
    if (lane >= o) c += cu, m += mu;
  }
  if (lane == 31) s.red[0][warp] = c, s.red[1][warp] = m;
  __syncthreads();
  unsigned long long bc = 0, bm = 0;
  tc = tm = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const unsigned long long x = s.red[0][w], y = s.red[1][w];
    if (w < warp) bc += x, bm += y;
    tc += x, tm += y;
  }
  c += bc, m += bm;
  __syncthreads();
}

struct Sampler {
  Shared& s;
  const float* xs;  // this CTA's logits, -inf beyond n up to a multiple of 4
  int n, base;      // how many, the first one's index
  int rank, size;
  Row row;
  cg::cluster_group cl;
  bool level0;      // the shares hold the bins' histogram with counts and weights
  unsigned long long ex_c, ex_m;  // of the last totals(): the share's count and weight before this thread's bins

  __device__ __forceinline__ Shared* of(int r) const { return cl.map_shared_rank(&s, r); }

  // ---- histograms ----
  __device__ __forceinline__ void clear(bool masses) {
    for (int b = threadIdx.x; b < kSmpBins; b += kSmpThreads) {
      s.cnt[b] = 0;
      if (masses) s.mass_lo[b] = s.mass_hi[b] = 0;
    }
    __syncthreads();
  }
  __device__ __forceinline__ void weigh(int b, unsigned long long q) {
    const uint32_t lo = (uint32_t)q, old = atomicAdd(&s.mass_lo[b], lo);
    const uint32_t up = (uint32_t)(q >> 32) + (old + lo < old ? 1u : 0u);
    if (up) atomicAdd(&s.mass_hi[b], up);
  }
  // Each CTA adds its share of the bins over the cluster, in place: nobody
  // else reads those here.
  __device__ __forceinline__ void add_up(bool masses) {
    cl.sync();
    const int share = kSmpBins / size;
    for (int b = rank * share + (int)threadIdx.x; b < (rank + 1) * share; b += kSmpThreads) {
      uint32_t c = 0;
      unsigned long long m = 0;
      for (int r0 = 0; r0 < size; r0 += 8) {
        uint32_t n[8], lo[8], hi[8];  // all loads before the sums
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          n[j] = lo[j] = hi[j] = 0;
          if (r0 + j < size) {
            const Shared* o = of(r0 + j);
            n[j] = o->cnt[b];
            if (masses) lo[j] = o->mass_lo[b], hi[j] = o->mass_hi[b];
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) c += n[j], m += ((unsigned long long)hi[j] << 32) + lo[j];
      }
      s.cnt[b] = c;
      if (masses) s.mass_lo[b] = (uint32_t)m, s.mass_hi[b] = (uint32_t)(m >> 32);
    }
    __syncthreads();
  }

  // The bins' counts, and the sum of this thread's weights if asked for.
  template <bool kWeights>
  __device__ __forceinline__ unsigned long long counts() {
    clear(false);
    unsigned long long z = 0;
    for (int i = threadIdx.x * 4; i < n; i += kSmpThreads * 4) {
      const float4 v = *reinterpret_cast<const float4*>(xs + i);
      const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (kWeights) z += row.mass(x[j]);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (x[j] > -INFINITY) atomicAdd(&s.cnt[row.bin(x[j])], 1u);
    }
    return z;
  }
  // The bins' counts and weights.
  __device__ __forceinline__ void histogram() {
    clear(true);
    for (int i = threadIdx.x * 4; i < n; i += kSmpThreads * 4) {
      const float4 v = *reinterpret_cast<const float4*>(xs + i);
      const float x[4] = {v.x, v.y, v.z, v.w};
      unsigned long long q[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) q[j] = row.mass(x[j]);  // apart from the atomics, to overlap
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (x[j] > -INFINITY) {
          const int b = row.bin(x[j]);
          atomicAdd(&s.cnt[b], 1u);
          weigh(b, q[j]);
        }
    }
    add_up(true);
    totals();
    level0 = true;
  }
  // The same of the keys in [lo, hi], by (hi - key) >> shift.
  __device__ __forceinline__ void histogram_of(uint32_t lo, uint32_t hi, int shift) {
    clear(true);
    for (int i = threadIdx.x; i < n; i += kSmpThreads) {
      const uint32_t key = key_of(xs[i]);
      if (key >= lo && key <= hi) {
        const int b = (int)((hi - key) >> shift);
        atomicAdd(&s.cnt[b], 1u);
        weigh(b, row.mass(xs[i]));
      }
    }
    add_up(true);
    totals();
    level0 = false;
  }

  // ---- sums over the bins ----
  // This thread's bins [b, e) of the CTA's share, and their count and weight.
  __device__ __forceinline__ void my_bins(int& b, int& e) const {
    const int share = kSmpBins / size, per = max(1, share / kSmpThreads);
    b = rank * share + min(share, (int)threadIdx.x * per);
    e = rank * share + min(share, ((int)threadIdx.x + 1) * per);
  }
  __device__ __forceinline__ unsigned long long bin_mass(int b) const {
    return ((unsigned long long)s.mass_hi[b] << 32) + s.mass_lo[b];
  }
  // Tells every CTA this one's sums, and waits for theirs.
  __device__ __forceinline__ void tell(unsigned long long c, unsigned long long m) {
    if ((int)threadIdx.x < size) {
      Shared* o = of(threadIdx.x);
      o->tot_c[rank] = c;
      o->tot_m[rank] = m;
    }
    cl.sync();
  }
  __device__ __forceinline__ void totals() {
    int b, e;
    my_bins(b, e);
    unsigned long long c = 0, m = 0, tc, tm;
    for (int i = b; i < e; ++i) c += s.cnt[i], m += bin_mass(i);
    ex_c = c, ex_m = m;
    scan2(s, c, m, tc, tm);
    ex_c = c - ex_c, ex_m = m - ex_m;
    tell(tc, tm);
  }
  __device__ __forceinline__ void before_me(unsigned long long& c, unsigned long long& m) const {
    for (int r = 0; r < rank; ++r) c += s.tot_c[r], m += s.tot_m[r];
  }
  // The first bin where, on top of what is above, the running count reaches
  // `count`, or (count == 0) the running weight reaches `mass` > 0.  The
  // target lies above what is above and is reached, so one bin has it.
  __device__ __forceinline__ Found find_bin(unsigned long long count, unsigned long long mass, int above_cnt,
                                            unsigned long long above_mass) {
    int b, e;
    my_bins(b, e);
    unsigned long long pc = above_cnt + ex_c, pm = above_mass + ex_m;
    before_me(pc, pm);
    for (int i = b; i < e; ++i) {
      const unsigned long long nc = pc + s.cnt[i], nm = pm + bin_mass(i);
      if (count ? pc < count && nc >= count : pm < mass && nm >= mass)
        for (int r = 0; r < size; ++r) of(r)->found = Found{i, (int)(nc - pc), (int)pc, pm};
      pc = nc, pm = nm;
    }
    cl.sync();
    return s.found;
  }

  // The smallest key whose bin is at most b.  Every thread of the cluster
  // finds the same.
  __device__ __forceinline__ uint32_t first_key(int b) const {
    const uint32_t top = key_of(row.top);
    auto in = [&](long long key) { return key > top || (key > kKeyNegInf && row.bin(value_of((uint32_t)key)) <= b); };
    // where bin b should end, give or take f32 roundings; else a search of all keys
    const int lane = threadIdx.x & 31;
    const float guess = fmaxf(row.top - ((float)b + 0.5f) / row.c_bins, -FLT_MAX);
    const long long g = (long long)key_of(guess + 0.0f) - 16;
    const unsigned in32 = __ballot_sync(0xffffffffu, in(g + lane));
    if (in32 != 0xffffffffu && in32 != 0u) return (uint32_t)(g + __ffs(in32) - 1);
    uint32_t lo = kKeyNegInf, hi = top;  // lo is out, hi is in
    while (hi - lo > 1) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if (in(mid)) hi = mid;
      else lo = mid;
    }
    return hi;
  }

  // ---- gathering ----
  __device__ __forceinline__ void empty_list() {  // the leader, before a cluster barrier
    if (rank == 0) {
      s.list[threadIdx.x] = s.list[threadIdx.x + kSmpThreads] = 0;
      if (threadIdx.x == 0) s.list_n = 0;
    }
  }
  // Gathers the tokens with logits in [lo, hi] (at most kSmpSort) into the
  // leader's list, sorted: largest first, equal ones by index.
  __device__ __forceinline__ void gather(float lo, float hi) {
    Shared* lead = of(0);
    for (int i = threadIdx.x * 4; i < n; i += kSmpThreads * 4) {
      const float4 v = *reinterpret_cast<const float4*>(xs + i);
      const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (x[j] >= lo && x[j] <= hi) {
          const int at = atomicAdd(&lead->list_n, 1);
          if (at < kSmpSort) lead->list[at] = ((unsigned long long)key_of(x[j]) << 32) | (uint32_t)~(base + i + j);
        }
    }
    cl.sync();
    if (rank != 0) return;
    // bitonic, places tid and tid + 512 in a thread (all keys differ: the
    // indexes do); empty places are 0
    int m = 32;
    while (m < s.list_n && m < kSmpSort) m <<= 1;
    const int i0 = threadIdx.x, i1 = i0 + kSmpThreads;
    unsigned long long v0 = s.list[i0], v1 = s.list[i1];
    auto swap = [&](unsigned long long v, unsigned long long o, int i, int k, int j) {
      const bool take_max = ((i & j) == 0) == ((i & k) == 0);  // runs with bit k clear descend
      return take_max ? (o > v ? o : v) : (o < v ? o : v);
    };
    for (int k = 2; k <= m; k <<= 1) {
      for (int j = k >> 1; j > 0; j >>= 1) {
        if (j == kSmpThreads) {
          const unsigned long long a = v0, b = v1;
          v0 = swap(a, b, i0, k, j);
          v1 = swap(b, a, i1, k, j);
        } else if (j >= 32) {
          __syncthreads();
          s.list[i0] = v0;
          s.list[i1] = v1;
          __syncthreads();
          v0 = swap(v0, s.list[i0 ^ j], i0, k, j);
          v1 = swap(v1, s.list[i1 ^ j], i1, k, j);
        } else {
          v0 = swap(v0, __shfl_xor_sync(0xffffffffu, v0, j), i0, k, j);
          if (m > kSmpThreads) v1 = swap(v1, __shfl_xor_sync(0xffffffffu, v1, j), i1, k, j);
        }
      }
    }
    __syncthreads();
    s.list[i0] = v0;
    s.list[i1] = v1;
    __syncthreads();
  }

  // The sorted list's tokens 2 tid and 2 tid + 1 and the running sums up to
  // them, on top of what is above.  Leader's block.
  __device__ __forceinline__ void sums(unsigned long long above, uint32_t (&key)[2], unsigned long long (&sum)[2]) {
    unsigned long long q[2], c = 0, tc, tm;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const unsigned long long v = s.list[2 * threadIdx.x + j];
      key[j] = (uint32_t)(v >> 32);
      q[j] = v ? row.mass(value_of(key[j])) : 0;
    }
    unsigned long long m = q[0] + q[1];
    scan2(s, c, m, tc, tm);
    sum[1] = above + m;
    sum[0] = sum[1] - q[1];
  }
  // How many of the leader's list's tokens satisfy a condition.
  __device__ __forceinline__ int how_many(bool a, bool b) const { return __syncthreads_count(a) + __syncthreads_count(b); }

  // The place where the running count reaches `count` (> 0), or the running
  // weight reaches `mass` (> 0, at most all), over all tokens.  Cluster-wide;
  // with kFinal the leader alone has the answer, with the token's index; else
  // every CTA has it, without.
  template <bool kFinal>
  __device__ __forceinline__ Place find(unsigned long long count, unsigned long long mass) {
    empty_list();
    Found f = find_bin(count, mass, 0, 0);
    uint32_t lo = first_key(f.bin), hi = f.bin ? first_key(f.bin - 1) - 1 : key_of(row.top);
    while (f.cnt > kSmpSort) {
      // the keys that are really there
      uint32_t l = 0xffffffffu, h = 0;
      for (int i = threadIdx.x; i < n; i += kSmpThreads) {
        const uint32_t key = key_of(xs[i]);
        if (key >= lo && key <= hi) l = min(l, key), h = max(h, key);
      }
      l = __reduce_min_sync(0xffffffffu, l);
      h = __reduce_max_sync(0xffffffffu, h);
      if ((threadIdx.x & 31) == 0) s.red[0][threadIdx.x >> 5] = ((unsigned long long)h << 32) | l;
      __syncthreads();
      if ((int)threadIdx.x < size) {
        for (int w = 0; w < kSmpThreads / 32; ++w)
          l = min(l, (uint32_t)s.red[0][w]), h = max(h, (uint32_t)(s.red[0][w] >> 32));
        Shared* o = of(threadIdx.x);
        o->lo[rank] = l;
        o->hi[rank] = h;
      }
      cl.sync();
      lo = 0xffffffffu, hi = 0;
      for (int r = 0; r < size; ++r) lo = min(lo, s.lo[r]), hi = max(hi, s.hi[r]);
      if (lo == hi) {  // equal logits: the place follows from their count, the index from their order
        const unsigned long long w = row.mass(value_of(lo));
        unsigned long long m = count ? count - f.above_cnt : w ? (mass - f.above_mass + w - 1) / w : 1;
        m = m < 1 ? 1 : m > (unsigned long long)f.cnt ? (unsigned long long)f.cnt : m;
        Place p{f.above_cnt + (int)m, f.above_mass + m * w, lo, kFinal ? nth(lo, (int)m) : -1};
        cl.sync();  // lo and hi may be written again from here on
        return p;
      }
      const int shift = max(0, 32 - __clz(hi - lo) - 11);
      histogram_of(lo, hi, shift);
      f = find_bin(count, mass, f.above_cnt, f.above_mass);
      hi -= (uint32_t)f.bin << shift;
      const uint32_t span = (1u << shift) - 1;
      lo = hi - lo > span ? hi - span : lo;
    }
    gather(value_of(lo), value_of(hi));
    if (rank == 0) {
      uint32_t key[2];
      unsigned long long sum[2];
      sums(f.above_mass, key, sum);
      const int left = s.list_n, i = 2 * threadIdx.x;
      auto before = [&](int j) {
        return i + j < left && (count ? (unsigned long long)(f.above_cnt + i + j + 1) < count : sum[j] < mass);
      };
      const int at = min(how_many(before(0), before(1)), left - 1);
      if (at >> 1 == (int)threadIdx.x) {
        const Place p{f.above_cnt + at + 1, sum[at & 1], key[at & 1], (int)~(uint32_t)s.list[at]};
        if (kFinal) s.place = p;
        else
          for (int r = 0; r < size; ++r) of(r)->place = p;
      }
      if (kFinal) __syncthreads();
    }
    if (!kFinal) cl.sync();
    const Place p = s.place;
    if (!kFinal) cl.sync();
    return p;
  }

  // The index of the m-th token (from 1) whose key is `key`; every CTA has it.
  __device__ __forceinline__ int nth(uint32_t key, int m) {
    const int per = (n + kSmpThreads - 1) / kSmpThreads, i0 = min(n, (int)threadIdx.x * per), i1 = min(n, i0 + per);
    unsigned long long mine = 0, none = 0, all, tm;
    const float x = value_of(key);
    for (int i = i0; i < i1; ++i) mine += xs[i] == x;
    unsigned long long incl = mine;
    scan2(s, incl, none, all, tm);
    if ((int)threadIdx.x < size) of(threadIdx.x)->same[rank] = (int)all;
    cl.sync();
    int before = 0;
    for (int r = 0; r < rank; ++r) before += s.same[r];
    const int lo = before + (int)(incl - mine);
    if (m > lo && m <= lo + (int)mine) {
      int at = lo;
      for (int i = i0; i < i1; ++i)
        if (xs[i] == x && ++at == m) {
          for (int r = 0; r < size; ++r) of(r)->word = base + i;
          break;
        }
    }
    cl.sync();
    const int index = s.word;
    cl.sync();
    return index;
  }
};

template <typename T>
__device__ __forceinline__ float as_float(T x);
template <>
__device__ __forceinline__ float as_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ float as_float<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float as_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__global__ void __launch_bounds__(kSmpThreads, 2) k_sample(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Shared& s = *reinterpret_cast<Shared*>(smem_raw);
  float* xs = reinterpret_cast<float*>(smem_raw + sizeof(Shared));
  cg::cluster_group cl = cg::this_cluster();
  const int size = (int)cl.num_blocks(), rank = (int)cl.block_rank(), b = blockIdx.x / size, tid = threadIdx.x;
  const int base = min(a.vocab, rank * a.slice), n = min(a.vocab, base + a.slice) - base;
  const T* x = static_cast<const T*>(a.logits) + b * a.stride + base;

  // the row (NaN as -inf, -0 as 0), the largest logit and the number above -inf
  float high = -INFINITY;
  int valid = 0;
  auto take = [&](float v) {
    v = v == v ? v + 0.0f : -INFINITY;
    high = fmaxf(high, v);
    valid += v > -INFINITY;
    return v;
  };
  constexpr int kVec = 16 / sizeof(T);
  int done = 0;
  if (aligned16(x)) {
    done = n / kVec * kVec;
#pragma unroll 4
    for (int i = tid * kVec; i < done; i += kSmpThreads * kVec) {
      const uint4 u = __ldcs(reinterpret_cast<const uint4*>(x + i));
      T v[kVec];
      memcpy(v, &u, 16);
#pragma unroll
      for (int j = 0; j < kVec; j += 4) {
        const float4 f = make_float4(take(as_float<T>(v[j])), take(as_float<T>(v[j + 1])), take(as_float<T>(v[j + 2])),
                                     take(as_float<T>(v[j + 3])));
        *reinterpret_cast<float4*>(xs + i + j) = f;
      }
    }
  }
  for (int i = done + tid; i < n; i += kSmpThreads) xs[i] = take(as_float<T>(x[i]));
  if (tid < 4 && n + tid < (n + 3) / 4 * 4) xs[n + tid] = -INFINITY;
  if (tid < kExpTable) s.table[tid] = exp2(-(double)tid / kExpTable);
  uint32_t top = __reduce_max_sync(0xffffffffu, key_of(high));
  valid = __reduce_add_sync(0xffffffffu, valid);
  if ((tid & 31) == 0) s.red[0][tid >> 5] = ((unsigned long long)top << 32) | (unsigned)valid;
  __syncthreads();
  if (tid == 0) {
    top = 0, valid = 0;
    for (int w = 0; w < kSmpThreads / 32; ++w)
      top = max(top, (uint32_t)(s.red[0][w] >> 32)), valid += (int)(uint32_t)s.red[0][w];
    s.top = top;
    s.valid = valid;
  }
  cl.sync();
  top = 0, valid = 0;
  for (int r = 0; r < size; ++r) {
    const Shared* o = cl.map_shared_rank(&s, r);
    top = max(top, o->top), valid += o->valid;
  }

  const float temp = a.temperature ? a.temperature[b] : 1.0f;
  const int k_in = a.top_k ? a.top_k[b] : 0;
  const float p_in = a.top_p ? a.top_p[b] : 1.0f, mp_in = a.min_p ? a.min_p[b] : 0.0f, u_in = a.uniform[b];
  const bool use_p = p_in < kTopPOff, use_mp = mp_in > 0.0f;
  const double u = u_in > 0.0f ? (u_in < 1.0f ? (double)u_in : 1.0) : 0.0;
  const bool writer = rank == 0 && tid == 0;
  Row row{};
  row.shift = a.shift;
  row.table = s.table;
  Sampler smp{s, xs, n, base, rank, size, row, cl, false, 0, 0};

  if (valid == 0) {  // nothing can be drawn; the same in every CTA
    cl.sync();         // the others have read this one's words
    if (writer) {
      a.tokens[b] = 0;
      if (a.probs) a.probs[b] = 0.0f;
      if (a.kept) a.kept[b] = 0;
    }
    return;
  }
  if (!(temp > kGreedyBelow) || k_in == 1) {
    const int at = smp.nth(top, 1);
    if (writer) {
      a.tokens[b] = at;
      if (a.probs) a.probs[b] = 1.0f;
      if (a.kept) a.kept[b] = 1;
    }
    return;
  }
  if (top == kKeyInf) {  // the tokens at +inf share the weight, whatever the rest
    for (int i = tid; i < n; i += kSmpThreads) {
      const bool in = xs[i] == INFINITY;
      xs[i] = in ? 0.0f : xs[i] > -INFINITY ? -FLT_MAX : -INFINITY;
    }
    top = key_of(0.0f);
    __syncthreads();
  }
  row.top = value_of(top);
  row.top64 = (double)row.top;
  row.c64 = -1.4426950408889634074 / (double)temp * kExpTable;
  row.c_bins = (float)(1.4426950408889634074 / (double)temp * kBinsPerOctave);
  row.d_max = fminf((float)(kSmpBins - 1) / row.c_bins, FLT_MAX);
  smp.row = row;

  const int k = k_in > 0 && k_in < valid ? k_in : valid;
  const bool any = use_p || use_mp || k < valid;
  int kept = valid;
  unsigned long long norm = 0;
  if (any) {
    // the bins that can hold kept tokens: up to where each filter's target is
    // surely reached, every token of a bin weighing at least the bin's end
    unsigned long long p_mass = 1;
    if (use_p) {
      unsigned long long z = smp.counts<true>(), c = 0, tc, tm;
      scan2(s, c, z, tc, tm);
      if (tid < size) cl.map_shared_rank(&s, tid)->z[rank] = tm;
    } else {
      smp.counts<false>();
    }
    smp.add_up(false);
    if (use_p) {
      unsigned long long z = 0;
      for (int r = 0; r < size; ++r) z += s.z[r];
      p_mass = (unsigned long long)fmax(1.0, ceil((double)p_in * (double)z));
    }
    smp.empty_list();
    int b0, b1;
    smp.my_bins(b0, b1);
    // bin b ends at b + 1/2, and f32 rounding moves a distance by less than 2^-20 of it
    unsigned long long c = 0, m = 0, tc, tm, pc = 0, pm = 0;
    for (int i = b0; i < b1; ++i) {
      c += s.cnt[i];
      if (use_p && i < kSmpBins - 1)
        m += (unsigned long long)((double)s.cnt[i] * exp2((-(double)i - 0.75) / kBinsPerOctave) * (double)(1ull << a.shift));
    }
    const unsigned long long c0 = c, m0 = m;
    scan2(s, c, m, tc, tm);
    smp.tell(tc, tm);
    smp.before_me(pc, pm);
    pc += c - c0, pm += m - m0;  // before this thread's bins
    const int min_bin =
        use_mp ? (int)fmin((double)kSmpBins, fmax(0.0, -log2((double)mp_in)) * kBinsPerOctave + 2.0) : kSmpBins;
    auto ended = [&](unsigned long long c, unsigned long long m, int b) {  // by the bins before b
      return c >= (unsigned long long)k || (use_p && m >= p_mass) || b >= min_bin;
    };
    if (b0 < b1 && !ended(pc, pm, b0) && ended(pc + c0, pm + m0, b1))
      for (int r = 0; r < size; ++r) cl.map_shared_rank(&s, r)->found = Found{b1 - 1, (int)(pc + c0), 0, 0};
    cl.sync();
    const Found last = s.found;
    if (last.cnt <= kSmpSort) {
      smp.gather(value_of(smp.first_key(last.bin)), row.top);
      if (rank == 0) {
        uint32_t key[2];
        unsigned long long sum[2];
        smp.sums(0, key, sum);
        const int left = s.list_n;
        const bool h0 = 2 * tid < left, h1 = 2 * tid + 1 < left;
        int m = min(k, left);
        if (use_p) m = min(m, smp.how_many(h0 && sum[0] < p_mass, h1 && sum[1] < p_mass) + 1);
        if (use_mp)
          m = min(m, smp.how_many(h0 && row.weight(value_of(key[0])) >= (double)mp_in,
                                  h1 && row.weight(value_of(key[1])) >= (double)mp_in));
        m = max(m, 1);
        if ((m - 1) >> 1 == tid) s.mark = sum[(m - 1) & 1];
        __syncthreads();
        const unsigned long long all = s.mark, target = (unsigned long long)ceil(u * (double)all);
        const int at = min(smp.how_many(h0 && sum[0] < target, h1 && sum[1] < target), m - 1);
        if (at >> 1 == tid) {
          a.tokens[b] = (int)~(uint32_t)s.list[at];
          if (a.probs)
            a.probs[b] = (float)(row.weight(value_of(key[at & 1])) * (double)(1ull << a.shift) / (double)all);
          if (a.kept) a.kept[b] = m;
        }
      }
      return;
    }
    cl.sync();  // found and tot may be written again from here on
    smp.histogram();
    kept = k;
    if (use_p) {
      const Place p = smp.find<false>(0, p_mass);
      if (p.n <= kept) kept = p.n, norm = p.mass;
    }
    if (use_mp) {
      unsigned long long likely = 0, c = 0, tc, tm;
      for (int i = tid; i < n; i += kSmpThreads) likely += xs[i] > -INFINITY && row.weight(xs[i]) >= (double)mp_in;
      scan2(s, c, likely, tc, tm);
      if (tid < size) cl.map_shared_rank(&s, tid)->z[rank] = tm;
      cl.sync();
      unsigned long long all = 0;
      for (int r = 0; r < size; ++r) all += s.z[r];
      cl.sync();
      if (all < (unsigned long long)kept) kept = (int)all, norm = 0;
    }
    kept = max(kept, 1);
    if (!smp.level0) smp.histogram();
    if (!norm) norm = smp.find<false>((unsigned long long)kept, 0).mass;
    if (!smp.level0) smp.histogram();
  } else {
    smp.histogram();
    for (int r = 0; r < size; ++r) norm += s.tot_m[r];
  }
  const unsigned long long target = (unsigned long long)fmax(1.0, ceil(u * (double)norm));
  const Place f = smp.find<true>(0, target < norm ? target : norm);
  if (writer) {
    a.tokens[b] = f.index;
    if (a.probs) a.probs[b] = (float)(row.weight(value_of(f.key)) * (double)(1ull << a.shift) / (double)norm);
    if (a.kept) a.kept[b] = kept;
  }
}

template <typename T>
cudaError_t launch_sample(const SampleArgs& a, int cluster, cudaStream_t st) {
  const size_t smem = sizeof(Shared) + (size_t)a.slice * 4;
  static OncePerDevice once;
  cudaError_t e = once([] {
    cudaError_t r = cudaFuncSetAttribute(k_sample<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)(sizeof(Shared) + (size_t)kSmpSlice * 4));
    if (r == cudaSuccess) r = cudaFuncSetAttribute(k_sample<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    return r;
  });
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * cluster));
  cfg.blockDim = dim3(kSmpThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_sample<T>, a);
}

static_assert(sizeof(Shared) % 16 == 0, "keys are 16-byte aligned");
static_assert(sizeof(Shared) + (size_t)kSmpSlice * 4 <= 232448, "a slice fits shared memory");
static_assert(2 * (sizeof(Shared) + (size_t)kSmpHalf * 4 + 1024) <= 228 * 1024, "two CTAs fit an SM");
static_assert((long long)kSmpSlice * kSmpMaxCluster >= kSmpMaxVocab, "a cluster holds a row");

}  // namespace
}  // namespace mcpo

using namespace mcpo;

extern "C" int minicpmo_gpu_sample(const void* logits, int dtype, size_t rows, size_t vocab, size_t stride,
                                   const float* temperature, const int32_t* top_k, const float* top_p,
                                   const float* min_p, const float* uniform, int32_t* tokens, float* probs,
                                   int32_t* kept, void* stream, char* error, size_t error_cap) {
  const char* op = "sample";
  const size_t esz = paged_type_bytes(dtype);
  if (!esz) return paged_error(error, error_cap, "error: %s: dtype %d is not F32, F16 or BF16", op, dtype);
  if (rows == 0) return 1;
  if (!logits || !uniform || !tokens) return paged_error(error, error_cap, "error: %s: null buffer", op);
  if (rows > (1u << 20) || vocab < 1 || vocab > (size_t)kSmpMaxVocab)
    return paged_error(error, error_cap, "error: %s: %zu rows of %zu tokens (at most %d)", op, rows, vocab, kSmpMaxVocab);
  if (stride < vocab || stride > (1ull << 40))
    return paged_error(error, error_cap, "error: %s: rows of %zu tokens, %zu apart", op, vocab, stride);
  if (reinterpret_cast<uintptr_t>(logits) % esz) return paged_error(error, error_cap, "error: %s: misaligned logits", op);
  if (!paged_on_device(logits, op, error, error_cap)) return 0;
  SampleArgs a{};
  a.logits = logits;
  a.stride = (long long)stride;
  a.rows = (int)rows;
  a.vocab = (int)vocab;
  int bits = 0;
  while ((1ull << bits) < vocab) ++bits;
  a.shift = 62 - bits < 50 ? 62 - bits : 50;
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  a.uniform = uniform;
  a.tokens = tokens;
  a.probs = probs;
  a.kept = kept;
  // CTAs per row: as few as hold it, two to an SM where 8 (the portable
  // cluster) can; more while there are SMs for them and each has 4096 tokens
  int cluster = 1;
  while (cluster < 8 && (size_t)cluster * kSmpHalf < vocab) cluster *= 2;
  while ((size_t)cluster * kSmpSlice < vocab) cluster *= 2;
  while (cluster < 8 && rows * cluster * 2 <= 148 && vocab >= (size_t)cluster * 2 * 4096) cluster *= 2;
  a.slice = (int)((vocab + cluster - 1) / cluster + 15) / 16 * 16;
  if (a.slice > kSmpSlice) a.slice = kSmpSlice;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == kF32   ? launch_sample<float>(a, cluster, st)
                        : dtype == kF16 ? launch_sample<__half>(a, cluster, st)
                                        : launch_sample<__nv_bfloat16>(a, cluster, st);
  if (e != cudaSuccess) return paged_error(error, error_cap, "error: %s: launch: %s", op, cudaGetErrorString(e));
  return 1;
}
