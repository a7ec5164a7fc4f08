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
// few f32 ones and one or two shared-memory atomics.
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

constexpr int kSmpThreads = 1024;
constexpr int kSmpBins = 2048;
constexpr int kSmpSort = 1024;       // tokens that one CTA sorts: one per thread
constexpr int kSmpSlice = 42 * 1024; // tokens of one CTA: their logits fill its shared memory
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
    const double t = ((double)x - top64) * c64;
    if (!(t < (double)(kExpTable * 53))) return 0;  // below half a unit for every shift
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

struct alignas(16) Shared {
  uint32_t cnt[kSmpBins];              // this CTA's histogram
  uint32_t mass_lo[kSmpBins], mass_hi[kSmpBins];
  uint32_t all_cnt[kSmpBins];          // the leader's: the cluster's histogram
  unsigned long long all_mass[kSmpBins];
  unsigned long long list[kSmpSort];   // gathered tokens, key in the upper half, ~index in the lower
  double table[kExpTable];
  unsigned long long red[64];
  // exchanged between the CTAs of the cluster
  uint32_t top[kSmpMaxCluster], lo[kSmpMaxCluster], hi[kSmpMaxCluster];
  int valid[kSmpMaxCluster], same[kSmpMaxCluster];
  unsigned long long z[kSmpMaxCluster];
  int list_n;
  int word;
  // the leader's decision, which every CTA reads
  int found_bin, found_cnt, above_cnt;
  unsigned long long above_mass, total;
  Place place;
};

__device__ __forceinline__ unsigned long long shfl_up64(unsigned long long v, int o) {
  return __shfl_up_sync(0xffffffffu, v, o);
}

// Inclusive block scan of (count, mass); red is the scratch.
__device__ __forceinline__ void scan2(unsigned long long& c, unsigned long long& m, unsigned long long* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long cu = shfl_up64(c, o), mu = shfl_up64(m, o);
    if (lane >= o) c += cu, m += mu;
  }
  if (lane == 31) red[warp] = c, red[32 + warp] = m;
  __syncthreads();
  if (warp == 0) {
    unsigned long long a = red[lane], b = red[32 + lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long au = shfl_up64(a, o), bu = shfl_up64(b, o);
      if (lane >= o) a += au, b += bu;
    }
    red[lane] = a, red[32 + lane] = b;
  }
  __syncthreads();
  if (warp) c += red[warp - 1], m += red[32 + warp - 1];
  __syncthreads();
}

__device__ __forceinline__ unsigned long long block_sum(unsigned long long v, unsigned long long* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (lane == 0) red[warp] = v;
  __syncthreads();
  unsigned long long s = red[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  __syncthreads();
  return s;
}

struct Sampler {
  Shared& s;
  const float* xs;  // this CTA's logits, -inf beyond n up to a multiple of 4
  int n, base;      // how many, the first one's index
  int rank, size;
  Row row;
  cg::cluster_group cl;
  bool level0;      // the leader holds the bins' histogram with weights

  // Adds the CTAs' histograms into the leader's all_cnt / all_mass.
  __device__ void add_up(bool masses) {
    cl.sync();
    // each CTA adds its share of the bins over the cluster
    Shared* lead = cl.map_shared_rank(&s, 0);
    const int share = kSmpBins / size;
    for (int b = rank * share + (int)threadIdx.x; b < (rank + 1) * share; b += kSmpThreads) {
      uint32_t c = 0;
      unsigned long long m = 0;
      for (int r = 0; r < size; ++r) {
        const Shared* o = cl.map_shared_rank(&s, r);
        c += o->cnt[b];
        if (masses) m += ((unsigned long long)o->mass_hi[b] << 32) + o->mass_lo[b];
      }
      lead->all_cnt[b] = c;
      lead->all_mass[b] = m;
    }
    cl.sync();
  }

  __device__ __forceinline__ void clear(bool masses) {
    for (int b = threadIdx.x; b < kSmpBins; b += kSmpThreads) {
      s.cnt[b] = 0;
      if (masses) s.mass_lo[b] = s.mass_hi[b] = 0;
    }
    __syncthreads();
  }

  __device__ __forceinline__ void count(int b, unsigned long long q) {
    atomicAdd(&s.cnt[b], 1u);
    const uint32_t lo = (uint32_t)q, old = atomicAdd(&s.mass_lo[b], lo);
    const uint32_t up = (uint32_t)(q >> 32) + (old + lo < old ? 1u : 0u);
    if (up) atomicAdd(&s.mass_hi[b], up);
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
      for (int j = 0; j < 4; ++j) {
        if (x[j] > -INFINITY) atomicAdd(&s.cnt[row.bin(x[j])], 1u);
        if (kWeights) z += row.mass(x[j]);
      }
    }
    add_up(false);
    level0 = false;
    return z;
  }

  // The bins' counts and weights.
  __device__ void histogram() {
    clear(true);
    for (int i = threadIdx.x * 4; i < n; i += kSmpThreads * 4) {
      const float4 v = *reinterpret_cast<const float4*>(xs + i);
      const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (x[j] > -INFINITY) count(row.bin(x[j]), row.mass(x[j]));
    }
    add_up(true);
    level0 = true;
  }

  // The same of the keys in [lo, hi], by (hi - key) >> shift.
  __device__ void histogram_of(uint32_t lo, uint32_t hi, int shift) {
    clear(true);
    for (int i = threadIdx.x; i < n; i += kSmpThreads) {
      const uint32_t key = key_of(xs[i]);
      if (key >= lo && key <= hi) count((int)((hi - key) >> shift), row.mass(xs[i]));
    }
    add_up(true);
    level0 = false;
  }

  // The smallest key whose bin is at most b.  Block-wide; every CTA of the
  // cluster finds the same.
  __device__ uint32_t first_key(int b) {
    const uint32_t top = key_of(row.top);
    uint32_t at = 0;  // keys below `at` are in later bins
#pragma unroll 1
    for (int sh = 22; sh >= 0; sh = sh > 2 ? sh - 10 : sh - 3) {
      const unsigned long long key = at + ((unsigned long long)threadIdx.x << sh);
      const bool in = key > top || (key > kKeyNegInf && row.bin(value_of((uint32_t)key)) <= b);
      const int out = kSmpThreads - __syncthreads_count(in);  // the candidates before the first that is in
      if (out) at += (uint32_t)(out - 1) << sh;
      if (sh == 2) {  // the last four keys, one after the other
        while (at <= kKeyNegInf || (at <= top && row.bin(value_of(at)) > b)) ++at;
        break;
      }
    }
    return at;
  }

  // The leader's bin where the running count reaches `count`, or (count == 0)
  // the running weight reaches `mass`; what is above it is added to
  // s.above_cnt / s.above_mass.  The last non-empty bin if neither does.
  // Leader's whole block.
  __device__ void find_bin(unsigned long long count, unsigned long long mass) {
    const int b0 = 2 * threadIdx.x;
    const unsigned long long c0 = s.all_cnt[b0], c1 = s.all_cnt[b0 + 1], m0 = s.all_mass[b0], m1 = s.all_mass[b0 + 1];
    unsigned long long c = c0 + c1, m = m0 + m1;
    scan2(c, m, s.red);
    const unsigned long long base_c = s.above_cnt, base_m = s.above_mass;
    if (threadIdx.x == 0) s.found_bin = -1;
    __syncthreads();
    // first bin that reaches the target: exactly one thread and bin
    const unsigned long long pc = base_c + c - c0 - c1, pm = base_m + m - m0 - m1;  // before this thread's bins
    const bool r0 = count ? pc + c0 >= count : pm + m0 >= mass && c0;
    const bool r1 = count ? pc + c0 + c1 >= count : pm + m0 + m1 >= mass && c1;
    int mine = -1;
    if (r0 && c0) mine = b0;
    else if (r1 && c1) mine = b0 + 1;
    // the least such bin over the block (a target of weight 0 is reached at once)
    int least = mine < 0 ? INT_MAX : mine, last = c1 ? b0 + 1 : c0 ? b0 : -1;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
      last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
    }
    if ((threadIdx.x & 31) == 0) s.red[threadIdx.x >> 5] = (unsigned)least | ((unsigned long long)(unsigned)(last + 1) << 32);
    __syncthreads();
    least = INT_MAX, last = -1;
    for (int w = 0; w < kSmpThreads / 32; ++w) {
      least = min(least, (int)(uint32_t)s.red[w]);
      last = max(last, (int)(s.red[w] >> 32) - 1);
    }
    const int bin = least == INT_MAX ? last : least;
    if (bin >> 1 == (int)threadIdx.x) {
      s.found_bin = bin;
      s.found_cnt = (int)(bin & 1 ? c1 : c0);
      s.above_cnt = (int)(pc + (bin & 1 ? c0 : 0));
      s.above_mass = pm + (bin & 1 ? m0 : 0);
    }
    __syncthreads();
  }

  // Gathers the tokens with logits in [lo, hi] (at most kSmpSort) into the
  // leader's list, sorted.
  __device__ void gather(float lo, float hi) {
    Shared* lead = cl.map_shared_rank(&s, 0);
    if (rank == 0) {
      s.list[threadIdx.x] = 0;
      if (threadIdx.x == 0) s.list_n = 0;
    }
    cl.sync();
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
    // bitonic, largest first (all keys differ: the indexes do); empty places are 0
    int m = 32;
    while (m < s.list_n) m <<= 1;
    if (m > kSmpSort) m = kSmpSort;
    const int i = threadIdx.x;
    unsigned long long v = s.list[i];
    for (int k = 2; k <= m; k <<= 1) {
      for (int j = k >> 1; j > 0; j >>= 1) {
        unsigned long long o;
        if (j >= 32) {
          __syncthreads();
          s.list[i] = v;
          __syncthreads();
          o = s.list[i ^ j];
        } else {
          o = __shfl_xor_sync(0xffffffffu, v, j);
        }
        const bool up = (i & k) != 0, low = (i & j) == 0;  // `up`: this run ascends
        const bool take_max = low != up;
        v = take_max ? (o > v ? o : v) : (o < v ? o : v);
      }
    }
    __syncthreads();
    s.list[i] = v;
    __syncthreads();
  }

  // The sorted list's token and running sums of this thread, on top of what is above.
  __device__ __forceinline__ void sums(uint32_t& key, unsigned long long& q, unsigned long long& mass) {
    const unsigned long long v = s.list[threadIdx.x];
    key = (uint32_t)(v >> 32);
    q = v ? row.mass(value_of(key)) : 0;
    unsigned long long c = 0, m = q;
    scan2(c, m, s.red);
    mass = s.above_mass + m;
  }

  // The place where the running count reaches `count` (> 0), or the running
  // weight reaches `mass`, over all tokens.  Cluster-wide; the answer in every
  // CTA.  with_index: also the token's index.
  __device__ Place find(unsigned long long count, unsigned long long mass, bool with_index) {
    Shared* lead = cl.map_shared_rank(&s, 0);
    if (!level0) histogram();
    if (rank == 0) {
      if (threadIdx.x == 0) s.above_cnt = 0, s.above_mass = 0;
      __syncthreads();
      find_bin(count, mass);
    }
    cl.sync();
    int bin = lead->found_bin, cnt = lead->found_cnt;
    uint32_t lo = first_key(bin), hi = bin ? first_key(bin - 1) - 1 : key_of(row.top);
    while (cnt > kSmpSort) {
      // the keys that are really there
      uint32_t l = 0xffffffffu, h = 0;
      for (int i = threadIdx.x; i < n; i += kSmpThreads) {
        const uint32_t key = key_of(xs[i]);
        if (key >= lo && key <= hi) l = min(l, key), h = max(h, key);
      }
      l = __reduce_min_sync(0xffffffffu, l);
      h = __reduce_max_sync(0xffffffffu, h);
      __syncthreads();
      if ((threadIdx.x & 31) == 0) s.red[threadIdx.x >> 5] = ((unsigned long long)h << 32) | l;
      __syncthreads();
      if ((int)threadIdx.x < size) {
        for (int w = 0; w < kSmpThreads / 32; ++w) l = min(l, (uint32_t)s.red[w]), h = max(h, (uint32_t)(s.red[w] >> 32));
        Shared* o = cl.map_shared_rank(&s, threadIdx.x);
        o->lo[rank] = l;
        o->hi[rank] = h;
      }
      cl.sync();
      lo = 0xffffffffu, hi = 0;
      for (int r = 0; r < size; ++r) lo = min(lo, s.lo[r]), hi = max(hi, s.hi[r]);
      if (lo == hi) {  // equal logits: the place follows from their count, the index from their order
        const unsigned long long w = row.mass(value_of(lo)), above_m = lead->above_mass;
        const int above_c = lead->above_cnt;
        unsigned long long m;
        if (count) m = count - above_c;
        else m = w ? (mass > above_m ? (mass - above_m + w - 1) / w : 1) : 1;
        m = m < 1 ? 1 : m > (unsigned long long)cnt ? (unsigned long long)cnt : m;
        Place f{above_c + (int)m, above_m + m * w, lo, with_index ? nth(lo, (int)m) : -1};
        cl.sync();  // the leader's words may change from here on
        return f;
      }
      const int shift = max(0, 32 - __clz(hi - lo) - 11);
      histogram_of(lo, hi, shift);
      if (rank == 0) find_bin(count, mass);
      cl.sync();
      bin = lead->found_bin, cnt = lead->found_cnt;
      hi -= (uint32_t)bin << shift;
      const uint32_t span = (1u << shift) - 1;
      lo = hi - lo > span ? hi - span : lo;
    }
    gather(value_of(lo), value_of(hi));
    if (rank == 0) {
      uint32_t key;
      unsigned long long w, sum;
      sums(key, w, sum);
      const int left = s.list_n;
      const bool before = (int)threadIdx.x < left && (count ? s.above_cnt + threadIdx.x + 1 < count : sum < mass);
      const int at = min(__syncthreads_count(before), left - 1);
      if ((int)threadIdx.x == at) s.place = Place{s.above_cnt + at + 1, sum, key, (int)~(uint32_t)s.list[at]};
    }
    cl.sync();
    const Place f = lead->place;
    cl.sync();
    return f;
  }

  // The index of the m-th token (from 1) whose key is `key`.
  __device__ int nth(uint32_t key, int m) {
    const int per = (n + kSmpThreads - 1) / kSmpThreads, i0 = min(n, (int)threadIdx.x * per), i1 = min(n, i0 + per);
    unsigned long long mine = 0, none = 0;
    const float x = value_of(key);
    for (int i = i0; i < i1; ++i) mine += xs[i] == x;
    unsigned long long incl = mine;
    scan2(incl, none, s.red);
    if (threadIdx.x == kSmpThreads - 1) s.word = (int)incl;
    __syncthreads();
    if ((int)threadIdx.x < size) cl.map_shared_rank(&s, threadIdx.x)->same[rank] = s.word;
    cl.sync();
    int before = 0;
    for (int r = 0; r < rank; ++r) before += s.same[r];
    const int lo = before + (int)(incl - mine);
    if (m > lo && m <= lo + (int)mine) {
      int at = lo;
      for (int i = i0; i < i1; ++i)
        if (xs[i] == x && ++at == m) {
          for (int r = 0; r < size; ++r) cl.map_shared_rank(&s, r)->word = base + i;
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
__global__ void __launch_bounds__(kSmpThreads) k_sample(const SampleArgs a) {
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
  if ((tid & 31) == 0) s.red[tid >> 5] = ((unsigned long long)top << 32) | (unsigned)valid;
  cl.sync();  // red is written; every CTA of the cluster runs, so their shared memory can be
  if (tid < size) {
    top = 0, valid = 0;
    for (int w = 0; w < kSmpThreads / 32; ++w) top = max(top, (uint32_t)(s.red[w] >> 32)), valid += (int)(uint32_t)s.red[w];
    Shared* o = cl.map_shared_rank(&s, tid);
    o->top[rank] = top;
    o->valid[rank] = valid;
  }
  cl.sync();
  top = 0, valid = 0;
  for (int r = 0; r < size; ++r) top = max(top, s.top[r]), valid += s.valid[r];

  const float temp = a.temperature ? a.temperature[b] : 1.0f;
  const int k_in = a.top_k ? a.top_k[b] : 0;
  const float p_in = a.top_p ? a.top_p[b] : 1.0f, mp_in = a.min_p ? a.min_p[b] : 0.0f, u_in = a.uniform[b];
  const bool use_p = p_in < kTopPOff, use_mp = mp_in > 0.0f;
  const double u = u_in > 0.0f ? (u_in < 1.0f ? (double)u_in : 1.0) : 0.0;
  const bool writer = rank == 0 && tid == 0;
  Row row{};
  row.shift = a.shift;
  row.table = s.table;
  Sampler smp{s, xs, n, base, rank, size, row, cl, false};

  if (valid == 0) {  // nothing can be drawn; the same in every CTA
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
  Shared* lead = cl.map_shared_rank(&s, 0);
  int kept = valid;
  unsigned long long norm;
  if (any) {
    // the bins that can hold kept tokens: up to where each filter's target is
    // surely reached, every token of a bin weighing at least the bin's end
    unsigned long long p_mass = 0;
    if (use_p) {
      unsigned long long z = block_sum(smp.counts<true>(), s.red);
      if (tid < size) cl.map_shared_rank(&s, tid)->z[rank] = z;
      cl.sync();
      z = 0;
      for (int r = 0; r < size; ++r) z += s.z[r];
      p_mass = (unsigned long long)ceil(fmax(0.0, (double)p_in) * (double)z);
    } else {
      smp.counts<false>();
    }
    if (rank == 0) {
      const int b0 = 2 * tid;
      const unsigned long long c0 = s.all_cnt[b0], c1 = s.all_cnt[b0 + 1];
      // bin b ends at b + 1/2, and f32 rounding moves a distance by less than 2^-20 of it
      const double unit = (double)(1ull << a.shift);
      const double w0 = exp2((-(double)b0 - 0.75) / kBinsPerOctave), w1 = exp2((-(double)b0 - 1.75) / kBinsPerOctave);
      unsigned long long c = c0 + c1;
      unsigned long long m = (unsigned long long)((double)c0 * w0 * unit) +
                             (b0 + 1 == kSmpBins - 1 ? 0ull : (unsigned long long)((double)c1 * w1 * unit));
      scan2(c, m, s.red);
      const int min_bin = use_mp ? (int)fmin((double)kSmpBins, fmax(0.0, -log2((double)mp_in)) * kBinsPerOctave + 2.0) : kSmpBins;
      // pairs of bins before which some filter has ended
      const bool open = !(c >= (unsigned long long)k) && !(use_p && m >= p_mass) && b0 + 2 <= min_bin;
      const int pairs = __syncthreads_count(open);
      if (tid == min(pairs, kSmpThreads - 1)) {
        s.found_bin = b0 + 1;
        s.found_cnt = (int)c;
      }
    }
    cl.sync();
    const int last_bin = lead->found_bin, cnt = lead->found_cnt;
    if (cnt <= kSmpSort) {
      const uint32_t lo = smp.first_key(last_bin);
      if (writer) s.above_cnt = 0, s.above_mass = 0;
      smp.gather(value_of(lo), row.top);
      if (rank == 0) {
        uint32_t key;
        unsigned long long q, sum;
        smp.sums(key, q, sum);
        const bool here = tid < s.list_n;
        const double w = here ? row.weight(value_of(key)) : 0.0;
        int m = min(k, s.list_n);
        const int below = __syncthreads_count(here && sum < p_mass);
        if (use_p) m = min(m, below + 1);
        const int likely = __syncthreads_count(here && w >= (double)mp_in);
        if (use_mp) m = min(m, likely);
        m = max(m, 1);
        __syncthreads();
        if (tid == m - 1) s.above_mass = sum;
        __syncthreads();
        const unsigned long long all = s.above_mass;
        const unsigned long long target = (unsigned long long)ceil(u * (double)all);
        const int at = min(__syncthreads_count(here && sum < target), m - 1);
        if (tid == at) {
          a.tokens[b] = (int)~(uint32_t)s.list[at];
          if (a.probs) a.probs[b] = (float)(w * (double)(1ull << a.shift) / (double)all);
          if (a.kept) a.kept[b] = m;
        }
      }
      return;
    }
    cl.sync();
    kept = k;
    if (use_p) kept = min(kept, smp.find(0, p_mass, false).n);
    if (use_mp) {
      int likely = 0;
      for (int i = tid; i < n; i += kSmpThreads)
        likely += xs[i] > -INFINITY && row.weight(xs[i]) >= (double)mp_in;
      const unsigned long long mine = block_sum((unsigned long long)likely, s.red);
      if (tid < size) cl.map_shared_rank(&s, tid)->z[rank] = mine;
      cl.sync();
      unsigned long long all = 0;
      for (int r = 0; r < size; ++r) all += s.z[r];
      cl.sync();
      kept = min(kept, (int)all);
    }
    kept = max(kept, 1);
    norm = smp.find((unsigned long long)kept, 0, false).mass;
  } else {
    smp.histogram();
    if (rank == 0) {
      const unsigned long long z = block_sum(s.all_mass[tid] + s.all_mass[kSmpThreads + tid], s.red);
      if (tid == 0) s.total = z;
    }
    cl.sync();
    norm = lead->total;
  }
  const unsigned long long target = (unsigned long long)ceil(u * (double)norm);
  Place f = smp.find(0, target < norm ? target : norm, true);
  if (f.n > kept) f = smp.find((unsigned long long)kept, 0, true);  // tokens of no weight at the end
  if (writer) {
    a.tokens[b] = f.index;
    const double w = row.weight(value_of(f.key));
    if (a.probs) a.probs[b] = (float)(w * (double)(1ull << a.shift) / (double)norm);
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
  // CTAs per row: as few as hold it, more while there are SMs for them and
  // each still has 4096 tokens
  int cluster = 1;
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
