// paged.cu -- page planning and the K/V append of the paged serving step.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <stdint.h>

#include "gemv.cuh"
#include "paged.cuh"

namespace mcpo {

bool paged_on_device(const void* p, const char* op, char* err, size_t cap) {
  int dev = -1;
  cudaPointerAttributes at{};
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaPointerGetAttributes(&at, p);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    paged_error(err, cap, "error: %s: %s", op, cudaGetErrorString(e));
    return false;
  }
  if (at.type == cudaMemoryTypeManaged) return true;
  if (at.type != cudaMemoryTypeDevice || at.device != dev) {
    paged_error(err, cap, "error: %s: the buffers are not memory of the current device %d", op, dev);
    return false;
  }
  return true;
}

bool paged_cache_ok(const minicpmo_paged_cache* c, const char* op, char* err, size_t cap) {
  if (!c || !c->k || !c->v) return paged_error(err, cap, "error: %s: null cache", op), false;
  const size_t esz = paged_type_bytes(c->dtype);
  if (!esz) return paged_error(err, cap, "error: %s: cache dtype %d is not F32, F16 or BF16", op, c->dtype), false;
  if (c->page_size < 8 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
    return paged_error(err, cap, "error: %s: page_size %u is not a power of two in 8..256", op, c->page_size), false;
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return paged_error(err, cap, "error: %s: head_dim %u is not 64, 128 or 256", op, c->head_dim), false;
  if (c->kv_heads < 1 || c->kv_heads > 1024 || c->n_pages < 1 || c->n_pages > 0x7fffffffull)
    return paged_error(err, cap, "error: %s: %u kv heads, %llu pages", op, c->kv_heads,
                       (unsigned long long)c->n_pages), false;
  const uint64_t hs = c->head_stride, ts = c->token_stride, ps = c->page_stride, lim = 1ull << 40;
  if (hs > lim || ts > lim || ps > lim || ps * esz > (1ull << 62) / c->n_pages)
    return paged_error(err, cap, "error: %s: cache strides out of range", op), false;
  const bool tokens_out = hs >= c->head_dim && ts >= (uint64_t)(c->kv_heads - 1) * hs + c->head_dim &&
                          ps >= (uint64_t)(c->page_size - 1) * ts + (uint64_t)(c->kv_heads - 1) * hs + c->head_dim;
  const bool heads_out = ts >= c->head_dim && hs >= (uint64_t)(c->page_size - 1) * ts + c->head_dim &&
                         ps >= (uint64_t)(c->kv_heads - 1) * hs + (uint64_t)(c->page_size - 1) * ts + c->head_dim;
  if (!tokens_out && !heads_out)
    return paged_error(err, cap, "error: %s: the cache's rows overlap (strides page %llu token %llu head %llu)", op,
                       (unsigned long long)ps, (unsigned long long)ts, (unsigned long long)hs), false;
  if (!aligned16(c->k) || !aligned16(c->v) || hs * esz % 16 || ts * esz % 16 || ps * esz % 16)
    return paged_error(err, cap, "error: %s: cache pointers and strides must be multiples of 16 bytes", op), false;
  return true;
}

namespace {

namespace cg = cooperative_groups;

// ---------------------------------------------------------------------
// plan
// ---------------------------------------------------------------------
// held = ceil(len / ps), need = ceil((len + new) / ps) - held; exclusive
// prefix sums of new tokens, needed pages and released pages over the
// requests place every token and page.  The work is a few bytes per request,
// page and token, so the time is the chain of dependent steps: one launch,
// the requests' loads, a block scan, then independent stores.  Every CTA of
// the one cluster scans all requests itself (no exchange between CTAs); the
// cluster barrier between the last read of lens and ring_state and the first
// write lets the outputs be the inputs' own buffers.  Tokens and pages are
// spread over the cluster flat, each finding its request by binary search in
// the shared prefix sums, so that one long prompt does not wait on one
// thread.  32 requests of one new token take 4.5 us, 512 with 40,000 tokens 9.9;
// a call's time on the host, 22 us with the wrapper's outputs, is above both.
constexpr int kPlanThreads = 1024;
constexpr int kPlanCluster = 8;  // the portable limit

struct PlanArgs {
  const int32_t *lens, *new_lens;
  int n_req;
  int32_t* table;
  long long max_pages, table_stride;
  int32_t* ring;
  long long ring_cap;
  const int64_t* ring_state;
  int page_shift;
  int tokens;
  int32_t* lens_out;
  int64_t* ring_out;
  int32_t *cu_new, *positions;
  int64_t* slots;
  int32_t* status;
};

// Inclusive scan of v over the block; *total gets the block's sum.  Two
// barriers; red has 32 entries.
__device__ __forceinline__ long long block_scan(long long v, long long* red, long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) red[warp] = v;
  __syncthreads();
  if (warp == 0) {
    long long w = red[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += u;
    }
    red[lane] = w;
  }
  __syncthreads();
  *total = red[31];
  return v + (warp ? red[warp - 1] : 0);
}

// The r with pre[r] <= x < pre[r + 1] (pre non-decreasing, pre[0] = 0, x <
// pre[n]).
__device__ __forceinline__ int find_request(const int* pre, int n, int x) {
  int lo = 0, hi = n;  // pre[lo] <= x < pre[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) k_paged_plan(const PlanArgs a) {
  extern __shared__ int plan_smem[];
  __shared__ long long red[3][32];
  __shared__ int flags_s;
  const int n = a.n_req, tid = threadIdx.x;
  int* len_s = plan_smem;          // [n]
  int* cu_s = len_s + n;           // [n + 1] new tokens before request r
  int* need_s = cu_s + n + 1;      // [n + 1] pages taken before it
  int* back_s = need_s + n + 1;    // [n + 1] pages released before it
  const int page = 1 << a.page_shift;
  if (tid == 0) flags_s = 0;
  __syncthreads();

  const long long head = a.ring_state[0], tail = a.ring_state[1];
  const int per = (n + kPlanThreads - 1) / kPlanThreads;
  const int r0 = min(n, tid * per), r1 = min(n, r0 + per);
  long long news = 0, need = 0, back = 0;
  int flags = 0;
  for (int r = r0; r < r1; ++r) {
    const int len = a.lens[r], add = a.new_lens[r];
    len_s[r] = len;
    if (len < 0 || add < -1) {
      flags |= 8;
      continue;
    }
    const long long after = (long long)len + max(add, 0);
    const long long held = ((long long)len + page - 1) >> a.page_shift, want = (after + page - 1) >> a.page_shift;
    if (want > a.max_pages || after > INT_MAX) flags |= 2;
    news += max(add, 0);
    need += want - held;
    if (add < 0) back += held;
  }
  long long all_new, all_need, all_back;
  long long pn = block_scan(news, red[0], &all_new) - news;
  long long pd = block_scan(need, red[1], &all_need) - need;
  long long pb = block_scan(back, red[2], &all_back) - back;
  if (head < 0 || tail < head || tail - head > a.ring_cap || tail - head + all_back > a.ring_cap) flags |= 16;
  if (all_need > tail - head) flags |= 1;
  if (all_new > a.tokens) flags |= 4;
  if (flags) atomicOr(&flags_s, flags);
  __syncthreads();
  flags = flags_s;
  if (!flags) {  // the sums fit 32 bits: tokens and ring_cap do
    for (int r = r0; r < r1; ++r) {
      const int len = len_s[r], add = a.new_lens[r];
      const int held = (int)(((long long)len + page - 1) >> a.page_shift);
      cu_s[r] = (int)pn;
      need_s[r] = (int)pd;
      back_s[r] = (int)pb;
      pn += max(add, 0);
      pd += (((long long)len + max(add, 0) + page - 1) >> a.page_shift) - held;
      if (add < 0) pb += held;
    }
    if (tid == 0) {
      cu_s[n] = (int)all_new;
      need_s[n] = (int)all_need;
      back_s[n] = (int)all_back;
    }
  }
  // every CTA has read lens, new_lens and ring_state before any writes
  cg::this_cluster().sync();

  const int rank = (int)cg::this_cluster().block_rank(), size = (int)cg::this_cluster().num_blocks();
  const int t0 = rank * kPlanThreads + tid, step = size * kPlanThreads;
  if (t0 == 0) {
    a.ring_out[0] = flags ? head : head + all_need;
    a.ring_out[1] = flags ? tail : tail + all_back;
    a.status[0] = flags;
    const long long left = flags ? tail - head : tail + all_back - head - all_need;
    a.status[1] = (int)(left < 0 ? 0 : left > INT_MAX ? INT_MAX : left);
  }
  if (flags) {
    for (int r = t0; r <= n; r += step) {
      a.cu_new[r] = 0;
      if (r < n) a.lens_out[r] = len_s[r];
    }
    for (int t = t0; t < a.tokens; t += step) {
      a.positions[t] = 0;
      a.slots[t] = -1;
    }
    return;
  }
  const long long h0 = head % a.ring_cap, e0 = tail % a.ring_cap;
  for (int r = t0; r <= n; r += step) {
    a.cu_new[r] = cu_s[r];
    if (r < n) {
      // a finished request released its pages (all of len's) or had none;
      // new_lens is an input of its own, so it can still be read
      a.lens_out[r] = a.new_lens[r] < 0 ? 0 : len_s[r] + cu_s[r + 1] - cu_s[r];
    }
  }
  for (int p = t0; p < (int)all_need; p += step) {
    const int r = find_request(need_s, n, p);
    const long long held = ((long long)len_s[r] + page - 1) >> a.page_shift;
    long long at = h0 + p;
    if (at >= a.ring_cap) at -= a.ring_cap;
    a.table[r * a.table_stride + held + (p - need_s[r])] = a.ring[at];
  }
  for (int p = t0; p < (int)all_back; p += step) {
    const int r = find_request(back_s, n, p);
    long long at = e0 + p;
    if (at >= a.ring_cap) at -= a.ring_cap;
    a.ring[at] = a.table[r * a.table_stride + (p - back_s[r])];
  }
  for (int t = t0; t < a.tokens; t += step) {
    if (t >= (int)all_new) {
      a.positions[t] = 0;
      a.slots[t] = -1;
      continue;
    }
    const int r = find_request(cu_s, n, t);
    const int pos = len_s[r] + t - cu_s[r];
    const long long held = ((long long)len_s[r] + page - 1) >> a.page_shift, j = pos >> a.page_shift;
    int id;
    if (j < held) {
      id = a.table[r * a.table_stride + j];
    } else {  // a page taken in this call: from the ring, which it is not written to here
      long long at = h0 + need_s[r] + (j - held);
      if (at >= a.ring_cap) at -= a.ring_cap;
      id = a.ring[at];
    }
    a.positions[t] = pos;
    a.slots[t] = id < 0 ? -1 : ((long long)id << a.page_shift) + (pos & (page - 1));
  }
}

// ---------------------------------------------------------------------
// append
// ---------------------------------------------------------------------
// A row of head_dim values is held by head_dim / 8 lanes, 4 values of the
// first half and the 4 they rotate with in each, so that loads and stores
// are 8 or 16 bytes per lane and the rotation needs no exchange; the sum of
// squares is a butterfly over those lanes.  HBM-bound: every value is read
// and written once, the inputs with loads that do not stay in the caches.  A
// group of lanes takes two rows of one token, with the token's table values
// loaded once for them: more rows cost occupancy and the smallest calls.  At
// 8192 tokens of 32 + 2 x 8 heads of 128, f32 into bf16, and at 32 tokens into
// f16: 58.9 and 2.75 us, 5.2 TB/s of the values and tables for the former; 4
// rows 58.0 and 3.6 us, CTAs of 256 threads 68.9 and 2.75; loads that stay in
// the caches, at 4 rows, 64.8 us.
constexpr int kAppendRows = 2;
constexpr int kAppendThreads = 128;

struct AppendArgs {
  const void *q, *k, *v;
  int n_tokens, q_heads, kv_heads;
  long long q_stride, k_stride, v_stride;
  const float *q_norm, *k_norm;
  float eps;
  const float *rope_cos, *rope_sin;
  int rope_context;
  const int32_t* positions;
  const int64_t* slots;
  void* q_out;
  long long q_out_stride;
  void *kc, *vc;
  long long n_slots, page_stride, token_stride, head_stride;
  int page_shift;
  int32_t* status;
};

template <typename T>
__device__ __forceinline__ float4 load4(const T* p);
template <>
__device__ __forceinline__ float4 load4<float>(const float* p) {
  return __ldcs(reinterpret_cast<const float4*>(p));
}
template <>
__device__ __forceinline__ float4 load4<__half>(const __half* p) {
  const uint2 u = __ldcs(reinterpret_cast<const uint2*>(p));
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
template <>
__device__ __forceinline__ float4 load4<__nv_bfloat16>(const __nv_bfloat16* p) {
  const uint2 u = __ldcs(reinterpret_cast<const uint2*>(p));
  return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                     __uint_as_float(u.y & 0xffff0000u));
}

template <typename T>
__device__ __forceinline__ void store4(T* p, float4 x);
template <>
__device__ __forceinline__ void store4<float>(float* p, float4 x) {
  *reinterpret_cast<float4*>(p) = x;
}
template <>
__device__ __forceinline__ void store4<__half>(__half* p, float4 x) {
  __half2 a = __floats2half2_rn(x.x, x.y), b = __floats2half2_rn(x.z, x.w);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
}
template <>
__device__ __forceinline__ void store4<__nv_bfloat16>(__nv_bfloat16* p, float4 x) {
  __nv_bfloat162 a = __floats2bfloat162_rn(x.x, x.y), b = __floats2bfloat162_rn(x.z, x.w);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
}

template <typename TI, typename TC, int HD>
__global__ void __launch_bounds__(kAppendThreads) k_paged_append(const AppendArgs a) {
  constexpr int kLanes = HD / 8;  // lanes of a row
  const int group = (int)((blockIdx.x * kAppendThreads + threadIdx.x) / kLanes), l = threadIdx.x % kLanes;
  const int rows = a.q_heads + 2 * a.kv_heads;
  const int chunks = (rows + kAppendRows - 1) / kAppendRows;
  // groups of one warp may be past the end: they take part in the shuffles
  const bool in = group < a.n_tokens * chunks;
  const int t = in ? group / chunks : 0, row0 = in ? (group % chunks) * kAppendRows : 0;
  const long long slot = in ? a.slots[t] : -1;
  const int pos = in ? a.positions[t] : 0;
  bool live = slot >= 0;
  if (live && (slot >= a.n_slots || pos < 0 || pos >= a.rope_context)) {
    live = false;
    if (a.status && row0 == 0 && l == 0) atomicOr(a.status, slot >= a.n_slots ? 2 : 1);
  }
  const int d0 = 4 * l, d1 = HD / 2 + 4 * l;
  float4 x[kAppendRows], y[kAppendRows], c = {}, s = {};
#pragma unroll
  for (int i = 0; i < kAppendRows; ++i) {
    const int row = row0 + i;
    x[i] = y[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live && row < rows) {
      const TI* p;
      if (row < a.q_heads) p = static_cast<const TI*>(a.q) + t * a.q_stride + (long long)row * HD;
      else if (row < a.q_heads + a.kv_heads) p = static_cast<const TI*>(a.k) + t * a.k_stride + (long long)(row - a.q_heads) * HD;
      else p = static_cast<const TI*>(a.v) + t * a.v_stride + (long long)(row - a.q_heads - a.kv_heads) * HD;
      x[i] = load4(p + d0);
      y[i] = load4(p + d1);
    }
  }
  if (live) {
    c = *reinterpret_cast<const float4*>(a.rope_cos + (long long)pos * (HD / 2) + d0);
    s = *reinterpret_cast<const float4*>(a.rope_sin + (long long)pos * (HD / 2) + d0);
  }
  const long long page = slot >> a.page_shift, off = slot & ((1ll << a.page_shift) - 1);
#pragma unroll
  for (int i = 0; i < kAppendRows; ++i) {
    const int row = row0 + i;
    const bool is_q = row < a.q_heads, is_v = row >= a.q_heads + a.kv_heads;
    const float* w = is_q ? a.q_norm : a.k_norm;
    float ss = x[i].x * x[i].x + x[i].y * x[i].y + x[i].z * x[i].z + x[i].w * x[i].w;
    ss += y[i].x * y[i].x + y[i].y * y[i].y + y[i].z * y[i].z + y[i].w * y[i].w;
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (!live || row >= rows) continue;
    if (is_v) {
      TC* dst = static_cast<TC*>(a.vc) + page * a.page_stride + off * a.token_stride +
                (long long)(row - a.q_heads - a.kv_heads) * a.head_stride;
      store4(dst + d0, x[i]);
      store4(dst + d1, y[i]);
      continue;
    }
    if (w) {
      const float inv = 1.0f / sqrtf(ss / (float)HD + a.eps);
      const float4 w0 = *reinterpret_cast<const float4*>(w + d0), w1 = *reinterpret_cast<const float4*>(w + d1);
      x[i] = make_float4(x[i].x * inv * w0.x, x[i].y * inv * w0.y, x[i].z * inv * w0.z, x[i].w * inv * w0.w);
      y[i] = make_float4(y[i].x * inv * w1.x, y[i].y * inv * w1.y, y[i].z * inv * w1.z, y[i].w * inv * w1.w);
    }
    const float4 u = make_float4(x[i].x * c.x - y[i].x * s.x, x[i].y * c.y - y[i].y * s.y, x[i].z * c.z - y[i].z * s.z,
                                 x[i].w * c.w - y[i].w * s.w);
    const float4 z = make_float4(y[i].x * c.x + x[i].x * s.x, y[i].y * c.y + x[i].y * s.y, y[i].z * c.z + x[i].z * s.z,
                                 y[i].w * c.w + x[i].w * s.w);
    TC* dst = is_q ? static_cast<TC*>(a.q_out) + t * a.q_out_stride + (long long)row * HD
                   : static_cast<TC*>(a.kc) + page * a.page_stride + off * a.token_stride +
                         (long long)(row - a.q_heads) * a.head_stride;
    store4(dst + d0, u);
    store4(dst + d1, z);
  }
}

template <typename TI, typename TC>
cudaError_t append_hd(const AppendArgs& a, int hd, cudaStream_t st) {
  const int rows = a.q_heads + 2 * a.kv_heads, chunks = (rows + kAppendRows - 1) / kAppendRows;
  const long long threads = (long long)a.n_tokens * chunks * (hd / 8);
  const unsigned grid = (unsigned)((threads + kAppendThreads - 1) / kAppendThreads);
  switch (hd) {
    case 64: k_paged_append<TI, TC, 64><<<grid, kAppendThreads, 0, st>>>(a); break;
    case 128: k_paged_append<TI, TC, 128><<<grid, kAppendThreads, 0, st>>>(a); break;
    default: k_paged_append<TI, TC, 256><<<grid, kAppendThreads, 0, st>>>(a); break;
  }
  return cudaGetLastError();
}

template <typename TI>
cudaError_t append_cache(const AppendArgs& a, int hd, int dtype, cudaStream_t st) {
  if (dtype == kF32) return append_hd<TI, float>(a, hd, st);
  if (dtype == kF16) return append_hd<TI, __half>(a, hd, st);
  return append_hd<TI, __nv_bfloat16>(a, hd, st);
}

}  // namespace
}  // namespace mcpo

using namespace mcpo;

extern "C" {

int minicpmo_gpu_paged_plan(const int32_t* lens, const int32_t* new_lens, size_t n_req, int32_t* block_table,
                            size_t max_pages, size_t table_stride, int32_t* free_ring, size_t ring_capacity,
                            const int64_t* ring_state, size_t page_size, size_t token_capacity, int32_t* lens_out,
                            int64_t* ring_state_out, int32_t* cu_new, int32_t* positions, int64_t* slots,
                            int32_t* status, void* stream, char* error, size_t error_cap) {
  const char* op = "paged plan";
  if (!lens || !new_lens || !block_table || !free_ring || !ring_state || !lens_out || !ring_state_out || !cu_new ||
      !status || (token_capacity && (!positions || !slots)))
    return paged_error(error, error_cap, "error: %s: null buffer", op);
  if (n_req < 1 || n_req > MINICPMO_PAGED_MAX_REQUESTS)
    return paged_error(error, error_cap, "error: %s: %zu requests outside 1..%d", op, n_req, MINICPMO_PAGED_MAX_REQUESTS);
  if (page_size < 8 || page_size > 256 || (page_size & (page_size - 1)))
    return paged_error(error, error_cap, "error: %s: page_size %zu is not a power of two in 8..256", op, page_size);
  if (max_pages < 1 || max_pages > (size_t)INT_MAX || table_stride < max_pages || table_stride > (1ull << 40))
    return paged_error(error, error_cap, "error: %s: table rows of %zu pages, %zu apart", op, max_pages, table_stride);
  if (ring_capacity < 1 || ring_capacity > (size_t)INT_MAX / 2)
    return paged_error(error, error_cap, "error: %s: ring capacity %zu", op, ring_capacity);
  if (token_capacity > (size_t)INT_MAX / 2)
    return paged_error(error, error_cap, "error: %s: token capacity %zu", op, token_capacity);
  if (cu_new == lens || cu_new == new_lens || lens_out == new_lens)
    return paged_error(error, error_cap, "error: %s: only lens_out and ring_state_out may be inputs' buffers", op);
  if (!paged_on_device(lens, op, error, error_cap)) return 0;
  PlanArgs a{};
  a.lens = lens;
  a.new_lens = new_lens;
  a.n_req = (int)n_req;
  a.table = block_table;
  a.max_pages = (long long)max_pages;
  a.table_stride = (long long)table_stride;
  a.ring = free_ring;
  a.ring_cap = (long long)ring_capacity;
  a.ring_state = ring_state;
  a.page_shift = __builtin_ctzll(page_size);
  a.tokens = (int)token_capacity;
  a.lens_out = lens_out;
  a.ring_out = ring_state_out;
  a.cu_new = cu_new;
  a.positions = positions;
  a.slots = slots;
  a.status = status;
  const size_t smem = (4 * n_req + 3) * sizeof(int);
  static_assert((4 * MINICPMO_PAGED_MAX_REQUESTS + 3) * sizeof(int) <= 160 * 1024, "plan prefix sums fit shared memory");
  static OncePerDevice once;
  cudaError_t e = once([] {
    return cudaFuncSetAttribute(k_paged_plan, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
  });
  if (e == cudaSuccess) {
    // one CTA does a decode step; a cluster where tokens or requests give each CTA a turn of work
    const size_t most = token_capacity > n_req ? token_capacity : n_req;
    size_t ctas = 1;
    while (ctas < kPlanCluster && ctas * kPlanThreads < most) ctas *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kPlanThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctas > 1 ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, k_paged_plan, a);
  }
  if (e != cudaSuccess) return paged_error(error, error_cap, "error: %s: launch: %s", op, cudaGetErrorString(e));
  return 1;
}

int minicpmo_gpu_paged_append(const minicpmo_paged_cache* cache, const void* q, const void* k, const void* v,
                              int in_dtype, size_t n_tokens, size_t q_heads, size_t q_stride, size_t k_stride,
                              size_t v_stride, const float* q_norm, const float* k_norm, float eps,
                              const float* rope_cos, const float* rope_sin, size_t rope_context,
                              const int32_t* positions, const int64_t* slots, void* q_out, size_t q_out_stride,
                              int32_t* status, void* stream, char* error, size_t error_cap) {
  const char* op = "paged append";
  if (!paged_cache_ok(cache, op, error, error_cap)) return 0;
  const size_t hd = cache->head_dim, isz = paged_type_bytes(in_dtype), csz = paged_type_bytes(cache->dtype);
  if (!isz) return paged_error(error, error_cap, "error: %s: input dtype %d is not F32, F16 or BF16", op, in_dtype);
  if (n_tokens == 0) return 1;
  if (!k || !v || !positions || !slots || !rope_cos || !rope_sin || (q_heads && (!q || !q_out)))
    return paged_error(error, error_cap, "error: %s: null buffer", op);
  if (q_heads > 8192 || n_tokens > (1u << 24) || rope_context < 1 || rope_context > (size_t)INT_MAX)
    return paged_error(error, error_cap, "error: %s: %zu tokens, %zu q heads, %zu table rows", op, n_tokens, q_heads,
                       rope_context);
  // the grid counts threads in 31 bits
  if (n_tokens * ((q_heads + 2 * (size_t)cache->kv_heads) / kAppendRows + 1) * (hd / 8) > (1ull << 31) - kAppendThreads)
    return paged_error(error, error_cap, "error: %s: too many rows in one call", op);
  if (k_stride < cache->kv_heads * hd || v_stride < cache->kv_heads * hd ||
      (q_heads && (q_stride < q_heads * hd || q_out_stride < q_heads * hd)))
    return paged_error(error, error_cap, "error: %s: tokens' rows overlap", op);
  if (!aligned16(k) || !aligned16(v) || k_stride * isz % 16 || v_stride * isz % 16 || !aligned16(rope_cos) ||
      !aligned16(rope_sin) || (q_norm && !aligned16(q_norm)) || (k_norm && !aligned16(k_norm)) ||
      (q_heads && (!aligned16(q) || !aligned16(q_out) || q_stride * isz % 16 || q_out_stride * csz % 16)))
    return paged_error(error, error_cap, "error: %s: pointers and strides must be multiples of 16 bytes", op);
  if (!paged_on_device(cache->k, op, error, error_cap)) return 0;
  AppendArgs a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.n_tokens = (int)n_tokens;
  a.q_heads = (int)q_heads;
  a.kv_heads = (int)cache->kv_heads;
  a.q_stride = (long long)q_stride;
  a.k_stride = (long long)k_stride;
  a.v_stride = (long long)v_stride;
  a.q_norm = q_norm;
  a.k_norm = k_norm;
  a.eps = eps;
  a.rope_cos = rope_cos;
  a.rope_sin = rope_sin;
  a.rope_context = (int)rope_context;
  a.positions = positions;
  a.slots = slots;
  a.q_out = q_out;
  a.q_out_stride = (long long)q_out_stride;
  a.kc = cache->k;
  a.vc = cache->v;
  a.page_shift = __builtin_ctz(cache->page_size);
  a.n_slots = (long long)cache->n_pages << a.page_shift;
  a.page_stride = (long long)cache->page_stride;
  a.token_stride = (long long)cache->token_stride;
  a.head_stride = (long long)cache->head_stride;
  a.status = status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = in_dtype == kF32   ? append_cache<float>(a, (int)hd, cache->dtype, st)
                  : in_dtype == kF16 ? append_cache<__half>(a, (int)hd, cache->dtype, st)
                                     : append_cache<__nv_bfloat16>(a, (int)hd, cache->dtype, st);
  if (e != cudaSuccess) return paged_error(error, error_cap, "error: %s: launch: %s", op, cudaGetErrorString(e));
  return 1;
}

}  // extern "C"
