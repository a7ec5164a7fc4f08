// paged_attn.cu -- attention of new tokens over a paged cache.
//
// With s_i = scale * log2(e) * q . K_i over the keys i that a row sees, the
// running maximum m and sum l of a softmax in base 2 give, tile after tile,
//   m' = max(m, max_i s_i), l' = l 2^(m - m') + sum_i 2^(s_i - m'),
//   o' = o 2^(m - m') + sum_i 2^(s_i - m') V_i;  out = o / l.
// Pieces of the keys join the same way.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <stdint.h>

#include "paged.cuh"
#include "paged_attn.cuh"
#include "tma.cuh"

namespace mcpo {
namespace {

// 16 bytes global -> shared, zeros when !in.
__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool in) {
  const int n = in ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Ends a piece of a block that several CTAs share: true in the CTA that
// finished last, which then adds the pieces.  Block-wide.
__device__ __forceinline__ bool paged_last(const PagedAttnArgs& a, const PagedPiece& p, unsigned* flag_s) {
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    const unsigned t = atomicAdd(&a.tickets[p.first_cta], 1u);
    const bool last = t == (unsigned)p.n_ctas - 1;
    if (last) a.tickets[p.first_cta] = 0u;
    *flag_s = last;
  }
  __syncthreads();
  const bool last = *flag_s != 0;
  if (last) __threadfence();
  __syncthreads();
  return last;
}

// ---------------------------------------------------------------------
// f32: FMAs
// ---------------------------------------------------------------------
constexpr int kSimtRows = 16, kSimtKeys = 32, kSimtThreads = 128;

template <int HD>
struct SimtSmem {
  float q[kSimtRows][HD];
  float k[2][kSimtKeys][HD + 4];
  float v[2][kSimtKeys][HD];
  float p[kSimtRows][kSimtKeys];
};

template <int HD>
__global__ void __launch_bounds__(kSimtThreads) k_paged_attn_f32(const PagedAttnArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  SimtSmem<HD>& s = *reinterpret_cast<SimtSmem<HD>*>(smem_raw);
  __shared__ PagedShared sched;
  __shared__ unsigned last_s;
  constexpr int kCols = HD / 16;  // accumulator columns of a thread, for each of its two rows
  const int tid = threadIdx.x, x = tid & 15, y = tid >> 4;  // rows 2y, 2y + 1
  const int block_tokens = kSimtRows / a.group;
  const float* qg = static_cast<const float*>(a.q);
  const float* kg = static_cast<const float*>(a.kc);
  const float* vg = static_cast<const float*>(a.vc);
  PagedWalk<kSimtKeys> walk(a, &sched, block_tokens, 1);
  PagedPiece p;
  while (walk.next(&p)) {
    const int t0 = p.b * block_tokens, rows = min(block_tokens, p.req.n_new - t0) * a.group;
    const int seen = paged_seen(p.req, p.b, block_tokens);
    auto load = [&](int tile, int st) {
      for (int e = tid; e < kSimtKeys * HD / 4; e += kSimtThreads) {
        const int key = e / (HD / 4), c = e % (HD / 4) * 4, pos = tile * kSimtKeys + key;
        bool in = pos < seen;
        long long at = 0;
        if (in) {
          const int id = a.table[p.r * a.table_stride + (pos >> a.page_shift)];
          in = id >= 0 && id < a.n_pages;
          if (in) at = id * a.page_stride + (pos & ((1 << a.page_shift) - 1)) * a.token_stride + p.h * a.head_stride + c;
        }
        cp_async16(&s.k[st][key][c], kg + at, in);
        cp_async16(&s.v[st][key][c], vg + at, in);
      }
      cp_async_commit();
    };
    load(p.tile0, 0);
    for (int e = tid; e < kSimtRows * HD / 4; e += kSimtThreads) {
      const int row = e / (HD / 4), c = e % (HD / 4) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row < rows)
        v = *reinterpret_cast<const float4*>(qg + (p.req.q0 + t0 + row / a.group) * a.q_stride +
                                             (long long)(p.h * a.group + row % a.group) * HD + c);
      *reinterpret_cast<float4*>(&s.q[row][c]) = v;
    }
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, acc[2][kCols];
    int see[2];  // keys that each row sees
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = 2 * y + i;
      see[i] = row < rows ? max(0, p.req.len - p.req.n_new + t0 + row / a.group + 1) : 0;
#pragma unroll
      for (int c = 0; c < kCols; ++c) acc[i][c] = 0.f;
    }
    for (int tile = p.tile0; tile < p.tile1; ++tile) {
      const int st = (tile - p.tile0) & 1, key0 = tile * kSimtKeys;
      if (tile + 1 < p.tile1) {
        load(tile + 1, st ^ 1);
        cp_async_wait<1>();
      } else {
        cp_async_wait<0>();
      }
      __syncthreads();
      float sc[2][2] = {};
#pragma unroll 4
      for (int d = 0; d < HD; d += 4) {
        const float4 q0 = *reinterpret_cast<const float4*>(&s.q[2 * y][d]);
        const float4 q1 = *reinterpret_cast<const float4*>(&s.q[2 * y + 1][d]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float4 k4 = *reinterpret_cast<const float4*>(&s.k[st][x + 16 * j][d]);
          sc[0][j] = fmaf(q0.x, k4.x, fmaf(q0.y, k4.y, fmaf(q0.z, k4.z, fmaf(q0.w, k4.w, sc[0][j]))));
          sc[1][j] = fmaf(q1.x, k4.x, fmaf(q1.y, k4.y, fmaf(q1.z, k4.z, fmaf(q1.w, k4.w, sc[1][j]))));
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          sc[i][j] = key0 + x + 16 * j < see[i] ? sc[i][j] * a.scale_log2 : -INFINITY;
          mx = fmaxf(mx, sc[i][j]);
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float mn = fmaxf(m[i], mx), base = mn == -INFINITY ? 0.f : mn;
        const float corr = exp2f(m[i] - base);
        m[i] = mn;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float w = exp2f(sc[i][j] - base);
          sum += w;
          s.p[2 * y + i][x + 16 * j] = w;
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        l[i] = l[i] * corr + sum;
#pragma unroll
        for (int c = 0; c < kCols; ++c) acc[i][c] *= corr;
      }
      __syncwarp();
      const bool all = key0 + kSimtKeys <= see[0] && key0 + kSimtKeys <= see[1];
#pragma unroll 4
      for (int key = 0; key < kSimtKeys; ++key) {
        float w0 = s.p[2 * y][key], w1 = s.p[2 * y + 1][key];
        // a key that a row does not see adds nothing, whatever V holds there
        const bool on0 = all || key0 + key < see[0], on1 = all || key0 + key < see[1];
#pragma unroll
        for (int c = 0; c < kCols; c += 4) {
          const float4 v4 = *reinterpret_cast<const float4*>(&s.v[st][key][x * 4 + c * 16]);
          if (on0) {
            acc[0][c] = fmaf(w0, v4.x, acc[0][c]);
            acc[0][c + 1] = fmaf(w0, v4.y, acc[0][c + 1]);
            acc[0][c + 2] = fmaf(w0, v4.z, acc[0][c + 2]);
            acc[0][c + 3] = fmaf(w0, v4.w, acc[0][c + 3]);
          }
          if (on1) {
            acc[1][c] = fmaf(w1, v4.x, acc[1][c]);
            acc[1][c + 1] = fmaf(w1, v4.y, acc[1][c + 1]);
            acc[1][c + 2] = fmaf(w1, v4.z, acc[1][c + 2]);
            acc[1][c + 3] = fmaf(w1, v4.w, acc[1][c + 3]);
          }
        }
      }
      __syncthreads();
    }
    bool write = p.n_ctas == 1;
    if (!write) {
      float* part = a.partial + paged_slot(blockIdx.x, p.first_cta) * kSimtRows * (HD + 4);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float* row = part + (2 * y + i) * (HD + 4);
#pragma unroll
        for (int c = 0; c < kCols; c += 4)
          *reinterpret_cast<float4*>(row + 4 + x * 4 + c * 16) =
              make_float4(acc[i][c], acc[i][c + 1], acc[i][c + 2], acc[i][c + 3]);
        if (x == 0) row[0] = m[i], row[1] = l[i];
      }
      if (paged_last(a, p, &last_s)) {
        write = true;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          m[i] = -INFINITY, l[i] = 0.f;
          for (int c = 0; c < p.n_ctas; ++c)
            m[i] = fmaxf(m[i], __ldcg(a.partial + paged_slot(p.first_cta + c, p.first_cta) * kSimtRows * (HD + 4) +
                                      (2 * y + i) * (HD + 4)));
          const float base = m[i] == -INFINITY ? 0.f : m[i];
#pragma unroll
          for (int c = 0; c < kCols; ++c) acc[i][c] = 0.f;
          for (int c = 0; c < p.n_ctas; ++c) {
            const float* row = a.partial + paged_slot(p.first_cta + c, p.first_cta) * kSimtRows * (HD + 4) +
                               (2 * y + i) * (HD + 4);
            const float f = exp2f(__ldcg(row) - base);
            l[i] += __ldcg(row + 1) * f;
#pragma unroll
            for (int cc = 0; cc < kCols; cc += 4) {
              const float4 v4 = __ldcg(reinterpret_cast<const float4*>(row + 4 + x * 4 + cc * 16));
              acc[i][cc] += v4.x * f;
              acc[i][cc + 1] += v4.y * f;
              acc[i][cc + 2] += v4.z * f;
              acc[i][cc + 3] += v4.w * f;
            }
          }
        }
      }
    }
    if (write) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = 2 * y + i;
        if (row >= rows) continue;
        const long long t = p.req.q0 + t0 + row / a.group;
        const int head = p.h * a.group + row % a.group;
        const float inv = see[i] > 0 ? 1.0f / l[i] : 0.f;
        float* o = static_cast<float*>(a.out) + t * a.out_stride + (long long)head * HD;
#pragma unroll
        for (int c = 0; c < kCols; c += 4)
          *reinterpret_cast<float4*>(o + x * 4 + c * 16) =
              see[i] > 0 ? make_float4(acc[i][c] * inv, acc[i][c + 1] * inv, acc[i][c + 2] * inv, acc[i][c + 3] * inv)
                         : make_float4(0.f, 0.f, 0.f, 0.f);
        if (a.lse && x == 0)
          a.lse[t * a.q_heads + head] = see[i] > 0 ? 0.693147180559945309f * (m[i] + log2f(l[i])) : -INFINITY;
      }
    }
    __syncthreads();  // the next piece's loads overwrite the tiles
  }
}

template <typename K>
cudaError_t big_smem(K kernel, size_t bytes) {
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}

cudaError_t sm_count(int* n) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(n, cudaDevAttrMultiProcessorCount, dev);
  return e;
}

template <int HD>
cudaError_t launch_f32(const PagedAttnArgs& a, cudaStream_t st) {
  int sms = 0;
  cudaError_t e = sm_count(&sms);
  if (e == cudaSuccess) e = big_smem(k_paged_attn_f32<HD>, sizeof(SimtSmem<HD>));
  if (e != cudaSuccess) return e;
  const int ctas = HD == 256 ? sms : 2 * sms;  // residents by shared memory
  k_paged_attn_f32<HD><<<ctas < kPagedMaxCtas ? ctas : kPagedMaxCtas, kSimtThreads, sizeof(SimtSmem<HD>), st>>>(a);
  return cudaGetLastError();
}

}  // namespace
}  // namespace mcpo

using namespace mcpo;

extern "C" int minicpmo_gpu_paged_attention(const minicpmo_paged_cache* cache, const void* q, size_t n_tokens,
                                            size_t q_heads, size_t q_stride, const int32_t* block_table,
                                            size_t max_pages, size_t table_stride, const int32_t* lens,
                                            const int32_t* cu_new, size_t n_req, float scale, void* out,
                                            size_t out_stride, float* lse, void* workspace, void* stream, char* error,
                                            size_t error_cap) {
  const char* op = "paged attention";
  if (!paged_cache_ok(cache, op, error, error_cap)) return 0;
  if (n_tokens == 0) return 1;
  if (!q || !block_table || !lens || !cu_new || !out || !workspace)
    return paged_error(error, error_cap, "error: %s: null buffer", op);
  if (n_req < 1 || n_req > MINICPMO_PAGED_MAX_REQUESTS)
    return paged_error(error, error_cap, "error: %s: %zu requests outside 1..%d", op, n_req, MINICPMO_PAGED_MAX_REQUESTS);
  const size_t kv = cache->kv_heads, hd = cache->head_dim, esz = paged_type_bytes(cache->dtype);
  if (q_heads < kv || q_heads % kv || q_heads / kv > kPagedMaxGroup)
    return paged_error(error, error_cap, "error: %s: %zu q heads over %zu kv heads (need a multiple, at most %d each)",
                       op, q_heads, kv, kPagedMaxGroup);
  if (n_tokens > (1u << 24)) return paged_error(error, error_cap, "error: %s: %zu tokens", op, n_tokens);
  if (max_pages < 1 || max_pages > (size_t)INT_MAX / cache->page_size || table_stride < max_pages ||
      table_stride > (1ull << 40))
    return paged_error(error, error_cap, "error: %s: table rows of %zu pages, %zu apart", op, max_pages, table_stride);
  if (q_stride < q_heads * hd || out_stride < q_heads * hd || q_stride > (1ull << 40) || out_stride > (1ull << 40))
    return paged_error(error, error_cap, "error: %s: tokens' rows overlap", op);
  if (!aligned16(q) || !aligned16(out) || q_stride * esz % 16 || out_stride * esz % 16 ||
      (reinterpret_cast<uintptr_t>(workspace) & 255))
    return paged_error(error, error_cap,
                       "error: %s: pointers and strides must be multiples of 16 bytes, the workspace of 256", op);
  if (!(scale > -INFINITY && scale < INFINITY)) return paged_error(error, error_cap, "error: %s: scale is not finite", op);
  if (!paged_on_device(cache->k, op, error, error_cap) || !paged_on_device(workspace, op, error, error_cap)) return 0;
  PagedAttnArgs a{};
  a.q = q;
  a.out = out;
  a.lse = lse;
  a.kc = cache->k;
  a.vc = cache->v;
  a.table = block_table;
  a.lens = lens;
  a.cu = cu_new;
  a.q_stride = (long long)q_stride;
  a.out_stride = (long long)out_stride;
  a.table_stride = (long long)table_stride;
  a.page_stride = (long long)cache->page_stride;
  a.token_stride = (long long)cache->token_stride;
  a.head_stride = (long long)cache->head_stride;
  a.n_tokens = (int)n_tokens;
  a.n_req = (int)n_req;
  a.q_heads = (int)q_heads;
  a.kv_heads = (int)kv;
  a.group = (int)(q_heads / kv);
  a.max_pages = (long long)max_pages;
  a.n_pages = (long long)cache->n_pages;
  a.page_shift = __builtin_ctz(cache->page_size);
  a.scale_log2 = (float)((double)scale * 1.4426950408889634074);
  a.tickets = static_cast<unsigned*>(workspace);
  a.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kPagedMaxCtas * sizeof(unsigned));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaErrorNotSupported;
  if (cache->dtype == kF32)
    e = hd == 64 ? launch_f32<64>(a, st) : hd == 128 ? launch_f32<128>(a, st) : launch_f32<256>(a, st);
  if (e != cudaSuccess) return paged_error(error, error_cap, "error: %s: launch: %s", op, cudaGetErrorString(e));
  return 1;
}
