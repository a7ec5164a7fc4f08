// paged_attn.cu -- attention of new tokens over a paged cache.
//
// With s_i = scale * log2(e) * q . K_i over the keys i that a row sees, the
// running maximum m and sum l of a softmax in base 2 give, tile after tile,
//   m' = max(m, max_i s_i), l' = l 2^(m - m') + sum_i 2^(s_i - m'),
//   o' = o 2^(m - m') + sum_i 2^(s_i - m') V_i;  out = o / l.
// Pieces of the keys join the same way.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <stdint.h>

#include "paged.cuh"
#include "paged_attn.cuh"
#include "paged_attn_tc.cuh"
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
// f32 products keep f32's accuracy on the FMA units; split into tf32 or bf16
// parts for the matrix units they took longer (three m16n8k8 tf32 products per
// step: 126 us where this takes less than half).  What bounds an FMA kernel is
// shared-memory reads, so threads take 4 x 4 tiles: for the scores a warp has
// all 16 rows x 32 keys over a quarter of head_dim (8 reads of 16 bytes per 64
// FMAs; the four warps' sums are added on the way to the softmax), for the
// output all rows x a quarter of the columns (2 reads per 16 FMAs).  Rows and
// keys are dealt out so that a warp's reads meet all banks.  Five requests of up
// to 33 new tokens behind up to 1000 (16 heads, 8 K/V heads of 128): 60 us.
constexpr int kSimtRows = 16, kSimtKeys = 32, kSimtThreads = 128;

template <int HD>
struct SimtSmem {
  float q[kSimtRows][HD + 4];
  float k[2][kSimtKeys][HD + 4];
  float v[2][kSimtKeys][HD];
  float part[4][kSimtRows][kSimtKeys + 8];  // scores over a warp's part of head_dim
  float p[kSimtRows][kSimtKeys + 4];
  float corr[kSimtRows], m[kSimtRows], l[kSimtRows];
};
template <int HD>
constexpr int kSimtCtas = HD == 64 ? 4 : HD == 128 ? 2 : 1;  // per SM, by shared memory

template <int HD>
__global__ void __launch_bounds__(kSimtThreads, kSimtCtas<HD>) k_paged_attn_f32(const PagedAttnArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  SimtSmem<HD>& s = *reinterpret_cast<SimtSmem<HD>*>(smem_raw);
  __shared__ PagedShared sched;
  __shared__ unsigned last_s;
  constexpr int kC = HD / 32;  // output columns of a thread, for each of its four rows
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rg = lane >> 3, kl = lane & 7;
  const int col = warp * (HD / 4) + kl * kC;  // rows 4 i + rg, i < 4
  const int srow = tid >> 3, skey = (tid & 7) * 4;  // in the softmax: a row, four keys
  const int block_tokens = kSimtRows / a.group;
  const float* qg = static_cast<const float*>(a.q);
  const float* kg = static_cast<const float*>(a.kc);
  const float* vg = static_cast<const float*>(a.vc);
  PagedWalk<kSimtKeys> walk;
  walk.start(a, &sched, block_tokens, 0, 3, 0.f);  // a unit takes long next to a join here: 1 instead of 0 made 16,000 keys 40% slower
  PagedPiece p;
  while (walk.next(a, &p)) {
    const int t0 = p.b * block_tokens, rows = min(block_tokens, p.req.n_new - t0) * a.group;
    const int seen = paged_seen(p.req, p.b, block_tokens);
    const int32_t* table = a.table + p.r * a.table_stride;
    auto page = [&](int tile) {  // of this warp's 8 keys of a tile
      const int pos = tile * kSimtKeys + warp * 8;
      return tile < p.tile1 && pos < seen ? table[pos >> a.page_shift] : -1;
    };
    auto load = [&](int tile, int st, int id) {
      const bool there = id >= 0 && id < a.n_pages;
      const long long base = there ? id * a.page_stride + p.h * a.head_stride : 0;
#pragma unroll
      for (int j = 0; j < HD / 16; ++j) {
        const int e = lane + 32 * j, key = warp * 8 + e / (HD / 4), c = e % (HD / 4) * 4, pos = tile * kSimtKeys + key;
        const bool in = there && pos < seen;
        const long long at = in ? base + (pos & ((1 << a.page_shift) - 1)) * a.token_stride + c : 0;
        cp_async16(&s.k[st][key][c], kg + at, in);
        cp_async16(&s.v[st][key][c], vg + at, in);
      }
      cp_async_commit();
    };
    load(p.tile0, 0, page(p.tile0));
    int next_page = page(p.tile0 + 1);
    for (int e = tid; e < kSimtRows * HD / 4; e += kSimtThreads) {
      const int row = e / (HD / 4), c = e % (HD / 4) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row < rows)
        v = *reinterpret_cast<const float4*>(qg + (p.req.q0 + t0 + row / a.group) * a.q_stride +
                                             (long long)(p.h * a.group + row % a.group) * HD + c);
      *reinterpret_cast<float4*>(&s.q[row][c]) = v;
    }
    // keys that a row sees (rows without a token: all, so that they mask nothing)
    auto sees = [&](int row) {
      return row < rows ? max(0, p.req.len - p.req.n_new + t0 + row / a.group + 1) : INT_MAX;
    };
    const int see_s = sees(srow), see_all = max(0, p.req.len - p.req.n_new + t0 + 1);
    const int see[4] = {sees(rg), sees(4 + rg), sees(8 + rg), sees(12 + rg)};
    float m = -INFINITY, l = 0.f, acc[4][kC];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < kC; ++c) acc[i][c] = 0.f;
    for (int tile = p.tile0; tile < p.tile1; ++tile) {
      const int st = (tile - p.tile0) & 1, key0 = tile * kSimtKeys;
      cp_async_wait<0>();
      __syncthreads();  // this tile is there, and everyone is done with the last one
      if (tile + 1 < p.tile1) {
        load(tile + 1, st ^ 1, next_page);
        next_page = page(tile + 2);
      }
      float sc[4][4] = {};
#pragma unroll 2
      for (int d = warp * (HD / 4); d < (warp + 1) * (HD / 4); d += 4) {
        float4 q4[4], k4[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          q4[i] = *reinterpret_cast<const float4*>(&s.q[4 * i + rg][d]);
          k4[i] = *reinterpret_cast<const float4*>(&s.k[st][8 * i + kl][d]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) sc[i][j] = fmaf(q4[i].x, k4[j].x, sc[i][j]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) sc[i][j] = fmaf(q4[i].y, k4[j].y, sc[i][j]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) sc[i][j] = fmaf(q4[i].z, k4[j].z, sc[i][j]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) sc[i][j] = fmaf(q4[i].w, k4[j].w, sc[i][j]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s.part[warp][4 * i + rg][8 * j + kl] = sc[i][j];
      __syncthreads();
      {
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float4 y = *reinterpret_cast<const float4*>(&s.part[w][srow][skey]);
          x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
        }
        const int left = see_s - key0 - skey;  // of the four keys, those that the row sees
        x.x = left > 0 ? x.x * a.scale_log2 : -INFINITY;
        x.y = left > 1 ? x.y * a.scale_log2 : -INFINITY;
        x.z = left > 2 ? x.z * a.scale_log2 : -INFINITY;
        x.w = left > 3 ? x.w * a.scale_log2 : -INFINITY;
        float mx = fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w));
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float mn = fmaxf(m, mx), base = mn == -INFINITY ? 0.f : mn, corr = exp2f(m - base);
        m = mn;
        x = make_float4(exp2f(x.x - base), exp2f(x.y - base), exp2f(x.z - base), exp2f(x.w - base));
        float sum = (x.x + x.y) + (x.z + x.w);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        l = l * corr + sum;
        *reinterpret_cast<float4*>(&s.p[srow][skey]) = x;
        if ((tid & 7) == 0) s.corr[srow] = corr;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f = s.corr[4 * i + rg];
#pragma unroll
        for (int c = 0; c < kC; ++c) acc[i][c] *= f;
      }
      auto value = [&](int key, float (&v)[kC]) {
        const float* at = &s.v[st][key][col];
        if constexpr (kC == 2) {
          const float2 x = *reinterpret_cast<const float2*>(at);
          v[0] = x.x, v[1] = x.y;
        } else {
#pragma unroll
          for (int c = 0; c < kC; c += 4) {
            const float4 x = *reinterpret_cast<const float4*>(at + c);
            v[c] = x.x, v[c + 1] = x.y, v[c + 2] = x.z, v[c + 3] = x.w;
          }
        }
      };
      if (key0 + kSimtKeys <= see_all) {
#pragma unroll 2
        for (int key = 0; key < kSimtKeys; key += 4) {
          float4 w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const float4*>(&s.p[4 * i + rg][key]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float v[kC];
            value(key + j, v);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float x = j == 0 ? w[i].x : j == 1 ? w[i].y : j == 2 ? w[i].z : w[i].w;
#pragma unroll
              for (int c = 0; c < kC; ++c) acc[i][c] = fmaf(x, v[c], acc[i][c]);
            }
          }
        }
      } else {
        // a key that a row does not see adds nothing, whatever V holds there
#pragma unroll 4
        for (int key = 0; key < kSimtKeys; ++key) {
          float v[kC];
          value(key, v);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = s.p[4 * i + rg][key];
            const bool on = key0 + key < see[i];
#pragma unroll
            for (int c = 0; c < kC; ++c) acc[i][c] = on ? fmaf(x, v[c], acc[i][c]) : acc[i][c];
          }
        }
      }
    }
    if ((tid & 7) == 0) s.m[srow] = m, s.l[srow] = l;
    __syncthreads();
    float rm[4], rl[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) rm[i] = s.m[4 * i + rg], rl[i] = s.l[4 * i + rg];
    bool write = p.n_ctas == 1;
    constexpr int kLd = HD + 4;
    if (!write) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float* row = a.partial + (paged_slot(blockIdx.x, p.first_cta) * kSimtRows + 4 * i + rg) * kLd;
#pragma unroll
        for (int c = 0; c < kC; c += 2) *reinterpret_cast<float2*>(row + 4 + col + c) = make_float2(acc[i][c], acc[i][c + 1]);
        if (warp == 0 && kl == 0) *reinterpret_cast<float2*>(row) = make_float2(rm[i], rl[i]);
      }
      if (paged_last(a, p, &last_s)) {
        write = true;
        const float* row0 = a.partial + rg * kLd;
        auto at = [&](int k, int i) {
          return row0 + (paged_slot(p.first_cta + k, p.first_cta) * kSimtRows + 4 * i) * kLd;
        };
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          rm[i] = -INFINITY, rl[i] = 0.f;
#pragma unroll
          for (int c = 0; c < kC; ++c) acc[i][c] = 0.f;
        }
#pragma unroll 4
        for (int k = 0; k < p.n_ctas; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) rm[i] = fmaxf(rm[i], __ldcg(at(k, i)));
#pragma unroll 2
        for (int k = 0; k < p.n_ctas; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(at(k, i)));
            const float f = exp2f(ml.x - (rm[i] == -INFINITY ? 0.f : rm[i]));
            rl[i] += ml.y * f;
#pragma unroll
            for (int c = 0; c < kC; c += 2) {
              const float2 v = __ldcg(reinterpret_cast<const float2*>(at(k, i) + 4 + col + c));
              acc[i][c] += v.x * f, acc[i][c + 1] += v.y * f;
            }
          }
      }
    }
    if (write) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 4 * i + rg;
        if (row >= rows) continue;
        const long long t = p.req.q0 + t0 + row / a.group;
        const int head = p.h * a.group + row % a.group;
        const bool any = see[i] > 0;
        const float inv = any ? 1.0f / rl[i] : 0.f;
        float* o = static_cast<float*>(a.out) + t * a.out_stride + (long long)head * HD + col;
#pragma unroll
        for (int c = 0; c < kC; c += 2)
          *reinterpret_cast<float2*>(o + c) = any ? make_float2(acc[i][c] * inv, acc[i][c + 1] * inv) : make_float2(0.f, 0.f);
        if (a.lse && warp == 0 && kl == 0)
          a.lse[t * a.q_heads + head] = any ? 0.693147180559945309f * (rm[i] + log2f(rl[i])) : -INFINITY;
      }
    }
    __syncthreads();  // the next piece's loads overwrite the tiles
  }
}

// ---------------------------------------------------------------------
// f16, bf16: few rows per request (decode, speculated tokens)
// ---------------------------------------------------------------------
// HBM-bound: K and V of a request are read once for the up to 16 rows (tokens
// x q heads of the group) of a block, and 16 rows are one m16n8k16 tile, so
// the legacy matrix instructions are far from their limit.  Each of the four
// warps takes 16 of a tile's 64 keys with its own ring of cp.async stages, its
// own maximum, sum and accumulator: nothing in the key loop waits on another
// warp; the four join once per piece.  16 keys lie in one page (two for pages
// of 8), so one table entry, fetched a tile ahead, addresses a warp's rows.
// 32 sequences of up to 4096 positions (8 K/V heads of 128, f16) take 64 us,
// 5.1 TB/s of K and V; 96 of 8000 reach 6.2.
constexpr int kMmaRows = 16, kMmaWarps = 4, kMmaKeys = 16, kMmaTile = kMmaWarps * kMmaKeys, kMmaThreads = kMmaWarps * 32;

template <int HD>
struct MmaCfg {
  // Three CTAs of two stages hide a piece's beginning and end better than two
  // of three: 64.8 against 67.8 us for 32 sequences of up to 4096 positions.
  static constexpr int kStages = HD == 64 ? 4 : HD == 128 ? 2 : 3;
  static constexpr int kTileBytes = kMmaKeys * HD * 2;  // a warp's K (or V) rows of one stage
  static constexpr int kSmem = kMmaWarps * kStages * 2 * kTileBytes;
  static constexpr int kCtas = HD == 256 ? 1 : 3;  // per SM
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

template <typename T, int HD>
__global__ void __launch_bounds__(kMmaThreads, MmaCfg<HD>::kCtas) k_paged_attn_mma(const PagedAttnArgs a) {
  using Cfg = MmaCfg<HD>;
  constexpr int kChunks = HD / 8;                      // 16-byte chunks of a row
  constexpr int kCopies = kMmaKeys * kChunks / 32;     // of a lane, per K (or V) tile
  constexpr int kStages = Cfg::kStages;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  __shared__ PagedShared sched;
  __shared__ unsigned last_s;
  __shared__ float stat_s[kMmaWarps][2][kMmaRows];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r4 = lane >> 2, c4 = lane & 3;
  uint8_t* ring = smem_raw + warp * kStages * 2 * Cfg::kTileBytes;
  const uint32_t ring_a = smem_addr(ring);
  const int block_tokens = kMmaRows / a.group;
  PagedWalk<kMmaTile> walk;
  // join_units: one request of 4,000 keys takes 25.3, 19.5 and 21.9 us at 0, 1/4 and 1
  walk.start(a, &sched, block_tokens, 0, 1, 0.3f);
  PagedPiece p;
  while (walk.next(a, &p)) {
    const int t0 = p.b * block_tokens, rows = min(block_tokens, p.req.n_new - t0) * a.group;
    const int seen = paged_seen(p.req, p.b, block_tokens);
    const int n_tiles = p.tile1 - p.tile0, key_first = p.tile0 * kMmaTile + warp * kMmaKeys;
    const int32_t* table = a.table + p.r * a.table_stride;
    const T* kg = static_cast<const T*>(a.kc) + p.h * a.head_stride;
    const T* vg = static_cast<const T*>(a.vc) + p.h * a.head_stride;
    // the pages of a warp's 16 keys of tile i: rows 0-7 and 8-15
    auto ids = [&](int i, int& id0, int& id1) {
      const int key = key_first + i * kMmaTile;
      id0 = i < n_tiles && key < seen ? table[key >> a.page_shift] : -1;
      id1 = i < n_tiles && key + 8 < seen ? table[(key + 8) >> a.page_shift] : -1;
    };
    auto load = [&](int i, int id0, int id1) {
      if (i < n_tiles) {
        const int key0 = key_first + i * kMmaTile;
        const uint32_t dst = ring_a + (i % kStages) * 2 * Cfg::kTileBytes;
#pragma unroll
        for (int j = 0; j < kCopies; ++j) {
          const int e = lane + 32 * j, row = e / kChunks, c = e % kChunks;
          const int id = row < 8 ? id0 : id1;
          const bool in = key0 + row < seen && id >= 0 && id < a.n_pages;
          const long long at =
              in ? id * a.page_stride + ((key0 + row) & ((1 << a.page_shift) - 1)) * a.token_stride + c * 8 : 0;
          const uint32_t d = dst + row * HD * 2 + ((c ^ (row & 7)) << 4);
          const int n = in ? 16 : 0;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(kg + at), "r"(n) : "memory");
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d + Cfg::kTileBytes), "l"(vg + at), "r"(n)
                       : "memory");
        }
      }
      cp_async_commit();
    };
    int id0, id1;
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
      ids(i, id0, id1);
      load(i, id0, id1);
    }
    ids(kStages - 1, id0, id1);

    uint32_t qf[HD / 16][4];
    int see[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = r4 + 8 * i;
      see[i] = row < rows ? max(0, p.req.len - p.req.n_new + t0 + row / a.group + 1) : 0;
      const T* qr = static_cast<const T*>(a.q) + (p.req.q0 + t0 + row / a.group) * a.q_stride +
                    (long long)(p.h * a.group + row % a.group) * HD + c4 * 2;
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        qf[k][i] = row < rows ? *reinterpret_cast<const uint32_t*>(qr + k * 16) : 0u;
        qf[k][2 + i] = row < rows ? *reinterpret_cast<const uint32_t*>(qr + k * 16 + 8) : 0u;
      }
    }
    // keys that every row of the block sees: before them nothing is masked
    const int see_all = max(0, p.req.len - p.req.n_new + t0 + 1);
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[HD / 8][4];
#pragma unroll
    for (int c = 0; c < HD / 8; ++c) o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f;

    for (int i = 0; i < n_tiles; ++i) {
      cp_async_wait<kStages - 2>();
      __syncwarp();
      load(i + kStages - 1, id0, id1);  // into the stage that the last iteration read
      ids(i + kStages, id0, id1);
      const int key0 = key_first + i * kMmaTile;
      if (key0 >= seen) continue;
      const uint32_t kt = ring_a + (i % kStages) * 2 * Cfg::kTileBytes, vt = kt + Cfg::kTileBytes;
      float sc[2][4] = {};
      {
        const int row = (lane & 7) + ((lane & 16) >> 1);  // matrices: keys 0-7 | 0-7 | 8-15 | 8-15, halves of 16 values
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          uint32_t b[4];
          const int c = 2 * k + ((lane >> 3) & 1);
          ldsm4(b, kt + row * HD * 2 + ((c ^ (row & 7)) << 4));
          Frag<T>::mma(sc[0], qf[k], b[0], b[1]);
          Frag<T>::mma(sc[1], qf[k], b[2], b[3]);
        }
      }
      const bool partial = key0 + kMmaKeys > see_all;
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = sc[n][e] * a.scale_log2;
          if (partial && key0 + n * 8 + c4 * 2 + (e & 1) >= see[e >> 1]) v = -INFINITY;
          sc[n][e] = v;
          mx[e >> 1] = fmaxf(mx[e >> 1], v);
        }
      float base[2], corr[2];
      bool moved = false;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
        const float mn = fmaxf(m[r], mx[r]);
        base[r] = mn == -INFINITY ? 0.f : mn;
        corr[r] = paged_exp2(m[r] - base[r]);
        moved |= mn > m[r];
        m[r] = mn;
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int r = 0; r < 2; ++r) l[r] *= corr[r];
#pragma unroll
        for (int c = 0; c < HD / 8; ++c) {
          o[c][0] *= corr[0], o[c][1] *= corr[0];
          o[c][2] *= corr[1], o[c][3] *= corr[1];
        }
      }
      uint32_t pf[4];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] = paged_exp2(sc[n][e] - base[e >> 1]);
          l[e >> 1] += w[e];
        }
        pf[2 * n] = Frag<T>::pack(w[0], w[1]);
        pf[2 * n + 1] = Frag<T>::pack(w[2], w[3]);
      }
      bool wild = false;
      if (partial) {
        // a key that a row does not see adds nothing, whatever V holds there;
        // 0 * inf would, so a tile with such values goes another way
#pragma unroll
        for (int j = 0; j < kCopies; ++j) {
          const uint4 v = *reinterpret_cast<const uint4*>(ring + (i % kStages) * 2 * Cfg::kTileBytes + Cfg::kTileBytes +
                                                          (lane + 32 * j) * 16);
          wild |= not_finite<T>(v.x) || not_finite<T>(v.y) || not_finite<T>(v.z) || not_finite<T>(v.w);
        }
        wild = __any_sync(0xffffffffu, wild);
      }
      if (!wild) {
        const int row = lane & 15;  // matrices: keys 0-7 | 8-15 of 8 values, twice
#pragma unroll
        for (int c = 0; c < HD / 16; ++c) {
          uint32_t b[4];
          const int ch = 2 * c + (lane >> 4);
          ldsm4t(b, vt + row * HD * 2 + ((ch ^ (row & 7)) << 4));
          Frag<T>::mma(o[2 * c], pf, b[0], b[1]);
          Frag<T>::mma(o[2 * c + 1], pf, b[2], b[3]);
        }
      } else {
        for (int key = 0; key < kMmaKeys; ++key) {
          // the weights of rows r4 and r4 + 8 for this key, from the lane of the quad that has them
          const int src = (lane & ~3) | ((key & 7) >> 1);
          const float2 lo = Frag<T>::unpack(__shfl_sync(0xffffffffu, pf[key < 8 ? 0 : 2], src));
          const float2 hi = Frag<T>::unpack(__shfl_sync(0xffffffffu, pf[key < 8 ? 1 : 3], src));
          const float w0 = key & 1 ? lo.y : lo.x, w1 = key & 1 ? hi.y : hi.x;
          const bool on0 = key0 + key < see[0], on1 = key0 + key < see[1];
#pragma unroll
          for (int c = 0; c < HD / 8; ++c) {
            const float2 v = Frag<T>::unpack(*reinterpret_cast<const uint32_t*>(
                ring + (i % kStages) * 2 * Cfg::kTileBytes + Cfg::kTileBytes + key * HD * 2 + ((c ^ (key & 7)) << 4) + c4 * 4));
            if (on0) o[c][0] += w0 * v.x, o[c][1] += w0 * v.y;
            if (on1) o[c][2] += w1 * v.x, o[c][3] += w1 * v.y;
          }
        }
      }
    }
    cp_async_wait<0>();

    // the four warps' sums, on the largest of their maxima
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (c4 == 0) {
        stat_s[warp][0][r4 + 8 * r] = m[r];
        stat_s[warp][1][r4 + 8 * r] = l[r];
      }
    }
    __syncthreads();  // every warp is done with its ring
    float* osum = reinterpret_cast<float*>(smem_raw);  // [warp][row][HD + 4]
    constexpr int kLd = HD + 4;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = r4 + 8 * r;
      float mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < kMmaWarps; ++w) mm = fmaxf(mm, stat_s[w][0][row]);
      const float f = paged_exp2(m[r] - (mm == -INFINITY ? 0.f : mm));
      float* dst = osum + (warp * kMmaRows + row) * kLd + c4 * 2;
#pragma unroll
      for (int c = 0; c < HD / 8; ++c)
        *reinterpret_cast<float2*>(dst + c * 8) = make_float2(o[c][2 * r] * f, o[c][2 * r + 1] * f);
    }
    __syncthreads();
    // from here on a thread has HD / 8 columns of one row, in groups of 4
    const int row = tid >> 3, col = (tid & 7) * 4;
    float mm = -INFINITY, ll = 0.f;
#pragma unroll
    for (int w = 0; w < kMmaWarps; ++w) mm = fmaxf(mm, stat_s[w][0][row]);
    const float mbase = mm == -INFINITY ? 0.f : mm;
#pragma unroll
    for (int w = 0; w < kMmaWarps; ++w) ll += stat_s[w][1][row] * paged_exp2(stat_s[w][0][row] - mbase);
    float4 acc[HD / 32];
#pragma unroll
    for (int c = 0; c < HD / 32; ++c) {
      acc[c] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kMmaWarps; ++w) {
        const float4 v = *reinterpret_cast<const float4*>(osum + (w * kMmaRows + row) * kLd + col + 32 * c);
        acc[c].x += v.x, acc[c].y += v.y, acc[c].z += v.z, acc[c].w += v.w;
      }
    }
    bool write = p.n_ctas == 1;
    if (!write) {
      float* part = a.partial + (paged_slot(blockIdx.x, p.first_cta) * kMmaRows + row) * kLd;
      if (row < rows) {
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) *reinterpret_cast<float4*>(part + 4 + col + 32 * c) = acc[c];
        if (col == 0) *reinterpret_cast<float2*>(part) = make_float2(mm, ll);
      }
      if (paged_last(a, p, &last_s)) {
        write = true;
        if (row < rows) {
          mm = -INFINITY, ll = 0.f;
#pragma unroll 8
          for (int c = 0; c < p.n_ctas; ++c)
            mm = fmaxf(mm, __ldcg(a.partial + (paged_slot(p.first_cta + c, p.first_cta) * kMmaRows + row) * kLd));
          const float b = mm == -INFINITY ? 0.f : mm;
#pragma unroll
          for (int c = 0; c < HD / 32; ++c) acc[c] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll(HD == 256 ? 2 : 4)
          for (int k = 0; k < p.n_ctas; ++k) {
            const float* src = a.partial + (paged_slot(p.first_cta + k, p.first_cta) * kMmaRows + row) * kLd;
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(src));
            const float f = paged_exp2(ml.x - b);
            ll += ml.y * f;
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) {
              const float4 v = __ldcg(reinterpret_cast<const float4*>(src + 4 + col + 32 * c));
              acc[c].x += v.x * f, acc[c].y += v.y * f, acc[c].z += v.z * f, acc[c].w += v.w * f;
            }
          }
        }
      }
    }
    if (write && row < rows) {
      const bool any = p.req.len - p.req.n_new + t0 + row / a.group + 1 > 0;
      const long long t = p.req.q0 + t0 + row / a.group;
      const int head = p.h * a.group + row % a.group;
      const float inv = any ? 1.0f / ll : 0.f;
      T* dst = static_cast<T*>(a.out) + t * a.out_stride + (long long)head * HD + col;
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) {
        uint2 u = make_uint2(0u, 0u);
        if (any) u = make_uint2(Frag<T>::pack(acc[c].x * inv, acc[c].y * inv), Frag<T>::pack(acc[c].z * inv, acc[c].w * inv));
        *reinterpret_cast<uint2*>(dst + 32 * c) = u;
      }
      if (a.lse && col == 0)
        a.lse[t * a.q_heads + head] = any ? 0.693147180559945309f * (mm + log2f(ll)) : -INFINITY;
    }
    __syncthreads();  // the next piece's loads overwrite the sums
  }
}

// The kernel's shared memory and the SM count, set up once per device.
template <auto kKernel>
cudaError_t ready(size_t smem, int* sms) {
  static OncePerDevice once;
  static int count[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64) return cudaErrorInvalidDevice;
  e = once([&] {
    cudaError_t r = cudaDeviceGetAttribute(&count[dev], cudaDevAttrMultiProcessorCount, dev);
    if (r == cudaSuccess) r = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    return r;
  });
  *sms = count[dev];
  return e;
}

template <int HD>
cudaError_t launch_f32(const PagedAttnArgs& a, cudaStream_t st) {
  int sms = 0;
  const cudaError_t e = ready<k_paged_attn_f32<HD>>(sizeof(SimtSmem<HD>), &sms);
  if (e != cudaSuccess) return e;
  const int ctas = kSimtCtas<HD> * sms;
  k_paged_attn_f32<HD><<<ctas < kPagedMaxCtas ? ctas : kPagedMaxCtas, kSimtThreads, sizeof(SimtSmem<HD>), st>>>(a);
  return cudaGetLastError();
}

template <typename T, int HD>
cudaError_t launch_mma(const PagedAttnArgs& a, cudaStream_t st) {
  using Cfg = MmaCfg<HD>;
  static_assert(Cfg::kSmem >= kMmaWarps * kMmaRows * (HD + 4) * 4, "the joined sums fit the rings");
  int sms = 0;
  const cudaError_t e = ready<k_paged_attn_mma<T, HD>>(Cfg::kSmem, &sms);
  if (e != cudaSuccess) return e;
  const int ctas = Cfg::kCtas * sms;
  k_paged_attn_mma<T, HD><<<ctas < kPagedMaxCtas ? ctas : kPagedMaxCtas, kMmaThreads, Cfg::kSmem, st>>>(a);
  return cudaGetLastError();
}

// cuTensorMapEncodeTiled, from the driver.
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static const EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeFn>(f);
  }();
  return fn;
}

// A 4-D map of 16-bit values read in boxes of 64 x box[0..2] with the
// 128-byte swizzle; strides in values.
bool encode4(CUtensorMap* m, bool bf16, const void* base, const uint64_t (&dims)[4], const uint64_t (&strides)[3],
             const uint32_t (&box)[3]) {
  const cuuint64_t d[4] = {dims[0], dims[1], dims[2], dims[3]};
  const cuuint64_t st[3] = {strides[0] * 2, strides[1] * 2, strides[2] * 2};
  const cuuint32_t b[4] = {64, box[0], box[1], box[2]}, one[4] = {1, 1, 1, 1};
  return encode_fn() &&
         encode_fn()(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base),
                     d, st, b, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// False where the driver does not take the strides: the other kernel does.
bool tc_maps(TcMaps* m, const PagedAttnArgs& a, int hd, bool bf16) {
  const uint64_t h = (uint64_t)hd, page = 1ull << a.page_shift, hs = a.head_stride, ts = a.token_stride, ps = a.page_stride;
  const uint32_t rows = (uint32_t)(page < kTcKeys ? page : kTcKeys);
  const uint64_t g = (uint64_t)a.group;
  m->heads_inner = hs <= ts;
  const uint64_t kd_h[4] = {h, (uint64_t)a.kv_heads, page, (uint64_t)a.n_pages}, ks_h[3] = {hs, ts, ps};
  const uint64_t kd_t[4] = {h, page, (uint64_t)a.kv_heads, (uint64_t)a.n_pages}, ks_t[3] = {ts, hs, ps};
  const uint32_t kb_h[3] = {1, rows, 1}, kb_t[3] = {rows, 1, 1};
  for (int i = 0; i < 2; ++i) {
    CUtensorMap* map = i ? &m->v : &m->k;
    const void* base = i ? a.vc : a.kc;
    if (!(m->heads_inner ? encode4(map, bf16, base, kd_h, ks_h, kb_h) : encode4(map, bf16, base, kd_t, ks_t, kb_t)))
      return false;
  }
  const uint64_t qd[4] = {h, g, (uint64_t)a.kv_heads, (uint64_t)a.n_tokens}, qs[3] = {h, g * h, (uint64_t)a.q_stride};
  const uint32_t qb[3] = {(uint32_t)g, 1, (uint32_t)(kTcRows / g)};
  return encode4(&m->q, bf16, a.q, qd, qs, qb);
}

template <typename T, int HD>
cudaError_t launch_tc(const PagedAttnArgs& a, const TcMaps& m, cudaStream_t st) {
  int sms = 0;
  const cudaError_t e = ready<k_paged_attn_tc<T, HD>>(TcCfg<HD>::kSmem, &sms);
  if (e != cudaSuccess) return e;
  k_paged_attn_tc<T, HD><<<sms < kTcMaxCtas ? sms : kTcMaxCtas, kTcThreads, TcCfg<HD>::kSmem, st>>>(a, m);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_16(const PagedAttnArgs& a, int hd, cudaStream_t st) {
  // Many rows per request: 256-row blocks on the tensor cores.  Few: 16-row
  // blocks, whose time is the K/V stream's.  Behind 4,000 keys (8 K/V heads of
  // 128, bf16), 16-row against 256-row blocks: 32 requests of 21 rows 88 and
  // 118 us, of 42 147 and 118; 8 of 22 41 and 49, of 45 57 and 50; one request
  // has few blocks to share the SMs out to, and a join: 128 rows 35 and 45, 256
  // 52 and 47.
  if (hd <= 128 && a.scale_log2 > 0.f && (long long)a.n_tokens * a.group >= 40ll * a.n_req &&
      (long long)a.n_tokens * a.q_heads >= 1536) {
    TcMaps m;
    if (tc_maps(&m, a, hd, Frag<T>::kExp == 0x7f807f80u))
      return hd == 64 ? launch_tc<T, 64>(a, m, st) : launch_tc<T, 128>(a, m, st);
  }
  return hd == 64 ? launch_mma<T, 64>(a, st) : hd == 128 ? launch_mma<T, 128>(a, st) : launch_mma<T, 256>(a, st);
}

// the workspace: tickets, the error word, then two pieces of a block for every CTA
constexpr size_t kHeadBytes = kPagedMaxCtas * sizeof(unsigned) + 256;
static_assert(kHeadBytes + (size_t)kPagedMaxCtas * 2 * kMmaRows * 260 * 4 <= MINICPMO_PAGED_WORKSPACE_BYTES, "workspace");
static_assert(kHeadBytes + (size_t)kTcMaxCtas * 2 * 256 * 132 * 4 <= MINICPMO_PAGED_WORKSPACE_BYTES, "workspace");
static_assert(2 * kTcMaxCtas <= kPagedMaxCtas, "tickets");

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
  if (max_pages < 1 || max_pages > (size_t)(1 << 30) / cache->page_size || table_stride < max_pages ||
      table_stride > (1ull << 40))
    return paged_error(error, error_cap, "error: %s: table rows of %zu pages, %zu apart", op, max_pages, table_stride);
  if (q_stride < q_heads * hd || out_stride < q_heads * hd || q_stride > (1ull << 40) || out_stride > (1ull << 40))
    return paged_error(error, error_cap, "error: %s: tokens' rows overlap", op);
  if (!aligned16(q) || !aligned16(out) || q_stride * esz % 16 || out_stride * esz % 16 ||
      (reinterpret_cast<uintptr_t>(workspace) & 255))
    return paged_error(error, error_cap,
                       "error: %s: pointers and strides must be multiples of 16 bytes, the workspace of 256", op);
  if (!(scale > -INFINITY && scale < INFINITY)) return paged_error(error, error_cap, "error: %s: scale is not finite", op);
  if (!paged_on_device(cache->k, op, error, error_cap)) return 0;
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
  a.err = reinterpret_cast<int*>(a.tickets + kPagedMaxCtas);
  a.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kHeadBytes);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaErrorNotSupported;
  if (cache->dtype == kF32)
    e = hd == 64 ? launch_f32<64>(a, st) : hd == 128 ? launch_f32<128>(a, st) : launch_f32<256>(a, st);
  else if (cache->dtype == kF16)
    e = launch_16<__half>(a, (int)hd, st);
  else
    e = launch_16<__nv_bfloat16>(a, (int)hd, st);
  if (e != cudaSuccess) return paged_error(error, error_cap, "error: %s: launch: %s", op, cudaGetErrorString(e));
  return 1;
}
