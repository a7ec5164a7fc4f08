// paged_attn.cuh -- the work split of the paged attention kernels.
//
// A unit of work is one tile of KT keys for one block of new tokens of one
// request and one kv head (all q heads of the group are rows of the block, so
// K and V are read once for them).  The units of all requests, in the order
// request, kv head, block, tile, are cut into equal contiguous ranges, one per
// CTA: ragged lengths leave no CTA with more than one unit above the average,
// whatever the mix of long and short requests, and the lengths stay on the
// device.  A cut within `snap` units of a block's end moves there, since a
// piece costs as much as a few units.  A block whose tiles lie in several
// ranges is computed in pieces;
// each piece leaves its sums in the workspace, and the CTA that finishes last
// adds them in the ranges' order, so the result does not depend on timing.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

namespace mcpo {

constexpr int kPagedMaxCtas = 1024;  // tickets in the workspace
constexpr int kPagedMaxGroup = 16;   // q heads per kv head

struct PagedAttnArgs {
  const void* q;
  void* out;
  float* lse;
  const void *kc, *vc;
  const int32_t *table, *lens, *cu;
  long long q_stride, out_stride, table_stride, page_stride, token_stride, head_stride;
  int n_tokens, n_req, q_heads, kv_heads, group;
  long long max_pages, n_pages;
  int page_shift;
  float scale_log2;     // scale * log2(e): scores are kept in base 2
  unsigned* tickets;    // [kPagedMaxCtas], zero at rest
  int* err;             // raised by a bounded wait that gave up
  float* partial;       // [CTA][2][rows of a block][head_dim + 2]
};

// One request's share of the batch.
struct PagedReq {
  int q0, n_new, len, blocks;
};

__device__ __forceinline__ PagedReq paged_req(const PagedAttnArgs& a, int r, int block_tokens) {
  PagedReq q;
  const int c0 = a.cu[r], c1 = a.cu[r + 1], len = a.lens[r];
  q.q0 = min(max(c0, 0), a.n_tokens);
  q.n_new = min(max(c1, q.q0), a.n_tokens) - q.q0;
  const long long most = a.max_pages << a.page_shift;
  q.len = (int)min((long long)max(len, 0), most);
  q.blocks = (q.n_new + block_tokens - 1) / block_tokens;
  return q;
}

// Keys that the last token of block b sees, and its tiles (at least one, so
// that blocks that see nothing are written too).
__device__ __forceinline__ int paged_seen(const PagedReq& q, int b, int block_tokens) {
  const int last = min(q.n_new, (b + 1) * block_tokens) - 1;
  return max(0, q.len - q.n_new + last + 1);
}
template <int KT>
__device__ __forceinline__ int paged_tiles(const PagedReq& q, int b, int block_tokens) {
  return max(1, (paged_seen(q, b, block_tokens) + KT - 1) / KT);
}
template <int KT>
__device__ __forceinline__ long long paged_head_units(const PagedReq& q, int block_tokens) {
  long long u = 0;
  for (int b = 0; b < q.blocks; ++b) u += paged_tiles<KT>(q, b, block_tokens);
  return u;
}

struct PagedShared {
  long long red[32];
  int longest[32];
  long long total, before;  // all units; those before request r
  int r;                    // the request of this CTA's first unit
};

// A piece of one block: tiles [tile0, tile1) of n_tiles.
struct PagedPiece {
  PagedReq req;
  int r, h, b, tile0, tile1, n_tiles;
  int first_cta, n_ctas;  // the CTAs that share the block
};

template <int KT>
struct PagedWalk {
  int block_tokens, ctas, snap;
  long long total, u, u1;  // this CTA's next and last unit
  PagedReq req;
  int r, h, b;
  long long block0;  // unit of the block's first tile

  // A cut x inside the block [b0, b0 + n), moved to its start or end when near.
  __device__ __forceinline__ long long cut(long long x, long long b0, int n) const {
    const int d = min(snap, n / 2);
    return x <= b0 + d ? b0 : x >= b0 + n - d ? b0 + n : x;
  }
  // The last CTA whose unmoved cut is at or before x.
  __device__ __forceinline__ int cta_of(long long x) const { return (int)(((x + 1) * ctas - 1) / total); }

  // The request, head and block that hold unit x (x < total).  Block-wide.
  __device__ __forceinline__ void locate(const PagedAttnArgs& a, PagedShared* s, long long x, long long ex, long long mine,
                                         int r0, int r1) {
    __syncthreads();
    if (x >= ex && x < ex + mine) {  // the thread whose requests hold it finds which
      long long at = ex;
      for (int i = r0; i < r1; ++i) {
        const long long ui = paged_head_units<KT>(paged_req(a, i, block_tokens), block_tokens) * a.kv_heads;
        if (x < at + ui) {
          s->r = i;
          s->before = at;
          break;
        }
        at += ui;
      }
    }
    __syncthreads();
    r = s->r;
    req = paged_req(a, r, block_tokens);
    const long long off = x - s->before, per_head = paged_head_units<KT>(req, block_tokens);
    h = (int)(off / per_head);
    b = 0;
    block0 = s->before + h * per_head;
    for (int n = paged_tiles<KT>(req, 0, block_tokens); x >= block0 + n; n = paged_tiles<KT>(req, b, block_tokens)) {
      block0 += n;
      ++b;
    }
  }

  __device__ __forceinline__ void next_block(const PagedAttnArgs& a) {
    if (++b == req.blocks) {
      b = 0;
      if (++h == a.kv_heads) {
        h = 0;
        do {
          req = paged_req(a, ++r, block_tokens);
        } while (req.blocks == 0);
      }
    }
  }

  // Block-wide: every thread of the CTA calls it, and gets the same walk.
  __device__ __forceinline__ void start(const PagedAttnArgs& a, PagedShared* s, int block_tokens_, int snap_, int min_units,
                                        float join_units) {
    block_tokens = block_tokens_;
    snap = snap_;
    const int n = a.n_req, nt = blockDim.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (n + nt - 1) / nt, r0 = min(n, tid * per), r1 = min(n, r0 + per);
    long long mine = 0;
    int longest = 0;  // units of the longest block
    for (int i = r0; i < r1; ++i) {
      const PagedReq q = paged_req(a, i, block_tokens);
      mine += paged_head_units<KT>(q, block_tokens);
      if (q.blocks > 0) longest = max(longest, paged_tiles<KT>(q, q.blocks - 1, block_tokens));
    }
    longest = __reduce_max_sync(0xffffffffu, longest);
    mine *= a.kv_heads;
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) s->red[warp] = incl, s->longest[warp] = longest;
    __syncthreads();
    long long base = 0, all = 0;
    for (int w = 0; w < nt / 32; ++w) {
      if (w < warp) base += s->red[w];
      all += s->red[w];
      longest = max(longest, s->longest[w]);
    }
    const long long ex = base + incl - mine;
    total = all;
    // Pieces of c units make the longest block of n take about c for its own
    // piece and join_units * n / c for the join, one piece behind the other:
    // least at c = sqrt(join_units * n), and no CTA takes less than that while
    // there are more CTAs than the units need.
    const int least = max(min_units, (int)sqrtf(join_units * (float)longest));
    ctas = (int)min((long long)gridDim.x, max(1ll, total / least));
    u = u1 = total;
    if ((int)blockIdx.x >= ctas || total == 0) return;  // the same for the whole block
    const long long x0 = (long long)blockIdx.x * total / ctas, x1 = (long long)(blockIdx.x + 1) * total / ctas;
    if (x1 < total) {
      locate(a, s, x1, ex, mine, r0, r1);
      u1 = cut(x1, block0, paged_tiles<KT>(req, b, block_tokens));
    }
    locate(a, s, x0, ex, mine, r0, r1);
    const int len = paged_tiles<KT>(req, b, block_tokens);
    u = cut(x0, block0, len);
    if (u < u1 && u == block0 + len) {
      block0 = u;
      next_block(a);
    }
  }

  // The next piece of this CTA's range; false at its end.
  __device__ __forceinline__ bool next(const PagedAttnArgs& a, PagedPiece* p) {
    if (u >= u1) return false;
    const int n = paged_tiles<KT>(req, b, block_tokens), d = min(snap, n / 2);
    p->req = req;
    p->r = r;
    p->h = h;
    p->b = b;
    p->n_tiles = n;
    p->tile0 = (int)(u - block0);
    p->tile1 = (int)min((long long)n, u1 - block0);
    // the CTAs whose moved ranges meet the block: from the last cut that is at
    // or moves to its start, to the last one before those that move to its end
    p->first_cta = cta_of(block0 + d);
    p->n_ctas = max(0, cta_of(block0 + n - d - 1) - p->first_cta) + 1;
    u = block0 + p->tile1;
    if (p->tile1 == n && u < u1) {
      block0 = u;
      next_block(a);
    }
    return true;
  }
};

// The workspace slot of CTA `cta`'s piece of a block that begins in
// first_cta: a CTA holds at most one block that began before it (0) and one
// that goes on behind it (1).
__device__ __forceinline__ long long paged_slot(int cta, int first_cta) { return 2ll * cta + (cta == first_cta ? 1 : 0); }

__device__ __forceinline__ float paged_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What the kernels of 16-bit types need to know of them.
template <typename T>
struct Frag;
template <>
struct Frag<__half> {
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }
  static constexpr uint32_t kExp = 0x7c007c00u;  // exponent bits of both values
};
template <>
struct Frag<__nv_bfloat16> {
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
  static constexpr uint32_t kExp = 0x7f807f80u;
};

// Whether either 16-bit value of u is infinite or NaN.
template <typename T>
__device__ __forceinline__ bool not_finite(uint32_t u) {
  const uint32_t e = u & Frag<T>::kExp;
  return (e & 0xffffu) == (Frag<T>::kExp & 0xffffu) || (e >> 16) == (Frag<T>::kExp >> 16);
}

}  // namespace mcpo
