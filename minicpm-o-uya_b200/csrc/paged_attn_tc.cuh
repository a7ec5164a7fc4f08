// paged_attn_tc.cuh -- paged attention on the tcgen05 tensor cores, for
// chunks of many new tokens (f16 or bf16, head_dim 64 or 128).
//
// A block is two tiles of 128 rows (tokens x q heads of a kv head).  Per step
// of 64 keys, S = Q K^T goes to tensor memory (64 f32 columns), one thread per
// row turns it into weights P that overwrite the first 32 columns as 16-bit
// values, and O += P V reads them from there.  Each tile has two such S/P
// buffers, so Q K^T of the next step runs while the softmax of this one does:
// with one buffer of 128 keys the chain softmax -> P V -> Q K^T took 4070
// cycles per 128 keys, of which the tensor cores worked 2048.  64 keys cost
// shared-memory bandwidth (Q is read again for each), about 2560 cycles per 128
// keys.  Now a step of both tiles takes about 1930 cycles (1280 of MMAs, 1024
// of exponentials): 4 chunks of up to 2048 tokens behind up to 16,384 keys (32
// heads, 8 K/V heads of 128, bf16) take 1.44 to 1.7 ms with the clock, up to
// 960 TFLOP/s.  The softmax's latency, one thread per row, is what is left.
// Roles: warps 0-3 and 4-7 are the softmax of tile 0 and 1, warps 8 and 9 issue
// their MMAs (in step i P V (i), then Q K^T (i + 2) into the buffer that P was
// in; the queue of MMAs is short, and one thread's waits for both tiles left
// the tensor cores idle for a third of the time), warp 10 the TMA loads of Q
// and of K and V pages (a ring of 64-key stages that both tiles read); warp 11
// only fills the warpgroup, whose registers go to the softmax warps.
//
// Rows keep the maximum they began with until a score exceeds it by 2^8;
// weights up to 2^8 lose nothing in these types, and the accumulator is
// rescaled only then.  Tensor memory: S/P of tile t in columns 128 t and
// 128 t + 64, O in 256 + head_dim t.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "paged_attn.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace mcpo {

constexpr int kTcRows = 128, kTcKeys = 64, kTcThreads = 384;
constexpr int kTcMaxCtas = 240;  // by the workspace
constexpr uint32_t kTcTmem = 512;

template <int HD>
struct TcCfg {
  static constexpr int kStageBytes = kTcKeys * HD * 2;
  static constexpr int kStages = 8;
  static constexpr int kHalves = HD / 64;  // 128-byte column blocks of a row
  static constexpr int kQBytes = kTcRows * HD * 2;
  static constexpr int kSmem = 2 * kQBytes + kStages * kStageBytes + 1024;  // with slack for the 1 KB alignment
};

// One lane of the warp.  tcgen05 operands sit in uniform registers; behind
// this predicate (and not behind lane == 0) the compiler knows that one thread
// is active, and an MMA takes a few instructions instead of about 100 cycles.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}

struct TcMaps {
  CUtensorMap q, k, v;
  int heads_inner;  // K/V map's dimensions: (hd, heads, tokens, pages), else (hd, tokens, heads, pages)
};

// Shared-memory operands with the 128-byte swizzle, as the low word of their
// descriptor (start address, and the leading offset in 16-byte units); the high
// word is the same for all: 8-row groups 1 KB apart.  K-major: rows of 128
// bytes.  MN-major: rows (k) of 64 values, the next 64 `lead` bytes further.
// Offsets within an operand are added to the low word, / 16.
constexpr uint32_t kTcDescHigh = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t tc_low(uint32_t saddr, uint32_t lead) { return (saddr >> 4) | ((lead >> 4) << 16); }
__device__ __forceinline__ uint64_t tc_desc(uint32_t low) { return ((uint64_t)kTcDescHigh << 32) | low; }

__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}

// 32 consecutive columns of this thread's lane; wait with tc_wait_ld before use.
__device__ __forceinline__ void tc_ld32(uint32_t addr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tc_ld16(uint32_t addr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
__device__ __forceinline__ void tc_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tc_st32(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// Makes the registers of the loads above depend on the wait.
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tc_tma_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_addr(bar))
      : "memory");
}

__device__ __forceinline__ uint64_t f2_pack(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 f2_unpack(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ uint64_t f2_all(float x) { return f2_pack(x, x); }

// How often a stage or buffer has been used decides the parity to wait for;
// the n-th of K and V loads of a block of n_steps, K(0) K(1) V(0) K(2) V(1) ...
__device__ __forceinline__ uint32_t tc_k_load(int i) { return i ? 2 * i - 1 : 0; }
__device__ __forceinline__ uint32_t tc_v_load(int i, int n_steps) { return i + 1 < n_steps ? 2 * i + 2 : 2 * i + 1; }

struct TcShared {
  uint64_t q_full, q_empty;
  uint64_t kv_full[8], kv_empty[8];
  uint64_t s_full[2][2], p_full[2][2];  // [tile][buffer]
  uint64_t pv_done[2][2], epi_done[2];
  uint32_t tmem;
  int abort_;
  unsigned last[2];
  // Values of V that are not finite, in steps that some row sees only part of:
  // they are 0 for the product, and here is, per column, the first key that
  // holds +inf, -inf or NaN.
  int wild;
  int first[3][128];
  // Counts that only grow (a tile can be several steps or short blocks ahead
  // of the other, which the parity of a barrier could not tell): warps that
  // have made a step's V finite, and warps of tile 1 that have written a block.
  unsigned v_fine, tile1_done;
};

__device__ __forceinline__ void tc_count(unsigned* n) {
  asm volatile("red.release.cta.shared::cta.add.u32 [%0], 1;" ::"r"(smem_addr(n)) : "memory");
}
// Bounded wait for a count.
__device__ __forceinline__ bool tc_counted(const unsigned* n, unsigned want, int* err, volatile int* abort_s) {
  for (int i = 0; i < kWaitLimit; ++i) {
    unsigned v;
    asm volatile("ld.acquire.cta.shared::cta.u32 %0, [%1];" : "=r"(v) : "r"(smem_addr(n)) : "memory");
    if ((int)(v - want) >= 0) return true;
    if ((i & 63) == 63 && *abort_s) return false;
  }
  *abort_s = 1;
  if (err) atomicExch(err, 1);
  return false;
}

// Issues tile t's MMAs of all the CTA's pieces.
template <typename T, int HD>
__device__ __forceinline__ void tc_issue(const PagedAttnArgs& a, TcShared& s, PagedWalk<kTcKeys>& walk, PagedPiece& p, int t,
                                         uint32_t q_a, uint32_t kv_a, uint32_t tmem, int tile_tokens) {
  using Cfg = TcCfg<HD>;
  constexpr uint32_t kType = Frag<T>::kExp == 0x7f807f80u ? 1u : 0u;  // 1: bf16
  constexpr uint32_t kBase = (1u << 4) | (kType << 7) | (kType << 10) | ((uint32_t)(kTcRows >> 4) << 24);
  constexpr uint32_t kDescS = kBase | ((uint32_t)(kTcKeys >> 3) << 17);
  constexpr uint32_t kDescO = kBase | (1u << 16) | ((uint32_t)(HD >> 3) << 17);  // V is MN-major
  constexpr int kStages = Cfg::kStages;
  volatile int* abort_s = &s.abort_;
  const uint32_t q_low = tc_low(q_a + t * Cfg::kQBytes, 16), k_low = tc_low(kv_a, 16), v_low = tc_low(kv_a, kTcKeys * 128);
  const uint32_t s_t = tmem + t * 128, o_t = tmem + 256 + t * HD;
  uint32_t stage_n = 0, piece_n = 0, p_parity = 0, epi_n = 0, checked = 0;  // p_parity: a bit per buffer
  bool ok = true;
  auto qk = [&](int buf, uint32_t st) {
    const uint32_t kl = k_low + st * (Cfg::kStageBytes >> 4);
#pragma unroll
    for (int k = 0; k < HD / 16; ++k)
      tc_mma_ss(s_t + buf * 64, tc_desc(q_low + (((k >> 2) * (kTcRows * 128) + (k & 3) * 32) >> 4)),
                tc_desc(kl + (((k >> 2) * (kTcKeys * 128) + (k & 3) * 32) >> 4)), kDescS, k != 0);
    umma_commit(&s.s_full[t][buf]);
  };
  auto loaded = [&](uint32_t load) {  // waits for a load, and gives its stage
    const uint32_t n = stage_n + load;
    ok = ok && gwait(&s.kv_full[n % kStages], (n / kStages) & 1, a.err, abort_s);
    return n % kStages;
  };
  while (ok && walk.next(a, &p)) {
    const int t0 = p.b * 2 * tile_tokens, n = p.tile1 - p.tile0, first_key = p.tile0 * kTcKeys;
    const bool two = p.req.n_new - t0 > tile_tokens;
    const int see_all = max(0, p.req.len - p.req.n_new + t0 + 1);  // of the block's first token
    if (t == 1 && !two) {
      // nothing to issue, but every load is waited for and released by both
      // issuers: a parity says where a barrier is only to one who follows it
      ok = gwait(&s.q_full, piece_n & 1, a.err, abort_s);
      if (ok) mbar_arrive(&s.q_empty);
      ++piece_n;
      for (int i = 0; ok && i < 2 * n; ++i) {
        const uint32_t st = loaded(i);
        if (ok) mbar_arrive(&s.kv_empty[st]);
      }
      stage_n += 2 * n;
      checked += max(0, n - max(0, (see_all - first_key) / kTcKeys));  // steps whose V tile 0 has checked
      continue;
    }
    ok = gwait(&s.q_full, piece_n & 1, a.err, abort_s);
    ++piece_n;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (!ok || i >= n) break;
      const uint32_t ks = loaded(tc_k_load(i));
      if (!ok) break;
      tc_fence_after();
      qk(i, ks);
      umma_commit(&s.kv_empty[ks]);
      if (i + 1 == n) umma_commit(&s.q_empty);
    }
    // O is written from here on: the softmax warps have read the last block's
    if (epi_n) ok = ok && gwait(&s.epi_done[t], (epi_n - 1) & 1, a.err, abort_s);
    for (int i0 = 0; ok && i0 < n; i0 += 2) {
#pragma unroll
      for (int buf = 0; buf < 2; ++buf) {
        const int i = i0 + buf;
        if (!ok || i >= n) break;
        const uint32_t vs = loaded(tc_v_load(i, n));
        if (t == 1 && first_key + (i + 1) * kTcKeys > see_all)
          ok = ok && tc_counted(&s.v_fine, 4 * ++checked, a.err, abort_s);
        ok = ok && gwait(&s.p_full[t][buf], (p_parity >> buf) & 1, a.err, abort_s);
        if (!ok) break;
        p_parity ^= 1u << buf;
        tc_fence_after();
        const uint32_t vl = v_low + vs * (Cfg::kStageBytes >> 4);
#pragma unroll
        for (int k = 0; k < kTcKeys / 16; ++k)
          tc_mma_ts(o_t, s_t + buf * 64 + k * 8, tc_desc(vl + ((k * 2048) >> 4)), kDescO, k != 0 || i != 0);
        umma_commit(&s.pv_done[t][buf]);
        umma_commit(&s.kv_empty[vs]);
        if (i + 2 < n) {
          const uint32_t ks = loaded(tc_k_load(i + 2));
          if (!ok) break;
          tc_fence_after();
          qk(buf, ks);
          umma_commit(&s.kv_empty[ks]);
          if (i + 3 == n) umma_commit(&s.q_empty);
        }
      }
    }
    stage_n += 2 * n;
    ++epi_n;
  }
}

template <typename T, int HD>
__global__ void __launch_bounds__(kTcThreads, 1)
    k_paged_attn_tc(const PagedAttnArgs a, const __grid_constant__ TcMaps maps) {
  using Cfg = TcCfg<HD>;
  constexpr int kStages = Cfg::kStages, kHalves = Cfg::kHalves, kLd = HD + 4;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  __shared__ TcShared s;
  __shared__ PagedShared sched;
  uint8_t* smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
  const uint32_t q_a = smem_addr(smem), kv_a = q_a + 2 * Cfg::kQBytes;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort_s = &s.abort_;

  if (tid == 0) {
    mbar_init(&s.q_full, 1);
    mbar_init(&s.q_empty, 2);  // both issuers
    for (int i = 0; i < kStages; ++i) mbar_init(&s.kv_full[i], 1), mbar_init(&s.kv_empty[i], 2);
    for (int t = 0; t < 2; ++t) {
      for (int b = 0; b < 2; ++b) mbar_init(&s.s_full[t][b], 1), mbar_init(&s.p_full[t][b], 4), mbar_init(&s.pv_done[t][b], 1);
      mbar_init(&s.epi_done[t], 4);
    }
    s.wild = 0;
    s.v_fine = s.tile1_done = 0;
    s.abort_ = 0;
    mbar_fence_init();
  }
  if (warp == 8) tmem_alloc(&s.tmem, kTcTmem);
  const int tile_tokens = kTcRows / a.group, block_tokens = 2 * tile_tokens;
  // every warp walks the CTA's pieces by itself, its lane 0 for it, with the
  // state in shared memory: the softmax rows need the registers
  __shared__ PagedWalk<kTcKeys> walks[kTcThreads / 32];
  __shared__ PagedPiece pieces[kTcThreads / 32];
  {
    PagedWalk<kTcKeys> walk;
    // join_units: 64 tokens behind 4,000 take 64, 55 and 43 us at 0, 1/4 and 1,
    // 512 behind 200 18.2, 18.0 and 22.7.
    walk.start(a, &sched, block_tokens, 4, 1, 0.5f);  // has barriers: the inits above are seen behind them
    if (lane == 0) walks[warp] = walk;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem;
  const PagedPiece& p = pieces[warp];
  auto next_piece = [&]() -> bool {
    __syncwarp();
    bool more = false;
    if (lane == 0) more = walks[warp].next(a, &pieces[warp]);
    return __shfl_sync(0xffffffffu, (int)more, 0) != 0;
  };

  // 384 threads start with 168 registers each (64512): 208 * 256 + 80 * 128 = 63488
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == 10) {
    // ---- loads, by one thread: boxes are a page's rows x 64 values ----
    if (elect_one()) {
      constexpr int kBoxes = kTcKeys / 8;  // of the smallest page
      const int box_rows = min(1 << a.page_shift, kTcKeys);
      const uint32_t box_bytes = box_rows * 128;
      uint32_t stage_n = 0, piece_n = 0;
      bool ok = true;
      while (ok && walks[warp].next(a, &pieces[warp])) {
        const int t0 = p.b * block_tokens, seen = paged_seen(p.req, p.b, block_tokens), n = p.tile1 - p.tile0, h = p.h;
        const bool two = p.req.n_new - t0 > tile_tokens;
        if (piece_n) ok = gwait(&s.q_empty, (piece_n - 1) & 1, a.err, abort_s);
        if (!ok) break;
        const uint32_t bytes = (uint32_t)(tile_tokens * a.group * HD * 2);
        mbar_arrive_expect_tx(&s.q_full, two ? 2 * bytes : bytes);
        for (int t = 0; t < (two ? 2 : 1); ++t)
          for (int c = 0; c < kHalves; ++c)
            tc_tma_4d(q_a + t * Cfg::kQBytes + c * (kTcRows * 128), &maps.q, c * 64, 0, h,
                      p.req.q0 + t0 + t * tile_tokens, &s.q_full);
        ++piece_n;
        const int32_t* table = a.table + p.r * a.table_stride;
        const int first_key = p.tile0 * kTcKeys;
        // the pages of a step's keys that the block sees; fetched a step before they are needed
        struct Ids {
          int n, id[kBoxes];
        };
        auto fetch = [&](int i) {
          Ids d;
          const int key0 = first_key + i * kTcKeys, left = i < n ? min(kTcKeys, seen - key0) : 0;
          d.n = left > 0 ? (left + box_rows - 1) / box_rows : 0;
#pragma unroll
          for (int b = 0; b < kBoxes; ++b) d.id[b] = b < d.n ? table[(key0 + b * box_rows) >> a.page_shift] : 0;
          return d;
        };
        auto load = [&](const CUtensorMap* map, const Ids& d, int i) {
          const uint32_t st = stage_n % kStages;
          if (stage_n >= kStages) ok = gwait(&s.kv_empty[st], (stage_n / kStages - 1) & 1, a.err, abort_s);
          if (!ok) return;
          ++stage_n;
          mbar_arrive_expect_tx(&s.kv_full[st], d.n * kHalves * box_bytes);
          const int row = (first_key + i * kTcKeys) & ((1 << a.page_shift) - 1);  // of pages longer than a step
          const uint32_t dst = kv_a + st * Cfg::kStageBytes;
#pragma unroll
          for (int b = 0; b < kBoxes; ++b) {
            if (b >= d.n) break;
            int id = d.id[b];
            if (id < 0 || id >= a.n_pages) id = (int)a.n_pages;  // out of the map: zeros
#pragma unroll
            for (int c = 0; c < kHalves; ++c) {
              const uint32_t at = dst + c * (kTcKeys * 128) + b * box_bytes;
              if (maps.heads_inner) tc_tma_4d(at, map, c * 64, h, row, id, &s.kv_full[st]);
              else tc_tma_4d(at, map, c * 64, row, h, id, &s.kv_full[st]);
            }
          }
        };
        Ids now = fetch(0), next = fetch(1);
        load(&maps.k, now, 0);
        for (int i = 0; ok && i < n; ++i) {
          const Ids after = fetch(i + 2);
          if (i + 1 < n) load(&maps.k, next, i + 1);
          if (ok) load(&maps.v, now, i);
          now = next;
          next = after;
        }
      }
      // copies in flight land before the shared memory goes
      if (piece_n) mbar_wait(&s.q_full, (piece_n - 1) & 1, a.err);
      for (uint32_t i = stage_n > kStages ? stage_n - kStages : 0; i < stage_n; ++i)
        mbar_wait(&s.kv_full[i % kStages], (i / kStages) & 1, a.err);
    }
    __syncwarp();
    } else if (warp < 10) {
      // ---- MMAs of tile t, by one thread ----
      if (elect_one()) tc_issue<T, HD>(a, s, walks[warp], pieces[warp], warp - 8, q_a, kv_a, tmem, tile_tokens);
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ---- softmax of tile t: thread = row ----
    const int t = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_t = tmem + lane_base + t * 128, o_t = tmem + lane_base + 256 + t * HD;
    uint32_t s_parity = 0, pv_n[2] = {0, 0}, stage_n = 0, pairs = 0;  // s_parity: a bit per buffer; blocks with two tiles
    // P V of step i of this block is done (that of step i - 2 is known to be)
    auto pv_wait = [&](int i) {
      const uint32_t n = (i & 1 ? pv_n[1] : pv_n[0]) + (i >> 1);
      return __all_sync(0xffffffffu, gwait(&s.pv_done[t][i & 1], n & 1, a.err, abort_s)) != 0;
    };
    bool ok = true;
    while (ok && next_piece()) {
      const int t0 = p.b * block_tokens, n = p.tile1 - p.tile0;
      const int rows = min(tile_tokens, p.req.n_new - t0 - t * tile_tokens) * a.group;
      if (rows <= 0) {
        stage_n += 2 * n;
        continue;
      }
      const int tok = t0 + t * tile_tokens + row / a.group;  // of the request's new tokens
      const bool valid = row < rows;
      // rows without a token see everything: what they compute is dropped
      const int see = valid ? max(0, p.req.len - p.req.n_new + tok + 1) : INT_MAX;
      const int see_all = max(0, p.req.len - p.req.n_new + t0 + 1);  // of the block's first token
      // `first` and `wild` are written from here on: tile 1 has read the last blocks'
      if (t == 0) ok = __all_sync(0xffffffffu, tc_counted(&s.tile1_done, 4 * pairs, a.err, abort_s));
      if (!ok) break;
      pairs += p.req.n_new - t0 > tile_tokens;
      const int first_key = p.tile0 * kTcKeys;
      float m = -INFINITY, l = 0.f, top = 0.f;
      // Steps of which every row sees all come first; the others have their own
      // copy of the code, which costs the first ones nothing (10% in one loop).
      const int n_full = min(n, max(0, (see_all - first_key) / kTcKeys));
      // Step i's scores, as soon as they are there (and, before them, its V).
      auto scores = [&](int i, float (&x)[kTcKeys], auto partial) {
        const int key0 = first_key + i * kTcKeys, buf = i & 1;
        if (decltype(partial)::value && t == 0) {
          // V must be finite where weights are 0
          const uint32_t vn = stage_n + tc_v_load(i, n), vs = vn % kStages;
          ok = __all_sync(0xffffffffu, gwait(&s.kv_full[vs], (vn / kStages) & 1, a.err, abort_s));
          if (!ok) return;
          uint8_t* v = smem + 2 * Cfg::kQBytes + vs * Cfg::kStageBytes;
          if (i == n_full) {  // the piece's first such step
            for (int e = tid; e < 3 * 128; e += 128) s.first[e / 128][e % 128] = INT_MAX;
            if (tid == 0) s.wild = 0;
            asm volatile("bar.sync 1, 128;" ::: "memory");
          }
          const int end = paged_seen(p.req, p.b, block_tokens) - key0;
          constexpr uint32_t kExp = Frag<T>::kExp, kOne = (kExp & ~(kExp << 1)) & 0x0fff0fffu;  // the exponents' lowest bits
          uint32_t hit = 0;
#pragma unroll 2
          for (int e = tid; e < Cfg::kStageBytes / 16; e += 128) {  // an exponent of ones carries into the sign's place
            const uint4 u = *reinterpret_cast<const uint4*>(v + e * 16);
            hit |= ((u.x & kExp) + kOne) | ((u.y & kExp) + kOne) | ((u.z & kExp) + kOne) | ((u.w & kExp) + kOne);
          }
          if (hit & 0x80008000u) {
#pragma unroll 1
            for (int e = tid; e < Cfg::kStageBytes / 16; e += 128) {
              const uint4 w4 = *reinterpret_cast<const uint4*>(v + e * 16);
              const int key = (e >> 3) % kTcKeys, half = (e >> 3) / kTcKeys, col = half * 64 + (((e & 7) ^ (key & 7)) << 3);
              uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const uint32_t bits = (w[k >> 1] >> (16 * (k & 1))) & 0xffffu, ex = kExp & 0xffffu;
                if ((bits & ex) != ex) continue;
                w[k >> 1] &= k & 1 ? 0x0000ffffu : 0xffff0000u;
                if (key >= end) continue;  // behind the request: nobody sees it
                const int kind = (bits & 0x7fffu) != ex ? 2 : bits >> 15;
                atomicMin(&s.first[kind][col + k], key0 + key);
                s.wild = 1;
              }
              *reinterpret_cast<uint4*>(v + e * 16) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) tc_count(&s.v_fine);
        }
        ok = __all_sync(0xffffffffu, gwait(&s.s_full[t][buf], (s_parity >> buf) & 1, a.err, abort_s));
        if (!ok) return;
        s_parity ^= 1u << buf;
        tc_fence_after();
        tc_ld32(s_t + buf * 64, x);
        tc_ld32(s_t + buf * 64 + 32, x + 32);
      };
      // Once they have landed: what the row does not see, and the largest.
      auto landed = [&](float (&x)[kTcKeys]) {
        tc_wait_ld();
#pragma unroll
        for (int c = 0; c < kTcKeys; ++c) asm volatile("" : "+f"(x[c]));
      };
      auto largest = [&](int i, float (&x)[kTcKeys], auto partial) {
        if constexpr (decltype(partial)::value) {
          const int lim = see - (first_key + i * kTcKeys);
#pragma unroll
          for (int c = 0; c < kTcKeys; ++c) x[c] = c < lim ? x[c] : -INFINITY;
        }
        float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int c = 4; c < kTcKeys; c += 4)
#pragma unroll
          for (int k = 0; k < 4; ++k) mx[k] = fmaxf(mx[k], x[c + k]);
        top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale_log2;
      };
      // Step i: x holds its scores, top their largest.
      auto step = [&](int i, float (&x)[kTcKeys]) {
        const int buf = i & 1;
        const bool up = top > m + 8.0f || (m == -INFINITY && top > -INFINITY);
        float f = 1.0f;
        if (up) {
          f = paged_exp2(m - top);
          m = top;
          l *= f;
        }
        if (i > 0 && __any_sync(0xffffffffu, up)) {
          // O up to the last step, once its P V is done
          ok = pv_wait(i - 1);
          if (!ok) return;
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < HD; c += 16) {
            float o[16];
            tc_ld16(o_t + c, o);
            tc_wait_ld();
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              asm volatile("" : "+f"(o[k]));
              o[k] *= f;
            }
            tc_st16(o_t + c, reinterpret_cast<const uint32_t*>(o));
          }
        }
        const float base = m == -INFINITY ? 0.f : m;
        const uint64_t sc2 = f2_all(a.scale_log2), mb2 = f2_all(-base);
        uint64_t sum[2] = {f2_pack(l, 0.f), f2_pack(0.f, 0.f)};
        uint32_t pk[kTcKeys / 2];
#pragma unroll
        for (int k = 0; k < kTcKeys / 2; ++k) {
          const float2 v = f2_unpack(f2_fma(f2_pack(x[2 * k], x[2 * k + 1]), sc2, mb2));
          const float w0 = paged_exp2(v.x), w1 = paged_exp2(v.y);
          sum[k & 1] = f2_add(sum[k & 1], f2_pack(w0, w1));
          pk[k] = Frag<T>::pack(w0, w1);
        }
        tc_st32(s_t + buf * 64, pk);
        const float2 s0 = f2_unpack(sum[0]), s1 = f2_unpack(sum[1]);
        l = (s0.x + s0.y) + (s1.x + s1.y);
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.p_full[t][buf]);
      };
      auto one = [&](int i, auto partial) {
        float x[kTcKeys];
        scores(i, x, partial);
        if (!ok) return;
        landed(x);
        largest(i, x, partial);
        step(i, x);
      };
      for (int i = 0; ok && i < n_full; ++i) one(i, std::false_type());
      for (int i = n_full; ok && i < n; ++i) one(i, std::true_type());
      stage_n += 2 * n;
      if (!ok) break;
      ok = pv_wait(n - 1);
      if (!ok) break;
      pv_n[0] += (n + 1) / 2;
      pv_n[1] += n / 2;
      tc_fence_after();
      // ---- O: to out, or to the workspace and joined by the CTA that is last ----
      const bool whole = p.n_ctas == 1;
      const float inv = see > 0 ? 1.0f / l : 0.f;
      const bool wild = s.wild != 0 && p.tile1 * kTcKeys > see_all;
      const long long tok_g = p.req.q0 + tok;
      const int head = p.h * a.group + row % a.group;
      // A piece's O is stored by fours of columns, the rows of each next to one
      // another: a warp's 32 threads, one row each, store and load 512 bytes in
      // a row.  (With the rows of O end to end a store took 8,700 cycles and a
      // join of 17 pieces 135,000; these take 3,800 and 61,000.)
      float* const part0 = a.partial + t * 128 * kLd;
      const long long slot_f = 256ll * kLd;
      float* part = part0 + paged_slot(blockIdx.x, p.first_cta) * slot_f;
      T* dst = static_cast<T*>(a.out) + tok_g * a.out_stride + (long long)head * HD;
      auto store = [&](int c, const float (&o)[32], float inv) {  // 32 columns of out
#pragma unroll
        for (int k = 0; k < 32; k += 8) {
          uint4 u;
          u.x = Frag<T>::pack(o[k] * inv, o[k + 1] * inv);
          u.y = Frag<T>::pack(o[k + 2] * inv, o[k + 3] * inv);
          u.z = Frag<T>::pack(o[k + 4] * inv, o[k + 5] * inv);
          u.w = Frag<T>::pack(o[k + 6] * inv, o[k + 7] * inv);
          *reinterpret_cast<uint4*>(dst + c + k) = u;
        }
      };
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        float o[32];
        tc_ld32(o_t + c, o);
        tc_wait_ld();
#pragma unroll
        for (int k = 0; k < 32; ++k) asm volatile("" : "+f"(o[k]));
        if (!valid) continue;
        if (l == 0.f) {  // no key of this piece is seen: O may hold 0 * what the others saw
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = 0.f;
        } else if (wild) {
#pragma unroll 1
          for (int k = 0; k < 32; ++k) {
            const bool pos = s.first[0][c + k] < see, neg = s.first[1][c + k] < see, nan = s.first[2][c + k] < see;
            float add = 0.f;
            if (nan || (pos && neg)) add = NAN;
            else if (pos) add = INFINITY;
            else if (neg) add = -INFINITY;
            if (add != 0.f) {
#pragma unroll
              for (int q = 0; q < 32; ++q)
                if (q == k) o[q] += add;
            }
          }
        }
        if (whole) {
          store(c, o, inv);
        } else {
#pragma unroll
          for (int k = 0; k < 32; k += 4)
            *reinterpret_cast<float4*>(part + ((c + k) / 4 * 128 + row) * 4) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
        }
      }
      if (valid && whole && a.lse)
        a.lse[tok_g * a.q_heads + head] = see > 0 ? 0.693147180559945309f * (m + log2f(l)) : -INFINITY;
      if (valid && !whole) *reinterpret_cast<float2*>(part + 128 * HD + 2 * row) = make_float2(m, l);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&s.epi_done[t]);
        if (t == 1) tc_count(&s.tile1_done);
      }
      if (!whole) {
        __threadfence();
        if (t == 0) asm volatile("bar.sync 1, 128;" ::: "memory");
        else asm volatile("bar.sync 2, 128;" ::: "memory");
        if ((tid & 127) == 0) {
          unsigned* ticket = &a.tickets[2 * p.first_cta + t];
          const bool last = atomicAdd(ticket, 1u) == (unsigned)p.n_ctas - 1;
          if (last) *ticket = 0u;
          s.last[t] = last;
        }
        if (t == 0) asm volatile("bar.sync 1, 128;" ::: "memory");
        else asm volatile("bar.sync 2, 128;" ::: "memory");
        if (s.last[t]) {
          __threadfence();
          auto at = [&](int k) { return part0 + paged_slot(p.first_cta + k, p.first_cta) * slot_f; };
          auto stat = [&](int k) { return __ldcg(reinterpret_cast<const float2*>(at(k) + 128 * HD + 2 * row)); };
          float mm = -INFINITY, ll = 0.f;
          if (valid) {
#pragma unroll 8
            for (int k = 0; k < p.n_ctas; ++k) mm = fmaxf(mm, stat(k).x);
            const float b = mm == -INFINITY ? 0.f : mm;
#pragma unroll 4
            for (int k = 0; k < p.n_ctas; ++k) {
              const float2 ml = stat(k);
              ll += ml.y == 0.f ? 0.f : ml.y * paged_exp2(ml.x - b);
            }
            const float iv = see > 0 ? 1.0f / ll : 0.f;
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
              float o[32];
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = 0.f;
#pragma unroll 2
              for (int k = 0; k < p.n_ctas; ++k) {
                const float2 ml = stat(k);
                float4 v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = __ldcg(reinterpret_cast<const float4*>(at(k) + ((c / 4 + j) * 128 + row) * 4));
                const float g = ml.y == 0.f ? 0.f : paged_exp2(ml.x - b);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                  o[4 * j] += v[j].x * g, o[4 * j + 1] += v[j].y * g, o[4 * j + 2] += v[j].z * g, o[4 * j + 3] += v[j].w * g;
              }
              store(c, o, iv);
            }
          }
          if (valid && a.lse)
            a.lse[tok_g * a.q_heads + head] = see > 0 ? 0.693147180559945309f * (mm + log2f(ll)) : -INFINITY;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, kTcTmem);
  }
}

}  // namespace mcpo
