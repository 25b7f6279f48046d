// attn_paged.cuh -- attention of a planned batch over the paged KV cache on the tensor cores.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = 2^(c (s_ij - m_i)),  s_ij = q_i . k_j,
//   c = scale log2 e,
// one pass over the keys: m_i is a running reference maximum and l_i = sum p_ij and the
// unnormalised o_i follow it.  m_i is only moved when a score passes it by more than 8 / c
// (probabilities then stay below 2^8), so the o accumulators are rescaled rarely instead
// of at every tile; any reference gives the same quotient.  s, m, l and o are fp32; p is
// rounded to bf16 as the matrix operand (v is bf16: both operands have one type), which is
// the one rounding besides the output's.
//
// Persistent, warp-specialized, one CTA per SM; the CTA walks the plan's items (paged.cuh),
// longest first, CTA order reversed every other pass so that loads even out.  A tile has
// the query tokens' g heads as rows, so the K / V of a kv head are read once for the whole
// group.  640 threads:
//   warps 0-15      softmax: scores from tensor memory, maximum, p to tensor memory (as the
//                   next product's A operand) and the item's epilogue.  Warpgroups 0, 1 take
//                   accumulator half 0 and 2, 3 half 1 (head_dim 256: all four the one
//                   half); a half's warpgroups share its rows and split the columns, the
//                   rows' maxima meeting in shared memory.  Four such warps per scheduler
//                   instead of two: one alone issues every fourth cycle at best;
//   warp 16         K / V producer: page ids of 32 pieces at a time, one TMA copy per page
//                   piece and 64 columns into the ring, 128-byte swizzle;
//   warp 17         owns the tensor memory; one lane issues all MMAs and commits;
//   warp 18         the next item's description and Q, as soon as the last score product has
//                   read the buffer (warp 19 is idle).
// Shared memory: Q 64 KB, a ring of five 32-KB chunks (128 keys x 128 columns of K or V).
// Tensor memory: scores S0 S1 (128 columns each; the p of 32 keys are written over the first
// half of their scores' columns, which no other warp reads), sums O0 O1.
//
// Three ways through one loop:
//   head_dim 128, many rows: half h has its own 128 rows, S_h, O_h; every K / V chunk is
//     used by both, and half 1's products run while half 0's softmax does;
//   head_dim 128, few rows (up to 128: single tokens) and two key tiles or more: both halves
//     have the same rows and take alternate key tiles, each with its own m, l, O, and leave a
//     part each to be joined;
//   head_dim 256: 128 rows, S0 and S1 take alternate key tiles of one softmax, O0 O1 are
//     the two column halves of one sum.
// In all of them the scores of tile t + 1 (or + 2) are computed while the softmax of tile t
// runs, and the issuing order makes every hazard on S, P and O an in-order one: the product
// that overwrites S_h is issued after the one that reads P_h, and a commit that announces
// S_h covers all earlier products, so the softmax may touch O_h as soon as it holds S_h
// (head_dim 256: after a commit of its own).  The product that adds to O_h is issued only
// when every warp of the half has rescaled its columns of it, or read them out for the last
// item.
//
// Measured (32 query and 8 kv heads of 128): a causal prompt of 16384 1.88 ms = 1170 TFLOP/s in a burst
// (2.13 ms when repeated until the power cap takes the clock down), of 2048 47 us; 8 tokens behind
// 17.9k to 32.8k keys (836 MB) 137-143 us = 5.8-6.1 TB/s.  A unit of 256 rows x 128 keys takes 1.95 us
// (head_dim 256, 128 rows: 1.6-1.7 us) where its products alone take 1.15: a half's scores, maximum,
// probabilities and sums follow one another, two halves fill each other's gaps, and a third set of
// scores has no room in tensor memory.  Around an item 3-4 us, around a call (with the join) 9-10 us.
//
// Stale memory: a K / V row at or past the request's length (or before the window) may hold
// anything.  Scores are masked by selection, and V rows outside [klo, len) are zeroed in
// shared memory before their product, since 0 * NaN is NaN.  (V at positions in between has to be
// finite: one that is not reaches that column of every row of the tile.)
//
// Every mbarrier wait is bounded by %globaltimer; one that runs out sets bit 1 of *error
// and an abort flag that every other wait checks.  Before the CTA gives up shared or
// tensor memory it waits (2 s bound) for the copies and MMAs in flight; bit 2 means that
// this ran out too and the tensor memory was kept.
#pragma once

#include <cuda.h>

#include <climits>

#include "paged.cuh"

namespace spark {
namespace paged {
namespace tc {

constexpr int kThreads = 640;
constexpr int kSoftmaxWarps = 16;
constexpr int kProducerWarp = 16, kMmaWarp = 17, kQWarp = 18;
constexpr int kStages = 5;
constexpr int kChunk = 32 * 1024;  // 128 keys x 128 columns
constexpr int kSub = 16 * 1024;    // 128 keys x 64 columns (one swizzle row of 128 bytes)
constexpr int kOffRing = 64 * 1024;
constexpr int kOffX = kOffRing + kStages * kChunk;  // row values shared by a half's warpgroups: [4][128]
constexpr int kOffBar = kOffX + 4 * 128 * 4;
constexpr int kBarFull = 0, kBarEmpty = kBarFull + kStages, kBarQFull = kBarEmpty + kStages,
              kBarQEmpty = kBarQFull + 2, kBarS = kBarQEmpty + 2, kBarP = kBarS + 2, kBarP2 = kBarP + 2,
              kBarO = kBarP2 + 2, kBarPV = kBarO + 2, kBarX = kBarPV + 2, kBarDrain = kBarX + 8,
              kNumBars = kBarDrain + 1;
constexpr int kOffMisc = kOffBar + 8 * kNumBars;  // tensor-memory base, abort flag, drained flag
constexpr int kOffItem = (kOffMisc + 16 + 15) / 16 * 16;  // two items and their kv heads, 64 bytes each
constexpr int kSmemBytes = kOffItem + 2 * 64;
constexpr int kTmemCols = 512;
constexpr int kColS = 0, kColO = 256;
constexpr unsigned long long kWaitNs = 500ull * 1000 * 1000;
constexpr unsigned long long kDrainNs = 2000ull * 1000 * 1000;
static_assert(kSmemBytes <= 227 * 1024, "shared memory");

// instruction descriptors (kind::f16): fp32 D, bf16 A and B, N = 128, M = 128; scores: both
// operands K-major; sums: B (= V, keys x columns) N-major (bit 16)
constexpr uint32_t kIdescS = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
constexpr uint32_t kIdescO = kIdescS | (1u << 16);

// 128-byte-swizzled operand tiles.  K-major (Q, K): 8-row groups 1024 bytes apart, 16
// columns = 32 bytes along the row.  N-major (V): 64-column blocks kSub apart (leading
// offset), 8-key groups 1024 bytes apart, 16 keys = 2048 bytes.
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) |
         (2ull << 61);
}
__device__ __forceinline__ uint64_t desc_v(uint32_t addr) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(kSub >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}

__device__ __forceinline__ unsigned long long now_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}

__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float ldsf(uint32_t addr) { return __uint_as_float(lds32(addr)); }
__device__ __forceinline__ void stsf(uint32_t addr, float v) {
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

// Wait for the phase of `parity`; false: limit_ns ran out or another role gave up (abort: the
// shared address of its flag, or 0).  The
// clock and the flag are looked at every 16th try only.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, unsigned long long limit_ns,
                                         uint32_t abort) {
  unsigned long long t0 = 0;
  for (uint32_t spin = 1;; spin++) {
    uint32_t done;
    asm volatile(
        "{.reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p;}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return true;
    if ((spin & 15u) == 0) {
      if (abort && lds32(abort)) return false;
      const unsigned long long t = now_ns();
      if (t0 == 0) t0 = t;
      else if (t - t0 >= limit_ns) return false;
    }
  }
}
// one look
__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{.reg .pred p; mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p;}"
               : "=r"(done)
               : "r"(bar), "r"(parity)
               : "memory");
  return done != 0;
}
__device__ __forceinline__ void bar_init(uint32_t bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::
          "r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accum) {
  asm volatile(
      "{.reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;}" ::"r"(d), "l"(a),
      "l"(b), "r"(id), "r"(accum)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t accum) {
  asm volatile(
      "{.reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;}" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"(accum)
      : "memory");
}
// true in one lane of the (converged) warp, the same one every time
__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile("{.reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p;}" : "=r"(e));
  return e != 0;
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of this warp's 32 lanes (the caller waits)
__device__ __forceinline__ void tm_load32(uint32_t addr, float* v) {
  uint32_t* u = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
        "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
        "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(addr));
}
// the wait ties the registers, so that no use moves above it
__device__ __forceinline__ void tm_wait32(float* v) {
  uint32_t* u = reinterpret_cast<uint32_t*>(v);
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(u[0]), "+r"(u[1]), "+r"(u[2]), "+r"(u[3]), "+r"(u[4]), "+r"(u[5]), "+r"(u[6]), "+r"(u[7]),
                 "+r"(u[8]), "+r"(u[9]), "+r"(u[10]), "+r"(u[11]), "+r"(u[12]), "+r"(u[13]), "+r"(u[14]),
                 "+r"(u[15]), "+r"(u[16]), "+r"(u[17]), "+r"(u[18]), "+r"(u[19]), "+r"(u[20]), "+r"(u[21]),
                 "+r"(u[22]), "+r"(u[23]), "+r"(u[24]), "+r"(u[25]), "+r"(u[26]), "+r"(u[27]), "+r"(u[28]),
                 "+r"(u[29]), "+r"(u[30]), "+r"(u[31])
               :
               : "memory");
}
__device__ __forceinline__ void tm_load16(uint32_t addr, float* v) {
  uint32_t* u = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(u[0]), "+r"(u[1]), "+r"(u[2]), "+r"(u[3]), "+r"(u[4]), "+r"(u[5]), "+r"(u[6]), "+r"(u[7]),
                 "+r"(u[8]), "+r"(u[9]), "+r"(u[10]), "+r"(u[11]), "+r"(u[12]), "+r"(u[13]), "+r"(u[14]),
                 "+r"(u[15])
               :
               : "memory");
}
__device__ __forceinline__ void tm_store16(uint32_t addr, const uint32_t* u) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(
          u[0]),
      "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]), "r"(u[10]),
      "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(addr)
      : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// p = 2^(s c + neg) of 16 scores: sums in fp32, the bf16 pairs to tensor memory.  Every
// exponential is the special-function unit's (a relative error of 2^-22, a NaN stays one, an
// infinite difference is 0 or infinite).
__device__ __forceinline__ void probs16(const float* s, u64 c2, u64 neg2, u64 (&sum)[2], uint32_t addr) {
  uint32_t pk[8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    float x, y;
    unpack2(fma2(pack2(s[2 * i], s[2 * i + 1]), c2, neg2), x, y);
    x = ex2(x);
    y = ex2(y);
    sum[i & 1] = add2(sum[i & 1], pack2(x, y));
    pk[i] = pack_bf16(x, y);
  }
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(pk[0]), "r"(pk[1]),
               "r"(pk[2]), "r"(pk[3]), "r"(pk[4]), "r"(pk[5]), "r"(pk[6]), "r"(pk[7]), "r"(addr)
               : "memory");
}

// 32 bytes (wide) or two times 16 to global memory
__device__ __forceinline__ void store32(void* dst, const uint32_t* v, bool wide) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(dst)[0] = make_uint4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<uint4*>(dst)[1] = make_uint4(v[4], v[5], v[6], v[7]);
  }
}
__device__ __forceinline__ int warp_min_i(int v) { return __reduce_min_sync(0xffffffffu, v); }

// The CTA's i-th work index (item x kv head): forward and backward through the CTAs in
// turn, so that a CTA that got a long item of one pass gets a short one of the next.
__device__ __forceinline__ uint32_t work_index(uint32_t pass) {
  return pass * gridDim.x + ((pass & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
}

struct TcArgs {
  AttnArgs a;
  int piece;  // keys per TMA copy: the largest power of two up to 128 that divides a page
  bool wide;  // out and its strides are multiples of 32 bytes
  unsigned long long limit_ns;
};

// Positions of K tile t and V tile t of n in the item's sequence of K / V tiles: d K tiles
// lead, then V_t, K_{t+d} alternate.
__device__ __forceinline__ int k_index(int t, int d) { return t < d ? t : 2 * t - d + 1; }
__device__ __forceinline__ int v_index(int t, int n, int d) {
  const int lead = d < n ? d : n, past = t - (n - lead);
  return lead + 2 * t - (past > 0 ? past : 0);
}

// Tensor maps: tmq over q [tokens][nq][D], box {64, g, 128 / g}; tmk, tmv over the caches as
// rows of D, box {64, piece}; all with the 128-byte swizzle.
template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    attn_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                const __grid_constant__ CUtensorMap tmv, const __grid_constant__ TcArgs args) {
  constexpr int NC = D / 128;  // chunks per K or V tile
  const AttnArgs& p = args.a;
  const unsigned long long limit_ns = args.limit_ns;
  // (swizzled tiles want 1024-byte alignment; there is no room for slack, and no static
  // shared memory in front: checked once, all threads together)
  extern __shared__ __align__(1024) unsigned char gbase[];
  const uint32_t base = (uint32_t)__cvta_generic_to_shared(gbase);
  if (base & 1023u) {
    if (threadIdx.x == 0) atomicOr(p.error, 1);
    return;
  }
  const uint32_t bars = base + kOffBar;
  const uint32_t tslot = base + kOffMisc;
  const uint32_t abort_flag = base + kOffMisc + 4;
  volatile int* drained_flag = reinterpret_cast<volatile int*>(gbase + kOffMisc + 8);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  auto bar = [&](int i) { return bars + 8u * (uint32_t)i; };
  auto fail = [&]() {
    atomicOr(p.error, 1);
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(abort_flag), "r"(1) : "memory");
  };

  if (tid == 0) {
    for (int s = 0; s < kStages; s++) {
      bar_init(bar(kBarFull + s), 1);
      bar_init(bar(kBarEmpty + s), 1);
    }
    for (int h = 0; h < 2; h++) {
      bar_init(bar(kBarQFull + h), 1);
      bar_init(bar(kBarQEmpty + h), 1 + kSoftmaxWarps);  // the last score product's commit, the softmax warps
      bar_init(bar(kBarS + h), 1);
      bar_init(bar(kBarP + h), D == 128 ? 8 : 16);
      bar_init(bar(kBarP2 + h), 8);
      bar_init(bar(kBarO + h), 1);
      bar_init(bar(kBarPV + h), 1);
    }
    for (int i = 0; i < 8; i++) bar_init(bar(kBarX + i), D == 128 ? 2 : 4);
    bar_init(bar(kBarDrain), 1);
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(abort_flag), "r"(0) : "memory");
    *drained_flag = 1;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tslot), "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tslot) : "memory");
  pdl_wait();
  const Header* hdr = reinterpret_cast<const Header*>(p.plan);
  const Item* items = reinterpret_cast<const Item*>(p.plan + p.lay.items);
  const bool fits = plan_fits<D>(p, hdr);
  if (!fits && blockIdx.x == 0 && tid == 0) atomicOr(p.error, kBadPlan);
  const uint32_t nwork = fits ? (uint32_t)hdr->items * (uint32_t)p.nkv : 0;
  const int g = p.nq / p.nkv;

  if (warp >= kSoftmaxWarps) {
    if (warp == kProducerWarp) {
      // ---------------------------------------------------------------- K / V producer
      uint32_t ring = 0;
      bool ok = true;
      const int pr = args.piece, pp = kKeyTile / pr;
      const int64_t rows_total = p.num_blocks * p.nkv * p.bs;
      for (uint32_t pass = 0; ok; pass++) {
        const uint32_t w = work_index(pass);
        if (pass && w >= nwork) break;
        const Item it = items[w / p.nkv];  // (the first one's load does not wait for the header)
        if (w >= nwork) break;
        const int kvh = (int)(w % p.nkv);
        const int n = it.nkt;
        if (n == 0) continue;
        const int d = (D == 256 || (it.flags & kFlagFew)) ? 2 : 1;
        // row of the cache that piece x (of pr keys, counted from key0) starts at; -1: the
        // piece holds no key of the item and is not read
        auto piece_row = [&](int x) -> int {
          const int key = it.key0 + x * pr;
          if (x >= n * pp || key >= it.len || key + pr <= it.klo) return -1;
          const int pg = key / p.bs;
          const int id =
              pg < p.table_width && it.req < p.table_rows ? __ldg(p.table + it.req * p.table_stride + pg) : -1;
          if (id < 0 || id >= p.num_blocks) {
            atomicOr(p.error, kBadPage);
            return (int)rows_total;  // outside the map: zeros
          }
          return (int)(((int64_t)id * p.nkv + kvh) * p.bs + (key - pg * p.bs));
        };
        int win[2] = {-1, -1}, rows[2] = {-1, -1};  // 32 pieces each for K and V
        auto load = [&](int v, int t) -> bool {
          const int x0 = t * pp;
          if (win[v] != (x0 >> 5)) {
            win[v] = x0 >> 5;
            rows[v] = piece_row((x0 & ~31) + lane);
          }
          const int row = __shfl_sync(0xffffffffu, rows[v], (x0 & 31) + (lane & (pp - 1)));
          const bool mine = lane < pp && row >= 0;
          const uint32_t live = __popc(__ballot_sync(0xffffffffu, mine));
          const CUtensorMap* map = v ? &tmv : &tmk;
#pragma unroll
          for (int c = 0; c < NC; c++) {
            const uint32_t s = ring % kStages;
            const bool free_ok = bar_wait(bar(kBarEmpty + s), ((ring / kStages) & 1) ^ 1, limit_ns, abort_flag);
            if (!__all_sync(0xffffffffu, free_ok)) return false;
            if (lane == 0) bar_expect_tx(bar(kBarFull + s), live * (uint32_t)(pr * 256));
            __syncwarp();
            if (mine) {
              const uint32_t dst = base + kOffRing + s * kChunk + (uint32_t)(lane * pr * 128);
              tma_2d(dst, map, c * 128, row, bar(kBarFull + s));
              tma_2d(dst + kSub, map, c * 128 + 64, row, bar(kBarFull + s));
            }
            ring++;
          }
          return true;
        };
        for (int t = 0; t < d && t < n && ok; t++) ok = load(0, t);
        for (int t = 0; t < n && ok; t++) {
          ok = load(1, t);
          if (ok && t + d < n) ok = load(0, t + d);
        }
      }
      if (!ok && lane == 0) fail();
      // every issued copy lands before the CTA can give its shared memory up
      bool drained = true;
      for (uint32_t i = ring > (uint32_t)kStages ? ring - kStages : 0; i < ring; i++)
        drained &= bar_wait(bar(kBarFull + i % kStages), (i / kStages) & 1, kDrainNs, 0);
      if (!drained && lane == 0) {
        atomicOr(p.error, 2);
        *drained_flag = 0;
      }
      __syncwarp();
    } else if (warp == kQWarp) {
      // ---------------------------------------------------------------- Q
      if (lane == 0) {
        uint32_t qi = 0, loaded = 0;  // items described; slots whose latest phase is a load of Q
        bool ok = true, prev_whole = false;
        const uint32_t box = (uint32_t)(g * p.lay.half_tok) * 128u;
        // item i is over with its slot (i & 1): read by all, its score products done
        auto over = [&](uint32_t i) { return bar_wait(bar(kBarQEmpty + (i & 1)), (i >> 1) & 1, limit_ns, abort_flag); };
        for (uint32_t pass = 0;; pass++, qi++) {
          const uint32_t w = work_index(pass);
          Item it;
          int kvh = 0;
          if (!pass || w < nwork) {
            it = items[w / p.nkv];
            kvh = (int)(w % p.nkv);
          }
          const bool have = w < nwork;
          // Items that fill the Q buffer wait for the one before; those of few rows take a
          // half of it in turn
          const bool whole = have && it.nkt > 0 && (D == 256 || !(it.flags & kFlagFew));
          if ((qi >= 2 && !over(qi - 2)) || (qi >= 1 && (whole || prev_whole) && !over(qi - 1))) {
            ok = false;
            break;
          }
          prev_whole = whole;
          const uint32_t q = qi & 1, full = bar(kBarQFull + q);
          loaded &= ~(1u << q);  // (the slot's last load was used: its item is over)
          Item* slot = reinterpret_cast<Item*>(gbase + kOffItem + 64 * q);
          if (!have) {
            slot->nkt = -1;
            bar_arrive(full);
            break;
          }
          *slot = it;
          *reinterpret_cast<int*>(gbase + kOffItem + 64 * q + sizeof(Item)) = kvh;
          if (it.nkt == 0) {
            bar_arrive(full);
            continue;
          }
          const int halves = D == 128 && whole ? 2 : 1;
          const uint32_t dst = base + (whole ? 0u : q * kChunk);
          bar_expect_tx(full, box * (uint32_t)(halves * (D / 64)));
          for (int h = 0; h < halves; h++)
            for (int c = 0; c < D / 64; c++)
              tma_3d(dst + (uint32_t)(h * kChunk + c * kSub), &tmq, c * 64, kvh * g, it.tok0 + h * p.lay.half_tok, full);
          loaded |= 1u << q;
        }
        if (!ok) fail();
        // a load still in flight is its slot's latest phase, that of the last item with this
        // parity below qi (an older phase could not be told from a newer one)
        for (uint32_t q = 0; q < 2; q++) {
          if (!(loaded >> q & 1)) continue;
          const uint32_t i = qi - 1 - ((qi - 1 - q) & 1);
          if (!bar_wait(bar(kBarQFull + q), (i >> 1) & 1, kDrainNs, 0)) {
            atomicOr(p.error, 2);
            *drained_flag = 0;
          }
        }
      }
      __syncwarp();
    } else if (warp == kMmaWarp) {
      // ---------------------------------------------------------------- MMA issuer
      // (the whole warp walks the loop, so that addresses and descriptors are warp-uniform
      // values in uniform registers; one lane, always the same, issues.  Issued from a
      // one-lane branch instead, an MMA took about 80 cycles to hand over.)
      {
        uint32_t qi = 0, np[2] = {0, 0};
        bool ok = true;
        // head_dim 256: mostly what is waited for is done, and one look at all of it together costs
        // 200 cycles in which the tensor pipe runs dry, a look at each as much again (one unit
        // 1.87 -> 1.68 us).  At head_dim 128 probabilities are mostly waited for: looks in front of
        // the wait cost 2%.
        auto ready = [&](int i, uint32_t parity) -> bool { return __all_sync(0xffffffffu, bar_test(bar(i), parity)); };
        auto wait = [&](int i, uint32_t parity) -> bool {
          return (D == 256 && ready(i, parity)) || __all_sync(0xffffffffu, bar_wait(bar(i), parity, limit_ns, abort_flag));
        };
        // A place in the ring; chunks are used in ring order, but for the scores of a next item
        // that are issued early
        struct Pos {
          uint32_t s, ph;
        };
        Pos cur{0, 0};
        auto step = [](Pos r, int k) -> Pos {  // (k < kStages)
          r.s += (uint32_t)k;
          if (r.s >= (uint32_t)kStages) {
            r.s -= kStages;
            r.ph ^= 1;
          }
          return r;
        };
        // the tile at r is in shared memory and phase `parity` of barrier i (-1: none) is over
        auto ready_tile = [&](Pos r, int i, uint32_t parity) -> bool {
          const Pos x = step(r, NC - 1);
          const bool a = bar_test(bar(kBarFull + r.s), r.ph), b = NC == 1 || bar_test(bar(kBarFull + x.s), x.ph);
          return __all_sync(0xffffffffu, a && b && (i < 0 || bar_test(bar(i), parity)));
        };
        auto full_tile = [&](Pos r) -> bool {
          if (ready_tile(r, -1, 0)) return true;
          bool f = wait(kBarFull + r.s, r.ph);
          if (NC == 2) f = f && wait(kBarFull + step(r, 1).s, step(r, 1).ph);
          return f;
        };
        auto stage = [&](Pos r) { return base + kOffRing + r.s * kChunk; };
        // S_h = Q_q K^T of the tile at r; then, all announced from the same lane's turn, the
        // scores, the tile's place (`done`) and a barrier of the caller's (or -1)
        auto scores = [&](int h, int q, Pos r, bool done, int also) {
#pragma unroll
          for (int c = 0; c < NC; c++) {
            const uint64_t kd = desc_k(stage(step(r, c))), qd = desc_k(base + (uint32_t)(q * kChunk + c * kChunk));
            if (elect_one()) {
#pragma unroll
              for (int j = 0; j < 8; j++) {
                const uint32_t off = (uint32_t)((j >> 2) * (kSub >> 4) + 2 * (j & 3));
                mma_ss(tmem + kColS + h * 128, qd + off, kd + off, kIdescS, (c | j) != 0);
              }
              if (c == NC - 1) {
                commit(bar(kBarS + h));
                if (done) {
                  commit(bar(kBarEmpty + r.s));
                  if (NC == 2) commit(bar(kBarEmpty + step(r, 1).s));
                }
                if (also >= 0) commit(bar(also));
              }
            }
            __syncwarp();
          }
        };
        // O += P_h V of the tile at r (`fresh`: V has not been waited for), in two steps: the
        // first 64 keys' probabilities are multiplied while the others are still computed.
        // `seen`: in, whether to look for the tile at `next` on the way; out, whether it is there.
        auto sums = [&](int h, int o, Pos r, uint32_t accum, bool fresh, bool done, int also, bool& seen,
                        Pos next) -> bool {
#pragma unroll
          for (int k = 0; k < 2; k++) {
            const int pb = (k ? kBarP2 : kBarP) + h;
            const uint32_t pp = np[h] & 1;
            if (k == 0 && fresh) {
              if (!ready_tile(r, pb, pp) && !(full_tile(r) && wait(pb, pp))) return false;
            } else if (k == 1 && seen) {
              seen = ready_tile(next, pb, pp);
              if (!seen && !wait(pb, pp)) return false;
            } else if (!wait(pb, pp)) {
              return false;
            }
            fence_after();
#pragma unroll
            for (int c = 0; c < NC; c++) {
              const uint64_t vd = desc_v(stage(step(r, c)));
              if (elect_one()) {
#pragma unroll
                for (int j = 4 * k; j < 4 * k + 4; j++)
                  mma_ts(tmem + kColO + (o + c) * 128, tmem + kColS + h * 128 + 32 * (j >> 1) + 8 * (j & 1),
                         vd + j * (2048 >> 4), kIdescO, accum | (j != 0));
                if (k == 1 && c == NC - 1) {
                  if (D == 256) commit(bar(kBarPV + h));
                  if (done) {
                    commit(bar(kBarEmpty + r.s));
                    if (NC == 2) commit(bar(kBarEmpty + step(r, 1).s));
                  }
                  if (also >= 0) commit(bar(also));
                }
              }
              __syncwarp();
            }
          }
          np[h]++;
          return true;
        };
        auto announce = [&](int i) {
          if (elect_one()) commit(bar(i));
          __syncwarp();
        };
        // tiles and mode of the item in slot i & 1
        auto describe = [&](uint32_t i, int& tiles, bool& alternate) {
          const Item* slot = reinterpret_cast<const Item*>(gbase + kOffItem + 64 * (i & 1));
          tiles = __shfl_sync(0xffffffffu, slot->nkt, 0);
          alternate = D == 256 || (__shfl_sync(0xffffffffu, slot->flags, 0) & kFlagFew);
        };
        // Alternating tiles: the scores of tile t of item i (its K at r), into buffer b
        auto alt_scores = [&](uint32_t i, int t, int n, int b, Pos r) {
          fence_after();
          scores(b, D == 256 ? 0 : (int)(i & 1), r, true, t + 1 == n ? kBarQEmpty + (int)(i & 1) : -1);
        };
        bool first0 = false;  // half 0's first scores of this item were issued behind the last one's
        int early = 0;      // score tiles of this item that were issued behind the last one's
        uint32_t par = 0;   // score buffer of the item's first alternating tile
        // What was read of the next item ahead of its turn is kept: once its scores are issued
        // the slot may move on, and its phase could no longer be told from the next but one.
        bool known = false, next_alt = false;
        int next_n = 0;
        for (;; qi++) {
          int n = next_n;
          bool alternate = next_alt;
          if (!known) {
            if (!(ok = wait(kBarQFull + (qi & 1), (qi >> 1) & 1))) break;
            describe(qi, n, alternate);
          }
          known = false;
          if (n < 0) break;
          if (n == 0) {
            if (lane == 0) bar_arrive(bar(kBarQEmpty + (qi & 1)));
            continue;
          }
          if (!alternate) {
            if (!(ok = full_tile(cur))) break;
            fence_after();
            if (!first0) scores(0, 0, cur, false, -1);
            first0 = false;
            scores(1, 1, cur, true, n == 1 ? kBarQEmpty + (int)(qi & 1) : -1);
            cur = step(cur, 1);
            bool unseen = false;  // (no look for the next K on the way: see wait)
            for (int t = 0; t + 1 < n && ok; t++) {
              const Pos rv = cur, rk = step(cur, 1);
              for (int h = 0; h < 2; h++) {
                if (!(ok = sums(h, h, rv, t > 0, h == 0, h == 1, -1, unseen, rk))) break;
                if (h == 0) {
                  if (!(ok = full_tile(rk))) break;
                  fence_after();
                }
                scores(h, h, rk, h == 1, h == 1 && t + 2 == n ? kBarQEmpty + (int)(qi & 1) : -1);
              }
              cur = step(cur, 2);
            }
            if (!ok) break;
            const Pos rv = cur;
            cur = step(cur, 1);
            if (!(ok = sums(0, 0, rv, n > 1, true, false, kBarO, unseen, cur))) break;
            // half 0's first scores of the next item, if its Q and K are there already, so that
            // they are done when the half's warps have written this one's rows (1% of a prompt
            // of 2048; inside the loop above the same look cost the other tiles 2%)
            if (ready(kBarQFull + ((qi + 1) & 1), ((qi + 1) >> 1) & 1)) {
              describe(qi + 1, next_n, next_alt);
              known = true;
              if (!next_alt && next_n > 0 && ready_tile(cur, -1, 0)) {
                fence_after();
                scores(0, 0, cur, false, -1);
                first0 = true;
              }
            }
            if (!(ok = sums(1, 1, rv, n > 1, false, true, kBarO + 1, unseen, cur))) break;
          } else {
            for (int t = early; t < 2 && t < n && ok; t++) {
              const Pos rk = step(cur, NC * t);
              if (!(ok = full_tile(rk))) break;
              alt_scores(qi, t, n, (par + t) & 1, rk);
            }
            if (!ok) break;
            early = 0;
            cur = step(cur, NC * (n < 2 ? n : 2));
            for (int t = 0; t < n; t++) {
              const int b = (par + t) & 1;
              const bool end = D == 256 ? t + 1 == n : t + 2 >= n;  // of this buffer's sums
              bool seen = t + 2 < n;
              if (!(ok = sums(b, D == 128 ? b : 0, cur, D == 128 ? t > 1 : t > 0, true, true,
                              end ? kBarO + (D == 128 ? b : 0) : -1, seen, step(cur, NC))))
                break;
              cur = step(cur, NC);
              if (t + 2 < n) {
                if (!(ok = seen || full_tile(cur))) break;
                alt_scores(qi, t + 2, n, b, cur);
                cur = step(cur, NC);
                continue;
              }
              // The next item's first scores fill the gap while this one's last softmax
              // runs, if its Q and K are there already (nothing is waited for).
              if (!known && ready(kBarQFull + ((qi + 1) & 1), ((qi + 1) >> 1) & 1)) {
                describe(qi + 1, next_n, next_alt);
                known = true;
              }
              for (; known && next_alt && early < t + 3 - n && early < next_n; early++) {
                const Pos rk = step(step(cur, NC * (n - 1 - t)), NC * early);  // behind this item's last V
                if (!ready_tile(rk, -1, 0)) break;
                alt_scores(qi + 1, early, next_n, (par + n + early) & 1, rk);
              }
            }
            if (!ok) break;
            par = (par + n) & 1;
          }
        }
        if (!ok && lane == 0) fail();
        announce(kBarDrain);  // tracks every MMA issued before it
        if (!bar_wait(bar(kBarDrain), 0, kDrainNs, 0) && lane == 0) {
          atomicOr(p.error, 2);
          *drained_flag = 0;
        }
      }
      __syncwarp();
    }
  } else {
    // ---------------------------------------------------------------- softmax and epilogue
    // SP warpgroups share the rows of a half (a thread of each owns the same row), 128 / SP
    // score columns and 64 sum columns each
    constexpr int SP = D == 128 ? 2 : 4, NQ = 4 / SP;
    const int wg = warp >> 2, h = D == 128 ? wg >> 1 : 0, sp = D == 128 ? wg & 1 : wg, r = tid & 127;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const int* lens = reinterpret_cast<const int*>(p.plan + p.lay.lens);
    const float c = p.scale * kLog2e;
    const uint32_t xs = base + kOffX + (uint32_t)(h * SP * 128 + r) * 4;  // [warpgroup][row]
    const int xbar = kBarX + h * 4 + (warp & 3);
    uint32_t ns[2] = {0, 0}, no = 0, npv[2] = {0, 0}, ring0 = 0, qi = 0, nx = 0, par = 0;
    bool ok = true, unread = false;
    auto wait = [&](int i, uint32_t parity) {
      return __all_sync(0xffffffffu, bar_wait(bar(i), parity, limit_ns, abort_flag));
    };
    // Warpgroup j's value of this row is at xs + 512 j.  The next values may be written over
    // these once all have read them.  head_dim 128, maxima: they follow the next scores of the
    // same buffer, which every partner's probabilities precede.  head_dim 256, whose next
    // scores are in the other buffer and may be there already, and an item's last exchange:
    // each warp reports that it has read (unread: that report is still to be awaited).
    auto exchange = [&](float v) -> bool {
      if (unread) {
        if (!wait(xbar, nx++ & 1)) return false;
        unread = false;
      }
      stsf(xs + 512 * sp, v);
      __syncwarp();
      if (lane == 0) bar_arrive(bar(xbar));
      return wait(xbar, nx++ & 1);
    };
    const int row_tok = r / g, head_row = r - row_tok * g;  // this thread's row: token of the half, head of the group
    for (;; qi++) {
      const int q = qi & 1;
      if (!(ok = wait(kBarQFull + q, (qi >> 1) & 1))) break;
      const Item it = *reinterpret_cast<const Item*>(gbase + kOffItem + 64 * q);
      const int kvh = *reinterpret_cast<const int*>(gbase + kOffItem + 64 * q + sizeof(Item));
      const int n = it.nkt;
      if (n < 0) break;
      __syncwarp();
      if (lane == 0) bar_arrive(bar(kBarQEmpty + q));  // this warp is done with the slot
      const bool few = D == 128 && (it.flags & kFlagFew), alt = D == 256 || few;
      // alternating tiles: the item's tile t is in score buffer (par + t) & 1; few rows: this
      // half has the tiles of its own buffer, t0, t0 + 2 ..
      const int t0 = few ? (int)(h ^ par) : 0;
      const int local = row_tok + (D == 128 && !few ? h * p.lay.half_tok : 0);  // token of the item
      const bool valid = r < g * p.lay.half_tok && local < it.ntok && it.tok0 + local < p.tokens;
      const int2 kk = valid ? row_keys(it, lens, p.window, local) : make_int2(0, 0);
      const bool any_valid = __any_sync(0xffffffffu, valid);
      // keys that some row (lo0, hi1) / every row (lo1, hi0) of the warp sees
      const int lo0 = warp_min_i(valid ? kk.x : INT_MAX), lo1 = -warp_min_i(valid ? -kk.x : INT_MAX);
      const int hi0 = warp_min_i(valid ? kk.y : INT_MAX), hi1 = -warp_min_i(valid ? -kk.y : INT_MAX);
      // head_dim 256: the sums of tile t are done.  The two score buffers' tiles have a
      // barrier each: a parity tells a phase from its neighbours only, and when the sums of
      // tile t are asked for (by the softmax of tile t + 1) those of tile t - 2 were announced
      // before the scores of tile t, and those of tile t + 2 cannot have begun.
      auto sums_done = [&](int t) {
        const uint32_t b = (par + t) & 1;
        return wait(kBarPV + b, (npv[b] + (uint32_t)(t >> 1)) & 1);
      };
      // (rows beyond the item's have no say in when the reference moves: with m at infinity
      // it never does for them, and what lies in them does not show in the others' rounding)
      float m = valid ? -INFINITY : INFINITY, l = 0.0f;
      const uint32_t ob = lanes + kColO + (D == 128 ? h * 128 : 0) + sp * 64;
      for (int t = t0; t < n; t += few ? 2 : 1) {
        const int b = D == 256 ? (int)((par + t) & 1) : h;  // score buffer
        const bool first = few ? t < 2 : t == 0;
        const uint32_t sb = lanes + kColS + b * 128;
        if (!(ok = wait(kBarS + b, ns[b]++ & 1))) break;
        fence_after();
        const int k0 = it.key0 + t * kKeyTile;
        // V rows that hold no key of the request (stale) are zeroed before their product
        const int tail = it.len - k0, front = it.klo - k0;
        if ((tail < kKeyTile || front > 0) && (alt || h == 0)) {
          if (D == 256 && t > 0) {  // (then the ring position read below is this tile's)
            if (!(ok = sums_done(t - 1))) break;
          }
          const uint32_t rv = ring0 + (uint32_t)(NC * v_index(t, n, alt ? 2 : 1));
          const int z0 = front > 0 ? front : 0, z1 = tail < kKeyTile ? tail : kKeyTile;
          for (int cc = 0; cc < NC && ok; cc++) {
            const uint32_t st = (rv + cc) % kStages;
            if (!(ok = wait(kBarFull + st, ((rv + cc) / kStages) & 1))) break;
            unsigned char* vb = gbase + kOffRing + st * kChunk;
            for (int i = sp * 128 + r; i < 128 * 16; i += SP * 128) {  // (row, 16 bytes of its two swizzle rows)
              const int row = i >> 4, q = i & 15;
              if (row < z0 || row >= z1)
                *reinterpret_cast<uint4*>(vb + (q >> 3) * kSub + row * 128 + (q & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
          }
          if (!ok) break;
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        // this warp's share of the first (k = 0) or last 64 keys' probabilities is written
        // (head_dim 256: warpgroups 2 and 3 have no share of the first, but that product adds to
        // all columns of O and reads V rows that they zeroed: they announce k = 0 too, once
        // they are done with both)
        auto announce = [&](int k) {
          wait_st();
          fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive(bar((k ? kBarP2 : kBarP) + b));
        };
        if (any_valid && k0 < hi1 && k0 + kKeyTile > lo0) {
          const bool edge = k0 < lo1 || k0 + kKeyTile > hi0;  // some row sees a part of the tile only
          const int col0 = kk.x - k0 - 32 * sp, cols = kk.y - kk.x;
          float s[32];
          auto load = [&](int q) {
            tm_load32(sb + 64 * q + 32 * sp, s);
            tm_wait32(s);
            if (edge) {
#pragma unroll
              for (int i = 0; i < 32; i++)
                s[i] = cols > 0 && (uint32_t)(i + 64 * q - col0) < (uint32_t)cols ? s[i] : -INFINITY;
            }
          };
          float mn = -INFINITY;
#pragma unroll
          for (int q = NQ - 1; q >= 0; q--) {  // (the first 32 scores stay for the second pass)
            load(q);
            float a = max3(mn, s[0], s[1]), b = max3(s[2], s[3], s[4]);
#pragma unroll
            for (int i = 5; i < 29; i += 4) {
              a = max3(a, s[i], s[i + 1]);
              b = max3(b, s[i + 2], s[i + 3]);
            }
            mn = max3(fmaxf(a, s[29]), fmaxf(b, s[30]), s[31]);
          }
          if (!(ok = exchange(mn))) break;
#pragma unroll
          for (int j = 0; j < SP; j++) mn = fmaxf(mn, ldsf(xs + 512 * j));
          if (D == 256) {
            __syncwarp();
            if (lane == 0) bar_arrive(bar(xbar));
            unread = true;
          }
          mn = fmaxf(m, mn);
          if (first) {
            m = mn;
          } else if (__any_sync(0xffffffffu, (mn - m) * c > 8.0f)) {
            const float f = mn == -INFINITY ? 1.0f : ex2((m - mn) * c);
            m = mn;
            l *= f;
            if (D == 256) {  // the product before this one has to be done with O
              if (!(ok = sums_done(t - 1))) break;
              fence_after();
            }
#pragma unroll 1
            for (int i = 0; i < 4; i++) {
              float o[16];
              tm_load16(ob + 16 * i, o);
#pragma unroll
              for (int j = 0; j < 16; j++) o[j] *= f;
              tm_store16(ob + 16 * i, reinterpret_cast<const uint32_t*>(o));
            }
          }
          if (D == 256 && sp >= 2) announce(0);
          const float neg = m == -INFINITY ? 0.0f : -m * c;
          const u64 neg2 = pack2(neg, neg), c2 = pack2(c, c);
          u64 sum[2] = {0, 0};
          // (not unrolled: both halves' probabilities side by side spill 28 bytes; packed prompts 184.6
          // -> 182.6, long shared prefix 90.4 -> 88.2, 8 x 2048 prefix 15.3 -> 14.9 us)
#pragma unroll 1
          for (int q = 0; q < NQ; q++) {
            if (q > 0) load(q);
            const uint32_t pb = sb + 64 * q + 32 * sp;
            probs16(s, c2, neg2, sum, pb);
            probs16(s + 16, c2, neg2, sum, pb + 8);
            announce(D == 128 ? q : sp >> 1);
          }
          float s0, s1;
          unpack2(add2(sum[0], sum[1]), s0, s1);
          l += s0 + s1;
        } else {
          if (D == 256 && sp >= 2) announce(0);
          uint32_t z[16];
#pragma unroll
          for (int i = 0; i < 16; i++) z[i] = 0;
#pragma unroll
          for (int q = 0; q < NQ; q++) {
            tm_store16(sb + 64 * q + 32 * sp, z);
            announce(D == 128 ? q : sp >> 1);
          }
        }
      }
      if (!ok) break;
      ring0 += (uint32_t)(2 * NC * n);
      npv[par] += (uint32_t)((n + 1) >> 1);
      npv[par ^ 1] += (uint32_t)(n >> 1);
      if (alt) par = (par + n) & 1;
      // -------------------------------------------------------------- epilogue
      const int mine = few ? (n + 1 - t0) / 2 : n;  // this half's tiles
      if (mine > 0) {
        if (!(ok = wait(kBarO + h, no++ & 1))) break;
        fence_after();
        // (only now: the products took every partner's last probabilities, so the maxima have
        // been read)
        if (any_valid) {  // the row's sum over all columns, added in warpgroup order
          if (!(ok = exchange(l))) break;
          l = 0.0f;
#pragma unroll
          for (int j = 0; j < SP; j++) l += ldsf(xs + 512 * j);
          __syncwarp();
          if (lane == 0) bar_arrive(bar(xbar));
          unread = true;
        }
      }
      if (any_valid) {
        const int tok = it.tok0 + local, head = kvh * g + head_row;
        const float inv = l != 0.0f ? 1.0f / l : 0.0f;  // (no key at all: zero)
        // (few rows: the even tiles' part, then the odd ones')
        const int64_t prow = (int64_t)(it.part + (t0 * it.ntok + local) * g + head_row) * p.nkv + kvh;
        // (loads of tensor memory in flight together, as far as the registers go: one after
        // the other a wide window takes 4% longer, all four at head_dim 128 the rest 2%)
#pragma unroll(D == 128 ? 2 : 4)
        for (int i = 0; i < 4; i++) {
          const int col = sp * 64 + 16 * i;
          float o[16] = {};
          if (mine > 0) tm_load16(ob + 16 * i, o);
          if (valid && it.part < 0) {
            uint32_t v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = pack_bf16(o[2 * j] * inv, o[2 * j + 1] * inv);
            store32(p.out + tok * p.o_tok + head * p.o_head + col, v, args.wide);
          } else if (valid && l != 0.0f) {
            float* dst = p.part_o + prow * D + col;
#pragma unroll
            for (int j = 0; j < 16; j += 8) store32(dst + j, reinterpret_cast<const uint32_t*>(o) + j, true);
          }
          __syncwarp();  // (the next load is the whole warp's)
        }
        if (valid && it.part >= 0 && sp == 0) p.part_ml[prow] = make_float2(m * c, l);
      }
    }
    if (!ok) fail();
  }

  fence_before();
  __syncthreads();
  if (warp == kMmaWarp && *drained_flag) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
}

}  // namespace tc
}  // namespace paged
}  // namespace spark
