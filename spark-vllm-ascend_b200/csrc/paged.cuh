// paged.cuh -- kernels of a batch of requests over the paged KV cache: block tables and
// slot maps from request lengths, the per-head norm + rotation + store of new rows, the
// work list of the paged attention, and the join of its partial results.
//
// All metadata lives on the device and is checked there: lengths, page ids and slots that
// do not fit are recorded in the caller's error word (kBad*) and never dereferenced.
#pragma once

#include "common.cuh"

namespace spark {
namespace paged {

// error word bits (the attention kernel's wait codes 1 and 2 are in attn_paged.cuh)
constexpr int kBadLength = 4;    // a length out of range, or starts that go down
constexpr int kNoPages = 8;      // the free list is shorter than the pages needed
constexpr int kTableWidth = 16;  // a request is longer than its block table row
constexpr int kNoRows = 32;      // more tokens than output rows
constexpr int kBadPage = 64;     // a block table entry outside the cache
constexpr int kBadPosition = 128;  // a position outside the rotation table
constexpr int kBadSlot = 256;    // a slot outside the cache
constexpr int kBadPlan = 512;    // a plan made for another shape or window, or none

// ------------------------------------------------------------------ block tables and slot maps
// Requests r = 0 .. R-1 with ctx[r] cached and nw[r] new tokens:
//   start[r] = sum of nw below r, len[r] = ctx[r] + nw[r];
//   pages ceil(ctx / bs) .. ceil(len / bs) - 1 of request r are the next ids of the free
//   list, in request order (free == nullptr: the table holds them already);
//   token t of request r: position ctx[r] + t - start[r], slot = page * bs + offset.
// Every CTA scans the R lengths itself (R <= kPlanMaxReqs: 8 bytes each, from L2) and
// keeps token starts and page starts in shared memory, so one launch does it all: the
// tokens and the new table entries are then dealt to all threads of the grid, a token
// finding its request by binary search.  All or nothing: when something does not fit,
// every CTA sees it in its own scan, no page is taken and the batch comes out empty.
constexpr int kPlanThreads = 512;
constexpr int kPlanMaxReqs = 8192;

struct PlanArgs {
  const int32_t *ctx, *nw, *free_ids, *free_head;
  int32_t *free_head_out, *table, *query_start, *seq_lens;
  int64_t *positions, *slots;
  int64_t table_stride;
  int reqs, num_free, width, bs, rows;
  int *counter, *error;
};

// inclusive scan over the CTA of two values per thread (sums of up to 8192 int32 values:
// 64 bits); returns the CTA totals in tot
__device__ __forceinline__ void block_scan2(long long& a, long long& b, long long (&tot)[2], long long (*ws)[2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) {
      a += x;
      b += y;
    }
  }
  if (lane == 31) {
    ws[warp][0] = a;
    ws[warp][1] = b;
  }
  __syncthreads();
  const int nw = blockDim.x >> 5;  // (at most 32 warps: every warp scans their totals)
  long long x = lane < nw ? ws[lane][0] : 0, y = lane < nw ? ws[lane][1] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) {
      x += u;
      y += v;
    }
  }
  const long long pa = __shfl_sync(0xffffffffu, x, (warp + 31) & 31), pb = __shfl_sync(0xffffffffu, y, (warp + 31) & 31);
  tot[0] = __shfl_sync(0xffffffffu, x, 31);
  tot[1] = __shfl_sync(0xffffffffu, y, 31);
  if (warp) {
    a += pa;
    b += pb;
  }
  __syncthreads();
}

// largest r with start[r] <= i (start ascending, start[0] = 0)
__device__ __forceinline__ int find_request(const int* start, int reqs, int i) {
  int lo = 0, hi = reqs - 1;
  while (lo < hi) {
    const int m = (lo + hi + 1) >> 1;
    if (start[m] <= i) lo = m;
    else hi = m - 1;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(PlanArgs p) {
  extern __shared__ int plan_sm[];
  __shared__ long long ws[kPlanThreads / 32][2];
  __shared__ int bad_s;
  int* start = plan_sm;              // [R + 1]
  int* page0 = plan_sm + p.reqs + 1;  // [R + 1] new pages below request r
  int* ctx_s = page0 + p.reqs + 1;    // [R] cached tokens
  const int tid = threadIdx.x, R = p.reqs, bs = p.bs;
  pdl_wait();
  if (tid == 0) bad_s = 0;
  __syncthreads();
  const int head = p.free_ids ? p.free_head[0] : 0;
  long long t_sum = 0, p_sum = 0;
  int bad = 0;
  for (int r0 = 0; r0 < R; r0 += kPlanThreads) {
    const int r = r0 + tid;
    long long n = 0, np = 0;
    int c = 0;
    if (r < R) {
      c = p.ctx[r];
      const long long w = p.nw[r];
      if (c < 0 || w < 0 || c + w > 0x7fffffffLL) bad |= kBadLength;
      else {
        const int need = (int)((c + w + bs - 1) / bs), have = (int)(((long long)c + bs - 1) / bs);
        if (need > p.width) bad |= kTableWidth;
        n = w;
        np = p.free_ids ? need - have : 0;
      }
    }
    long long tot[2], a = n, b = np;
    block_scan2(a, b, tot, ws);
    if (r < R) {  // (sums past int32 are refused below before they are read)
      start[r] = (int)(t_sum + a - n);
      page0[r] = (int)(p_sum + b - np);
      ctx_s[r] = c;
    }
    t_sum += tot[0];
    p_sum += tot[1];
  }
  if (tid == 0) {
    start[R] = (int)t_sum;
    page0[R] = (int)p_sum;
  }
  if (t_sum > p.rows) bad |= kNoRows;
  if (p.free_ids && (head < 0 || p_sum > (long long)p.num_free - head)) bad |= kNoPages;
  if (bad) atomicOr(&bad_s, bad);
  __syncthreads();
  bad = bad_s;
  if (bad && blockIdx.x == 0 && tid == 0) atomicOr(p.error, bad);
  const int tokens = bad ? 0 : (int)t_sum, pages = bad ? 0 : (int)p_sum;
  const int gtid = blockIdx.x * kPlanThreads + tid, gthreads = gridDim.x * kPlanThreads;
  for (int r = gtid; r <= R; r += gthreads) {  // (R <= kPlanMaxReqs)
    p.query_start[r] = bad ? 0 : start[r];
    if (r < R) p.seq_lens[r] = bad ? 0 : ctx_s[r] + (start[r + 1] - start[r]);
  }
  // (unsigned: the step past 2^31 - 1 rows or pages is not one below zero)
  for (uint32_t i = gtid; i < (uint32_t)pages; i += gthreads) {
    const int r = find_request(page0, R, i);
    const int first = (int)(((long long)ctx_s[r] + bs - 1) / bs);
    p.table[r * p.table_stride + first + (i - page0[r])] = p.free_ids[head + i];
  }
  for (uint32_t i = gtid; i < (uint32_t)p.rows; i += gthreads) {
    long long pos = 0, slot = -1;
    if (i < (uint32_t)tokens) {
      const int r = find_request(start, R, i);
      const int c = ctx_s[r], at = c + (i - start[r]);  // (below seq_lens[r]: fits)
      const int pg = at / bs, first = (int)(((long long)c + bs - 1) / bs);
      pos = at;
      // a page taken in this call is read from the free list: another CTA may not have
      // written its table entry yet
      const int id = p.free_ids && pg >= first ? p.free_ids[head + page0[r] + pg - first]
                                               : p.table[r * p.table_stride + pg];
      if (id >= 0) slot = (long long)id * bs + (at - pg * bs);
      else atomicOr(p.error, kBadPage);
    }
    p.positions[i] = pos;
    p.slots[i] = slot;
  }
  if (p.free_head_out) {  // after every CTA has read free_head (the two may be one tensor)
    __syncthreads();
    if (tid == 0) {
      __threadfence();
      if (atomicAdd(p.counter, 1) == (int)gridDim.x - 1) {
        *p.counter = 0;
        p.free_head_out[0] = head + pages;
      }
    }
  }
}

// ------------------------------------------------------------------ norm + rotation + store
// One pass over the rows of a fused qkv output: per head of q and k
//   y = x * rsqrt(mean(x^2) + eps) * gamma          (gamma == nullptr: y = x)
//   (y_i, y_{i + r/2}) -> (y_i c_i - y_{i+r/2} s_i, y_{i+r/2} c_i + y_i s_i),  i < r/2
// in fp32, rounded to bf16 once at the end (the input's own rounding is the last one
// before it: no bf16 between the norm and the rotation); q to q_out, k and v to the pages
// at slot_mapping.  D / 8 lanes hold one head, 8 elements (16 bytes) each: the norm is a
// butterfly over them and the rotation partner is the lane r / 16 away.
struct RopeArgs {
  const uint16_t *qkv, *qg, *kg, *cos_sin;
  const int64_t *positions, *slots;
  uint16_t *k_cache, *v_cache, *q_out;
  int64_t row_stride, max_pos, num_slots;
  float eps;
  int rows, nq, nkv, rot, bs;
  int* error;
};

// packed pairs of fp32 (each half rounded as the scalar operation)
typedef unsigned long long u64;
__device__ __forceinline__ u64 pack2(float lo, float hi) {
  u64 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(u64 v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ u64 fma2(u64 a, u64 b, u64 c) {
  u64 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ u64 add2(u64 a, u64 b) {
  u64 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ u64 mul2(u64 a, u64 b) {
  u64 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ void unpack8(const uint4 u, u64 (&v)[4]) {
  v[0] = pack2(bf_lo(u.x), bf_hi(u.x));
  v[1] = pack2(bf_lo(u.y), bf_hi(u.y));
  v[2] = pack2(bf_lo(u.z), bf_hi(u.z));
  v[3] = pack2(bf_lo(u.w), bf_hi(u.w));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint4 pack8(const u64 (&v)[4]) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    float a, b;
    unpack2(v[j], a, b);
    w[j] = pack_bf16(a, b);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// D / 16 lanes hold a head, 16 elements each: two runs of 8 that are rotation partners (i ..
// i + 7 and i + r/2 ..), or two of the unrotated rest; so the norm's butterfly is the only
// exchange between lanes.  A CTA is 128 threads of one row (blockIdx.y: which heads).  Memory
// bound with two dependent loads (position, then rotation row) in a row's chain: small CTAs
// at 48 registers, ten or more to an SM, hide that best (16111 rows of 24 heads of 256: 80
// us, 4.9 TB/s; 256 threads 97-109 us, persistent CTAs reading four rows ahead 137 us).
constexpr int kRopeMaxThreads = 128;

template <int D>
__global__ void __launch_bounds__(kRopeMaxThreads, 10) rope_store_kernel(RopeArgs p) {
  constexpr int L = D / 16;  // lanes per head
  const int nh = p.nq + 2 * p.nkv;
  const int sub = threadIdx.x % L, h = blockIdx.y * (blockDim.x / L) + threadIdx.x / L;
  const bool head_ok = h < nh, is_v = h >= p.nq + p.nkv, is_k = !is_v && h >= p.nq;
  const int half = p.rot >> 1, hl = half >> 3;
  const bool rotated = head_ok && !is_v && sub < hl;
  const int e0 = sub < hl ? 8 * sub : 8 * (hl + sub);
  const int e1 = e0 + (sub < hl ? half : 8 * (L - hl));
  const int64_t row = blockIdx.x;
  pdl_wait();
  uint4 w0 = make_uint4(0, 0, 0, 0), w1 = w0, g0 = w0, g1 = w0, cw = w0, sw = w0;
  int64_t pos = 0, slot = -1;
  const bool norm = p.qg && head_ok && !is_v;
  if (head_ok) {
    const uint16_t* x_at = p.qkv + row * p.row_stride + h * D;
    if (!is_v) pos = p.positions[row];
    if (is_v || is_k) slot = p.slots[row];
    w0 = ldg_stream(x_at + e0);
    w1 = ldg_stream(x_at + e1);
  }
  if (norm) {
    const uint16_t* gamma = is_k ? p.kg : p.qg;
    g0 = __ldg(reinterpret_cast<const uint4*>(gamma + e0));
    g1 = __ldg(reinterpret_cast<const uint4*>(gamma + e1));
  }
  const bool pos_ok = pos >= 0 && pos < p.max_pos;
  if (rotated && pos_ok) {
    cw = __ldg(reinterpret_cast<const uint4*>(p.cos_sin + pos * p.rot + e0));
    sw = __ldg(reinterpret_cast<const uint4*>(p.cos_sin + pos * p.rot + e1));
  }
  u64 x[4], y[4];
  unpack8(w0, x);
  unpack8(w1, y);
  if (p.qg) {  // (uniform: the shuffles are the whole warp's)
    u64 s2 = mul2(x[0], x[0]);
#pragma unroll
    for (int j = 1; j < 4; j++) s2 = fma2(x[j], x[j], s2);
#pragma unroll
    for (int j = 0; j < 4; j++) s2 = fma2(y[j], y[j], s2);
    float a, b;
    unpack2(s2, a, b);
    a += b;
#pragma unroll
    for (int o = L / 2; o >= 1; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    if (norm) {
      const float inv = rsqrtf(a * (1.0f / D) + p.eps);
      const u64 inv2 = pack2(inv, inv);
      u64 g[4];
      unpack8(g0, g);
#pragma unroll
      for (int j = 0; j < 4; j++) x[j] = mul2(mul2(x[j], inv2), g[j]);
      unpack8(g1, g);
#pragma unroll
      for (int j = 0; j < 4; j++) y[j] = mul2(mul2(y[j], inv2), g[j]);
    }
  }
  if (rotated) {
    u64 c[4], s[4];
    unpack8(cw, c);
    unpack8(sw, s);
    const u64 minus = pack2(-1.0f, -1.0f);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const u64 xs = mul2(x[j], s[j]), ys = mul2(mul2(y[j], s[j]), minus);
      x[j] = add2(mul2(x[j], c[j]), ys);
      y[j] = add2(mul2(y[j], c[j]), xs);
    }
  }
  if (!head_ok) return;
  if (!is_v) {
    w0 = pack8(x);
    w1 = pack8(y);
  }
  uint16_t* dst;
  if (!pos_ok) {
    if (sub == 0) atomicOr(p.error, kBadPosition);
    return;
  }
  if (!is_v && !is_k) {
    dst = p.q_out + (row * p.nq + h) * D;
  } else {
    if (slot < 0) return;  // padding
    if (slot >= p.num_slots) {
      if (sub == 0) atomicOr(p.error, kBadSlot);
      return;
    }
    int64_t blk, off;
    if (slot <= 0x7fffffff) {  // (a 64-bit division costs as much as the row's arithmetic)
      blk = (uint32_t)slot / (uint32_t)p.bs;
      off = (uint32_t)slot - (uint32_t)blk * (uint32_t)p.bs;
    } else {
      blk = slot / p.bs;
      off = slot - blk * p.bs;
    }
    const int kh = h - p.nq - (is_v ? p.nkv : 0);
    dst = (is_v ? p.v_cache : p.k_cache) + ((blk * p.nkv + kh) * p.bs + off) * D;
  }
  *reinterpret_cast<uint4*>(dst + e0) = w0;
  *reinterpret_cast<uint4*>(dst + e1) = w1;
}

// ------------------------------------------------------------------ attention work list
// The attention kernel walks items: a tile of consecutive query tokens of one request (the
// rows of a tile are its tokens x the g query heads of a kv head) against a run of 128-key
// tiles.  The list is per kv head (item i stands for nkv of them).  A tile whose run is
// long against the even share of all work is cut into parts, whose unnormalised sums go to
// the partial buffers and are joined by combine_kernel.
constexpr int kKeyTile = 128;

struct alignas(16) Item {
  int tok0, ntok;   // query tokens
  int pos0;         // position of the first one (kFlagLens: unused)
  int req;          // block table row
  int key0, nkt;    // first key (a multiple of kKeyTile), key tiles
  int klo, khi;     // keys of the part: [klo, khi)
  int len;          // keys the request holds: rows of its pages at or past it are stale
  int flags;
  int part;         // first partial row, or -1: the part is the whole tile
  int pad;
};
constexpr int kFlagFew = 1;   // the tokens fit half a tile: the two halves take alternate key tiles, a part each
constexpr int kFlagLens = 2;  // row limits are the requests' lengths (shared prefix), not causal
static_assert(sizeof(Item) == 48, "items are three 16-byte words");

struct alignas(16) Entry {  // rows to join: tokens tok0 .. tok0 + ntok - 1, part i of a list at base + i * stride
  int tok0, ntok, base_a, n_a, stride_a, base_b, n_b, stride_b;
};

// What the plan was made for stands in its header: the attention compares it with its own
// arguments, since every offset and partial row below follows from them.
struct Shape {
  int max_tokens, max_reqs, nq, nkv, head_dim, window;
};
struct alignas(16) Header {
  int items, entries;
  int join_rows;  // rows of the largest entry
  int pad0;
  Shape shape;
  int pad1[6];
};
static_assert(sizeof(Header) == 64, "items start at a multiple of 16 bytes");

struct Layout {
  int tile_tok, half_tok, max_tiles, max_items, max_entries, budget, part_rows;
  int64_t items, entries, starts, tiles, bases, lens, bytes;
};

// Sizes of a plan for up to T tokens and R requests.  `budget` bounds the parts beyond one
// per tile (4 per SM over the kv heads), so that partial rows stay bounded.
__host__ __device__ inline Layout layout_of(int T, int R, int nq, int nkv, int D) {
  Layout l;
  const int g = nq / nkv;
  l.half_tok = 128 / g;
  l.tile_tok = D == 128 ? 2 * l.half_tok : l.half_tok;
  const int tk = T > R ? T : R;
  l.max_tiles = tk / l.tile_tok + R + 1;
  l.budget = 4 * kNumSMs / nkv + 1;
  l.max_items = l.max_tiles + l.budget;
  l.max_entries = R + l.budget;
  const int64_t rows = l.tile_tok < tk ? l.tile_tok : tk;
  l.part_rows = (int)((2 * (int64_t)l.budget * rows + 4 * (int64_t)R) * g);
  int64_t at = 0;  // every array starts on a 16-byte boundary
  auto take = [&at](int64_t bytes) {
    const int64_t o = at;
    at += (bytes + 15) / 16 * 16;
    return o;
  };
  take(sizeof(Header));
  l.items = take((int64_t)l.max_items * sizeof(Item));
  l.entries = take((int64_t)l.max_entries * sizeof(Entry));
  l.starts = take(((int64_t)R + 1) * sizeof(int));
  l.tiles = take((int64_t)l.max_tiles * sizeof(int2));
  l.bases = take((int64_t)l.max_tiles * sizeof(int2));
  l.lens = take(((int64_t)R + 1) * sizeof(int));
  // (one item per CTA is read before the header is known to match: any plan has room for them)
  const int64_t least = sizeof(Header) + (int64_t)kNumSMs * sizeof(Item);
  l.bytes = at > least ? at : least;
  return l;
}

struct AttnPlanArgs {
  const int32_t *query_start, *seq_lens, *prefix_len;  // prefix_len: the shared-prefix plan
  int reqs, tokens, max_reqs, nq, nkv, D, window;
  Layout lay;
  unsigned char* plan;
  int* error;
};

constexpr int kAttnPlanThreads = 1024;
constexpr int kBins = 1024;
constexpr int kPlanStarts = 1024, kPlanTiles = 1024;
// longest request: key positions are 32-bit numbers, also those of the tiles and page ids
// read ahead past its end
constexpr int kMaxKeys = 0x7fff0000;

// Tile i of the batch: everything but how it is cut.
struct Tile {
  int tok0, ntok, pos0, req, key0, nkt, klo, khi, len, flags;
};

__device__ __forceinline__ Tile prompt_tile(const AttnPlanArgs& p, int q0, int n, int len, int r, int k) {
  Tile t;
  const int off = k * p.lay.tile_tok;
  t.tok0 = q0 + off;
  t.ntok = n - off < p.lay.tile_tok ? n - off : p.lay.tile_tok;
  t.pos0 = len - n + off;  // (negative when the request has more queries than keys)
  t.req = r;
  t.len = len;
  const int last = t.pos0 + t.ntok;  // exclusive causal limit of the last row
  t.khi = last < 0 ? 0 : last;
  // (compared first: with a window near 2^31 the difference of a negative position wraps)
  t.klo = p.window > 0 && t.pos0 >= p.window ? t.pos0 + 1 - p.window : 0;
  t.key0 = t.klo / kKeyTile * kKeyTile;
  t.nkt = t.khi > t.klo ? (t.khi - t.key0 + kKeyTile - 1) / kKeyTile : 0;
  t.flags = p.D == 128 && t.ntok <= p.lay.half_tok && t.nkt > 1 ? kFlagFew : 0;
  return t;
}

__device__ __forceinline__ Tile prefix_tile(const AttnPlanArgs& p, const int* lens, int prefix, int npre, int i) {
  Tile t;
  t.pos0 = 0;
  t.flags = kFlagLens;
  if (i < npre) {  // a tile of requests against the prefix, through the first request's table
    t.tok0 = i * p.lay.tile_tok;
    t.ntok = p.reqs - t.tok0 < p.lay.tile_tok ? p.reqs - t.tok0 : p.lay.tile_tok;
    t.req = 0;
    t.klo = 0;
    t.khi = t.len = prefix;
  } else {  // one request's own keys
    t.tok0 = t.req = i - npre;
    t.ntok = 1;
    t.klo = prefix;
    t.khi = t.len = lens[t.req];
  }
  t.key0 = t.klo / kKeyTile * kKeyTile;
  t.nkt = t.khi > t.klo ? (t.khi - t.key0 + kKeyTile - 1) / kKeyTile : 0;
  if (p.D == 128 && t.ntok <= p.lay.half_tok && t.nkt > 1) t.flags |= kFlagFew;
  return t;
}

// Cost of a part in quarters of a key tile of many rows: the tiles (alternating halves take
// two at a time), what an item costs around them, and for a part that is joined the fp32
// sums of its rows.  Measured with the attention kernel: see there.
__host__ __device__ inline int part_cost(int flags, int parts, int tiles, int rows) {
  return tiles * ((flags & kFlagFew) ? 2 : 4) + 8 + (parts > 1 ? rows / 32 : 0);
}
constexpr int kPriceBins = 128;
__device__ __forceinline__ int price_bin(int cost, int top) {
  return min((int)((long long)cost * kPriceBins / (top + 1)), kPriceBins - 1);
}
__constant__ int kCuts[32] = {1,  2,  3,  4,  5,  6,  7,  8,  9,  10, 11, 12, 13, 14, 15, 16,
                              18, 20, 22, 24, 27, 30, 34, 37, 42, 48, 55, 64, 74, 96, 128, 148};

__global__ void __launch_bounds__(kAttnPlanThreads) attn_plan_kernel(AttnPlanArgs p) {
  __shared__ long long ws2[kAttnPlanThreads / 32][2];
  __shared__ int ws[kAttnPlanThreads / 32];
  __shared__ int hist[kBins];
  __shared__ int price[32 * (kPriceBins + 1)];
  // of small batches: first tile per request, and (key tiles, flags | rows << 8) per tile
  __shared__ int starts_s[kPlanStarts + 1];
  __shared__ int2 brief_s[kPlanTiles];
  __shared__ int entries_s, rows_s, bad_s, join_s, keys_s;
  const int tid = threadIdx.x, R = p.reqs;
  Header* hdr = reinterpret_cast<Header*>(p.plan);
  Item* items = reinterpret_cast<Item*>(p.plan + p.lay.items);
  Entry* entries = reinterpret_cast<Entry*>(p.plan + p.lay.entries);
  int* starts = R <= kPlanStarts ? starts_s : reinterpret_cast<int*>(p.plan + p.lay.starts);  // first tile of request r
  int2* tiles = reinterpret_cast<int2*>(p.plan + p.lay.tiles);  // (request, tile of the request)
  int2* bases = reinterpret_cast<int2*>(p.plan + p.lay.bases);  // (first partial row, parts)
  int* lens = reinterpret_cast<int*>(p.plan + p.lay.lens);
  pdl_wait();
  if (tid == 0) entries_s = rows_s = bad_s = join_s = keys_s = 0;
  __syncthreads();
  const bool prefix_kind = p.prefix_len != nullptr;
  int prefix = 0, npre = 0, nt = 0;
  // tiles per request
  if (prefix_kind) {
    prefix = p.prefix_len[0];
    if (prefix < 0 || prefix > kMaxKeys) {
      prefix = 0;
      if (tid == 0) bad_s = kBadLength;
    }
    int most = 0;
    for (int r = tid; r < R; r += kAttnPlanThreads) {
      const int n = p.seq_lens[r];
      const bool ok = n >= 0 && n <= kMaxKeys;
      if (!ok) atomicOr(&bad_s, kBadLength);
      lens[r] = ok ? n : 0;
      if (ok && n > most) most = n;
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if ((tid & 31) == 0 && most) atomicMax(&keys_s, most);
    npre = (R + p.lay.tile_tok - 1) / p.lay.tile_tok;
    nt = npre + R;
  } else {
    long long sum = 0;
    for (int r0 = 0; r0 < R; r0 += kAttnPlanThreads) {
      const int r = r0 + tid;
      long long n = 0, dummy = 0, tot[2];
      if (r < R) {
        const int q0 = p.query_start[r], q1 = p.query_start[r + 1], len = p.seq_lens[r];
        const bool ok = q0 >= 0 && q1 >= q0 && q1 <= p.tokens && len >= 0 && len <= kMaxKeys;
        if (!ok) atomicOr(&bad_s, kBadLength);
        lens[r] = ok ? len : 0;
        n = ok ? (q1 - q0 + p.lay.tile_tok - 1) / p.lay.tile_tok : 0;
      }
      long long a = n;
      block_scan2(a, dummy, tot, ws2);
      // (overlapping starts could list more tokens than there are: the excess is cut)
      if (r < R) {
        const long long s = sum + a - n;
        starts[r] = (int)(s < p.lay.max_tiles ? s : p.lay.max_tiles);
      }
      sum += tot[0];
    }
    if (sum > p.lay.max_tiles) {
      sum = p.lay.max_tiles;
      if (tid == 0) atomicOr(&bad_s, kBadLength);
    }
    nt = (int)sum;
  }
  __syncthreads();
  // (no request holds what lies behind the longest one: neither a page id nor finite values)
  if (prefix > keys_s) prefix = keys_s;
  bool allow_few = true;
  auto tile_at = [&](int i) {
    if (prefix_kind) return prefix_tile(p, lens, prefix, npre, i);
    const int2 t = tiles[i];
    const int q0 = p.query_start[t.x];
    Tile tile = prompt_tile(p, q0, p.query_start[t.x + 1] - q0, lens[t.x], t.x, t.y);
    if (!allow_few) tile.flags = 0;
    return tile;
  };
  const int g = p.nq / p.nkv;
  int longest = 0, few_rows = 0;
  for (int i = tid; i < nt; i += kAttnPlanThreads) {
    if (!prefix_kind) {
      const int r = find_request(starts, R, i);
      tiles[i] = make_int2(r, i - starts[r]);
    }
    const Tile t = tile_at(i);
    if (i < kPlanTiles) brief_s[i] = make_int2(t.nkt, t.flags | t.ntok * g << 8);
    longest = t.nkt > longest ? t.nkt : longest;
    if (t.flags & kFlagFew) few_rows += 2 * t.ntok * g;
  }
  longest = __reduce_max_sync(0xffffffffu, longest);
  few_rows = __reduce_add_sync(0xffffffffu, few_rows);
  if ((tid & 31) == 0) {
    ws[tid >> 5] = longest;
    ws2[tid >> 5][0] = few_rows;
  }
  __syncthreads();
  longest = __reduce_max_sync(0xffffffffu, ws[tid & 31]);
  long long few_all = 0;
  for (int w = 0; w < kAttnPlanThreads / 32; w++) few_all += ws2[w][0];
  __syncthreads();
  // many requests of some tokens each: enough tiles without, and their parts would not fit
  if (!prefix_kind && few_all > p.lay.part_rows / 2) allow_few = false;
  // How fine to cut: warp w prices "the longest tile in kCuts[w] parts, the others in parts
  // no longer than those" by dealing the parts out as the attention kernel will.  (A batch of
  // more than 8192 tiles balances without.)
  int cut = longest > 0 ? longest : 1;
  if (nt <= 8192 && longest > 1) {
    const int w = tid >> 5, lane = tid & 31;
    const int c = (longest + kCuts[w] - 1) / kCuts[w];
    int* h = price + w * (kPriceBins + 1);
    for (int b = lane; b <= kPriceBins; b += 32) h[b] = 0;
    const int top = part_cost(0, 2, c, p.lay.tile_tok * g);  // (no part costs more)
    __syncwarp();
    int extra = 0, rows = 0;
    for (int i = lane; i < nt; i += 32) {
      int nkt, flags, trows;
      if (i < kPlanTiles) {
        const int2 t = brief_s[i];
        nkt = t.x, flags = allow_few ? t.y & 255 : t.y & 255 & ~kFlagFew, trows = t.y >> 8;
      } else {
        const Tile t = tile_at(i);
        nkt = t.nkt, flags = t.flags, trows = t.ntok * g;
      }
      const int np = (nkt + c - 1) / c;
      if (np == 0) continue;
      extra += np - 1;
      const int each = (flags & kFlagFew) ? 2 : 1;
      if (np > 1 || prefix_kind || each == 2) rows += each * np * trows;
      const int lo = nkt / np, more = nkt - lo * np;  // `more` parts have one tile more
      const int joined = prefix_kind ? 2 : np;
      const int c0 = part_cost(flags, joined, lo, trows), c1 = part_cost(flags, joined, lo + 1, trows);
      if (np > more) atomicAdd(&h[price_bin(c0, top)], (np - more) * p.nkv);
      if (more) atomicAdd(&h[price_bin(c1, top)], more * p.nkv);
    }
    for (int o = 16; o >= 1; o >>= 1) {
      extra += __shfl_xor_sync(0xffffffffu, extra, o);
      rows += __shfl_xor_sync(0xffffffffu, rows, o);
    }
    __syncwarp();
    // bin counts -> parts in this bin and above it (costlier), by a suffix scan of 8 bins a lane
    int mine[kPriceBins / 32], sum = 0;
    for (int j = kPriceBins / 32 - 1; j >= 0; j--) mine[j] = sum += h[lane * (kPriceBins / 32) + j];
    int above = sum;
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_down_sync(0xffffffffu, above, o);
      if (lane + o < 32) above += v;
    }
    above -= sum;
    __syncwarp();
    for (int j = 0; j < kPriceBins / 32; j++) h[lane * (kPriceBins / 32) + j] = mine[j] + above;
    __syncwarp();
    const int parts = h[0];
    // the load of eight of the CTAs, four lanes each that take every fourth round, in the
    // kernel's back-and-forth order
    const int cta = (lane >> 2) * (kNumSMs - 1) / 7;
    int worst = 0;
    for (int round = lane & 3; (int64_t)round * kNumSMs < parts; round += 4) {
      const int at = round * kNumSMs + ((round & 1) ? kNumSMs - 1 - cta : cta);
      if (at >= parts) continue;
      int lo = 0, hi = kPriceBins - 1;  // largest bin with more than `at` parts in and above it
      while (lo < hi) {
        const int m = (lo + hi + 1) >> 1;
        if (h[m] > at) lo = m;
        else hi = m - 1;
      }
      worst += lo + 1;
    }
    worst += __shfl_xor_sync(0xffffffffu, worst, 1);
    worst += __shfl_xor_sync(0xffffffffu, worst, 2);
    worst = __reduce_max_sync(0xffffffffu, worst);
    // bins back to cost (rounded up); what does not fit the buffers is out
    const bool fits = extra <= p.lay.budget && rows <= p.lay.part_rows;
    const long long cost = fits ? (long long)worst * top : (1LL << 60);
    if (lane == 0) {
      ws2[w][0] = cost;
      ws2[w][1] = c;
    }
    __syncthreads();
    long long best = ws2[0][0];  // (whole tiles always fit)
    cut = (int)ws2[0][1];
    for (int i = 1; i < kAttnPlanThreads / 32; i++)
      if (ws2[i][0] < best) {
        best = ws2[i][0];
        cut = (int)ws2[i][1];
      }
    __syncthreads();
  }
  // longest parts first (a counting sort by length; the order inside a length does not
  // matter to any result)
  for (int b = tid; b < kBins; b += kAttnPlanThreads) hist[b] = 0;
  __syncthreads();
  const int top = part_cost(0, 2, cut, p.lay.tile_tok * g);
  auto bin_of = [&](const Tile& t, int joined, int keys) {
    return kBins - 1 - (int)((long long)min(part_cost(t.flags, joined, keys, t.ntok * g), top) * (kBins - 1) / top);
  };
  // a group of 32, 4 or 1 lanes per tile, which share its parts
  const int group = nt <= 32 ? 32 : nt <= 256 ? 4 : 1, sub = tid & (group - 1);
  const int per = kAttnPlanThreads / group, turns = (nt + per - 1) / per;
  for (int pass = 0; pass < 2; pass++) {
    for (int turn = 0; turn < turns; turn++) {  // (uniform: the shuffle is the whole warp's)
      const int i = turn * per + tid / group;
      Tile t;
      int np = 0, each = 1, base = -1;
      bool parts = false;
      if (i < nt) {
        t = tile_at(i);
        np = (t.nkt + cut - 1) / cut;
        if (np == 0 && !prefix_kind) np = 1;  // rows without keys are written as zeros
        each = (t.flags & kFlagFew) ? 2 : 1;
        parts = np > 1 || prefix_kind || each == 2;
        if (pass == 1 && sub == 0) {
          if (parts) base = atomicAdd(&rows_s, each * np * t.ntok * g);
          bases[i] = make_int2(base, each * np);
          if (parts && !prefix_kind) {
            const int e = atomicAdd(&entries_s, 1);
            entries[e] = {t.tok0, t.ntok, base, each * np, t.ntok * g, 0, 0, 0};
            atomicMax(&join_s, t.ntok * g);
          }
        }
      }
      base = __shfl_sync(0xffffffffu, base, (tid & 31) & ~(group - 1));
      for (int k = sub; k < np; k += group) {
        const int a = (int)((long long)k * t.nkt / np), b = (int)((long long)(k + 1) * t.nkt / np);
        const int slot = atomicAdd(&hist[bin_of(t, parts ? 2 : 1, b - a)], 1);
        if (pass == 1) {
          Item it;
          it.tok0 = t.tok0, it.ntok = t.ntok, it.pos0 = t.pos0, it.req = t.req;
          it.key0 = t.key0 + a * kKeyTile;
          it.nkt = b - a;
          it.klo = a ? it.key0 : t.klo;
          it.khi = k + 1 < np ? t.key0 + b * kKeyTile : t.khi;
          it.len = t.len, it.flags = t.flags;
          it.part = parts ? base + k * each * t.ntok * g : -1;
          it.pad = 0;
          items[slot] = it;
        }
      }
    }
    __syncthreads();
    if (pass == 0) {  // counts -> first slot of each bin
      long long a = tid < kBins ? hist[tid] : 0, n = a, dummy = 0, tot[2];
      block_scan2(a, dummy, tot, ws2);
      if (tid < kBins) hist[tid] = (int)(a - n);
      if (tid == 0) hdr->items = (int)tot[0];
      __syncthreads();
    }
  }
  if (prefix_kind) {
    for (int r = tid; r < R; r += kAttnPlanThreads) {
      const int i = r / p.lay.tile_tok;
      const Tile t = prefix_tile(p, lens, prefix, npre, i);
      const int2 a = bases[i], b = bases[npre + r];
      entries[r] = {r, 1, a.x + (r - t.tok0) * g, a.y, t.ntok * g, b.x, b.y, g};
    }
  }
  if (tid == 0) {
    hdr->entries = prefix_kind ? R : entries_s;
    hdr->join_rows = prefix_kind ? p.nq / p.nkv : join_s;
    hdr->shape = {p.tokens, p.max_reqs, p.nq, p.nkv, p.D, p.window};
    if (bad_s) atomicOr(p.error, bad_s);
  }
}

// ------------------------------------------------------------------ attention
struct AttnArgs {
  const uint16_t *q, *k_cache, *v_cache;
  int64_t q_tok, q_head, o_tok, o_head;  // strides in elements
  const int32_t* table;
  int64_t table_stride, num_blocks;
  int table_width, table_rows, bs, tokens, max_tokens, max_reqs, nq, nkv, window;
  float scale;
  const unsigned char* plan;
  Layout lay;
  float* part_o;    // [part rows][nkv][D] unnormalised sums
  float2* part_ml;  // [part rows][nkv]: (running maximum of scale * s * log2 e, sum)
  uint16_t* out;
  int* error;
};

// the plan is one of this call's shape and window
template <int D>
__device__ __forceinline__ bool plan_fits(const AttnArgs& p, const Header* hdr) {
  const Shape s = hdr->shape;
  return s.max_tokens == p.max_tokens && s.max_reqs == p.max_reqs && s.nq == p.nq && s.nkv == p.nkv &&
         s.head_dim == D && s.window == p.window;
}

// keys row (token i of the item) may see, within the item's part
__device__ __forceinline__ int2 row_keys(const Item& it, const int* lens, int window, int i) {
  int lo = it.klo, hi = it.khi;
  if (it.flags & kFlagLens) {
    const int n = lens[it.tok0 + i];
    hi = n < hi ? n : hi;
  } else {
    const int pos = it.pos0 + i;
    hi = pos + 1 < hi ? pos + 1 : hi;
    if (window > 0 && pos >= window && pos + 1 - window > lo) lo = pos + 1 - window;  // (see prompt_tile)
  }
  return make_int2(lo, hi);
}

// Join of the parts of cut tiles: with M = max m_i over a row's parts,
//   out = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i,
// the parts in list order whatever order they were computed in.  A row without any key is
// zero.  One warp per row: lanes hold 32 parts' (m, l) at a time, then the warp adds the
// parts' sums, four in flight.
constexpr int kJoinThreads = 256, kJoinFlight = 4;

template <int D>
__global__ void __launch_bounds__(kJoinThreads) combine_kernel(AttnArgs p) {
  constexpr int E = D / 32;  // elements of a lane, contiguous
  pdl_wait();
  const Header* hdr = reinterpret_cast<const Header*>(p.plan);
  const Entry* entries = reinterpret_cast<const Entry*>(p.plan + p.lay.entries);
  const int g = p.nq / p.nkv, lane = threadIdx.x & 31;
  const int n = plan_fits<D>(p, hdr) ? hdr->entries : 0, jr = hdr->join_rows;
  // (entries x kv heads x rows: below 2^31, checked on the host)
  const uint32_t total = (uint32_t)n * p.nkv * jr, step = gridDim.x * (kJoinThreads / 32);
  for (uint32_t w = blockIdx.x * (kJoinThreads / 32) + (threadIdx.x >> 5); w < total; w += step) {
    const uint32_t x = w / (uint32_t)jr, e = x / (uint32_t)p.nkv;
    const int row = (int)(w - x * jr), kvh = (int)(x - e * p.nkv);
    const Entry en = entries[e];
    const int tok = en.tok0 + row / g, head = kvh * g + row % g;
    if (row >= en.ntok * g || tok >= p.tokens) continue;
    const int parts = en.n_a + en.n_b;
    auto index = [&](int k) {
      const int64_t r = k < en.n_a ? en.base_a + (int64_t)k * en.stride_a
                                   : en.base_b + (int64_t)(k - en.n_a) * en.stride_b;
      return (r + row) * p.nkv + kvh;
    };
    float M = -INFINITY, l = 0.0f, o[E];
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = 0.0f;
    for (int k0 = 0; k0 < parts; k0 += 32) {
      // (parts without a key for this row have l = 0: their sums were not written)
      const float2 ml = k0 + lane < parts ? p.part_ml[index(k0 + lane)] : make_float2(-INFINITY, 0.0f);
      const float mn = fmaxf(M, warp_max(ml.y != 0.0f ? ml.x : -INFINITY));
      const float wt = ml.y != 0.0f ? exp2f(ml.x - mn) : 0.0f;
      const float a = M == -INFINITY ? 0.0f : exp2f(M - mn);
      M = mn;
      l = l * a + butterfly_sum<32>(wt * ml.y);
#pragma unroll
      for (int e = 0; e < E; e++) o[e] *= a;
      const int m = parts - k0 < 32 ? parts - k0 : 32;
      for (int k = 0; k < m; k += kJoinFlight) {
        float v[kJoinFlight][E], f[kJoinFlight];
#pragma unroll
        for (int j = 0; j < kJoinFlight; j++) {
          f[j] = __shfl_sync(0xffffffffu, wt, (k + j) & 31);
          const bool use = k + j < m && f[j] != 0.0f;
          const float4* src = reinterpret_cast<const float4*>(p.part_o + index(k0 + k + j) * D + lane * E);
#pragma unroll
          for (int e = 0; e < E; e += 4) {
            const float4 t = use ? src[e / 4] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            v[j][e] = t.x, v[j][e + 1] = t.y, v[j][e + 2] = t.z, v[j][e + 3] = t.w;
          }
          if (!use) f[j] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < kJoinFlight; j++)
#pragma unroll
          for (int e = 0; e < E; e++) o[e] = __fmaf_rn(v[j][e], f[j], o[e]);
      }
    }
    const float inv = 1.0f / l;
    uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + tok * p.o_tok + head * p.o_head + lane * E);
#pragma unroll
    for (int e = 0; e < E; e += 2) dst[e / 2] = l != 0.0f ? pack_bf16(o[e] * inv, o[e + 1] * inv) : 0;
  }
}

}  // namespace paged
}  // namespace spark
