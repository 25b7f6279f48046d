// paged.cu -- C ABI entry points of the paged-batch operators (include/spark_b200.h).
// Sizes, strides and alignments are checked here, before any launch.
#include <algorithm>
#include <cstdint>
#include <cstring>

#include "attn_paged.cuh"
#include "host.cuh"
#include "paged.cuh"
#include "spark_b200.h"

using namespace spark;

// bytes [at, at + n) of a tensor; an absent one overlaps nothing
struct Span {
  const void* at;
  int64_t n;
};
static bool overlap(const Span& a, const Span& b) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
  return a.at && b.at && a.n > 0 && b.n > 0 && x < y + (uintptr_t)b.n && y < x + (uintptr_t)a.n;
}
// a span and `rows` rows of `width` bytes, `pitch` apart: what lies between the rows is free
static bool overlap(const Span& a, const void* base, int64_t rows, int64_t pitch, int64_t width) {
  if (!overlap(a, Span{base, (rows - 1) * pitch + width})) return false;
  const int64_t d = (int64_t)(reinterpret_cast<uintptr_t>(a.at) - reinterpret_cast<uintptr_t>(base));
  return d < 0 || d % pitch < width || d % pitch + a.n > pitch;
}

template <int D>
static int attn_launch(const paged::AttnArgs& p, int64_t wait_ns, cudaStream_t stream) {
  const int g = p.nq / p.nkv;
  paged::tc::TcArgs t;
  t.a = p;
  t.piece = p.bs & -p.bs;
  if (t.piece > paged::kKeyTile) t.piece = paged::kKeyTile;
  t.wide = p.o_tok % 16 == 0 && p.o_head % 16 == 0 && aligned(p.out, 32);
  t.limit_ns = wait_ns < 0 ? paged::tc::kWaitNs : (unsigned long long)wait_ns;
  const CUtensorMapDataType bf = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const uint64_t rows = (uint64_t)p.num_blocks * p.nkv * p.bs;
  CUtensorMap mq, mk, mv;
  if (!encode_map3(&mq, bf, p.q, {(uint64_t)D, (uint64_t)p.nq, (uint64_t)p.tokens},
                   {(uint64_t)p.q_head * 2, (uint64_t)p.q_tok * 2}, {64u, (uint32_t)g, (uint32_t)p.lay.half_tok}) ||
      !encode_map(&mk, bf, p.k_cache, D, rows, D * 2, 64, (uint32_t)t.piece, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !encode_map(&mv, bf, p.v_cache, D, rows, D * 2, 64, (uint32_t)t.piece, CU_TENSOR_MAP_SWIZZLE_128B))
    return SPARK_ERR_LAUNCH;
  const int grid = (int)std::min<int64_t>((int64_t)p.lay.max_items * p.nkv, std::min(num_sms(), kNumSMs));
  const int st = launch(paged::tc::attn_kernel<D>, dim3(grid), dim3(paged::tc::kThreads), paged::tc::kSmemBytes,
                        stream, mq, mk, mv, t);
  if (st) return st;
  // one row of a join per warp and pass; the device knows how many there are
  const int64_t join_rows = (int64_t)p.lay.max_entries * p.nkv * std::min(p.lay.tile_tok, p.tokens) * g;
  const int per_cta = paged::kJoinThreads / 32;
  const int cgrid = (int)std::min<int64_t>((join_rows + per_cta - 1) / per_cta, 4LL * num_sms());
  return launch(paged::combine_kernel<D>, dim3(cgrid), dim3(paged::kJoinThreads), 0, stream, p);
}

extern "C" {

int spark_paged_plan(const int32_t* ctx_lens, const int32_t* new_lens, int reqs, const int32_t* free_blocks,
                     int num_free, const int32_t* free_head, int32_t* free_head_out, int32_t* block_table,
                     int64_t table_stride, int table_width, int block_size, int rows, int32_t* query_start,
                     int32_t* seq_lens, int64_t* positions, int64_t* slot_mapping, int* counter, int* error,
                     void* stream) {
  if (!ctx_lens || !new_lens || !block_table || !query_start || !seq_lens || !error || !counter)
    return SPARK_ERR_INVALID_ARG;
  if (rows > 0 && (!positions || !slot_mapping)) return SPARK_ERR_INVALID_ARG;
  if (free_blocks ? (!free_head || !free_head_out) : (free_head || free_head_out)) return SPARK_ERR_INVALID_ARG;
  if (reqs <= 0 || rows < 0 || num_free < 0 || block_size <= 0 || table_width <= 0 || table_stride < table_width)
    return SPARK_ERR_UNSUPPORTED_SHAPE;
  if (reqs > paged::kPlanMaxReqs) return SPARK_ERR_TOO_LARGE;
  // every CTA reads all lengths and the free list, while others write already (the head may be
  // advanced in place: it is written when all have read it)
  const int64_t tokens = 8 * (int64_t)rows;
  const Span in[] = {{ctx_lens, 4 * (int64_t)reqs}, {new_lens, 4 * (int64_t)reqs}, {free_blocks, 4 * (int64_t)num_free},
                     {free_head == free_head_out ? nullptr : free_head, 4}};
  const Span out[] = {{query_start, 4 * ((int64_t)reqs + 1)}, {seq_lens, 4 * (int64_t)reqs}, {positions, tokens},
                      {slot_mapping, tokens}, {free_head_out, 4}, {counter, 4}, {error, 4}};
  auto on_table = [&](const Span& t) { return overlap(t, block_table, reqs, 4 * table_stride, 4 * table_width); };
  for (const Span& i : in)
    if (on_table(i)) return SPARK_ERR_INVALID_ARG;
  for (const Span& o : out) {
    if (on_table(o)) return SPARK_ERR_INVALID_ARG;
    for (const Span& i : in)
      if (overlap(o, i)) return SPARK_ERR_INVALID_ARG;
    for (const Span& other : out)
      if (&other != &o && overlap(o, other)) return SPARK_ERR_INVALID_ARG;
  }
  paged::PlanArgs p;
  memset(&p, 0, sizeof(p));
  p.ctx = ctx_lens, p.nw = new_lens, p.free_ids = free_blocks, p.free_head = free_head;
  p.free_head_out = free_head_out, p.table = block_table, p.query_start = query_start, p.seq_lens = seq_lens;
  p.positions = positions, p.slots = slot_mapping, p.table_stride = table_stride;
  p.reqs = reqs, p.num_free = num_free, p.width = table_width, p.bs = block_size, p.rows = rows;
  p.counter = counter, p.error = error;
  const int64_t units = std::max<int64_t>(rows, reqs);
  const int grid = (int)std::min<int64_t>((units + paged::kPlanThreads - 1) / paged::kPlanThreads, num_sms());
  return launch(paged::paged_plan_kernel, dim3(grid), dim3(paged::kPlanThreads), (3 * (size_t)reqs + 2) * 4,
                as_stream(stream), p);
}

int spark_qk_norm_rope_store_rows(const uint16_t* qkv, int64_t row_stride, int rows, int nq, int nkv, int head_dim,
                                  const uint16_t* q_gamma, const uint16_t* k_gamma, float eps,
                                  const uint16_t* cos_sin, int64_t max_pos, int rotary_dim, const int64_t* positions,
                                  const int64_t* slot_mapping, int block_size, int64_t num_blocks, uint16_t* k_cache,
                                  uint16_t* v_cache, uint16_t* q_out, int* error, void* stream) {
  if (!cos_sin || !positions || !slot_mapping || !k_cache || !v_cache || !error) return SPARK_ERR_INVALID_ARG;
  if ((q_gamma == nullptr) != (k_gamma == nullptr)) return SPARK_ERR_INVALID_ARG;
  if (rows < 0 || nq <= 0 || nkv <= 0 || (head_dim != 128 && head_dim != 256) || rotary_dim <= 0 ||
      rotary_dim % 16 || rotary_dim > head_dim || max_pos <= 0 || block_size <= 0 || num_blocks <= 0)
    return SPARK_ERR_UNSUPPORTED_SHAPE;
  if (row_stride < (int64_t)(nq + 2 * nkv) * head_dim) return SPARK_ERR_UNSUPPORTED_SHAPE;
  if (rows == 0) return SPARK_OK;
  if (!qkv || !q_out) return SPARK_ERR_INVALID_ARG;
  if (row_stride % 8 || !aligned(qkv, 16) || !aligned(cos_sin, 16) || !aligned(k_cache, 16) ||
      !aligned(v_cache, 16) || !aligned(q_out, 16) || (q_gamma && (!aligned(q_gamma, 16) || !aligned(k_gamma, 16))))
    return SPARK_ERR_ALIGNMENT;
  // rows are read and written in any order (a single one may be rotated in place)
  const int64_t cache = num_blocks * nkv * block_size * (int64_t)head_dim * 2;
  const Span x{qkv, ((rows - 1) * row_stride + (int64_t)(nq + 2 * nkv) * head_dim) * 2},
      y{q_out, (int64_t)rows * nq * head_dim * 2}, k{k_cache, cache}, v{v_cache, cache};
  if ((overlap(x, y) && !(rows == 1 && q_out == qkv)) || overlap(x, k) || overlap(x, v) || overlap(y, k) ||
      overlap(y, v) || overlap(k, v))
    return SPARK_ERR_INVALID_ARG;
  paged::RopeArgs p;
  memset(&p, 0, sizeof(p));
  p.qkv = qkv, p.qg = q_gamma, p.kg = k_gamma, p.cos_sin = cos_sin, p.positions = positions, p.slots = slot_mapping;
  p.k_cache = k_cache, p.v_cache = v_cache, p.q_out = q_out, p.row_stride = row_stride, p.max_pos = max_pos;
  p.num_slots = num_blocks * block_size, p.eps = eps, p.rows = rows, p.nq = nq, p.nkv = nkv, p.rot = rotary_dim;
  p.bs = block_size, p.error = error;
  const int lanes = (nq + 2 * nkv) * (head_dim / 16);  // 16 elements a thread
  const int threads = std::min((lanes + 31) / 32 * 32, paged::kRopeMaxThreads);
  const int gy = (lanes + threads - 1) / threads;
  if (gy > 65535) return SPARK_ERR_TOO_LARGE;
  const dim3 grid(rows, gy);
  if (head_dim == 128) return launch(paged::rope_store_kernel<128>, grid, dim3(threads), 0, as_stream(stream), p);
  return launch(paged::rope_store_kernel<256>, grid, dim3(threads), 0, as_stream(stream), p);
}

// ------------------------------------------------------------------ paged attention
static int check_attn_shape(int max_tokens, int max_reqs, int nq, int nkv, int head_dim) {
  if (max_tokens <= 0 || max_reqs <= 0 || nq <= 0 || nkv <= 0 || nq % nkv || nq / nkv > 128 ||
      (head_dim != 128 && head_dim != 256))
    return SPARK_ERR_UNSUPPORTED_SHAPE;
  // tile, item and partial-row counts are 32-bit
  if (max_tokens > (1 << 22) || max_reqs > (1 << 16) || nkv > 4096) return SPARK_ERR_TOO_LARGE;
  const paged::Layout l = paged::layout_of(max_tokens, max_reqs, nq, nkv, head_dim);
  if ((int64_t)l.max_items * nkv > (1 << 30) ||
      (int64_t)l.max_entries * nkv * l.tile_tok * (nq / nkv) > (1LL << 30))
    return SPARK_ERR_TOO_LARGE;
  return SPARK_OK;
}

int64_t spark_attn_plan_bytes(int max_tokens, int max_reqs, int nq, int nkv, int head_dim) {
  if (check_attn_shape(max_tokens, max_reqs, nq, nkv, head_dim)) return -1;
  return paged::layout_of(max_tokens, max_reqs, nq, nkv, head_dim).bytes;
}

int64_t spark_attn_part_rows(int max_tokens, int max_reqs, int nq, int nkv, int head_dim) {
  if (check_attn_shape(max_tokens, max_reqs, nq, nkv, head_dim)) return -1;
  return paged::layout_of(max_tokens, max_reqs, nq, nkv, head_dim).part_rows;
}

int spark_attn_plan(const int32_t* query_start, const int32_t* seq_lens, const int32_t* prefix_len, int reqs,
                    int max_tokens, int max_reqs, int nq, int nkv, int head_dim, int window, void* plan, int* error,
                    void* stream) {
  if (!seq_lens || !plan || !error || (query_start == nullptr) == (prefix_len == nullptr))
    return SPARK_ERR_INVALID_ARG;
  int st = check_attn_shape(max_tokens, max_reqs, nq, nkv, head_dim);
  if (st) return st;
  if (reqs < 0 || reqs > max_reqs || (prefix_len && reqs > max_tokens) || window < 0 || (prefix_len && window))
    return SPARK_ERR_UNSUPPORTED_SHAPE;
  if (!aligned(plan, 16)) return SPARK_ERR_ALIGNMENT;
  paged::AttnPlanArgs p;
  memset(&p, 0, sizeof(p));
  p.query_start = query_start, p.seq_lens = seq_lens, p.prefix_len = prefix_len;
  p.reqs = reqs, p.tokens = max_tokens, p.max_reqs = max_reqs, p.nq = nq, p.nkv = nkv, p.D = head_dim, p.window = window;
  p.lay = paged::layout_of(max_tokens, max_reqs, nq, nkv, head_dim);
  p.plan = static_cast<unsigned char*>(plan), p.error = error;
  return launch(paged::attn_plan_kernel, dim3(1), dim3(paged::kAttnPlanThreads), 0, as_stream(stream), p);
}

int spark_attn_paged_bounded(const uint16_t* q, int64_t q_tok_stride, int64_t q_head_stride, int tokens,
                             const uint16_t* k_cache, const uint16_t* v_cache, int64_t num_blocks, int block_size,
                             const int32_t* block_table, int64_t table_stride, int table_width, int table_rows,
                             int max_tokens, int max_reqs, int nq, int nkv, int head_dim, int window, float scale,
                             const void* plan, float* part_o, float* part_ml, uint16_t* out, int64_t out_tok_stride,
                             int64_t out_head_stride, int* error, int64_t wait_ns, void* stream) {
  if (!k_cache || !v_cache || !block_table || !plan || !part_o || !part_ml || !error) return SPARK_ERR_INVALID_ARG;
  int st = check_attn_shape(max_tokens, max_reqs, nq, nkv, head_dim);
  if (st) return st;
  if (tokens < 0 || tokens > max_tokens || num_blocks <= 0 || block_size < 16 || block_size % 16 ||
      table_width <= 0 || table_rows <= 0 || table_stride < 0 || window < 0 || !(scale > 0.0f) || scale > 1e30f)
    return SPARK_ERR_UNSUPPORTED_SHAPE;
  if (tokens == 0) return SPARK_OK;
  if (!q || !out) return SPARK_ERR_INVALID_ARG;
  if ((tokens > 1 && (q_tok_stride <= 0 || out_tok_stride <= 0)) ||
      (nq > 1 && (q_head_stride <= 0 || out_head_stride <= 0)))
    return SPARK_ERR_UNSUPPORTED_SHAPE;
  if (tokens == 1) q_tok_stride = (int64_t)nq * head_dim;  // (of no meaning: any valid pitch)
  if (nq == 1) q_head_stride = head_dim;
  // tensor-map coordinates are 32-bit rows of the caches
  if (num_blocks * nkv * block_size > 0x7fffffffLL - 128) return SPARK_ERR_TOO_LARGE;
  if (q_tok_stride % 8 || q_head_stride % 8 || out_tok_stride % 8 || out_head_stride % 8 || !aligned(q, 16) ||
      !aligned(k_cache, 16) || !aligned(v_cache, 16) || !aligned(out, 16) || !aligned(plan, 16) ||
      !aligned(part_o, 32) || !aligned(part_ml, 8))
    return SPARK_ERR_ALIGNMENT;
  paged::AttnArgs p;
  memset(&p, 0, sizeof(p));
  p.q = q, p.k_cache = k_cache, p.v_cache = v_cache, p.table = block_table, p.table_stride = table_stride;
  p.q_tok = q_tok_stride, p.q_head = q_head_stride, p.o_tok = out_tok_stride, p.o_head = out_head_stride;
  p.num_blocks = num_blocks, p.table_width = table_width, p.table_rows = table_rows, p.bs = block_size, p.tokens = tokens;
  p.max_tokens = max_tokens, p.max_reqs = max_reqs;
  p.nq = nq, p.nkv = nkv, p.window = window, p.scale = scale;
  p.plan = static_cast<const unsigned char*>(plan);
  p.lay = paged::layout_of(max_tokens, max_reqs, nq, nkv, head_dim);
  p.part_o = part_o, p.part_ml = reinterpret_cast<float2*>(part_ml), p.out = out, p.error = error;
  if (head_dim == 128) return attn_launch<128>(p, wait_ns, as_stream(stream));
  return attn_launch<256>(p, wait_ns, as_stream(stream));
}

int spark_attn_paged(const uint16_t* q, int64_t q_tok_stride, int64_t q_head_stride, int tokens,
                     const uint16_t* k_cache, const uint16_t* v_cache, int64_t num_blocks, int block_size,
                     const int32_t* block_table, int64_t table_stride, int table_width, int max_tokens, int max_reqs,
                     int nq, int nkv, int head_dim, int window, float scale, const void* plan, float* part_o,
                     float* part_ml, uint16_t* out, int64_t out_tok_stride, int64_t out_head_stride, int* error,
                     int64_t wait_ns, void* stream) {
  return spark_attn_paged_bounded(q, q_tok_stride, q_head_stride, tokens, k_cache, v_cache, num_blocks, block_size,
                                  block_table, table_stride, table_width, max_reqs, max_tokens, max_reqs, nq, nkv,
                                  head_dim, window, scale, plan, part_o, part_ml, out, out_tok_stride,
                                  out_head_stride, error, wait_ns, stream);
}

}  // extern "C"
