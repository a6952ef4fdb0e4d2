// Attention over the 8-bit paged cache, and attention for trees of drafted
// tokens over either cache.
//
// Query rows of a sequence follow its committed tokens; row j of n sees the
// keys a mask gives it: all positions up to its own (causal), or the
// committed ones and its ancestors among the drafted (tree).  For the cached
// row (codes c, scale s) of a key, score and output are
//   x_t = scale * s_t * (q . c_t),   o = sum_t w_t s'_t c'_t / sum_t w_t,
//   w_t = exp(x_t - max)
// with the codes taken as they are and the scales applied to fp32 values.  The
// kernels are in kv_tiles.h and kv_narrow.h; here are the ancestor bits, how a
// call is split into launches, and the entry points.
#include <algorithm>
#include <atomic>

#include "kv_attention.h"

namespace lv {

// Ancestor bits: thread per drafted token walks up its parents, whose indices
// fall, so that every walk ends.  Bound by the latency of that chain, one read
// from L2 a level.
__global__ __launch_bounds__(256) void tree_mask_kernel(const int32_t* __restrict__ parents,
                                                        const int32_t* __restrict__ cu,
                                                        int num_seqs, int num_tokens,
                                                        uint64_t* __restrict__ mask, int words) {
  const int row = blockIdx.x * 256 + threadIdx.x;
  if (row >= num_tokens) return;
  int lo = 0, hi = num_seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= row) lo = mid; else hi = mid - 1;
  }
  const int q0 = cu[lo];
  if (q0 < 0 || row < q0 || row >= cu[lo + 1]) return;
  uint64_t* out = mask + (int64_t)row * words;
  int at = row - q0;
  for (int w = words - 1; w >= 0; --w) {     // the walk meets the words from the last down
    uint64_t bits = 0;
    while (at >= 64 * w) {
      if (at < 64 * (w + 1)) bits |= 1ull << (at & 63);
      const int up = parents[q0 + at];
      at = up < at ? up : -1;
      if (at < 0) break;
    }
    out[w] = bits;
  }
}

LV_ERROR_WORD_READER(read_errors_tree)

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
namespace {

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

// CUs of the current device (looked up once per device).
int device_cus() {
  static std::atomic<int> known[64];
  int dev = 0, n = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  n = known[dev].load(std::memory_order_relaxed);
  if (n > 0) return n;
  if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0)
    n = 256;
  known[dev].store(n, std::memory_order_relaxed);
  return n;
}

// How the sequences of a part are launched.  Everything here follows from the
// sizes the caller names, never from what is in device memory.  `codes`: an
// 8-bit cache whose strides the narrow kernel takes.
TilePlan plan_tiles(int seq_begin, int n_seqs, int max_q, int num_heads, int num_kv_heads,
                    int head_dim, int max_blocks, lv_dtype dtype, bool codes) {
  TilePlan p{};
  p.seq_begin = seq_begin;
  p.n_seqs = n_seqs;
  p.max_q = max_q;
  const int64_t rows = std::max<int64_t>(1, (int64_t)max_q * (num_heads / num_kv_heads));
  const bool f32 = dtype == LV_F32;
  const int64_t cus = device_cus();
  const int64_t groups = (int64_t)n_seqs * num_kv_heads;
  auto units_of = [&](int r) { return groups * ((rows + r - 1) / r); };
  p.rw = rows <= 32 ? 1 : rows <= 64 ? 2 : rows <= 128 || f32 ? 4 : 8;
  p.waves = 4;
  // Eight wavefronts (one workgroup a CU, two for four) pay where a workgroup
  // stays with long rows: few units, or long contexts of codes, whose way into
  // LDS they share.  Where there are many short units two workgroups hide each
  // other's starts.  us with eight | four: 48 trees of 40-64 tokens at 500-4000
  // 136 | 142, of 12-16 tokens 100 | 114, 4 over codes at 2000-16000 39 | 50, two
  // chunks of 700-1024 at 15000-19000 372 | 413, 60 chunks of 100 at 0-3000
  // 170 | 188; 256 trees of 40-64 at 300-1000 317 | 224, at 1000-3000 616 | 537,
  // 60 chunks of 100 at 0-300 60 | 51.  33-64 rows on four wavefronts are half
  // a unit of RW = 4, since RW = 2 on four has too few registers (48 trees of
  // 20-32 tokens at 500-4000 173, RW = 4 125, RW = 2 on eight 102).  Up to 32
  // rows over codes stay with four (16 trees of 4-8 tokens at 2000-16000 98 |
  // 72).  fp32 keeps to four: its registers and LDS are those of one wavefront a
  // SIMD.
  if (!f32) {
    const int wide = std::max(p.rw, 2);
    if (max_blocks > 32 && (p.rw > 1 || !codes) &&
        ((codes && max_blocks > 128) || 2 * units_of(32 * wide) <= 3 * cus)) {
      p.rw = wide;
      p.waves = 8;
    } else if (p.rw > 1) {
      p.rw = 4;
    }
  }
  const int r = 32 * p.rw, kt = p.rw == 4 && p.waves == 4 ? 64 : 128;
  const int64_t units = units_of(r);
  const int64_t tiles = std::max<int64_t>(1, ((int64_t)max_blocks * kBs + kt - 1) / kt);
  p.nq = (int)((rows + r - 1) / r);
  p.list = units * tiles;
  const int64_t at_once = cus * (f32 || p.waves == 8 ? 1 : 2);
  p.ranges = (int)std::min<int64_t>(p.list, at_once);
  p.grid = p.ranges;
  const bool one_round = units <= at_once;
  const int64_t all = (groups + kXcds - 1) / kXcds * kXcds * p.nq;
  if (all < (1ll << 31)) {
    // Contexts of a few tiles are not split where all units run at once (a join
    // takes as long as two tiles or three: 3 decode rows of 40-300 keys 7.9 us,
    // split, by the narrow kernel, 10.4, and 11.0 where the table is wide; up to 8 tiles a tree of 700
    // keys takes 15.0, split 13.4).  Where there are half as many units again as
    // run at once, the kernel looks whether they need to be (15 chunks of 512
    // at 0-3071 203 us, split 265).
    p.direct = one_round && tiles <= 4 ? 3 : tiles <= 2 ? 2 : 2 * units >= 3 * p.ranges ? 1 : 0;
    if (p.direct) p.grid = (int)std::max<int64_t>(all, p.direct == 1 ? p.ranges : 0);
  }
  p.slot_heads = 1;
  p.slot_rows = (int)std::min<int64_t>(rows, r);
  // (64 decode rows of 256-4096 keys, 8 heads a kv head: 40.6 us, as tiles 45.3;
  // 256 of 16-2048, 2 heads: 103, as tiles 174)
  if (codes && !f32 && rows <= 8 && p.direct != 3) {
    p.rw = 0;
    p.direct = 0;
    p.slot_heads = std::min(num_kv_heads, 8);
    while (num_kv_heads % p.slot_heads != 0) --p.slot_heads;
    p.list = (int64_t)n_seqs * (num_kv_heads / p.slot_heads) * std::max(1, (max_blocks + 1) / 2);
    p.grid = p.ranges = (int)std::min<int64_t>(p.list, cus * (8 / p.slot_heads));
  }
  if (p.direct < 2) {
    const size_t slots = (size_t)2 * p.ranges * p.slot_heads * p.slot_rows;
    p.head_bytes = align256((size_t)p.ranges * 2 * 16);
    p.ml_bytes = align256(slots * 8);
    p.acc_bytes = align256(slots * head_dim * 4);
  }
  return p;
}

size_t plan_bytes(const TilePlan& p) { return p.head_bytes + p.ml_bytes + p.acc_bytes; }

// The parts of a call, one launch (and its join) each: its decode rows, then its
// other sequences, kPartSeqs at a time.  f(plan) until one does not return LV_OK.
template <typename F>
int for_each_part(int num_seqs, int num_decodes, int max_query_len, int num_heads,
                  int num_kv_heads, int head_dim, int max_blocks, lv_dtype dtype, bool codes, F f) {
  for (int i = 0, n; i < num_seqs; i += n) {
    const bool decodes = i < num_decodes;
    n = std::min(kPartSeqs, (decodes ? num_decodes : num_seqs) - i);
    if (const int rc = f(plan_tiles(i, n, decodes ? 1 : max_query_len, num_heads, num_kv_heads,
                                    head_dim, max_blocks, dtype, codes));
        rc != LV_OK)
      return rc;
  }
  return LV_OK;
}

size_t workspace_size(int num_seqs, int num_decodes, int max_query_len, int num_heads,
                      int num_kv_heads, int head_dim, int max_blocks, lv_dtype dtype) {
  // (of an 8-bit cache or not: the larger need)
  if (num_seqs <= 0 || num_kv_heads <= 0 || num_heads < num_kv_heads || max_blocks < 0) return 0;
  size_t need = 0;
  for (const bool codes : {false, true})
    for_each_part(num_seqs, num_decodes, max_query_len, num_heads, num_kv_heads, head_dim,
                  max_blocks, dtype, codes, [&](const TilePlan& p) {
                    need = std::max(need, plan_bytes(p));
                    return LV_OK;
                  });
  return need;
}

int launch_part(const Call& a, const TilePlan& p, char* ws) {
  if (a.dtype == LV_F32) return launch_tiles_f32(a, p, ws);
  if (a.dtype == LV_F16) return launch_tiles_f16(a, p, ws);
  return launch_tiles_bf16(a, p, ws);
}

int launch(const Call& a, int num_decodes, int max_query_len, void* ws) {
  // (the narrow kernel's offsets within a block are 32 bits wide)
  const bool codes = a.code >= 0 && a.c.tok <= (1 << 26);
  return for_each_part(a.b.num_seqs, num_decodes, max_query_len, a.r.num_heads, a.r.num_kv_heads,
                       a.d, a.b.max_blocks, a.dtype, codes,
                       [&](const TilePlan& p) { return launch_part(a, p, (char*)ws); });
}

// The checks common to the attention entries; fills `a` but for the cache.
int check_call(const char* who, Call& a, int num_decodes, const void* query, int64_t q_stride,
               const int32_t* tables, int max_blocks, const int32_t* cu, const int32_t* ctx,
               int num_seqs, int64_t num_tokens, int max_query_len, int num_heads,
               int num_kv_heads, int head_dim, int block_size, float scale, void* out,
               int64_t out_stride, const void* ws, size_t ws_bytes, lv_dtype dtype) {
  LV_REQUIRE(dtype == LV_F32 || dtype == LV_F16 || dtype == LV_BF16, "%s: bad dtype", who);
  LV_REQUIRE(num_seqs >= 0 && num_tokens >= 0 && max_blocks >= 0 && max_query_len >= 0,
             "%s: negative size", who);
  LV_REQUIRE(num_tokens < (1ll << 31), "%s: num_tokens does not fit in 32 bits", who);
  LV_REQUIRE(max_blocks < (1 << 27), "%s: max_blocks * 16 does not fit in 32 bits", who);
  LV_REQUIRE(num_heads > 0 && num_kv_heads > 0 && num_heads % num_kv_heads == 0,
             "%s: num_heads must be a multiple of num_kv_heads", who);
  if ((head_dim != 64 && head_dim != 128) || block_size != kBs || num_heads > 65535) {
    set_error("%s: head_dim %d, block_size %d, %d heads (head_dim 64 or 128, block_size 16 and "
              "up to 65535 heads are supported)", who, head_dim, block_size, num_heads);
    return LV_ERR_UNSUPPORTED;
  }
  if (num_seqs == 0 || num_tokens == 0) return LV_OK;
  LV_REQUIRE(query && out && ctx && (tables || max_blocks == 0), "%s: null pointer", who);
  LV_REQUIRE(cu || num_tokens == num_seqs, "%s: without cu_seqlens every sequence has one row",
             who);
  const int64_t row = (int64_t)num_heads * head_dim;
  LV_REQUIRE((q_stride >= row && out_stride >= row) || num_tokens == 1,
             "%s: token stride smaller than num_heads*head_dim", who);
  const size_t es = dtype_size(dtype);
  LV_REQUIRE(aligned16(query) && aligned16(out) && (q_stride * es) % 16 == 0 &&
                 (out_stride * es) % 16 == 0,
             "%s: query and out rows must be 16-byte aligned", who);
  a.b.block_tables = tables; a.b.max_blocks = max_blocks;
  a.b.cu = cu; a.b.ctx = ctx;
  a.b.num_seqs = num_seqs; a.b.num_tokens = (int)num_tokens;
  a.r.q = query; a.r.q_stride = q_stride; a.r.out = out; a.r.out_stride = out_stride;
  a.r.num_heads = num_heads; a.r.num_kv_heads = num_kv_heads;
  a.r.scale_log2 = scale * 1.4426950408889634f;
  a.d = head_dim; a.dtype = dtype;
  if (num_seqs > 16384) {
    set_error("%s: %d sequences (up to 16384 are supported)", who, num_seqs);
    return LV_ERR_UNSUPPORTED;
  }
  bool fits = max_query_len * (int64_t)(num_heads / num_kv_heads) < (1ll << 30);
  for (const bool codes : {false, true})
    for_each_part(num_seqs, num_decodes, max_query_len, num_heads, num_kv_heads, head_dim,
                  max_blocks, dtype, codes, [&](const TilePlan& p) {
                    fits = fits && p.list < (1ll << 31) - (1 << 16);
                    return LV_OK;
                  });
  LV_REQUIRE(fits, "%s: too many keys and rows for 32-bit offsets", who);
  const size_t need = workspace_size(num_seqs, num_decodes, max_query_len, num_heads, num_kv_heads,
                                     head_dim, max_blocks, dtype);
  if (need > 0 && (!ws || ((uintptr_t)ws & 255) != 0 || ws_bytes < need)) {
    set_error("%s: workspace of %zu bytes (256-byte aligned) needed, got %zu", who, need,
              ws ? ws_bytes : (size_t)0);
    return LV_ERR_WORKSPACE;
  }
  return LV_OK;
}

void use_cache(Call& a, const lv_quant_cache* c) {
  a.c = KvView{{c->key_dev, c->value_dev}, {c->key_scale_dev, c->value_scale_dev},
               c->stride_block, c->stride_token, c->stride_head,
               c->scale_stride_block, c->scale_stride_token, c->scale_stride_head, c->num_blocks};
  a.code = c->code;
}

int check_mask(const char* who, Call& a, const uint64_t* mask, int words, int max_query_len,
               int64_t num_tokens) {
  LV_REQUIRE(words >= 1 && (int64_t)words * 64 >= max_query_len,
             "%s: mask_words * 64 must be at least max_query_len", who);
  LV_REQUIRE((mask && ((uintptr_t)mask & 7) == 0) || num_tokens == 0,
             "%s: null or unaligned tree_mask", who);
  a.b.mask = mask;
  a.b.mask_words = words;
  a.tree = true;
  return LV_OK;
}

}  // namespace
}  // namespace lv

extern "C" size_t lv_paged_attention_quant_workspace_size(int32_t num_seqs, int32_t num_decodes,
                                                          int64_t num_tokens,
                                                          int32_t max_query_len,
                                                          int32_t num_heads,
                                                          int32_t num_kv_heads, int32_t head_dim,
                                                          int32_t max_blocks, lv_dtype dtype) {
  return lv::workspace_size(num_seqs, num_decodes, max_query_len, num_heads, num_kv_heads,
                            head_dim, max_blocks, dtype);
}

extern "C" size_t lv_tree_attention_workspace_size(int32_t num_seqs, int64_t num_tokens,
                                                   int32_t max_query_len, int32_t num_heads,
                                                   int32_t num_kv_heads, int32_t head_dim,
                                                   int32_t max_blocks, lv_dtype dtype) {
  return lv::workspace_size(num_seqs, 0, max_query_len, num_heads, num_kv_heads, head_dim,
                            max_blocks, dtype);
}

extern "C" int lv_paged_attention_quant(
    const void* query_dev, int64_t q_stride_t, const lv_quant_cache* cache,
    const int32_t* block_tables_dev, int32_t max_blocks, const int32_t* cu_seqlens_dev,
    const int32_t* context_lens_dev, int32_t num_seqs, int32_t num_decodes, int64_t num_tokens,
    int32_t max_query_len, int32_t num_heads, float scale, void* out_dev, int64_t out_stride_t,
    void* workspace_dev, size_t workspace_bytes, lv_dtype dtype, void* stream) {
  using namespace lv;
  constexpr const char* who = "lv_paged_attention_quant";
  clear_error();
  if (const int rc = check_quant_cache(who, cache); rc != LV_OK) return rc;
  LV_REQUIRE(num_decodes >= 0 && num_decodes <= num_seqs && num_decodes <= num_tokens,
             "%s: num_decodes %d outside [0, num_seqs]", who, num_decodes);
  Call a{};
  if (const int rc = check_call(who, a, num_decodes, query_dev, q_stride_t, block_tables_dev, max_blocks,
                                cu_seqlens_dev, context_lens_dev, num_seqs, num_tokens,
                                max_query_len, num_heads, cache->num_kv_heads, cache->head_dim,
                                cache->block_size, scale, out_dev, out_stride_t, workspace_dev,
                                workspace_bytes, dtype);
      rc != LV_OK || num_seqs == 0 || num_tokens == 0)
    return rc;
  use_cache(a, cache);
  a.stream = (hipStream_t)stream;
  return launch(a, num_decodes, max_query_len, workspace_dev);
}

extern "C" int lv_tree_attention(
    const void* query_dev, int64_t q_stride_t, const void* key_cache_dev,
    const void* value_cache_dev, int64_t num_cache_blocks, const int32_t* block_tables_dev,
    int32_t max_blocks, const int32_t* cu_seqlens_dev, const int32_t* context_lens_dev,
    const uint64_t* tree_mask_dev, int32_t mask_words, int32_t num_seqs, int64_t num_tokens,
    int32_t max_query_len, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t block_size, float scale, void* out_dev, int64_t out_stride_t, void* workspace_dev,
    size_t workspace_bytes, lv_dtype dtype, void* stream) {
  using namespace lv;
  constexpr const char* who = "lv_tree_attention";
  clear_error();
  Call a{};
  if (const int rc = check_mask(who, a, tree_mask_dev, mask_words, max_query_len, num_tokens);
      rc != LV_OK)
    return rc;
  LV_REQUIRE(num_cache_blocks > 0, "%s: bad cache geometry", who);
  if (const int rc = check_call(who, a, 0, query_dev, q_stride_t, block_tables_dev, max_blocks,
                                cu_seqlens_dev, context_lens_dev, num_seqs, num_tokens,
                                max_query_len, num_heads, num_kv_heads, head_dim, block_size,
                                scale, out_dev, out_stride_t, workspace_dev, workspace_bytes,
                                dtype);
      rc != LV_OK || num_seqs == 0 || num_tokens == 0)
    return rc;
  LV_REQUIRE(cu_seqlens_dev, "%s: null cu_seqlens", who);
  LV_REQUIRE(key_cache_dev && value_cache_dev && aligned16(key_cache_dev) &&
                 aligned16(value_cache_dev),
             "%s: null or unaligned cache", who);
  const int64_t tok = (int64_t)num_kv_heads * head_dim;
  a.c = KvView{{key_cache_dev, value_cache_dev}, {nullptr, nullptr}, kBs * tok, tok, head_dim,
               0, 0, 0, num_cache_blocks};
  a.code = -1;
  a.stream = (hipStream_t)stream;
  return launch(a, 0, max_query_len, workspace_dev);
}

extern "C" int lv_tree_attention_quant(
    const void* query_dev, int64_t q_stride_t, const lv_quant_cache* cache,
    const int32_t* block_tables_dev, int32_t max_blocks, const int32_t* cu_seqlens_dev,
    const int32_t* context_lens_dev, const uint64_t* tree_mask_dev, int32_t mask_words,
    int32_t num_seqs, int64_t num_tokens, int32_t max_query_len, int32_t num_heads, float scale,
    void* out_dev, int64_t out_stride_t, void* workspace_dev, size_t workspace_bytes,
    lv_dtype dtype, void* stream) {
  using namespace lv;
  constexpr const char* who = "lv_tree_attention_quant";
  clear_error();
  if (const int rc = check_quant_cache(who, cache); rc != LV_OK) return rc;
  Call a{};
  if (const int rc = check_mask(who, a, tree_mask_dev, mask_words, max_query_len, num_tokens);
      rc != LV_OK)
    return rc;
  if (const int rc = check_call(who, a, 0, query_dev, q_stride_t, block_tables_dev, max_blocks,
                                cu_seqlens_dev, context_lens_dev, num_seqs, num_tokens,
                                max_query_len, num_heads, cache->num_kv_heads, cache->head_dim,
                                cache->block_size, scale, out_dev, out_stride_t, workspace_dev,
                                workspace_bytes, dtype);
      rc != LV_OK || num_seqs == 0 || num_tokens == 0)
    return rc;
  LV_REQUIRE(cu_seqlens_dev, "%s: null cu_seqlens", who);
  use_cache(a, cache);
  a.stream = (hipStream_t)stream;
  return launch(a, 0, max_query_len, workspace_dev);
}

extern "C" int lv_tree_mask(const int32_t* parents_dev, const int32_t* cu_seqlens_dev,
                            int32_t num_seqs, int64_t num_tokens, uint64_t* tree_mask_dev,
                            int32_t mask_words, void* stream) {
  using namespace lv;
  clear_error();
  LV_REQUIRE(num_seqs >= 0 && num_tokens >= 0 && num_tokens < (1ll << 31),
             "lv_tree_mask: bad sizes");
  LV_REQUIRE(mask_words >= 1 && mask_words <= 16, "lv_tree_mask: mask_words must be 1 to 16");
  if (num_seqs == 0 || num_tokens == 0) return LV_OK;
  LV_REQUIRE(parents_dev && cu_seqlens_dev && tree_mask_dev && ((uintptr_t)tree_mask_dev & 7) == 0,
             "lv_tree_mask: null or unaligned pointer");
  tree_mask_kernel<<<(unsigned)((num_tokens + 255) / 256), 256, 0, (hipStream_t)stream>>>(
      parents_dev, cu_seqlens_dev, num_seqs, (int)num_tokens, tree_mask_dev, mask_words);
  return check_launch("lv_tree_mask");
}
