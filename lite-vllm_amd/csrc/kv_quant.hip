// The quantised K/V cache's writers and reader.
//
//  * kv_scatter_quant: K and V rows of the step's tokens into the cache at
//      slot_mapping, as codes and a scale per (token, kv head) -- the 8-bit
//      form of Attention.forward's scatter (reference
//      litevllm/layers/attention.py:79-84, write_to_cache 17-33).
//  * kv_gather_quant: the values of the rows at given slots.
//  * qk_norm_rope_cache_quant: the attention prologue of a layer (reference
//      models/qwen3.py:75-84, layers/rotary_emb.py:92-117) ending in such a
//      write.  q and k stay in fp32 from the projection to the query's
//      rounding and the codes.
//
// All three move each byte once and are bound by HBM, or by latency for a
// decode step's few rows.  A lane owns 8 dims (in the prologue 8 rotation
// pairs), so a row's codes go out 8 bytes a lane and its scale is a maximum
// over D / 8 (D / 16) lanes by row operations, with no LDS.  Wider lanes (16
// dims) would halve the lanes that a few rows keep busy; narrower ones would
// not fill a 16-byte load of 16-bit values.
#include "lv_common.h"
#include "lv_quant.h"

namespace lv {

constexpr int kQuantThreads = 256;

// Where the cache's codes and scales lie; strides in elements.
struct QuantView {
  uint8_t* code[2];     // key, value
  float* scale[2];
  int64_t blk, tok, head;        // of the codes
  int64_t sblk, stok, shead;     // of the scales
  int64_t num_slots;
  int block_size, block_shift;   // shift: log2 of the size, or -1
};

// Scatter and gather: 64-bit divisions took more instructions than the rest of a
// row, so the workgroup divides once, in scalars, and a lane divides the small
// rest (7872 tokens written and read back 26.2 -> 25.0 us).  The prologue, which
// waits longer for its loads, divides: with these it took 30.0 us for 4099
// tokens, read back, against 26.4.
struct RowOf { int64_t token; int head_slot; };
template <int W>
__device__ __forceinline__ RowOf row_of(int per_token) {
  const int64_t first = (int64_t)blockIdx.x * (kQuantThreads / W);
  const int64_t t0 = first / per_token;
  const unsigned rem = (unsigned)(first - t0 * per_token) + threadIdx.x / W;
  const unsigned up = rem / (unsigned)per_token;
  return {t0 + up, (int)(rem - up * per_token)};
}

struct SlotOf { int64_t block; int offset; };
__device__ __forceinline__ SlotOf slot_of(const QuantView& c, int64_t slot) {
  if (c.block_shift >= 0)
    return {slot >> c.block_shift, (int)(slot & (c.block_size - 1))};
  const int64_t blk = slot / c.block_size;
  return {blk, (int)(slot - blk * c.block_size)};
}

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, float* x) {
  if constexpr (VEC && elem<T>::kPer16B == 8) {
    elem<T>::unpack(load16(p), x);
  } else if constexpr (VEC) {
    elem<T>::unpack(load16(p), x);
    elem<T>::unpack(load16(p + 4), x + 4);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = elem<T>::load(p + i);
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, const float* x) {
  if constexpr (VEC && elem<T>::kPer16B == 8) {
    store16(p, pack16<T>(x));
  } else if constexpr (VEC) {
    store16(p, pack16<T>(x));
    store16(p + 4, pack16<T>(x + 4));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) elem<T>::store(p + i, x[i]);
  }
}

template <typename C>
__device__ __forceinline__ void store_codes8(uint8_t* p, const float* y) {
  *reinterpret_cast<uint2*>(p) = make_uint2(code<C>::pack4(y), code<C>::pack4(y + 4));
}

// W = D / 8 lanes per (token, K or V, kv head): code = x / max|x| * top, the
// exact quotient (lv_quant.h).  7872 bf16 tokens of 8 heads of 128 to e4m3:
// 14.1 us, 49 MB at 3.5 TB/s; the exact quotients' vector instructions and HBM
// (10 us) overlap in part.  61 tokens: 3.5 us, one chain of slot,
// scale and store.
template <typename T, typename C, int D, bool VEC>
__global__ __launch_bounds__(kQuantThreads) void kv_scatter_quant_kernel(
    const T* __restrict__ key, int64_t key_stride, const T* __restrict__ value,
    int64_t value_stride, QuantView c, const int64_t* __restrict__ slots, int64_t num_tokens,
    int num_kv_heads) {
  constexpr int W = D / 8;
  const int i = (threadIdx.x & (W - 1)) * 8;
  const RowOf row = row_of<W>(2 * num_kv_heads);
  const int64_t t = row.token;
  if (t >= num_tokens) return;      // whole groups leave together (W divides 64)
  const int hs = row.head_slot;
  const int kv = hs >= num_kv_heads, head = hs - kv * num_kv_heads;
  const int64_t slot = slots[t];
  float x[8];       // (loaded beside the slot, not after it)
  load8<T, VEC>((kv ? value + t * value_stride : key + t * key_stride) + (int64_t)head * D + i, x);
  if (slot < 0) return;                      // padding
  if (slot >= c.num_slots) {                 // outside the cache: not written, reported
    if (hs == 0 && i == 0) report_device_error(LV_DEVERR_SLOT);
    return;
  }
  const float scale = row_scale<C, W, 8>(x);
  const auto [blk, off] = slot_of(c, slot);
  store_codes8<C>(c.code[kv] + blk * c.blk + off * c.tok + head * c.head + i, x);
  if (i == 0) c.scale[kv][blk * c.sblk + off * c.stok + head * c.shead] = scale;
}

// value = code * scale, one rounding.  Rows at slots outside the cache
// (negative: padding) are zeros.  The same 7872 tokens read back: 11.4 us,
// 4.3 TB/s, bound by HBM; 61 tokens: 3.0 us, bound by the chain slot, code,
// store.
template <typename T, typename C, int D, bool VEC>
__global__ __launch_bounds__(kQuantThreads) void kv_gather_quant_kernel(
    QuantView c, const int64_t* __restrict__ slots, int64_t num_tokens, int num_kv_heads,
    T* __restrict__ key, int64_t key_stride, T* __restrict__ value, int64_t value_stride) {
  constexpr int W = D / 8;
  const int i = (threadIdx.x & (W - 1)) * 8;
  const RowOf row = row_of<W>(2 * num_kv_heads);
  const int64_t t = row.token;
  if (t >= num_tokens) return;
  const int hs = row.head_slot;
  const int kv = hs >= num_kv_heads, head = hs - kv * num_kv_heads;
  const int64_t slot = slots[t];
  float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (slot >= c.num_slots && hs == 0 && i == 0) report_device_error(LV_DEVERR_SLOT);
  if (slot >= 0 && slot < c.num_slots) {
    const auto [blk, off] = slot_of(c, slot);
    const uint2 w = *reinterpret_cast<const uint2*>(c.code[kv] + blk * c.blk + off * c.tok +
                                                    head * c.head + i);
    const float scale = c.scale[kv][blk * c.sblk + off * c.stok + head * c.shead];
    code<C>::unpack4(w.x, x);
    code<C>::unpack4(w.y, x + 4);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] *= scale;
  }
  store8<T, VEC>((kv ? value + t * value_stride : key + t * key_stride) + (int64_t)head * D + i, x);
}

// W = D / 16 lanes per (token, head slot), head slots as in
// qk_norm_rope_cache: queries, keys, values.  Lane i owns the rotation pairs
// (8 i + j, 8 i + j + D / 2), so the rotation crosses no lanes: per row the
// norm's sum of squares, x cos - y sin and y cos + x sin in fp32, and for K and V
// the scale and codes of the fp32 result (rounding it to T first would be a
// second rounding of what is rounded to 8 bits).  Slot, position, row and norm
// weights are read at once; cos and sin follow the position.  256 tokens of
// 16 + 8 + 8 heads of 128: 4.2 us, bound by that chain.
template <typename T, typename C, int D, bool VEC>
__global__ __launch_bounds__(kQuantThreads) void qk_norm_rope_cache_quant_kernel(
    const T* __restrict__ qkv, int64_t qkv_stride, const T* __restrict__ q_norm_w,
    const T* __restrict__ k_norm_w, const T* __restrict__ cos_cache,
    const T* __restrict__ sin_cache, int64_t max_position, const int64_t* __restrict__ positions,
    const int64_t* __restrict__ slots, T* __restrict__ q_out, int64_t q_out_stride, QuantView c,
    int64_t num_tokens, int num_heads, int num_kv_heads, float eps) {
  constexpr int HALF = D / 2, W = HALF / 8;
  const int i = (threadIdx.x & (W - 1)) * 8;
  const int per_token = num_heads + 2 * num_kv_heads;
  const int64_t row = ((int64_t)blockIdx.x * kQuantThreads + threadIdx.x) / W;
  const int64_t t = row / per_token;
  if (t >= num_tokens) return;
  const int hs = (int)(row - t * per_token);
  const int64_t pos = positions[t];
  const int64_t slot = slots[t];
  const T* src = qkv + t * qkv_stride + (int64_t)hs * D + i;
  float x[16];       // the pairs' first members, then their second ones
  load8<T, VEC>(src, x);
  load8<T, VEC>(src + HALF, x + 8);
  const bool is_q = hs < num_heads, is_v = hs >= num_heads + num_kv_heads;
  const T* nw = is_q ? q_norm_w : is_v ? nullptr : k_norm_w;
  float w[16];
  if (nw) {
    load8<T, VEC>(nw + i, w);
    load8<T, VEC>(nw + i + HALF, w + 8);
  }
  if (!is_q) {       // padding, and slots outside the cache (reported): nothing is written
    if (slot >= c.num_slots && hs == num_heads && i == 0) report_device_error(LV_DEVERR_SLOT);
    if (slot < 0 || slot >= c.num_slots) return;
  }
  if (!is_v) {
    // a position without a cos / sin row makes the output NaN
    const bool pos_ok = pos >= 0 && pos < max_position;
    const int64_t prow = (pos_ok ? pos : 0) * HALF + i;
    float cs[8], sn[8];
    load8<T, VEC>(cos_cache + prow, cs);
    load8<T, VEC>(sin_cache + prow, sn);
    if (nw) {
      float ss = 0.0f;
#pragma unroll
      for (int j = 0; j < 16; ++j) ss += x[j] * x[j];
      ss = group_sum<W>(ss);
      const float inv = rsqrtf(ss / (float)D + eps);
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = x[j] * inv * w[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float co = pos_ok ? cs[j] : __builtin_nanf(""), si = pos_ok ? sn[j] : __builtin_nanf("");
      const float a = x[j], b = x[j + 8];
      x[j] = a * co - b * si;
      x[j + 8] = b * co + a * si;
    }
    if (is_q) {
      T* dst = q_out + t * q_out_stride + (int64_t)hs * D + i;
      store8<T, VEC>(dst, x);
      store8<T, VEC>(dst + HALF, x + 8);
      return;
    }
  }
  const int head = hs - num_heads - (is_v ? num_kv_heads : 0);
  const float scale = row_scale<C, W, 16>(x);
  const int64_t blk = slot / c.block_size;
  const int off = (int)(slot - blk * c.block_size);
  uint8_t* dst = c.code[is_v] + blk * c.blk + off * c.tok + head * c.head + i;
  store_codes8<C>(dst, x);
  store_codes8<C>(dst + HALF, x + 8);
  if (i == 0) c.scale[is_v][blk * c.sblk + off * c.stok + head * c.shead] = scale;
}

LV_ERROR_WORD_READER(read_errors_quant)

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

// Checks a cache description; the message names `who`.
int check_quant_cache(const char* who, const lv_quant_cache* c) {
  LV_REQUIRE(c != nullptr, "%s: null cache", who);
  LV_REQUIRE(c->code == LV_INT8 || c->code == LV_E4M3, "%s: bad code type", who);
  LV_REQUIRE(c->num_blocks > 0 && c->block_size > 0 && c->num_kv_heads > 0,
             "%s: bad cache geometry", who);
  LV_REQUIRE(c->key_dev && c->value_dev && c->key_scale_dev && c->value_scale_dev,
             "%s: null cache pointer", who);
  const int64_t sizes[3] = {c->num_blocks, c->block_size, c->num_kv_heads};
  const int64_t strides[3] = {c->stride_block, c->stride_token, c->stride_head};
  const int64_t sstrides[3] = {c->scale_stride_block, c->scale_stride_token,
                               c->scale_stride_head};
  for (int i = 0; i < 3; ++i) {
    LV_REQUIRE(strides[i] % 16 == 0 && (strides[i] >= c->head_dim || sizes[i] == 1),
               "%s: cache strides must be multiples of 16 and at least head_dim", who);
    LV_REQUIRE(sstrides[i] > 0 || sizes[i] == 1, "%s: scale strides must be positive", who);
  }
  LV_REQUIRE(aligned16(c->key_dev) && aligned16(c->value_dev), "%s: codes not 16-byte aligned",
             who);
  LV_REQUIRE(((uintptr_t)c->key_scale_dev & 3) == 0 && ((uintptr_t)c->value_scale_dev & 3) == 0,
             "%s: scales not 4-byte aligned", who);
  return LV_OK;
}

namespace {

QuantView view_of(const lv_quant_cache* c) {
  QuantView v;
  v.code[0] = (uint8_t*)c->key_dev;
  v.code[1] = (uint8_t*)c->value_dev;
  v.scale[0] = c->key_scale_dev;
  v.scale[1] = c->value_scale_dev;
  v.blk = c->stride_block; v.tok = c->stride_token; v.head = c->stride_head;
  v.sblk = c->scale_stride_block; v.stok = c->scale_stride_token; v.shead = c->scale_stride_head;
  v.block_size = c->block_size;
  v.block_shift = (c->block_size & (c->block_size - 1)) == 0 ? __builtin_ctz(c->block_size) : -1;
  v.num_slots = c->num_blocks * c->block_size;
  return v;
}

// Workgroups for `rows` rows of `lanes` lanes; 0 if there are too many.
unsigned grid_of(int64_t rows, int lanes) {
  const int64_t g = (rows * lanes + kQuantThreads - 1) / kQuantThreads;
  return g < (1ll << 31) ? (unsigned)g : 0u;
}

template <typename F>
int by_code(int code, F&& f) {
  return code == LV_INT8 ? f(int8_code{}) : f(e4m3_code{});
}
template <typename F>
int by_type(lv_dtype dt, F&& f) {
  return dt == LV_F32 ? f(float{}) : dt == LV_F16 ? f(f16{}) : f(bf16{});
}
template <typename F>
int by_dim(int d, F&& f) {
  return d == 64 ? f(std::integral_constant<int, 64>{})
       : d == 128 ? f(std::integral_constant<int, 128>{})
                  : f(std::integral_constant<int, 256>{});
}
template <typename F>
int by_bool(bool b, F&& f) {
  return b ? f(std::true_type{}) : f(std::false_type{});
}

bool aligned_rows(const void* p, int64_t stride, lv_dtype dt) {
  return aligned16(p) && (stride * (int64_t)dtype_size(dt)) % 16 == 0;
}

int check_common(const char* who, const lv_quant_cache* c, lv_dtype dt, int64_t num_tokens) {
  LV_REQUIRE(dt == LV_F32 || dt == LV_F16 || dt == LV_BF16, "%s: bad dtype", who);
  LV_REQUIRE(num_tokens >= 0, "%s: negative num_tokens", who);
  if (const int rc = check_quant_cache(who, c); rc != LV_OK) return rc;
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) {
    set_error("%s: head_dim %d (64, 128 and 256 are supported)", who, c->head_dim);
    return LV_ERR_UNSUPPORTED;
  }
  return LV_OK;
}

}  // namespace
}  // namespace lv

extern "C" int lv_kv_scatter_quant(const void* key_dev, int64_t key_stride_t,
                                   const void* value_dev, int64_t value_stride_t,
                                   const lv_quant_cache* cache, const int64_t* slot_mapping_dev,
                                   int64_t num_tokens, lv_dtype dtype, void* stream) {
  using namespace lv;
  clear_error();
  if (const int rc = check_common("lv_kv_scatter_quant", cache, dtype, num_tokens); rc != LV_OK)
    return rc;
  if (num_tokens == 0) return LV_OK;
  LV_REQUIRE(key_dev && value_dev && slot_mapping_dev, "lv_kv_scatter_quant: null pointer");
  const int hkv = cache->num_kv_heads, d = cache->head_dim;
  LV_REQUIRE((key_stride_t >= (int64_t)hkv * d && value_stride_t >= (int64_t)hkv * d) ||
                 num_tokens == 1,
             "lv_kv_scatter_quant: token stride smaller than num_kv_heads*head_dim");
  const bool vec = aligned_rows(key_dev, key_stride_t, dtype) &&
                   aligned_rows(value_dev, value_stride_t, dtype);
  const unsigned grid = grid_of(num_tokens * 2 * hkv, d / 8);
  LV_REQUIRE(grid > 0, "lv_kv_scatter_quant: too many rows for one launch");
  const QuantView v = view_of(cache);
  return by_type(dtype, [&](auto t) {
    return by_code(cache->code, [&](auto c) {
      return by_dim(d, [&](auto dim) {
        return by_bool(vec, [&](auto al) {
          using T = decltype(t);
          kv_scatter_quant_kernel<T, decltype(c), decltype(dim)::value, decltype(al)::value>
              <<<grid, kQuantThreads, 0, (hipStream_t)stream>>>(
                  (const T*)key_dev, key_stride_t, (const T*)value_dev, value_stride_t, v,
                  slot_mapping_dev, num_tokens, hkv);
          return check_launch("lv_kv_scatter_quant");
        });
      });
    });
  });
}

extern "C" int lv_kv_gather_quant(const lv_quant_cache* cache, const int64_t* slots_dev,
                                  int64_t num_tokens, void* key_dev, int64_t key_stride_t,
                                  void* value_dev, int64_t value_stride_t, lv_dtype dtype,
                                  void* stream) {
  using namespace lv;
  clear_error();
  if (const int rc = check_common("lv_kv_gather_quant", cache, dtype, num_tokens); rc != LV_OK)
    return rc;
  if (num_tokens == 0) return LV_OK;
  LV_REQUIRE(key_dev && value_dev && slots_dev, "lv_kv_gather_quant: null pointer");
  const int hkv = cache->num_kv_heads, d = cache->head_dim;
  LV_REQUIRE((key_stride_t >= (int64_t)hkv * d && value_stride_t >= (int64_t)hkv * d) ||
                 num_tokens == 1,
             "lv_kv_gather_quant: token stride smaller than num_kv_heads*head_dim");
  const bool vec = aligned_rows(key_dev, key_stride_t, dtype) &&
                   aligned_rows(value_dev, value_stride_t, dtype);
  const unsigned grid = grid_of(num_tokens * 2 * hkv, d / 8);
  LV_REQUIRE(grid > 0, "lv_kv_gather_quant: too many rows for one launch");
  const QuantView v = view_of(cache);
  return by_type(dtype, [&](auto t) {
    return by_code(cache->code, [&](auto c) {
      return by_dim(d, [&](auto dim) {
        return by_bool(vec, [&](auto al) {
          using T = decltype(t);
          kv_gather_quant_kernel<T, decltype(c), decltype(dim)::value, decltype(al)::value>
              <<<grid, kQuantThreads, 0, (hipStream_t)stream>>>(
                  v, slots_dev, num_tokens, hkv, (T*)key_dev, key_stride_t, (T*)value_dev,
                  value_stride_t);
          return check_launch("lv_kv_gather_quant");
        });
      });
    });
  });
}

extern "C" int lv_qk_norm_rope_cache_quant(
    const void* qkv_dev, int64_t qkv_stride_t, const void* q_norm_weight_dev,
    const void* k_norm_weight_dev, const void* cos_dev, const void* sin_dev, int64_t max_position,
    const int64_t* positions_dev, const int64_t* slot_mapping_dev, void* q_out_dev,
    int64_t q_out_stride_t, const lv_quant_cache* cache, int64_t num_tokens, int32_t num_heads,
    float eps, lv_dtype dtype, void* stream) {
  using namespace lv;
  clear_error();
  if (const int rc = check_common("lv_qk_norm_rope_cache_quant", cache, dtype, num_tokens);
      rc != LV_OK)
    return rc;
  LV_REQUIRE(num_heads > 0 && max_position > 0, "lv_qk_norm_rope_cache_quant: bad sizes");
  if (num_tokens == 0) return LV_OK;
  LV_REQUIRE(qkv_dev && cos_dev && sin_dev && positions_dev && slot_mapping_dev && q_out_dev,
             "lv_qk_norm_rope_cache_quant: null pointer");
  const int hkv = cache->num_kv_heads, d = cache->head_dim;
  const int64_t per_token = (int64_t)num_heads + 2 * (int64_t)hkv;
  LV_REQUIRE((qkv_stride_t >= per_token * d && q_out_stride_t >= (int64_t)num_heads * d) ||
                 num_tokens == 1,
             "lv_qk_norm_rope_cache_quant: token stride smaller than the row");
  const bool vec = aligned_rows(qkv_dev, qkv_stride_t, dtype) &&
                   aligned_rows(q_out_dev, q_out_stride_t, dtype) && aligned16(cos_dev) &&
                   aligned16(sin_dev) && aligned16(q_norm_weight_dev) &&
                   aligned16(k_norm_weight_dev);
  const unsigned grid = grid_of(num_tokens * per_token, d / 16);
  LV_REQUIRE(grid > 0, "lv_qk_norm_rope_cache_quant: too many rows for one launch");
  const QuantView v = view_of(cache);
  return by_type(dtype, [&](auto t) {
    return by_code(cache->code, [&](auto c) {
      return by_dim(d, [&](auto dim) {
        return by_bool(vec, [&](auto al) {
          using T = decltype(t);
          qk_norm_rope_cache_quant_kernel<T, decltype(c), decltype(dim)::value,
                                          decltype(al)::value>
              <<<grid, kQuantThreads, 0, (hipStream_t)stream>>>(
                  (const T*)qkv_dev, qkv_stride_t, (const T*)q_norm_weight_dev,
                  (const T*)k_norm_weight_dev, (const T*)cos_dev, (const T*)sin_dev, max_position,
                  positions_dev, slot_mapping_dev, (T*)q_out_dev, q_out_stride_t, v, num_tokens,
                  num_heads, hkv, eps);
          return check_launch("lv_qk_norm_rope_cache_quant");
        });
      });
    });
  });
}
