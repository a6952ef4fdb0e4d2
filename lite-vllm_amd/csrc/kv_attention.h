// What the attention kernels over paged caches share (kv_attention.hip,
// kv_tiles.h): the cache, batch and rows of a call, and one launch part of it.
#pragma once
#include <type_traits>

#include "lv_common.h"
#include "lv_quant.h"

namespace lv {

// A paged cache of element or code type; strides in elements.
struct KvView {
  const void* kv[2];
  const float* scale[2];         // 8-bit caches only
  int64_t blk, tok, head;
  int64_t sblk, stok, shead;
  int64_t num_blocks;
};

struct Batch {
  const int32_t* block_tables; int max_blocks;
  const int32_t* cu; const int32_t* ctx;
  const uint64_t* mask; int mask_words;      // trees only
  int num_seqs; int num_tokens;
};

struct Rows {
  const void* q; int64_t q_stride;
  void* out; int64_t out_stride;
  int num_heads, num_kv_heads;
  float scale_log2;
};

constexpr int kBs = 16;
constexpr float kNegBig = -3.40282347e38f;     // under every finite score

template <typename C> struct cached {          // 8-bit codes
  static constexpr bool kCodes = true;
  static constexpr int kBytes = 1;
  static constexpr int kPer16B = 16;
  __device__ __forceinline__ static void unpack(const uint4& v, float* out) {
    code<C>::unpack4(v.x, out);
    code<C>::unpack4(v.y, out + 4);
    code<C>::unpack4(v.z, out + 8);
    code<C>::unpack4(v.w, out + 12);
  }
};
template <typename T> struct cached_elem : elem<T> { static constexpr bool kCodes = false; };
template <> struct cached<float> : cached_elem<float> {};
template <> struct cached<f16> : cached_elem<f16> {};
template <> struct cached<bf16> : cached_elem<bf16> {};

// A sequence's query rows [q0, q0 + n) and its keys [0, ctx), clamped to the
// batch's tensors.
struct Seq { int q0, n, ctx; };
__device__ __forceinline__ Seq sequence(const Batch& b, int i) {
  Seq s;
  s.q0 = b.cu ? b.cu[i] : i;
  const int q1 = b.cu ? b.cu[i + 1] : i + 1;
  s.q0 = min(max(s.q0, 0), b.num_tokens);
  s.n = min(max(q1 - s.q0, 0), b.num_tokens - s.q0);
  s.ctx = min(max(b.ctx[i], 0), b.max_blocks * kBs);
  return s;
}

__device__ __forceinline__ int physical_block(const Batch& b, int64_t num_blocks, int seq,
                                              int blk) {
  const int id = b.block_tables[(int64_t)seq * b.max_blocks + blk];
  if (id >= 0 && id < num_blocks) return id;
  report_device_error(LV_DEVERR_BLOCK_ID);     // clamped and reported
  return 0;
}

// A call of one of the entry points.
struct Call {
  Batch b; KvView c; Rows r;
  int d; lv_dtype dtype; int code;     // code: lv_code, or -1 for a cache of dtype
  bool tree;
  hipStream_t stream;
};

// Sequences of a launch, at most.  A kernel keeps their offsets in LDS beside its
// tiles: for so many the largest tiles leave room (kv_launch.h asserts it).
constexpr int kPartSeqs = 4096;
constexpr size_t kOffsetBytes = (size_t)(kPartSeqs + 1) * 4;
constexpr size_t kLdsBytes = 160 * 1024;

// The sequences [seq_begin, seq_begin + n_seqs) of a call, max_q rows each at
// most: their kernel, its launch and its workspace.
struct TilePlan {
  int seq_begin, n_seqs, max_q;
  int rw;                   // tile kernel: 32-row groups of a unit, 1, 2, 4 or 8; 0: narrow kernel
  int waves;                // and its wavefronts
  int64_t list;             // tiles of all units, at most
  int grid, ranges;         // workgroups; ranges that the list is split into
  int direct, nq;           // (see TileArgs)
  int slot_heads, slot_rows;
  size_t head_bytes, ml_bytes, acc_bytes;
};

// One translation unit per query type.
int launch_tiles_bf16(const Call& a, const TilePlan& p, char* ws);
int launch_tiles_f16(const Call& a, const TilePlan& p, char* ws);
int launch_tiles_f32(const Call& a, const TilePlan& p, char* ws);

}  // namespace lv
