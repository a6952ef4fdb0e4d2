// Attention over paged caches on the matrix cores (the kernel and its launch;
// included by one translation unit per query type).
#pragma once
#include <utility>

#include "kv_attention.h"
#include "lv_attn.h"
#include "lv_mfma.h"

namespace lv {

// ---------------------------------------------------------------------------
// Tiles on the matrix cores.
//
// The query rows of a sequence that read one kv head are its (token, head of
// the group) pairs; a unit is up to R = 32 RW of them and the keys they need,
// in tiles of KT.  All units' tiles form one list, which a fixed grid of
// workgroups splits into equal contiguous ranges: the work is even however
// unlike the contexts are, and nothing about them has to be known on the
// host.  A unit inside one range is written to `out`; the pieces of one that
// spans several go to the workspace (m, l, O / l in fp32) and attn_join_kernel
// joins them.  Where there are many units and none is long against a range, a
// workgroup takes a whole unit instead (direct), longest sequences and last
// rows first, so that there are no pieces: 15 chunks of 512 tokens at offsets
// of 0-3071, 2 query heads for each of 8 kv heads (480 units of 256 rows),
// 265 -> 203 us.
//
// A workgroup is 4 or 8 wavefronts: RW groups of 32 rows times KW = WAVES / RW
// parts of every tile's keys, so that few rows (RW = 1: decodes, small trees)
// still use four wavefronts; the KW states are merged through LDS when a piece
// ends.  Eight halve what each does to bring a tile into LDS, and the pieces
// (the host's rule and its measurements are in plan_tiles).
// Per tile:
//   * the next tile's rows are loaded from HBM into registers while this one
//     is computed, then turned into 16-bit operands (codes are exact in bf16
//     and fp16) and written to LDS, swizzled (ChunkLds);
//   * S^T = K Q^T, v_mfma_f32_32x32x16: a lane ends with one query row (its
//     column) against 16 of each 32 keys;
//   * x = S^T * (scale of the key's row * scale), masked by position or tree;
//     maximum (raised rarely), weights and their sum in fp32;
//   * O^T += V^T P^T with P = weight * scale of the value's row.
// The scales of a score's keys come from LDS as one register, 16 lanes holding
// 16 keys, and by DPP into the instruction that takes them: read as they lie
// for 16 keys (b128, the same for 32 lanes) they were most of the LDS time (two
// chunks of 700-1024 tokens at 15000-19000, 8 query heads a kv head, 309 -> 292
// us; trees of 25-60 tokens at 2000-16000 213 -> 198; both with weights of one
// part).
//
// Weights.  A weight rounded to bf16 (2^-8) or, for an fp16 output, to fp16
// (2^-11) errs as much as the output's own rounding does, and the keys' errors
// do not cancel.  So P is as many 16-bit parts as leave nothing of that: two fp16
// ones (2^-22) over codes and fp16 caches, two bf16 ones (2^-15) over a bf16
// cache, three bf16 ones, all the bits, for fp32 queries.  (One fp16 part put fp16
// outputs a third further from 64 bits than fp32 weights do, 2.7e-4 instead of
// 2.1e-4, and bf16 ones half a percent, 1.664e-3 instead of 1.655e-3.  The second
// costs 16 products a tile and an instruction a score: the chunks above 292 ->
// 377 us and the trees over codes 195 -> 243, both fp16, the mixed step 318 -> 359,
// bf16.)
// Over codes, with y = x + log2(scale of the value's row), P = exp2(y - reference)
// takes no multiplication, the weights' sum is sum P / scale, and the reference
// follows the largest y, so that the largest P of a row is between 2^10 and 2^15
// whatever the scales are and what fp16 cannot hold of the smallest, 2^-25, is
// 2^-35 of it.  The sum y is rounded to the last place of the score, as the score
// was when it was scaled: one rounding beside the D of its products.
// Scales outside [2^-60, 2^20] of the unit's first ones, and ones that are not
// finite, make the piece careful (below).
// fp32 queries are three bf16 parts (all their bits), others are taken as
// they are.  An fp32 cache keeps fp32 operands and v_mfma_f32_32x32x2 (157
// TFLOP/s at most; six products of bf16 parts would need three times the LDS):
// trees of 40-64 tokens at 500-4000, 48 sequences, 8 kv heads of 128: 594 us.
//
// What bounds it: the chunks above, at 373 us, the issue of one SIMD's two
// wavefronts (registers allow no third), whose products (46% of the cycles) and
// vector instructions (52%) overlap little.  Over a 16-bit cache the one tile that
// is on its way from HBM while another is computed: those trees in bf16 take 132 us,
// 3.6 TB/s, with products 29% and vector instructions 36% of the cycles.
//
// Zero weights times a value that is not finite make NaN: a piece whose sums
// are not finite is computed again key by key (careful), where a key that a
// row does not see is not read.
// ---------------------------------------------------------------------------
struct TileArgs {
  Batch b; KvView c; Rows r;
  int seq_begin, n_seqs, max_q;
  int ranges;               // ranges of the list
  int direct;               // a workgroup per unit: 1 if no unit is long, 2 always, 3 always
                            // and in no order (all run at once)
  int nq;                   // row tiles of a unit's sequence, at most
  int slot_heads, slot_rows;   // kv heads of a workspace slot, rows of each
  int4* head;               // [ranges][2]: the unit that crosses a range's start
  float* ml;                // [2 ranges][slot_heads][slot_rows][2]
  float* acc;               // [2 ranges][slot_heads][slot_rows][D]
};

struct Unit {
  int seq, q0, n, rows, committed, kend, kvh, row0, ntiles;
  int unit2;     // the V scales' unit is 2^unit2 (16-bit queries over codes)
};

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
// The same in all lanes: said to the compiler, which does not see it of what
// comes out of LDS, so that all that follows from a unit is scalar.
__device__ __forceinline__ void make_uniform(Unit& u) {
  u.seq = uniform(u.seq); u.q0 = uniform(u.q0); u.n = uniform(u.n); u.rows = uniform(u.rows);
  u.committed = uniform(u.committed); u.kend = uniform(u.kend); u.kvh = uniform(u.kvh);
  u.row0 = uniform(u.row0); u.ntiles = uniform(u.ntiles);
}

template <int RW_, int WAVES_> struct TileCfg {
  static constexpr int RW = RW_, WAVES = WAVES_, THREADS = 64 * WAVES;
  static constexpr int R = 32 * RW, KW = WAVES / RW;
  static constexpr int KT = WAVES == 4 && RW == 4 ? 64 : 128;   // keys per tile
  static constexpr int BPW = KT / (16 * WAVES);   // 16-token blocks a wavefront stages
  static constexpr int KPW = KT / KW;             // keys a wavefront computes
  static constexpr int SUB = KPW > 64 ? 2 : 1;    // in so many steps
  static constexpr int NST = RW >= 4 || WAVES == 8 ? 2 : 1;     // LDS stages
  static constexpr size_t lds(int d, int bytes) { // operands of so many bytes; without the
    return (size_t)NST * (KT * d * 2 * bytes + KT * 12) + 32 * WAVES * 8;      // list's offsets
  }
};

// Keys that row tile [row0, row0 + R) of a sequence needs.
template <bool TREE, int R>
__device__ __forceinline__ int keys_needed(int ctx, int committed, int rows, int row0, int g) {
  if (TREE) return ctx;
  return max(0, min(ctx, committed + (min(row0 + R, rows) - 1) / g + 1));
}

__device__ __forceinline__ Seq tile_sequence(const TileArgs& a, int i) {
  return sequence(a.b, a.seq_begin + i);
}

// Tiles of sequence i, over all its row tiles and kv heads.
template <bool TREE, typename F>
__device__ __forceinline__ int sequence_tiles(const TileArgs& a, const Seq& s, int g) {
  const int rows = min(s.n, a.max_q) * g;
  int sum = 0;
  if (TREE) {
    sum = (rows + F::R - 1) / F::R * max(1, (s.ctx + F::KT - 1) / F::KT);
  } else {
    for (int r0 = 0; r0 < rows; r0 += F::R)
      sum += max(1, (keys_needed<TREE, F::R>(s.ctx, s.ctx - s.n, rows, r0, g) + F::KT - 1) / F::KT);
  }
  return sum * a.r.num_kv_heads;
}

// Exclusive scan of the sequences' tiles into off[0 .. n_seqs]; returns the
// longest unit's tiles.
template <bool TREE, typename F>
__device__ int scan_tiles(const TileArgs& a, int g, int* off, int* part) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int per = (a.n_seqs + F::THREADS - 1) / F::THREADS;
  const int lo = min(a.n_seqs, t * per), hi = min(a.n_seqs, lo + per);
  int sum = 0, longest = 0;
  for (int i = lo; i < hi; ++i) {
    off[i] = sum;                       // within the thread's run
    const Seq s = tile_sequence(a, i);
    sum += sequence_tiles<TREE, F>(a, s, g);
    if (s.n > 0) longest = max(longest, (s.ctx + F::KT - 1) / F::KT);
  }
  longest = (int)group_umax<64>((uint32_t)longest);
  int incl = sum;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int u = __shfl_up(incl, d);
    if (lane >= d) incl += u;
  }
  if (lane == 63) part[wave] = incl;
  if (lane == 0) part[8 + wave] = longest;
  __syncthreads();
  int base = incl - sum;
  for (int w = 0; w < wave; ++w) base += part[w];
  for (int i = lo; i < hi; ++i) off[i] += base;
  if (t == F::THREADS - 1) off[a.n_seqs] = base + sum;
  for (int w = 0; w < F::WAVES; ++w) longest = max(longest, part[8 + w]);
  __syncthreads();
  return longest;
}

// The sequence that direct workgroups of rank r take: the r-th by descending
// context (ties by index) where they are few enough to rank, r otherwise.
constexpr int kRankMax = 256;
__device__ __forceinline__ int ranked_sequence(const TileArgs& a, int r, int* ctx, int* pick) {
  if (a.n_seqs > kRankMax || a.direct == 3) return r;
  const int t = threadIdx.x;
  const int mine = t < a.n_seqs ? tile_sequence(a, t).ctx : -1;
  if (t < kRankMax) ctx[t] = mine;
  __syncthreads();
  int before = 0;
  for (int i = 0; i < a.n_seqs; ++i) before += ctx[i] > mine || (ctx[i] == mine && i < t);
  if (t < a.n_seqs && before == r) *pick = t;
  __syncthreads();
  return *pick;
}

template <bool TREE, typename F>
__device__ __forceinline__ void set_rows(const TileArgs& a, Unit& u, int ctx, int g) {
  u.kend = keys_needed<TREE, F::R>(ctx, u.committed, u.rows, u.row0, g);
  u.ntiles = max(1, (u.kend + F::KT - 1) / F::KT);
}
__device__ __forceinline__ int set_seq(const TileArgs& a, Unit& u, int i, int g) {
  const Seq s = tile_sequence(a, i);
  u.seq = i; u.q0 = s.q0; u.n = s.n;
  u.rows = min(s.n, a.max_q) * g;
  u.committed = s.ctx - s.n;
  return s.ctx;
}

// The unit that holds place p of the list, and p's tile in it.
template <bool TREE, typename F>
__device__ __forceinline__ int locate(const TileArgs& a, const int* off, int p, int g, Unit& u) {
  int lo = 0, hi = a.n_seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (off[mid] <= p) lo = mid; else hi = mid - 1;
  }
  const int ctx = set_seq(a, u, lo, g);
  const int per_head = (off[lo + 1] - off[lo]) / a.r.num_kv_heads;
  int rem = p - off[lo];
  u.kvh = rem / per_head;
  rem -= u.kvh * per_head;
  for (u.row0 = 0;; u.row0 += F::R) {
    set_rows<TREE, F>(a, u, ctx, g);
    if (rem < u.ntiles || u.row0 + F::R >= u.rows) break;
    rem -= u.ntiles;
  }
  return rem;
}

template <bool TREE, typename F>
__device__ __forceinline__ Unit next_unit(const TileArgs& a, Unit u, int g) {
  u.row0 += F::R;
  int ctx = u.committed + u.n;
  if (u.row0 >= u.rows) {
    u.row0 = 0;
    if (++u.kvh == a.r.num_kv_heads) {
      u.kvh = 0;
      do ctx = set_seq(a, u, u.seq + 1, g); while (u.rows == 0 && u.seq + 1 < a.n_seqs);
    }
  }
  set_rows<TREE, F>(a, u, ctx, g);
  return u;
}

// 16 codes -> 16 operands of 16 bits (two 16-byte chunks).
template <typename O, typename C>
__device__ __forceinline__ void codes_to_operands(const uint4& w, uint4* out) {
  const uint32_t in[4] = {w.x, w.y, w.z, w.w};
  uint32_t o[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<C, e4m3_code>::value && std::is_same<O, bf16>::value) {
      o[2 * i] = __builtin_bit_cast(uint32_t,
                                    __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(in[i], 1.0f, false));
      o[2 * i + 1] = __builtin_bit_cast(
          uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(in[i], 1.0f, true));
    } else if constexpr (std::is_same<C, e4m3_code>::value) {
      o[2 * i] = __builtin_bit_cast(uint32_t,
                                    __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(in[i], 1.0f, false));
      o[2 * i + 1] = __builtin_bit_cast(
          uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(in[i], 1.0f, true));
    } else if constexpr (std::is_same<O, bf16>::value) {
      float f[4];
      code<C>::unpack4(in[i], f);
      o[2 * i] = float_to_bf16_pair(f[0], f[1]);
      o[2 * i + 1] = float_to_bf16_pair(f[2], f[3]);
    } else {
      // bytes c + 128 under the exponent of 1024: the fp16 value 1152 + c
      const uint32_t u = in[i] ^ 0x80808080u;
      const f16x2_t off = {(_Float16)1152.0f, (_Float16)1152.0f};
      o[2 * i] = __builtin_bit_cast(
          uint32_t, __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off);
      o[2 * i + 1] = __builtin_bit_cast(
          uint32_t, __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off);
    }
  }
  out[0] = make_uint4(o[0], o[1], o[2], o[3]);
  out[1] = make_uint4(o[4], o[5], o[6], o[7]);
}

// Pairs of fp32 values as their leading bf16 / fp16 parts, taken off them unless
// they are the last.
template <typename O>
__device__ __forceinline__ uint32_t take_part(float& a, float& b, bool last) {
  if constexpr (std::is_same<O, bf16>::value) {
    if (last) return float_to_bf16_pair(a, b);
    const uint32_t w = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    a -= __uint_as_float(w << 16);
    b -= __uint_as_float(w & 0xffff0000u);
    return w;
  } else {
    const uint32_t w = __builtin_bit_cast(
        uint32_t, __builtin_convertvector(f32x2_t{a, b}, f16x2_t));     // one instruction
    if (!last) {
      a -= f16_bits_to_float(w & 0xffffu);
      b -= f16_bits_to_float(w >> 16);
    }
    return w;
  }
}

// The same for a leading fp16 part w and all that it leaves, as fp16: one
// instruction a value (v_fma_mix, which the compiler does not make of a
// difference).
__device__ __forceinline__ uint32_t rest_of(uint32_t w, float a, float b) {
  float minus = -1.0f;
  asm("" : "+s"(minus));
  const f16x2_t h = __builtin_bit_cast(f16x2_t, w);
  const f16x2_t r = {(_Float16)fmaf((float)h[0], minus, a), (_Float16)fmaf((float)h[1], minus, b)};
  return __builtin_bit_cast(uint32_t, r);
}

// Waits here for the loads of these registers.  Left alone, the compiler waits
// at their first use, which lies in a loop, and so on every pass for whatever
// loads are then in flight.
template <int N>
__device__ __forceinline__ void settle(uint4 (&q)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(q[i].x), "+v"(q[i].y), "+v"(q[i].z), "+v"(q[i].w));
}

// Lane I of every 16 lanes' x, in all of them: part of the instruction that
// takes it (DPP).
template <int I> __device__ __forceinline__ float row_lane(float x) {
  return __uint_as_float(
      (uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), 0x150 + I, 0xf, 0xf, true));
}
using Sixteen = std::make_integer_sequence<int, 16>;
// x[i] times, plus lane i's value (not contracted to one instruction: that has
// no DPP form).
template <int... I>
__device__ __forceinline__ void scale_rows(f32x16_t& x, float mul, std::integer_sequence<int, I...>) {
#pragma clang fp contract(off)
  ((x[I] = row_lane<I>(mul) * x[I]), ...);
}
template <int... I>
__device__ __forceinline__ void add_rows(f32x16_t& x, float add, std::integer_sequence<int, I...>) {
#pragma clang fp contract(off)
  ((x[I] = row_lane<I>(add) + x[I]), ...);
}
// sum + the sum of x[i] times lane i's value.  (The compiler does not make this
// form itself.  All lanes are on.  The first wait states are those that DPP and the results of
// exp2 need, which it does not add before assembly.)
__device__ __forceinline__ float sum_rows(const f32x16_t& x, float mul, float sum) {
#define LV_FMAC(i, r) "v_fmac_f32_dpp %0, %1, %" #r " row_newbcast:" #i " row_mask:0xf bank_mask:0xf\n"
  asm("s_nop 1\n"
      LV_FMAC(0, 2) LV_FMAC(1, 3) LV_FMAC(2, 4) LV_FMAC(3, 5)
      LV_FMAC(4, 6) LV_FMAC(5, 7) LV_FMAC(6, 8) LV_FMAC(7, 9)
      : "+&v"(sum)
      : "v"(mul), "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "v"(x[4]), "v"(x[5]), "v"(x[6]),
        "v"(x[7]));
  asm("s_nop 1\n"
      LV_FMAC(8, 2) LV_FMAC(9, 3) LV_FMAC(10, 4) LV_FMAC(11, 5)
      LV_FMAC(12, 6) LV_FMAC(13, 7) LV_FMAC(14, 8) LV_FMAC(15, 9)
      : "+&v"(sum)
      : "v"(mul), "v"(x[8]), "v"(x[9]), "v"(x[10]), "v"(x[11]), "v"(x[12]), "v"(x[13]), "v"(x[14]),
        "v"(x[15]));
#undef LV_FMAC
  return sum;
}

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

__device__ __forceinline__ void team_barrier() {
  wait_lds();                      // (loads into registers stay in flight)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <typename T, typename C> struct Operands {
  static constexpr bool kCodes = cached<C>::kCodes;
  using K = typename std::conditional<std::is_same<T, f16>::value, f16, bf16>::type;
  static constexpr bool kF32 = std::is_same<T, float>::value;
  static constexpr bool kLog = kCodes && !kF32;   // P = exp2(x + log2 of V's scale)
  using V = typename std::conditional<kCodes, typename std::conditional<kF32, bf16, f16>::type,
                                      K>::type;
  static constexpr int QP = kF32 ? 3 : 1;    // parts of a query, of a weight
  static constexpr int PP = kF32 ? 3 : 2;
  static constexpr bool kWide = std::is_same<C, float>::value;   // fp32 operands
  // A row's reference is set kLift (in log2 units) under the score that sets it
  // and again when a score passes it by kTop: fp16 weights then lie high enough
  // that the fixed step of the smallest ones, 2^-24, weighs nothing.
  static constexpr float kLift = std::is_same<V, f16>::value ? 10.0f : 0.0f;
  static constexpr float kTop = std::is_same<V, f16>::value ? 15.0f : 8.0f;
};

// What the tile kernel has in LDS besides its tiles and offsets.
constexpr size_t kTileStaticLds = (16 + kRankMax + 4) * sizeof(int);

// Wavefronts per SIMD: the three parts of fp32 queries need the registers of two.
template <typename T> constexpr int kTileWaves = std::is_same<T, float>::value ? 1 : 2;

template <typename T, typename C, int D, typename F, bool TREE>
__global__ __launch_bounds__(F::THREADS, kTileWaves<T>)
void attn_tile_kernel(TileArgs a) {
  constexpr int RW = F::RW;
  using P = Operands<T, C>;
  using E = cached<C>;
  using L = ChunkLds<D, 4>;
  using KM = Mfma32<typename P::K>;
  using VM = Mfma32<typename P::V>;
  constexpr bool kCodes = P::kCodes;
  constexpr int KT = F::KT, KW = F::KW, KPW = F::KPW, KB = KPW / F::SUB / 32,
                BPW = F::BPW;
  constexpr int QSTEPS = D / 16, DBLK = D / 32;
  constexpr int CPR = D / E::kPer16B;             // 16-byte chunks of a cached row
  constexpr int RPL = 64 / CPR;                   // rows of a wavefront-wide load
  constexpr int LPB = kBs / RPL;                  // loads of a block's K or V
  constexpr int OPC = E::kPer16B < 8 ? 1 : E::kPer16B / 8;             // operand chunks of a cached chunk
  constexpr bool kWide = P::kWide;
  static_assert(16 % RPL == 0, "whole loads per block");
  // K and V tiles, then the scales of their keys; the merge of a piece's parts
  // reuses the tiles (WAVES x 32 rows x D floats, which fill them for eight
  // wavefronts)
  extern __shared__ __align__(16) unsigned char s_dyn[];
  // (of K or V, in 16-bit places)
  constexpr int NST = F::NST, TILE = KT * D * (kWide ? 2 : 1);
  static_assert(KW == 1 || F::WAVES * 32 * D * 4 <= NST * 2 * TILE * 2, "the merge fits the tiles");
  uint16_t* const s_kv = reinterpret_cast<uint16_t*>(s_dyn);       // [NST][K, V][TILE]
  // [NST][KT] each: K's scales; V's scales, or their logarithms and inverses
  float* const s_sc = reinterpret_cast<float*>(s_kv + NST * 2 * TILE);
  float2* const s_ml = reinterpret_cast<float2*>(s_sc + NST * 3 * KT);   // [WAVES][32]
  int* const s_off = reinterpret_cast<int*>(s_ml + 32 * F::WAVES);
  __shared__ int s_part[16], s_ctx[kRankMax], s_pick;

  const int H = a.r.num_heads, Hkv = a.r.num_kv_heads;
  const int G = H / Hkv;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rg = wave % RW, kg = wave / RW;
  const int lr = lane & 31, h = lane >> 5;

  int r0 = 0, r1 = 1, w = 0, t = 0, per = 1;
  bool direct = a.direct >= 2;
  if (!direct) {
    const int longest = uniform(scan_tiles<TREE, F>(a, G, s_off, s_part));
    const int total = uniform(s_off[a.n_seqs]);
    per = max(1, (int)(((int64_t)total + a.ranges - 1) / a.ranges));
    direct = a.direct == 1 && longest <= 2 * per;
    const int b = (int)blockIdx.x;
    // neighbouring ranges on one XCD: they read the same cached rows
    w = a.ranges % kXcds == 0 ? b % kXcds * (a.ranges / kXcds) + b / kXcds : b;
    if (b < a.ranges && threadIdx.x == 0) a.head[2 * w] = make_int4(0, 0, 0, 0);
    if (!direct) {
      if (b >= a.ranges) return;
      r0 = (int)min((int64_t)total, (int64_t)w * per);
      r1 = (int)min((int64_t)total, (int64_t)(w + 1) * per);
      if (r0 >= r1) return;
    }
  }
  Unit U;
  if (direct) {
    // all row tiles of a (sequence, kv head) on one XCD
    const int slot = (int)blockIdx.x / kXcds;
    const int grp = slot / a.nq * kXcds + (int)blockIdx.x % kXcds;
    if (grp >= a.n_seqs * Hkv) return;
    const int seq = uniform(ranked_sequence(a, grp / Hkv, s_ctx, &s_pick));
    const int ctx = set_seq(a, U, seq, G);
    U.kvh = grp % Hkv;
    U.row0 = (a.nq - 1 - slot % a.nq) * F::R;
    if (U.row0 >= U.rows) return;
    set_rows<TREE, F>(a, U, ctx, G);
    make_uniform(U);
  } else {
    t = uniform(locate<TREE, F>(a, s_off, r0, G, U));
    make_uniform(U);
    if (t > 0 && threadIdx.x == 0) {
      // the range starts inside a unit; if that unit starts in the range
      // before, this range's workgroup of the join takes it
      const int start = r0 - t, end = start + U.ntiles;
      if (start >= r0 - per) {
        a.head[2 * w] = make_int4((end - 1) / per - w + 2, U.q0, U.kvh, U.row0);
        a.head[2 * w + 1] = make_int4(min(F::R, U.rows - U.row0), 0, 0, 0);
      }
    }
  }

  // -- loading -------------------------------------------------------------
  // What follows from the unit alone is set once a piece (set_piece).
  uint4 kraw[BPW][LPB], vraw[BPW][LPB];
  float sraw = 0.0f;             // a scale (K of keys 0 .., then V) of the wavefront's blocks
  int ids[BPW], id_first = 0;
  const char *kbase = nullptr, *vbase = nullptr;
  const float* sbase = nullptr;
  const int lrow = lane / CPR, lchunk = lane % CPR;
  int64_t loff[LPB];
#pragma unroll
  for (int i = 0; i < LPB; ++i)
    loff[i] = (int64_t)(RPL * i + lrow) * a.c.tok * E::kBytes + 16 * lchunk;
  auto load_ids = [&](int first) {
    const int last = (U.kend - 1) / kBs;
#pragma unroll
    for (int j = 0; j < BPW; ++j) {
      ids[j] = 0;
      if (U.kend > 0)
        ids[j] = physical_block(a.b, a.c.num_blocks, a.seq_begin + U.seq,
                                min((first + lane) * (KT / kBs) + wave * BPW + j, last));
    }
    id_first = first;
  };
  auto load_tile = [&](int tile) {
    if (tile - id_first >= 64) load_ids(tile);
    int phys[BPW];     // (read by all lanes: a readlane under a branch sees stale copies)
#pragma unroll
    for (int j = 0; j < BPW; ++j) phys[j] = __builtin_amdgcn_readlane(ids[j], tile - id_first);
#pragma unroll
    for (int j = 0; j < BPW; ++j) {
      const int64_t at = (int64_t)phys[j] * a.c.blk * E::kBytes;
#pragma unroll
      for (int i = 0; i < LPB; ++i) {
        kraw[j][i] = load16(kbase + at + loff[i]);
        vraw[j][i] = load16(vbase + at + loff[i]);
      }
    }
    if constexpr (kCodes) {
      const int block = lane & 16 ? phys[BPW - 1] : phys[0];
      sraw = sbase[block * a.c.sblk];
    }
  };
  // Loads the piece's first tile; what they wait for one after the other (block
  // table, then rows) is in flight with the look at the V scales.
  auto set_piece = [&](int first) {
    kbase = (const char*)a.c.kv[0] + U.kvh * a.c.head * E::kBytes;
    vbase = (const char*)a.c.kv[1] + U.kvh * a.c.head * E::kBytes;
    load_ids(first);
    const int key = first * KT + lane;
    int block = 0;
    if (P::kLog && key < U.kend)
      block = physical_block(a.b, a.c.num_blocks, a.seq_begin + U.seq, key / kBs);
    if constexpr (kCodes) {
      // lanes 0 .. 16 BPW - 1 the K scales, the next as many the V scales
      const bool of_v = (lane / (16 * BPW)) & 1;
      sbase = (of_v ? a.c.scale[1] : a.c.scale[0]) + (lane & 15) * a.c.stok + U.kvh * a.c.shead;
    }
    load_tile(first);
    if constexpr (P::kLog) {     // the unit of the V scales: the largest of the first 64
      float v = 0.0f;
      if (key < U.kend)
        v = a.c.scale[1][block * a.c.sblk + (key % kBs) * a.c.stok + U.kvh * a.c.shead];
      v = group_max<64>(v > 0.0f && v < __builtin_inff() ? v : 0.0f);
      const int e = uniform((int)(__float_as_uint(v) >> 23));      // 0: no scale
      U.unit2 = e > 0 ? min(max(e - 127, -100), 100) : 0;
    }
  };
  auto write_tile = [&](int tile, int st) {
    uint16_t* const Ks = s_kv + st * 2 * TILE;
    uint16_t* const Vs = Ks + TILE;
    const int key0 = tile * KT + wave * 16 * BPW;
    const bool tail = key0 + 16 * BPW > U.kend;
#pragma unroll
    for (int j = 0; j < BPW; ++j)
#pragma unroll
      for (int i = 0; i < LPB; ++i) {
        const int row = 16 * (wave * BPW + j) + RPL * i + lrow;    // of the tile
        if (tail && tile * KT + row >= U.kend) vraw[j][i] = make_uint4(0, 0, 0, 0);
        if constexpr (kWide) {
          store16(Ks + 2 * row * D + 8 * (lchunk ^ (row & 15)), kraw[j][i]);
          store16(Vs + 2 * row * D + 8 * (lchunk ^ (2 * (row & 4))), vraw[j][i]);
        } else {
          uint4 ko[OPC], vo[OPC];
          if constexpr (kCodes) {
            codes_to_operands<typename P::K, C>(kraw[j][i], ko);
            codes_to_operands<typename P::V, C>(vraw[j][i], vo);
          } else {
            ko[0] = kraw[j][i];
            vo[0] = vraw[j][i];
          }
#pragma unroll
          for (int c = 0; c < OPC; ++c) {
            store16(Ks + L::at(row, lchunk * OPC + c), ko[c]);
            store16(Vs + L::at(row, lchunk * OPC + c), vo[c]);
          }
        }
      }
    if constexpr (kCodes) {
      const int key = lane % (16 * BPW), kv = lane / (16 * BPW);
      const int row = 16 * wave * BPW + key;
      float* const sc = s_sc + st * 3 * KT;
      const bool in = tile * KT + row < U.kend;
      if (kv == 0) sc[row] = sraw * a.r.scale_log2;
      if (kv == 1) {
        if constexpr (P::kLog) {
          const float v = sraw * pow2(-U.unit2);
          const bool ok = v >= 0x1p-60f && v <= 0x1p20f;
          sc[KT + row] = !in ? 0.0f : ok ? __builtin_amdgcn_logf(v) : v == 0.0f ? -60.0f : 0.0f;
          sc[2 * KT + row] = !in ? 0.0f : ok ? __builtin_amdgcn_rcpf(v)
                                       : v == 0.0f ? 0x1p60f : __builtin_nanf("");
        } else {
          sc[KT + row] = in ? sraw : 0.0f;
        }
      }
    }
  };

  // -- a piece's state -------------------------------------------------------
  using qv8 = typename KM::v8;
  qv8 qf[kWide ? 1 : P::QP][kWide ? 1 : QSTEPS];
  float4 qw[kWide ? D / 8 : 1];              // fp32 operands: dims 8 i + 4 h ...
  f32x16_t o[DBLK];
  float m_run = kNegBig, l_run = 0.0f;
  int qrow = 0, qhead = 0, lim = 0;          // this lane's row, head and last key
  bool live = false;

  auto start = [&]() {
    const int idx = U.row0 + 32 * rg + lr;
    live = idx < U.rows;
    const int use = live ? idx : U.row0;
    qrow = U.q0 + use / G;
    qhead = U.kvh * G + use % G;
    lim = TREE ? U.kend - 1 : min(U.committed + use / G, U.kend - 1);
    const T* qp = (const T*)a.r.q + (int64_t)qrow * a.r.q_stride + (int64_t)qhead * D + 8 * h;
    if constexpr (kWide) {
      uint4 raw[D / 8];
#pragma unroll
      for (int s = 0; s < D / 8; ++s) raw[s] = load16(qp - 4 * h + 8 * s);
      settle(raw);
#pragma unroll
      for (int s = 0; s < D / 8; ++s) qw[s] = __builtin_bit_cast(float4, raw[s]);
    } else if constexpr (P::QP == 1) {
      uint4 raw[QSTEPS];
#pragma unroll
      for (int s = 0; s < QSTEPS; ++s) raw[s] = load16(qp + 16 * s);
      settle(raw);
#pragma unroll
      for (int s = 0; s < QSTEPS; ++s) qf[0][s] = __builtin_bit_cast(qv8, raw[s]);
    } else {
#pragma unroll
      for (int s = 0; s < QSTEPS; ++s) {
        float x[8];
        elem<float>::unpack(load16(qp + 16 * s), x);
        elem<float>::unpack(load16(qp + 16 * s + 4), x + 4);
#pragma unroll
        for (int p = 0; p < P::QP; ++p) {
          uint32_t part[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            part[i] = take_part<bf16>(x[2 * i], x[2 * i + 1], p + 1 == P::QP);
          qf[p][s] = __builtin_bit_cast(qv8, make_uint4(part[0], part[1], part[2], part[3]));
        }
      }
    }
#pragma unroll
    for (int b = 0; b < DBLK; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[b][i] = 0.0f;
    m_run = kNegBig;
    l_run = 0.0f;
  };

  // Score i of 32 keys is key 8 (i / 4) + i % 4 + 4 h; the lane that holds that
  // key's scales for its 16 lanes is i.
  const int own_key = 8 * ((lane & 15) >> 2) + (lane & 3) + 4 * h;
  // Byte offsets in a stage of this lane's operands: the swizzle is an XOR of
  // the chunk, so the chunk of k-step s (dim block b) is one more XOR away.
  const uint32_t k_at = 2 * (lr * D + 8 * (h ^ L::swz(lr)));      // ^ 32 s
  uint32_t v_at[2];                                               // ^ 64 b
  {
    const int vrow = 4 * h + ((lane & 15) >> 2), dim = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
    for (int i = 0; i < 2; ++i) v_at[i] = 2 * (L::at(vrow + 8 * i, dim >> 3) + (dim & 7));
  }

  // Bits of the 32 drafted keys from t0 on that this lane's row sees; keys
  // before the first drafted one are committed: seen.
  auto tree_window = [&](int t0) -> uint32_t {
    const uint64_t* row = a.b.mask + (int64_t)qrow * a.b.mask_words;
    if (t0 <= -32) return ~0u;
    if (t0 < 0) return (uint32_t)(row[0] << -t0) | ((1u << -t0) - 1);
    const int i = t0 >> 6, s = t0 & 63;
    uint64_t v = i < a.b.mask_words ? row[i] >> s : 0;
    if (s > 32 && i + 1 < a.b.mask_words) v |= row[i + 1] << (64 - s);
    return (uint32_t)v;
  };

  auto compute = [&](int tile, int st, int sub) {
    const int off = kg * KPW + 32 * KB * sub;      // this wavefront's first key of the step
    const int k0 = tile * KT + off;
    const uint32_t kt = (uint32_t)(2 * st * 2 * TILE + (kWide ? 4 : 2) * off * D);
    const uint32_t vt = kt + 2 * TILE;
    const float* const s_ks = s_sc + st * 3 * KT + off;
    const float* const s_vs = s_ks + KT;
    // Four K operands in flight: read j + 4 goes out when product j has taken
    // its buffer (left to itself, the compiler waits out each read in turn).
    f32x16_t sv[KB];
    __builtin_amdgcn_s_setprio(1);
    if constexpr (kWide) {
      // a step of two dims: d from half h = 0, d + 4 from h = 1
      constexpr int NJ = KB * (D / 8);
      auto kread = [&](int j) __attribute__((always_inline)) {
        const int chunk = 2 * (j % (D / 8)) + h;
        return *reinterpret_cast<const float4*>(
            s_dyn + kt + 4 * (32 * (j / (D / 8)) + lr) * D + 16 * (chunk ^ (lr & 15)));
      };
      float4 ka[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) ka[j] = kread(j);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        __builtin_amdgcn_sched_barrier(0);
        const int kb = j / (D / 8), s = j % (D / 8);
        if (s == 0) sv[kb] = f32x16_t{};
        sv[kb] = mfma32_f32(ka[j & 1].x, qw[s].x, sv[kb]);
        sv[kb] = mfma32_f32(ka[j & 1].y, qw[s].y, sv[kb]);
        sv[kb] = mfma32_f32(ka[j & 1].z, qw[s].z, sv[kb]);
        sv[kb] = mfma32_f32(ka[j & 1].w, qw[s].w, sv[kb]);
        if (j + 2 < NJ) ka[j & 1] = kread(j + 2);
      }
      __builtin_amdgcn_sched_barrier(0);
    } else {
      constexpr int NJ = KB * QSTEPS;
      auto kread = [&](int j) __attribute__((always_inline)) {
        return *reinterpret_cast<const uint4*>(
            s_dyn + ((kt + k_at) ^ (32 * (j % QSTEPS))) + 64 * (j / QSTEPS) * D);
      };
      uint4 ka[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) ka[j] = kread(j);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        __builtin_amdgcn_sched_barrier(0);
        const int kb = j / QSTEPS, s = j % QSTEPS;
#pragma unroll
        for (int p = P::QP - 1; p >= 0; --p)       // the small parts first
          sv[kb] = KM::run(__builtin_bit_cast(qv8, ka[j & 3]), qf[p][s],
                           s || p + 1 < P::QP ? sv[kb] : f32x16_t{});
        if (j + 4 < NJ) ka[j & 3] = kread(j + 4);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    // x in log2 units; the first key that some row may not see
    float mx = kNegBig;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      if constexpr (kCodes) {
        scale_rows(sv[kb], s_ks[32 * kb + own_key], Sixteen{});
        if constexpr (P::kLog) add_rows(sv[kb], s_vs[32 * kb + own_key], Sixteen{});
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) sv[kb][i] *= a.r.scale_log2;
      }
    }
    const int open = TREE ? U.committed : U.committed + U.row0 / G + 1;
    if (k0 + 32 * KB > min(open, U.kend)) {            // the same in all lanes
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const int kk = k0 + 32 * kb;
        uint32_t win = ~0u;
        if constexpr (TREE) win = tree_window(kk - U.committed);
        const int d = lim - kk - 4 * h;
        win >>= 4 * h;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int at = 8 * (i >> 2) + (i & 3);
          if (at > d || !((win >> at) & 1)) sv[kb][i] = -__builtin_inff();
        }
      }
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sv[kb][i]);
    mx = xor32_max(mx);
    float alpha = 1.0f;
    if (mx > m_run + P::kTop) {
      alpha = fast_exp2(m_run - (mx - P::kLift));
      m_run = mx - P::kLift;
    }
    if (__ballot(alpha != 1.0f)) {                 // rare after a row's first tile
      l_run *= alpha;
#pragma unroll
      for (int b = 0; b < DBLK; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[b][i] *= alpha;
    }
    i16x4_t vlo[2][DBLK], vhi[2][DBLK];
    auto vread = [&](int buf, int step) __attribute__((always_inline)) {
#pragma unroll
      for (int b = 0; b < DBLK; ++b) {
        vlo[buf][b] = lds_read_tr16(reinterpret_cast<const uint16_t*>(
            s_dyn + ((vt + v_at[0]) ^ (64 * b)) + 32 * step * D));
        vhi[buf][b] = lds_read_tr16(reinterpret_cast<const uint16_t*>(
            s_dyn + ((vt + v_at[1]) ^ (64 * b)) + 32 * step * D));
      }
    };
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
      for (int i = 0; i < 16; ++i) sv[kb][i] = fast_exp2(sv[kb][i] - m_run);
      if constexpr (P::kLog) {
        l_run = sum_rows(sv[kb], s_vs[KT + 32 * kb + own_key], l_run);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) l_run += sv[kb][i];
        if constexpr (kCodes)
          scale_rows(sv[kb], s_vs[32 * kb + own_key], Sixteen{});
      }
      if constexpr (kWide) {
        // a step of two keys: 8 q4 + e from half h = 0, 4 more from h = 1, as
        // the scores lie
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = 32 * kb + 8 * (i >> 2) + (i & 3) + 4 * h;
#pragma unroll
          for (int b = 0; b < DBLK; ++b) {
            const float v = *reinterpret_cast<const float*>(
                s_dyn + vt + 4 * key * D + 16 * ((8 * b + (lr >> 2)) ^ (8 * h)) + 4 * (lr & 3));
            o[b] = mfma32_f32(v, sv[kb][i], o[b]);
          }
        }
        continue;
      }
      uint32_t pw[P::PP][8];
#pragma unroll
      for (int p = 0; p < P::PP; ++p)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float x = sv[kb][2 * i], y = sv[kb][2 * i + 1];
          if constexpr (P::PP == 2 && std::is_same<typename P::V, f16>::value) {
            pw[p][i] = p == 0 ? take_part<f16>(x, y, true) : rest_of(pw[0][i], x, y);
          } else {
            pw[p][i] = take_part<typename P::V>(x, y, p + 1 == P::PP);
            sv[kb][2 * i] = x;
            sv[kb][2 * i + 1] = y;
          }
        }
      // Each step's V operands are read while the step before is multiplied.
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        if (kb == 0 && s == 0) vread(0, 0);
        if (2 * kb + s + 1 < 2 * KB) vread((s + 1) & 1, 2 * kb + s + 1);
#pragma unroll
        for (int p = P::PP - 1; p >= 0; --p) {
          const uint32_t* pp = &pw[p][4 * s];
          const auto pb = __builtin_bit_cast(typename VM::v8, make_uint4(pp[0], pp[1], pp[2], pp[3]));
#pragma unroll
          for (int b = 0; b < DBLK; ++b) {
            const i16x8_t va = __builtin_shufflevector(vlo[s][b], vhi[s][b], 0, 1, 2, 3, 4, 5, 6, 7);
            o[b] = VM::run(__builtin_bit_cast(typename VM::v8, va), pb, o[b]);
          }
        }
      }
    }
  };

  // The piece's tiles [t0, t1) again, key by key: a lane's row against every
  // key of this wavefront that it sees, in the same dims.
  auto careful = [&](int t0, int t1) {
    m_run = kNegBig;
    l_run = 0.0f;
#pragma unroll
    for (int b = 0; b < DBLK; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[b][i] = 0.0f;
    const T* qp = (const T*)a.r.q + (int64_t)qrow * a.r.q_stride + (int64_t)qhead * D;
#pragma unroll 1
    for (int i = t0 * KPW; i < t1 * KPW; ++i) {
      const int key = i / KPW * KT + kg * KPW + i % KPW;
      if (key >= U.kend) continue;
      bool sees = key <= lim;
      if (TREE && key >= U.committed) {
        const int tt = key - U.committed;
        sees = sees && (tt >> 6) < a.b.mask_words &&
               (a.b.mask[(int64_t)qrow * a.b.mask_words + (tt >> 6)] >> (tt & 63)) & 1;
      }
      if (!sees) continue;
      const int64_t phys = physical_block(a.b, a.c.num_blocks, a.seq_begin + U.seq, key / kBs);
      const int64_t at = phys * a.c.blk + (key % kBs) * a.c.tok + U.kvh * a.c.head;
      const char* kp = (const char*)a.c.kv[0] + at * E::kBytes;
      float x = 0.0f;
#pragma unroll 1
      for (int d = 0; d < D; d += E::kPer16B) {
        float kf[E::kPer16B];
        E::unpack(load16(kp + d * E::kBytes), kf);
#pragma unroll
        for (int e = 0; e < E::kPer16B; ++e) x = fmaf(elem<T>::load(qp + d + e), kf[e], x);
      }
      x *= a.r.scale_log2;
      float vs = 1.0f;
      if constexpr (kCodes) {
        const int64_t so = phys * a.c.sblk + (key % kBs) * a.c.stok + U.kvh * a.c.shead;
        x *= a.c.scale[0][so];
        vs = a.c.scale[1][so];
      }
      const float mn = fmaxf(m_run, x), alpha = fast_exp2(m_run - mn);
      const float p = fast_exp2(x - mn);
      m_run = mn;
      l_run = l_run * alpha + (h == 0 ? p : 0.0f);   // both halves hold the row
      const char* vp = (const char*)a.c.kv[1] + (at + 4 * h) * E::kBytes;
#pragma unroll
      for (int b = 0; b < DBLK; ++b)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          float v[4];
          const char* vq = vp + (32 * b + 8 * q4) * E::kBytes;
          if constexpr (kCodes) {
            code<C>::unpack4(*reinterpret_cast<const uint32_t*>(vq), v);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = elem<C>::load((const C*)vq + e);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) o[b][4 * q4 + e] = fmaf(p * vs, v[e], o[b][4 * q4 + e] * alpha);
        }
    }
  };

  // Four dims of a row: to the output, or to the piece's slot.
  auto put = [&](int slot, int idx, int d, float x0, float x1, float x2, float x3) {
    if (slot < 0) {
      T* op = (T*)a.r.out + (int64_t)qrow * a.r.out_stride + (int64_t)qhead * D + d;
      if constexpr (std::is_same<T, float>::value)
        *reinterpret_cast<float4*>(op) = make_float4(x0, x1, x2, x3);
      else
        *reinterpret_cast<uint2*>(op) = make_uint2(Mfma32<T>::pack2(x0, x1), Mfma32<T>::pack2(x2, x3));
    } else {
      *reinterpret_cast<float4*>(a.acc + ((int64_t)slot * a.slot_rows + idx) * D + d) =
          make_float4(x0, x1, x2, x3);
    }
  };
  auto finish = [&](int t0, int t1) {
    float all = l_run, unit = P::kLog ? pow2(U.unit2) : 1.0f;
#pragma unroll
    for (int b = 0; b < DBLK; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) all += o[b][i];
    if (__ballot(!(fabsf(all) < __builtin_inff()))) {
      careful(t0, t1);
      unit = 1.0f;
    }
    const bool whole = t0 == 0 && t1 == U.ntiles;
    const int slot = whole ? -1 : 2 * w + (t0 == 0 ? 1 : 0);
    const int idx = 32 * rg + lr;                  // the row's place in the unit
    l_run = xor32_sum(l_run);
    if constexpr (KW == 1) {
      const float inv = l_run != 0.0f ? unit / l_run : 0.0f;
      if (!live) return;
      if (!whole && h == 0)
        *reinterpret_cast<float2*>(a.ml + ((int64_t)slot * a.slot_rows + idx) * 2) =
            make_float2(m_run, l_run);
#pragma unroll
      for (int b = 0; b < DBLK; ++b)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4)
          put(slot, idx, 32 * b + 8 * q4 + 4 * h, o[b][4 * q4] * inv, o[b][4 * q4 + 1] * inv,
              o[b][4 * q4 + 2] * inv, o[b][4 * q4 + 3] * inv);
    } else {
      constexpr int GRP = DBLK * 4 / KW;           // groups of four dims each wavefront ends with
      float4* const xo = reinterpret_cast<float4*>(s_dyn);     // [WAVES][DBLK * 4][64]
      team_barrier();                              // nobody reads the tiles any more
#pragma unroll
      for (int b = 0; b < DBLK; ++b)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4)
          xo[(wave * (DBLK * 4) + 4 * b + q4) * 64 + lane] =
              make_float4(o[b][4 * q4] * unit, o[b][4 * q4 + 1] * unit, o[b][4 * q4 + 2] * unit,
                          o[b][4 * q4 + 3] * unit);
      if (h == 0) s_ml[wave * 32 + lr] = make_float2(m_run, l_run);
      team_barrier();
      float2 ml[KW];
      float m = kNegBig, l = 0.0f;
#pragma unroll
      for (int k = 0; k < KW; ++k) {
        ml[k] = s_ml[(k * RW + rg) * 32 + lr];
        m = fmaxf(m, ml[k].x);
      }
#pragma unroll
      for (int k = 0; k < KW; ++k) {
        ml[k].x = fast_exp2(ml[k].x - m);
        l += ml[k].x * ml[k].y;
      }
      const float inv = l != 0.0f ? 1.0f / l : 0.0f;
      if (live && !whole && h == 0 && kg == 0)
        *reinterpret_cast<float2*>(a.ml + ((int64_t)slot * a.slot_rows + idx) * 2) =
            make_float2(m, l);
#pragma unroll
      for (int i = 0; i < GRP; ++i) {
        const int grp = kg * GRP + i;
        float4 s = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < KW; ++k) {
          const float4 v = xo[((k * RW + rg) * (DBLK * 4) + grp) * 64 + lane];
          s.x = fmaf(v.x, ml[k].x, s.x); s.y = fmaf(v.y, ml[k].x, s.y);
          s.z = fmaf(v.z, ml[k].x, s.z); s.w = fmaf(v.w, ml[k].x, s.w);
        }
        if (live)
          put(slot, idx, 32 * (grp >> 2) + 8 * (grp & 3) + 4 * h, s.x * inv, s.y * inv,
              s.z * inv, s.w * inv);
      }
      team_barrier();                              // the next tile may be written
    }
  };

  // -- the range ---------------------------------------------------------------
  for (int p = r0;;) {
    const int t1 = direct ? U.ntiles : min(U.ntiles, t + (r1 - p));
    set_piece(t);
    start();
    if constexpr (NST == 2) {
      // one tile computed, the next in registers on its way to the other stage,
      // the one after that being loaded: one barrier per tile
      write_tile(t, 0);
      if (t + 1 < t1) load_tile(t + 1);
      team_barrier();
      for (int i = t, st = 0; i < t1; ++i, st ^= 1) {
        // Of eight wavefronts the second four, which share the SIMDs of the
        // first, write half a tile later: one multiplies while the other does
        // not (214 -> 202 us for trees of 25-60 tokens over codes, with weights of
        // one part).
#pragma unroll 1
        for (int sub = 0; sub < F::SUB; ++sub) {
          if (i + 1 < t1 && sub == (F::SUB == 2 ? wave >> 2 : 0)) {
            write_tile(i + 1, st ^ 1);
            if (i + 2 < t1) load_tile(i + 2);
          }
          compute(i, st, sub);
        }
        team_barrier();
      }
    } else {
      for (int i = t; i < t1; ++i) {
        if constexpr (RW > 1) team_barrier();      // the last tile has been read
        write_tile(i, 0);
        if (i + 1 < t1) load_tile(i + 1);
        if constexpr (RW > 1) team_barrier();
        else wait_lds();
        compute(i, 0, 0);
      }
    }
    finish(t, t1);
    p += t1 - t;
    if (direct || p >= r1) break;
    U = next_unit<TREE, F>(a, U, G);
    make_uniform(U);
    t = 0;
  }
}

// Joins the pieces of the units that span several ranges: workgroup (w, y)
// the unit that crosses the start of range w and begins in range w - 1, its
// rows rows_per y ...  Its pieces lie in slots 2 (w - 1) + 1, 2 w, 2 (w + 1),
// ...  D / 4 lanes per row, `rows_per` rows at a time, the rest of the
// workgroup the row's other pieces; four pieces' loads are in flight at once
// (two sequences of 131000 tokens over 2048 ranges, 128 pieces a row: 18.5 ->
// 9.6 us).
template <typename T, int D>
__global__ __launch_bounds__(256) void attn_join_kernel(TileArgs a, int rows_per) {
  constexpr int LPR = D / 4, TEAMS = 256 / LPR, U = 4;
  __shared__ float2 s_ml[TEAMS];
  __shared__ float4 s_o[TEAMS][LPR];
  const int w = blockIdx.x + 1;
  const int4 hd = a.head[2 * w];
  if (hd.x == 0) return;
  const int nrows = a.head[2 * w + 1].x;
  const int team = threadIdx.x / LPR, d = 4 * (threadIdx.x % LPR);
  const int parts = TEAMS / rows_per;          // pieces taken side by side
  const int slot_rows = a.slot_heads * a.slot_rows;
  const int row = (int)blockIdx.y * rows_per + team / parts;   // of the slot
  const int head = row / a.slot_rows, own = row - head * a.slot_rows;
  const bool on = head < a.slot_heads && own < nrows;
  float m = kNegBig, l = 0.0f, o[4] = {};
  auto fold = [&](const float2& ml, const float4& v, float weight) {
    const float mn = fmaxf(m, ml.x), f0 = fast_exp2(m - mn), f1 = weight * fast_exp2(ml.x - mn);
    m = mn;
    l = l * f0 + ml.y * fast_exp2(ml.x - mn);
    o[0] = o[0] * f0 + v.x * f1; o[1] = o[1] * f0 + v.y * f1;
    o[2] = o[2] * f0 + v.z * f1; o[3] = o[3] * f0 + v.w * f1;
  };
  if (on) {
    for (int i = team % parts; i < hd.x; i += U * parts) {
      float2 ml[U];
      float4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int e = min(i + u * parts, hd.x - 1);
        const int64_t slot = e == 0 ? 2 * (w - 1) + 1 : 2 * (w - 1 + e);
        ml[u] = *reinterpret_cast<const float2*>(a.ml + (slot * slot_rows + row) * 2);
        v[u] = *reinterpret_cast<const float4*>(a.acc + (slot * slot_rows + row) * D + d);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * parts < hd.x) fold(ml[u], v[u], ml[u].y);
    }
  }
  if (parts > 1) {
    if (d == 0) s_ml[team] = make_float2(m, l);
    s_o[team][d / 4] = make_float4(o[0], o[1], o[2], o[3]);
    __syncthreads();
    if (team % parts != 0 || !on) return;
    for (int k = 1; k < parts; ++k) fold(s_ml[team + k], s_o[team + k][d / 4], 1.0f);
  }
  if (!on) return;
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;
  const int g = a.r.num_heads / a.r.num_kv_heads;
  const int idx = hd.w + own;
  T* op = (T*)a.r.out + (int64_t)(hd.y + idx / g) * a.r.out_stride +
          (int64_t)((hd.z + head) * g + idx % g) * D + d;
#pragma unroll
  for (int i = 0; i < 4; ++i) elem<T>::store(op + i, o[i] * inv);
}

}  // namespace lv
