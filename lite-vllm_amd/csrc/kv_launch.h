// Launches of the attention kernels over paged caches (included by one
// translation unit per query type).
#pragma once
#include "kv_narrow.h"
#include "kv_tiles.h"

namespace lv {

inline TileArgs tile_args(const Call& a, const TilePlan& p, char* ws) {
  TileArgs t{};
  t.b = a.b; t.c = a.c; t.r = a.r;
  t.seq_begin = p.seq_begin; t.n_seqs = p.n_seqs; t.max_q = p.max_q;
  t.ranges = p.ranges;
  t.direct = p.direct;
  t.nq = p.nq;
  t.slot_heads = p.slot_heads;
  t.slot_rows = p.slot_rows;
  t.head = reinterpret_cast<int4*>(ws);
  t.ml = reinterpret_cast<float*>(ws + p.head_bytes);
  t.acc = reinterpret_cast<float*>(ws + p.head_bytes + p.ml_bytes);
  return t;
}

template <typename T, int D>
int launch_join(const Call& a, const TilePlan& p, const TileArgs& t) {
  if (p.ranges < 2) return LV_OK;
  constexpr int TEAMS = 256 / (D / 4);
  // few rows may have many pieces: the teams share them
  const int rows = p.slot_heads * p.slot_rows;
  const int rows_per = p.slot_rows <= 8 ? 1 : TEAMS;
  attn_join_kernel<T, D><<<dim3((unsigned)p.ranges - 1, (unsigned)((rows + rows_per - 1) / rows_per)),
                           256, 0, a.stream>>>(t, rows_per);
  return check_launch("attn_join_kernel");
}

template <typename T, typename C, int D, bool TREE, int RW, int WAVES>
int launch_tile_kernel(const Call& a, const TilePlan& p, char* ws) {
  using F = TileCfg<RW, WAVES>;
  const TileArgs t = tile_args(a, p, ws);
  constexpr size_t tiles = F::lds(D, Operands<T, C>::kWide ? 4 : 2);
  static_assert(tiles + kOffsetBytes + kTileStaticLds <= kLdsBytes, "LDS of a CU");
  const size_t lds = tiles + (size_t)(p.n_seqs + 1) * 4;
  attn_tile_kernel<T, C, D, F, TREE><<<(unsigned)p.grid, F::THREADS, lds, a.stream>>>(t);
  if (const int rc = check_launch("attn_tile_kernel"); rc != LV_OK || p.direct >= 2)
    return rc;
  return launch_join<T, D>(a, p, t);
}

template <typename T, typename C, int D, bool TREE>
int launch_narrow_kernel(const Call& a, const TilePlan& p, char* ws) {
  const TileArgs t = tile_args(a, p, ws);
  static_assert(kNarrowWaves * 2 * NarrowStage<D>::BYTES + kOffsetBytes + kNarrowWaves * 4 <=
                    kLdsBytes, "LDS of a CU");
  const size_t lds = (size_t)p.slot_heads * 2 * NarrowStage<D>::BYTES + (size_t)(p.n_seqs + 1) * 4;
  attn_narrow_kernel<T, C, D, TREE>
      <<<(unsigned)p.grid, (unsigned)(64 * p.slot_heads), lds, a.stream>>>(t);
  if (const int rc = check_launch("attn_narrow_kernel"); rc != LV_OK) return rc;
  return launch_join<T, D>(a, p, t);
}

template <typename T, typename C, int D, bool TREE>
int launch_tiles_rw(const Call& a, const TilePlan& p, char* ws) {
  if (p.rw == 1) return launch_tile_kernel<T, C, D, TREE, 1, 4>(a, p, ws);
  if constexpr (std::is_same<T, float>::value) {
    if (p.rw == 2) return launch_tile_kernel<T, C, D, TREE, 2, 4>(a, p, ws);
  } else if (p.waves == 8) {
    if (p.rw == 2) return launch_tile_kernel<T, C, D, TREE, 2, 8>(a, p, ws);
    if (p.rw == 4) return launch_tile_kernel<T, C, D, TREE, 4, 8>(a, p, ws);
    return launch_tile_kernel<T, C, D, TREE, 8, 8>(a, p, ws);
  }
  return launch_tile_kernel<T, C, D, TREE, 4, 4>(a, p, ws);
}

template <typename T, typename C, int D>
int launch_tiles_d(const Call& a, const TilePlan& p, char* ws) {
  if constexpr (cached<C>::kCodes && !std::is_same<T, float>::value) {
    if (p.rw == 0)
      return a.tree ? launch_narrow_kernel<T, C, D, true>(a, p, ws)
                    : launch_narrow_kernel<T, C, D, false>(a, p, ws);
  }
  if (a.tree) return launch_tiles_rw<T, C, D, true>(a, p, ws);
  if constexpr (cached<C>::kCodes) return launch_tiles_rw<T, C, D, false>(a, p, ws);
  return LV_ERR_UNSUPPORTED;
}

template <typename T>
int launch_tiles(const Call& a, const TilePlan& p, char* ws) {
  if (a.code == LV_INT8)
    return a.d == 64 ? launch_tiles_d<T, int8_code, 64>(a, p, ws)
                     : launch_tiles_d<T, int8_code, 128>(a, p, ws);
  if (a.code == LV_E4M3)
    return a.d == 64 ? launch_tiles_d<T, e4m3_code, 64>(a, p, ws)
                     : launch_tiles_d<T, e4m3_code, 128>(a, p, ws);
  return a.d == 64 ? launch_tiles_d<T, T, 64>(a, p, ws) : launch_tiles_d<T, T, 128>(a, p, ws);
}

}  // namespace lv
