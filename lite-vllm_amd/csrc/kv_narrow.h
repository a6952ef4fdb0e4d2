// Attention of few query rows per sequence (decode rows, small trees) over the
// 8-bit paged cache.
//
// Up to 8 rows read each cached row here, so HBM is the bound and everything
// else has to stay out of its way.  The list is that of all sequences' tiles of
// 32 keys, a workgroup owns a contiguous range of it, and its wavefronts are
// the kv heads (up to 8): they walk the same tiles side by side, so that a
// block's rows of all heads, one run of memory, are read together (a wavefront
// with a range of its own over one head's tiles reads runs of 2 KiB and half
// lines of scales: 110 us for 256 sequences of 16-2048 tokens against 96).
// A barrier every few tiles, with no wait for loads, keeps them together.
//   * Codes and scales go from HBM to LDS directly (global_load_lds), two
//     stages of one tile, waits by vmcnt; tile i + 1 is in flight while tile i
//     is computed.
//   * S^T = K Q^T on 16x16x32: a lane's 16 bytes of LDS are 16 codes of one
//     key, i.e. the operands of two products; the query is laid out to match.
//   * O^T += V^T P^T on 16x16x32 over the tile's 32 keys: V^T by the 8-bit
//     LDS transpose read (a lane gets 8 keys of one dim), 8 products for 128
//     dims.  The 16 columns are the rows' leading parts of P, then their
//     second parts (bf16 each, 16 bits together), so both are one product.
// Codes become bf16 (for fp16 queries K's become fp16) in registers, exactly:
// about 200 of the 350 vector instructions of a tile.
//
// LDS row r (a key) holds its 16-byte chunk j at j ^ swz(r), which keeps the K
// reads (16 rows, one chunk) and the transpose reads (rows 4 g .. and 16 + 4 g
// .., one chunk) free of bank conflicts.
#pragma once
#include "kv_tiles.h"

namespace lv {

constexpr int kNarrowKeys = 32;
constexpr int kNarrowWaves = 8;      // kv heads of a workgroup, at most
constexpr int kNarrowSync = 3;       // barrier every 4 tiles

template <int D> struct NarrowStage {
  static constexpr int CPR = D / 16;               // 16-byte chunks per row
  static constexpr int RPL = 64 / CPR;             // rows of a wavefront-wide load
  static constexpr int LOADS = kNarrowKeys / RPL;  // loads of a tile's K or V
  static constexpr int KV = kNarrowKeys * D;       // bytes of a tile's K or V
  static constexpr int BYTES = 2 * KV + 2 * kNarrowKeys * 4;
  static constexpr int PER = 2 * LOADS + 1;        // vector-memory operations of a stage
  __device__ __forceinline__ static int swz(int row) {
    if constexpr (D == 128) return ((row >> 1) & 7) ^ (row & 16 ? 4 : 0);
    return ((row >> 2) & 3) ^ (row & 16 ? 2 : 0);
  }
  __device__ __forceinline__ static int at(int row, int chunk) {
    return row * D + 16 * (chunk ^ swz(row));
  }
};

__device__ __forceinline__ float xor16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return __uint_as_float(threadIdx.x & 16 ? r[0] : r[1]);
}

typedef int i32x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ i32x2_t lds_read_tr8(const unsigned char* p) {
  return __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2_t*)p);
}

// 4 codes -> 4 operands of 16 bits.
template <typename O, typename C>
__device__ __forceinline__ void codes4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  uint4 out[2];
  codes_to_operands<O, C>(make_uint4(w, 0, 0, 0), out);
  lo = out[0].x;
  hi = out[0].y;
}

template <typename T, typename C, int D, bool TREE>
__global__ __launch_bounds__(64 * kNarrowWaves, 1) void attn_narrow_kernel(TileArgs a) {
  using S = NarrowStage<D>;
  using KO = typename Operands<T, C>::K;
  using KM = Mfma16<KO>;
  using VM = Mfma16<bf16>;
  constexpr int QS = D / 32;                       // products of K Q^T per 16 keys
  constexpr int NB = D / 16;                       // 16-dim blocks of O^T
  extern __shared__ __align__(16) unsigned char s_dyn[];
  __shared__ int s_part[kNarrowWaves];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int waves = (int)blockDim.x >> 6;          // kv heads of the workgroup
  int* const s_off = reinterpret_cast<int*>(s_dyn + waves * 2 * S::BYTES);

  const int H = a.r.num_heads, Hkv = a.r.num_kv_heads;
  const int G = H / Hkv;
  const int groups = Hkv / waves;                  // groups of kv heads
  // tiles of every sequence: all its rows form one unit per group of heads
  {
    const int t = threadIdx.x, nt = blockDim.x;
    const int per = (a.n_seqs + nt - 1) / nt;
    const int lo = min(a.n_seqs, t * per), hi = min(a.n_seqs, lo + per);
    int sum = 0;
    for (int i = lo; i < hi; ++i) {
      s_off[i] = sum;
      const Seq s = tile_sequence(a, i);
      if (s.n > 0) sum += groups * max(1, (s.ctx + kNarrowKeys - 1) / kNarrowKeys);
    }
    int incl = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int u = __shfl_up(incl, d);
      if (lane >= d) incl += u;
    }
    if (lane == 63) s_part[wave] = incl;
    __syncthreads();
    int base = incl - sum;
    for (int w = 0; w < wave; ++w) base += s_part[w];
    for (int i = lo; i < hi; ++i) s_off[i] += base;
    if (t == nt - 1) s_off[a.n_seqs] = base + sum;
    __syncthreads();
  }
  const int total = s_off[a.n_seqs];
  const int w = (int)blockIdx.x;                   // the workgroup's range
  const int ranges = (int)gridDim.x;
  const int per = max(1, (int)(((int64_t)total + ranges - 1) / ranges));
  const int r0 = (int)min((int64_t)total, (int64_t)w * per);
  const int r1 = (int)min((int64_t)total, (int64_t)(w + 1) * per);
  if (threadIdx.x == 0) a.head[2 * w] = make_int4(0, 0, 0, 0);
  if (r0 >= r1) return;

  const int col = lane & 15, g = lane >> 4;
  const unsigned char* const stage0 = s_dyn + wave * 2 * S::BYTES;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)stage0);

  // Load u of a tile fills rows RPL u ..: lane l's 16 bytes land in slot
  // l % CPR of row RPL u + l / CPR, which holds chunk slot ^ swz(row).
  uint32_t goff[S::LOADS];
#pragma unroll
  for (int u = 0; u < S::LOADS; ++u) {
    const int r = S::RPL * u + lane / S::CPR;
    goff[u] = (uint32_t)((r & 15) * (int)a.c.tok) + 16u * ((lane % S::CPR) ^ S::swz(r));
  }
  const float* const sbase = (lane < 32 ? a.c.scale[0] : a.c.scale[1]) + (lane & 15) * a.c.stok;
  auto stage = [&](int s, int id0, int id1, int kvh) __attribute__((always_inline)) {
    const uint32_t dst = lds0 + s * S::BYTES;
    const uint64_t at0 = (uint64_t)((int64_t)id0 * a.c.blk + kvh * a.c.head);
    const uint64_t at1 = (uint64_t)((int64_t)id1 * a.c.blk + kvh * a.c.head);
    const int64_t sc = (int64_t)(lane & 16 ? id1 : id0) * a.c.sblk + kvh * a.c.shead;
    wait_lds();      // the stage's last reads have returned
#pragma unroll
    for (int u = 0; u < S::LOADS; ++u)
      load_lds16_stream((uint64_t)a.c.kv[0] + (2 * u < S::LOADS ? at0 : at1), goff[u],
                        dst + 1024 * u);
#pragma unroll
    for (int u = 0; u < S::LOADS; ++u)
      load_lds16_stream((uint64_t)a.c.kv[1] + (2 * u < S::LOADS ? at0 : at1), goff[u],
                        dst + S::KV + 1024 * u);
    load_lds4_async(sbase + sc, dst + 2 * S::KV);
  };

  int koff[2][D / 64], voff[NB];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int s = 0; s < D / 64; ++s) koff[t][s] = S::at(16 * t + col, 4 * s + g);
  {
    const int r = col >> 1, row = (r < 4 ? 0 : 12) + 4 * g + r;
#pragma unroll
    for (int b = 0; b < NB; ++b) voff[b] = S::at(row, b) + 8 * (col & 1);
  }

  // -- a piece's state -------------------------------------------------------
  uint4 qf[QS];
  f32x4_t o[NB];
  float m = kNegBig, l = 0.0f;
  int seq = -1, kvh = 0, kend = 0, committed = 0, rows = 0, first = 0;
  int qrow = 0, qhead = 0, lim = 0, cols = 1;
  bool live = false;

  auto start = [&](int sq, int kv, int tile) __attribute__((always_inline)) {
    const Seq s = tile_sequence(a, sq);
    seq = sq; kvh = kv; first = tile;
    kend = s.ctx;
    committed = s.ctx - s.n;
    rows = min(s.n, a.max_q) * G;
    cols = rows <= 1 ? 1 : rows <= 2 ? 2 : rows <= 4 ? 4 : 8;
    const int r = col & (cols - 1);
    live = col < rows;
    const int use = r < rows ? r : 0;
    qrow = s.q0 + use / G;
    qhead = kv * G + use % G;
    lim = TREE ? kend - 1 : min(committed + use / G, kend - 1);
    const T* qp = (const T*)a.r.q + (int64_t)qrow * a.r.q_stride + (int64_t)qhead * D + 16 * g;
#pragma unroll
    for (int i = 0; i < QS; ++i) qf[i] = load16(qp + 64 * (i >> 1) + 8 * (i & 1));
    settle(qf);
#pragma unroll
    for (int b = 0; b < NB; ++b) o[b] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    m = kNegBig;
    l = 0.0f;
  };

  auto sees_drafted = [&](int t) {
    return (t >> 6) < a.b.mask_words &&
           (a.b.mask[(int64_t)qrow * a.b.mask_words + (t >> 6)] >> (t & 63)) & 1;
  };

  auto process = [&](int s, int tile) __attribute__((always_inline)) {
    unsigned char* const kt = s_dyn + wave * 2 * S::BYTES + s * S::BYTES;
    unsigned char* const vt = kt + S::KV;
    float* const sc = reinterpret_cast<float*>(vt + S::KV);
    const int k0 = tile * kNarrowKeys;
    const int left = kend - k0;                    // keys of the tile in the context
    if (left < kNarrowKeys) {
      // rows past the context may hold anything: zero their V and its scales
      for (int c = lane; c < kNarrowKeys * S::CPR; c += 64)
        if (c / S::CPR >= left)
          *reinterpret_cast<uint4*>(vt + 16 * c) = make_uint4(0, 0, 0, 0);
      if (lane >= 32 && lane - 32 >= left) sc[lane] = 0.0f;
    }
    float x[8], vs[8];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f32x4_t acc = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        uint4 op[2];
        codes_to_operands<KO, C>(*reinterpret_cast<const uint4*>(kt + koff[t][i]), op);
        acc = KM::run32(op[0], qf[2 * i], acc);
        acc = KM::run32(op[1], qf[2 * i + 1], acc);
      }
      const float4 ks = *reinterpret_cast<const float4*>(sc + 16 * t + 4 * g);
      const float4 v4 = *reinterpret_cast<const float4*>(sc + 32 + 16 * t + 4 * g);
      x[4 * t] = acc[0] * ks.x; x[4 * t + 1] = acc[1] * ks.y;
      x[4 * t + 2] = acc[2] * ks.z; x[4 * t + 3] = acc[3] * ks.w;
      vs[4 * t] = v4.x; vs[4 * t + 1] = v4.y; vs[4 * t + 2] = v4.z; vs[4 * t + 3] = v4.w;
    }
    float mx = kNegBig;
    const int open = TREE ? committed : committed + 1;
    const bool masked = k0 + kNarrowKeys > min(open, kend);     // the same in all lanes
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= a.r.scale_log2;
    if (masked) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int key = k0 + 16 * (e >> 2) + 4 * g + (e & 3);
        bool sees = key <= lim;
        if (TREE && key >= committed) sees = sees && sees_drafted(key - committed);
        if (!sees) x[e] = -__builtin_inff();
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) mx = fmaxf(mx, x[e]);
    mx = fmaxf(mx, xor16(mx));
    mx = xor32_max(mx);
    if (__ballot(mx > m + 8.0f)) {                 // rare after a row's first tile
      if (mx > m + 8.0f) {
        const float alpha = fast_exp2(m - mx);
        m = mx;
        l *= alpha;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[b][e] *= alpha;
      }
    }
    const bool second = (col & cols) != 0;         // this column holds the second parts
    float z[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float p = fast_exp2(x[e] - m);
      l += p;
      z[e] = p * vs[e];
      const float head = __uint_as_float(__float_as_uint(z[e]) & 0xffff0000u);
      z[e] = second ? z[e] - head : head;
    }
    const uint4 pw = make_uint4(float_to_bf16_pair(z[0], z[1]), float_to_bf16_pair(z[2], z[3]),
                                float_to_bf16_pair(z[4], z[5]), float_to_bf16_pair(z[6], z[7]));
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const i32x2_t w8 = lds_read_tr8(vt + voff[b]);
      uint4 va;
      codes4<bf16, C>((uint32_t)w8.x, va.x, va.y);
      codes4<bf16, C>((uint32_t)w8.y, va.z, va.w);
      o[b] = VM::run32(va, pw, o[b]);
    }
  };

  // Tiles [t0, t1) again, key by key (see the tile kernel).
  auto careful = [&](int t0, int t1) {
    m = kNegBig;
    l = 0.0f;
#pragma unroll
    for (int b = 0; b < NB; ++b) o[b] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    if (col >= cols) return;
    const T* qp = (const T*)a.r.q + (int64_t)qrow * a.r.q_stride + (int64_t)qhead * D;
    const int end = min(t1 * kNarrowKeys, kend);
#pragma unroll 1
    for (int key = t0 * kNarrowKeys; key < end; ++key) {
      bool sees = key <= lim;
      if (TREE && key >= committed) sees = sees && sees_drafted(key - committed);
      if (!sees) continue;
      const int64_t phys = physical_block(a.b, a.c.num_blocks, a.seq_begin + seq, key / kBs);
      const int64_t at = phys * a.c.blk + (key % kBs) * a.c.tok + kvh * a.c.head;
      const int64_t so = phys * a.c.sblk + (key % kBs) * a.c.stok + kvh * a.c.shead;
      float x = 0.0f;
#pragma unroll 1
      for (int d = 0; d < D; d += 16) {
        float kf[16];
        cached<C>::unpack(load16((const char*)a.c.kv[0] + at + d), kf);
#pragma unroll
        for (int e = 0; e < 16; ++e) x = fmaf(elem<T>::load(qp + d + e), kf[e], x);
      }
      x *= a.r.scale_log2 * a.c.scale[0][so];
      const float mn = fmaxf(m, x), alpha = fast_exp2(m - mn), p = fast_exp2(x - mn);
      const float z = p * a.c.scale[1][so];
      m = mn;
      l = l * alpha + (g == 0 ? p : 0.0f);         // the four lanes of a column share the row
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float v[4];
        code<C>::unpack4(*reinterpret_cast<const uint32_t*>((const char*)a.c.kv[1] + at + 16 * b + 4 * g), v);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[b][e] = fmaf(z, v[e], o[b][e] * alpha);
      }
    }
  };

  auto finish = [&](int t1) {
    float all = 0.0f;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) all += o[b][e];
    if (__ballot(col < 2 * cols && !(fabsf(all) < __builtin_inff()))) careful(first, t1);
    // (columns past the two parts' hold products of no use)
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[b][e] += __shfl(o[b][e], lane + cols);
    float L = l + xor16(l);
    L = xor32_sum(L);
    const int ntiles = max(1, (kend + kNarrowKeys - 1) / kNarrowKeys);
    const bool whole = first == 0 && t1 == ntiles;
    if (!live) return;
    const float inv = L != 0.0f ? 1.0f / L : 0.0f;
    if (whole) {
      T* op = (T*)a.r.out + (int64_t)qrow * a.r.out_stride + (int64_t)qhead * D + 4 * g;
#pragma unroll
      for (int b = 0; b < NB; ++b)
        *reinterpret_cast<uint2*>(op + 16 * b) =
            make_uint2(Mfma32<T>::pack2(o[b][0] * inv, o[b][1] * inv),
                       Mfma32<T>::pack2(o[b][2] * inv, o[b][3] * inv));
      return;
    }
    const int64_t at =
        ((int64_t)(2 * w + (first == 0 ? 1 : 0)) * waves + wave) * a.slot_rows + col;
    if (g == 0) *reinterpret_cast<float2*>(a.ml + at * 2) = make_float2(m, L);
#pragma unroll
    for (int b = 0; b < NB; ++b)
      *reinterpret_cast<float4*>(a.acc + at * D + 16 * b + 4 * g) =
          make_float4(o[b][0] * inv, o[b][1] * inv, o[b][2] * inv, o[b][3] * inv);
  };

  // -- the range -----------------------------------------------------------------
  int last_tile = 0;
  for (int base = r0; base < r1; base += 64) {
    // lane l resolves place base + l of the list
    const int cnt = min(64, r1 - base);
    const int p = min(base + lane, r1 - 1);
    int lo = 0, hi = a.n_seqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_off[mid] <= p) lo = mid; else hi = mid - 1;
    }
    const int nt = (s_off[lo + 1] - s_off[lo]) / groups;
    const int rem = p - s_off[lo];
    const int e_seq = lo, e_grp = rem / nt, e_tile = rem - e_grp * nt;
    int e_id0 = 0, e_id1 = 0;
    {
      const Seq s = tile_sequence(a, lo);
      const int last = (s.ctx - 1) / kBs;
      if (s.ctx > 0) {
        e_id0 = physical_block(a.b, a.c.num_blocks, a.seq_begin + lo, min(2 * e_tile, last));
        e_id1 = physical_block(a.b, a.c.num_blocks, a.seq_begin + lo, min(2 * e_tile + 1, last));
      }
    }
    if (base == r0 && threadIdx.x == 0 && e_tile > 0 && r0 - e_tile >= r0 - per) {
      // the range starts inside a unit that starts in the range before: this
      // range's workgroup of the join takes it
      const Seq s = tile_sequence(a, lo);
      a.head[2 * w] = make_int4((r0 - e_tile + nt - 1) / per - w + 2, s.q0, e_grp * waves, 0);
      a.head[2 * w + 1] = make_int4(min(s.n, a.max_q) * G, 0, 0, 0);
    }
    auto get = [&](int v, int i) { return __builtin_amdgcn_readlane(v, i); };
    stage(0, get(e_id0, 0), get(e_id1, 0), get(e_grp, 0) * waves + wave);
    for (int i = 0; i < cnt; ++i) {
      if ((i & kNarrowSync) == 0) __builtin_amdgcn_s_barrier();
      const int sq = get(e_seq, i), kv = get(e_grp, i) * waves + wave, tile = get(e_tile, i);
      if (sq != seq || kv != kvh) {
        if (seq >= 0) finish(last_tile + 1);
        start(sq, kv, tile);
      }
      if (i + 1 < cnt)
        stage((i + 1) & 1, get(e_id0, i + 1), get(e_id1, i + 1),
              get(e_grp, i + 1) * waves + wave);
      if (i + 1 < cnt) wait_vmem<S::PER>();        // tile i has landed, i + 1 may not have
      else wait_vmem<0>();
      process(i & 1, tile);
      last_tile = tile;
    }
  }
  if (seq >= 0) finish(last_tile + 1);
}

}  // namespace lv
