// tree_tiles.hpp -- the tile machinery of the paged attention kernels: LDS
// layouts, HBM -> LDS transfers of K and V tiles from the pages, and the MFMA
// phase, for 64-key tiles and head sizes 64 and 128.  The scheme (transposed
// products, key order inside a tile, rings, phases) is described where the
// kernels are, in tree_attention.hip and scored_attention.hpp.
#pragma once

#include <hip/hip_runtime.h>

#include "half_types.hpp"
#include "lds_dma.hpp"

namespace cfa {
namespace tree {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kKT = 64;                       // keys per tile
constexpr int kWaves = 8;
constexpr int kNT = kWaves * 64;              // threads per work-group
// A wave owns QT 16-row query tiles: two, or one for at most 64 query rows
// (then one wave per SIMD is busy either way, with half the work per tile: a
// draft level of 8 sequences x 8 nodes, head_dim 64, 13.5 -> 12.3 us).  From
// 65 to 128 rows one tile a wave would make all eight waves read every K and V
// operand from LDS instead of four: 31 nodes at head_dim 128 39.4 -> 47.7 us.
constexpr int kRowsOneTile = 64;
constexpr int kMaxRows = kWaves * 2 * 16;     // query rows per work-group
constexpr int kKStages = 4;                   // K-tile ring (tile u: stage u % 4)
constexpr int kVStages = 5;                   // V-tile ring (read one iteration after K)
constexpr float kRescaleSlack = 8.0f;         // log2 units

// Layout constants of head size D (64 or 128): K / V rows of D bf16 values,
// D / 8 16-byte chunks each.
template <int D, int QT = 2>
struct Geo {
  static_assert(D == 64 || D == 128, "head_dim 64 or 128");
  static constexpr int kRowBytes = D * 2;             // one K or V row
  static constexpr int kTileBytes = kKT * kRowBytes;  // 8 or 16 KiB
  static constexpr int kChunks = D / 8;               // 16-byte chunks per row
  static constexpr int kRowsPerLoad = 1024 / kRowBytes;  // rows per 1 KiB transfer
  static constexpr int kLoadsPerTile = 2 * (8 / kRowsPerLoad);  // K + V transfers per wave
  static constexpr int kKK = D / 32;                  // k-slices of the QK product
  static constexpr int kDT = D / 16;                  // 16-row blocks of O^T
  static constexpr int kMfma = 2 * kDT * QT + 2 * QT + 4 * kKK * QT;  // per MFMA phase
};
#ifndef CFA_TA_SGB
#define CFA_TA_SGB 1
#endif
constexpr int kMaxGroups = 1024;              // 16-key groups per split (page lookup table)
constexpr int kMaxTilesPerSplit = kMaxGroups / (kKT / 16);

// The matrix product of one 16 x 16 x 32 tile, by element type.
template <class T>
struct Mfma;
template <>
struct Mfma<BF16> {
  typedef bf16x8 frag;
  static __device__ __forceinline__ f32x4 run(frag a, frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mfma<FP16> {
  typedef f16x8 frag;
  static __device__ __forceinline__ f32x4 run(frag a, frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

__device__ __forceinline__ uint4 ld_g16(const uint16_t *p) {
  return *reinterpret_cast<const uint4 *>(p);
}

// Key (tile-relative) held by K-tile LDS row R.
__device__ __forceinline__ int k_key_of_row(int R) {
  return (R & ~31) + ((R >> 2) & 3) * 8 + ((R >> 4) & 1) * 4 + (R & 3);
}

// LDS swizzles (16-byte chunk c of a row sits at position c ^ swizzle):
//   K-tile row R:  D = 128: R % 16;  D = 64: (R / 2) % 8.  A 16-row MFMA
//     operand read then touches every bank once per 16 lanes.
//   V-tile row key: twice the 32-byte block swizzle vh, the same for keys k
//     and k + 4 (one transposed-read pair); D = 128: (key % 4) | 4 ((key / 8)
//     % 2); D = 64: ((key / 2) % 2) | 2 ((key / 8) % 2).  The four rows of one
//     transposed read then land in distinct banks.
template <int D>
__device__ __forceinline__ int k_swz(int R) {
  return D == 128 ? (R & 15) : ((R >> 1) & 7);
}
template <int D>
__device__ __forceinline__ int v_swz(int key) {
  return D == 128 ? (((key & 3) | ((key >> 1) & 4)) << 1) : ((((key >> 1) & 1) | ((key >> 2) & 2)) << 1);
}

// Key positions that a transfer reads lie below nkeys and, with kFrom, at
// `from` or behind it; others re-read the nearest of those.
template <bool kFrom>
__device__ __forceinline__ int clamp_pos(int pos, int from, int nkeys) {
  pos = min(pos, nkeys - 1);
  return kFrom ? max(pos, from) : pos;
}

// Pool element offset of the row holding position gstart = clamp_pos(16 gi),
// the first row 16-key group gi reads.  Page index and block id
// are clamped into the table and the pool, so a corrupt table can never send
// a load outside the pool.
template <int D, bool kFrom = false, class A>
__device__ __forceinline__ long long group_row_offset(const A &a, const int32_t *btb, int gi,
                                                      int nkeys, int h, int from = 0) {
  const int gstart = clamp_pos<kFrom>(gi * 16, from, nkeys);
  const int page = min(gstart / a.bs, a.max_blocks - 1);
  const int blk = min(max(btb[page], 0), a.num_blocks - 1);
  return (((long long)blk * a.num_layers + a.layer) * a.Hkv + h) * ((long long)a.bs * D) +
         (long long)(gstart - page * a.bs) * D;
}

__device__ __forceinline__ long long uniform_i64(long long v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)((unsigned long long)v >> 32));
  return (long long)(((unsigned long long)hi << 32) | lo);
}

// Issue this wave's share of the tile at key kbase: K-tile LDS rows 8w..8w+7
// and V keys 8w..8w+7, in 1 KiB transfers of 1024 / (2 D) rows.  Each
// transfer stays inside one 16-key group, and a group never straddles a page
// (block_size % 16 == 0).  Keys at or past nkeys re-read key nkeys - 1: a
// finite, in-bounds row that the mask then hides.  kt and vt point to the row
// offsets (group_row_offset) of the K and V group that the wave moves: of the
// tile's groups 2 (w / 4) + w % 2 and w / 2.
template <int D, bool kFrom = false, class A>
__device__ __forceinline__ void issue_tile(const A &a, const long long *kt, const long long *vt, int kbase,
                                           int nkeys, uint8_t *kdst, uint8_t *vdst, int wave,
                                           int lane, int from = 0) {
  using Gm = Geo<D>;
  constexpr int RPL = Gm::kRowsPerLoad;
  const int sub = lane / Gm::kChunks, pc = lane % Gm::kChunks;
  {
    // K: the wave's rows hold keys of the tile's 16-group 2 (w / 4) + (w % 2)
    const int gi = kbase / 16 + 2 * (wave >> 2) + (wave & 1);
    const int gstart = clamp_pos<kFrom>(gi * 16, from, nkeys);
    const uint16_t *base = a.kpool + uniform_i64(*kt);
#pragma unroll
    for (int j = 0; j < 8 / RPL; ++j) {
      const int R = 8 * wave + RPL * j + sub;
      const int c = pc ^ k_swz<D>(R);
      const int pos = clamp_pos<kFrom>(kbase + k_key_of_row(R), from, nkeys);
      dma16(base + ((pos - gstart) * D + c * 8),
            (CFA_LDS void *)(kdst + (8 * wave + RPL * j) * Gm::kRowBytes));
    }
  }
  {
    // V: keys 8w..8w+7, in the tile's 16-group w / 2
    const int gi = kbase / 16 + (wave >> 1);
    const int gstart = clamp_pos<kFrom>(gi * 16, from, nkeys);
    const uint16_t *base = a.vpool + uniform_i64(*vt);
#pragma unroll
    for (int j = 0; j < 8 / RPL; ++j) {
      const int key = 8 * wave + RPL * j + sub;
      const int c = pc ^ v_swz<D>(key);
      const int pos = clamp_pos<kFrom>(kbase + key, from, nkeys);
      dma16(base + ((pos - gstart) * D + c * 8),
            (CFA_LDS void *)(vdst + (8 * wave + RPL * j) * Gm::kRowBytes));
    }
  }
}

// Per-lane byte offsets, within their 16-key group, of this lane's K and V
// transfers (issue_tile's rows and chunks) for a tile that lies wholly below
// nkeys, where no position is clamped: the same for every such tile.
template <int D>
struct DmaOffs {
  uint32_t k[8 / Geo<D>::kRowsPerLoad], v[8 / Geo<D>::kRowsPerLoad];
};
template <int D>
__device__ __forceinline__ DmaOffs<D> dma_offsets(int wave, int lane) {
  using Gm = Geo<D>;
  constexpr int RPL = Gm::kRowsPerLoad;
  const int sub = lane / Gm::kChunks, pc = lane % Gm::kChunks;
  DmaOffs<D> o;
#pragma unroll
  for (int j = 0; j < 8 / RPL; ++j) {
    const int R = 8 * wave + RPL * j + sub;
    const int kin = k_key_of_row(R) - 32 * (wave >> 2) - 16 * (wave & 1);  // key in its group
    o.k[j] = (uint32_t)((kin * D + (pc ^ k_swz<D>(R)) * 8) * 2);
    const int key = 8 * wave + RPL * j + sub;
    const int vin = key - 16 * (wave >> 1);
    o.v[j] = (uint32_t)((vin * D + (pc ^ v_swz<D>(key)) * 8) * 2);
  }
  return o;
}

// issue_tile for a tile with kbase + 64 <= nkeys, from the precomputed
// offsets: per transfer only the group's page base, which is uniform.
template <int D, class A>
__device__ __forceinline__ void issue_tile_full(const A &a, const long long *kt, const long long *vt,
                                                const DmaOffs<D> &off, uint8_t *kdst, uint8_t *vdst,
                                                int wave) {
  using Gm = Geo<D>;
  constexpr int RPL = Gm::kRowsPerLoad;
  const uint16_t *kb = a.kpool + uniform_i64(*kt);
  const uint16_t *vb = a.vpool + uniform_i64(*vt);
#pragma unroll
  for (int j = 0; j < 8 / RPL; ++j)
    dma16_s(kb, off.k[j], (CFA_LDS void *)(kdst + (8 * wave + RPL * j) * Gm::kRowBytes));
#pragma unroll
  for (int j = 0; j < 8 / RPL; ++j)
    dma16_s(vb, off.v[j], (CFA_LDS void *)(vdst + (8 * wave + RPL * j) * Gm::kRowBytes));
}

// Visibility of the 64 keys kbase.. of a tile to a query whose ancestor mask
// (bits < N) is anc: context positions (< ctx) are all visible, tree position
// ctx + j is visible iff bit j of anc is set, positions past the tree never.
__device__ __forceinline__ uint64_t tile_visibility(int kbase, int ctx, uint64_t anc) {
  const int nctx = ctx - kbase;  // context keys at the start of the tile
  const uint64_t ctx_bits = nctx >= 64 ? ~0ull : (nctx <= 0 ? 0ull : ((1ull << nctx) - 1));
  // tile key k is tree node k - nctx
  const uint64_t tree_bits = nctx >= 0 ? (nctx >= 64 ? 0ull : anc << nctx)
                                       : (-nctx >= 64 ? 0ull : anc >> -nctx);
  return ctx_bits | tree_bits;
}

// Maximum over lanes l, l ^ 16, l ^ 32 and l ^ 48 (the four lanes holding
// one query column) without an LDS round trip: each permlane swap returns the
// lane's own value and its partner's (in one order or the other), so the max
// of the pair is the max of the two lanes.
__device__ __forceinline__ float column_max(float v) {
  const auto r32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r32[0]), __uint_as_float(r32[1]));
  const auto r16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r16[0]), __uint_as_float(r16[1]));
}

// Per-wave state of the pipelined loop: 16-row query tiles qt of this wave,
// scores of one 64-key tile s[qt][blk][T] (keys blk*32 + 8g + 4T + i) and its
// 16-bit probabilities p[qt][blk] (keys blk*32 + 8g + 0..7).
template <int QT>
struct Scores {
  f32x4 s[QT][2][2];
};
template <int QT, class T = BF16>
struct Probs {
  typename Mfma<T>::frag p[QT][2];
};

template <int D, int QT, class T = BF16>
struct Lane {
  typename Mfma<T>::frag qf[QT][D / 32];  // Q^T columns, scaled if the kernel wants it
  int koff[D / 32];        // K-tile LDS byte offsets of this lane's operand reads
  int vbase, vh;           // V-tile transposed-read offset and swizzle
  int g;                   // lane / 16
};

// S^T = K Q^T - base: the accumulators start at -b so that the products come
// out relative to the column's exponent base.
template <int D, int QT, class E = BF16>
__device__ __forceinline__ void qk_tile(const Lane<D, QT, E> &ln, const uint8_t *Ks, const float *b,
                                        Scores<QT> &S) {
#pragma unroll
  for (int qt = 0; qt < QT; ++qt)
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
      for (int T = 0; T < 2; ++T) S.s[qt][blk][T] = f32x4{-b[qt], -b[qt], -b[qt], -b[qt]};
#pragma unroll
  for (int kk = 0; kk < D / 32; ++kk)
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
      for (int T = 0; T < 2; ++T) {
        const uint4 kv = *reinterpret_cast<const uint4 *>(Ks + (blk * 32 + T * 16) * Geo<D>::kRowBytes +
                                                          ln.koff[kk]);
        const auto kf = __builtin_bit_cast(typename Mfma<E>::frag, kv);
#pragma unroll
        for (int qt = 0; qt < QT; ++qt)
          S.s[qt][blk][T] = Mfma<E>::run(kf, ln.qf[qt][kk], S.s[qt][blk][T]);
      }
}

// Online-softmax bookkeeping of one column: b is the exponent base (log2
// units) the scores are relative to, valid says b has been set.
template <int QT>
struct Softmax {
  float b[QT];
  bool valid[QT];
};

// MFMA phase of tile t: O^T += V_t^T P^T and l += 1^T P^T, then
// S = K_{t+1} Q^T - b (tile t+1's scores; for the last tile the stage read is
// stale and the result unused).  The QK products run k-slice outermost so
// that eight independent accumulation chains interleave: a dependent MFMA
// issued right behind its predecessor stalls the matrix pipe.  Lane (g, col)
// reads V rows blk*32 + 8g + 0..7 at d = dt*16 + col through two transposed
// 4x16 reads.
template <int D, int QT, class E = BF16, int READS = 2>
__device__ __forceinline__ void mfma_phase(const Lane<D, QT, E> &ln, const uint8_t *Knext, const uint8_t *Vs,
                                           const float *b, const Probs<QT, E> &P, Scores<QT> &S,
                                           f32x4 (&o)[QT][D / 16], f32x4 (&lacc)[QT]) {
  constexpr int RB = Geo<D>::kRowBytes;
  typename Mfma<E>::frag ones;
#pragma unroll
  for (int j = 0; j < 8; ++j) ones[j] = (typename E::elem)1.0f;
  f32x4 negb[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) negb[qt] = f32x4{-b[qt], -b[qt], -b[qt], -b[qt]};
  // the column sums first: they read no LDS, so they cover the latency of
  // the phase's first operand reads (about 1.5%)
#pragma unroll
  for (int blk = 0; blk < 2; ++blk)
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
      lacc[qt] = Mfma<E>::run(ones, P.p[qt][blk], lacc[qt]);
#pragma unroll
  for (int blk = 0; blk < 2; ++blk) {
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) {
      const uint8_t *vp = Vs + blk * 32 * RB + ln.vbase + ((dt ^ ln.vh) << 5);
      const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((CFA_LDS i16x4 *)vp);
      const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((CFA_LDS i16x4 *)(vp + 4 * RB));
      const auto vf = __builtin_bit_cast(typename Mfma<E>::frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
        o[qt][dt] = Mfma<E>::run(vf, P.p[qt][blk], o[qt][dt]);
    }
  }
#pragma unroll
  for (int kk = 0; kk < D / 32; ++kk)
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
      for (int T = 0; T < 2; ++T) {
        const auto kf = __builtin_bit_cast(
            typename Mfma<E>::frag, *reinterpret_cast<const uint4 *>(Knext + (blk * 32 + T * 16) * RB + ln.koff[kk]));
#pragma unroll
        for (int qt = 0; qt < QT; ++qt)
          S.s[qt][blk][T] =
              Mfma<E>::run(kf, ln.qf[qt][kk], kk == 0 ? negb[qt] : S.s[qt][blk][T]);
      }
#if CFA_TA_SGB
  // software pipeline of the operand reads: four fragments ahead, then READS
  // reads after every pair of MFMAs
  __builtin_amdgcn_sched_group_barrier(0x0100, 8, 0);
#pragma unroll
  for (int j = 0; j < Geo<D, QT>::kMfma / 2; ++j) {
    __builtin_amdgcn_sched_group_barrier(0x0008, 2, 0);
    __builtin_amdgcn_sched_group_barrier(0x0100, READS, 0);
  }
#endif
}

}  // namespace tree
}  // namespace cfa
