// scored_attention.hpp -- attention over the paged cache whose scores are
// capped by a tanh, biased by distance or cut by a sliding window: draft trees
// and single tokens (cfa_tree_attention_scored), and chunks of prompts
// (cfa_prompt_attention).
//
// For a query at position p and a key at position k that its mask leaves:
//   s = scale q.k;  s = cap tanh(s / cap);  s -= slope_h (p - k)
//   visible only while p - k < window
//   out = sum exp(s) v / sum exp(s)          (a row without keys: zeros)
// A tree node's position is ctx + its depth, its visible keys the context and
// its ancestors; token i of a prompt's chunk stands at ctx + i and sees every
// key up to itself.
//
// The tiles, rings, transposed products and phases are those of
// tree_attention.hip (tree_tiles.hpp): one work-group takes up to 256 query
// rows (the G = Hq / Hkv heads of a KV head times 256 / G tokens; 128 or 64 rows
// where those would leave CUs idle) over a split of the keys; its waves keep Q^T in
// registers while 64-key tiles of K and V stream through LDS, and each lane owns one
// query column.  What differs:
//  * Q stays as it is and the scale is applied to the products in fp32 (one
//    fma a score, with the base): a pre-scaled Q would be rounded once more.
//  * tanh.  While every |s / cap| of a wave's tile is below 1/2, tanh(t) / t is
//    a polynomial of degree 3 in t^2 (least maximum relative error on that
//    range, 5.4e-7): it keeps small scores exact under a large cap, where 1 -
//    2 / (1 + e^2t) cancels, and with its coefficients in the products' units it
//    is five fp32 operations, against two transcendental ones (16 cycles each)
//    and three others.  Tiles beyond that take the exponential form (a prompt of
//    8192, cap 50: 553 us with scores of deviation 2, 581 with 7, 596 with 12 and
//    more, where every tile does; in fp16 648, 737, 763).
//  * Capped scores without a bias lie in [-cap, cap], so bf16 probabilities
//    need no running maximum while 2^(cap log2 e) times a sum of values stays
//    in fp32's range (kFixedCap): P = exp2(s), no maxima, no rescaling.  Others
//    keep the lazy base of tree_attention.hip.  P's rounding to the element
//    type (the second product's operand) is the only one before the output's: the
//    matrix instruction takes both operands in one type, and the row's sum is of
//    the rounded values.  2-norm of the error against 64 bits in bf16: 0.0017 for
//    the output's rounding alone, 0.0018 with P's under a base (the largest is then
//    exact), 0.0022 without one.
//  * Keys in front of the window's first are not read: a tile's transfers are
//    clamped to the first visible position of its rows (their pages may be
//    gone or reused), and whole tiles in front of it are skipped.
//  * Splits are cut on the device, from each block's own first and last tile,
//    and leave fp32 sums for a log-sum-exp merge.
//
// Bound: prompts by the matrix products and the scores' vector work beside them
// (8192 tokens, 32 heads of 128 over 8: 485 us, 1134 TFLOP/s, matrix and vector units
// each busy 54% of the cycles, in phases of two waves a SIMD; capped at 50 553, 46 and
// 62%; biased 547; both 726, 34 and 61%, with 1.9 times the plain one's vector
// instructions, and 847 where every tile takes the exponential form; a window of 1024
// 156: four rounds of work-groups of 18 tiles at 1.6 us, and 6.8 each in front of the
// first tile and for the output); single tokens by HBM (64 sequences to 4096 keys,
// capped: 125 us, 5.4 TB/s); trees by both (16 of 63 nodes behind 4096, capped: 98 us
// with the merge, 690 TFLOP/s, 3 TB/s); small calls by latency (about 4.5 us in front
// of the first tile, 0.8 to 1.6 a tile, 1.5 for the output, 4 for a merge).
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "abi_internal.hpp"
#include "tree_tiles.hpp"

namespace cfa {
namespace scored {

using namespace cfa::tree;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// tanh(t) / t = kT0 + kT1 t^2 + kT2 t^4 + kT3 t^6 for |t| <= kTanhSmall
constexpr float kTanhSmall = 0.5f;
constexpr float kT0 = 0.9999994557706551f, kT1 = -0.3332631793391637f, kT2 = 0.13190296581701041f,
                kT3 = -0.04440222555554884f;
// cap log2(e) up to which exp2 needs no base: sums of 2^24 keys times values
// of 2^20 stay below 2^127, and 2^-80 is a normal bf16
constexpr float kFixedCap = 80.0f;
constexpr int kPeekSteps = 4;  // tiles of a split from which the last one is seen first

struct Args {
  const uint16_t *q;      // [rows of tokens, Hq, D]
  const uint16_t *kpool;  // [blocks, layers, Hkv, bs, D]
  const uint16_t *vpool;
  const int32_t *bt;      // [B, max_blocks]
  const int32_t *ctx;     // [B]
  const uint64_t *mask;   // trees: [N] or [B, N]; null: prompts
  long long mask_sb;
  const int32_t *cu;      // prompts: [B + 1]
  const float *slopes;    // [Hq] or null
  uint16_t *out;          // [tokens, Hq, D]
  float *part_o;          // [S, tokens, Hq, D] unnormalised sums
  float2 *part_ml;        // [S, tokens, Hq] (exponent base in log2 units, sum)
  int T, B, N, q0, Nq;    // tokens in all; trees: nodes, first query node, queries
  int Hq, Hkv, G, TQ;     // TQ: tokens per block
  int max_blocks, num_blocks, num_layers, layer, bs;
  int splits, window;
  int past;               // partials are stored past the caches
  float scale, cap;       // scale as given, or with a cap scale / cap
  // with a cap: its score in log2 units is x (k0 + k1 x^2 + k2 x^4 + k3 x^6) for
  // a product |x| <= small
  float k0, k1, k2, k3, small;
};

// The block of query tokens of a work-group.
struct Block {
  int b, t0, nt, i0;  // sequence, first token (global), tokens, the first's index in it
  int ctx;            // as given
};

// Inclusive sum over the wave's lanes, within the vector registers.
__device__ __forceinline__ int lane_scan(int v) {
#define CFA_SCAN_STEP(ctrl, rows) v += __builtin_amdgcn_update_dpp(0, v, ctrl, rows, 0xf, false);
  CFA_SCAN_STEP(0x111, 0xf)  // from 1, 2, 4 and 8 lanes in front, in rows of 16
  CFA_SCAN_STEP(0x112, 0xf)
  CFA_SCAN_STEP(0x114, 0xf)
  CFA_SCAN_STEP(0x118, 0xf)
  CFA_SCAN_STEP(0x142, 0xa)  // lane 15 to the next row
  CFA_SCAN_STEP(0x143, 0xc)  // lane 31 to the upper half
#undef CFA_SCAN_STEP
  return v;
}

// Trees: block = sequence * ceil(Nq / TQ) + part, with the sequences in the order
// of falling length where one wave can rank them: the work-groups that start
// last are then the short ones (64 single tokens over 1024 to 4096 keys, 126 us
// against 172 in the batch's order).  Prompts: the blocks of all
// sequences are numbered through, each sequence's last (longest) one first.
__device__ __forceinline__ bool find_block(const Args &a, int id, int lane, Block &k) {
  if (a.mask) {
    const int per = (a.Nq + a.TQ - 1) / a.TQ;
    k.b = id / per;
    if (a.B > 1 && a.B <= 64) {
      const int mine = lane < a.B ? a.ctx[lane] : 0;
      int rank = 0;
      for (int j = 0; j < a.B; ++j) {
        const int c = __builtin_amdgcn_readlane(mine, j);
        rank += c > mine || (c == mine && j < lane);
      }
      k.b = __ffsll((unsigned long long)__ballot(lane < a.B && rank == k.b)) - 1;
      k.ctx = __builtin_amdgcn_readlane(mine, k.b);
    } else {
      k.ctx = a.ctx[k.b];
    }
    k.i0 = (id % per) * a.TQ;
    k.t0 = k.b * a.Nq + k.i0;
    k.nt = min(a.TQ, a.Nq - k.i0);
    return true;
  }
  int before = 0;  // blocks of the sequences in front of this round's
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int b = b0 + lane;
    int len = 0, at = 0, ctx = 0;
    if (b < a.B) {
      at = a.cu[b];
      ctx = a.ctx[b];
      // (an end behind the tokens there are, or in front of the start, is cut)
      len = at < 0 ? 0 : max(min(a.cu[b + 1], a.T) - at, 0);
    }
    const int n = (len + a.TQ - 1) / a.TQ;
    const int upto = lane_scan(n);
    const uint64_t hit = __ballot(before + upto > id);
    if (hit) {
      const int w = __ffsll((unsigned long long)hit) - 1;
      const int nb = __builtin_amdgcn_readlane(n, w);
      const int r = id - before - __builtin_amdgcn_readlane(upto, w) + nb;  // among its blocks
      k.b = b0 + w;
      k.i0 = (nb - 1 - r) * a.TQ;
      k.t0 = __builtin_amdgcn_readlane(at, w) + k.i0;
      k.nt = min(a.TQ, __builtin_amdgcn_readlane(len, w) - k.i0);
      k.ctx = __builtin_amdgcn_readlane(ctx, w);
      return true;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// What a query row's scores need besides its Q, in LDS: registers held across
// the MFMA phase are what its operand reads are scheduled ahead with (four more,
// and the compiler drops that schedule: 692 against 519 us for the plain prompt).
struct Row {
  uint64_t anc;   // trees: visible nodes (ancestors inside the window); prompts:
                  // the keys up to the row's own, of those that the table covers
  int pos;        // position
  int first;      // first visible position (window), else 0
  float slope2;   // distance bias: slope * log2(e)
};

template <int D, int QT, class T, bool CAP, bool BIAS, bool FIXED>
__device__ __forceinline__ void raw_scores(const Lane<D, QT, T> &ln, const float (&base_of)[QT],
                                           const Args &a, float k0, float cap2, int kbase, int ctx,
                                           int least, int most_first, const Row *rows,
                                           const float *move, Scores<QT> &S) {
  const bool tree = a.mask != nullptr;
  // tanh: the polynomial while the whole wave's tile is small
  bool small = true;
  if constexpr (CAP) {
    float m = 0.0f;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
#pragma unroll
      for (int blk = 0; blk < 2; ++blk)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) m = fmaxf(m, fabsf(S.s[qt][blk][t][i]));
    // (NaN, lost by fmaxf, stays NaN in either form)
    small = __ballot(m > a.small) == 0;
  }
  // f(score, what to add to it): every score of the tile.  (The choice of form
  // stays outside: as a condition inside the loops it became a branch a score,
  // 964 us against 567 for the capped prompt of 8192.)
  auto every = [&](auto f) {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      float base = FIXED ? 0.0f : -base_of[qt], slope = 0.0f;
      if constexpr (BIAS) {  // of the lane's first key; exact until rounded once
        slope = rows[qt * 16].slope2;
        base += slope * (float)(kbase + 8 * ln.g - rows[qt * 16].pos);
      }
#pragma unroll
      for (int blk = 0; blk < 2; ++blk)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            S.s[qt][blk][t][i] =
                f(S.s[qt][blk][t][i],
                  BIAS ? fmaf(slope, (float)(blk * 32 + 4 * t + i), base) : base);
    }
  };
  if constexpr (!CAP) {
    every([&](float x, float add) { return fmaf(x, k0, add); });
  } else if (small) {
    every([&](float x, float add) {
      const float w = x * x;
      float p = fmaf(w, a.k3, a.k2);
      p = fmaf(w, p, a.k1);
      p = fmaf(w, p, a.k0);
      return FIXED ? x * p : fmaf(x, p, add);
    });
  } else {
    every([&](float x, float add) {
      const float r = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * k0));
      return fmaf(r, -2.0f * cap2, FIXED ? cap2 : cap2 + add);
    });
  }
  if (BIAS && tree && kbase + kKT > ctx) {
    // a tree key stands at ctx + its depth, not at its slot
    const float *mv = move + (kbase + 8 * ln.g - ctx);
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float by = mv[blk * 32 + 4 * t + i];
#pragma unroll
          for (int qt = 0; qt < QT; ++qt)
            S.s[qt][blk][t][i] = fmaf(rows[qt * 16].slope2, by, S.s[qt][blk][t][i]);
        }
  }
  if (kbase + kKT > least || kbase < most_first) {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      // bit k: tile key k is visible to this column
      const Row r = rows[qt * 16];
      uint64_t vis;
      if (tree) {
        vis = tile_visibility(kbase, ctx, r.anc);
      } else {
        const int n = (int)r.anc - kbase;
        vis = n >= 64 ? ~0ull : (n <= 0 ? 0ull : ((1ull << n) - 1));
      }
      const int cut = min(r.first, tree ? ctx : r.first) - kbase;  // keys in front
      if (cut > 0) vis = cut >= 64 ? 0ull : vis >> cut << cut;
      vis >>= 8 * ln.g;
#pragma unroll
      for (int blk = 0; blk < 2; ++blk)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            S.s[qt][blk][t][i] =
                ((vis >> (blk * 32 + 4 * t + i)) & 1ull) ? S.s[qt][blk][t][i] : -INFINITY;
    }
  }
}

template <int QT>
__device__ __forceinline__ float score_max(const Scores<QT> &S, int qt) {
  float v = -INFINITY;
#pragma unroll
  for (int blk = 0; blk < 2; ++blk)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) v = fmaxf(v, S.s[qt][blk][t][i]);
  return column_max(v);
}

// Scores of one tile to probabilities; the columns' lazy bases b (log2 units; 0:
// none yet, where the sum is 0 too) where FIXED does not hold.
template <int D, int QT, class T, bool FIXED>
__device__ __forceinline__ void score_phase(Scores<QT> &S, float (&b)[QT], f32x4 (&o)[QT][D / 16],
                                            f32x4 (&lacc)[QT], Probs<QT, T> &P) {
  if constexpr (!FIXED) {
    float mx[QT];
    bool any = false;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      mx[qt] = score_max(S, qt);
      const bool unset = b[qt] == 0.0f && lacc[qt][0] == 0.0f && mx[qt] > -INFINITY;
      mx[qt] = mx[qt] > kRescaleSlack || unset ? mx[qt] : 0.0f;  // what the base moves by
      any |= mx[qt] != 0.0f;
    }
    if (__ballot(any) != 0) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        // (a base falls only while the sums are still 0)
        const float alpha = __builtin_amdgcn_exp2f(-fmaxf(mx[qt], 0.0f));
        b[qt] += mx[qt];
        lacc[qt] *= alpha;
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) o[qt][dt] *= alpha;
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
          for (int t = 0; t < 2; ++t) S.s[qt][blk][t] -= mx[qt];
      }
    }
  }
#pragma unroll
  for (int qt = 0; qt < QT; ++qt)
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          P.p[qt][blk][t * 4 + i] =
              (typename T::elem)__builtin_amdgcn_exp2f(S.s[qt][blk][t][i]);
      // keep the exponentials in this phase (see tree_attention.hip)
      asm volatile("" ::"v"(P.p[qt][blk]));
    }
}

template <int D, int QT, class T, bool CAP, bool BIAS, bool FIXED>
__global__ __launch_bounds__(kNT) void scored_attn_kernel(Args a) {
  using Gm = Geo<D>;
  constexpr int kTileBytes = Gm::kTileBytes;
  constexpr int kLoadsPerTile = Gm::kLoadsPerTile;
  __shared__ __align__(16) uint8_t kring[kKStages * kTileBytes];
  __shared__ __align__(16) uint8_t vring[kVStages * kTileBytes];
  // row offsets of the split's 16-key groups; a ring, refilled half a ring at a
  // time in longer splits (its size, and the rows', let two work-groups of one
  // query tile and head_dim 64 share a CU's LDS)
  constexpr int kRing = D == 64 ? 512 : 1024;
  __shared__ long long gtab[kRing];
  __shared__ long long gpeek[kKT / 16];
  // trees: how far node j's position lies from its slot, at 64 + j; 0 around them
  __shared__ float smove[192];
  __shared__ Row srow[QT == 1 ? kMaxRows / 2 : kMaxRows];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, g = lane >> 4;
  const int split = blockIdx.x % a.splits, rest = blockIdx.x / a.splits;
  const int h = rest % a.Hkv;
  Block blk;
  if (!__builtin_amdgcn_readfirstlane(find_block(a, rest / a.Hkv, lane, blk))) return;
  // (the same in every lane; told to the compiler, since everything that steers
  // the loop and its transfers follows from them)
  blk.b = __builtin_amdgcn_readfirstlane(blk.b);
  blk.t0 = __builtin_amdgcn_readfirstlane(blk.t0);
  blk.nt = __builtin_amdgcn_readfirstlane(blk.nt);
  blk.i0 = __builtin_amdgcn_readfirstlane(blk.i0);
  blk.ctx = __builtin_amdgcn_readfirstlane(blk.ctx);
  const int b = blk.b, rows = blk.nt * a.G;
  const bool tree = a.mask != nullptr;

  // positions past the block table are never read: a tree's context is cut to
  // leave room for its nodes, a prompt's keys end with the table
  const int cap_keys = a.max_blocks * a.bs;
  const int last = tree ? a.N : blk.i0 + blk.nt;  // keys behind the context
  const int ctx = min(max(blk.ctx, 0), tree ? max(cap_keys - last, 0) : 0x7fffffff - last);
  int nkeys = min(ctx + last, cap_keys);  // trees: cut behind the last visible node

  Lane<D, QT, T> ln;
  float base[QT];  // exponent bases
  Row row[QT];
  bool qvalid[QT];
  ln.g = g;
  int low;  // the first query's position (trees: the shallowest's)
  if (tree) {
    const uint64_t nodes = a.N >= 64 ? ~0ull : ((1ull << a.N) - 1);
    uint64_t mine = lane < a.N ? a.mask[(long long)b * a.mask_sb + lane] & nodes : 0ull;
    const int depth = max((int)__popcll(mine) - 1, 0);
    if (BIAS && wave < 3) {
      const int node = lane + 64 * (wave - 1);  // wave 1 holds the nodes
      smove[64 + node] = node >= 0 && node < a.N ? (float)(depth - node) : 0.0f;
    }
    const int j = a.q0 + blk.i0;
    if (a.window > 0)  // nodes that lie `window` and more above are out of it
      for (int m = 0; m < a.N; ++m)
        if (depth - __builtin_amdgcn_readlane(depth, m) >= a.window) mine &= ~(1ull << m);
    const bool asks = lane >= j && lane < j + blk.nt;
    int d = asks ? depth : 64, behind = asks && mine ? 64 - __clzll((long long)mine) : 0;
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) {
      d = min(d, __shfl_xor(d, s, 64));
      behind = max(behind, __shfl_xor(behind, s, 64));
    }
    low = ctx + __builtin_amdgcn_readfirstlane(d);
    nkeys = ctx + __builtin_amdgcn_readfirstlane(behind);
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int r = (wave * QT + qt) * 16 + col;
      qvalid[qt] = r < rows;
      const int node = j + (qvalid[qt] ? r / a.G : 0);
      const uint64_t anc = __shfl((unsigned long long)mine, node, 64);
      row[qt].pos = ctx + __shfl(depth, node, 64);
      row[qt].anc = qvalid[qt] ? anc : 0ull;
    }
  } else {
    low = ctx + blk.i0;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int r = (wave * QT + qt) * 16 + col;
      qvalid[qt] = r < rows;
      row[qt].pos = low + (qvalid[qt] ? r / a.G : 0);
      row[qt].anc = min(row[qt].pos + 1, nkeys);
    }
  }
  const int high = tree ? ctx + 63 : low + blk.nt - 1;  // no query stands behind it
  // the first position that any row sees, and the last first one
  const int from = a.window > 0 ? min(max(low - a.window + 1, 0), tree ? ctx : nkeys - 1) : 0;
  const int most_first = a.window > 0 ? max(high - a.window + 1, 0) : 0;
  // keys below it are visible to all (but the window)
  const int least = tree ? ctx : min(low + 1, nkeys);
  const int tlo = from / kKT, thi = (nkeys + kKT - 1) / kKT;
  const int tps = (thi - tlo + a.splits - 1) / a.splits;
  const int t0 = tlo + split * tps, t1 = min(thi, t0 + tps);
  const int steps = from < nkeys ? t1 - t0 : 0;
  constexpr float kLog2e = 1.4426950408889634f;
  const float cap2 = a.cap * kLog2e;
  // without a cap: score in log2 units = product * k0; with one: e^(2 s / cap)
  // = exp2(product * k0)
  const float k0 = (CAP ? 2.0f : 1.0f) * a.scale * kLog2e;

#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int r = (wave * QT + qt) * 16 + col;
    const int nl = qvalid[qt] ? r / a.G : 0, hg = qvalid[qt] ? r % a.G : 0;
    const int head = h * a.G + hg;
    row[qt].first = a.window > 0 ? max(row[qt].pos - a.window + 1, 0) : 0;
    row[qt].slope2 = BIAS ? a.slopes[head] * kLog2e : 0.0f;
    if (g == 0) srow[r] = row[qt];
    base[qt] = 0.0f;
    const uint16_t *qp = a.q + (((long long)blk.t0 + nl) * a.Hq + head) * D;
#pragma unroll
    for (int kk = 0; kk < D / 32; ++kk) {
      const uint4 v = qvalid[qt] ? ld_g16(qp + kk * 32 + g * 8) : make_uint4(0, 0, 0, 0);
      ln.qf[qt][kk] = __builtin_bit_cast(typename Mfma<T>::frag, v);
    }
  }
#pragma unroll
  for (int kk = 0; kk < D / 32; ++kk)
    ln.koff[kk] = col * Gm::kRowBytes + (((kk * 4 + g) ^ k_swz<D>(col)) << 4);
  {
    const int vrow = 8 * g + (col >> 2);
    ln.vh = v_swz<D>(vrow) >> 1;
    ln.vbase = vrow * Gm::kRowBytes + ((col >> 1) & 1) * 16 + (col & 1) * 8;
  }

  const DmaOffs<D> doff = dma_offsets<D>(wave, lane);
  auto issue_from = [&](const long long *tab, int u, uint8_t *kdst, uint8_t *vdst) {
    const int kbase = (t0 + u) * kKT;
    const long long *kt = tab + 2 * (wave >> 2) + (wave & 1);
    const long long *vt = tab + (wave >> 1);
    if (kbase + kKT <= nkeys && kbase >= from)
      issue_tile_full<D>(a, kt, vt, doff, kdst, vdst, wave);
    else
      issue_tile<D, true>(a, kt, vt, kbase, nkeys, kdst, vdst, wave, lane, from);
  };
  auto issue = [&](int u, uint8_t *kdst, uint8_t *vdst) {
    issue_from(gtab + u * (kKT / 16) % kRing, u, kdst, vdst);
  };
  const int32_t *btb = a.bt + (long long)b * a.max_blocks;
  constexpr int kPerTile = kKT / 16;
  const int ng = steps * kPerTile;
  auto look_up = [&](int first, int n) {
    for (int i = first + tid; i < min(first + n, ng); i += kNT) {
      gtab[i % kRing] =
          group_row_offset<D, true>(a, btb, t0 * kPerTile + i, nkeys, h, from);
    }
  };
  look_up(0, kRing);
  // Under a distance bias the last tile's keys, the nearest, set the exponent
  // bases before the first tile: from far to near, steep slopes would rescale
  // the outputs at every tile (the biased prompt of 8192 693 us against 546).
  const bool peek = BIAS && steps >= kPeekSteps;
  if (BIAS && tid < kPerTile)
    gpeek[tid] = group_row_offset<D, true>(a, btb, (t1 - 1) * kPerTile + tid, nkeys, h, from);
  wait_vmcnt<0>();
  __syncthreads();

  f32x4 o[QT][D / 16];
  f32x4 lacc[QT];
  const Row *const rows_at = srow + wave * QT * 16 + col;
  float zero[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    zero[qt] = 0.0f;
    lacc[qt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) o[qt][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  if (steps > 0) {
    // the phases and barriers of tree_attention.hip's loop
    // (the last K stage and V stage are free until the loop)
    if (peek)
      issue_from(gpeek, steps - 1, kring + (kKStages - 1) * kTileBytes,
                 vring + (kVStages - 1) * kTileBytes);
    for (int u = 0; u < min(3, steps); ++u)
      issue(u, kring + (u % kKStages) * kTileBytes, vring + (u % kVStages) * kTileBytes);
    Scores<QT> S;
    const bool busy = wave * QT * 16 < rows;  // wave-uniform
    if constexpr (BIAS) {
      if (peek) {
        wait_vmcnt<3 * kLoadsPerTile>();
        block_barrier();
        if (busy) {
          qk_tile(ln, kring + (kKStages - 1) * kTileBytes, zero, S);
          raw_scores<D, QT, T, CAP, BIAS, FIXED>(ln, base, a, k0, cap2, (t1 - 1) * kKT, ctx, least,
                                                 most_first, rows_at, smove + 64, S);
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) {
            const float m = score_max(S, qt);
            base[qt] = m > -INFINITY ? m : 0.0f;
          }
        }
        block_barrier();
      }
    }
    const int later = min(3, steps) - 1;
    if (later >= 2) wait_vmcnt<2 * kLoadsPerTile>();
    else if (later == 1) wait_vmcnt<kLoadsPerTile>();
    else wait_vmcnt<0>();
    block_barrier();
    const bool lag = wave >= kWaves / 2;
    if (lag) block_barrier();
    Probs<QT, T> P;
    if (busy) qk_tile(ln, kring, zero, S);
    for (int u = 0; u < steps; ++u) {
      const int kbase = (t0 + u) * kKT;
      const int ahead = u + 3;
      // (both halves' groups were in use until now: the one in front of this step
      // has no readers left, and its new entries have them half a ring on)
      if (u > 0 && u % (kRing / kPerTile / 2) == 0) {
        look_up(u * kPerTile + kRing / 2, kRing / 2);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
      if (!lag) {
        block_barrier();
      } else {
        if (u + 2 < steps) wait_vmcnt<kLoadsPerTile>();
        else wait_vmcnt<0>();
        block_barrier();
      }
      if (ahead < steps)
        issue(ahead, kring + (ahead % kKStages) * kTileBytes,
              vring + (ahead % kVStages) * kTileBytes);
      if (busy) {
        raw_scores<D, QT, T, CAP, BIAS, FIXED>(ln, base, a, k0, cap2, kbase, ctx, least, most_first,
                                               rows_at, smove + 64, S);
        score_phase<D, QT, T, FIXED>(S, base, o, lacc, P);
      }
      if (!lag) {
        if (ahead < steps) wait_vmcnt<2 * kLoadsPerTile>();
        else if (u + 2 < steps) wait_vmcnt<kLoadsPerTile>();
        else wait_vmcnt<0>();
        block_barrier();
      } else {
        block_barrier();
      }
      __builtin_amdgcn_s_setprio(1);
      if (busy)
        // (one query tile has half the products per operand read)
        mfma_phase<D, QT, T, QT == 1 ? 4 : 2>(ln, kring + ((u + 1) % kKStages) * kTileBytes,
                   vring + (u % kVStages) * kTileBytes, zero, P, S, o, lacc);
      __builtin_amdgcn_s_setprio(0);
    }
    if (!lag) block_barrier();
  }

  // Results pass the caches, since what these hold dirty at a kernel's end delays the
  // next (32 prompts of 256 tokens 72.0 -> 64.5 us, one of 8192 494 -> 492); partials
  // only up to 24 MB (one tree of 63 nodes, 16 MB: 30.4 -> 27.3), since the merge finds
  // part of more in them (256 tokens behind 8000, 34 MB: 50.8 -> 52.6).
  if (a.splits == 1) {
    // through LDS (the K ring's, once every wave is done with it), so that whole rows
    // are stored, 16 bytes a lane; 16-byte chunk c of row r lies at c ^ r % (D / 8)
    constexpr int kChunks = D / 8;
    __syncthreads();
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int r0 = (wave * QT + qt) * 16;
      uint8_t *const tile = kring + r0 * D * 2;
      const float ls = lacc[qt][0], inv = ls != 0.0f ? 1.0f / ls : 0.0f;
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) {
        uint2 w;
        w.x = pack2<T>(o[qt][dt][0] * inv, o[qt][dt][1] * inv);
        w.y = pack2<T>(o[qt][dt][2] * inv, o[qt][dt][3] * inv);
        const int c = (dt * 2 + (g >> 1)) ^ (col % kChunks);
        *reinterpret_cast<uint2 *>(tile + col * D * 2 + c * 16 + (g & 1) * 8) = w;
      }
#pragma unroll
      for (int i = 0; i < kChunks / 4; ++i) {
        const int x = i * 64 + lane, rr = x / kChunks, c = x % kChunks, r = r0 + rr;
        const u32x4 v = *reinterpret_cast<const u32x4 *>(
            tile + rr * D * 2 + ((c ^ (rr % kChunks)) << 4));
        const long long orow = ((long long)blk.t0 + r / a.G) * a.Hq + (long long)h * a.G + r % a.G;
        if (r < rows)
          __builtin_nontemporal_store(v, reinterpret_cast<u32x4 *>(a.out + orow * D + c * 8));
      }
    }
    return;
  }
  auto put = [&](f32x4 *at, f32x4 v) {
    // (the empty asm keep the compiler from joining the two into a plain store)
    if (a.past) {
      asm volatile("");
      __builtin_nontemporal_store(v, at);
    } else {
      *at = v;
      asm volatile("");
    }
  };
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const float ls = lacc[qt][0];
    if (!qvalid[qt]) continue;
    const int r = (wave * QT + qt) * 16 + col;
    const long long orow = ((long long)blk.t0 + r / a.G) * a.Hq + (long long)h * a.G + r % a.G;
    const long long prow = (long long)split * a.T * a.Hq + orow;
    float *pp = a.part_o + prow * D;
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt)
      put(reinterpret_cast<f32x4 *>(pp + dt * 16 + 4 * g), o[qt][dt]);
    if (g == 0) a.part_ml[prow] = make_float2(ls != 0.0f ? base[qt] : -INFINITY, ls);
  }
}

// Log-sum-exp merge of the splits: out = sum_s w_s o_s / sum_s w_s l_s with
// w_s = 2^(b_s - max b); four values a thread, D / 4 threads a row.  Rows of
// tokens that belong to no prompt are left alone.  Every value is touched once, so
// loads and stores pass the caches (16 trees of 63 nodes, two splits: the whole call
// 102 -> 97 us).
// REGS: splits whose loads are issued in one round, 4 for up to 4 splits, else 8 (16
// trees of 63 nodes, two splits: in kernel traces 8.8 us with 4 and 10.9 with 8; by
// itself, launched over and over, 10.2 with 2 or 4, 12.3 with 8, 17 with 16; one
// token behind 8000, 32 splits: 14.3, 11.0, 9.6, 9.6 with 2, 4, 8 and 16).
template <int D, class T, int REGS>
__global__ __launch_bounds__(256) void scored_merge_kernel(Args a) {
  constexpr int kTPR = D / 4;
  const long long row = (long long)blockIdx.x * (256 / kTPR) + threadIdx.x / kTPR;
  const int e = (threadIdx.x % kTPR) * 4;
  const long long rows = (long long)a.T * a.Hq;
  if (row >= rows) return;
  if (a.cu) {
    const long long t = row / a.Hq;
    if (t < a.cu[0] || t >= a.cu[a.B]) return;
  }
  float M = -INFINITY, L = 0.0f;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s0 = 0; s0 < a.splits; s0 += REGS) {
    float2 ml[REGS];
    f32x4 v[REGS];
#pragma unroll
    for (int s = 0; s < REGS; ++s) {
      if (s0 + s < a.splits) {
        const long long p = (long long)(s0 + s) * rows + row;
        ml[s] = a.part_ml[p];
        v[s] = __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>(a.part_o + p * D + e));
      }
    }
    float m = M;
#pragma unroll
    for (int s = 0; s < REGS; ++s)
      if (s0 + s < a.splits) m = fmaxf(m, ml[s].x);
    const float base = m == -INFINITY ? 0.0f : m;
    const float w0 = __builtin_amdgcn_exp2f(M - base);
    L *= w0;
    acc *= w0;
#pragma unroll
    for (int s = 0; s < REGS; ++s)
      if (s0 + s < a.splits) {
        const float w = __builtin_amdgcn_exp2f(ml[s].x - base);
        L += w * ml[s].y;
        acc += w * v[s];
      }
    M = m;
  }
  const float inv = L != 0.0f ? 1.0f / L : 0.0f;
  uint2 w;
  w.x = pack2<T>(acc[0] * inv, acc[1] * inv);
  w.y = pack2<T>(acc[2] * inv, acc[3] * inv);
  __builtin_nontemporal_store(u32x2{w.x, w.y}, reinterpret_cast<u32x2 *>(a.out + row * D + e));
}

template <int D, int QT, class T>
int launch_scores(const Args &a, unsigned grid, hipStream_t st) {
  const bool cap = a.cap > 0.0f, bias = a.slopes != nullptr;
  const bool fixed = cap && !bias && std::is_same<T, BF16>::value &&
                     a.cap * 1.4426950408889634f <= kFixedCap;
#define CFA_SCORED(C, B, F)                                                                  \
  CFA_LAUNCH("scored_attn", (scored_attn_kernel<D, QT, T, C, B, F>), dim3(grid), dim3(kNT), 0, \
             st, a)
  if (cap && bias) CFA_SCORED(true, true, false);
  else if (fixed) {
    if constexpr (std::is_same<T, BF16>::value) CFA_SCORED(true, false, true);
  } else if (cap) CFA_SCORED(true, false, false);
  else if (bias) CFA_SCORED(false, true, false);
  else CFA_SCORED(false, false, false);
#undef CFA_SCORED
  return CFA_OK;
}

template <int D, class T>
int launch(const Args &a, bool one, unsigned grid, hipStream_t st) {
  const int rc = one ? launch_scores<D, 1, T>(a, grid, st) : launch_scores<D, 2, T>(a, grid, st);
  if (rc != CFA_OK || a.splits == 1) return rc;
  const long long rows = (long long)a.T * a.Hq;
  const int per = 256 / (D / 4);
  const dim3 merges((unsigned)((rows + per - 1) / per));
  if (a.splits <= 4)
    CFA_LAUNCH("scored_merge", (scored_merge_kernel<D, T, 4>), merges, dim3(256), 0, st, a);
  else
    CFA_LAUNCH("scored_merge", (scored_merge_kernel<D, T, 8>), merges, dim3(256), 0, st, a);
  return CFA_OK;
}

}  // namespace scored
}  // namespace cfa
