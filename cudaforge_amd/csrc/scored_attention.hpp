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
// rows (the G = Hq / Hkv heads of a KV head times 256 / G tokens) over a split
// of the keys; its waves keep Q^T in registers while 64-key tiles of K and V
// stream through LDS, and each lane owns one query column.  What differs:
//  * Q stays as it is and the scale is applied to the products in fp32 (one
//    fma a score, with the base): a pre-scaled Q would be rounded once more.
//  * tanh.  While every |s / cap| of a wave's tile is below 3/4, tanh(t) / t is
//    a polynomial of degree 4 in t^2 (least maximum relative error on that
//    range, 5.7e-7): it keeps small scores exact under a large cap, where 1 -
//    2 / (1 + e^2t) cancels, and is six fp32 operations against two
//    transcendental ones (16 cycles each) and three others.  Tiles beyond that
//    take the exponential form.
//  * Capped scores without a bias lie in [-cap, cap], so bf16 probabilities
//    need no running maximum while 2^(cap log2 e) times a sum of values stays
//    in fp32's range (kFixedCap): P = exp2(s), no maxima, no rescaling.  Others
//    keep the lazy base of tree_attention.hip.  P's rounding to the element
//    type (the second product's operand) is the only one before the output's.
//  * Keys in front of the window's first are not read: a tile's transfers are
//    clamped to the first visible position of its rows (their pages may be
//    gone or reused), and whole tiles in front of it are skipped.
//  * Splits are cut on the device, from each block's own first and last tile,
//    and leave fp32 sums for a log-sum-exp merge.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "abi_internal.hpp"
#include "tree_tiles.hpp"

namespace cfa {
namespace scored {

using namespace cfa::tree;

// tanh(t) / t = kT0 + kT1 t^2 + ... + kT4 t^8 for |t| <= kTanhSmall
constexpr float kTanhSmall = 0.75f;
constexpr float kT0 = 0.9999994349232844f, kT1 = -0.3332825152895064f, kT2 = 0.13258983189591972f,
                kT3 = -0.05005630179239906f, kT4 = 0.012929631620462257f;
// cap log2(e) up to which exp2 needs no base: sums of 2^24 keys times values
// of 2^20 stay below 2^127, and 2^-80 is a normal bf16
constexpr float kFixedCap = 80.0f;

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
  int blocks;             // blocks launched (trees: B * ceil(Nq / TQ))
  int max_blocks, num_blocks, num_layers, layer, bs;
  int splits, window;
  float scale, cap;       // scale as given, or with a cap scale / cap
};

// The block of query tokens of a work-group.
struct Block {
  int b, t0, nt, i0;  // sequence, first token (global), tokens, the first's index in it
};

// Trees: block = sequence * ceil(Nq / TQ) + part.  Prompts: the blocks of all
// sequences are numbered through, each sequence's last (longest) one first.
__device__ __forceinline__ bool find_block(const Args &a, int id, int lane, Block &k) {
  if (a.mask) {
    const int per = (a.Nq + a.TQ - 1) / a.TQ;
    k.b = id / per;
    k.i0 = (id % per) * a.TQ;
    k.t0 = k.b * a.Nq + k.i0;
    k.nt = min(a.TQ, a.Nq - k.i0);
    return true;
  }
  int before = 0;  // blocks of the sequences in front of this round's
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int b = b0 + lane;
    int len = 0, at = 0;
    if (b < a.B) {
      at = a.cu[b];
      // (an end behind the tokens there are, or in front of the start, is cut)
      len = at < 0 ? 0 : max(min(a.cu[b + 1], a.T) - at, 0);
    }
    const int n = (len + a.TQ - 1) / a.TQ;
    int upto = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(upto, o, 64);
      if (lane >= o) upto += v;
    }
    const uint64_t hit = __ballot(before + upto > id);
    if (hit) {
      const int w = __ffsll((unsigned long long)hit) - 1;
      const int r = id - before - __shfl(upto - n, w, 64);  // place among its blocks
      const int wl = __shfl(len, w, 64), nb = __shfl(n, w, 64);
      k.b = b0 + w;
      k.i0 = (nb - 1 - r) * a.TQ;
      k.t0 = __shfl(at, w, 64) + k.i0;
      k.nt = min(a.TQ, wl - k.i0);
      return true;
    }
    before += __shfl(upto, 63, 64);
  }
  return false;
}

// What a lane knows of its query column besides Q.
struct Column {
  uint64_t anc;  // trees: visible nodes (ancestors inside the window)
  int pos;       // position
  int first;     // first visible position (window), else 0
  float slope2;  // slope * log2(e)
};

// Scores of one tile in log2 units less the base (S in: raw products), masked,
// to probabilities; the lazy maximum where kFixed does not hold.
template <int D, int QT, class T, bool CAP, bool BIAS, bool FIXED>
__device__ __forceinline__ void score_phase(const Lane<D, QT, T> &ln, const Column (&cl)[QT],
                                            const Args &a, float k0, float cap2, int kbase, int ctx,
                                            int least, int most_first, const int *sdepth,
                                            Scores<QT> &S, Softmax<QT> &sm,
                                            f32x4 (&o)[QT][D / 16], f32x4 (&lacc)[QT],
                                            Probs<QT, T> &P) {
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
    // a.scale = sm_scale / cap; NaN (lost by fmaxf) stays NaN in either form
    small = __ballot(m * fabsf(a.scale) > kTanhSmall) == 0;
  }
  const bool tree_keys = tree && kbase + kKT > ctx;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    float base = FIXED ? 0.0f : -sm.b[qt];
    const float slope = BIAS ? cl[qt].slope2 : 0.0f;
    if constexpr (BIAS)  // of the lane's first key; exact until rounded once
      base += slope * (float)(kbase + 8 * ln.g - cl[qt].pos);
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int off = blk * 32 + 4 * t + i;
          float add = BIAS ? fmaf(slope, (float)off, base) : base;
          const float x = S.s[qt][blk][t][i];
          if constexpr (CAP) {
            if (small) {
              const float u = x * a.scale, w = u * u;
              float p = fmaf(w, kT4, kT3);
              p = fmaf(w, p, kT2);
              p = fmaf(w, p, kT1);
              p = fmaf(w, p, kT0);
              S.s[qt][blk][t][i] = fmaf(u * cap2, p, add);
            } else {
              const float r = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * k0));
              S.s[qt][blk][t][i] = fmaf(r, -2.0f * cap2, cap2 + add);
            }
          } else {
            S.s[qt][blk][t][i] = fmaf(x, k0, add);
          }
        }
    if constexpr (BIAS) {
      if (tree_keys) {
        // a tree key's distance is the difference of the depths
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int slot = kbase + 8 * ln.g + blk * 32 + 4 * t + i;
              const int j = min(max(slot - ctx, 0), 63);
              const int moved = slot >= ctx ? ctx + sdepth[j] - slot : 0;
              S.s[qt][blk][t][i] = fmaf(slope, (float)moved, S.s[qt][blk][t][i]);
            }
      }
    }
  }
  if (kbase + kKT > least || kbase < most_first) {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      // bit k: tile key k is visible to this column
      uint64_t vis;
      if (tree) {
        vis = tile_visibility(kbase, ctx, cl[qt].anc);
      } else {
        const int n = cl[qt].pos + 1 - kbase;
        vis = n >= 64 ? ~0ull : (n <= 0 ? 0ull : ((1ull << n) - 1));
      }
      const int cut = min(cl[qt].first, tree ? ctx : cl[qt].first) - kbase;  // keys in front
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
  if constexpr (!FIXED) {
    float mx[QT];
    bool resc[QT];
    bool any = false;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      float v = -INFINITY;
#pragma unroll
      for (int blk = 0; blk < 2; ++blk)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) v = fmaxf(v, S.s[qt][blk][t][i]);
      mx[qt] = column_max(v);
      resc[qt] = mx[qt] > -INFINITY && (!sm.valid[qt] || mx[qt] > kRescaleSlack);
      any |= resc[qt];
    }
    if (__ballot(any) != 0) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        const float d = resc[qt] ? mx[qt] : 0.0f;
        const float alpha =
            resc[qt] ? (sm.valid[qt] ? __builtin_amdgcn_exp2f(-d) : 0.0f) : 1.0f;
        sm.b[qt] += d;
        sm.valid[qt] = sm.valid[qt] || resc[qt];
        lacc[qt] *= alpha;
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) o[qt][dt] *= alpha;
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
          for (int t = 0; t < 2; ++t) S.s[qt][blk][t] -= d;
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
  // row offsets of the split's 16-key groups; a ring of kMaxGroups, refilled
  // half a ring at a time in longer splits
  __shared__ long long gtab[kMaxGroups];
  __shared__ int sdepth[64];
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
  const int b = blk.b, rows = blk.nt * a.G;
  const bool tree = a.mask != nullptr;

  // positions past the block table are never read (lengths beyond the table's
  // capacity are clamped rather than trusted)
  const int cap_keys = a.max_blocks * a.bs;
  const int last = tree ? a.N : blk.i0 + blk.nt;  // keys behind the context
  const int ctx = min(max(a.ctx[b], 0), max(cap_keys - last, 0));
  const int nkeys = min(ctx + last, cap_keys);

  Lane<D, QT, T> ln;
  Column cl[QT];
  bool qvalid[QT];
  ln.g = g;
  int low;  // the first query's position (trees: the shallowest's)
  if (tree) {
    const uint64_t nodes = a.N >= 64 ? ~0ull : ((1ull << a.N) - 1);
    const uint64_t mine = lane < a.N ? a.mask[(long long)b * a.mask_sb + lane] & nodes : 0ull;
    const int depth = max((int)__popcll(mine) - 1, 0);
    if (wave == 0) sdepth[lane] = depth;
    const int j = a.q0 + blk.i0;
    int d = lane >= j && lane < j + blk.nt ? depth : 64;
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) d = min(d, __shfl_xor(d, s, 64));
    low = ctx + __builtin_amdgcn_readfirstlane(d);
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int r = (wave * QT + qt) * 16 + col;
      qvalid[qt] = r < rows;
      const int node = j + (qvalid[qt] ? r / a.G : 0);
      uint64_t anc = __shfl((unsigned long long)mine, node, 64);
      const int dq = __shfl(depth, node, 64);
      cl[qt].pos = ctx + dq;
      if (a.window > 0)  // nodes that lie `window` and more above are out of it
        for (int m = 0; m < a.N; ++m)
          if (dq - __shfl(depth, m, 64) >= a.window) anc &= ~(1ull << m);
      cl[qt].anc = qvalid[qt] ? anc : 0ull;
    }
  } else {
    low = ctx + blk.i0;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int r = (wave * QT + qt) * 16 + col;
      qvalid[qt] = r < rows;
      cl[qt].pos = low + (qvalid[qt] ? r / a.G : 0);
      cl[qt].anc = 0;
    }
  }
  const int high = tree ? ctx + 63 : low + blk.nt - 1;  // no query stands behind it
  // the first position that any row sees, and the last first one
  const int from = a.window > 0 ? min(max(low - a.window + 1, 0), tree ? ctx : nkeys - 1) : 0;
  const int most_first = a.window > 0 ? max(high - a.window + 1, 0) : 0;
  const int least = tree ? ctx : low + 1;  // keys below it are visible to all (but the window)
  const int tlo = from / kKT, thi = (nkeys + kKT - 1) / kKT;
  const int tps = (thi - tlo + a.splits - 1) / a.splits;
  const int t0 = tlo + split * tps, t1 = min(thi, t0 + tps);
  const int g0 = t0 * (kKT / 16);
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
    cl[qt].first = a.window > 0 ? max(cl[qt].pos - a.window + 1, 0) : 0;
    cl[qt].slope2 = BIAS ? a.slopes[head] * kLog2e : 0.0f;
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
  auto issue = [&](int u, uint8_t *kdst, uint8_t *vdst) {
    const int kbase = u * kKT, gi = kbase / 16 - g0;
    const long long *kt = gtab + (gi + 2 * (wave >> 2) + (wave & 1)) % kMaxGroups;
    const long long *vt = gtab + (gi + (wave >> 1)) % kMaxGroups;
    if (kbase + kKT <= nkeys && kbase >= from)
      issue_tile_full<D>(a, kt, vt, doff, kdst, vdst, wave);
    else
      issue_tile<D, true>(a, kt, vt, kbase, nkeys, kdst, vdst, wave, lane, from);
  };
  const int32_t *btb = a.bt + (long long)b * a.max_blocks;
  const int ng = (t1 - t0) * (kKT / 16);
  auto look_up = [&](int first, int n) {
    for (int i = first + tid; i < min(first + n, ng); i += kNT)
      gtab[i % kMaxGroups] = group_row_offset<D, true>(a, btb, g0 + i, nkeys, h, from);
  };
  look_up(0, kMaxGroups);
  wait_vmcnt<0>();
  __syncthreads();

  f32x4 o[QT][D / 16];
  f32x4 lacc[QT];
  Softmax<QT> sm;
  float zero[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    zero[qt] = 0.0f;
    sm.b[qt] = 0.0f;
    sm.valid[qt] = FIXED;
    lacc[qt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) o[qt][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  if (t0 < t1) {
    // the phases and barriers of tree_attention.hip's loop
    for (int u = t0; u < min(t0 + 3, t1); ++u)
      issue(u, kring + ((u - t0) % kKStages) * kTileBytes,
            vring + ((u - t0) % kVStages) * kTileBytes);
    const int later = min(t0 + 3, t1) - 1 - t0;
    if (later >= 2) wait_vmcnt<2 * kLoadsPerTile>();
    else if (later == 1) wait_vmcnt<kLoadsPerTile>();
    else wait_vmcnt<0>();
    block_barrier();
    const bool lag = wave >= kWaves / 2;
    if (lag) block_barrier();
    Scores<QT> S;
    Probs<QT, T> P;
    const bool busy = wave * QT * 16 < rows;  // wave-uniform
    if (busy) qk_tile(ln, kring, zero, S);
    for (int t = t0; t < t1; ++t) {
      const int kbase = t * kKT;
      const int u = t + 3 - t0;
      // (both halves' groups were in use until now: the one in front of this
      // tile has no readers left, and its new entries have them 125 tiles on)
      if (t > t0 && (t - t0) % (kMaxTilesPerSplit / 2) == 0) {
        look_up((t - t0) * (kKT / 16) + kMaxGroups / 2, kMaxGroups / 2);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
      if (!lag) {
        block_barrier();
      } else {
        if (t + 2 < t1) wait_vmcnt<kLoadsPerTile>();
        else wait_vmcnt<0>();
        block_barrier();
      }
      if (t + 3 < t1)
        issue(t + 3, kring + (u % kKStages) * kTileBytes, vring + (u % kVStages) * kTileBytes);
      if (busy)
        score_phase<D, QT, T, CAP, BIAS, FIXED>(ln, cl, a, k0, cap2, kbase, ctx, least, most_first,
                                                sdepth, S, sm, o, lacc, P);
      if (!lag) {
        if (t + 3 < t1) wait_vmcnt<2 * kLoadsPerTile>();
        else if (t + 2 < t1) wait_vmcnt<kLoadsPerTile>();
        else wait_vmcnt<0>();
        block_barrier();
      } else {
        block_barrier();
      }
      __builtin_amdgcn_s_setprio(1);
      if (busy)
        mfma_phase(ln, kring + ((t + 1 - t0) % kKStages) * kTileBytes,
                   vring + ((t - t0) % kVStages) * kTileBytes, zero, P, S, o, lacc);
      __builtin_amdgcn_s_setprio(0);
    }
    if (!lag) block_barrier();
  }

#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const float ls = lacc[qt][0];
    if (!qvalid[qt]) continue;
    const int r = (wave * QT + qt) * 16 + col;
    const long long row = ((long long)blk.t0 + r / a.G) * a.Hq + (long long)h * a.G + r % a.G;
    if (a.splits == 1) {
      uint16_t *op = a.out + row * D;
      const float inv = ls != 0.0f ? 1.0f / ls : 0.0f;
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) {
        uint2 w;
        w.x = pack2<T>(o[qt][dt][0] * inv, o[qt][dt][1] * inv);
        w.y = pack2<T>(o[qt][dt][2] * inv, o[qt][dt][3] * inv);
        *reinterpret_cast<uint2 *>(op + dt * 16 + 4 * g) = w;
      }
    } else {
      const long long prow = (long long)split * a.T * a.Hq + row;
      float *pp = a.part_o + prow * D;
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt)
        *reinterpret_cast<f32x4 *>(pp + dt * 16 + 4 * g) = o[qt][dt];
      if (g == 0) a.part_ml[prow] = make_float2(sm.valid[qt] ? sm.b[qt] : -INFINITY, ls);
    }
  }
}

// Log-sum-exp merge of the splits: out = sum_s w_s o_s / sum_s w_s l_s with
// w_s = 2^(b_s - max b); four values a thread, D / 4 threads a row.  Rows of
// tokens that belong to no prompt are left alone.
constexpr int kMergeRegs = 8;  // splits whose loads are issued in one round
template <int D, class T>
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
  for (int s0 = 0; s0 < a.splits; s0 += kMergeRegs) {
    float2 ml[kMergeRegs];
    f32x4 v[kMergeRegs];
#pragma unroll
    for (int s = 0; s < kMergeRegs; ++s) {
      if (s0 + s < a.splits) {
        const long long p = (long long)(s0 + s) * rows + row;
        ml[s] = a.part_ml[p];
        v[s] = *reinterpret_cast<const f32x4 *>(a.part_o + p * D + e);
      }
    }
    float m = M;
#pragma unroll
    for (int s = 0; s < kMergeRegs; ++s)
      if (s0 + s < a.splits) m = fmaxf(m, ml[s].x);
    const float base = m == -INFINITY ? 0.0f : m;
    const float w0 = __builtin_amdgcn_exp2f(M - base);
    L *= w0;
    acc *= w0;
#pragma unroll
    for (int s = 0; s < kMergeRegs; ++s)
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
  *reinterpret_cast<uint2 *>(a.out + row * D + e) = w;
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
  CFA_LAUNCH("scored_merge", (scored_merge_kernel<D, T>), dim3((unsigned)((rows + per - 1) / per)),
             dim3(256), 0, st, a);
  return CFA_OK;
}

}  // namespace scored
}  // namespace cfa
