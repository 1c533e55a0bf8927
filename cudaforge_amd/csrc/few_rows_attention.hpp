// few_rows_attention.hpp -- attention of few query rows over the paged cache of e4m3
// codes: single tokens, small draft trees and short chunks (scored_attention.hpp's
// formulas, rows of G heads times tokens).
//
// With at most 32 query rows the products are small and the bytes are all: what
// counts is how many of them are on their way.  So no tile is shared.  Each of a
// work-group's four waves takes every fourth 64-key tile of the split for itself, from
// the last (nearest) on, and the waves meet only at the end, where their sums are
// joined in LDS by the largest of their exponent bases.
//   K  straight into registers: a lane holds 16 codes of a key at a time, which are
//      two operands of eight; the head's elements are taken in that order, Q's too.
//      A conversion scales as it goes (the row's scale is a power of two).
//   V  through the wave's own LDS, codes as they are (half the LDS bytes of 16-bit
//      tiles); a transposed read gives a lane eight keys of one element, and since
//      each key has a scale of its own, the scale goes to the key's probability:
//      p' = p 2^e, rounded to bf16; the row's sum is of what p' was rounded to, over 2^e.
//   The next tile's K and V are asked for as soon as the present tile's products with
//   Q have read its K.
// Measured, 32 heads of 128 over 8: 64 single tokens behind 1024 to 4096 keys 74 us, 4.6
// TB/s of codes (132 with the tiles that a work-group shares, which are turned into 16
// bits first); one token behind 1000 keys of its window 8.5, of which about 5 pass in
// front of the first tile, and 2.4 for the merge.
// p' needs fp32's range: the scales of a tile's keys lie 2^30 and more apart, and the
// largest may be that of a key that a row does not see.  V's codes are therefore taken as
// bf16, exactly, whatever q's type, and p' as bf16 too; for fp16 q in two parts, the
// rounded value and the rest, which keep 16 bits of it, and then the sum is of p (16 trees
// of 8 nodes over 4096 keys, bf16 q: 37 us with one part, 41 with two; fp16 40, and 39
// with p' in fp16 relative to the largest scale met, which lost the small values beside a
// large one).
#pragma once

#include "scored_attention.hpp"

namespace cfa {
namespace scored {

typedef int i32x2 __attribute__((ext_vector_type(2)));

constexpr int kFewWaves = 4;
constexpr int kFewNT = kFewWaves * 64;
constexpr int kFewTiles = 2;  // at most so many 16-row query tiles
// work-groups that a CU holds at once (LDS at head_dim 128, registers at 64)
constexpr int few_groups(int D, int QT) { return D == 64 && QT == 1 ? 3 : 2; }

template <int D, int QT, class T, bool CAP, bool BIAS, bool SINKS>
__global__ __launch_bounds__(kFewNT, few_groups(D, QT)) void few_rows_kernel(Args a) {
  constexpr int kTileBytes = kKT * D;  // of codes
  constexpr int kHalves = D / 64;      // 16-code loads of a lane for one key
  constexpr int kRowsPerLoad = 1024 / D;
  constexpr int kParts = std::is_same<T, BF16>::value ? 1 : 2;  // of a probability
  constexpr int kMerge = QT * 16 * (D + 4);  // floats of a wave's sums
  constexpr int kStageBytes = kFewWaves * 2 * kTileBytes;
  constexpr int kMergeBytes = kFewWaves * kMerge * 4;
  __shared__ __align__(16) uint8_t lds[kStageBytes > kMergeBytes ? kStageBytes : kMergeBytes];
  __shared__ float smove[192];
  __shared__ Row srow[QT * 16];
  __shared__ float sbase[kFewWaves][QT * 16], ssum[kFewWaves][QT * 16];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, g = lane >> 4;
  const int split = blockIdx.x % a.splits, rest = blockIdx.x / a.splits;
  const int h = rest % a.Hkv;
  View view;
  Row row[QT];
  bool qvalid[QT];
  if (!look_round<QT, BIAS, SINKS>(a, rest / a.Hkv, split, 0, wave, lane, view, row, qvalid, smove))
    return;
  const Block &blk = view.blk;
  const int from = view.from, sinks = view.sinks, nkeys = view.nkeys;
  constexpr float kLog2e = 1.4426950408889634f;
  const float cap2 = a.cap * kLog2e;
  const float k0 = (CAP ? 2.0f : 1.0f) * a.scale * kLog2e;

  Lane<D, QT, T> ln;
  ln.g = g;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int r = qt * 16 + col;
    const int nl = qvalid[qt] ? r / a.G : 0, hg = qvalid[qt] ? r % a.G : 0;
    const int head = h * a.G + hg;
    row[qt].first = a.window > 0 ? max(row[qt].pos - a.window + 1, 0) : 0;
    row[qt].slope2 = BIAS ? a.slopes[head] * kLog2e : 0.0f;
    if (wave == 0 && g == 0) srow[r] = row[qt];
    const uint16_t *qp = a.q + (((long long)blk.t0 + nl) * a.Hq + head) * D;
#pragma unroll
    for (int kk = 0; kk < D / 32; ++kk) {  // the elements of K's operands, see above
      const uint4 v = qvalid[qt] ? ld_g16(qp + (kk >> 1) * 64 + g * 16 + (kk & 1) * 8)
                                 : make_uint4(0, 0, 0, 0);
      ln.qf[qt][kk] = __builtin_bit_cast(typename Mfma<T>::frag, v);
    }
  }
  __syncthreads();

  const int32_t *btb = a.bt + (long long)blk.b * a.max_blocks;
  uint8_t *const vlds = lds + wave * 2 * kTileBytes;
  // K keys of this lane's operand rows: key blk * 32 + 4 T + kkey
  const int kkey = 8 * (col >> 2) + (col & 3);

  // Row offsets of the 16-key groups of the wave's next 16 tiles, one a lane: group
  // l % 4 of tile i - 4 (l / 4).  The block numbers of a batch are asked for a batch
  // ahead, so that no tile's transfers wait for them.
  auto first_of = [&](int i) {
    const int gi = view.key_of<SINKS>(i - kFewWaves * (lane >> 2)) / 16 + (lane & 3);
    return clamp_pos<true>(gi * 16, gi * 16, from, sinks, nkeys);
  };
  auto block_of = [&](int first) { return btb[min(max(first, 0) / a.bs, a.max_blocks - 1)]; };
  auto offset_of = [&](int block, int first) {
    const long long blk = min(max(block, 0), a.num_blocks - 1);
    first = max(first, 0);
    return ((blk * a.num_layers + a.layer) * a.Hkv + h) * ((long long)a.bs * D) +
           (long long)(first - min(first / a.bs, a.max_blocks - 1) * a.bs) * D;
  };
  auto group_of = [&](long long offs, int j) {
    return (long long)(((unsigned long long)(uint32_t)__builtin_amdgcn_readlane(
                            (int)((unsigned long long)offs >> 32), j)
                        << 32) |
                       (uint32_t)__builtin_amdgcn_readlane((int)offs, j));
  };
  auto is_full = [&](int kbase) {
    return (kbase + kKT <= nkeys && kbase >= from) || (SINKS && kbase + kKT <= sinks);
  };
  // where key `key` of the tile lies behind its group's row offset, in rows
  auto in_group = [&](int kbase, int key, bool full) {
    if (full) return key & 15;
    const int group = kbase + (key & ~15);
    return clamp_pos<true>(kbase + key, group, from, sinks, nkeys) -
           clamp_pos<true>(group, group, from, sinks, nkeys);
  };

  uint4 kraw[2][2][kHalves];  // [blk][T]
  uint32_t kbyte[2][2];
  uint2 vbyte[2];  // of keys blk * 32 + 8 g + 0 .. 7
  auto ask = [&](int i, long long offs, int n, int stage) {  // n: the tile's place in offs
    const int kbase = view.key_of<SINKS>(i);
    const bool full = is_full(kbase);
    long long go[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) go[j] = group_of(offs, 4 * n + j);
#pragma unroll
    for (int j = 0; j < kTileBytes / 1024; ++j) {
      const int key = j * kRowsPerLoad + lane / (D / 16);
      const int swz = D == 128 ? key & 7 : (key >> 1) & 3;
      const int grp = j * kRowsPerLoad / 16;
      const uint32_t off = (uint32_t)(in_group(kbase, key, full) * D + ((lane % (D / 16)) ^ swz) * 16);
      dma16((const uint8_t *)a.vpool + go[grp] + off,
            (CFA_LDS void *)(vlds + stage * kTileBytes + j * 1024));
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const long long kgo = col >> 3 ? go[2 * b + 1] : go[2 * b];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int in = in_group(kbase, b * 32 + 4 * t + kkey, full);
        const uint8_t *kp = (const uint8_t *)a.kpool + kgo + (long long)in * D + g * 16;
#pragma unroll
        for (int hf = 0; hf < kHalves; ++hf)
          kraw[b][t][hf] = *reinterpret_cast<const uint4 *>(kp + hf * 64);
        kbyte[b][t] = a.kscale[kgo / D + in];
      }
      const long long vgo = g >> 1 ? go[2 * b + 1] : go[2 * b];
      vbyte[b] = *reinterpret_cast<const uint2 *>(a.vscale + (vgo / D & ~15LL) + 8 * (g & 1));
    }
    // (the loads stay here, in front of what the present tile is still to do)
    asm volatile("" ::: "memory");
  };

  f32x4 o[QT][D / 16];
  float base[QT], sum[QT];
  bool set[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    base[qt] = sum[qt] = 0.0f;
    set[qt] = false;
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) o[qt][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const Row *const rows_at = srow + col;

  // (a split without keys has no tile, also where the window's first tile is numbered)
  int i = (view.steps > 0 ? view.t1 : view.t0) - 1 - wave;
  int stage = 0, n = 0;
  long long offs = 0;
  int next_block = 0;
  if (i >= view.t0) {
    offs = offset_of(block_of(first_of(i)), first_of(i));
    ask(i, offs, 0, 0);
    next_block = block_of(first_of(i - 16 * kFewWaves));
  }
  for (; i >= view.t0; i -= kFewWaves, stage ^= 1) {
    const int kbase = view.key_of<SINKS>(i);
    const bool full = is_full(kbase);
    wait_vmcnt<0>();
    asm volatile("" ::: "memory");
    // S^T = K Q^T
    Scores<QT> S;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int t = 0; t < 2; ++t) S.s[qt][b][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int kk = 0; kk < D / 32; ++kk)
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const uint4 w = kraw[b][t][kk >> 1];
          const uint32_t lo = kk & 1 ? w.z : w.x, hi = kk & 1 ? w.w : w.y;
          const float s = e4m3::scale(kbyte[b][t]);
          const uint4 v = make_uint4(
              e4m3::unpack_pair<T, false>(lo, s), e4m3::unpack_pair<T, true>(lo, s),
              e4m3::unpack_pair<T, false>(hi, s), e4m3::unpack_pair<T, true>(hi, s));
          const auto kf = __builtin_bit_cast(typename Mfma<T>::frag, v);
#pragma unroll
          for (int qt = 0; qt < QT; ++qt)
            S.s[qt][b][t] = Mfma<T>::run(kf, ln.qf[qt][kk], S.s[qt][b][t]);
        }
    // V's scales: bytes to factors of the probabilities (of keys that were re-read: 0)
    uint32_t vb[2][2] = {{vbyte[0].x, vbyte[0].y}, {vbyte[1].x, vbyte[1].y}};
    if (!full) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int key = b * 32 + 8 * g + 4 * t + k, group = kbase + (key & ~15);
            if (clamp_pos<true>(kbase + key, group, from, sinks, nkeys) != kbase + key)
              vb[b][t] &= ~(255u << (8 * k));
          }
    }
    const int ahead = i - kFewWaves;
    if (ahead >= view.t0) {
      if (++n == 16) {
        n = 0;
        offs = offset_of(next_block, first_of(ahead));
        next_block = block_of(first_of(ahead - 16 * kFewWaves));
      }
      ask(ahead, offs, n, stage ^ 1);
    }
    raw_scores<D, QT, T, CAP, BIAS, false, SINKS>(ln, base, a, k0, cap2, kbase, view.ctx, view.least,
                                                  view.most_first, rows_at, smove + 64, S);
    float by[QT];
    bool any = false;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const float mx = score_max(S, qt);
      by[qt] = mx > kRescaleSlack || (!set[qt] && mx > -INFINITY) ? mx : 0.0f;
      set[qt] = set[qt] || mx > -INFINITY;
      any |= by[qt] != 0.0f;
    }
    if (__ballot(any) != 0) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        // (a base falls only while the sums are still 0)
        const float alpha = __builtin_amdgcn_exp2f(-fmaxf(by[qt], 0.0f));
        base[qt] += by[qt];
        sum[qt] *= alpha;
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) o[qt][dt] *= alpha;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int t = 0; t < 2; ++t) S.s[qt][b][t] -= by[qt];
      }
    }
    // O^T += V^T P^T, 32 keys at a time
    const uint8_t *const vs = vlds + stage * kTileBytes;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      u32x4 p[QT], rest[QT];
      float part[QT] = {};
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
          // two keys' scales as a bf16 pair, and one over them
          const uint32_t pair =
              __builtin_amdgcn_perm(0u, vb[b][t], k == 0 ? 0x0c010c00u : 0x0c030c02u) << 7;
          const uint32_t back = 0x7f007f00u - pair;
          float f0, f1;
          unpack2<BF16>(pair, f0, f1);
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) {
            const float x0 = __builtin_amdgcn_exp2f(S.s[qt][b][t][k]);
            const float x1 = __builtin_amdgcn_exp2f(S.s[qt][b][t][k + 1]);
            const uint32_t high = pack2<BF16>(x0 * f0, x1 * f1);
            p[qt][t * 2 + k / 2] = high;
            if constexpr (kParts == 2) {
              float h0, h1;
              unpack2<BF16>(high, h0, h1);
              rest[qt][t * 2 + k / 2] = pack2<BF16>(x0 * f0 - h0, x1 * f1 - h1);
              sum[qt] += x0 + x1;
            } else {  // of the rounded ones
              part[qt] = dot2(BF16{}, high, back, part[qt]);
            }
          }
        }
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) sum[qt] += part[qt];
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) {
        const int key = b * 32 + 8 * g + (col >> 1);
        const int swz = D == 128 ? key & 7 : (key >> 1) & 3;
        const i32x2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
            (CFA_LDS i32x2 *)(vs + key * D + ((dt ^ swz) << 4) + (col & 1) * 8));
        const uint4 v = make_uint4(
            e4m3::unpack_pair<BF16, false>(w.x, 1.0f), e4m3::unpack_pair<BF16, true>(w.x, 1.0f),
            e4m3::unpack_pair<BF16, false>(w.y, 1.0f), e4m3::unpack_pair<BF16, true>(w.y, 1.0f));
        typedef Mfma<BF16>::frag frag;
        const auto vf = __builtin_bit_cast(frag, v);
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
          o[qt][dt] = Mfma<BF16>::run(vf, __builtin_bit_cast(frag, p[qt]), o[qt][dt]);
          if constexpr (kParts == 2)
            o[qt][dt] = Mfma<BF16>::run(vf, __builtin_bit_cast(frag, rest[qt]), o[qt][dt]);
        }
      }
    }
  }

  // The waves' sums: a row's is over the four lanes of its column.
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    sum[qt] += __shfl_xor(sum[qt], 16, 64);
    sum[qt] += __shfl_xor(sum[qt], 32, 64);
    if (g == 0) {
      sbase[wave][qt * 16 + col] = sum[qt] != 0.0f ? base[qt] : -INFINITY;
      ssum[wave][qt * 16 + col] = sum[qt];
    }
  }
  __syncthreads();  // every wave is done with its V
  float *const merge = reinterpret_cast<float *>(lds);
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int r = qt * 16 + col;
    float m = sbase[0][r];
#pragma unroll
    for (int w = 1; w < kFewWaves; ++w) m = fmaxf(m, sbase[w][r]);
    const float mine = sum[qt] != 0.0f ? __builtin_amdgcn_exp2f(base[qt] - m) : 0.0f;
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt)
      *reinterpret_cast<f32x4 *>(merge + (wave * QT * 16 + r) * (D + 4) + dt * 16 + 4 * g) =
          o[qt][dt] * mine;
  }
  __syncthreads();
  for (int x = tid; x < QT * 16 * (D / 4); x += kFewNT) {
    const int r = x / (D / 4), e = x % (D / 4) * 4;
    if (r >= view.rows) continue;
    float m = sbase[0][r], l = 0.0f;
#pragma unroll
    for (int w = 1; w < kFewWaves; ++w) m = fmaxf(m, sbase[w][r]);
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) {
      acc += *reinterpret_cast<const f32x4 *>(merge + (w * QT * 16 + r) * (D + 4) + e);
      const float s = ssum[w][r];
      l += s != 0.0f ? __builtin_amdgcn_exp2f(sbase[w][r] - m) * s : 0.0f;
    }
    const long long orow =
        ((long long)blk.t0 + r / a.G) * a.Hq + (long long)h * a.G + r % a.G;
    if (a.splits == 1) {
      const float inv = l != 0.0f ? 1.0f / l : 0.0f;
      uint2 w;
      w.x = pack2<T>(acc[0] * inv, acc[1] * inv);
      w.y = pack2<T>(acc[2] * inv, acc[3] * inv);
      *reinterpret_cast<uint2 *>(a.out + orow * D + e) = w;
    } else {
      const long long prow = (long long)split * a.T * a.Hq + orow;
      *reinterpret_cast<f32x4 *>(a.part_o + prow * D + e) = acc;
      if (e == 0) a.part_ml[prow] = make_float2(m, l);
    }
  }
}

template <int D, int QT, class T>
int launch_few_scores(const Args &a, unsigned grid, hipStream_t st) {
  const bool cap = a.cap > 0.0f, bias = a.slopes != nullptr;
#define CFA_FEW(C, B)                                                                           \
  do {                                                                                          \
    if (a.sinks > 0)                                                                            \
      CFA_LAUNCH("few_rows_attn", (few_rows_kernel<D, QT, T, C, B, true>), dim3(grid),       \
                 dim3(kFewNT), 0, st, a);                                                       \
    else                                                                                        \
      CFA_LAUNCH("few_rows_attn", (few_rows_kernel<D, QT, T, C, B, false>), dim3(grid),      \
                 dim3(kFewNT), 0, st, a);                                                       \
  } while (0)
  if (cap && bias) CFA_FEW(true, true);
  else if (cap) CFA_FEW(true, false);
  else if (bias) CFA_FEW(false, true);
  else CFA_FEW(false, false);
#undef CFA_FEW
  return CFA_OK;
}

template <int D, class T>
int launch_few(const Args &a, bool one, unsigned grid, hipStream_t st) {
  const int rc = one ? launch_few_scores<D, 1, T>(a, grid, st)
                     : launch_few_scores<D, 2, T>(a, grid, st);
  return rc != CFA_OK ? rc : launch_merge<D, T>(a, st);
}

}  // namespace scored
}  // namespace cfa
