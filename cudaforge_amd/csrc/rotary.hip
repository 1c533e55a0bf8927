// rotary.hip -- RMSNorm of every q and k head, rotary positions and the write
// of k and v into the paged cache, one pass over a QKV projection.
//
// For token t and q or k head x of D elements (fp32 arithmetic, one rounding):
//   y = x * rsqrt(mean(x^2) + eps) * w                 (w given; else y = x)
//   pairs (a, b) of the first R elements, at angle p_t f_i (position times the
//   pair's frequency), as halves (i, i + R/2) or as neighbours (2i, 2i + 1):
//   (a, b) -> factor * (a cos - b sin, b cos + a sin)
// v is copied.  q goes to q_out [T, Hq, D], k and v to the sequence's slots
// base[b] + j of pool[block][layer][kv_head][slot][D], as they are or as e4m3
// codes with a scale a row (e4m3.hpp): v's elements, and k's results in 64 bits.
//
// Angles.  At position 100000 an fp32 product p f is off by up to 0.004
// radians, more than bf16 resolves.  Frequencies are therefore 64-bit
// fractions of a turn: p times the fraction, modulo 2^64, is the angle modulo
// a whole turn without any rounding, for every 32-bit position of either sign,
// and its upper 32 bits go to the sine and cosine (which take turns).
//
// Bound: HBM.  Each element is read and written once (D bytes * 4 a head and
// token), the arithmetic hides under that.  A head is one group of D / 8 lanes
// (16 bytes a lane): its sum of squares stays in the group, and a half-layout
// pair is one exchange between two of its lanes.  A wave keeps one token, so
// that its angles and the norms' weights are formed once for its heads.  8149
// tokens of 48 heads of 128: 51 us, 3.9 TB/s (pages scattered, 256 bytes a row); 504
// tokens 7 us, 8 tokens 5.  Into e4m3 pages (184 MB): 61 us for the 8149, 6 for 8, with
// keys in 64 bits.  In fp32 56 to 60, but then 12 to 26 of 8.4 million codes were other
// than their exact values', against none.
#include <hip/hip_runtime.h>

#include "abi_internal.hpp"
#include "e4m3.hpp"
#include "half_types.hpp"
#include "packed_tokens.hpp"

namespace cfa {
namespace rotary {

constexpr int kIter = 4;   // rows of a lane group whose loads are in flight at once
constexpr int kWaves = 4;  // waves per work-group, each with its own (token, heads)
enum Layout { kHalf = 0, kHalfAny = 1, kNeighbours = 2 };

struct Args {
  const uint16_t *q, *k, *v;
  long long q_st, q_sh, k_st, k_sh, v_st, v_sh;  // elements
  const int32_t *pos;  // [T]
  const int32_t *cu;   // [B + 1], or null: token t is b = t / n, j = t % n
  int T, B, n, Hq, Hkv, D, R;
  const uint64_t *turns;  // [R / 2]
  float factor;
  const void *q_w, *k_w;  // [D] or null
  int w_f32;
  float eps;
  uint16_t *q_out;
  void *kc, *vc;
  uint8_t *ks, *vs;  // e4m3: scales [blocks, layers, Hkv, bs]
  int num_blocks, max_blocks, bs;
  const int32_t *block_tables, *base;
  long long blk_stride, layer_off, head_stride;  // elements
  int chunks, rounds;        // waves a token; rounds of rows a wave
  int kv_chunks, kv_rounds;  // e4m3: the same of its k and v rows, `chunks` of its q rows
};

// Sum over the LPR lanes of a head, every lane gets it.
template <int LPR>
__device__ __forceinline__ float group_sum(float v) {
#define CFA_DPP(ctrl) \
  v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), ctrl, 0xf, 0xf, true))
  CFA_DPP(0xB1);                           // lane ^ 1
  CFA_DPP(0x4E);                           // lane ^ 2
  if constexpr (LPR >= 8) CFA_DPP(0x141);  // mirrored in 8 lanes: the other quad
  if constexpr (LPR >= 16) CFA_DPP(0x140);  // mirrored in 16 lanes: the other 8
#undef CFA_DPP
  if constexpr (LPR >= 32) v += __shfl_xor(v, 16, 64);
  return v;
}

template <int LPR>
__device__ __forceinline__ double group_sum(double v) {
#pragma unroll
  for (int d = 1; d < LPR; d *= 2) v += __shfl_xor(v, d, 64);
  return v;
}

// Largest over the LPR lanes of a head, every lane gets it.
template <int LPR>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
#define CFA_DPP(ctrl) \
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xf, 0xf, true))
  CFA_DPP(0xB1);  // the lanes of group_sum
  CFA_DPP(0x4E);
  if constexpr (LPR >= 8) CFA_DPP(0x141);
  if constexpr (LPR >= 16) CFA_DPP(0x140);
#undef CFA_DPP
  if constexpr (LPR >= 32) v = max(v, (uint32_t)__shfl_xor((int)v, 16, 64));
  return v;
}

// Sixteen bytes at any element: views of a projection may begin anywhere, and an
// access that an address splits costs little (eight of 2 bytes: four times as many).
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 at_element __attribute__((aligned(2)));
__device__ __forceinline__ uint4 load8(const void *p) {
  const u32x4 w = *reinterpret_cast<const at_element *>(p);
  return make_uint4(w.x, w.y, w.z, w.w);
}
// Past the caches: 8149 tokens 54.2 -> 50.9 us, and with the attention that reads them
// next 31.6 -> 29.7 (4 chunks of 256), 556 -> 558 (one of 8192).
__device__ __forceinline__ void store8(uint16_t *p, const uint32_t (&w)[4]) {
  __builtin_nontemporal_store(u32x4{w[0], w[1], w[2], w[3]}, reinterpret_cast<at_element *>(p));
}

template <class T>
__device__ __forceinline__ void unpack8(const uint4 &v, float (&x)[8]) {
  unpack2<T>(v.x, x[0], x[1]);
  unpack2<T>(v.y, x[2], x[3]);
  unpack2<T>(v.z, x[4], x[5]);
  unpack2<T>(v.w, x[6], x[7]);
}

// Weights e .. e + 7 of a norm (1 where there is none).
template <class T>
__device__ __forceinline__ void weights8(const void *w, int f32, int e, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = 1.0f;
  if (!w) return;
  if (f32) {
    const float *p = reinterpret_cast<const float *>(w) + e;
    const uint4 a = load8(p), b = load8(p + 4);
    const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(u[i]);
  } else {
    unpack8<T>(load8(reinterpret_cast<const uint16_t *>(w) + e), x);
  }
}

// One of them.
template <class T>
__device__ __forceinline__ float weight(const void *w, int f32, int e) {
  if (!w) return 1.0f;
  if (f32) return reinterpret_cast<const float *>(w)[e];
  return (float)reinterpret_cast<const typename T::elem *>(w)[e];
}

// N frequencies from number i on.
template <int N>
__device__ __forceinline__ void turns_at(const Args &a, int i, uint64_t (&t)[N]) {
#pragma unroll
  for (int k = 0; k < N; k += 2) {
    const uint4 v = load8(a.turns + i + k);
    t[k] = ((uint64_t)v.y << 32) | v.x;
    t[k + 1] = ((uint64_t)v.w << 32) | v.z;
  }
}

// factor * (cos, sin) of position p on a pair's frequency.  The instructions take turns; over
// [-1/2, 1/2] they are off by at most 2^-22.9 (six million values measured),
// where the library's cospi and sinpi take some 30 instructions each.
__device__ __forceinline__ void angle(const Args &a, int p, uint64_t turns, float &cs, float &sn) {
  const uint64_t turn = turns * (uint64_t)(int64_t)p;
  const float f = (float)(int32_t)(turn >> 32) * 0x1p-32f;  // [-1/2, 1/2] turns
  cs = a.factor * __builtin_amdgcn_cosf(f);
  sn = a.factor * __builtin_amdgcn_sinf(f);
}

// The same in 64 bits, for what becomes codes: there a rounding on the way in can move
// the result by a whole step of 2^-3, so keys are formed in 64 bits and rounded once.
// The turn less its nearest quarter is exact in integers; over [-1/8, 1/8] turns
// sin(2 pi f) / f and cos(2 pi f) are polynomials in f^2, fitted for the least relative
// error (2^-37 and 2^-34).
__device__ __forceinline__ void fine_angle(const Args &a, int p, uint64_t turns, double &cs,
                                           double &sn) {
  const uint64_t turn = turns * (uint64_t)(int64_t)p;
  const uint32_t quarter = (uint32_t)((turn + (1ull << 61)) >> 62);
  const double f = (double)(int64_t)(turn - ((uint64_t)quarter << 62)) * 0x1p-64;
  const double z = f * f;
  const double sine =
      f * (6.283185307151002 +
           z * (-41.341702150556394 +
                z * (81.60520380748551 + z * (-76.69777415285763 + z * 41.46989043587605))));
  const double cosine =
      0.9999999999439374 +
      z * (-19.739208633036213 +
           z * (64.9393107446243 + z * (-85.44229797458063 + z * 59.202796144154824)));
  const double along = (double)a.factor * (quarter & 1 ? sine : cosine);
  const double across = (double)a.factor * (quarter & 1 ? cosine : sine);
  cs = (quarter + 1) & 2 ? -along : along;
  sn = quarter & 2 ? -across : across;
}

// 1 / sqrt(mean) in 64 bits: the instruction's (some 2^-23) and a step of Newton's (none
// where that is 0 or infinite).
__device__ __forceinline__ double fine_rsqrt(double mean) {
  const double r = __builtin_amdgcn_rsq(mean);
  if (!(r > 0.0 && r < INFINITY)) return r;
  return r + 0.5 * r * (1.0 - mean * r * r);
}

// v as fp32, rounded to odd: toward zero, with the last bit set where bits were lost, so
// that the code's rounding behind it is v's own (no second rounding to a tie).
__device__ __forceinline__ float round_to_odd(double v) {
  const float f = (float)v;
  const double d = f;
  uint32_t w = __float_as_uint(f);
  w -= __builtin_fabs(d) > __builtin_fabs(v) ? 1u : 0u;
  w |= d != v ? 1u : 0u;
  return __uint_as_float(w);
}

// One wave = one token and `rounds` times ITER * 64 / LPR consecutive rows of its
// Hq q heads, Hkv k heads and Hkv v heads.
template <class T, int LPR, int LAYOUT, int ITER>
__global__ __launch_bounds__(kWaves * 64) void qk_norm_rope_kv_kernel(Args a) {
  constexpr int RPW = 64 / LPR;
  const int lane = threadIdx.x & 63, l = lane % LPR;
  const long long item = (long long)blockIdx.x * kWaves + (threadIdx.x >> 6);
  const int t = (int)(item / a.chunks), chunk = (int)(item % a.chunks);
  if (t >= a.T) return;
  const int e = 8 * l, H = a.Hq + 2 * a.Hkv;
  const bool mine = e < a.D;
  const int row0 = chunk * a.rounds * ITER * RPW + lane / LPR;

  uint4 raw[ITER];
  auto load = [&](int round) {
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
      const int row = row0 + (round * ITER + it) * RPW;
      raw[it] = make_uint4(0, 0, 0, 0);
      if (row < H && mine) {
        const uint16_t *src =
            row < a.Hq ? a.q + t * a.q_st + row * a.q_sh
                       : row < a.Hq + a.Hkv ? a.k + t * a.k_st + (row - a.Hq) * a.k_sh
                                            : a.v + t * a.v_st + (row - a.Hq - a.Hkv) * a.v_sh;
        raw[it] = load8(src + e);
      }
    }
  };
  load(0);
  int b, j;
  if (!place_token(a, t, lane, b, j)) return;
  // this lane's cosines and sines: c[i], s[i] of element e + i, the sine with
  // the sign that its partner's value takes
  float c[8], s[8], wq[8], wk[8];
  const int half = a.R / 2;
  const int p = a.pos[t];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    c[i] = 1.0f;
    s[i] = 0.0f;
  }
  if constexpr (LAYOUT == kNeighbours) {
    if (e + 8 <= a.R) {
      uint64_t f[4];
      turns_at<4>(a, e / 2, f);
#pragma unroll
      for (int i = 0; i < 8; i += 2) angle(a, p, f[i / 2], c[i], s[i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i += 2)
        if (e + i < a.R) angle(a, p, a.turns[(e + i) / 2], c[i], s[i + 1]);
    }
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      c[i + 1] = c[i];
      s[i] = -s[i + 1];
    }
  } else if constexpr (LAYOUT == kHalf) {
    if (e < a.R) {  // a lane's eight lie in one half
      const bool first = e < half;
      uint64_t f[8];
      turns_at<8>(a, first ? e : e - half, f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        angle(a, p, f[i], c[i], s[i]);
        s[i] = first ? -s[i] : s[i];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (e + i < a.R) {
        const bool first = e + i < half;
        angle(a, p, a.turns[first ? e + i : e + i - half], c[i], s[i]);
        if (first) s[i] = -s[i];
      }
    }
  }
  if (mine) {
    weights8<T>(a.q_w, a.w_f32, e, wq);
    weights8<T>(a.k_w, a.w_f32, e, wk);
  }
  // the page of this token's slot
  const long long slot = (long long)a.base[b] + j;
  const long long page = slot / a.bs;
  int blk = -1;
  if (slot >= 0 && page < a.max_blocks) blk = a.block_tables[(long long)b * a.max_blocks + page];
  const bool mapped = blk >= 0 && blk < a.num_blocks;
  const long long at = blk * a.blk_stride + a.layer_off + (slot - page * a.bs) * a.D;

  for (int round = 0; round < a.rounds; ++round) {
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
      const int row = row0 + (round * ITER + it) * RPW;
      const bool is_q = row < a.Hq, is_v = row >= a.Hq + a.Hkv;
      float x[8], y[8];
      unpack8<T>(raw[it], x);
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
      ss = group_sum<LPR>(ss);
      const bool norm = (is_q ? a.q_w : a.k_w) != nullptr;
      const float inv = norm ? rsqrtf(ss / (float)a.D + a.eps) : 1.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= inv * (is_q ? wq[i] : wk[i]);
      if constexpr (LAYOUT == kHalf) {
        // R / 2 is a multiple of 8: the partner's elements are one lane's
        const int to = e < half ? lane + half / 8 : (e < a.R ? lane - half / 8 : lane);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = __shfl(x[i], to, 64);
      } else if constexpr (LAYOUT == kHalfAny) {
        // element by element: partner e + i +- R / 2, in lane (e + i +- R / 2) / 8
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int el = e + i;
          const int pe = el < half ? el + half : (el < a.R ? el - half : el);
          const int from = lane - l + pe / 8;
          float v = 0.0f;
#pragma unroll
          for (int m = 0; m < 8; ++m) {
            const float got = __shfl(x[m], from, 64);
            if (pe % 8 == m) v = got;
          }
          y[i] = v;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = x[i ^ 1];
      }
      if (row >= H || !mine) continue;
      // (elements behind the rotated ones are selected, not turned by 0: they
      // may be infinite)
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = e + i < a.R ? x[i] * c[i] + y[i] * s[i] : x[i];
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = pack2<T>(x[2 * i], x[2 * i + 1]);
      if (is_v) {  // as it is
        w[0] = raw[it].x;
        w[1] = raw[it].y;
        w[2] = raw[it].z;
        w[3] = raw[it].w;
      }
      if (is_q)
        store8(a.q_out + ((long long)t * a.Hq + row) * a.D + e, w);
      else if (mapped)
        store8((is_v ? (uint16_t *)a.vc + (row - a.Hq - a.Hkv) * a.head_stride
                          : (uint16_t *)a.kc + (row - a.Hq) * a.head_stride) + at + e, w);
    }
    if (round + 1 < a.rounds) load(round + 1);
  }
}

// The same into e4m3 pools.  q rows, in the arithmetic above (and its bits), and k and v
// rows are different waves', which then hold one kind of angles and weights each: four
// waves a SIMD, where both kinds took 142 registers and left three.  (8149 tokens: 61 us;
// without the bound on registers 130 of them, and 71.)  Partners exchange the elements as
// they are read, exact in fp32, and what multiplies them is formed in 64 bits once a wave.
template <class T, int LPR, int LAYOUT, int ITER>
__global__ __launch_bounds__(kWaves * 64, LAYOUT != kHalfAny ? 4 : 1) void
qk_norm_rope_kv_e4m3_kernel(Args a) {
  constexpr int RPW = 64 / LPR;
  const int lane = threadIdx.x & 63, l = lane % LPR;
  const long long item = (long long)blockIdx.x * kWaves + (threadIdx.x >> 6);
  const int all = a.chunks + a.kv_chunks;
  const int t = (int)(item / all), chunk = (int)(item % all);
  if (t >= a.T) return;
  const int e = 8 * l;
  const bool kv = __builtin_amdgcn_readfirstlane(chunk) >= a.chunks;
  const int rounds = kv ? a.kv_rounds : a.rounds;
  const int H = !kv ? a.Hq : a.Hq + 2 * a.Hkv;  // the wave's rows end here
  const bool mine = e < a.D;
  const int row0 = (kv ? a.Hq + (chunk - a.chunks) * rounds * ITER * RPW
                       : chunk * rounds * ITER * RPW) + lane / LPR;

  uint4 raw[ITER];
  auto load = [&](int round) {
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
      const int row = row0 + (round * ITER + it) * RPW;
      raw[it] = make_uint4(0, 0, 0, 0);
      if (row < H && mine) {
        const uint16_t *src =
            row < a.Hq ? a.q + t * a.q_st + row * a.q_sh
                       : row < a.Hq + a.Hkv ? a.k + t * a.k_st + (row - a.Hq) * a.k_sh
                                            : a.v + t * a.v_st + (row - a.Hq - a.Hkv) * a.v_sh;
        raw[it] = load8(src + e);
      }
    }
  };
  load(0);
  int b, j;
  if (!place_token(a, t, lane, b, j)) return;
  const int half = a.R / 2;
  const int p = a.pos[t];
  // the page of this token's slot
  const long long slot = (long long)a.base[b] + j;
  const long long page = slot / a.bs;
  int blk = -1;
  if (slot >= 0 && page < a.max_blocks) blk = a.block_tables[(long long)b * a.max_blocks + page];
  const bool mapped = blk >= 0 && blk < a.num_blocks;
  const long long at = blk * a.blk_stride + a.layer_off + (slot - page * a.bs) * a.D;
  // of the partners' p
  __shared__ __align__(16) float swap[LAYOUT == kHalfAny ? kWaves * 64 * 8 : 1];
  auto exchange = [&](const float(&p)[8], float(&y)[8]) {
    if constexpr (LAYOUT == kHalf) {
      // R / 2 is a multiple of 8: the partner's elements are one lane's
      const int to = e < half ? lane + half / 8 : (e < a.R ? lane - half / 8 : lane);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = __shfl(p[i], to, 64);
    } else if constexpr (LAYOUT == kHalfAny) {
      // element by element, through the wave's LDS (in order within a wave)
      float *const own = swap + (threadIdx.x & ~63) * 8;
      float4 *const mine8 = reinterpret_cast<float4 *>(own + lane * 8);
      mine8[0] = make_float4(p[0], p[1], p[2], p[3]);
      mine8[1] = make_float4(p[4], p[5], p[6], p[7]);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int el = e + i;
        y[i] = own[(lane - l) * 8 + (el < half ? el + half : (el < a.R ? el - half : el))];
      }
      __builtin_amdgcn_wave_barrier();
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = p[i ^ 1];
    }
  };

  // turn(frequency, i, whether it is the pair's first) for each of the lane's elements
  // e + i that turn (neighbours: for the pairs' first ones)
  auto angles = [&](auto turn) {
    if constexpr (LAYOUT == kNeighbours) {
      if (e + 8 <= a.R) {
        uint64_t f[4];
        turns_at<4>(a, e / 2, f);
#pragma unroll
        for (int i = 0; i < 8; i += 2) turn(f[i / 2], i, true);
      } else {
#pragma unroll
        for (int i = 0; i < 8; i += 2)
          if (e + i < a.R) turn(a.turns[(e + i) / 2], i, true);
      }
    } else if constexpr (LAYOUT == kHalf) {
      if (e < a.R) {  // a lane's eight lie in one half
        const bool first = e < half;
        uint64_t f[8];
        turns_at<8>(a, first ? e : e - half, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) turn(f[i], i, first);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (e + i < a.R) {
          const bool first = e + i < half;
          turn(a.turns[first ? e + i : e + i - half], i, first);
        }
      }
    }
  };

  if (kv) {
    // element e + i of a key is x ca[i] + y cb[i], y its partner in the pair: the norm's
    // weights times the cosine, and the partner's times the sine with its sign
    double ca[8], cb[8];
    {
      float w[8], wp[8];
      weights8<T>(a.k_w, a.w_f32, mine ? e : 0, w);
      if constexpr (LAYOUT == kHalf) {
        weights8<T>(a.k_w, a.w_f32, e < half ? e + half : e < a.R ? e - half : 0, wp);
      } else if constexpr (LAYOUT == kNeighbours) {
#pragma unroll
        for (int i = 0; i < 8; ++i) wp[i] = w[i ^ 1];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ca[i] = w[i];
        cb[i] = 0.0;
      }
      auto turn = [&](uint64_t turns, int i, bool front) {
        double cs, sn;
        fine_angle(a, p, turns, cs, sn);
        ca[i] = w[i] * cs;
        if constexpr (LAYOUT == kHalfAny)
          wp[i] = weight<T>(a.k_w, a.w_f32, front ? e + i + half : e + i - half);
        cb[i] = wp[i] * (front ? -sn : sn);
        if constexpr (LAYOUT == kNeighbours) {
          ca[i + 1] = w[i + 1] * cs;
          cb[i + 1] = wp[i + 1] * sn;
        }
      };
      angles(turn);
    }
    for (int round = 0; round < rounds; ++round) {
#pragma unroll
      for (int it = 0; it < ITER; ++it) {
        const int row = row0 + (round * ITER + it) * RPW;
        const bool is_v = row >= a.Hq + a.Hkv;
        float x[8], y[8];
        unpack8<T>(raw[it], x);
        if (__builtin_amdgcn_readfirstlane(row - lane / LPR) < a.Hq + a.Hkv) {  // keys
          double ss = 0.0;
#pragma unroll
          for (int i = 0; i < 8; ++i) ss += (double)x[i] * x[i];
          const double inv = a.k_w ? fine_rsqrt(group_sum<LPR>(ss) / a.D + (double)a.eps) : 1.0;
          exchange(x, y);
          // (elements behind the rotated ones are selected, not turned by 0: they may be
          // infinite)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const double own = (double)x[i] * ca[i];
            const double key = (e + i < a.R ? own + (double)y[i] * cb[i] : own) * inv;
            x[i] = is_v ? x[i] : round_to_odd(key);
          }
        }
        // the whole group finds the row's scale
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, mine ? e4m3::magnitude(x[i]) : 0u);
        const uint32_t byte = e4m3::scale_byte(group_max<LPR>(top));
        if (row >= H || !mine || !mapped) continue;
        const float inv = e4m3::inverse_scale(byte);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = e4m3::codable<T>(x[i]) * inv;
        const long long head = is_v ? row - a.Hq - a.Hkv : row - a.Hq;
        uint2 w;
        w.x = e4m3::pack4(x[0], x[1], x[2], x[3]);
        w.y = e4m3::pack4(x[4], x[5], x[6], x[7]);
        *reinterpret_cast<uint2 *>((uint8_t *)(is_v ? a.vc : a.kc) + head * a.head_stride + at +
                                   e) = w;
        if (l == 0) (is_v ? a.vs : a.ks)[head * a.bs + at / a.D] = (uint8_t)byte;
      }
      if (round + 1 < rounds) load(round + 1);
    }
    return;
  }

  // this lane's cosines and sines: c[i], s[i] of element e + i, the sine with
  // the sign that its partner's value takes
  float c[8], s[8], w8[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    c[i] = 1.0f;
    s[i] = 0.0f;
  }
  angles([&](uint64_t turns, int i, bool front) {
    float cs, sn;
    angle(a, p, turns, cs, sn);
    c[i] = cs;
    s[i] = front ? -sn : sn;
    if constexpr (LAYOUT == kNeighbours) {
      c[i + 1] = cs;
      s[i + 1] = sn;
    }
  });
  if (mine) weights8<T>(a.q_w, a.w_f32, e, w8);
  for (int round = 0; round < rounds; ++round) {
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
      const int row = row0 + (round * ITER + it) * RPW;
      float x[8], y[8];
      unpack8<T>(raw[it], x);
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
      ss = group_sum<LPR>(ss);
      const float inv = a.q_w ? rsqrtf(ss / (float)a.D + a.eps) : 1.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= inv * w8[i];
      exchange(x, y);
      if (row >= H || !mine) continue;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = e + i < a.R ? x[i] * c[i] + y[i] * s[i] : x[i];
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = pack2<T>(x[2 * i], x[2 * i + 1]);
      store8(a.q_out + ((long long)t * a.Hq + row) * a.D + e, w);
    }
    if (round + 1 < rounds) load(round + 1);
  }
}

template <class T, int LPR, int LAYOUT, bool E4M3>
int launch(Args a, hipStream_t st) {
  constexpr int RPW = 64 / LPR;
  const int H = a.Hq + 2 * a.Hkv;
  const long long few = (long long)a.T * ((H + RPW - 1) / RPW);
  const int rows = E4M3 ? a.Hq : H;
  auto up = [](int n, int per) { return (n + per - 1) / per; };
  auto groups = [&](int iter, bool all) {
    a.rounds = all ? up(rows, iter * RPW) : 1;
    a.chunks = up(rows, iter * a.rounds * RPW);
    a.kv_rounds = E4M3 ? (all ? up(2 * a.Hkv, iter * RPW) : 1) : 0;
    a.kv_chunks = E4M3 ? up(2 * a.Hkv, iter * a.kv_rounds * RPW) : 0;
    return ((long long)a.T * (a.chunks + a.kv_chunks) + kWaves - 1) / kWaves;
  };
  // `few`: waves of one row a lane group.  A token's heads all in one wave where
  // that leaves 8192 waves of kIter rows' work (angles and weights are then formed
  // once a token), else kIter rows a group where that leaves 2048 waves, else one.
  // us, 48 heads of 128, one row a group / kIter rows / all heads in a wave: 504
  // tokens 10.1 / 10.6 / 14, 2000 tokens 22 / 19.6 / 20.5, 3200 tokens 36 / 27 / 24, 8149
  // tokens 104 / 73 / 58.  With 2 / 6 / 8 / 12 rows in flight: 59.5 / 59.2 / 62 / 69.
  const bool many = few >= 8192, all = few >= 8192 * kIter;
  const long long n = many ? groups(kIter, all) : groups(1, false);
  if (n * kWaves * 64 >= 1LL << 32)  // a launch's threads
    return abi::fail_arg("too many tokens and heads for one call");
  const dim3 grid((unsigned)n);
  if constexpr (E4M3) {
    if (many)
      CFA_LAUNCH("qk_norm_rope_kv", (qk_norm_rope_kv_e4m3_kernel<T, LPR, LAYOUT, kIter>),
                 grid, dim3(kWaves * 64), 0, st, a);
    else
      CFA_LAUNCH("qk_norm_rope_kv", (qk_norm_rope_kv_e4m3_kernel<T, LPR, LAYOUT, 1>),
                 grid, dim3(kWaves * 64), 0, st, a);
  } else {
    if (many)
      CFA_LAUNCH("qk_norm_rope_kv", (qk_norm_rope_kv_kernel<T, LPR, LAYOUT, kIter>),
                 grid, dim3(kWaves * 64), 0, st, a);
    else
      CFA_LAUNCH("qk_norm_rope_kv", (qk_norm_rope_kv_kernel<T, LPR, LAYOUT, 1>),
                 grid, dim3(kWaves * 64), 0, st, a);
  }
  return CFA_OK;
}

template <class T, int LPR, bool E4M3>
int launch_layout(const Args &a, int layout, hipStream_t st) {
  switch (layout) {
    case kHalf: return launch<T, LPR, kHalf, E4M3>(a, st);
    case kHalfAny: return launch<T, LPR, kHalfAny, E4M3>(a, st);
    default: return launch<T, LPR, kNeighbours, E4M3>(a, st);
  }
}

template <class T, bool E4M3>
int launch_type(const Args &a, int layout, hipStream_t st) {
  if (a.D <= 32) return launch_layout<T, 4, E4M3>(a, layout, st);
  if (a.D <= 64) return launch_layout<T, 8, E4M3>(a, layout, st);
  if (a.D <= 128) return launch_layout<T, 16, E4M3>(a, layout, st);
  return launch_layout<T, 32, E4M3>(a, layout, st);
}

}  // namespace rotary
}  // namespace cfa

extern "C" int cfa_qk_norm_rope_kv_e4m3(
    const void *q, int64_t q_stride_t, int64_t q_stride_h, const void *k, int64_t k_stride_t,
    int64_t k_stride_h, const void *v, int64_t v_stride_t, int64_t v_stride_h, int fp16,
    const int32_t *positions, int T, int B, const int32_t *cu_seqlens, int n_q_heads,
    int n_kv_heads, int head_dim, int rotary_dim, const uint64_t *turns, float factor,
    int interleaved, const void *q_norm, const void *k_norm, int norm_f32, float eps, void *q_out,
    void *k_pool, void *v_pool, uint8_t *k_scales, uint8_t *v_scales, int num_blocks,
    int num_layers, int layer, int block_size, const int32_t *block_tables, int max_blocks_per_seq,
    const int32_t *base_lens, void *stream) {
  using namespace cfa::abi;
  using namespace cfa::rotary;
  clear_error();
  if (T < 0 || B < 0 || n_q_heads <= 0 || n_kv_heads <= 0)
    return fail_arg("need T, B >= 0 and positive head counts");
  if (head_dim <= 0 || head_dim % 8 || head_dim > 256)
    return fail_arg("head_dim must be a multiple of 8, at most 256");
  if (!k_scales != !v_scales) return fail_arg("k_scales and v_scales go together");
  const bool e4m3 = k_scales != nullptr;
  if (e4m3 && head_dim % 16) return fail_arg("e4m3 pools need head_dim to be a multiple of 16");
  if (e4m3 && (((uintptr_t)k_pool | (uintptr_t)v_pool) & 15) != 0)
    return fail_arg("e4m3 pools must be 16-byte aligned");
  if (rotary_dim < 0 || rotary_dim % 2 || rotary_dim > head_dim)
    return fail_arg("rotary_dim must be even, between 0 and head_dim");
  if (num_blocks <= 0 || num_layers <= 0 || layer < 0 || layer >= num_layers || block_size <= 0 ||
      max_blocks_per_seq < 0)
    return fail_arg("bad pool geometry (num_blocks, num_layers, layer, block_size)");
  if (T == 0 || B == 0) return CFA_OK;
  if (!q || !k || !v || !positions || !q_out || !k_pool || !v_pool || !base_lens ||
      (rotary_dim > 0 && !turns) || (max_blocks_per_seq > 0 && !block_tables))
    return fail_arg("null pointer argument");
  if ((long long)T * ((n_q_heads + 2LL * n_kv_heads + 1) / 2) >= (1LL << 26))
    return fail_arg("too many tokens and heads for one call (T * heads of 2^27 and more)");
  if (!cu_seqlens && T % B) return fail_arg("without cu_seqlens T must be a multiple of B");
  Args a{};
  a.q = (const uint16_t *)q;
  a.k = (const uint16_t *)k;
  a.v = (const uint16_t *)v;
  a.q_st = q_stride_t;
  a.q_sh = q_stride_h;
  a.k_st = k_stride_t;
  a.k_sh = k_stride_h;
  a.v_st = v_stride_t;
  a.v_sh = v_stride_h;
  a.pos = positions;
  a.cu = cu_seqlens;
  a.T = T;
  a.B = B;
  a.n = T / B;
  a.Hq = n_q_heads;
  a.Hkv = n_kv_heads;
  a.D = head_dim;
  a.R = rotary_dim;
  a.turns = turns;
  a.factor = factor;
  a.q_w = q_norm;
  a.k_w = k_norm;
  a.w_f32 = norm_f32;
  a.eps = eps;
  a.q_out = (uint16_t *)q_out;
  a.kc = k_pool;
  a.vc = v_pool;
  a.ks = k_scales;
  a.vs = v_scales;
  a.num_blocks = num_blocks;
  a.max_blocks = max_blocks_per_seq;
  a.bs = block_size;
  a.block_tables = block_tables;
  a.base = base_lens;
  a.head_stride = (long long)block_size * head_dim;
  a.blk_stride = (long long)num_layers * n_kv_heads * a.head_stride;
  a.layer_off = (long long)layer * n_kv_heads * a.head_stride;
  const int layout = interleaved ? kNeighbours : (rotary_dim % 16 == 0 ? kHalf : kHalfAny);
  hipStream_t st = (hipStream_t)stream;
  if (e4m3)
    return fp16 ? launch_type<cfa::FP16, true>(a, layout, st)
                : launch_type<cfa::BF16, true>(a, layout, st);
  return fp16 ? launch_type<cfa::FP16, false>(a, layout, st)
              : launch_type<cfa::BF16, false>(a, layout, st);
}

extern "C" int cfa_qk_norm_rope_kv(
    const void *q, int64_t q_stride_t, int64_t q_stride_h, const void *k, int64_t k_stride_t,
    int64_t k_stride_h, const void *v, int64_t v_stride_t, int64_t v_stride_h, int fp16,
    const int32_t *positions, int T, int B, const int32_t *cu_seqlens, int n_q_heads,
    int n_kv_heads, int head_dim, int rotary_dim, const uint64_t *turns, float factor,
    int interleaved, const void *q_norm, const void *k_norm, int norm_f32, float eps, void *q_out,
    void *k_pool, void *v_pool, int num_blocks, int num_layers, int layer, int block_size,
    const int32_t *block_tables, int max_blocks_per_seq, const int32_t *base_lens, void *stream) {
  return cfa_qk_norm_rope_kv_e4m3(q, q_stride_t, q_stride_h, k, k_stride_t, k_stride_h, v,
                                  v_stride_t, v_stride_h, fp16, positions, T, B, cu_seqlens,
                                  n_q_heads, n_kv_heads, head_dim, rotary_dim, turns, factor,
                                  interleaved, q_norm, k_norm, norm_f32, eps, q_out, k_pool,
                                  v_pool, nullptr, nullptr, num_blocks, num_layers, layer,
                                  block_size, block_tables, max_blocks_per_seq, base_lens, stream);
}
