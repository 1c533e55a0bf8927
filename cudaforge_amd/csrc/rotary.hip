// rotary.hip -- RMSNorm of every q and k head, rotary positions and the write
// of k and v into the paged cache, one pass over a QKV projection.
//
// For token t and q or k head x of D elements (fp32 arithmetic, one rounding):
//   y = x * rsqrt(mean(x^2) + eps) * w                 (w given; else y = x)
//   pairs (a, b) of the first R elements, at angle p_t f_i (position times the
//   pair's frequency), as halves (i, i + R/2) or as neighbours (2i, 2i + 1):
//   (a, b) -> factor * (a cos - b sin, b cos + a sin)
// v is copied.  q goes to q_out [T, Hq, D], k and v to the sequence's slots
// base[b] + j of pool[block][layer][kv_head][slot][D].
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
// tokens 7 us, 8 tokens 5.
#include <hip/hip_runtime.h>

#include "abi_internal.hpp"
#include "half_types.hpp"

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
  uint16_t *q_out, *kc, *vc;
  int num_blocks, max_blocks, bs;
  const int32_t *block_tables, *base;
  long long blk_stride, layer_off, head_stride;
  int chunks, rounds;  // waves a token; rounds of rows a wave
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

// The sequence b and the place j in it of token t; false where t belongs to
// none (in front of the first, or behind the last).
__device__ __forceinline__ bool place(const Args &a, int t, int lane, int &b, int &j) {
  if (!a.cu) {
    b = t / a.n;
    j = t - b * a.n;
    return true;
  }
  b = 0;  // ends at or before t
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const bool ended = b0 + lane < a.B && a.cu[b0 + lane + 1] <= t;
    b += __popcll(__ballot(ended));
  }
  if (b >= a.B) return false;
  j = t - a.cu[b];
  return j >= 0;
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
  if (!place(a, t, lane, b, j)) return;
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
        store8((is_v ? a.vc + (row - a.Hq - a.Hkv) * a.head_stride
                          : a.kc + (row - a.Hq) * a.head_stride) + at + e, w);
    }
    if (round + 1 < a.rounds) load(round + 1);
  }
}

template <class T, int LPR, int LAYOUT>
int launch(Args a, hipStream_t st) {
  constexpr int RPW = 64 / LPR;
  const int H = a.Hq + 2 * a.Hkv;
  const long long few = (long long)a.T * ((H + RPW - 1) / RPW);
  auto grid = [&](int iter, int rounds) {
    a.rounds = rounds;
    a.chunks = (H + iter * rounds * RPW - 1) / (iter * rounds * RPW);
    return dim3((unsigned)(((long long)a.T * a.chunks + kWaves - 1) / kWaves));
  };
  // `few`: waves of one row a lane group.  A token's heads all in one wave where
  // that leaves 8192 waves of kIter rows' work (angles and weights are then formed
  // once a token), else kIter rows a group where that leaves 2048 waves, else one.
  // us, 48 heads of 128, one row a group / kIter rows / all heads in a wave: 504
  // tokens 10.1 / 10.6 / 14, 2000 tokens 22 / 19.6 / 20.5, 3200 tokens 36 / 27 / 24, 8149
  // tokens 104 / 73 / 58.  With 2 / 6 / 8 / 12 rows in flight: 59.5 / 59.2 / 62 / 69.
  if (few >= 8192 * kIter) {
    const int all = (H + kIter * RPW - 1) / (kIter * RPW);
    CFA_LAUNCH("qk_norm_rope_kv", (qk_norm_rope_kv_kernel<T, LPR, LAYOUT, kIter>),
               grid(kIter, all), dim3(kWaves * 64), 0, st, a);
  } else if (few >= 8192) {
    CFA_LAUNCH("qk_norm_rope_kv", (qk_norm_rope_kv_kernel<T, LPR, LAYOUT, kIter>),
               grid(kIter, 1), dim3(kWaves * 64), 0, st, a);
  } else {
    CFA_LAUNCH("qk_norm_rope_kv", (qk_norm_rope_kv_kernel<T, LPR, LAYOUT, 1>), grid(1, 1),
               dim3(kWaves * 64), 0, st, a);
  }
  return CFA_OK;
}

template <class T, int LPR>
int launch_layout(const Args &a, int layout, hipStream_t st) {
  switch (layout) {
    case kHalf: return launch<T, LPR, kHalf>(a, st);
    case kHalfAny: return launch<T, LPR, kHalfAny>(a, st);
    default: return launch<T, LPR, kNeighbours>(a, st);
  }
}

template <class T>
int launch_type(const Args &a, int layout, hipStream_t st) {
  if (a.D <= 32) return launch_layout<T, 4>(a, layout, st);
  if (a.D <= 64) return launch_layout<T, 8>(a, layout, st);
  if (a.D <= 128) return launch_layout<T, 16>(a, layout, st);
  return launch_layout<T, 32>(a, layout, st);
}

}  // namespace rotary
}  // namespace cfa

extern "C" int cfa_qk_norm_rope_kv(
    const void *q, int64_t q_stride_t, int64_t q_stride_h, const void *k, int64_t k_stride_t,
    int64_t k_stride_h, const void *v, int64_t v_stride_t, int64_t v_stride_h, int fp16,
    const int32_t *positions, int T, int B, const int32_t *cu_seqlens, int n_q_heads,
    int n_kv_heads, int head_dim, int rotary_dim, const uint64_t *turns, float factor,
    int interleaved, const void *q_norm, const void *k_norm, int norm_f32, float eps, void *q_out,
    void *k_pool, void *v_pool, int num_blocks, int num_layers, int layer, int block_size,
    const int32_t *block_tables, int max_blocks_per_seq, const int32_t *base_lens, void *stream) {
  using namespace cfa::abi;
  using namespace cfa::rotary;
  clear_error();
  if (T < 0 || B < 0 || n_q_heads <= 0 || n_kv_heads <= 0)
    return fail_arg("need T, B >= 0 and positive head counts");
  if (head_dim <= 0 || head_dim % 8 || head_dim > 256)
    return fail_arg("head_dim must be a multiple of 8, at most 256");
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
  a.kc = (uint16_t *)k_pool;
  a.vc = (uint16_t *)v_pool;
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
  return fp16 ? launch_type<cfa::FP16>(a, layout, st)
              : launch_type<cfa::BF16>(a, layout, st);
}
