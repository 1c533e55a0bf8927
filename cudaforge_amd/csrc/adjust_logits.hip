// adjust_logits.hip -- logits on their way to the sampler or the verification:
// penalties of repeated tokens, biases and grammar masks, for single rows and for
// the nodes of a draft tree (each behind its own path).
//
// Row i of sequence b, token v, in fp32 with one rounding at the end:
//   c = times v stands in the sequence's generated tokens and on the row's path
//   x = x > 0 ? x / r : x r      where v stands there or in the prompt
//   x = x - (f c + p [c > 0]) + bias(v)
//   x = -inf                     where the row's mask has no bit for v
//
// A work-group owns a slice of the vocabulary of one sequence.  It counts the
// sequence's tokens that fall into the slice in LDS (whole numbers, so the order of
// the atomics leaves no trace) and lists those that occur.  Then, row by row, it
// streams the slice through with the mask alone, and a thread for each listed token
// (and for each token on the row's path) computes that one and stores it over what
// was streamed: few tokens of a slice are touched, but some in nearly every wave's
// vector, which would take all of them through the penalties.
//
// Bound: HBM, every logit read and written once, and in front of that each
// work-group's count (4 us for 2000 tokens, while nothing streams: 8192 tokens a slice
// keep it to sixteen of a vocabulary of 128256).  us a call, bf16: 64 rows of 128256
// alone 7.3, behind 2000 tokens each 11.3, and with biases and masks 13.5; 504 nodes of
// 8 trees to fp32 (388 MB) 71, behind 2000 tokens 88 (4.4 TB/s; a copy of the same
// tensors takes 67), behind 8000 108 (145 if they are all different).  Each group counts
// all of its sequence's history, so that long ones cost: behind 30000 and 100000 such
// tokens one row 19 and 49, 64 rows 44 and 111, the trees 218 and 427.  With the
// penalties in the streaming loop, instead of behind it for the listed tokens, the rows
// took 17.3 and the trees 90.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "abi_internal.hpp"
#include "half_types.hpp"
#include "lds_dma.hpp"

namespace cfa {
namespace logits {

constexpr int NT = 512;  // threads of a work-group
constexpr int kVec = 8;  // logits of a lane at a time
constexpr int VECS = 2;  // of those a lane has in a row
constexpr int kSlice = VECS * NT * kVec;  // tokens of a slice
constexpr int kMaxNodes = 64;
constexpr int kFewBiases = 256;  // biases that are listed and searched, not tabled

struct FP32 {
  typedef float elem;
};

struct Args {
  const void *in;
  void *out;
  long long in_sb, in_sn, out_sb, out_sn;  // elements
  int B, N, V, slices, per;                // rows of a sequence; slices of a row; rows a group
  const int32_t *history, *lens, *prompts;
  int L;
  const float *rep, *freq, *pres;
  float rep0, freq0, pres0;
  const int32_t *nodes;  // [B, N] or null
  const uint64_t *mask;
  long long mask_sb;
  const int32_t *bias_tokens;
  const float *bias_values;
  long long bias_sb;
  int K;
  const uint32_t *allowed;
  const int32_t *index;
  int words, masks;
  int in_place;
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 at_half __attribute__((aligned(2)));
typedef u32x4 at_word __attribute__((aligned(4)));
typedef i32x4 at_token __attribute__((aligned(4)));

// Eight values as they lie in memory, from any element on.
template <class T>
struct Raw {
  u32x4 w[sizeof(typename T::elem) / 2];
};
template <class T>
__device__ __forceinline__ void fetch8(const void *p, Raw<T> &r) {
  if constexpr (__is_same(T, FP32)) {
    r.w[0] = reinterpret_cast<const at_word *>(p)[0];
    r.w[1] = reinterpret_cast<const at_word *>(p)[1];
  } else {
    r.w[0] = *reinterpret_cast<const at_half *>(p);
  }
}
// (past the caches: 64 rows of 128256 in bf16 8.5 -> 7.3 us, without anything to do)
template <class T>
__device__ __forceinline__ void store8(void *p, const Raw<T> &r) {
  if constexpr (__is_same(T, FP32)) {
    __builtin_nontemporal_store(r.w[0], reinterpret_cast<at_word *>(p));
    __builtin_nontemporal_store(r.w[1], reinterpret_cast<at_word *>(p) + 1);
  } else {
    __builtin_nontemporal_store(r.w[0], reinterpret_cast<at_half *>(p));
  }
}
// The eight in the output's type, -inf where `ok` has no bit (bits are kept where
// the type is).
template <class TI, class TO>
__device__ __forceinline__ void masked8(const Raw<TI> &r, uint32_t ok, Raw<TO> &y) {
  if constexpr (__is_same(TO, FP32)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (__is_same(TI, FP32)) {
        y.w[0][i] = r.w[0][i];
        y.w[1][i] = r.w[1][i];
      } else {
        float lo, hi;
        unpack2<TI>(r.w[0][i], lo, hi);
        y.w[i / 2][2 * (i % 2)] = __float_as_uint(lo);
        y.w[i / 2][2 * (i % 2) + 1] = __float_as_uint(hi);
      }
    }
    if (ok != 255u)
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        if (!(ok >> i & 1)) y.w[i / 4][i % 4] = 0xff800000u;
  } else {
    y.w[0] = r.w[0];
    constexpr uint32_t inf = __is_same(TO, BF16) ? 0xff80u : 0xfc00u;
    if (ok != 255u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!(ok >> (2 * i) & 1)) y.w[0][i] = (y.w[0][i] & 0xffff0000u) | inf;
        if (!(ok >> (2 * i + 1) & 1)) y.w[0][i] = (y.w[0][i] & 0xffffu) | inf << 16;
      }
  }
}

constexpr uint32_t kInPrompt = 0x80000000u;

// LDS: counts [slice] (bit 31: in the prompt), with many biases their numbers + 1
// [slice], the bitmap of touched tokens [slice / 32], how many tokens and biases are
// listed [4], few biases' (place << 16 | number) [kFewBiases], and the touched tokens'
// places, 16 bits each.
static size_t lds_bytes(int L, int K) {
  const long long listed = std::min<long long>((long long)L + K, kSlice);
  return (size_t)kSlice * (K > kFewBiases ? 8 : 4) + kSlice / 8 + 16 +
         (K > 0 && K <= kFewBiases ? kFewBiases * 4 : 0) + 2 * listed;
}

// A lane's vectors of a row are loaded a row ahead, those of the first row in front of
// the counting.
template <class TI, class TO>
__global__ __launch_bounds__(NT) void adjust_logits_kernel(Args a) {
  constexpr int kIn = sizeof(typename TI::elem), kOut = sizeof(typename TO::elem);
  extern __shared__ __align__(16) uint32_t lds[];
  const bool many = a.K > kFewBiases;
  uint32_t *const count = lds, *const bias = lds + kSlice;
  uint32_t *const touched = lds + (many ? 2 : 1) * kSlice;
  uint32_t *const listed = touched + kSlice / 32;
  uint32_t *const biases = listed + 4;
  uint16_t *const list =
      reinterpret_cast<uint16_t *>(biases + (a.K > 0 && !many ? kFewBiases : 0));
  const int tid = threadIdx.x, lane = tid & 63;
  const int v0 = (int)(blockIdx.x % a.slices) * kSlice;
  const int rest = blockIdx.x / a.slices;
  const int parts = (a.N + a.per - 1) / a.per;
  const int b = rest / parts, i0 = rest % parts * a.per, i1 = min(a.N, i0 + a.per);
  const int vn = min(kSlice, a.V - v0);  // tokens of this slice

  Raw<TI> raw[VECS];
  uint32_t allow[VECS];  // a bit for each token of a vector
  const uint8_t *next_bits = nullptr;
  auto row_in = [&](int i) {
    return (const uint8_t *)a.in + (b * a.in_sb + i * a.in_sn + v0) * (long long)kIn;
  };
  auto fetch = [&](int i) {
    next_bits = nullptr;
    if (a.allowed) {
      const long long row = (long long)b * a.N + i;
      const long long m = a.index ? a.index[row] : row;
      if (m >= 0 && m < a.masks)
        next_bits = (const uint8_t *)(a.allowed + m * a.words) + v0 / 8;
    }
#pragma unroll
    for (int u = 0; u < VECS; ++u) {
      const int p = (u * NT + tid) * kVec;
      if (p + kVec <= vn && !a.in_place) fetch8<TI>(row_in(i) + p * kIn, raw[u]);
      allow[u] = next_bits && p < vn ? next_bits[p / 8] : 255u;
    }
  };
  // everything that the first row and the counting wait for is asked for at once (of
  // the history its first kAhead * NT * 4 tokens, before it is known how many count)
  const int32_t *const tokens = a.history + (long long)b * a.L;
  constexpr int kAhead = 2;
  const int fours = a.L / 4;
  i32x4 t[kAhead];
  auto ask = [&](int j) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (j + u * NT < fours)
        t[u] = *reinterpret_cast<const at_token *>(tokens + 4 * (j + u * NT));
  };
  ask(tid);
  fetch(i0);
  const int len = a.history ? min(max(a.lens ? a.lens[b] : a.L, 0), a.L) : 0;
  const int prompt = a.prompts ? a.prompts[b] : 0;

  const bool any = a.history || a.K > 0;  // something may be listed
  if (any) {
    const int total = kSlice * (many ? 2 : 1) + kSlice / 32 + 4;
    for (int i = tid * 4; i < total; i += NT * 4)
      *reinterpret_cast<u32x4 *>(lds + i) = u32x4{0, 0, 0, 0};
    __syncthreads();
  }
  auto enlist = [&](uint32_t at) {
    const uint32_t bit = 1u << (at % 32);
    if (!(atomicOr(&touched[at / 32], bit) & bit)) list[atomicAdd(listed, 1u)] = (uint16_t)at;
  };
  auto counted = [&](int32_t token, int i) {
    const uint32_t at = (uint32_t)token - (uint32_t)v0;
    if (at < (uint32_t)vn && i < len) {
      if (i < prompt) atomicOr(&count[at], kInPrompt);
      else atomicAdd(&count[at], 1u);
      enlist(at);
    }
  };
  for (int j = tid; j < fours; j += NT * kAhead) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (j + u * NT < fours)
#pragma unroll
        for (int k = 0; k < 4; ++k) counted(t[u][k], 4 * (j + u * NT) + k);
    ask(j + NT * kAhead);
  }
  if (tid < (a.L & 3)) counted(tokens[4 * fours + tid], 4 * fours + tid);
  const int32_t *const bias_tokens = a.bias_tokens + b * a.bias_sb;
  const float *const bias_values = a.bias_values + b * a.bias_sb;
  for (int i = tid; i < a.K; i += NT) {
    const uint32_t at = (uint32_t)bias_tokens[i] - (uint32_t)v0;
    if (at < (uint32_t)vn) {
      if (many) atomicMax(&bias[at], (uint32_t)i + 1);
      else biases[atomicAdd(listed + 1, 1u)] = at << 16 | (uint32_t)i;
      enlist(at);
    }
  }
  const float rep = a.rep ? a.rep[b] : a.rep0, freq = a.freq ? a.freq[b] : a.freq0;
  const float pres = a.pres ? a.pres[b] : a.pres0;
  // a lane's node and its token's place in the slice
  uint32_t node_at = 0xffffffffu;
  if (a.nodes && lane < a.N) node_at = (uint32_t)a.nodes[(long long)b * a.N + lane] - (uint32_t)v0;
  const uint64_t here = __ballot(node_at < (uint32_t)vn);
  int n_list = 0, n_biases = 0;
  if (any) {
    __syncthreads();
    n_list = listed[0];
    n_biases = listed[1];
  }

  for (int i = i0; i < i1; ++i) {
    uint8_t *out = (uint8_t *)a.out + (b * a.out_sb + i * a.out_sn + v0) * (long long)kOut;
    const uint64_t path = a.nodes ? a.mask[b * a.mask_sb + i] & here : 0;
    const uint8_t *const bits = next_bits;
    Raw<TI> now[VECS];
    uint32_t ok[VECS];
#pragma unroll
    for (int u = 0; u < VECS; ++u) {
      now[u] = raw[u];
      ok[u] = allow[u];
    }
    if (i + 1 < i1) fetch(i + 1);
#pragma unroll
    for (int u = 0; u < VECS; ++u) {
      const int p = (u * NT + tid) * kVec, n = min(kVec, vn - p);
      if (n <= 0 || (a.in_place && ok[u] == 255u)) continue;
      if (n == kVec) {
        if (a.in_place) fetch8<TI>(row_in(i) + p * kIn, now[u]);
        Raw<TO> y;
        masked8<TI, TO>(now[u], ok[u], y);
        store8<TO>(out + p * kOut, y);
      } else {
        for (int k = 0; k < n; ++k) {
          const auto x = reinterpret_cast<const typename TI::elem *>(row_in(i))[p + k];
          reinterpret_cast<typename TO::elem *>(out)[p + k] =
              ok[u] >> k & 1 ? (typename TO::elem)x : (typename TO::elem)(-INFINITY);
        }
      }
    }
    if (n_list == 0 && path == 0) continue;
    // the row is stored, and has arrived: what follows is stored over parts of it
    wait_vmcnt<0>();
    __syncthreads();
    // the listed tokens, and behind them those on the path (each once, and not the
    // listed ones)
    for (int e = tid; e < n_list + (path ? a.N : 0); e += NT) {
      uint32_t at;
      bool mine = true;
      if (e < n_list) {
        at = list[e];
      } else {
        const int node = e - n_list;
        mine = path >> node & 1;
        at = mine ? (uint32_t)a.nodes[(long long)b * a.N + node] - (uint32_t)v0 : 0u;
        mine = mine && !(any && touched[at / 32] >> (at % 32) & 1);
        for (uint64_t left = path & ((1ull << node) - 1); left; left &= left - 1)
          mine = mine && (uint32_t)a.nodes[(long long)b * a.N + __ffsll((unsigned long long)left) -
                                           1] - (uint32_t)v0 != at;
      }
      if (!mine || (bits && !(bits[at / 8] >> (at % 8) & 1))) continue;
      const uint32_t w = any ? count[at] : 0;
      uint32_t c = w & ~kInPrompt;
      for (uint64_t left = path; left; left &= left - 1)
        c += __builtin_amdgcn_readlane(node_at, __ffsll((unsigned long long)left) - 1) == at;
      float x = (float)reinterpret_cast<const typename TI::elem *>(row_in(i))[at];
      if (w | c) x = x > 0.0f ? x / rep : x * rep;
      if (c) x -= freq * (float)c + pres;
      if (many) {
        if (const uint32_t which = bias[at]) x += bias_values[which - 1];
      } else {
        int last = -1;
        for (int i = 0; i < n_biases; ++i)
          if (biases[i] >> 16 == at) last = max(last, (int)(biases[i] & 0xffffu));
        if (last >= 0) x += bias_values[last];
      }
      reinterpret_cast<typename TO::elem *>(out)[at] = (typename TO::elem)x;
    }
  }
}

template <class TI, class TO>
int launch(const Args &a, unsigned groups, hipStream_t st) {
  CFA_LAUNCH("adjust_logits", (adjust_logits_kernel<TI, TO>), dim3(groups), dim3(NT),
             lds_bytes(a.L, a.K), st, a);
  return CFA_OK;
}

}  // namespace logits
}  // namespace cfa

extern "C" int cfa_adjust_logits(
    const void *logits, int64_t stride_b, int64_t stride_n, int type, int B, int N, int V,
    const int32_t *history, const int32_t *history_lens, const int32_t *prompt_lens, int L,
    const float *repetition, float repetition0, const float *frequency, float frequency0,
    const float *presence, float presence0, const int32_t *node_tokens, const uint64_t *tree_mask,
    int64_t tree_mask_stride_b, const int32_t *bias_tokens, const float *bias_values,
    int64_t bias_stride_b, int K, const int32_t *allowed, int words, int masks,
    const int32_t *allowed_index, void *out, int64_t out_stride_b, int64_t out_stride_n,
    int out_f32, void *stream) {
  using namespace cfa::abi;
  using namespace cfa::logits;
  clear_error();
  if (B < 0 || N < 0 || V <= 0 || L < 0 || K < 0)
    return fail_arg("need B, N, L, K >= 0 and V > 0");
  if (type < 0 || type > 2) return fail_arg("type must be 0 (fp32), 1 (bf16) or 2 (fp16)");
  if (node_tokens && N > kMaxNodes) return fail_arg("at most 64 tree nodes");
  if (!node_tokens != !tree_mask) return fail_arg("node_tokens and tree_mask go together");
  if (!repetition && !(repetition0 > 0.0f && std::isfinite(repetition0)))
    return fail_arg("repetition must be positive and finite");
  if ((!frequency && !std::isfinite(frequency0)) || (!presence && !std::isfinite(presence0)))
    return fail_arg("frequency and presence must be finite");
  if (allowed && ((long long)words * 32 < V || masks < 0))
    return fail_arg("allowed needs a bit for every token");
  if (B == 0 || N == 0) return CFA_OK;
  if (!logits || !out || (L > 0 && !history) || (K > 0 && (!bias_tokens || !bias_values)))
    return fail_arg("null pointer argument");
  Args a{};
  a.in = logits;
  a.out = out;
  a.in_sb = stride_b;
  a.in_sn = stride_n;
  a.out_sb = out_stride_b;
  a.out_sn = out_stride_n;
  a.B = B;
  a.N = N;
  a.V = V;
  a.history = L > 0 ? history : nullptr;
  a.lens = history_lens;
  a.prompts = prompt_lens;
  a.L = L;
  a.rep = repetition;
  a.rep0 = repetition0;
  a.freq = frequency;
  a.freq0 = frequency0;
  a.pres = presence;
  a.pres0 = presence0;
  a.nodes = node_tokens;
  a.mask = tree_mask;
  a.mask_sb = tree_mask_stride_b;
  a.bias_tokens = bias_tokens;
  a.bias_values = bias_values;
  a.bias_sb = bias_stride_b;
  a.K = K;
  a.allowed = (const uint32_t *)allowed;
  a.index = allowed_index;
  a.words = words;
  a.masks = masks;
  const bool f32 = type == 0 || out_f32;
  a.in_place = out == logits && (type == 0) == f32 && out_stride_b == stride_b &&
               out_stride_n == stride_n;
  a.slices = (int)(((long long)V + kSlice - 1) / kSlice);
  // Two rows of a sequence share a count where that leaves eight work-groups a CU (which
  // holds four at once).  us with 1 / 2 / 4 rows: 8 trees of 63 nodes behind
  // 2000 tokens 96 / 90 / 97, behind 8000 120 / 108 / 116; of 8 nodes 13.9 / 14.5 / 16.0.
  a.per = L > 0 && (long long)a.slices * N * B >= 16 * (long long)device_cu_count() ? 2 : 1;
  const long long groups = (long long)a.slices * ((N + a.per - 1) / a.per) * B;
  if (groups >= 1LL << 22) return fail_arg("too many rows for one call");
  hipStream_t st = (hipStream_t)stream;
  const unsigned g = (unsigned)groups;
  switch (type) {
    case 0: return launch<FP32, FP32>(a, g, st);
    case 1: return f32 ? launch<cfa::BF16, FP32>(a, g, st) : launch<cfa::BF16, cfa::BF16>(a, g, st);
    default: return f32 ? launch<cfa::FP16, FP32>(a, g, st) : launch<cfa::FP16, cfa::FP16>(a, g, st);
  }
}
