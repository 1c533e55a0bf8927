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
// One pass: a work-group owns a slice of the vocabulary of one sequence.  It counts
// the sequence's tokens that fall into the slice in LDS (whole numbers, so the order
// of the atomics leaves no trace), and then streams the slice of each of its rows
// through, eight logits a lane.  A bitmap says which tokens are touched at all: the
// other ones (nearly all) need no look at their counts.  The tokens on a row's path
// are at most 64, and a ballot finds those in the slice.
//
// Bound: HBM, every logit read and written once.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "abi_internal.hpp"
#include "half_types.hpp"

namespace cfa {
namespace logits {

constexpr int kNT = 256;
constexpr int kVec = 8;  // logits of a lane at a time
constexpr int kMaxNodes = 64;

struct FP32 {
  typedef float elem;
};

struct Args {
  const void *in;
  void *out;
  long long in_sb, in_sn, out_sb, out_sn;  // elements
  int B, N, V, slice, slices, per;         // rows of a sequence; tokens of a slice; rows a group
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
typedef u32x4 at_half __attribute__((aligned(2)));
typedef u32x4 at_word __attribute__((aligned(4)));

// Eight values from any element on.
template <class T>
__device__ __forceinline__ void load8(const void *p, float (&x)[kVec]) {
  if constexpr (__is_same(T, FP32)) {
    const at_word *w = reinterpret_cast<const at_word *>(p);
    const u32x4 a = w[0], b = w[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = __uint_as_float(a[i]);
      x[4 + i] = __uint_as_float(b[i]);
    }
  } else {
    const u32x4 a = *reinterpret_cast<const at_half *>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) unpack2<T>(a[i], x[2 * i], x[2 * i + 1]);
  }
}
template <class T>
__device__ __forceinline__ void store8(void *p, const float (&x)[kVec]) {
  if constexpr (__is_same(T, FP32)) {
    u32x4 a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = __float_as_uint(x[i]);
      b[i] = __float_as_uint(x[4 + i]);
    }
    at_word *w = reinterpret_cast<at_word *>(p);
    w[0] = a;
    w[1] = b;
  } else {
    u32x4 a;
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = pack2<T>(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<at_half *>(p) = a;
  }
}
template <class T>
__device__ __forceinline__ float load1(const void *p) {
  if constexpr (__is_same(T, FP32)) return *reinterpret_cast<const float *>(p);
  else return (float)*reinterpret_cast<const typename T::elem *>(p);
}

constexpr uint32_t kInPrompt = 0x80000000u;

// LDS: counts [slice] (bit 31: in the prompt), biases' numbers + 1 [slice] where
// there are biases, and the bitmap of touched tokens [slice / 32].
template <class TI, class TO>
__global__ __launch_bounds__(kNT) void adjust_logits_kernel(Args a) {
  extern __shared__ __align__(16) uint32_t lds[];
  uint32_t *const count = lds, *const bias = lds + a.slice;
  uint32_t *const touched = lds + (a.K > 0 ? 2 : 1) * a.slice;
  const int tid = threadIdx.x, lane = tid & 63;
  const int v0 = (int)(blockIdx.x % a.slices) * a.slice;
  const int rest = blockIdx.x / a.slices;
  const int parts = (a.N + a.per - 1) / a.per;
  const int b = rest / parts, i0 = rest % parts * a.per, i1 = min(a.N, i0 + a.per);
  const int vn = min(a.slice, a.V - v0);  // tokens of this slice

  const int total = a.slice * (a.K > 0 ? 2 : 1) + a.slice / 32;
  for (int i = tid * 4; i < total; i += kNT * 4)
    *reinterpret_cast<u32x4 *>(lds + i) = u32x4{0, 0, 0, 0};
  __syncthreads();
  const int len = a.history ? min(max(a.lens ? a.lens[b] : a.L, 0), a.L) : 0;
  const int prompt = a.prompts ? a.prompts[b] : 0;
  const int32_t *const tokens = a.history + (long long)b * a.L;
  for (int i = tid; i < len; i += kNT) {
    const uint32_t at = (uint32_t)tokens[i] - (uint32_t)v0;
    if (at < (uint32_t)vn) {
      if (i < prompt) atomicOr(&count[at], kInPrompt);
      else atomicAdd(&count[at], 1u);
      atomicOr(&touched[at / 32], 1u << (at % 32));
    }
  }
  for (int i = tid; i < a.K; i += kNT) {
    const uint32_t at = (uint32_t)a.bias_tokens[b * a.bias_sb + i] - (uint32_t)v0;
    if (at < (uint32_t)vn) {
      atomicMax(&bias[at], (uint32_t)i + 1);  // of one token's the last
      atomicOr(&touched[at / 32], 1u << (at % 32));
    }
  }
  const float rep = a.rep ? a.rep[b] : a.rep0, freq = a.freq ? a.freq[b] : a.freq0;
  const float pres = a.pres ? a.pres[b] : a.pres0;
  // a lane's node and its token's place in the slice
  uint32_t node_at = 0xffffffffu;
  if (a.nodes && lane < a.N) node_at = (uint32_t)a.nodes[(long long)b * a.N + lane] - (uint32_t)v0;
  const uint64_t here = __ballot(node_at < (uint32_t)vn);
  __syncthreads();

  for (int i = i0; i < i1; ++i) {
    const uint8_t *in = (const uint8_t *)a.in +
                        (b * a.in_sb + i * a.in_sn + v0) * (long long)sizeof(typename TI::elem);
    uint8_t *out = (uint8_t *)a.out +
                   (b * a.out_sb + i * a.out_sn + v0) * (long long)sizeof(typename TO::elem);
    const uint64_t path = a.nodes ? a.mask[b * a.mask_sb + i] & here : 0;
    const uint8_t *allowed = nullptr;  // a byte for eight tokens
    if (a.allowed) {
      const long long row = (long long)b * a.N + i;
      const long long m = a.index ? a.index[row] : row;
      if (m >= 0 && m < a.masks)
        allowed = (const uint8_t *)(a.allowed + m * a.words) + v0 / 8;
    }
    for (int p = tid * kVec; p < vn; p += kNT * kVec) {
      uint32_t look = (touched[p / 32] >> (p % 32)) & 255u;
      uint32_t ok = allowed ? allowed[p / 8] : 255u;
      for (uint64_t left = path; left; left &= left - 1) {
        const uint32_t at = __builtin_amdgcn_readlane(node_at, __ffsll((unsigned long long)left) - 1) - (uint32_t)p;
        if (at < kVec) look |= 1u << at;
      }
      if (a.in_place && look == 0 && ok == 255u) continue;
      const int n = min(kVec, vn - p);
      float x[kVec];
      if (n == kVec) {
        load8<TI>(in + p * (int)sizeof(typename TI::elem), x);
      } else {
        for (int k = 0; k < kVec; ++k)
          x[k] = k < n ? load1<TI>(in + (p + k) * (int)sizeof(typename TI::elem)) : 0.0f;
      }
      if (look) {
#pragma unroll
        for (int k = 0; k < kVec; ++k) {
          if (!(look >> k & 1)) continue;
          const uint32_t w = count[p + k];
          uint32_t c = w & ~kInPrompt;
          for (uint64_t left = path; left; left &= left - 1)
            c += __builtin_amdgcn_readlane(node_at, __ffsll((unsigned long long)left) - 1) == (uint32_t)(p + k);
          if (w | c) x[k] = x[k] > 0.0f ? x[k] / rep : x[k] * rep;
          if (c) x[k] -= freq * (float)c + pres;
          const uint32_t which = a.K > 0 ? bias[p + k] : 0;
          if (which) x[k] += a.bias_values[b * a.bias_sb + which - 1];
        }
      }
#pragma unroll
      for (int k = 0; k < kVec; ++k) x[k] = ok >> k & 1 ? x[k] : -INFINITY;
      if (n == kVec) {
        store8<TO>(out + p * (int)sizeof(typename TO::elem), x);
      } else {
        for (int k = 0; k < n; ++k)
          reinterpret_cast<typename TO::elem *>(out)[p + k] = (typename TO::elem)x[k];
      }
    }
  }
}

template <class TI, class TO>
int launch(const Args &a, hipStream_t st) {
  const long long parts = (a.N + a.per - 1) / a.per;
  const size_t lds = (size_t)a.slice * (a.K > 0 ? 8 : 4) + a.slice / 8;
  CFA_LAUNCH("adjust_logits", (adjust_logits_kernel<TI, TO>),
             dim3((unsigned)(a.slices * parts * a.B)), dim3(kNT), lds, st, a);
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
  if (!repetition && !(repetition0 > 0.0f)) return fail_arg("repetition must be positive");
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
  a.slice = 4096;
  a.slices = (V + a.slice - 1) / a.slice;
  a.per = 8;
  const long long groups = (long long)a.slices * ((N + a.per - 1) / a.per) * B;
  if (groups >= 1LL << 24) return fail_arg("too many rows for one call");
  hipStream_t st = (hipStream_t)stream;
  switch (type) {
    case 0: return launch<FP32, FP32>(a, st);
    case 1: return f32 ? launch<cfa::BF16, FP32>(a, st) : launch<cfa::BF16, cfa::BF16>(a, st);
    default: return f32 ? launch<cfa::FP16, FP32>(a, st) : launch<cfa::FP16, cfa::FP16>(a, st);
  }
}
