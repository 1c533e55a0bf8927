// sample_rows.hip -- draws from rows of logits, each row with a temperature,
// top-k, top-p and min-p of its own (cfa_sample_rows).
//
// With x a row, T its temperature and M its maximum:
//   w_i = exp((x_i - M) / T),  Z = sum w_i
// in the order of falling x (equal values: lower index first) the first n
// tokens are kept, those with
//   rank < top_k,  mass in front of it < top_p Z,  w >= min_p
// (rank 0 always), and u in [0, 1) draws the first kept index whose kept mass
// up to and with itself exceeds u times the kept mass.  T <= 0 keeps rank 0.
//
// The result is a whole number, decided by comparisons of sums over 10^5
// tokens: fp32 sums (2^-24 each) would flip about one draw in a hundred.
// Weights are therefore formed in fp64 and kept as fractions of 36 bits of a
// power of two near their slice's largest (2^-37 of it off at most, where fp32
// sums of a row are off by 2^-24): sums of whole numbers are exact whatever
// their order, so the histograms' atomics leave the same bits every time, and
// equal weights have exact multiples.
//
// Two launches (three with probabilities):
//  1. slice_kernel, a work-group per 8192 tokens: the slice's maximum, then a
//     histogram of counts and masses over bins of 1/16 octave of weight.  The
//     bins lie on one grid of x / T, so that slices' histograms add up with a
//     shift, and the maximum of the row is not needed first.
//  2. row_kernel, a work-group per row: adds the histograms, finds the bin that
//     holds the end of the kept tokens, lists its tokens (one pass over the
//     row, from cache) and selects among them by radix, to the exact token;
//     then each draw's slice from the slices' kept masses, and the token by a
//     scan of that slice.
// Bound: the first launch by vector arithmetic, the weights' in fp64 above all (64
// bf16 rows of 128256: 16.4 us, 1.0 TB/s; 72 fp32 rows 19.3 us, 1.9 TB/s; the vector
// units issue in 92 and 90% of the cycles of busy CUs, LDS is used in 33%), the second
// by one CU's reading of its row (40 to 85 GB/s) and its dependent phases (31.6 and
// 36.9 us, on 64 and 72 of 256 CUs, vector units 57 and 51%; one row of 32000 15.4),
// the probabilities by HBM (72 rows 12.9 us, 5.7 TB/s).
#include <hip/hip_runtime.h>

#include "abi_internal.hpp"
#include "half_types.hpp"
#include "row_codes.hpp"

namespace cfa {
namespace rows {

constexpr int kNT = 1024;
constexpr int kPer = 8;              // consecutive tokens of a thread
constexpr int kSlice = kNT * kPer;   // tokens of a slice
constexpr int kMaxSlices = 128;      // V <= 2^20
constexpr int kBins = 512;           // 32 octaves, the last bin takes the rest
constexpr int kDigits = 1024;        // radix of the selection inside a bin
constexpr int kList = 8192;          // tokens of a bin that fit LDS
constexpr int kWaveList = kList / (kNT / 64);
constexpr int kFew = 64;             // tokens that one wave ranks by itself
constexpr int kFrac = 36;            // fraction bits of a weight (below 2)
constexpr int kSumBits = 50;         // 8192 weights; a bin's count lies above their sum

struct Args {
  const void *rows;
  long long stride;
  int R, V, draws, slices;
  const float *temp, *top_p, *min_p;  // [R] or null: the scalar
  const int32_t *top_k;
  float temp0, top_p0, min_p0;
  int top_k0;
  const float *u;  // [R, draws]
  int32_t *tokens;
  float *probs;
  // workspace
  float *smax;               // [R, slices]
  unsigned long long *hist;  // [R, slices, kBins]: count << kSumBits | mass
  struct Kept *kept;         // [R]
};

// What row_kernel leaves for the probabilities.
struct Kept {
  double c, top, scale;  // bins per unit of x; bin of 2^0; 1 / kept mass
  uint32_t key;          // kept: a larger code, or this one up to index `last`
  int last;
};

template <int TYPE>
__device__ __forceinline__ float load1(const Args &a, long long row, int i) {
  if constexpr (TYPE == kF32) {
    return Code<TYPE>::clean(reinterpret_cast<const float *>(a.rows)[row * a.stride + i]);
  } else {
    const uint16_t v = reinterpret_cast<const uint16_t *>(a.rows)[row * a.stride + i];
    float lo, hi;
    if constexpr (TYPE == kBF16) unpack2<BF16>(v, lo, hi);
    else unpack2<FP16>(v, lo, hi);
    return Code<TYPE>::clean(lo);
  }
}

// Tokens i .. i + 7 of a row as they are (all of them in the row), by 16-byte loads
// at any element: rows of an odd length begin anywhere (50257 fp32 tokens by single
// loads 41 us in the second launch, against 20 now).
template <int TYPE>
struct Raw {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  typedef u32x4 at_element __attribute__((aligned(2)));
  uint4 v[TYPE == kF32 ? 2 : 1];
  __device__ __forceinline__ void load(const Args &a, long long row, int i) {
    const char *p = reinterpret_cast<const char *>(a.rows) +
                    (row * a.stride + i) * (TYPE == kF32 ? 4 : 2);
#pragma unroll
    for (int k = 0; k < (TYPE == kF32 ? 2 : 1); ++k) {
      const u32x4 w = reinterpret_cast<const at_element *>(p)[k];
      v[k] = make_uint4(w.x, w.y, w.z, w.w);
    }
  }
  // A value's bits where most() has a word's upper ones.
  static __device__ __forceinline__ int word(float x) {
    return TYPE == kFP16 ? (int)pack1<FP16>(x) << 16 : __float_as_int(x);
  }
  // The largest of its values' bits as whole numbers (of 16-bit values, with the
  // lower neighbour's behind them: no less than their own).
  __device__ __forceinline__ int most() const {
    const int *w = reinterpret_cast<const int *>(v);
    int m = w[0];
#pragma unroll
    for (int k = 0; k < (TYPE == kF32 ? 8 : 4); ++k) {
      m = max(m, w[k]);
      if constexpr (TYPE != kF32) m = max(m, w[k] << 16);
    }
    return m;
  }
  __device__ __forceinline__ void get(float (&x)[kPer]) const {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(v);
#pragma unroll
    for (int k = 0; k < kPer / (TYPE == kF32 ? 1 : 2); ++k) {
      if constexpr (TYPE == kF32) x[k] = __uint_as_float(w[k]);
      else if constexpr (TYPE == kBF16) unpack2<BF16>(w[k], x[2 * k], x[2 * k + 1]);
      else unpack2<FP16>(w[k], x[2 * k], x[2 * k + 1]);
    }
  }
};

// Tokens i .. i + 7 of a row (-inf behind its end).
template <int TYPE>
__device__ __forceinline__ void load8(const Args &a, long long row, int i, float (&x)[kPer]) {
  if (i + kPer <= a.V) {
    Raw<TYPE> v;
    v.load(a, row, i);
    v.get(x);
#pragma unroll
    for (int k = 0; k < kPer; ++k) x[k] = Code<TYPE>::clean(x[k]);
  } else {
#pragma unroll
    for (int k = 0; k < kPer; ++k) x[k] = i + k < a.V ? load1<TYPE>(a, row, i + k) : -INFINITY;
  }
}

// A row's settings.
struct Rule {
  double c;      // kSub log2(e) / T: bins per unit of x
  double p;      // top_p, or above 1: off
  double t, m;   // temperature, min_p (0: off)
  uint32_t k;    // top_k (all ones: off)
};
__device__ __forceinline__ Rule rule_of(const Args &a, int r) {
  const float t = a.temp ? a.temp[r] : a.temp0;
  const float p = a.top_p ? a.top_p[r] : a.top_p0;
  const float m = a.min_p ? a.min_p[r] : a.min_p0;
  const int k = a.top_k ? a.top_k[r] : a.top_k0;
  Rule q;
  const bool greedy = !(t > 0.0f);
  q.t = greedy ? 1.0 : (double)fminf(t, FLT_MAX);
  q.c = kSub * 1.4426950408889634074 / q.t;
  q.p = !greedy && p < 1.0f ? (double)p : 2.0;
  q.m = !greedy && m > 0.0f ? (double)m : 0.0;
  q.k = greedy || m > 1.0f ? 1u : (k > 0 ? (uint32_t)k : 0xffffffffu);
  return q;
}

// 2^((r - 1/2) / 16) for r in [0, 1): Taylor series, (ln 2 / 32)^6 / 720 = 2^-42
// off at most.
__device__ __forceinline__ double exp2_sub(double r) {
  constexpr double g = 0.69314718055994530942 / kSub;
  const double h = r - 0.5;
  double p = g * g * g * g * g / 120.0;
  p = fma(p, h, g * g * g * g / 24.0);
  p = fma(p, h, g * g * g / 6.0);
  p = fma(p, h, g * g / 2.0);
  p = fma(p, h, g);
  return fma(p, h, 1.0);
}

// Bin and weight of x: bins above `top` (a bin that begins an octave), and
// 2^(bits + (x c - top) / 16).  table[j] = 2^((j + 1/2) / 16).
struct Weight {
  int rel;
  double w;
};
__device__ __forceinline__ Weight weigh(float x, double c, double top, const double *table,
                                        int bits) {
  // z rounded before floor(z) is taken off it: an fma would leave the product's
  // rounding error, which for values near fp32's largest exceeds a bin by far
#pragma clang fp contract(off)
  const double z = (double)x * c, q = floor(z);
  const int rel = (int)fmax(q - top, -65536.0);
  return Weight{rel, ldexp(table[rel & (kSub - 1)] * exp2_sub(z - q), (rel >> 4) + bits)};
}
__device__ __forceinline__ double weight(float x, double c, double top, const double *table) {
  return weigh(x, c, top, table, 0).w;
}
// A weight of kFrac fraction bits as a whole number below 2^(kFrac + 1): rounded
// to nearest by the addition of 2^52, whose fraction then is the value.
__device__ __forceinline__ unsigned long long whole(double w) {
  const double v = fmin(w, (double)((2ull << kFrac) - 1)) + 4503599627370496.0;
  return (unsigned long long)__double_as_longlong(v) & 0xfffffffffffffull;
}
__device__ __forceinline__ unsigned long long fixed(float x, double c, double top,
                                                    const double *table) {
  return whole(weigh(x, c, top, table, kFrac).w);
}
__device__ __forceinline__ uint32_t count_of(unsigned long long h) {
  return (uint32_t)(h >> kSumBits);
}
__device__ __forceinline__ unsigned long long mass_of(unsigned long long h) {
  return h & ((1ull << kSumBits) - 1);
}
// Whole octaves below bin q.
__device__ __forceinline__ double octave(double q) { return floor(q / kSub) * kSub; }

__device__ __forceinline__ void fill_table(double *table) {
  if (threadIdx.x < kSub) table[threadIdx.x] = exp2((threadIdx.x + 0.5) / kSub);
}

__device__ __forceinline__ float block_max(float v, float *red) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int i = 1; i < kNT / 64; ++i) v = fmaxf(v, red[i]);
  __syncthreads();
  return v;
}

// The row and slice of a work-group.  Work-groups go to the 8 XCDs in turn:
// row r's take numbers that are r modulo 8, as row_kernel's own, so that the
// row and its histograms are in the L2 of the XCD that reads them next.
__device__ __forceinline__ bool place(const Args &a, int &r, int &s) {
  const int g = blockIdx.x / (8 * a.slices), i = blockIdx.x % (8 * a.slices);
  r = g * 8 + i % 8;
  s = i / 8;
  return r < a.R;
}

template <int TYPE>
__global__ __launch_bounds__(kNT) void slice_kernel(Args a) {
  __shared__ unsigned long long hist[kBins];
  __shared__ double table[kSub];
  __shared__ float red[kNT / 64];
  int r, s;
  if (!place(a, r, s)) return;
  const int tid = threadIdx.x;
  float x[kPer];
  load8<TYPE>(a, r, s * kSlice + tid * kPer, x);
  if (tid < kBins) hist[tid] = 0;
  fill_table(table);
  const Rule q = rule_of(a, r);
  float mx = x[0];
#pragma unroll
  for (int k = 1; k < kPer; ++k) mx = fmaxf(mx, x[k]);
  mx = block_max(mx, red);
  const long long at = (long long)r * a.slices + s;
  if (tid == 0) a.smax[at] = mx;
  if (mx == -INFINITY) {  // nothing to count; the row skips the slice
    return;
  }
  const double qtop = floor((double)mx * q.c), top = octave(qtop);
  const int rtop = (int)(qtop - top);
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    if (x[k] == -INFINITY) continue;
    const Weight w = weigh(x[k], q.c, top, table, kFrac);
    const int d = min(rtop - w.rel, kBins - 1);
    atomicAdd(&hist[d], (1ull << kSumBits) | whole(w.w));
  }
  __syncthreads();
  if (tid < kBins) a.hist[at * kBins + tid] = hist[tid];
}

// Inclusive sums over the wave's lanes, by data movement inside the vector
// registers (a shuffle through LDS costs about ten times as long).
#define CFA_SCAN_STEP(ctrl, rows)                                                              \
  {                                                                                            \
    n += __builtin_amdgcn_update_dpp(0, n, ctrl, rows, 0xf, false);                            \
    const uint64_t b_ = __double_as_longlong(m);                                               \
    const uint32_t l_ = __builtin_amdgcn_update_dpp(0, (uint32_t)b_, ctrl, rows, 0xf, false);  \
    const uint32_t h_ =                                                                        \
        __builtin_amdgcn_update_dpp(0, (uint32_t)(b_ >> 32), ctrl, rows, 0xf, false);          \
    m += __longlong_as_double(((uint64_t)h_ << 32) | l_);                                      \
  }
__device__ __forceinline__ void wave_scan(uint32_t &n, double &m) {
  CFA_SCAN_STEP(0x111, 0xf)  // from 1, 2, 4 and 8 lanes in front, in rows of 16
  CFA_SCAN_STEP(0x112, 0xf)
  CFA_SCAN_STEP(0x114, 0xf)
  CFA_SCAN_STEP(0x118, 0xf)
  CFA_SCAN_STEP(0x142, 0xa)  // lane 15 to the next row
  CFA_SCAN_STEP(0x143, 0xc)  // lane 31 to the upper half
}
#undef CFA_SCAN_STEP
__device__ __forceinline__ void wave_scan(uint64_t &m) {
#define CFA_SCAN_STEP(ctrl, rows)                                                              \
  {                                                                                            \
    const uint32_t l_ = __builtin_amdgcn_update_dpp(0, (uint32_t)m, ctrl, rows, 0xf, false);   \
    const uint32_t h_ =                                                                        \
        __builtin_amdgcn_update_dpp(0, (uint32_t)(m >> 32), ctrl, rows, 0xf, false);           \
    m += ((uint64_t)h_ << 32) | l_;                                                            \
  }
  CFA_SCAN_STEP(0x111, 0xf)
  CFA_SCAN_STEP(0x112, 0xf)
  CFA_SCAN_STEP(0x114, 0xf)
  CFA_SCAN_STEP(0x118, 0xf)
  CFA_SCAN_STEP(0x142, 0xa)
  CFA_SCAN_STEP(0x143, 0xc)
#undef CFA_SCAN_STEP
}

__device__ __forceinline__ double read_lane(double v, int lane) {
  const uint64_t b = __double_as_longlong(v);
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)b, lane);
  const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(b >> 32), lane);
  return __longlong_as_double(((uint64_t)hi << 32) | lo);
}

// Inclusive sums over the work-group's threads, in their order: (n, m) of the
// thread and those in front of it.  One barrier; `turn` alternates between
// calls, so that the next call's waves do not overwrite what is still read.
struct Partials {
  uint32_t n[2][kNT / 64];
  double m[2][kNT / 64];
};
__device__ __forceinline__ void block_scan(uint32_t &n, double &m, Partials &ps, int turn) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  wave_scan(n, m);
  if (lane == 63) {
    ps.n[turn][wave] = n;
    ps.m[turn][wave] = m;
  }
  __syncthreads();
  // every wave sums the partials of the waves in front of it in the same order
  uint32_t bn = lane < kNT / 64 ? ps.n[turn][lane] : 0;
  double bm = lane < kNT / 64 ? ps.m[turn][lane] : 0.0;
  wave_scan(bn, bm);
  if (wave > 0) {
    n += __builtin_amdgcn_readlane(bn, wave - 1);
    m += read_lane(bm, wave - 1);
  }
}

// The code of the least finite value x with floor(x c) >= q (c > 0).
template <int TYPE>
__device__ __forceinline__ uint32_t first_code(double q, double c) {
  using C = Code<TYPE>;
  const double guess = fmin(fmax(q / c, -(double)C::kMost), (double)C::kMost);
  uint32_t k = C::of((float)guess + 0.0f);
  while (k > C::lowest() && floor((double)C::value(k) * c) >= q) --k;
  while (k < C::most() && floor((double)C::value(k) * c) < q) ++k;
  return k;
}

// log2(m) for 0 < m <= 1 (of 1: 0, without any rounding).
__device__ __forceinline__ double log2_of(double m, const double *table) {
  if (m == 1.0) return 0.0;
  const int e = ilogb(m);
  const double f = ldexp(m, -e);  // [1, 2)
  return e + log2_from(f, __builtin_amdgcn_logf((float)f), table);
}

// f(code, index, at) for the tokens of a row with codes klo .. khi, `at`
// numbering those of this wave; returns how many they are.  One CU reads the
// whole row, so it is bound by instructions: the loads of several rounds are in
// flight before the first comparison; eight tokens a lane that all lie below a
// positive border are passed over by their largest word alone (as whole numbers,
// whose order is that of positive floats); the others are marked in a mask, and
// each lane then visits its own (a branch a token for whole waves, with its
// visits one by one, took 15 us against 6 where a hundredth are hits).
template <int TYPE, int kRounds, class F>
__device__ __forceinline__ uint32_t each_in_row(const Args &a, long long r, uint32_t klo,
                                                uint32_t khi, F f) {
  using C = Code<TYPE>;
  uint32_t got = 0;
  const Span<TYPE> in(klo, khi);
  if (in.none) return got;
  const bool positive = in.least > 0.0f;
  const int border = Raw<TYPE>::word(in.least);
  auto marks = [&](const float (&x)[kPer]) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) m |= in.holds(x[j]) ? 1u << j : 0u;
    return m;
  };
  // the marked tokens of a round of eights that begin at base + k kSlice
  auto visit = [&](uint64_t mask, int base) {
    uint32_t at = __popcll(mask);
    uint64_t upto = at;
    wave_scan(upto);
    const uint32_t all = __builtin_amdgcn_readlane((uint32_t)upto, 63);
    at = got + (uint32_t)upto - at;
    while (mask) {
      const int b = __ffsll((unsigned long long)mask) - 1;
      mask &= mask - 1;
      const int i = base + (b >> 3) * kSlice + (b & 7);
      f(C::of(load1<TYPE>(a, r, i)), i, at++);
    }
    got += all;
  };
  const int t0 = threadIdx.x * kPer;
  for (int b = 0; b < a.V; b += kRounds * kSlice) {
    uint64_t mask = 0;
    Raw<TYPE> v[kRounds];
#pragma unroll
    for (int k = 0; k < kRounds; ++k)
      if (b + k * kSlice + t0 + kPer <= a.V) v[k].load(a, r, b + k * kSlice + t0);
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      const int i = b + k * kSlice + t0;
      float x[kPer];
      if (i + kPer <= a.V) {
        if (positive && __ballot(v[k].most() >= border) == 0) continue;
        v[k].get(x);
        mask |= (uint64_t)marks(x) << (8 * k);
      } else if (i < a.V) {
        load8<TYPE>(a, r, i, x);
        mask |= (uint64_t)marks(x) << (8 * k);
      }
    }
    if (__ballot(mask != 0)) visit(mask, b + t0);
  }
  return got;
}

// The first thread for which `ends` holds, with what it brings (-1: none).  One
// barrier; `turn` as in block_scan.
struct Ends {
  int tid[2][kNT / 64];
  uint32_t before[2][kNT / 64], own[2][kNT / 64];
  double mass[2][kNT / 64];
};
struct End {
  int tid;
  uint32_t before, own;  // tokens in front of it, and its own
  double mass;           // mass in front of it
};
__device__ __forceinline__ End first_end(bool ends, uint32_t before, uint32_t own, double mass,
                                         Ends &es, int turn) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t any = __ballot(ends);
  if (any == 0) {
    if (lane == 0) es.tid[turn][wave] = -1;
  } else if (lane == __ffsll((unsigned long long)any) - 1) {
    es.tid[turn][wave] = threadIdx.x;
    es.before[turn][wave] = before;
    es.own[turn][wave] = own;
    es.mass[turn][wave] = mass;
  }
  __syncthreads();
  const uint64_t waves = __ballot(lane < kNT / 64 && es.tid[turn][lane % (kNT / 64)] >= 0);
  if (waves == 0) return End{-1, 0, 0, 0.0};
  const int w = __ffsll((unsigned long long)waves) - 1;
  return End{es.tid[turn][w], es.before[turn][w], es.own[turn][w], es.mass[turn][w]};
}

template <int TYPE>
__global__ __launch_bounds__(kNT) void row_kernel(Args a) {
  using C = Code<TYPE>;
  __shared__ uint32_t list_key[kList];  // a part for each wave
  __shared__ int list_idx[kList];
  __shared__ uint32_t list_n[kNT / 64];
  __shared__ uint32_t dcnt[kDigits];
  __shared__ unsigned long long dmass[kDigits];
  __shared__ double table[kSub];
  // per slice: its largest bin below the row's and its unit's octaves, in
  // these units; the mass it keeps, in its own unit
  __shared__ int sshift[kMaxSlices], soct[kMaxSlices];
  __shared__ unsigned long long skept[kMaxSlices];
  __shared__ Partials ps;
  __shared__ Ends es;
  __shared__ uint32_t deep_n;
  __shared__ unsigned long long deep_m;
  __shared__ int draw_last;
  __shared__ uint32_t sel_key;
  __shared__ int sel_last;
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Rule q = rule_of(a, r);
  int turn = 0;
  auto scan = [&](uint32_t &n, double &m) {
    block_scan(n, m, ps, turn & 1);
    ++turn;
  };
  auto first = [&](bool ends, uint32_t before, uint32_t own, double mass) {
    const End e = first_end(ends, before, own, mass, es, turn & 1);
    ++turn;
    return e;
  };

  // every wave takes the row's maximum from the slices' (no barrier)
  float mx = -INFINITY, mine = -INFINITY;
  for (int s = lane; s < a.slices; s += 64) mx = fmaxf(mx, a.smax[(long long)r * a.slices + s]);
  if (tid < a.slices) mine = a.smax[(long long)r * a.slices + tid];
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
  if (mx == -INFINITY) {  // every token is masked
    if (tid < a.draws) a.tokens[(long long)r * a.draws + tid] = -1;
    if (tid == 0 && a.probs) a.kept[r] = Kept{q.c, 0.0, 0.0, 0xffffffffu, -1};
    return;
  }
  const double qtop = floor((double)mx * q.c), top = octave(qtop);
  fill_table(table);
  if (tid < a.slices) {
    const double sq = floor((double)mine * q.c);
    // (a slice of masked tokens alone has no histogram: shift -1.  Kept in range
    // whatever the workspace holds: calls that share one at once, which they must
    // not, get wrong tokens but read nothing outside of it.)
    sshift[tid] = mine == -INFINITY ? -1 : (int)fmin(fmax(qtop - sq, 0.0), (double)kBins);
    soct[tid] = mine == -INFINITY ? 0 : (int)fmin(fmax((top - octave(sq)) / kSub, 0.0), 4000.0);
    skept[tid] = 0;
  }
  if (tid == 0) {
    deep_n = 0;
    deep_m = 0;
  }
  __syncthreads();

  // the row's histogram: thread b takes bin b % kBins of every other slice, in
  // units of the row's largest octave; the last bin takes what lies behind
  uint32_t n = 0;
  double m = 0.0;
  const int bin = tid % kBins;
  constexpr int kHalves = kNT / kBins, kRound = 8;
  for (int s0 = tid / kBins; s0 < a.slices; s0 += kRound * kHalves) {
    unsigned long long w[kRound];
#pragma unroll
    for (int k = 0; k < kRound; ++k) {  // every load in flight before the first sum
      const int s = s0 + k * kHalves;
      const int shift = s < a.slices ? sshift[s] : -1;
      const int from = bin == kBins - 1 ? bin : bin - shift;
      const bool ok = shift >= 0 && from >= 0;
      const long long at = ((long long)r * a.slices + s) * kBins + from;
      w[k] = ok ? a.hist[at] : 0;
    }
#pragma unroll
    for (int k = 0; k < kRound; ++k) {
      const int s = s0 + k * kHalves;
      if (s >= a.slices) continue;
      n += count_of(w[k]);
      m += ldexp((double)mass_of(w[k]), -soct[s]);
    }
  }
  // bins that the shift moves behind the last (32 octaves down: next to no mass,
  // in whole units so that the order does not matter), one wave a slice
  for (int s = wave; s < a.slices; s += kNT / 64) {
    for (int b = max(kBins - 1 - sshift[s], 0) + lane; b < kBins - 1; b += 64) {
      const long long at = ((long long)r * a.slices + s) * kBins + b;
      const unsigned long long d = a.hist[at];
      if (d) {
        atomicAdd(&deep_n, count_of(d));
        atomicAdd(&deep_m, soct[s] < 64 ? mass_of(d) >> soct[s] : 0ull);
      }
    }
  }
  double *half_m = reinterpret_cast<double *>(dmass);
  if (tid >= kBins) {
    dcnt[tid - kBins] = n;
    half_m[tid - kBins] = m;
  }
  // the code of the least value that min-p keeps, and its bin
  uint32_t least = C::lowest();
  if (q.m > 0.0 && q.m <= 1.0) {
    const double xm = mx + kSub * log2_of(q.m, table) / q.c;
    least = C::of((float)fmax(xm, -(double)C::kMost) + 0.0f);
    while (least > C::lowest() && (double)C::value(least) >= xm) --least;
    while ((double)C::value(least) < xm) ++least;  // (ends at the maximum's)
  }
  const int bin_m = (int)fmin(qtop - floor((double)C::value(least) * q.c), (double)(kBins - 1));
  __syncthreads();
  if (tid < kBins) {
    n += dcnt[tid];
    m += half_m[tid];
    if (tid == kBins - 1) {
      n += deep_n;
      m += (double)deep_m;
    }
  } else {
    n = 0;
    m = 0.0;
  }
  const uint32_t bn = n;
  const double bm = m;
  scan(n, m);
  // (bins from kBins on add nothing: the last thread's sum is Z)
  if (tid == kNT - 1) half_m[kDigits - 1] = m;
  __syncthreads();
  const double limit = q.p <= 1.0 ? fmax(q.p * half_m[kDigits - 1], 1e-300) : INFINITY;
  // the first bin that is not kept as a whole (min-p's at the latest)
  const End crit = first(tid < kBins && (n > q.k || m >= limit || tid == bin_m), n - bn, bn, m - bm);
  // (where neither top-k nor top-p ends in it and min-p takes off nothing, every
  // token is kept)
  const bool all = least == C::lowest() && crit.tid == bin_m && crit.before + crit.own <= q.k &&
                   limit == INFINITY;
  uint32_t room = q.k - crit.before;  // tokens that may still be kept
  double left = limit - crit.mass;    // the mass in front of a kept one stays below it
  uint32_t bin_lo, bin_hi;
  {
    // odd lanes: the first key of the bin in front
    const double qb = qtop - crit.tid + (lane & 1);
    const uint32_t k = first_code<TYPE>(qb, q.c);
    bin_lo = crit.tid == kBins - 1 ? C::lowest() : __builtin_amdgcn_readlane(k, 0);
    bin_hi = crit.tid == 0 ? C::of(mx) : __builtin_amdgcn_readlane(k, 1) - 1;
  }

  // each slice's mass in whole kept bins, one wave a slice
  for (int s = wave; s < a.slices; s += kNT / 64) {
    const int bins = sshift[s] < 0 ? 0 : (all ? kBins : crit.tid - sshift[s]);
    const long long at = ((long long)r * a.slices + s) * kBins;
    unsigned long long w[kBins / 64];
#pragma unroll
    for (int k = 0; k < kBins / 64; ++k) {
      const int b = k * 64 + lane;
      w[k] = b < bins ? mass_of(a.hist[at + b]) : 0ull;
    }
    uint64_t sum = 0;
#pragma unroll
    for (int k = 0; k < kBins / 64; ++k) sum += w[k];
    wave_scan(sum);
    if (lane == 63) skept[s] = sum;
  }

  // select inside the bin: codes lo .. hi hold the end
  uint32_t lo = bin_lo, hi = bin_hi, now = crit.own;
  bool listed = false, whole = false;
  // f(code, index) for the tokens in lo .. hi
  auto each = [&](auto f) {
    if (listed) {
      for (uint32_t i = lane; i < list_n[wave]; i += 64) {
        const uint32_t key = list_key[wave * kWaveList + i];
        if (key >= lo && key <= hi) f(key, list_idx[wave * kWaveList + i]);
      }
    } else {
      each_in_row<TYPE, 1>(a, r, lo, hi, [&](uint32_t k, int i, uint32_t) { f(k, i); });
    }
  };
  // the tokens in lo .. hi to the waves' lists; false where one does not hold them
  auto gather = [&]() {
    const uint32_t got = each_in_row<TYPE, TYPE == kF32 ? 2 : 4>(a, r, lo, hi, [&](uint32_t k, int i, uint32_t at) {
      if (at < kWaveList) {
        list_key[wave * kWaveList + at] = k;
        list_idx[wave * kWaveList + at] = i;
      }
    });
    if (lane == 0) list_n[wave] = got;
    __syncthreads();
    listed = __ballot(lane < kNT / 64 && list_n[lane % (kNT / 64)] > kWaveList) == 0;
    return listed;
  };
  // at most kFew tokens in lo .. hi: the first wave holds one a lane and counts,
  // for each, the tokens and the mass in front of it
  auto few = [&]() {
    __syncthreads();
    if (wave == 0) {
      // (the list may hold others too: its tokens in the range, packed to the
      // lanes from 0 on)
      uint32_t k = 0;
      int i = 0, got = 0;
      for (int p = 0; p < kNT / 64; ++p) {
        for (uint32_t j0 = 0; j0 < list_n[p]; j0 += 64) {
          const uint32_t j = p * kWaveList + j0 + lane;
          const uint32_t kj = j0 + lane < list_n[p] ? list_key[j] : 0;
          const bool in = j0 + lane < list_n[p] && kj >= lo && kj <= hi;
          const uint64_t b = __ballot(in);
          const int to = got + (int)__popcll(b & ((1ull << lane) - 1));
          if (in && to < kFew) {
            dcnt[to] = kj;
            dcnt[kFew + to] = list_idx[j];
          }
          got = min(got + (int)__popcll(b), kFew);
        }
      }
      const bool live = lane < got;
      k = live ? dcnt[lane] : 0;
      i = live ? (int)dcnt[kFew + lane] : 0;
      const unsigned long long w = live ? fixed(C::value(k), q.c, top, table) : 0;
      uint32_t ahead = 0;
      unsigned long long mass = 0;
      for (int j = 0; j < got; ++j) {
        const uint32_t kj = __builtin_amdgcn_readlane(k, j);
        const int ij = __builtin_amdgcn_readlane(i, j);
        const uint32_t lo_j = __builtin_amdgcn_readlane((uint32_t)w, j);
        const uint32_t hi_j = __builtin_amdgcn_readlane((uint32_t)(w >> 32), j);
        const unsigned long long wj = ((unsigned long long)hi_j << 32) | lo_j;
        const bool front = kj > k || (kj == k && ij < i);
        ahead += front;
        mass += front ? wj : 0;
      }
      const bool keep = live && ahead < room && (double)mass < left;
      // kept tokens are the first in the order: the one with most ahead is last
      const int n_kept = __popcll(__ballot(keep));
      if (n_kept == 0) {
        if (lane == 0) {
          sel_key = hi;
          sel_last = -1;
          // (none of them: whatever lies above the range stays)
          if (hi != 0xffffffffu) sel_key = hi + 1, sel_last = 0x7fffffff;
        }
      } else if (keep && (int)ahead == n_kept - 1) {
        sel_key = k;
        sel_last = i;
      }
    }
    __syncthreads();
  };
  bool cut = !all && (now > room || left < INFINITY);  // (otherwise min-p alone ends the row here)
  bool done = false;
  uint32_t fits = kList;  // tokens that are tried to be listed
  while (!all) {
    if (!listed && now <= fits) {
      whole = gather() && lo == bin_lo && hi == bin_hi;
      fits = kWaveList;
    }
    if (!cut || lo >= hi) break;
    if (listed && now <= kFew) {
      few();
      done = true;
      break;
    }
    const int bits = 32 - __clz(hi - lo), shift = max(bits - 10, 0);
    __syncthreads();
    dcnt[tid] = 0;
    dmass[tid] = 0;
    __syncthreads();
    each([&](uint32_t key, int) {
      const uint32_t d = (hi - key) >> shift;
      atomicAdd(&dcnt[d], 1u);
      atomicAdd(&dmass[d], fixed(C::value(key), q.c, top, table));
    });
    __syncthreads();
    const uint32_t dn = dcnt[tid];
    const double dm = (double)dmass[tid];
    n = dn;
    m = dm;
    scan(n, m);
    const End e = first(dn > 0 && (n > room || m >= left), n - dn, dn, m - dm);
    if (e.tid < 0) {  // all of these are kept
      cut = false;
      break;
    }
    room -= e.before;
    left -= e.mass;
    now = e.own;
    hi -= (uint32_t)e.tid << shift;
    lo = max(lo, hi - ((1u << shift) - 1));
  }
  // equal values: the first ones by index
  uint32_t key = lo;
  int last = 0x7fffffff;
  if (done) {
    key = sel_key;
    last = sel_last;
  } else if (cut) {
    const double w = (double)fixed(C::value(key), q.c, top, table);
    uint32_t keep = min(room, now);
    if (w > 0.0 && left < INFINITY)
      keep = (uint32_t)fmin((double)keep, fmax(ceil(left / w), 0.0));
    if (keep == 0) {
      last = -1;
    } else if (keep < now) {
      // the index of number `keep`: its 1024 tokens first, then itself
      int base = 0;
      for (int level = 1; level >= 0; --level) {
        __syncthreads();
        dcnt[tid] = 0;
        __syncthreads();
        each([&](uint32_t k, int i) {
          if (k != key) return;
          if (level == 1) atomicAdd(&dcnt[i >> 10], 1u);
          else if (i >> 10 == base) atomicAdd(&dcnt[i & 1023], 1u);
        });
        __syncthreads();
        const uint32_t dn = dcnt[tid];
        n = dn;
        m = 0.0;
        scan(n, m);
        const End e = first(n >= keep, n - dn, dn, 0.0);
        if (level == 1) {
          base = e.tid;
          keep -= e.before;
        } else {
          last = (base << 10) + e.tid;
        }
      }
    }
  }
  if (all) key = C::lowest();
  if (key < least) {  // min-p ends it first
    key = least;
    last = 0x7fffffff;
  }

  // the bin's kept tokens, to their slices' masses
  auto own_top = [&](int s) { return top - (double)kSub * soct[s]; };
  auto add = [&](uint32_t k, int i) {
    if (k > key || (k == key && i <= last))
      atomicAdd(&skept[i / kSlice], fixed(C::value(k), q.c, own_top(i / kSlice), table));
  };
  __syncthreads();
  if (whole) {
    for (uint32_t i = lane; i < list_n[wave]; i += 64)
      add(list_key[wave * kWaveList + i], list_idx[wave * kWaveList + i]);
  } else if (!all) {
    each_in_row<TYPE, 1>(a, r, max(key, bin_lo), bin_hi,
                      [&](uint32_t k, int i, uint32_t) { add(k, i); });
  }
  __syncthreads();
  // the slices' masses up to and with each, in the row's unit (lane s: slices
  // s and 64 + s)
  double upto[kMaxSlices / 64], own[kMaxSlices / 64], total = 0.0;
#pragma unroll
  for (int k = 0; k < kMaxSlices / 64; ++k) {
    const int s = k * 64 + lane;
    uint32_t none = 0;
    own[k] = s < a.slices ? ldexp((double)skept[s], -soct[s]) : 0.0;
    upto[k] = own[k];
    wave_scan(none, upto[k]);
    upto[k] += total;
    total = read_lane(upto[k], 63);
  }
  if (tid == 0 && a.probs)
    a.kept[r] = Kept{q.c, top, (double)(1ull << kFrac) / total, key, last};

  for (int d = 0; d < a.draws; ++d) {
    // the slice, then the token
    const double want = (double)a.u[(long long)r * a.draws + d] * total;
    int at = -1;
    double rest = INFINITY;
#pragma unroll
    for (int k = 0; k < kMaxSlices / 64; ++k) {
      const uint64_t hit = __ballot(own[k] > 0.0 && upto[k] > want);
      if (at < 0 && hit) {
        const int w = __ffsll((unsigned long long)hit) - 1;
        at = k * 64 + w;
        rest = ldexp(want - (read_lane(upto[k], w) - read_lane(own[k], w)), soct[at]);
      }
    }
    if (at < 0) {  // u of 1 and above, or NaN: the last kept token
#pragma unroll
      for (int k = 0; k < kMaxSlices / 64; ++k) {
        const uint64_t some = __ballot(own[k] > 0.0);
        if (some) at = k * 64 + 63 - __clzll((long long)some);
      }
      at = max(at, 0);
    }
    float x[kPer];
    const int i0 = at * kSlice + tid * kPer;
    load8<TYPE>(a, r, i0, x);
    unsigned long long w[kPer], sum = 0;
    const double st = own_top(at);
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      w[k] = 0;
      const uint32_t kx = C::of(x[k]);
      if (x[k] != -INFINITY && (kx > key || (kx == key && i0 + k <= last)))
        w[k] = fixed(x[k], q.c, st, table);
      sum += w[k];
    }
    // (whole numbers below 2^55: their fp64 sums are off by 2^-53 at most)
    uint32_t none = 0;
    double c = (double)sum;
    scan(none, c);
    c -= (double)sum;
    int hit = -1, any = -1;
#pragma unroll
    for (int k = kPer - 1; k >= 0; --k) any = any < 0 && w[k] ? i0 + k : any;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      c += (double)w[k];
      hit = hit < 0 && w[k] && c > rest ? i0 + k : hit;
    }
    const End e = first(hit >= 0, (uint32_t)hit, 0, 0.0);
    if (e.tid >= 0) {
      if (tid == 0) a.tokens[(long long)r * a.draws + d] = (int)e.before;
    } else {  // none beyond it: the last of any weight
      if (tid == 0) draw_last = 0;
      __syncthreads();
      if (any >= 0) atomicMax(&draw_last, any);
      __syncthreads();
      if (tid == 0) a.tokens[(long long)r * a.draws + d] = draw_last;
      __syncthreads();
    }
  }
}

template <int TYPE>
__global__ __launch_bounds__(kNT) void probs_kernel(Args a) {
  __shared__ double table[kSub];
  int r, s;
  if (!place(a, r, s)) return;
  const int i0 = s * kSlice + threadIdx.x * kPer;
  float x[kPer];
  load8<TYPE>(a, r, i0, x);
  fill_table(table);
  const Kept k = a.kept[r];
  __syncthreads();
  float p[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const uint32_t key = Code<TYPE>::of(x[j]);
    const bool kept = x[j] != -INFINITY && (key > k.key || (key == k.key && i0 + j <= k.last));
    p[j] = kept ? (float)(weight(x[j], k.c, k.top, table) * k.scale) : 0.0f;
  }
  float *out = a.probs + (long long)r * a.V + i0;
  if (i0 + kPer <= a.V) {  // (rows of an odd length begin anywhere)
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    typedef f32x4 at_element __attribute__((aligned(4)));
    __builtin_nontemporal_store(f32x4{p[0], p[1], p[2], p[3]}, reinterpret_cast<at_element *>(out));
    __builtin_nontemporal_store(f32x4{p[4], p[5], p[6], p[7]},
                                reinterpret_cast<at_element *>(out) + 1);
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (i0 + j < a.V) out[j] = p[j];
  }
}

static size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

struct Layout {
  size_t smax, hist, kept, bytes;
  Layout(long long R, int V) {
    const size_t n = (size_t)R * ((V + kSlice - 1) / kSlice);
    smax = 0;
    hist = smax + align256(n * sizeof(float));
    kept = hist + align256(n * kBins * sizeof(unsigned long long));
    bytes = kept + align256((size_t)R * sizeof(Kept));
  }
};

template <int TYPE>
int launch(const Args &a, hipStream_t st) {
  const unsigned grid = (unsigned)((a.R + 7) / 8 * 8 * a.slices);
  CFA_LAUNCH("sample_slices", slice_kernel<TYPE>, dim3(grid), dim3(kNT), 0, st, a);
  CFA_LAUNCH("sample_rows", row_kernel<TYPE>, dim3(a.R), dim3(kNT), 0, st, a);
  if (a.probs)
    CFA_LAUNCH("sample_probs", probs_kernel<TYPE>, dim3(grid), dim3(kNT), 0, st, a);
  return CFA_OK;
}

}  // namespace rows
}  // namespace cfa

using namespace cfa::rows;

extern "C" size_t cfa_sample_rows_workspace_size(int R, int V) {
  if (R <= 0 || V <= 0 || V > kMaxSlices * kSlice) return 0;
  return Layout(R, V).bytes;
}

extern "C" int cfa_sample_rows(const void *rows, int64_t row_stride, int elem_type, int R, int V,
                               int draws, const float *temperature, float temperature_all,
                               const int32_t *top_k, int top_k_all, const float *top_p,
                               float top_p_all, const float *min_p, float min_p_all,
                               const float *uniforms, int32_t *out_tokens, float *out_probs,
                               void *workspace, size_t workspace_bytes, void *stream) {
  using namespace cfa::abi;
  clear_error();
  if (R < 0 || V <= 0 || V > kMaxSlices * kSlice)
    return fail_arg("need R >= 0 and 0 < V <= 2^20");
  if (elem_type < kF32 || elem_type > kFP16) return fail_arg("elem_type must be 0, 1 or 2");
  if (draws < 0 || draws > 64) return fail_arg("draws must be between 0 and 64");
  if (draws == 0 && !out_probs) return fail_arg("without draws out_probs is needed");
  if (R > 1 && row_stride < V) return fail_arg("row_stride must be at least V");
  if (R == 0) return CFA_OK;
  if (!rows || !workspace || (draws > 0 && (!uniforms || !out_tokens)))
    return fail_arg("null pointer argument");
  const Layout lay(R, V);
  if (workspace_bytes < lay.bytes)
    return fail_arg("workspace too small (see cfa_sample_rows_workspace_size)");
  if (((uintptr_t)workspace & 15) != 0 || ((uintptr_t)out_probs & 15) != 0)
    return fail_arg("workspace and out_probs must be 16-byte aligned");
  Args a{};
  a.rows = rows;
  a.stride = row_stride;
  a.R = R;
  a.V = V;
  a.draws = draws;
  a.slices = (V + kSlice - 1) / kSlice;
  if (((long long)R + 7) / 8 * 8 * a.slices * kNT >= (1LL << 32)) return fail_arg("too many rows for one call");
  if ((uintptr_t)rows % (elem_type == kF32 ? 4 : 2)) return fail_arg("rows must be aligned to its elements");
  a.temp = temperature;
  a.temp0 = temperature_all;
  a.top_k = top_k;
  a.top_k0 = top_k_all;
  a.top_p = top_p;
  a.top_p0 = top_p_all;
  a.min_p = min_p;
  a.min_p0 = min_p_all;
  a.u = uniforms;
  a.tokens = out_tokens;
  a.probs = out_probs;
  char *ws = (char *)workspace;
  a.smax = (float *)(ws + lay.smax);
  a.hist = (unsigned long long *)(ws + lay.hist);
  a.kept = (Kept *)(ws + lay.kept);
  hipStream_t st = (hipStream_t)stream;
  switch (elem_type) {
    case kF32: return launch<kF32>(a, st);
    case kBF16: return launch<kBF16>(a, st);
    default: return launch<kFP16>(a, st);
  }
}
