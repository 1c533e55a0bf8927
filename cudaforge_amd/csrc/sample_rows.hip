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
// Weights are therefore formed in fp64 and kept as 41-bit fractions of a power
// of two near their slice's largest, so that sums are exact whatever their
// order: the histograms' atomics leave the same bits every time.
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
// Bound: the rows' bytes once from HBM, then latency of the second launch.
#include <hip/hip_runtime.h>

#include <cfloat>

#include "abi_internal.hpp"
#include "half_types.hpp"

namespace cfa {
namespace rows {

constexpr int kNT = 1024;
constexpr int kPer = 8;              // consecutive tokens of a thread
constexpr int kSlice = kNT * kPer;   // tokens of a slice
constexpr int kMaxSlices = 128;      // V <= 2^20
constexpr int kSub = 16;             // bins per octave of weight
constexpr int kBins = 512;           // 32 octaves, the last bin takes the rest
constexpr int kDigits = 1024;        // radix of the selection inside a bin
constexpr int kList = 8192;          // tokens of a bin that fit LDS
constexpr int kFrac = 41;            // fraction bits of a weight

enum Type { kF32 = 0, kBF16 = 1, kFP16 = 2 };

struct Args {
  const void *rows;
  long long stride;
  int type, R, V, draws, slices, vec;
  const float *temp, *top_p, *min_p;  // [R] or null: the scalar
  const int32_t *top_k;
  float temp0, top_p0, min_p0;
  int top_k0;
  const float *u;  // [R, draws]
  int32_t *tokens;
  float *probs;
  // workspace
  float *smax;               // [R, slices]
  uint32_t *cnt;             // [R, slices, kBins]
  unsigned long long *mass;  // [R, slices, kBins]
  struct Kept *kept;         // [R]
};

// What row_kernel leaves for the probabilities.
struct Kept {
  double c, top, scale;  // bins per unit of x; bin of 2^0; 1 / kept mass
  uint32_t key;          // kept: a larger key, or this one up to index `last`
  int last;
};

// fp32 values as keys whose order is theirs.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}
constexpr uint32_t kKeyLowest = 0x00800000u;  // key_of(-FLT_MAX)

// A logit as the rules take it: NaN as -inf, +inf as the largest finite, -0 as 0.
__device__ __forceinline__ float clean(float x) {
  return x != x ? -INFINITY : fminf(x, FLT_MAX) + 0.0f;
}

template <int TYPE>
__device__ __forceinline__ float load1(const Args &a, long long row, int i) {
  if constexpr (TYPE == kF32) {
    return clean(reinterpret_cast<const float *>(a.rows)[row * a.stride + i]);
  } else {
    const uint16_t v = reinterpret_cast<const uint16_t *>(a.rows)[row * a.stride + i];
    float lo, hi;
    if constexpr (TYPE == kBF16) unpack2<BF16>(v, lo, hi);
    else unpack2<FP16>(v, lo, hi);
    return clean(lo);
  }
}

// Tokens i .. i + 7 of a row (-inf behind its end).
template <int TYPE>
__device__ __forceinline__ void load8(const Args &a, long long row, int i, float (&x)[kPer]) {
  if (a.vec && i + kPer <= a.V) {
    if constexpr (TYPE == kF32) {
      const float4 *p =
          reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(a.rows) + row * a.stride + i);
      const float4 v0 = p[0], v1 = p[1];
      x[0] = v0.x; x[1] = v0.y; x[2] = v0.z; x[3] = v0.w;
      x[4] = v1.x; x[5] = v1.y; x[6] = v1.z; x[7] = v1.w;
    } else {
      const uint4 v = *reinterpret_cast<const uint4 *>(
          reinterpret_cast<const uint16_t *>(a.rows) + row * a.stride + i);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (TYPE == kBF16) unpack2<BF16>(w[k], x[2 * k], x[2 * k + 1]);
        else unpack2<FP16>(w[k], x[2 * k], x[2 * k + 1]);
      }
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k) x[k] = clean(x[k]);
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

// 2^(r / 16) for r in [0, 1): Taylor, relative error below 2^-53.
__device__ __forceinline__ double exp2_sub(double r) {
  constexpr double g = 0.69314718055994530942 / kSub;
  double p = g * g * g * g * g * g * g / 5040.0;
  p = fma(p, r, g * g * g * g * g * g / 720.0);
  p = fma(p, r, g * g * g * g * g / 120.0);
  p = fma(p, r, g * g * g * g / 24.0);
  p = fma(p, r, g * g * g / 6.0);
  p = fma(p, r, g * g / 2.0);
  p = fma(p, r, g);
  return fma(p, r, 1.0);
}

// 2^((x c - top) / 16) with top a whole number of octaves; table = 2^(j / 16).
// A weight of 2^-1024 and below may come out as 0.
__device__ __forceinline__ double weight(float x, double c, double top, const double *table) {
  // z rounded before floor(z) is taken off it: an fma would leave the product's
  // rounding error, which for values near fp32's largest exceeds a bin by far
#pragma clang fp contract(off)
  const double z = (double)x * c, q = floor(z);
  const int rel = (int)fmax(q - top, -65536.0);
  return ldexp(table[rel & (kSub - 1)] * exp2_sub(z - q), rel >> 4);
}
// The same as a fraction of kFrac bits (at most 2^(kFrac + 1)).
__device__ __forceinline__ unsigned long long fixed(double w) {
  // rounded to nearest by the addition of 2^52, whose fraction then is the value
  const double v = w * (double)(1ull << kFrac) + 4503599627370496.0;
  return __double_as_longlong(v) & 0xfffffffffffffull;
}
// Whole octaves below bin q.
__device__ __forceinline__ double octave(double q) { return floor(q / kSub) * kSub; }

__device__ __forceinline__ void fill_table(double *table) {
  if (threadIdx.x < kSub) table[threadIdx.x] = exp2((double)threadIdx.x / kSub);
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

template <int TYPE>
__global__ __launch_bounds__(kNT) void slice_kernel(Args a) {
  __shared__ uint32_t cnt[kBins];
  __shared__ unsigned long long mass[kBins];
  __shared__ double table[kSub];
  __shared__ float red[kNT / 64];
  const int r = blockIdx.x / a.slices, s = blockIdx.x % a.slices, tid = threadIdx.x;
  float x[kPer];
  load8<TYPE>(a, r, s * kSlice + tid * kPer, x);
  if (tid < kBins) {
    cnt[tid] = 0;
    mass[tid] = 0;
  }
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
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    if (x[k] == -INFINITY) continue;
    const int d = (int)fmin(qtop - floor((double)x[k] * q.c), (double)(kBins - 1));
    atomicAdd(&cnt[d], 1u);
    atomicAdd(&mass[d], fixed(weight(x[k], q.c, top, table)));
  }
  __syncthreads();
  if (tid < kBins) {
    a.cnt[at * kBins + tid] = cnt[tid];
    a.mass[at * kBins + tid] = mass[tid];
  }
}

// Inclusive sums over the work-group's threads, in their order.
struct Sums {
  uint32_t n;
  double m;
};
__device__ __forceinline__ Sums block_scan(uint32_t n, double m, uint32_t *rn, double *rm) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t vn = __shfl_up(n, o, 64);
    const double vm = __shfl_up(m, o, 64);
    if (lane >= o) {
      n += vn;
      m += vm;
    }
  }
  if (lane == 63) {
    rn[wave] = n;
    rm[wave] = m;
  }
  __syncthreads();
  uint32_t bn = 0;
  double bm = 0.0;
  for (int i = 0; i < wave; ++i) {
    bn += rn[i];
    bm += rm[i];
  }
  __syncthreads();
  return Sums{n + bn, m + bm};
}
__device__ __forceinline__ unsigned long long block_scan_u64(unsigned long long m,
                                                             unsigned long long *red) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned long long v = __shfl_up(m, o, 64);
    if (lane >= o) m += v;
  }
  if (lane == 63) red[wave] = m;
  __syncthreads();
  unsigned long long b = 0;
  for (int i = 0; i < wave; ++i) b += red[i];
  __syncthreads();
  return m + b;
}

// The least finite fp32 x with floor(x c) >= q, as a key (c > 0).
__device__ __forceinline__ uint32_t first_key(double q, double c) {
  const double guess = fmin(fmax(q / c, -(double)FLT_MAX), (double)FLT_MAX);
  uint32_t k = key_of((float)guess + 0.0f);
  constexpr uint32_t kKeyMost = 0xff7fffffu;  // key_of(FLT_MAX)
  while (k > kKeyLowest && floor((double)of_key(k) * c) >= q) --k;
  while (k < kKeyMost && floor((double)of_key(k) * c) < q) ++k;
  return k;
}

template <int TYPE>
__global__ __launch_bounds__(kNT) void row_kernel(Args a) {
  __shared__ uint32_t list_key[kList];
  __shared__ int list_idx[kList];
  __shared__ uint32_t dcnt[kDigits];
  __shared__ unsigned long long dmass[kDigits];
  __shared__ double table[kSub];
  __shared__ float smax[kMaxSlices];
  __shared__ unsigned long long skept[kMaxSlices];  // kept mass, in the slice's own unit
  __shared__ double rm[kNT / 64];
  __shared__ uint32_t rn[kNT / 64];
  __shared__ unsigned long long ru[kNT / 64];
  __shared__ float rf[kNT / 64];
  __shared__ uint32_t found_n, list_n, found_d;
  __shared__ double found_m;
  __shared__ int found_i;
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Rule q = rule_of(a, r);
  fill_table(table);
  float mx = -INFINITY;
  if (tid < a.slices) mx = smax[tid] = a.smax[(long long)r * a.slices + tid];
  mx = block_max(mx, rf);
  if (mx == -INFINITY) {  // every token is masked
    if (tid < a.draws) a.tokens[(long long)r * a.draws + tid] = -1;
    if (tid == 0 && a.probs) a.kept[r] = Kept{q.c, 0.0, 0.0, 0xffffffffu, -1};
    return;
  }
  const double qtop = floor((double)mx * q.c), top = octave(qtop);

  // the row's histogram: thread b takes bin b % kBins of every other slice, in
  // units of the row's largest octave; the last bin takes what lies behind
  uint32_t n = 0, deep_n = 0;
  double m = 0.0, deep_m = 0.0;
  {
    const int bin = tid % kBins;
    for (int s = tid / kBins; s < a.slices; s += kNT / kBins) {
      if (smax[s] == -INFINITY) continue;
      const long long at = ((long long)r * a.slices + s) * kBins;
      const double sq = floor((double)smax[s] * q.c);
      const double shift = qtop - sq;  // bins further down
      const double unit = ldexp(1.0, (int)fmax((octave(sq) - top) / kSub, -2000.0));
      const double from = bin - shift;
      if (bin < kBins - 1 && from >= 0.0) {
        n += a.cnt[at + (int)from];
        m += unit * (double)a.mass[at + (int)from];
      }
      if (bin + shift >= kBins - 1) {
        deep_n += a.cnt[at + bin];
        deep_m += unit * (double)a.mass[at + bin];
      }
    }
  }
  const Sums deep = block_scan(deep_n, deep_m, rn, rm);  // the last thread has them all
  if (tid == kNT - 1) {
    found_n = deep.n;
    found_m = deep.m;
  }
  // both halves of the slices meet in the first kBins threads
  double *half_m = reinterpret_cast<double *>(dmass);
  if (tid >= kBins) {
    dcnt[tid - kBins] = n;
    half_m[tid - kBins] = m;
  }
  __syncthreads();
  if (tid < kBins) {
    n += dcnt[tid];
    m += half_m[tid];
    if (tid == kBins - 1) {
      n = found_n;
      m = found_m;
    }
  } else {
    n = 0;
    m = 0.0;
  }
  const Sums up = block_scan(n, m, rn, rm);
  if (tid == kNT - 1) found_m = up.m;  // Z
  if (tid == 0) found_d = kBins;
  __syncthreads();
  const double limit = q.p <= 1.0 ? fmax(q.p * found_m, 1e-300) : INFINITY;
  // the least value that min-p keeps, as a key
  uint32_t least = kKeyLowest;
  if (q.m > 0.0) {
    const double xm = fmin(mx + q.t * log(q.m), (double)mx);
    float f = (float)fmax(xm, -(double)FLT_MAX);
    uint32_t k = key_of(f + 0.0f);
    if ((double)f < xm) ++k;
    least = k;
  }
  const double bin_m = fmin(qtop - floor((double)of_key(least) * q.c), (double)(kBins - 1));
  const bool ends = tid < kBins && (up.n > q.k || up.m >= limit || tid == (int)bin_m);
  // the first bin that is not kept as a whole
  if (ends) atomicMin(&found_d, (uint32_t)tid);
  __syncthreads();
  const int crit = (int)found_d;  // < kBins: min-p's bin is one of them
  __syncthreads();
  if (tid == crit) {
    found_n = up.n - n;
    found_m = up.m - m;
    list_n = n;
  }
  if (tid < a.slices) skept[tid] = 0;
  __syncthreads();
  const uint32_t bin_n = list_n;
  uint32_t room = q.k - found_n;         // tokens that may still be kept
  double left = limit - found_m;         // mass in front of a kept one stays below it
  const uint32_t bin_lo = crit == kBins - 1 ? kKeyLowest : first_key(qtop - crit, q.c);
  const uint32_t bin_hi = crit == 0 ? key_of(mx) : first_key(qtop - crit + 1.0, q.c) - 1;
  __syncthreads();

  // select inside the bin: keys lo .. hi hold the end
  uint32_t lo = bin_lo, hi = bin_hi, now = bin_n;
  bool listed = false, whole = false;
  auto each_row = [&](uint32_t klo, uint32_t khi, auto f) {
    for (int i = tid * kPer; i < a.V; i += kSlice) {
      float x[kPer];
      load8<TYPE>(a, r, i, x);
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        const uint32_t key = key_of(x[k]);
        if (key >= klo && key <= khi) f(key, i + k);
      }
    }
  };
  auto each = [&](auto f) {
    if (listed) {
      for (uint32_t i = tid; i < list_n; i += kNT) {
        const uint32_t key = list_key[i];
        if (key >= lo && key <= hi) f(key, list_idx[i]);
      }
    } else {
      each_row(lo, hi, f);
    }
  };
  auto gather = [&]() {
    __syncthreads();
    if (tid == 0) list_n = 0;
    __syncthreads();
    whole = lo == bin_lo && hi == bin_hi;
    each_row(lo, hi, [&](uint32_t key, int i) {
      const uint32_t at = atomicAdd(&list_n, 1u);
      if (at < kList) {
        list_key[at] = key;
        list_idx[at] = i;
      }
    });
    __syncthreads();
    listed = true;
  };
  if (now <= kList) gather();
  bool cut = now > room || left < INFINITY;  // (otherwise min-p alone ends the row here)
  while (cut && lo < hi) {
    const int bits = 32 - __clz(hi - lo), shift = max(bits - 10, 0);
    __syncthreads();
    dcnt[tid] = 0;
    dmass[tid] = 0;
    __syncthreads();
    each([&](uint32_t key, int) {
      const uint32_t d = (hi - key) >> shift;
      atomicAdd(&dcnt[d], 1u);
      atomicAdd(&dmass[d], fixed(weight(of_key(key), q.c, top, table)));
    });
    __syncthreads();
    const uint32_t dn = dcnt[tid];
    const double dm = (double)dmass[tid];
    const Sums su = block_scan(dn, dm, rn, rm);
    if (tid == 0) found_d = kDigits;
    __syncthreads();
    if (dn > 0 && (su.n > room || su.m >= left)) atomicMin(&found_d, (uint32_t)tid);
    __syncthreads();
    const uint32_t d = found_d;
    __syncthreads();
    if (d == kDigits) {  // all of these are kept
      cut = false;
      break;
    }
    if (tid == (int)d) {
      found_n = su.n - dn;
      found_m = su.m - dm;
      found_i = (int)dn;
    }
    __syncthreads();
    room -= found_n;
    left -= found_m;
    now = (uint32_t)found_i;
    const uint32_t h0 = hi;
    hi = h0 - (d << shift);
    lo = max(lo, hi - ((1u << shift) - 1));
    if (!listed && now <= kList) gather();
  }
  // equal values: the first ones by index
  uint32_t key = lo;
  int last = 0x7fffffff;
  if (cut) {
    const double w = (double)fixed(weight(of_key(key), q.c, top, table));
    uint32_t keep = min(room, now);
    if (w > 0.0 && left < INFINITY) {
      const double by_mass = ceil(left / w);
      keep = (uint32_t)fmin((double)keep, fmax(by_mass, 0.0));
    }
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
        const Sums su = block_scan(dn, 0.0, rn, rm);
        if (su.n >= keep && su.n - dn < keep) {
          found_i = tid;
          found_n = su.n - dn;
        }
        __syncthreads();
        if (level == 1) {
          base = found_i;
          keep -= found_n;
        } else {
          last = (base << 10) + found_i;
        }
      }
    }
  }
  if (key < least) {  // min-p ends it first
    key = least;
    last = 0x7fffffff;
  }
  __syncthreads();

  // each slice's kept mass in its own unit: whole bins, and its part of the bin
  auto keeps = [&](uint32_t k, int i) { return k > key || (k == key && i <= last); };
  for (int s = wave; s < a.slices; s += kNT / 64) {
    if (smax[s] == -INFINITY) continue;
    const double shift = qtop - floor((double)smax[s] * q.c);
    const double bins = fmin(fmax(crit - shift, 0.0), (double)kBins);
    unsigned long long sum = 0;
    const long long at = ((long long)r * a.slices + s) * kBins;
    for (int b = lane; b < (int)bins; b += 64) sum += a.mass[at + b];
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (lane == 0 && sum) atomicAdd(&skept[s], sum);
  }
  auto own_top = [&](int s) { return octave(floor((double)smax[s] * q.c)); };
  auto add = [&](uint32_t k, int i) {
    if (!keeps(k, i)) return;
    const int s = i / kSlice;
    atomicAdd(&skept[s], fixed(weight(of_key(k), q.c, own_top(s), table)));
  };
  if (whole) {
    for (uint32_t i = tid; i < list_n; i += kNT) add(list_key[i], list_idx[i]);
  } else {
    each_row(bin_lo, bin_hi, add);
  }
  __syncthreads();
  auto unit = [&](int s) { return ldexp(1.0, (int)fmax((own_top(s) - top) / kSub, -2000.0)); };
  double total = 0.0;
  for (int s = 0; s < a.slices; ++s)
    if (skept[s]) total += unit(s) * (double)skept[s];
  if (tid == 0 && a.probs)
    a.kept[r] = Kept{q.c, top, (double)(1ull << kFrac) / total, key, last};

  for (int d = 0; d < a.draws; ++d) {
    // the slice, then the token
    const double want = (double)a.u[(long long)r * a.draws + d] * total;
    double upto = 0.0, before = 0.0;
    int at = 0;
    bool hit = false;
    for (int s = 0; s < a.slices && !hit; ++s) {
      if (!skept[s]) continue;
      before = upto;
      upto += unit(s) * (double)skept[s];
      at = s;
      hit = upto > want;
    }
    const double rest = hit ? (want - before) / unit(at) : INFINITY;
    float x[kPer];
    const int i0 = at * kSlice + tid * kPer;
    load8<TYPE>(a, r, i0, x);
    unsigned long long w[kPer], sum = 0;
    const double st = own_top(at);
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      w[k] = 0;
      if (x[k] != -INFINITY && keeps(key_of(x[k]), i0 + k)) w[k] = fixed(weight(x[k], q.c, st, table));
      sum += w[k];
    }
    unsigned long long c = block_scan_u64(sum, ru) - sum;
    if (tid == 0) {
      found_d = 0xffffffffu;  // the first beyond `rest`
      found_i = 0;            // the last of any weight
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      c += w[k];
      if (w[k]) {
        if ((double)c > rest) atomicMin(&found_d, (uint32_t)(i0 + k));
        atomicMax(&found_i, i0 + k);
      }
    }
    __syncthreads();
    if (tid == 0)
      a.tokens[(long long)r * a.draws + d] =
          found_d != 0xffffffffu ? (int)found_d : found_i;
    __syncthreads();
  }
}

template <int TYPE>
__global__ __launch_bounds__(kNT) void probs_kernel(Args a) {
  __shared__ double table[kSub];
  const int r = blockIdx.x / a.slices, s = blockIdx.x % a.slices;
  const int i0 = s * kSlice + threadIdx.x * kPer;
  float x[kPer];
  load8<TYPE>(a, r, i0, x);
  fill_table(table);
  const Kept k = a.kept[r];
  __syncthreads();
  float p[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const uint32_t key = key_of(x[j]);
    const bool kept = x[j] != -INFINITY && (key > k.key || (key == k.key && i0 + j <= k.last));
    p[j] = kept ? (float)(weight(x[j], k.c, k.top, table) * k.scale) : 0.0f;
  }
  float *out = a.probs + (long long)r * a.V + i0;
  if (a.V % 4 == 0 && i0 + kPer <= a.V) {
    reinterpret_cast<float4 *>(out)[0] = make_float4(p[0], p[1], p[2], p[3]);
    reinterpret_cast<float4 *>(out)[1] = make_float4(p[4], p[5], p[6], p[7]);
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (i0 + j < a.V) out[j] = p[j];
  }
}

static size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

struct Layout {
  size_t smax, cnt, mass, kept, bytes;
  Layout(long long R, int V) {
    const size_t n = (size_t)R * ((V + kSlice - 1) / kSlice);
    smax = 0;
    cnt = smax + align256(n * sizeof(float));
    mass = cnt + align256(n * kBins * sizeof(uint32_t));
    kept = mass + align256(n * kBins * sizeof(unsigned long long));
    bytes = kept + align256((size_t)R * sizeof(Kept));
  }
};

template <int TYPE>
int launch(const Args &a, hipStream_t st) {
  const unsigned grid = (unsigned)(a.R * a.slices);
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
  a.type = elem_type;
  a.R = R;
  a.V = V;
  a.draws = draws;
  a.slices = (V + kSlice - 1) / kSlice;
  if ((long long)R * a.slices * kNT >= (1LL << 32)) return fail_arg("too many rows for one call");
  const int size = elem_type == kF32 ? 4 : 2;
  a.vec = (uintptr_t)rows % 16 == 0 && row_stride * size % 16 == 0;
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
  a.cnt = (uint32_t *)(ws + lay.cnt);
  a.mass = (unsigned long long *)(ws + lay.mass);
  a.kept = (Kept *)(ws + lay.kept);
  hipStream_t st = (hipStream_t)stream;
  switch (elem_type) {
    case kF32: return launch<kF32>(a, st);
    case kBF16: return launch<kBF16>(a, st);
    default: return launch<kFP16>(a, st);
  }
}
