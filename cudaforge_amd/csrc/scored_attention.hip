// scored_attention.hip -- the entry points of scored_attention.hpp: argument
// checks, the plan of blocks and splits, and the workspace.
#include "scored_attention.hpp"

#include <algorithm>
#include <cmath>

namespace cfa {
namespace scored {

extern template int launch<64, BF16>(const Args &, bool, unsigned, hipStream_t);
extern template int launch<128, BF16>(const Args &, bool, unsigned, hipStream_t);
extern template int launch<64, FP16>(const Args &, bool, unsigned, hipStream_t);
extern template int launch<128, FP16>(const Args &, bool, unsigned, hipStream_t);

static size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

struct Plan {
  int TQ, splits;
  long long blocks;  // blocks to launch
  bool one;          // one 16-row query tile a wave
  size_t part_bytes(long long tokens, int Hq, int D) const {
    return align256((size_t)splits * tokens * Hq * D * 4);
  }
  size_t bytes(long long tokens, int Hq, int D) const {
    return splits == 1 ? 0
                       : part_bytes(tokens, Hq, D) +
                             align256((size_t)splits * tokens * Hq * sizeof(float2));
  }
};

// Query rows of a block (256 in two tiles a wave, or 128 or 64 in one) and splits of
// the keys, by the time that they would take.  In us, as measured over prompts of 128
// to 4096 tokens and trees of 31 and 63 nodes: a work-group's first transfers and
// output, and each of its tiles,
//    rows           256         128         64
//    head_dim 128   6.8 + 1.6   4.3 + 1.1   3.5 + 1.0
//    head_dim 64    4.5 + 1.4   3.0 + 1.0   2.5 + 0.84
// one work-group a CU (of one tile and head_dim 64, two with 1.4 to 2 times the
// throughput); a merge's launch 6, and the partials' bytes, written and read.  A call
// takes at least its longest work-group, the sum of all over the CUs (a prompt's
// have half the tiles of its last on average; trees' and tokens' come in whole
// rounds), and the tiles' bytes at 6 TB/s, from whichever cache.
// Fewer rows must gain 5%: they read keys and values more often.  us with 256 / 128 /
// 64 rows, head_dim 128: a prompt of 512 24.0 / 17.5 / 15.5, of 1024 36.5 / 26.2 / 29.7,
// of 2048 62 / 56 / 88, four of 512 24.4 / 29.9 / 40; one tree of 63 nodes behind 4096
// 26.9 / 21.8 / 21.4, 24 of them 159 / 193 / 223.  Splits, of a prompt's 64 tokens behind
// 8000: 208 without, 28 with 16.
// `longest` bounds a sequence's queries; tokens is the number of all.
static Plan plan(long long tokens, long long longest, int B, int G, int Hkv, int D, int max_keys,
                 int window, int num_splits, bool tree) {
  struct Rows {
    int rows;
    double first, tile, share;
  };
  static constexpr Rows kRows[2][3] = {
      {{kMaxRows, 6.8, 1.6, 1.0}, {kMaxRows / 2, 4.3, 1.1, 1.0}, {kRowsOneTile, 3.5, 1.0, 1.0}},
      {{kMaxRows, 4.5, 1.4, 1.0}, {kMaxRows / 2, 3.0, 1.0, 1.4}, {kRowsOneTile, 2.5, 0.84, 2.0}}};
  const double merged = (double)tokens * Hkv * G * D * 8 / 5.2e6;  // a split's bytes
  Plan p{};
  double least = 0.0;
  for (int i = 0; i < 3; ++i) {
    const Rows &c = kRows[D == 64][i];
    // (the fewest rows that hold a sequence's, or else a token's heads, are the last)
    const bool enough = i < 2 && std::max<long long>(longest, 1) * G <= kRows[D == 64][i + 1].rows;
    if (enough || (i > 0 && G > c.rows)) continue;
    const int TQ = (int)std::max(1LL, std::min(longest, (long long)c.rows / G));
    const long long blocks =
        tree ? (long long)B * ((longest + TQ - 1) / TQ) : tokens / TQ + B;
    const long long busy =  // blocks that have queries, about
        tree ? blocks
             : std::max(tokens / TQ + std::min<long long>(B, tokens) / 2,
                        std::max<long long>(1, std::min<long long>(B, tokens)));
    int tiles = (int)std::max(1LL, ((long long)max_keys + kKT - 1) / kKT);
    double mean = tiles;
    if (window > 0)
      mean = tiles = (int)std::min<long long>(
          tiles, ((long long)window + (tree ? 64 : TQ) + kKT - 2) / kKT + 1);
    else if (!tree)
      mean = std::max(1.0, tiles - 0.5 * (double)std::min<long long>(longest, max_keys) / kKT);
    const double cus = abi::device_cu_count(), items = (double)std::max(1LL, busy * Hkv);
    const double bytes = items * mean * kKT * D * 4 / 6e6;
    long long n = num_splits > 0 ? std::min(num_splits, tiles) : 1;
    while (true) {
      const long long per = (tiles + n - 1) / n;
      const double longest_of = c.first + c.tile * (double)per;
      const double a_cu = items * (double)n / cus;
      double time = std::max(longest_of, bytes);
      if (tree)
        time = std::max(time, std::ceil(a_cu) / c.share * longest_of);
      else
        time = std::max(time, a_cu / c.share * (std::max(c.first, 6.0) +
                                                c.tile * std::max(1.0, mean / (double)n)));
      if (n > 1) time += 6.0 + (double)n * merged;
      if (p.splits == 0 || time < least * (p.TQ == TQ ? 1.0 : 0.95)) {
        p.TQ = TQ;
        p.blocks = blocks;
        p.one = i > 0;
        p.splits = (int)n;
        least = time;
      }
      // (the next number of splits that makes them shorter, up to 4 rounds)
      if (num_splits > 0 || per == 1) break;
      n = (tiles + per - 2) / (per - 1);
      if (items * (double)n > 4.0 * c.share * cus) break;
    }
  }
  return p;
}

static int check_scores(float sm_scale, float soft_cap, int window) {
  using namespace cfa::abi;
  if (!std::isfinite(sm_scale)) return fail_arg("sm_scale must be finite");
  if (!(soft_cap == 0.0f || (soft_cap >= 1e-6f && std::isfinite(soft_cap))))
    return fail_arg("soft_cap must be 0 (no cap) or finite and at least 1e-6");
  // (the factor of a product in log2 units: infinite, it would make NaN of a 0)
  if (!std::isfinite((soft_cap > 0.0f ? 2.0f * (sm_scale / soft_cap) : sm_scale) * 1.4426951f))
    return fail_arg("sm_scale is out of fp32's range (of soft_cap, where there is one)");
  if (window < 0) return fail_arg("window must not be negative (0: none)");
  return CFA_OK;
}

static int check_heads(int Hq, int Hkv, int D) {
  using namespace cfa::abi;
  if (D != 64 && D != 128) return fail_arg("head_dim must be 64 or 128");
  if (Hkv <= 0 || Hq <= 0 || Hq % Hkv)
    return fail_arg("n_q_heads must be a positive multiple of n_kv_heads");
  if (Hq / Hkv > kMaxRows) return fail_arg("n_q_heads / n_kv_heads must be at most 256");
  return CFA_OK;
}

static int check_pool(int num_blocks, int num_layers, int layer, int block_size, int max_blocks) {
  using namespace cfa::abi;
  if (block_size <= 0 || block_size % 16) return fail_arg("block_size must be a multiple of 16");
  if (num_blocks <= 0 || num_layers <= 0 || layer < 0 || layer >= num_layers)
    return fail_arg("bad pool geometry (num_blocks, num_layers, layer)");
  if (max_blocks <= 0) return fail_arg("max_blocks_per_seq must be positive");
  if ((long long)max_blocks * block_size > 0x7fffff00LL)
    return fail_arg("a block table must cover less than 2^31 - 256 positions");
  return CFA_OK;
}

static int run(Args &a, const Plan &p, int D, int fp16, float sm_scale, float soft_cap,
               void *workspace, size_t workspace_bytes, void *stream) {
  using namespace cfa::abi;
  if ((((uintptr_t)a.q | (uintptr_t)a.kpool | (uintptr_t)a.vpool | (uintptr_t)a.out) & 15) != 0)
    return fail_arg("q, the pools and out must be 16-byte aligned");
  a.TQ = p.TQ;
  a.splits = p.splits;
  a.cap = soft_cap;
  a.scale = soft_cap > 0.0f ? sm_scale / soft_cap : sm_scale;
  if (soft_cap > 0.0f) {
    const double t = (double)sm_scale / soft_cap, unit = soft_cap * 1.4426950408889634 * t;
    a.k0 = (float)(unit * kT0);
    a.k1 = (float)(unit * kT1 * t * t);
    a.k2 = (float)(unit * kT2 * t * t * t * t);
    a.k3 = (float)(unit * kT3 * t * t * t * t * t * t);
    // a coefficient that fp32 does not hold (scores far below the cap) is left
    // out, and the polynomial kept to where its term is below 5e-7
    double far = kTanhSmall;
    if (std::fabs(a.k3) < 1e-37f) a.k3 = 0.0f, far = 0.14;
    if (std::fabs(a.k2) < 1e-37f) a.k2 = 0.0f, far = 0.04;
    if (std::fabs(a.k1) < 1e-37f) a.k1 = 0.0f, far = 0.001;
    const double small = t != 0.0 ? far / std::fabs(t) : 1e18;
    a.small = (float)std::min(small, 1e18);  // (x^2 stays in fp32's range)
    // a coefficient past fp32's range (scores far above the cap): no polynomial
    if (!std::isfinite(a.k1) || !std::isfinite(a.k2) || !std::isfinite(a.k3)) a.small = -1.0f;
  }
  const long long grid = (long long)p.splits * a.Hkv * p.blocks;
  if (grid * kNT >= (1LL << 32)) return fail_arg("too many queries for one call");
  if (p.splits > 1) {
    if ((long long)a.T * a.Hq * (D / 4) >= (1LL << 32))  // the merge's threads
      return fail_arg("too many queries for one call");
    if (!workspace || workspace_bytes < p.bytes(a.T, a.Hq, D))
      return fail_arg("workspace too small (see the entry point's _workspace_size)");
    if (((uintptr_t)workspace & 15) != 0) return fail_arg("workspace must be 16-byte aligned");
    a.part_o = (float *)workspace;
    a.part_ml = (float2 *)((char *)workspace + p.part_bytes(a.T, a.Hq, D));
  }
  a.past = (long long)p.splits * a.T * a.Hq * D * 4 <= 24LL << 20;
  hipStream_t st = (hipStream_t)stream;
  if (D == 128)
    return fp16 ? launch<128, FP16>(a, p.one, (unsigned)grid, st)
                : launch<128, BF16>(a, p.one, (unsigned)grid, st);
  return fp16 ? launch<64, FP16>(a, p.one, (unsigned)grid, st)
              : launch<64, BF16>(a, p.one, (unsigned)grid, st);
}

}  // namespace scored
}  // namespace cfa

using namespace cfa::scored;

extern "C" size_t cfa_tree_attention_scored_workspace_size(int B, int N, int n_q_heads,
                                                           int n_kv_heads, int head_dim,
                                                           int max_keys, int window,
                                                           int num_splits) {
  cfa::abi::clear_error();
  if (B <= 0 || N <= 0 || window < 0 || check_heads(n_q_heads, n_kv_heads, head_dim) != CFA_OK)
    return 0;
  const Plan p = plan((long long)B * N, N, B, n_q_heads / n_kv_heads, n_kv_heads, head_dim, max_keys,
                      window, num_splits, true);
  return p.bytes((long long)B * N, n_q_heads, head_dim);
}

extern "C" int cfa_tree_attention_scored(
    const void *q, const void *k_pool, const void *v_pool, int fp16, const int32_t *block_tables,
    int max_blocks_per_seq, const int32_t *ctx_lens, int num_blocks, int num_layers, int layer,
    int block_size, const uint64_t *tree_mask, int64_t tree_mask_stride_b, int B, int N,
    int first_node, int n_q_heads, int n_kv_heads, int head_dim, float sm_scale, float soft_cap,
    const float *alibi_slopes, int window, int max_keys, int num_splits, void *out,
    void *workspace, size_t workspace_bytes, void *stream) {
  using namespace cfa::abi;
  clear_error();
  if (!q || !k_pool || !v_pool || !block_tables || !ctx_lens || !tree_mask || !out)
    return fail_arg("null pointer argument");
  if (B <= 0 || N <= 0 || N > 64) return fail_arg("need B > 0 and 0 < N <= 64 tree nodes");
  if (first_node < 0 || first_node >= N) return fail_arg("need 0 <= first_node < N");
  if (int rc = check_heads(n_q_heads, n_kv_heads, head_dim)) return rc;
  if (int rc = check_pool(num_blocks, num_layers, layer, block_size, max_blocks_per_seq)) return rc;
  if (int rc = check_scores(sm_scale, soft_cap, window)) return rc;
  if (max_keys < N) return fail_arg("max_keys must be at least N (context + tree tokens)");
  if ((long long)max_blocks_per_seq * block_size < max_keys)
    return fail_arg("max_blocks_per_seq * block_size must cover max_keys");
  if (num_splits < 0) return fail_arg("num_splits must not be negative");
  Args a{};
  a.q = (const uint16_t *)q;
  a.kpool = (const uint16_t *)k_pool;
  a.vpool = (const uint16_t *)v_pool;
  a.bt = block_tables;
  a.ctx = ctx_lens;
  a.mask = tree_mask;
  a.mask_sb = tree_mask_stride_b;
  a.slopes = alibi_slopes;
  a.out = (uint16_t *)out;
  a.Nq = N - first_node;
  if ((long long)B * a.Nq >= (1LL << 31)) return fail_arg("too many queries for one call");
  a.T = B * a.Nq;
  a.B = B;
  a.N = N;
  a.q0 = first_node;
  a.Hq = n_q_heads;
  a.Hkv = n_kv_heads;
  a.G = n_q_heads / n_kv_heads;
  a.max_blocks = max_blocks_per_seq;
  a.num_blocks = num_blocks;
  a.num_layers = num_layers;
  a.layer = layer;
  a.bs = block_size;
  a.window = window;
  const Plan p = plan(a.T, a.Nq, B, a.G, n_kv_heads, head_dim, max_keys, window, num_splits,
                      true);
  return run(a, p, head_dim, fp16, sm_scale, soft_cap, workspace, workspace_bytes, stream);
}

extern "C" size_t cfa_prompt_attention_workspace_size(int T, int B, int n_q_heads, int n_kv_heads,
                                                      int head_dim, int max_query, int max_keys,
                                                      int window, int num_splits) {
  cfa::abi::clear_error();
  if (B <= 0 || T <= 0 || max_query <= 0 || window < 0 ||
      check_heads(n_q_heads, n_kv_heads, head_dim) != CFA_OK)
    return 0;
  const Plan p = plan(T, std::min(max_query, T), B, n_q_heads / n_kv_heads, n_kv_heads, head_dim,
                      max_keys, window, num_splits, false);
  return p.bytes(T, n_q_heads, head_dim);
}

extern "C" int cfa_prompt_attention(
    const void *q, const void *k_pool, const void *v_pool, int fp16, const int32_t *block_tables,
    int max_blocks_per_seq, const int32_t *ctx_lens, int num_blocks, int num_layers, int layer,
    int block_size, const int32_t *cu_seqlens, int T, int B, int n_q_heads, int n_kv_heads,
    int head_dim, float sm_scale, float soft_cap, const float *alibi_slopes, int window,
    int max_query, int max_keys, int num_splits, void *out, void *workspace,
    size_t workspace_bytes, void *stream) {
  using namespace cfa::abi;
  clear_error();
  if (T < 0 || B < 0) return fail_arg("need T, B >= 0");
  if (int rc = check_heads(n_q_heads, n_kv_heads, head_dim)) return rc;
  if (int rc = check_pool(num_blocks, num_layers, layer, block_size, max_blocks_per_seq)) return rc;
  if (int rc = check_scores(sm_scale, soft_cap, window)) return rc;
  if (max_query <= 0 || max_keys <= 0) return fail_arg("max_query and max_keys must be positive");
  if (num_splits < 0) return fail_arg("num_splits must not be negative");
  if (T == 0 || B == 0) return CFA_OK;
  if (!q || !k_pool || !v_pool || !block_tables || !ctx_lens || !cu_seqlens || !out)
    return fail_arg("null pointer argument");
  Args a{};
  a.q = (const uint16_t *)q;
  a.kpool = (const uint16_t *)k_pool;
  a.vpool = (const uint16_t *)v_pool;
  a.bt = block_tables;
  a.ctx = ctx_lens;
  a.cu = cu_seqlens;
  a.slopes = alibi_slopes;
  a.out = (uint16_t *)out;
  a.T = T;
  a.B = B;
  a.Hq = n_q_heads;
  a.Hkv = n_kv_heads;
  a.G = n_q_heads / n_kv_heads;
  a.max_blocks = max_blocks_per_seq;
  a.num_blocks = num_blocks;
  a.num_layers = num_layers;
  a.layer = layer;
  a.bs = block_size;
  a.window = window;
  const Plan p = plan(T, std::min(max_query, T), B, a.G, n_kv_heads, head_dim, max_keys, window,
                      num_splits, false);
  return run(a, p, head_dim, fp16, sm_scale, soft_cap, workspace, workspace_bytes, stream);
}
