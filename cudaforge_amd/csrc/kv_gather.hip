// kv_gather.hip -- rows of the paged cache, read back token by token: sequences'
// keys and values out of their pages into packed [T, Hkv, D] tensors of 16 bits,
// from pools of the same type or of e4m3 codes with a scale a row (e4m3.hpp).
//
// Token j of sequence b is the row at slot start[b] + j of
// pool[block][layer][kv_head][slot][D]; out = code 2^(byte - 127), exact in bf16.
//
// Bound: HBM.  A row's D codes are read and 2 D bytes written once; 16 codes a lane, a
// wave a token, whose page is looked up once for its heads.  8 sequences of 4096 tokens,
// 8 heads of 128 (202 MB): 45 us, 4.5 TB/s; one of 8149 tokens 12, 93 tokens 3.4.
#include <hip/hip_runtime.h>

#include "abi_internal.hpp"
#include "e4m3.hpp"
#include "packed_tokens.hpp"

namespace cfa {
namespace gather {

constexpr int kWaves = 4;

struct Args {
  const uint8_t *kpool, *vpool;
  const uint8_t *ks, *vs;  // null: pools of 16 bits
  const int32_t *bt, *start, *cu;
  uint8_t *k_out, *v_out;
  int T, B, n;
  int Hkv, D, max_blocks, num_blocks, num_layers, layer, bs;
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// One wave = one token: its K and V rows, 16 elements a lane.
template <class T, bool E4M3>
__global__ __launch_bounds__(kWaves * 64) void kv_gather_kernel(Args a) {
  const int lane = threadIdx.x & 63;
  const int t = blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (t >= a.T) return;
  int b, j;
  if (!place_token(a, t, lane, b, j)) return;
  const long long slot = (long long)a.start[b] + j;
  const long long page = slot / a.bs;
  int blk = -1;
  if (slot >= 0 && page < a.max_blocks) blk = a.bt[(long long)b * a.max_blocks + page];
  const bool mapped = blk >= 0 && blk < a.num_blocks;
  const int per = a.D / 16, items = 2 * a.Hkv * per;
  for (int i = lane; i < items; i += 64) {
    const int c = i % per, head = i / per % a.Hkv;
    const bool is_v = i >= a.Hkv * per;
    const long long row = (((long long)blk * a.num_layers + a.layer) * a.Hkv + head) * a.bs +
                          (slot - page * a.bs);
    u32x4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
    if (mapped) {
      const uint8_t *pool = is_v ? a.vpool : a.kpool;
      if constexpr (E4M3) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(pool + row * a.D + c * 16);
        const float s = e4m3::scale((is_v ? a.vs : a.ks)[row]);
        lo = u32x4{e4m3::unpack_pair<T, false>(w.x, s), e4m3::unpack_pair<T, true>(w.x, s),
                   e4m3::unpack_pair<T, false>(w.y, s), e4m3::unpack_pair<T, true>(w.y, s)};
        hi = u32x4{e4m3::unpack_pair<T, false>(w.z, s), e4m3::unpack_pair<T, true>(w.z, s),
                   e4m3::unpack_pair<T, false>(w.w, s), e4m3::unpack_pair<T, true>(w.w, s)};
      } else {
        const u32x4 *p = reinterpret_cast<const u32x4 *>(pool + (row * a.D + c * 16) * 2);
        lo = p[0];
        hi = p[1];
      }
    }
    u32x4 *out = reinterpret_cast<u32x4 *>((is_v ? a.v_out : a.k_out) +
                                           (((long long)t * a.Hkv + head) * a.D + c * 16) * 2);
    __builtin_nontemporal_store(lo, out);
    __builtin_nontemporal_store(hi, out + 1);
  }
}

template <class T>
int launch(const Args &a, hipStream_t st) {
  const dim3 grid((unsigned)(((long long)a.T + kWaves - 1) / kWaves));
  if (a.ks)
    CFA_LAUNCH("kv_gather", (kv_gather_kernel<T, true>), grid, dim3(kWaves * 64), 0, st, a);
  else
    CFA_LAUNCH("kv_gather", (kv_gather_kernel<T, false>), grid, dim3(kWaves * 64), 0, st, a);
  return CFA_OK;
}

}  // namespace gather
}  // namespace cfa

extern "C" int cfa_kv_gather(const void *k_pool, const void *v_pool, const uint8_t *k_scales,
                             const uint8_t *v_scales, int fp16, int num_blocks, int num_layers,
                             int layer, int n_kv_heads, int block_size, int head_dim,
                             const int32_t *block_tables, int max_blocks_per_seq,
                             const int32_t *starts, const int32_t *cu_seqlens, int T, int B,
                             void *k_out, void *v_out, void *stream) {
  using namespace cfa::abi;
  clear_error();
  if (T < 0 || B < 0 || n_kv_heads <= 0 || n_kv_heads > 65536)
    return fail_arg("need T, B >= 0 and 1 to 65536 heads");
  if (head_dim <= 0 || head_dim % 16 || head_dim > 256)
    return fail_arg("head_dim must be a multiple of 16, at most 256");
  if (num_blocks <= 0 || num_layers <= 0 || layer < 0 || layer >= num_layers || block_size <= 0 ||
      max_blocks_per_seq < 0)
    return fail_arg("bad pool geometry (num_blocks, num_layers, layer, block_size)");
  if (!k_scales != !v_scales) return fail_arg("k_scales and v_scales go together");
  if (T == 0 || B == 0) return CFA_OK;
  if (!k_pool || !v_pool || !starts || !k_out || !v_out ||
      (max_blocks_per_seq > 0 && !block_tables))
    return fail_arg("null pointer argument");
  if (!cu_seqlens && T % B) return fail_arg("without cu_seqlens T must be a multiple of B");
  if ((((uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)k_out | (uintptr_t)v_out) & 15) != 0)
    return fail_arg("the pools and outputs must be 16-byte aligned");
  // (a launch has less than 2^32 threads)
  if ((T + 3LL) / 4 >= 1 << 24) return fail_arg("too many tokens for one call (about 2^26)");
  cfa::gather::Args a{};
  a.kpool = (const uint8_t *)k_pool;
  a.vpool = (const uint8_t *)v_pool;
  a.ks = k_scales;
  a.vs = v_scales;
  a.bt = block_tables;
  a.start = starts;
  a.cu = cu_seqlens;
  a.k_out = (uint8_t *)k_out;
  a.v_out = (uint8_t *)v_out;
  a.T = T;
  a.B = B;
  a.n = T / B;
  a.Hkv = n_kv_heads;
  a.D = head_dim;
  a.max_blocks = max_blocks_per_seq;
  a.num_blocks = num_blocks;
  a.num_layers = num_layers;
  a.layer = layer;
  a.bs = block_size;
  hipStream_t st = (hipStream_t)stream;
  return fp16 ? cfa::gather::launch<cfa::FP16>(a, st) : cfa::gather::launch<cfa::BF16>(a, st);
}
