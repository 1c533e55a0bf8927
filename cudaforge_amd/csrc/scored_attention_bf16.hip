// scored_attention_bf16.hip -- the bf16 kernels of scored_attention.hpp.
#include "scored_attention.hpp"

namespace cfa {
namespace scored {
template int launch<64, BF16, false>(const Args &, bool, unsigned, hipStream_t);
template int launch<128, BF16, false>(const Args &, bool, unsigned, hipStream_t);
}  // namespace scored
}  // namespace cfa
