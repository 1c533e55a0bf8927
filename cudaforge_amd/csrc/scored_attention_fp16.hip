// scored_attention_fp16.hip -- the fp16 kernels of scored_attention.hpp.
#include "scored_attention.hpp"

namespace cfa {
namespace scored {
template int launch<64, FP16, false>(const Args &, bool, unsigned, hipStream_t);
template int launch<128, FP16, false>(const Args &, bool, unsigned, hipStream_t);
}  // namespace scored
}  // namespace cfa
