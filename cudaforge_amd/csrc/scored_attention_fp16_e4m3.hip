// scored_attention_fp16_e4m3.hip -- the fp16 kernels over e4m3 codes of scored_attention.hpp.
#include "scored_attention.hpp"

namespace cfa {
namespace scored {
template int launch<64, FP16, true>(const Args &, bool, unsigned, hipStream_t);
template int launch<128, FP16, true>(const Args &, bool, unsigned, hipStream_t);
}  // namespace scored
}  // namespace cfa
