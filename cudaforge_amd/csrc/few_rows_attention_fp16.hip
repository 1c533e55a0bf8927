// few_rows_attention_fp16.hip -- the fp16 kernels of few_rows_attention.hpp.
#include "few_rows_attention.hpp"

namespace cfa {
namespace scored {
template int launch_few<64, FP16>(const Args &, bool, unsigned, hipStream_t);
template int launch_few<128, FP16>(const Args &, bool, unsigned, hipStream_t);
}  // namespace scored
}  // namespace cfa
