// few_rows_attention_bf16.hip -- the bf16 kernels of few_rows_attention.hpp.
#include "few_rows_attention.hpp"

namespace cfa {
namespace scored {
template int launch_few<64, BF16>(const Args &, bool, unsigned, hipStream_t);
template int launch_few<128, BF16>(const Args &, bool, unsigned, hipStream_t);
}  // namespace scored
}  // namespace cfa
