// k_q4_f16.hip -- the kernels of sg_q4.h for fp16 rows.
#include "sg_q4.h"

namespace sgk {

hipError_t matmul_q4_f16(const sg_q4_args& a, hipStream_t s) { return sgq::by_weight<_Float16>(a, s); }

}  // namespace sgk
