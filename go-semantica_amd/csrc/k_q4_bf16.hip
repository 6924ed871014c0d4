// k_q4_bf16.hip -- the kernels of sg_q4.h for bf16 rows.
#include "sg_q4.h"

namespace sgk {

hipError_t matmul_q4_bf16(const sg_q4_args& a, hipStream_t s) { return sgq::by_weight<sgp::bf16_t>(a, s); }

}  // namespace sgk
