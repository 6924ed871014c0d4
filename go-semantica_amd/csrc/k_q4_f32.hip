// k_q4_f32.hip -- the kernels of sg_q4.h for float32 rows.
#include "sg_q4.h"

namespace sgk {

hipError_t matmul_q4_f32(const sg_q4_args& a, hipStream_t s) { return sgq::by_weight<float>(a, s); }

}  // namespace sgk
