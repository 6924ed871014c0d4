// k_attn_shared_f32.hip -- the kernels of sg_attn_shared.h for float32 queries.
#include "sg_attn_shared.h"

namespace sgk {

hipError_t attn_shared_f32(const sg_attn_shared_args& a, const sg_attn_list& list, bool q8, int D, hipStream_t s) {
  return sga::launch_type<float>(a, list, q8, D, s);
}

}  // namespace sgk
