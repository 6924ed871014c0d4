// k_attn_shared_f16.hip -- the kernels of sg_attn_shared.h for fp16 queries.
#include "sg_attn_shared.h"

namespace sgk {

hipError_t attn_shared_f16(const sg_attn_shared_args& a, const sg_attn_list& list, bool q8, int D, hipStream_t s) {
  return sga::launch_type<_Float16>(a, list, q8, D, s);
}

}  // namespace sgk
