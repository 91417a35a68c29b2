#include "norm_rotate.cuh"

namespace bdh {

BDH_NORM_ROTATE_OF(, __nv_bfloat16)

}  // namespace bdh
