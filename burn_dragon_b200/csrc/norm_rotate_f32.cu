#include "norm_rotate.cuh"

namespace bdh {

BDH_NORM_ROTATE_OF(, float)

}  // namespace bdh
