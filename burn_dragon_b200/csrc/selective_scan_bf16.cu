#include "selective_scan.cuh"

namespace bdh {

BDH_SCAN_OF(, __nv_bfloat16)

}  // namespace bdh
