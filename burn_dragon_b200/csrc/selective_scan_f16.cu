#include "selective_scan.cuh"

namespace bdh {

BDH_SCAN_OF(, __half)

}  // namespace bdh
