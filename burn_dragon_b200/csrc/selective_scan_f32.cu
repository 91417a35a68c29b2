#include "selective_scan.cuh"

namespace bdh {

BDH_SCAN_OF(, float)

}  // namespace bdh
