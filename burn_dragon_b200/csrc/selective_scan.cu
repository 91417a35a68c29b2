// C entries of the selective scan (selective_scan.cuh); each row type is compiled in a file of its own.
#include "selective_scan.cuh"

namespace bdh {

BDH_SCAN_OF(extern, float)
BDH_SCAN_OF(extern, __half)
BDH_SCAN_OF(extern, __nv_bfloat16)

}  // namespace bdh

using namespace bdh;

extern "C" void bdh_selective_scan_sizes(const BdhScanDesc* d, long long* marks, long long* fwd_scratch, long long* bwd_scratch) {
  *marks = *fwd_scratch = *bwd_scratch = 0;
  if (checked(*d) != BDH_OK) return;
  const Plan f = fwd_plan(*d), b = bwd_plan(*d);
  *marks = static_cast<long long>(d->B) * f.tiles * d->D * 4 * f.G;
  *fwd_scratch = seg_floats(*d, f);
  *bwd_scratch = seg_floats(*d, b) + bc_floats(*d, b) + da_floats(*d, b) + static_cast<long long>(d->B) * b.segs * d->D * 2;
}

extern "C" int bdh_selective_scan_fwd(const BdhScanDesc* d, float* marks, float* scratch, cudaStream_t s) {
  if (const int rc = checked(*d)) return rc;
  if (d->B == 0) return BDH_OK;
  if (d->T == 0) return BDH_ERR_ARGUMENT;
  switch (d->dtype) {
    case BDH_F32: return selective_scan_fwd_of<float>(*d, marks, scratch, s);
    case BDH_F16: return selective_scan_fwd_of<__half>(*d, marks, scratch, s);
  }
  return selective_scan_fwd_of<__nv_bfloat16>(*d, marks, scratch, s);
}

extern "C" int bdh_selective_scan_bwd(const BdhScanDesc* d, const float* marks, float* scratch, float* dA, float* dD, float* dbias, void* dB,
                                      void* dC, cudaStream_t s) {
  if (const int rc = checked(*d)) return rc;
  if (d->B == 0 || d->T == 0) return BDH_ERR_ARGUMENT;
  switch (d->dtype) {
    case BDH_F32: return selective_scan_bwd_of<float>(*d, marks, scratch, dA, dD, dbias, dB, dC, s);
    case BDH_F16: return selective_scan_bwd_of<__half>(*d, marks, scratch, dA, dD, dbias, dB, dC, s);
  }
  return selective_scan_bwd_of<__nv_bfloat16>(*d, marks, scratch, dA, dD, dbias, dB, dC, s);
}

extern "C" int bdh_selective_scan_step(const BdhScanDesc* d, const float* h, long long h_sb, float* out, long long out_sb,
                                       const unsigned char* active, cudaStream_t s) {
  if (const int rc = checked(*d)) return rc;
  if (d->B == 0) return BDH_OK;
  switch (d->dtype) {
    case BDH_F32: return selective_scan_step_of<float>(*d, h, h_sb, out, out_sb, active, s);
    case BDH_F16: return selective_scan_step_of<__half>(*d, h, h_sb, out, out_sb, active, s);
  }
  return selective_scan_step_of<__nv_bfloat16>(*d, h, h_sb, out, out_sb, active, s);
}
