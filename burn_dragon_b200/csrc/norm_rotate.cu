// C entries of the per-head norm and rotation (norm_rotate.cuh); each row type is compiled in a file of its own.
#include "norm_rotate.cuh"

namespace bdh {

BDH_NORM_ROTATE_OF(extern, float)
BDH_NORM_ROTATE_OF(extern, __half)
BDH_NORM_ROTATE_OF(extern, __nv_bfloat16)

}  // namespace bdh

using namespace bdh;

extern "C" int bdh_norm_rotate_fwd(const BdhNormRotateDesc* d, cudaStream_t s) {
  if (const int rc = checked(*d)) return rc;
  if (static_cast<long long>(d->B) * d->T == 0) return BDH_OK;
  switch (d->dtype) {
    case BDH_F32: return norm_rotate_fwd_of<float>(*d, s);
    case BDH_F16: return norm_rotate_fwd_of<__half>(*d, s);
  }
  return norm_rotate_fwd_of<__nv_bfloat16>(*d, s);
}

// Room for whichever kernel the pointers of the later call select.
extern "C" long long bdh_norm_rotate_scratch(const BdhNormRotateDesc* d, int want_weight, int want_bias, int want_angles) {
  if (d->B < 1 || d->T < 1 || d->Hq < 1 || d->Dh < 2) return 0;
  long long most = 0;
  for (int v : {4, 8})
    for (int nv : {1, 2, 4})
      for (int groups : {FEW, MANY}) {
        if (32 * v * nv < d->Dh) continue;
        const NormArgs a = args_for(*d, v, nv, groups);
        const BwdPlan p = bwd_plan(a, v * nv, want_weight || want_bias, want_bias || (want_weight && d->per_head), want_angles);
        most = p.partial + p.angles > most ? p.partial + p.angles : most;
      }
  return most;
}

extern "C" int bdh_norm_rotate_bwd(const BdhNormRotateDesc* d, float* dq_weight, float* dk_weight, float* dq_bias, float* dk_bias,
                                   float* dangles, float* scratch, cudaStream_t s) {
  if (const int rc = checked(*d)) return rc;
  if (static_cast<long long>(d->B) * d->T == 0) return BDH_ERR_ARGUMENT;
  if (dangles != nullptr && d->angles == nullptr) return BDH_ERR_ARGUMENT;
  const NormRotateGrads o{dq_weight, dk_weight, dq_bias, dk_bias, dangles, scratch};
  switch (d->dtype) {
    case BDH_F32: return norm_rotate_bwd_of<float>(*d, o, s);
    case BDH_F16: return norm_rotate_bwd_of<__half>(*d, o, s);
  }
  return norm_rotate_bwd_of<__nv_bfloat16>(*d, o, s);
}
