// Group norm of one position per sample: gradient.
#include "group_norm_rows.cuh"

void hdc::gn_rows_bwd(int dtype, const GnParams& p, const GnRowPlan& r, int ve, cudaStream_t s) {
  if (dtype == HDC_F32) gn_rows<float, true>(p, r, ve, s);
  else gn_rows<__nv_bfloat16, true>(p, r, ve, s);
}
