// Group norm of one position per sample: forward.
#include "group_norm_rows.cuh"

void hdc::gn_rows_fwd(int dtype, const GnParams& p, const GnRowPlan& r, int ve, cudaStream_t s) {
  if (dtype == HDC_F32) gn_rows<float, false>(p, r, ve, s);
  else gn_rows<__nv_bfloat16, false>(p, r, ve, s);
}
