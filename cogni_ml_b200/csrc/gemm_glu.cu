// The prefill product (gemm_prefill.cuh) with gate and up projection, activation and product in one launch: cogni_qmm_gemm_glu.
#include "gemm_prefill.cuh"

namespace cogni {

int launch_gemm_glu(const RowsCall &c, cudaStream_t s) {
  if (rows_kernel_takes(c)) return launch_gemm_rows_glu(c, s);
  return launch_gemm_form<kGlu>(c, s);
}

unsigned gemm_glu_timeouts() { return form_timeouts(); }
int gemm_glu_reset_timeouts() { return form_reset_timeouts(); }

}  // namespace cogni
