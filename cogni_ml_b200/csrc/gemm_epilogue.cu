// The prefill product (gemm_prefill.cuh) with bias, activation and residual in the epilogue: cogni_qmm_gemm_epilogue.
#include "gemm_prefill.cuh"

namespace cogni {

int launch_gemm_epilogue(const RowsCall &c, cudaStream_t s) {
  if (rows_kernel_takes(c)) return launch_gemm_rows_epilogue(c, s);
  return launch_gemm_form<kEpilogue>(c, s);
}

unsigned gemm_epilogue_timeouts() { return form_timeouts(); }
int gemm_epilogue_reset_timeouts() { return form_reset_timeouts(); }

}  // namespace cogni
