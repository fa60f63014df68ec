// The gated form of the product for few rows (gemm_rows.cuh).
#include "gemm_rows.cuh"

namespace cogni {

int launch_gemm_rows_glu(const RowsCall &c, cudaStream_t s) { return launch_rows<true>(c, s); }
unsigned gemm_rows_glu_timeouts() { return rows_timeouts(); }
int gemm_rows_glu_reset_timeouts() { return rows_reset_timeouts(); }

}  // namespace cogni
