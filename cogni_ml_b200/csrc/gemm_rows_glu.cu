// The gated form of the product for few rows (rows_stream.cuh, gemm_rows.cuh).
#include <cstdlib>

#include "rows_stream.cuh"

namespace cogni {

int launch_gemm_rows_glu(const RowsCall &c, cudaStream_t s) {
  const int st = launch_rows_stream<true>(c, s);
  return st == kNotTaken ? launch_rows<true>(c, s) : st;
}
unsigned gemm_rows_glu_timeouts() { return rows_timeouts(); }
int gemm_rows_glu_reset_timeouts() { return rows_reset_timeouts(); }

}  // namespace cogni
