// The gated form of the product for few rows (glu_sums.cuh, gemm_rows.cuh).
#include "glu_sums.cuh"

namespace cogni {
namespace {

template <int TYPE> int launch_typed(const RowsCall &c, cudaStream_t s) {
  if (c.m_rows <= 8) return launch_glu_sums<TYPE, 1>(c, s);
  // Measured against the kernel that rounds its weights, us: Q4_K 12288 x 4096, 16 / 24 / 32 rows 29.6 / 35.7 / 46.5 and
  // 38.0 / 44.2 / 51.0; 17408 x 5120 39.7 / 52.2 / 68.2 and 53.6 / 64.0 / 84.6; but few CTAs of 256 weight rows are slower
  // than more of 128: 4096 x 2048 10.1 / 11.8 / 14.6 and 9.3 / 10.4 / 11.9.
  if ((long long)c.n_out * c.k_in >= 1 << 24) {
    if (c.m_rows <= 16) return launch_glu_sums<TYPE, 2>(c, s);
    if constexpr (TYPE == kQ4_K) {  // Q5_K: two CTAs an SM have no room for more than 16 tokens
      if (c.m_rows <= 24) return launch_glu_sums<TYPE, 3>(c, s);
      if (c.m_rows <= 32) return launch_glu_sums<TYPE, 4>(c, s);
    }
  }
  return launch_rows<true>(c, s);
}

}  // namespace

int launch_gemm_rows_glu(const RowsCall &c, cudaStream_t s) {
  if (c.type == kQ4_K) return launch_typed<kQ4_K>(c, s);
  if (c.type == kQ5_K) return launch_typed<kQ5_K>(c, s);
  return launch_rows<true>(c, s);
}
unsigned gemm_rows_glu_timeouts() { return rows_timeouts(); }
int gemm_rows_glu_reset_timeouts() { return rows_reset_timeouts(); }

}  // namespace cogni
