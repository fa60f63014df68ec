// The plain form of the prefill product (gemm_prefill.cuh): cogni_qmm_gemm_bf16.
#include "gemm_prefill.cuh"

namespace cogni {

int g_prefill_force_bn = 0;
int g_prefill_stage_raw = 1;
int g_prefill_force_split = 0;
int g_prefill_pair = 1;
int g_prefill_two = 0;

int launch_gemm_prefill(int type, const void *d_w, const void *d_x_bf16, void *d_y, int out_type,
                        int m_rows, int n_out, int k_in, cudaStream_t s) {
  RowsCall c = {};
  c.type = type;
  c.w = d_w;
  c.x = d_x_bf16;
  c.x_stride = k_in;
  c.m_rows = m_rows; c.n_out = n_out; c.k_in = k_in;
  c.epi.y = d_y;
  c.epi.y_stride = n_out;
  c.epi.y_bf16 = out_type == COGNI_QMM_OUT_BF16;
  return launch_gemm_form<kPlain>(c, s);
}

void gemm_prefill_set_tile(int bn) { g_prefill_force_bn = bn; }
void gemm_prefill_set_split(int mode) { g_prefill_force_split = mode; }
void gemm_prefill_set_stage_raw(int on) { g_prefill_stage_raw = on; }
void gemm_prefill_set_pair(int on) { g_prefill_pair = on; }
void gemm_prefill_set_two(int on) { g_prefill_two = on; }

unsigned gemm_prefill_timeouts() { return form_timeouts(); }
int gemm_prefill_reset_timeouts() { return form_reset_timeouts(); }

}  // namespace cogni
