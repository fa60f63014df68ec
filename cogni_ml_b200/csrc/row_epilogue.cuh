// What happens to a sum of a product with an epilogue on its way to memory: bias, activation, residual
// or gating, one rounding to the output type.  Shared by the tensor-core prefill kernels
// (gemm_prefill.cuh) and the kernel for few rows (gemm_rows.cuh).
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/cogni_qmm.h"

namespace cogni {

// y[m, n] = residual[m, n] + act(sum + bias[n]), or act(sum_gate + bias[n]) * (sum_up + bias_up[n])
struct RowEpilogue {
  const float *bias, *bias_up;  // null: none
  const void *residual;         // null: none; may be y itself (same strides)
  void *y;
  long long residual_stride, y_stride;  // elements between rows
  int residual_bf16, y_bf16;
  int activation;
  int vec;  // rows are multiples of four outputs, and four from a multiple of four on are aligned for one access each
};

template <int V> struct IntConst { static constexpr int value = V; };

// Calls f with the activation as a constant, so that the choice costs one branch a tile and not one
// an element.
template <class F> __device__ __forceinline__ void with_activation(int act, F &&f) {
  switch (act) {
    case COGNI_QMM_ACT_RELU: f(IntConst<COGNI_QMM_ACT_RELU>{}); break;
    case COGNI_QMM_ACT_SILU: f(IntConst<COGNI_QMM_ACT_SILU>{}); break;
    case COGNI_QMM_ACT_GELU: f(IntConst<COGNI_QMM_ACT_GELU>{}); break;
    case COGNI_QMM_ACT_GELU_TANH: f(IntConst<COGNI_QMM_ACT_GELU_TANH>{}); break;
    case COGNI_QMM_ACT_SIGMOID: f(IntConst<COGNI_QMM_ACT_SIGMOID>{}); break;
    default: f(IntConst<COGNI_QMM_ACT_NONE>{}); break;
  }
}

// In f32.  The quotients are 0 where exp(-v) is above 2^126 (v < -87.3, __fdividef), which is within 2^-126 |v| of the value.
// __expf is off by 2 + 1.17 |v| units of 2^-23, so sigmoid and silu by 1e-5 of their value at v = -80 where that is 1e-35.  The tanh form is v * sigmoid(2 u), the same function without the cancellation of
// 1 + tanh(u) at negative u.
template <int ACT> __device__ __forceinline__ float activate(float v) {
  if (ACT == COGNI_QMM_ACT_RELU) return v < 0.f ? 0.f : v;  // NaN stays NaN
  if (ACT == COGNI_QMM_ACT_SILU) return __fdividef(v, 1.f + __expf(-v));
  if (ACT == COGNI_QMM_ACT_SIGMOID) return __fdividef(1.f, 1.f + __expf(-v));
  if (ACT == COGNI_QMM_ACT_GELU) return 0.5f * v * (1.f + erff(v * 0.70710678f));
  if (ACT == COGNI_QMM_ACT_GELU_TANH)
    return __fdividef(v, 1.f + __expf(-1.5957691f * (v + 0.044715f * v * v * v)));
  return v;
}

__device__ __forceinline__ float bf16_value(uint32_t bits16) { return __uint_as_float(bits16 << 16); }
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}

__device__ __forceinline__ void store_out(const RowEpilogue &e, int m, int n, float v) {
  const long long at = (long long)m * e.y_stride + n;
  if (e.y_bf16) reinterpret_cast<__nv_bfloat16 *>(e.y)[at] = __float2bfloat16_rn(v);
  else reinterpret_cast<float *>(e.y)[at] = v;
}
__device__ __forceinline__ void store_out4(const RowEpilogue &e, int m, int n, const float (&f)[4]) {
  const long long at = (long long)m * e.y_stride + n;
  if (e.y_bf16)
    *reinterpret_cast<uint2 *>(reinterpret_cast<__nv_bfloat16 *>(e.y) + at) =
        make_uint2(bf16_pair(f[0], f[1]), bf16_pair(f[2], f[3]));
  else
    *reinterpret_cast<float4 *>(reinterpret_cast<float *>(e.y) + at) = make_float4(f[0], f[1], f[2], f[3]);
}
// The residual of four outputs n .. n + 3 of row m in one access (RowEpilogue::vec), as read and as values; zero where there
// is none.
__device__ __forceinline__ uint4 residual4_bits(const RowEpilogue &e, int m, int n) {
  if (!e.residual) return make_uint4(0, 0, 0, 0);
  const long long at = (long long)m * e.residual_stride + n;
  if (e.residual_bf16) {
    const uint2 b = *reinterpret_cast<const uint2 *>(reinterpret_cast<const __nv_bfloat16 *>(e.residual) + at);
    return make_uint4(b.x, b.y, 0, 0);
  }
  return *reinterpret_cast<const uint4 *>(reinterpret_cast<const float *>(e.residual) + at);
}
__device__ __forceinline__ void residual4_values(const RowEpilogue &e, const uint4 &b, float (&r)[4]) {
  r[0] = e.residual_bf16 ? bf16_value(b.x) : __uint_as_float(b.x);
  r[1] = __uint_as_float(e.residual_bf16 ? b.x & 0xffff0000u : b.y);
  r[2] = e.residual_bf16 ? bf16_value(b.y) : __uint_as_float(b.z);
  r[3] = __uint_as_float(e.residual_bf16 ? b.y & 0xffff0000u : b.w);
}
// Residual and bias of four outputs n .. n + 3 (n a multiple of four below n_out) of row m.  Which accesses are taken is the same
// for all lanes: outputs behind the row's end read its last element, and are not stored.  (Plain loads, not through the
// read-only path: the residual may be the y that other threads write.)
__device__ __forceinline__ void load_residual4(const RowEpilogue &e, int m, int n, int n_out, float (&r)[4]) {
  if (e.vec || !e.residual) {
    residual4_values(e, residual4_bits(e, m, n), r);
    return;
  }
  const long long row = (long long)m * e.residual_stride;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const long long at = row + min(n + i, n_out - 1);
    r[i] = e.residual_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(e.residual)[at])
                           : reinterpret_cast<const float *>(e.residual)[at];
  }
}
__device__ __forceinline__ void load_bias4(const float *bias, int n, int n_out, float (&b)[4]) {
#pragma unroll
  for (int i = 0; i < 4; i++) b[i] = bias ? __ldg(bias + min(n + i, n_out - 1)) : 0.f;
}
__device__ __forceinline__ void store_outputs4(const RowEpilogue &e, int m, int n, int n_out, const float (&f)[4]) {
  if (e.vec) {
    store_out4(e, m, n, f);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (n + i < n_out) store_out(e, m, n + i, f[i]);
}
// Four outputs n .. n + 3 (n a multiple of four) of row m, those below n_out.
template <int ACT> __device__ __forceinline__ void epilogue_store4_as(const RowEpilogue &e, const float (&sum)[4], int m, int n, int n_out) {
  if (n >= n_out) return;
  float r[4], b[4], f[4];
  load_residual4(e, m, n, n_out, r);
  load_bias4(e.bias, n, n_out, b);
#pragma unroll
  for (int i = 0; i < 4; i++) f[i] = r[i] + activate<ACT>(sum[i] + b[i]);
  store_outputs4(e, m, n, n_out, f);
}
__device__ __forceinline__ void epilogue_store4(const RowEpilogue &e, const float (&sum)[4], int m, int n, int n_out) {
  with_activation(e.activation, [&](auto act) { epilogue_store4_as<decltype(act)::value>(e, sum, m, n, n_out); });
}
__device__ __forceinline__ void glu_store4(const RowEpilogue &e, const float (&gate)[4], const float (&up)[4], int m,
                                           int n, int n_out) {
  if (n >= n_out) return;
  float bg[4], bu[4], f[4];
  load_bias4(e.bias, n, n_out, bg);
  load_bias4(e.bias_up, n, n_out, bu);
  with_activation(e.activation, [&](auto act) {
#pragma unroll
    for (int i = 0; i < 4; i++) f[i] = activate<decltype(act)::value>(gate[i] + bg[i]) * (up[i] + bu[i]);
  });
  store_outputs4(e, m, n, n_out, f);
}

// Whether four consecutive elements of every row of n can be one access (rows `stride` elements apart), the last ones too: a
// row that ends inside four outputs goes element by element in all lanes.
inline bool rows_vec4(const void *p, long long stride, bool bf16, int n) {
  return (reinterpret_cast<uintptr_t>(p) & (bf16 ? 7 : 15)) == 0 && stride % 4 == 0 && n % 4 == 0;
}

// One call of a product with an epilogue, as the launchers take it.
struct RowsCall {
  int type;
  const void *w, *w_up;  // w_up: gated form
  const void *x;         // bf16, rows x_stride elements apart
  long long x_stride;
  int m_rows, n_out, k_in;
  int resident;
  int ks_begin, ks_end;  // tiles: the k-steps of 64 of one launch
  RowEpilogue epi;
};

// A tensor core truncates its f32 accumulator at every K = 16 step, which pulls a sum towards zero: by half a unit in the
// last place of the partial sum on average.  Measured over K = 2048 .. 32768, weights of four types and activations of
// mean 0 and 1/2, y comes out (1 - a K / 16) y, a = 1.30e-8 .. 1.58e-8: 1.34e-5 of the norm against f64 at K = 12288,
// where f32 sums in order have 1.4e-6.  So where y is f32, K is cut until no part is longer than this, into CTAs of a cluster (at
// most eight) or launches that follow one another, and the parts are added in f32, rounded to nearest: 6.7e-6.  Nothing else
// is done to a sum, so one that is exact at every step comes out exact.  In bf16 (2^-9) the truncation does not show.
constexpr int kMaxF32Part = 6144;

// Few rows go to the kernel that expands weights in registers (gemm_rows.cuh), more to the tensor-core tiles
// (gemm_prefill.cuh), whose expansion into shared memory does not get dearer with the tokens but is slow for Q6_K and Q8_0.
// Time of the first over that of the best tile, geometric means over drawn shapes:
//   6183 shapes, at 25-32 / 41-48 / 57-64 rows: Q4_K 0.96 / 1.12 / 1.3, Q5_K 0.97 / 1.05 / 1.5, IQ4_NL 0.88 / 1.13 / 1.3, Q8_0
//   0.57 / 0.74 / 0.87, Q6_K 0.49 / 0.68 / 0.80;
//   gated Q4_K and Q5_K, 60 shapes, at 9-16 / 18-24 / 26-32 rows: 0.77 / 0.98 / 1.15, below 2^21 weights a matrix 0.9 throughout.
inline bool rows_kernel_takes(const RowsCall &c) {
  if (c.type == COGNI_QMM_TYPE_Q6_K || c.type == COGNI_QMM_TYPE_Q8_0) return c.m_rows <= 64;
  const bool gated_k = c.w_up && (c.type == COGNI_QMM_TYPE_Q4_K || c.type == COGNI_QMM_TYPE_Q5_K);
  return c.m_rows <= (gated_k && (long long)c.n_out * c.k_in >= 1 << 21 ? 24 : 32);
}

}  // namespace cogni
