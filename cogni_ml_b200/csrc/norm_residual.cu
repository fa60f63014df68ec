// The norms around a block, with its gate and the residual addition (cogni_qmm_norm_residual):
//
//     h = residual + scale * gate * norm_post(block)        y = norm_pre(h)
//     rms:   norm(v) = v * rsqrt(mean(v^2) + eps) * w + b
//     layer: norm(v) = (v - mean(v)) * rsqrt(mean((v - mean(v))^2) + eps) * w + b
//
// One pass: a row is read once into registers, both norms are taken there, h and y are written once; the
// bytes are all that bounds it.  A row belongs to one CTA of 32 .. 1024 threads, each with one to four
// chunks of eight elements.  All loads of a row are issued before the first reduction; the CTAs of
// the other rows on the SM cover the reductions.  Sums are f32 trees over at most 32 values a thread
// (the layer norm's variance from the centred values), y and h are rounded once, and y is formed from
// the f32 h, before its rounding.
#include <cuda_bf16.h>

#include "qmm_common.cuh"
#include "row_epilogue.cuh"
#include "tma_pipe.cuh"

namespace cogni {
namespace {

struct NormSide {
  const float *w, *b;  // w null: no norm
  float eps;
  int layer;
};
struct NormParams {
  const void *residual, *block, *gate;  // block, gate: null = none
  void *h, *y;                          // null: not written
  long long residual_stride, block_stride, gate_stride, h_stride, y_stride;
  int residual_bf16, block_bf16, gate_bf16, h_bf16, y_bf16;
  float scale;
  NormSide post, pre;
  int n;
};

__device__ __forceinline__ void store8(void *p, bool bf16, long long at, const float (&v)[8]) {
  if (bf16) {
    *reinterpret_cast<uint4 *>(static_cast<__nv_bfloat16 *>(p) + at) =
        make_uint4(bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7]));
  } else {
    *reinterpret_cast<float4 *>(static_cast<float *>(p) + at) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4 *>(static_cast<float *>(p) + at + 4) = make_float4(v[4], v[5], v[6], v[7]);
  }
}
__device__ __forceinline__ void store1(void *p, bool bf16, long long at, float v) {
  if (bf16) static_cast<__nv_bfloat16 *>(p)[at] = __float2bfloat16_rn(v);
  else static_cast<float *>(p)[at] = v;
}

// Where a thread's chunk c lies in the row.  VEC: eight consecutive elements; else element i of it is
// blockDim.x * (8 c + i) + threadIdx.x, so that a warp's accesses stay contiguous at any alignment.
template <bool VEC> __device__ __forceinline__ int place(int c, int i) {
  return VEC ? 8 * ((int)blockDim.x * c + (int)threadIdx.x) + i : (int)blockDim.x * (8 * c + i) + (int)threadIdx.x;
}
// whether element i of chunk c lies in the row (VEC: n is a multiple of eight, a chunk does or does not)
template <bool VEC> __device__ __forceinline__ bool inside(int c, int i, int n) { return place<VEC>(c, VEC ? 0 : i) < n; }

// A chunk as it lies in memory.  Loading and converting are apart: a conversion in the branch of its type would wait for
// its load before the next array's is issued (333 rows x 2051, layer norms around a gate: 12.9 us so, 8.2 apart).
struct RawChunk { uint32_t w[8]; };
template <bool VEC> __device__ __forceinline__ void load_raw(const void *p, bool bf16, long long row, int c, int n, RawChunk &r) {
  if (VEC) {
    if (!inside<true>(c, 0, n)) return;
    const uint4 *a = reinterpret_cast<const uint4 *>(static_cast<const char *>(p) + (row + place<true>(c, 0)) * (bf16 ? 2 : 4));
    const uint4 lo = a[0];
    r.w[0] = lo.x; r.w[1] = lo.y; r.w[2] = lo.z; r.w[3] = lo.w;
    if (!bf16) {
      const uint4 hi = a[1];
      r.w[4] = hi.x; r.w[5] = hi.y; r.w[6] = hi.z; r.w[7] = hi.w;
    }
  } else if (bf16) {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (inside<false>(c, i, n)) r.w[i] = static_cast<const unsigned short *>(p)[row + place<false>(c, i)];
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (inside<false>(c, i, n)) r.w[i] = static_cast<const uint32_t *>(p)[row + place<false>(c, i)];
  }
}
template <bool VEC> __device__ __forceinline__ void convert(const RawChunk &r, bool bf16, float (&v)[8]) {
  if (!bf16) {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = __uint_as_float(r.w[i]);
  } else if (VEC) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      v[2 * i] = bf16_value(r.w[i]);
      v[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = bf16_value(r.w[i]);
  }
}
template <bool VEC> __device__ __forceinline__ void load_vector(const float *p, int c, int n, float (&v)[8]) {  // f32, the same for all rows
  RawChunk r;
  load_raw<VEC>(p, false, 0, c, n, r);
  convert<VEC>(r, false, v);
}
template <bool VEC> __device__ __forceinline__ void store_chunk(void *p, bool bf16, long long row, int c, int n, const float (&v)[8]) {
  if (VEC) {
    if (inside<true>(c, 0, n)) store8(p, bf16, row + place<true>(c, 0), v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (inside<false>(c, i, n)) store1(p, bf16, row + place<false>(c, i), v[i]);
  }
}

// The sum over the CTA, in an order that does not depend on timing.  `slots`: two sets of 32 floats
// used in turn, so that one barrier a sum is enough.
__device__ __forceinline__ float row_sum(float v, float *slots, int &turn) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  float *s = slots + 32 * (turn & 1);
  turn++;
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = (threadIdx.x & 31) < warps ? s[threadIdx.x & 31] : 0.f;
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int C, bool VEC>
__device__ __forceinline__ void normalise(const NormSide &s, float (&v)[C][8], int n, float *slots, int &turn) {
  float sum = 0.f, inv_n = 1.f / (float)n;
  if (s.layer) {
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (inside<VEC>(c, i, n)) sum += v[c][i];
    const float mean = row_sum(sum, slots, turn) * inv_n;
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int i = 0; i < 8; i++) v[c][i] -= mean;
  }
  sum = 0.f;
#pragma unroll
  for (int c = 0; c < C; c++)
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (inside<VEC>(c, i, n)) sum += v[c][i] * v[c][i];
  const float r = rsqrtf(row_sum(sum, slots, turn) * inv_n + s.eps);
#pragma unroll
  for (int c = 0; c < C; c++) {
    float w[8];
    load_vector<VEC>(s.w, c, n, w);
#pragma unroll
    for (int i = 0; i < 8; i++) v[c][i] = v[c][i] * r * w[i];
    if (s.b) {
      load_vector<VEC>(s.b, c, n, w);
#pragma unroll
      for (int i = 0; i < 8; i++) v[c][i] += w[i];
    }
  }
}

// Full occupancy (32 registers) for the vector form of one chunk: 4096 rows x 5120 with both norms 63 us at 40 registers,
// 58 at 32.  (Tried and slower: the rows past the L1, 62; the next row loaded beside this one's reductions, 76.)
template <int C, bool VEC>
__global__ void __launch_bounds__(1024, C == 1 && VEC ? 2 : 1) norm_residual_kernel(const NormParams p) {
  __shared__ float slots[64];
  int turn = 0;
  const long long m = blockIdx.x;
  pdl_wait_prior_grid();
  pdl_launch_dependents();
  float h[C][8], b[C][8];
  {
    RawChunk hr[C], br[C];
#pragma unroll
    for (int c = 0; c < C; c++) {
      if (p.block) load_raw<VEC>(p.block, p.block_bf16, m * p.block_stride, c, p.n, br[c]);
      load_raw<VEC>(p.residual, p.residual_bf16, m * p.residual_stride, c, p.n, hr[c]);
    }
#pragma unroll
    for (int c = 0; c < C; c++) {
      if (p.block) convert<VEC>(br[c], p.block_bf16, b[c]);
      convert<VEC>(hr[c], p.residual_bf16, h[c]);
    }
  }
  if (p.block) {
    if (p.post.w) normalise<C, VEC>(p.post, b, p.n, slots, turn);
#pragma unroll
    for (int c = 0; c < C; c++) {
      if (p.gate) {
        RawChunk r;
        float g[8];
        load_raw<VEC>(p.gate, p.gate_bf16, m * p.gate_stride, c, p.n, r);
        convert<VEC>(r, p.gate_bf16, g);
#pragma unroll
        for (int i = 0; i < 8; i++) b[c][i] *= g[i];
      }
#pragma unroll
      for (int i = 0; i < 8; i++) h[c][i] += p.scale * b[c][i];
    }
  }
  if (p.h) {
#pragma unroll
    for (int c = 0; c < C; c++) store_chunk<VEC>(p.h, p.h_bf16, m * p.h_stride, c, p.n, h[c]);
  }
  if (p.pre.w) {
    normalise<C, VEC>(p.pre, h, p.n, slots, turn);
#pragma unroll
    for (int c = 0; c < C; c++) store_chunk<VEC>(p.y, p.y_bf16, m * p.y_stride, c, p.n, h[c]);
  }
}

template <int C>
int launch_width(const NormParams &p, int m_rows, int threads, bool vec, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(m_rows);
  cfg.blockDim = dim3(threads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return (int)(vec ? cudaLaunchKernelEx(&cfg, norm_residual_kernel<C, true>, p)
                   : cudaLaunchKernelEx(&cfg, norm_residual_kernel<C, false>, p));
}

bool rows_vec8(const void *p, long long stride) {  // 16-byte accesses of eight elements (f32: two)
  return !p || ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride % 8 == 0);
}

}  // namespace

int launch_norm_residual(const cogni_qmm_norm_args &a, cudaStream_t s) {
  NormParams p = {};
  p.residual = a.residual; p.block = a.block; p.gate = a.block ? a.gate : nullptr;
  p.h = a.h; p.y = a.y;
  p.residual_stride = a.residual_stride; p.block_stride = a.block_stride; p.gate_stride = a.gate_stride;
  p.h_stride = a.h_stride; p.y_stride = a.y_stride;
  p.residual_bf16 = a.residual_type == COGNI_QMM_OUT_BF16; p.block_bf16 = a.block_type == COGNI_QMM_OUT_BF16;
  p.gate_bf16 = a.gate_type == COGNI_QMM_OUT_BF16; p.h_bf16 = a.h_type == COGNI_QMM_OUT_BF16;
  p.y_bf16 = a.y_type == COGNI_QMM_OUT_BF16;
  p.scale = a.scale;
  p.post = {a.block ? a.post.weight : nullptr, a.post.bias, a.post.eps, a.post.kind == COGNI_QMM_NORM_LAYER};
  p.pre = {a.pre.weight, a.pre.bias, a.pre.eps, a.pre.kind == COGNI_QMM_NORM_LAYER};
  p.n = a.n;
  const bool vec = a.n % 8 == 0 && rows_vec8(p.residual, p.residual_stride) && rows_vec8(p.block, p.block_stride) &&
                   rows_vec8(p.gate, p.gate_stride) && rows_vec8(p.h, p.h_stride) && rows_vec8(p.y, p.y_stride) &&
                   rows_vec8(p.post.w, 0) && rows_vec8(p.post.b, 0) && rows_vec8(p.pre.w, 0) && rows_vec8(p.pre.b, 0);
  // eight elements a thread up to 8192, beyond that up to 32
  const int chunks = (a.n + 7) / 8;
  const int per = chunks <= 1024 ? 1 : chunks <= 2048 ? 2 : 4;
  const int threads = ((chunks + per - 1) / per + 31) / 32 * 32;
  if (per == 1) return launch_width<1>(p, a.m_rows, threads, vec, s);
  if (per == 2) return launch_width<2>(p, a.m_rows, threads, vec, s);
  return launch_width<4>(p, a.m_rows, threads, vec, s);
}

}  // namespace cogni
