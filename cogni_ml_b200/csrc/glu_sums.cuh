// The gated form of Q4_K / Q5_K for few tokens: the sums of quant_sums.cuh, with the activations shared by the CTA.
//
// Every warp reads all of the activations from shared memory for every tile of 16 rows, which is more than the weights from
// nine tokens on.  So a warp has two tiles and reads them once for both, and the eight warps of the CTA (256 weight
// rows, half gate, half up; two CTAs an SM) go through the superblocks together, one superblock column of the rows and
// the tokens' 256 activations a stage, two stages.  K is cut for a cluster as in gemm_rows.cuh.  Warp w takes the
// activations' sums of group w before a superblock's products.
//   MMA rows g = 0 .. 7 are the rows 2 (g & 3) + (g >> 2) of their eight: rows are 144 (176) bytes apart, and an 8-byte load
// serves 16 lanes, four rows, at a time; every other row lies 32 (96) bytes on modulo 128.
// Bound (counters, Q4_K 12288 x 4096, one row): neither the copies (12 us alone, at 6.7 TB/s) nor the 400 instructions a tile
// and superblock (13 us alone) but that a CTA does the one while it waits for the other: 22 us.  Tried: three stages,
// 21.3; four warps a CTA, 23.5; 128 rows and a warp-private ring for every warp without clusters or barriers, 20.3, but slower
// where tokens x K leave that ring little room (8 rows of 17408 x 5120: 43.9 against 30.9).
#pragma once

#include "quant_sums.cuh"

namespace cogni {
namespace {

constexpr int kSumsWarps = 8, kSumsThreads = 32 * kSumsWarps;
constexpr int kSumsRows = 32 * kSumsWarps;   // A rows of a CTA
constexpr int kSumsOuts = kSumsRows / 2;
constexpr int kSumsStages = 2;
template <int TYPE, int NT> __host__ __device__ constexpr int sums_smem() {
  return kSumsStages * (kSumsRows * RowCfg<TYPE>::RS + 8 * NT * kTokenStride) + 8 * 8 * NT * 4 /*sums*/ + 64 /*barriers*/;
}

template <int TYPE, int NT>
__global__ void __launch_bounds__(kSumsThreads, 2)
    glu_sums_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_up, const RowsParams p) {
  using Cfg = RowCfg<TYPE>;
  constexpr int kStageBytes = kSumsRows * Cfg::RS;
  constexpr int kTokens = 8 * NT, kXBytes = kTokens * kTokenStride;
  static_assert(kTokens * (kSumsRows + 4) * 4 <= kSumsStages * kStageBytes, "the partial tile fits the ring");
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t *x0 = smem + kSumsStages * kStageBytes, *xsum0 = x0 + kSumsStages * kXBytes;
  const uint32_t bars = smem_u32(xsum0 + 8 * kTokens * 4);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * kSumsOuts, m0 = blockIdx.y * kTokens;
  const int sb0 = blockIdx.z * p.per, nsb = min(p.per, p.nsb - sb0);
  const int parts = gridDim.z, rank = blockIdx.z;
  const int raw_n0 = min(n0, p.n_out - p.box_rows);  // as in gemm_rows_kernel
  const int gr = 2 * (g & 3) + (g >> 2);             // the row of its eight that MMA row g stands for

  auto issue_weights = [&](int i) {
    if (tid == 0) {
      const uint32_t dst = smem_u32(smem) + (i % kSumsStages) * kStageBytes, full = bars + 8 * (i % kSumsStages);
      mbar_arrive_expect_tx(full, 2 * p.box_rows * Cfg::RS);
      const int at = (Cfg::SB * (sb0 + i)) >> 2;  // 4-byte elements, 16-byte boundaries
      tma_load_2d(dst, &tmap_w, at, raw_n0, full);
      tma_load_2d(dst + kSumsOuts * Cfg::RS, &tmap_up, at, raw_n0, full);
    }
  };
  auto issue_x = [&](int i) {
    const uint32_t dst = smem_u32(x0) + (i % kSumsStages) * kXBytes;
#pragma unroll
    for (int j = 0; j < kTokens * 32 / kSumsThreads; j++) {
      const int at = kSumsThreads * j + tid, token = at >> 5, c = at & 31;
      const bool in = m0 + token < p.m_rows;
      const __nv_bfloat16 *a = p.x + (in ? (long long)(m0 + token) * p.x_stride : 0) + (sb0 + i) * 256 + 8 * c;
      cp_async16(dst + token * kTokenStride + 16 * c, a, in ? 16 : 0);
    }
  };
  const uint8_t *x_lane = x0 + g * kTokenStride + 16 * t;

  if (tid == 0) {
    for (int i = 0; i < kSumsStages; i++) mbar_init(bars + 8 * i, 1);
    mbar_fence_init();
  }
  __syncthreads();
  pdl_launch_dependents();
  if (!p.resident) pdl_wait_prior_grid();
#pragma unroll
  for (int i = 0; i < kSumsStages - 1; i++)
    if (i < nsb) issue_weights(i);
  if (p.resident) pdl_wait_prior_grid();
#pragma unroll
  for (int i = 0; i < kSumsStages - 1; i++) {
    if (i < nsb) issue_x(i);
    cp_async_commit();
  }

  float acc[2][NT][4] = {};
  uint32_t rows[2][2];  // the lane's rows: tile, gate or up
#pragma unroll
  for (int u = 0; u < 2; u++) {
    const int r = min(n0 + 16 * warp + 8 * u + gr - raw_n0, p.box_rows - 1);
    rows[u][0] = r * Cfg::RS;
    rows[u][1] = (kSumsOuts + r) * Cfg::RS;
  }
  bool ok = true;
#pragma unroll 1
  for (int i = 0; i < nsb; i++) {
    cp_async_wait<kSumsStages - 2>();
    ok &= mbar_wait(bars + 8 * (i % kSumsStages), (i / kSumsStages) & 1);
    __syncthreads();  // stage i has landed for every warp, stage i - 1 is free
    if (i + kSumsStages - 1 < nsb) {
      issue_weights(i + kSumsStages - 1);
      issue_x(i + kSumsStages - 1);
    }
    cp_async_commit();
    const uint8_t *stage = smem + (i % kSumsStages) * kStageBytes, *x = x_lane + (i % kSumsStages) * kXBytes;
#pragma unroll
    for (int j = 0; j < NT; j++) {
      const float2 s = sum_group(lds128(x + j * 8 * kTokenStride + 64 * warp));
      if (g == 0) *reinterpret_cast<float2 *>(xsum0 + (warp * kTokens + 8 * j + 2 * t) * 4) = s;
    }
    __syncthreads();
    const uint8_t *const at[2][2] = {{stage + rows[0][0], stage + rows[0][1]}, {stage + rows[1][0], stage + rows[1][1]}};
    sums_tiles<TYPE, NT, 2>(at, [&](int j, int s) { return lds128(x + j * 8 * kTokenStride + 64 * s); }, xsum0 + 8 * t, t, acc);
  }
  cp_async_wait<0>();
  if (!ok) drain_copies_in_flight();
  __syncthreads();
  float *part = reinterpret_cast<float *>(smem);
#pragma unroll
  for (int u = 0; u < 2; u++) leave_tile<NT, kSumsRows>(acc[u], part, 32 * warp + 16 * u + gr, t);
  finish_rows<kTokens, kSumsRows, true, kSumsThreads>(p, part, m0, n0, parts, rank);
}

template <int TYPE, int NT> int launch_glu_sums(const RowsCall &c, cudaStream_t s) {
  static RowsOnce once;
  RowsParams p;
  CUtensorMap maps[2] = {};
  constexpr int kSmem = sums_smem<TYPE, NT>();
  static_assert(2 * (kSmem + 1024) <= 228 * 1024, "two CTAs an SM");
  int sms = 0, st = rows_configure(once, reinterpret_cast<const void *>(glu_sums_kernel<TYPE, NT>), kSmem, sms);
  if (!st) st = rows_params<TYPE, true>(c, RowCfg<TYPE>::RS, kSumsOuts, p, maps);
  if (st) return st;
  return rows_launch(once, glu_sums_kernel<TYPE, NT>, p, maps, kSumsOuts, 8 * NT, kSumsThreads, kSmem, sms, s);
}

}  // namespace
}  // namespace cogni
