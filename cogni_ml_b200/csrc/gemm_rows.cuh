// Products with an epilogue for few rows (1 .. 64 tokens a tile, sm_100a): weights streamed once from HBM,
// expanded to bf16 in registers, multiplied with mma.sync.
//
//     y[m, n] = residual[m, n] + act(sum_k x[m, k] bf16(dequant(W[n, k])) + bias[n])       GLU = false
//     y[m, n] = act(sum_k x Wg + bias_g) * (sum_k x Wu + bias_u)                           GLU = true
//
// A tensor-core tile of 128 tokens (gemm_prefill.cuh) spends its time on expanding weights into shared
// memory, whatever the number of tokens.  Here the weights never go back to shared memory: a warp owns 16
// weight rows (the M of mma.sync.m16n8k16), a lane the 64 weights of two of them in every superblock that
// share scales (Lane<TYPE>), which come out of the expansion in the A operand's register layout.  Which k an
// operand slot stands for is free as long as both operands agree: slot (t, i) of step s is the i-th of
// four consecutive weights of lane t, and the B operand is read from the activations accordingly.
//   * A CTA is eight warps (128 weight rows) and a part of K; the parts of a row block form a cluster and
//     meet in distributed shared memory (cluster_sum.cuh), so no workspace, no atomics, the same bits every
//     time.  K is cut where waves x superblocks come out least (rows_launch).
//   * A superblock column of the CTA's rows (one TMA box a matrix) and the tokens' 256 activations (16-byte
//     cp.async) are one stage of a ring; all loads of a short part are in flight at once.  Q6_K rows that
//     are not multiples of 16 bytes (k_in not a multiple of 2048) cannot be described to TMA: their
//     blocks come by cp.async too (STAGED = false).
//   * GLU: rows 0-7 of a warp's tile are the gate's, rows 8-15 the up matrix's.  Both sums of an output are
//     then in the same lane's accumulators.
// Weights are complete before the launch if `resident`: their first stages are then fetched before the wait
// for the preceding kernel (programmatic dependent launch).
#pragma once

#include <atomic>

#include "cluster_sum.cuh"
#include "expand.cuh"
#include "qmm_common.cuh"
#include "row_epilogue.cuh"
#include "tensor_map.cuh"
#include "tma_pipe.cuh"

namespace cogni {
namespace {

constexpr int kRowWarps = 8;
constexpr int kRowThreads = 32 * kRowWarps;
constexpr int kRowTile = 16 * kRowWarps;       // A rows of a CTA
constexpr int kTokenStride = 512 + 64;         // bytes of a token's 256 activations in shared memory: consecutive
                                               // tokens half a bank cycle apart

// SB: bytes of 256 weights of a row; RS: bytes of a row in a stage, which is the TMA box's width.  Lanes read 16
// bytes of two rows x four places 32 bytes apart at a time (RS an odd multiple of 16: distinct banks), or 4
// bytes of eight rows (Q8_0, IQ4_NL: RS = 16 modulo 128).  A Q6_K block, which starts on a 2-byte
// boundary, lies somewhere in a window of 240 bytes.
template <int TYPE> struct RowCfg;
template <> struct RowCfg<kQ4_K> { static constexpr int SB = 144, RS = 144; };
template <> struct RowCfg<kQ5_K> { static constexpr int SB = 176, RS = 176; };
template <> struct RowCfg<kQ6_K> { static constexpr int SB = 210, RS = 240; };
template <> struct RowCfg<kQ8_0> { static constexpr int SB = 272, RS = 272; };
template <> struct RowCfg<kIQ4_NL> { static constexpr int SB = 144, RS = 144; };
constexpr int kQ6Chunks = 14;  // 16-byte chunks that cover a block from the 16-byte boundary below it

template <int TYPE, int NT> __host__ __device__ constexpr int row_stage_bytes() { return kRowTile * RowCfg<TYPE>::RS + 8 * NT * kTokenStride; }
// stages: as many as let two CTAs share an SM, at most four
template <int TYPE, int NT> __host__ __device__ constexpr int row_stages() {
  constexpr int fit = (113 * 1024) / row_stage_bytes<TYPE, NT>();
  return fit < 2 ? 2 : fit > 4 ? 4 : fit;
}
template <int TYPE, int NT> __host__ __device__ constexpr int row_smem() {
  return row_stages<TYPE, NT>() * row_stage_bytes<TYPE, NT>() + 64 /*barriers*/;
}

struct RowsParams {
  const uint8_t *w, *w_up;
  const __nv_bfloat16 *x;
  long long x_stride, row_bytes;
  int m_rows, n_out, nsb, per;  // superblocks of a row, of a part
  int resident;
  int box_rows;  // rows of a TMA box: the tile's of a matrix, or all of them if there are fewer
  RowEpilogue epi;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, uint32_t bytes) {  // the rest is zero
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// Reads of staged bytes: ordinary loads (of shared memory, as the compiler sees from where the pointers come), so that
// they are ordered against the barriers and otherwise free to move among the MMAs.
__device__ __forceinline__ uint4 lds128(const uint8_t *a) { return *reinterpret_cast<const uint4 *>(a); }
__device__ __forceinline__ uint2 lds64(const uint8_t *a) { return *reinterpret_cast<const uint2 *>(a); }
__device__ __forceinline__ uint32_t lds32(const uint8_t *a) { return *reinterpret_cast<const uint32_t *>(a); }
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Four bytes to two bf16 pairs, in f32 as the dequantiser has it, then one rounding.  Without a minimum: d (byte - BIAS)
// as one fma on pairs.  The byte becomes a float by a permute that puts it into the mantissa of a power of
// two: 128 + byte (Q6_K, byte < 64, BIAS 32) or 2^15 + byte (bytes up to 255, BIAS 128); d has 18 (11) bits, so
// that power plus BIAS times d (160 = 5 * 2^5, 32896 = 257 * 2^7) is exact in f32 and so is the result.
template <int BIAS> __device__ __forceinline__ uint64_t scale_offset(float d) {
  const float c = BIAS == 32 ? -160.f * d : -32896.f * d;
  return f2_pack(c, c);
}
template <int BIAS> __device__ __forceinline__ uint64_t bytes2_float(uint32_t q, int i) {
  constexpr uint32_t base = BIAS == 32 ? 0x43000000u : 0x47000000u, sel = BIAS == 32 ? 0x7044u : 0x7604u;
  constexpr int shift = BIAS == 32 ? 8 : 4;
  return f2_pack(__uint_as_float(__byte_perm(q, base, sel + (i << shift))), __uint_as_float(__byte_perm(q, base, sel + ((i + 1) << shift))));
}
template <int BIAS> __device__ __forceinline__ void scale_word(uint32_t q, uint64_t d2, uint64_t c2, uint32_t &r0, uint32_t &r1) {
  r0 = f2_to_bf16x2(f2_fma(d2, bytes2_float<BIAS>(q, 0), c2));
  r1 = f2_to_bf16x2(f2_fma(d2, bytes2_float<BIAS>(q, 2), c2));
}
// With one: d * byte - m (2^23 + byte, whose bias comes off exactly).
__device__ __forceinline__ void scale_min_word(uint32_t q, uint64_t d2, uint64_t nm2, uint32_t &r0, uint32_t &r1) {
  const uint64_t off = f2_pack(-8388608.f, -8388608.f);
  r0 = f2_to_bf16x2(f2_fma(d2, f2_add(bytes2_biased(q, 0), off), nm2));
  r1 = f2_to_bf16x2(f2_fma(d2, f2_add(bytes2_biased(q, 2), off), nm2));
}
__device__ __forceinline__ float half_bits(uint32_t v) { return __half2float(__ushort_as_half((unsigned short)v)); }
__device__ __forceinline__ float small_byte(uint32_t v, int i) {
  return __uint_as_float(__byte_perm(v, 0x4B000000u, 0x7650 + i)) - 8388608.f;
}

// What lane t of a quad holds of one row in one superblock: 64 weights as eight runs ("chunks") of eight
// consecutive ones.  chunks(w): the two chunks w and 4 + w as four bf16 pairs each.  x_place(c): where the
// activations of the superblock's c-th eight elements (c = 0 .. 31) lie in a token's staged 512 bytes, in units of
// 16 bytes: chunk j of lane t at 4 j + t, so that a quad reads 64 contiguous bytes.
template <int TYPE> struct Lane;

// Q4_K / Q5_K: lane t has the 64-element group t, its low nibbles (sub-block 2t: chunks 0-3) and its high ones
// (sub-block 2t + 1: chunks 4-7).
template <int TYPE> struct LaneK45 {
  uint32_t q[8], h[TYPE == kQ5_K ? 8 : 1];
  uint64_t d[2], nm[2];  // of the two sub-blocks
  __device__ __forceinline__ void fetch(const uint8_t *row, int, int t) {
    const uint4 hdr = lds128(row);
    constexpr int at = TYPE == kQ5_K ? 48 : 16;
    const uint4 a = lds128(row + at + 32 * t), b = lds128(row + at + 16 + 32 * t);
    q[0] = a.x; q[1] = a.y; q[2] = a.z; q[3] = a.w; q[4] = b.x; q[5] = b.y; q[6] = b.z; q[7] = b.w;
    if constexpr (TYPE == kQ5_K) {
      const uint4 c = lds128(row + 16), e = lds128(row + 32);
      const uint32_t v[8] = {c.x, c.y, c.z, c.w, e.x, e.y, e.z, e.w};
#pragma unroll
      for (int i = 0; i < 8; i++) h[i] = v[i] >> (2 * t);  // the two sub-blocks' fifth bits are now bits 0 and 1
    }
    // the 6-bit scales and minimums of sub-blocks 2t, 2t + 1 in the low two bytes (dequant.cr:240-249)
    const int sh = 16 * (t & 1);
    const uint32_t u0 = hdr.y >> sh, u1 = hdr.z >> sh, u2 = hdr.w >> sh;
    const uint32_t sc = t < 2 ? u0 & 0x3f3fu : (u2 & 0x0f0fu) | ((u0 >> 2) & 0x3030u);
    const uint32_t mn = t < 2 ? u1 & 0x3f3fu : ((u2 >> 4) & 0x0f0fu) | ((u1 >> 2) & 0x3030u);
    const float df = half_bits(hdr.x & 0xffffu), dm = half_bits(hdr.x >> 16);
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const float s = __fmul_rn(df, small_byte(sc, i)), m = -__fmul_rn(dm, small_byte(mn, i));
      d[i] = f2_pack(s, s);
      nm[i] = f2_pack(m, m);
    }
  }
  __device__ __forceinline__ void chunks(int w, uint32_t (&lo)[4], uint32_t (&hi)[4]) const {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      uint32_t a = q[2 * w + i] & 0x0f0f0f0fu, b = (q[2 * w + i] >> 4) & 0x0f0f0f0fu;
      if constexpr (TYPE == kQ5_K) {
        a |= (h[2 * w + i] << 4) & 0x10101010u;
        b |= (h[2 * w + i] << 3) & 0x10101010u;
      }
      scale_min_word(a, d[0], nm[0], lo[2 * i], lo[2 * i + 1]);
      scale_min_word(b, d[1], nm[1], hi[2 * i], hi[2 * i + 1]);
    }
  }
  __device__ static __forceinline__ int x_place(int c) { return 4 * (c & 7) + (c >> 3); }
};
template <> struct Lane<kQ4_K> : LaneK45<kQ4_K> {};
template <> struct Lane<kQ5_K> : LaneK45<kQ5_K> {};

// Q6_K: lane t has half n = t >> 1 of the superblock, ql bytes 32 b .. 32 b + 31 of it (b = t & 1): the low nibbles
// are the half's run b (chunks 0-3), the high ones run 2 + b (chunks 4-7); a run has two scales.
template <> struct Lane<kQ6_K> {
  uint32_t ql[8], qh[8];
  uint64_t d[4], c[4];  // low run: elements 0-15, 16-31; high run
  // eight words from byte `at` (2-byte aligned) of a staged row on
  __device__ static __forceinline__ void words(const uint8_t *row, int at, uint32_t (&out)[8]) {
    const uint8_t *a = row + (at & ~15);
    const uint4 c0 = lds128(a), c1 = lds128(a + 16), c2 = lds128(a + 32);
    const uint32_t w[12] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w, c2.x, c2.y, c2.z, c2.w};
    const uint32_t sh = (uint32_t)(at & 2) * 8;
    switch ((at & 15) >> 2) {  // the same for all rows when rows are multiples of 16 bytes
      case 0:
#pragma unroll
        for (int i = 0; i < 8; i++) out[i] = __funnelshift_r(w[i], w[i + 1], sh);
        break;
      case 1:
#pragma unroll
        for (int i = 0; i < 8; i++) out[i] = __funnelshift_r(w[i + 1], w[i + 2], sh);
        break;
      case 2:
#pragma unroll
        for (int i = 0; i < 8; i++) out[i] = __funnelshift_r(w[i + 2], w[i + 3], sh);
        break;
      default:
#pragma unroll
        for (int i = 0; i < 8; i++) out[i] = __funnelshift_r(w[i + 3], i < 7 ? w[i + 4] : w[11], sh);
        break;
    }
  }
  __device__ __forceinline__ void fetch(const uint8_t *row, int off, int t) {
    const int n = t >> 1, b = t & 1;
    words(row, off + 32 * t, ql);
    words(row, off + 128 + 32 * n, qh);
#pragma unroll
    for (int i = 0; i < 8; i++) qh[i] >>= 2 * b;  // run b in bits 0-1, run 2 + b in bits 4-5
    // scales 8n + 2b, + 1 (low run) and + 4, + 5 (high run), each pair at an even address; then d
    auto pair16 = [&](int at) { return lds32(row + (at & ~3)) >> ((at & 2) * 8); };
    const uint32_t lo = pair16(off + 192 + 8 * n + 2 * b), hi = pair16(off + 196 + 8 * n + 2 * b);
    const float df = half_bits(pair16(off + 208) & 0xffffu);
    const int s[4] = {(int8_t)(lo & 0xff), (int8_t)((lo >> 8) & 0xff), (int8_t)(hi & 0xff), (int8_t)((hi >> 8) & 0xff)};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float v = __fmul_rn(df, (float)s[i]);
      d[i] = f2_pack(v, v);
      c[i] = scale_offset<32>(v);
    }
  }
  __device__ __forceinline__ void chunks(int w, uint32_t (&lo)[4], uint32_t (&hi)[4]) const {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const uint32_t l = ql[2 * w + i], h = qh[2 * w + i];
      scale_word<32>((l & 0x0f0f0f0fu) | ((h << 4) & 0x30303030u), d[w >> 1], c[w >> 1], lo[2 * i], lo[2 * i + 1]);
      scale_word<32>(((l >> 4) & 0x0f0f0f0fu) | (h & 0x30303030u), d[2 + (w >> 1)], c[2 + (w >> 1)], hi[2 * i], hi[2 * i + 1]);
    }
  }
  __device__ static __forceinline__ int x_place(int c) {
    return 4 * (4 * ((c >> 3) & 1) + (c & 3)) + 2 * (c >> 4) + ((c >> 2) & 1);
  }
};

// Q8_0 and IQ4_NL: lane t has blocks 2t (chunks 0-3) and 2t + 1 (chunks 4-7), as 16 words of offset bytes in
// element order.
template <int TYPE> struct LaneBlocks {
  uint32_t q[16];
  uint64_t d[2], c[2];
  __device__ __forceinline__ void fetch(const uint8_t *row, int, int t) {
    constexpr int QW = TYPE == kQ8_0 ? 8 : 4;   // words of quants in a block
    const uint8_t *a = row + (2 * QW + 1) * 4 * t;  // two blocks of 2 + 4 QW bytes
    uint32_t w[2 * QW + 1];
#pragma unroll
    for (int i = 0; i < 2 * QW + 1; i++) w[i] = lds32(a + 4 * i);
    const float d0 = half_bits(w[0] & 0xffffu), d1 = half_bits(w[QW] >> 16);
    d[0] = f2_pack(d0, d0);
    d[1] = f2_pack(d1, d1);
    c[0] = scale_offset<128>(d0);
    c[1] = scale_offset<128>(d1);
#pragma unroll
    for (int i = 0; i < QW; i++) {
      const uint32_t v0 = __funnelshift_r(w[i], w[i + 1], 16), v1 = w[QW + 1 + i];
      if constexpr (TYPE == kQ8_0) {
        q[i] = v0 ^ 0x80808080u;
        q[8 + i] = v1 ^ 0x80808080u;
      } else {  // element i: low nibble of byte i, element 16 + i: the high one
#pragma unroll
        for (int b = 0; b < 2; b++) {
          const uint32_t v = b ? v1 : v0, e = iq4nl_lookup4(v), f = iq4nl_lookup4(v >> 16);
          q[8 * b + i] = __byte_perm(e, f, 0x6420) ^ 0x80808080u;
          q[8 * b + 4 + i] = __byte_perm(e, f, 0x7531) ^ 0x80808080u;
        }
      }
    }
  }
  __device__ __forceinline__ void chunks(int w, uint32_t (&lo)[4], uint32_t (&hi)[4]) const {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      scale_word<128>(q[2 * w + i], d[0], c[0], lo[2 * i], lo[2 * i + 1]);
      scale_word<128>(q[8 + 2 * w + i], d[1], c[1], hi[2 * i], hi[2 * i + 1]);
    }
  }
  __device__ static __forceinline__ int x_place(int c) { return 4 * (c & 7) + (c >> 3); }
};
template <> struct Lane<kQ8_0> : LaneBlocks<kQ8_0> {};
template <> struct Lane<kIQ4_NL> : LaneBlocks<kIQ4_NL> {};

// The sums of a CTA's tile, left by its warps as [token][A row] f32 (rows kRows + 4 floats apart) in the idle
// ring, to its outputs, together with the other parts' of its cluster.
template <int kTokens, int kRows, bool GLU, int kThreads>
__device__ __forceinline__ void finish_rows(const RowsParams &p, const float *part, int m0, int n0, int parts, int rank) {
  constexpr int kOuts = GLU ? kRows / 2 : kRows;
  if (parts > 1) split_sync();
  else __syncthreads();
  const int live = min(kTokens, p.m_rows - m0);
  constexpr int kQuads = kOuts / 4;
  for (int i = rank * kThreads + threadIdx.x; i < live * kQuads; i += parts * kThreads) {
    const int token = i / kQuads, o = 4 * (i % kQuads);
    const int row = GLU ? 16 * (o >> 3) + (o & 7) : o;
    const uint32_t at = smem_u32(part + token * (kRows + 4) + row);
    const float4 a = sum_parts(at, parts);
    const float f[4] = {a.x, a.y, a.z, a.w};
    if constexpr (GLU) {
      const float4 b = sum_parts(at + 32, parts);
      const float u[4] = {b.x, b.y, b.z, b.w};
      glu_store4(p.epi, f, u, m0 + token, n0 + o, p.n_out);
    } else {
      epilogue_store4(p.epi, f, m0 + token, n0 + o, p.n_out);
    }
  }
  if (parts > 1) split_sync();  // nobody leaves while its partial tile is read
}
// One MMA tile's sums to its place there: A rows `row` and row + 8.
template <int NT, int kRows> __device__ __forceinline__ void leave_tile(const float (&acc)[NT][4], float *part, int row, int t) {
#pragma unroll
  for (int j = 0; j < NT; j++) {
    float *at = part + (8 * j + 2 * t) * (kRows + 4) + row;
    at[0] = acc[j][0];
    at[kRows + 4] = acc[j][1];
    at[8] = acc[j][2];
    at[kRows + 4 + 8] = acc[j][3];
  }
}

// Whether the tensor cores' sums, truncated at every step (kMaxF32Part), are taken a superblock at a time and added rounded to
// nearest: Q6_K 4096 x 12288, one row, 1.6e-6 -> 2.4e-7 of the norm, at the same time.  The gated form's bf16 result does not
// need it, and more than 32 tokens have no registers for it (3.4e-6).
template <int NT, bool GLU> constexpr bool kBySuperblock = !GLU && NT <= 4;

template <int TYPE, int NT, bool GLU, bool STAGED>
__global__ void __launch_bounds__(kRowThreads, 2)
    gemm_rows_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_up,
                     const RowsParams p) {
  using Cfg = RowCfg<TYPE>;
  constexpr int kStages = row_stages<TYPE, NT>(), kStageBytes = row_stage_bytes<TYPE, NT>();
  constexpr int kTokens = 8 * NT, kXOff = kRowTile * Cfg::RS;
  constexpr int kOuts = GLU ? kRowTile / 2 : kRowTile;
  static_assert(kTokens * (kRowTile + 4) * 4 <= kStages * kStageBytes, "the partial tile fits the ring");
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t smem0 = smem_u32(smem), bars = smem0 + kStages * kStageBytes;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * kOuts, m0 = blockIdx.y * kTokens;
  const int sb0 = blockIdx.z * p.per, nsb = min(p.per, p.nsb - sb0);
  const int parts = gridDim.z, rank = blockIdx.z;

  // The tile's rows of a matrix are kept inside it (boxes that reach beyond a matrix are avoided): the last block
  // fetches from raw_n0 on; its rows past the end are copies of the last one, whose sums are not stored.
  const int raw_n0 = STAGED ? min(n0, p.n_out - p.box_rows) : n0;
  // smem row of row r of the warp's tile
  auto stage_row = [&](int r) {
    const int mine = GLU ? 8 * warp + (r & 7) : 16 * warp + r;
    return (STAGED ? min(n0 + mine - raw_n0, p.box_rows - 1) : mine) + (GLU && r >= 8 ? kOuts : 0);
  };
  // byte offset of a row of its matrix, of the tile's smem row r (STAGED = false)
  auto row_offset = [&](int r) { return (long long)min(n0 + (GLU ? r & (kOuts - 1) : r), p.n_out - 1) * p.row_bytes; };
  auto issue_weights = [&](int i) {
    const uint32_t dst = smem0 + (i % kStages) * kStageBytes;
    if constexpr (STAGED) {
      if (tid == 0) {
        const uint32_t full = bars + 8 * (i % kStages);
        mbar_arrive_expect_tx(full, (GLU ? 2 : 1) * p.box_rows * Cfg::RS);
        // 4-byte elements; 16-byte boundaries
        const int at = (TYPE == kQ6_K ? min((Cfg::SB * (sb0 + i)) & ~15, (int)p.row_bytes - Cfg::RS) : Cfg::SB * (sb0 + i)) >> 2;
        tma_load_2d(dst, &tmap_w, at, raw_n0, full);
        if constexpr (GLU) tma_load_2d(dst + kOuts * Cfg::RS, &tmap_up, at, raw_n0, full);
      }
    } else {
      // from the 16-byte boundary below each block; in the last rows not beyond the matrix's end
      const long long w_bytes = (long long)p.n_out * p.row_bytes;
      const bool tail = n0 + kOuts >= p.n_out && sb0 + i + 1 == p.nsb;
#pragma unroll
      for (int j = 0; j < kRowTile * kQ6Chunks / kRowThreads; j++) {
        const int at = kRowThreads * j + tid, r = at / kQ6Chunks, c = at % kQ6Chunks;
        const uint8_t *base = GLU && r >= kOuts ? p.w_up : p.w;
        const long long off = ((row_offset(r) + (long long)(sb0 + i) * Cfg::SB) & ~15ll) + 16 * c;
        const int bytes = !tail || off + 16 <= w_bytes ? 16 : off < w_bytes ? (int)(w_bytes - off) : 0;
        cp_async16(dst + r * Cfg::RS + 16 * c, base + (bytes ? off : 0), bytes);
      }
    }
  };
  auto issue_x = [&](int i) {
    const uint32_t dst = smem0 + (i % kStages) * kStageBytes + kXOff;
#pragma unroll
    for (int j = 0; j < NT; j++) {
      const int at = kRowThreads * j + tid, token = at >> 5, c = at & 31;
      const bool in = m0 + token < p.m_rows;
      const __nv_bfloat16 *a = p.x + (in ? (long long)(m0 + token) * p.x_stride : 0) + (sb0 + i) * 256 + 8 * c;
      cp_async16(dst + token * kTokenStride + 16 * Lane<TYPE>::x_place(c), a, in ? 16 : 0);
    }
  };

  if constexpr (STAGED) {
    if (tid == 0) {
      for (int i = 0; i < kStages; i++) mbar_init(bars + 8 * i, 1);
      mbar_fence_init();
    }
    __syncthreads();
  }
  pdl_launch_dependents();
  if (!p.resident) pdl_wait_prior_grid();
#pragma unroll
  for (int i = 0; i < kStages - 1; i++)
    if (i < nsb) issue_weights(i);
  if (p.resident) pdl_wait_prior_grid();
#pragma unroll
  for (int i = 0; i < kStages - 1; i++) {
    if (i < nsb) issue_x(i);
    cp_async_commit();
  }

  float acc[NT][4] = {};
  const uint8_t *row0 = smem + stage_row(g) * Cfg::RS, *row1 = smem + stage_row(g + 8) * Cfg::RS;
  const uint8_t *x_lane = smem + kXOff + g * kTokenStride + 16 * t;
  const uint32_t off0 = STAGED ? 0u : (uint32_t)row_offset(stage_row(g)), off1 = STAGED ? 0u : (uint32_t)row_offset(stage_row(g + 8));
  bool ok = true;
#pragma unroll 1
  for (int i = 0; i < nsb; i++) {
    cp_async_wait<kStages - 2>();
    if constexpr (STAGED) {
      ok &= mbar_wait(bars + 8 * (i % kStages), (i / kStages) & 1);
      // the barrier orders the reads of stage i - 1 against threads, this against the TMA copy that fills it again (0.4 %)
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();  // stage i has landed for every warp, stage i - 1 is free
    if (i + kStages - 1 < nsb) {
      issue_weights(i + kStages - 1);
      issue_x(i + kStages - 1);
    }
    cp_async_commit();
    const uint32_t stage = (i % kStages) * kStageBytes;
    Lane<TYPE> r0, r1;
    const int at = Cfg::SB * (sb0 + i);  // Q6_K: where the block starts in its window
    const int in_window = TYPE == kQ6_K && STAGED ? at - min(at & ~15, (int)p.row_bytes - Cfg::RS) : 0;
    r0.fetch(row0 + stage, STAGED ? in_window : (off0 + at) & 15, t);
    r1.fetch(row1 + stage, STAGED ? in_window : (off1 + at) & 15, t);
    float sum[NT][4] = {};  // of this superblock
    float(&to)[NT][4] = kBySuperblock<NT, GLU> ? sum : acc;
#pragma unroll
    for (int w = 0; w < 4; w++) {
      uint32_t l0[4], h0[4], l1[4], h1[4];
      r0.chunks(w, l0, h0);
      r1.chunks(w, l1, h1);
#pragma unroll
      for (int j = 0; j < NT; j++) {
        const uint4 xl = lds128(x_lane + stage + j * 8 * kTokenStride + 64 * w);
        const uint4 xh = lds128(x_lane + stage + j * 8 * kTokenStride + 64 * (4 + w));
        mma_bf16(to[j], l0[0], l1[0], l0[1], l1[1], xl.x, xl.y);
        mma_bf16(to[j], l0[2], l1[2], l0[3], l1[3], xl.z, xl.w);
        mma_bf16(to[j], h0[0], h1[0], h0[1], h1[1], xh.x, xh.y);
        mma_bf16(to[j], h0[2], h1[2], h0[3], h1[3], xh.z, xh.w);
      }
    }
    if constexpr (kBySuperblock<NT, GLU>) {
#pragma unroll
      for (int j = 0; j < NT; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) acc[j][e] += sum[j][e];
    }
  }
  cp_async_wait<0>();
  if (!ok) drain_copies_in_flight();
  __syncthreads();

  float *part = reinterpret_cast<float *>(smem);
  leave_tile<NT, kRowTile>(acc, part, 16 * warp + g, t);
  finish_rows<kTokens, kRowTile, GLU, kRowThreads>(p, part, m0, n0, parts, rank);
}

// The kernel's parameters but for the split, and the weights' tensor maps (gate or only matrix, up matrix); `outs`: its
// outputs per CTA; box_row: bytes of a box's rows, 0: none.
template <int TYPE, bool GLU> int rows_params(const RowsCall &c, int box_row, int outs, RowsParams &p, CUtensorMap (&maps)[2]) {
  p.w = static_cast<const uint8_t *>(c.w);
  p.w_up = static_cast<const uint8_t *>(c.w_up);
  p.x = static_cast<const __nv_bfloat16 *>(c.x);
  p.x_stride = c.x_stride;
  p.nsb = c.k_in / 256;
  p.row_bytes = (long long)p.nsb * RowCfg<TYPE>::SB;
  p.m_rows = c.m_rows; p.n_out = c.n_out;
  p.resident = c.resident;
  p.epi = c.epi;
  p.box_rows = c.n_out < outs ? c.n_out : outs;
  if (!box_row) return COGNI_QMM_OK;  // no TMA
  EncodeTiledFn encode = encode_tiled_fn();
  if (!encode) return COGNI_QMM_ERR_DEVICE;
  // 4-byte elements: a box has at most 256 along a dimension
  const cuuint64_t dims[2] = {(cuuint64_t)p.row_bytes / 4, (cuuint64_t)c.n_out}, strides[1] = {(cuuint64_t)p.row_bytes};
  const cuuint32_t box[2] = {(cuuint32_t)box_row / 4, (cuuint32_t)p.box_rows}, estr[2] = {1, 1};
  for (int i = 0; i < (GLU ? 2 : 1); i++) {
    const CUresult r = encode(&maps[i], CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void *>(i ? c.w_up : c.w), dims, strides,
                              box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return (int)r;
  }
  return COGNI_QMM_OK;
}

typedef void (*RowsKernel)(CUtensorMap, CUtensorMap, RowsParams);

// Opts into the shared memory, once per device; `once` is the caller's, one per kernel.
struct RowsOnce {
  std::atomic<bool> configured[64];
  int sms[64];
  std::atomic<int> clusters[64][9];  // 1 + how many clusters of that many CTAs run at once
};
inline int rows_configure(RowsOnce &once, const void *kernel, int smem, int &sms) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return COGNI_QMM_ERR_DEVICE;
  if (!once.configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&once.sms[dev], cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return (int)e;
    once.configured[dev] = true;
  }
  sms = once.sms[dev];
  return COGNI_QMM_OK;
}

inline int rows_clusters(RowsOnce &once, RowsKernel kernel, int threads, int smem, int parts) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return 0;
  std::atomic<int> &slot = once.clusters[dev][parts];
  int v = slot.load();
  if (v == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1, 1, parts);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = parts;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 0) {
      cudaGetLastError();  // not cut into that many then
      n = 0;
    }
    v = n + 1;
    slot.store(v);
  }
  return v - 1;
}

// Chooses the split along K and launches.
inline int rows_launch(RowsOnce &once, RowsKernel kernel, RowsParams &p, const CUtensorMap (&maps)[2], int outs, int tokens, int threads, int smem,
                       int sms, cudaStream_t s) {
  const int blocks = (p.n_out + outs - 1) / outs, tiles = (p.m_rows + tokens - 1) / tokens;
  // Parts of K.  Clusters of n CTAs come in waves of as many as fit the GPU, two CTAs an SM; a CTA takes its superblocks
  // and a start and an end, beside another one not twice as long as alone.  Measured over every split, both forms, five types, 1 to
  // 48 tokens: with these constants 1.1 % over the best on average for 1024 to 17408 rows of 4096 to 17408 columns as layers have
  // them, 2.6 % for drawn shapes (126 of 1122 more than 10 %).  1.75 instead of 1.3 and 1.0 instead of 0.75 make that 0.9 %, but
  // 12288 x 4096 onto f32 takes 9 to 25 % longer with them.
  int parts = 1;
  double best = 1e30;
  for (int n = 1; n <= 8 && n <= p.nsb; n++) {
    const int per = (p.nsb + n - 1) / n;
    if ((n - 1) * per >= p.nsb) continue;  // a part would be empty
    const int at_once = rows_clusters(once, kernel, threads, smem, n);
    if (at_once == 0) continue;
    const long long clusters = (long long)blocks * tiles, rest = clusters % at_once * n;  // CTAs of the last wave
    const double load = clusters / at_once * 2.0 + (rest == 0 ? 0.0 : rest <= sms ? 1.3 : 2.0);
    double cost = load * (per + 0.75) + (n > 1 ? 0.5 : 0.0);
    if (!p.epi.y_bf16 && tokens > 32 && 256 * per > kMaxF32Part) cost += 1e7 * per;  // the shortest parts if none is short enough
    if (cost < best) { best = cost; parts = n; }
  }
  p.per = (p.nsb + parts - 1) / parts;
  parts = (p.nsb + p.per - 1) / p.per;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks, tiles, parts);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = parts;
  cfg.attrs = attr;
  cfg.numAttrs = parts > 1 ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, kernel, maps[0], maps[1], p);
}

template <int TYPE, int NT, bool GLU, bool STAGED> int launch_rows_tile(const RowsCall &c, cudaStream_t s) {
  static RowsOnce once;
  RowsParams p;
  CUtensorMap maps[2] = {};
  int sms = 0, st = rows_configure(once, reinterpret_cast<const void *>(gemm_rows_kernel<TYPE, NT, GLU, STAGED>), row_smem<TYPE, NT>(), sms);
  constexpr int outs = GLU ? kRowTile / 2 : kRowTile;
  if (!st) st = rows_params<TYPE, GLU>(c, STAGED ? RowCfg<TYPE>::RS : 0, outs, p, maps);
  if (st) return st;
  return rows_launch(once, gemm_rows_kernel<TYPE, NT, GLU, STAGED>, p, maps, outs, 8 * NT, kRowThreads, row_smem<TYPE, NT>(), sms, s);
}

template <int TYPE, bool GLU, bool STAGED> int launch_rows_width(const RowsCall &c, cudaStream_t s) {
  // the narrowest tile that holds all rows (rows_kernel_takes)
  if (c.m_rows <= 8) return launch_rows_tile<TYPE, 1, GLU, STAGED>(c, s);
  if (c.m_rows <= 16) return launch_rows_tile<TYPE, 2, GLU, STAGED>(c, s);
  if (c.m_rows <= 24) return launch_rows_tile<TYPE, 3, GLU, STAGED>(c, s);
  if constexpr (TYPE == kQ6_K || TYPE == kQ8_0) {
    if (c.m_rows > 48) return launch_rows_tile<TYPE, 8, GLU, STAGED>(c, s);
    if (c.m_rows > 32) return launch_rows_tile<TYPE, 6, GLU, STAGED>(c, s);
  }
  return launch_rows_tile<TYPE, 4, GLU, STAGED>(c, s);
}

template <bool GLU> int launch_rows(const RowsCall &c, cudaStream_t s) {
  switch (c.type) {
    case kQ4_K: return launch_rows_width<kQ4_K, GLU, true>(c, s);
    case kQ5_K: return launch_rows_width<kQ5_K, GLU, true>(c, s);
    case kQ6_K: return c.k_in % 2048 == 0 ? launch_rows_width<kQ6_K, GLU, true>(c, s) : launch_rows_width<kQ6_K, GLU, false>(c, s);
    case kQ8_0: return launch_rows_width<kQ8_0, GLU, true>(c, s);
    case kIQ4_NL: return launch_rows_width<kIQ4_NL, GLU, true>(c, s);
    default: return COGNI_QMM_ERR_TYPE;
  }
}

unsigned rows_timeouts() {
  unsigned v = 0;
  cudaMemcpyFromSymbol(&v, g_pipe_wait_timeouts, sizeof(v));
  return v;
}
int rows_reset_timeouts() {
  const unsigned zero = 0;
  return (int)cudaMemcpyToSymbol(g_pipe_wait_timeouts, &zero, sizeof(zero));
}

}  // namespace
}  // namespace cogni
