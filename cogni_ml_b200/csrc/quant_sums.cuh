// Q4_K / Q5_K products with a bf16 result by sums of raw quants per scale group on the tensor cores, scaled in f32:
//
//     sum_k x[k] (d q[k] - m)  over a group of 32  =  d sum_k x[k] (128 + q[k])  -  (m + 128 d) sum_k x[k]
//
// A quant becomes a bf16 operand by a byte permute (byte q under the byte 0x43 is 128 + q exactly): seven
// instructions per eight weights and lane where the expansion to rounded weights takes 23, and the ALU does two a
// cycle.  The weights enter unrounded; the 128 costs four bits of the f32 sums.  The K = 16 of an MMA has to lie in
// one group for all lanes, so lane t of a quad takes the eight weights 8 t .. of every group (bytes 8 t .. of 32;
// low nibbles one group, high ones the next).  Every lane decodes the scales of its two rows itself: four lanes do
// the same work, but exchanging them costs more shared-memory cycles than the weights.
#pragma once

#include "gemm_rows.cuh"

namespace cogni {
namespace {

__device__ __forceinline__ void mma_bf16_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                              uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// Four bytes below 128 as the bf16 pairs (128 + b0, 128 + b1), (128 + b2, 128 + b3).
__device__ __forceinline__ void bytes_plus128(uint32_t q, uint32_t &r0, uint32_t &r1) {
  r0 = __byte_perm(q, 0x43434343u, 0x4140);
  r1 = __byte_perm(q, 0x43434343u, 0x4342);
}

// The scales of a lane's two rows: groups 0-3 and 4-7 as bytes, d and -dmin of both rows as pairs.  d sc and -dmin m
// are rounded once: fma(2^23 + b, d, -2^23 d) = b d, the product with 2^23 being exact.
struct RowScales {
  uint32_t sc[2][2], mn[2][2];
  uint64_t d, nd, dm, ndm;
  __device__ __forceinline__ void fetch(const uint8_t *row0, const uint8_t *row1) {
    float df[2], mf[2];
#pragma unroll
    for (int r = 0; r < 2; r++) {
      const uint4 h = lds128(r ? row1 : row0);  // d, dmin, the 6-bit scales and minimums (dequant.cr:240-249)
      sc[r][0] = h.y & 0x3f3f3f3fu;
      mn[r][0] = h.z & 0x3f3f3f3fu;
      sc[r][1] = (h.w & 0x0f0f0f0fu) | ((h.y >> 2) & 0x30303030u);
      mn[r][1] = ((h.w >> 4) & 0x0f0f0f0fu) | ((h.z >> 2) & 0x30303030u);
      const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&h.x));
      df[r] = v.x;
      mf[r] = -v.y;
    }
    d = f2_pack(df[0], df[1]);
    dm = f2_pack(mf[0], mf[1]);
    const uint64_t bias = f2_pack(-8388608.f, -8388608.f);
    nd = f2_mul(bias, d);
    ndm = f2_mul(bias, dm);
  }
  // of group s, both rows: the scale d sc, and what goes to the sum of the activations, -(dmin m + 128 d sc)
  __device__ __forceinline__ void group(int s, float (&scale)[2], float (&offset)[2]) const {
    auto bytes = [&](const uint32_t (&v)[2][2]) {
      return f2_pack(__uint_as_float(__byte_perm(v[0][s >> 2], 0x4B000000u, 0x7650 + (s & 3))),
                     __uint_as_float(__byte_perm(v[1][s >> 2], 0x4B000000u, 0x7650 + (s & 3))));
    };
    const uint64_t ds = f2_fma(bytes(sc), d, nd);
    const uint64_t of = f2_fma(f2_pack(-128.f, -128.f), ds, f2_fma(bytes(mn), dm, ndm));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(scale[0]), "=f"(scale[1]) : "l"(ds));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(offset[0]), "=f"(offset[1]) : "l"(of));
  }
};

// One superblock of U tiles of 16 rows (the lane's two of each at rows[u]) against NT x 8 tokens: x_at(j, s) the
// lane's activations of group s, column 8 j + g; xs: the activations' sums, [group][token] f32, at tokens 2t, 2t + 1.
template <int TYPE, int NT, int U, class AT>
__device__ __forceinline__ void sums_tiles(const uint8_t *const (&rows)[U][2], const AT &x_at, const uint8_t *xs, int t,
                                           float (&acc)[U][NT][4]) {
  static_assert(TYPE == kQ4_K || TYPE == kQ5_K, "groups of 32 with a minimum");
  constexpr int kQuants = TYPE == kQ5_K ? 48 : 16;
  RowScales sc[U];
  uint2 fifth[U][2];  // Q5_K: the fifth bits of the lane's eight weights of every group, bit s for group s
#pragma unroll
  for (int u = 0; u < U; u++) {
    sc[u].fetch(rows[u][0], rows[u][1]);
    if (TYPE == kQ5_K) {
      fifth[u][0] = lds64(rows[u][0] + 16 + 8 * t);
      fifth[u][1] = lds64(rows[u][1] + 16 + 8 * t);
    }
  }
#pragma unroll
  for (int pair = 0; pair < 4; pair++) {
    uint2 q[U][2];
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int h = 0; h < 2; h++) q[u][h] = lds64(rows[u][h] + kQuants + 32 * pair + 8 * t);
#pragma unroll
    for (int hi = 0; hi < 2; hi++) {
      const int s = 2 * pair + hi;
      uint4 x[NT];
      uint2 n[NT];
#pragma unroll
      for (int j = 0; j < NT; j++) {
        x[j] = x_at(j, s);
        n[j] = lds64(xs + (s * 8 * NT + 8 * j) * 4);
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        uint32_t a[2][4];
        float d[2], c[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const uint32_t w[2] = {q[u][h].x, q[u][h].y};
#pragma unroll
          for (int e = 0; e < 2; e++) {
            uint32_t v = (hi ? w[e] >> 4 : w[e]) & 0x0f0f0f0fu;
            if constexpr (TYPE == kQ5_K) {
              const uint32_t f = e ? fifth[u][h].y : fifth[u][h].x;
              v |= (s < 4 ? f << (4 - s) : f >> (s - 4)) & 0x10101010u;
            }
            bytes_plus128(v, a[h][2 * e], a[h][2 * e + 1]);
          }
        }
        sc[u].group(s, d, c);
#pragma unroll
        for (int j = 0; j < NT; j++) {
          float sum[4];
          mma_bf16_zero(sum, a[0][0], a[1][0], a[0][1], a[1][1], x[j].x, x[j].y);
          mma_bf16(sum, a[0][2], a[1][2], a[0][3], a[1][3], x[j].z, x[j].w);
          float(&o)[4] = acc[u][j];
          o[0] = fmaf(d[0], sum[0], fmaf(c[0], __uint_as_float(n[j].x), o[0]));
          o[1] = fmaf(d[0], sum[1], fmaf(c[0], __uint_as_float(n[j].y), o[1]));
          o[2] = fmaf(d[1], sum[2], fmaf(c[1], __uint_as_float(n[j].x), o[2]));
          o[3] = fmaf(d[1], sum[3], fmaf(c[1], __uint_as_float(n[j].y), o[3]));
        }
      }
    }
  }
}
// The sums of the activations of one group, tokens 8 j + 2t and + 1, by MMAs with a matrix of ones; v: as x_at.
__device__ __forceinline__ float2 sum_group(const uint4 &v) {
  const uint32_t ones = 0x3f803f80u;
  float s[4];
  mma_bf16_zero(s, ones, ones, ones, ones, v.x, v.y);
  mma_bf16(s, ones, ones, ones, ones, v.z, v.w);
  return make_float2(s[0], s[1]);
}

}  // namespace
}  // namespace cogni
