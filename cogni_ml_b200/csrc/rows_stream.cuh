// Products with an epilogue for the fewest rows (1 .. 16 tokens, sm_100a): every warp streams weights of its own.
//
// With so few tokens the weights' bytes are the floor, and what keeps a kernel from it are the
// instructions per weight and whatever makes warps wait for one another.  So:
//   * A CTA per SM takes whole tiles of 16 weight rows (the M of mma.sync.m16n8k16) along all of K.  Its work is a
//     list of items, one superblock column of a tile each, in the order of the tiles; its sixteen warps take
//     equal runs of the list.  No split over CTAs, no cluster, no barrier in the loop: 12288 x 4096 with gate and
//     up, one row: 10.4 tiles an SM on average, 11 at most.
//   * A warp fetches its items itself, by TMA into a ring of its own, up to four boxes ahead: 16 rows (gate and up: 8
//     of each) of two superblocks where these are short, so that a row of a box is 240 bytes or more.  (Measured,
//     gate + up 12288 x 4096 Q4_K, copies alone: boxes of 8 rows x 144 bytes 12.1 us; 16-byte cp.async 8.3 us, but
//     it takes a shared-memory cycle per 32 bytes, as many as all the reads.)
//   * The activations of all of K lie in shared memory, m_rows tokens of them (lanes whose column stands for no token
//     read another one's; that column is never stored).  Shapes for which they do not fit go to gemm_rows.cuh.
//   * A warp adds up an item after the other in its accumulators and leaves them in shared memory when its run
//     leaves a tile; the parts of a tile are added in the order of the warps, the same every time.
// How an item is computed is the template parameter:
//   Rounded  weights expanded to bf16(dequant(W)) in registers (Lane<TYPE>, gemm_rows.cuh)
//   Sums     Q4_K / Q5_K with a bf16 result: sums of raw quants per scale group, scaled in f32,
//                sum_k x[k] (d q[k] - m)  over a group of 32  =  d sum_k x[k] (128 + q[k])  -  (m + 128 d) sum_k x[k]
//            A quant becomes a bf16 operand by a byte permute (byte q under the byte 0x43 is 128 + q exactly):
//            seven instructions per eight weights and lane where the expansion takes 23, and an ALU that does two
//            a cycle.  The weights enter unrounded; the 128 costs four bits of the f32 sums.
#pragma once

#include "gemm_rows.cuh"

namespace cogni {
namespace {

constexpr int kStreamWarps = 16;
constexpr int kStreamThreads = 32 * kStreamWarps;
constexpr int kStreamStages = 4;  // at most, of a warp's ring

// A box's superblocks, and the bytes of its rows (Q6_K: the window that holds a block, see RowCfg)
template <int TYPE> __host__ __device__ constexpr int box_sbs() { return RowCfg<TYPE>::SB < 200 ? 2 : 1; }
template <int TYPE> __host__ __device__ constexpr int box_row() { return box_sbs<TYPE>() * RowCfg<TYPE>::RS; }

struct StreamParams {
  RowsParams r;
  int tiles;             // of all rows
  int tiles_per_cta, stages;
  int x_stride;          // bytes between the tokens of the staged activations
  int off_ring, off_sums, off_part;  // shared memory, after the activations
};

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

// An item, Rounded: the lane's two rows at row0 / row1 (Q6_K: the block `off` bytes into them), the superblock's
// activations of the lane's column at x (the quad's bytes already chosen).
template <int TYPE, int NT> struct Rounded {
  static constexpr bool kSums = false;
  __device__ static __forceinline__ int x_place(int c) { return Lane<TYPE>::x_place(c); }
  __device__ static __forceinline__ void item(const uint8_t *row0, const uint8_t *row1, int off0, int off1,
                                              const uint8_t *const (&x)[NT], const uint8_t *, int t, float (&acc)[NT][4]) {
    Lane<TYPE> r0, r1;
    r0.fetch(row0, off0, t);
    r1.fetch(row1, off1, t);
#pragma unroll
    for (int w = 0; w < 4; w++) {
      uint32_t l0[4], h0[4], l1[4], h1[4];
      r0.chunks(w, l0, h0);
      r1.chunks(w, l1, h1);
#pragma unroll
      for (int j = 0; j < NT; j++) {
        const uint4 xl = lds128(x[j] + 64 * w), xh = lds128(x[j] + 64 * (4 + w));
        mma_bf16(acc[j], l0[0], l1[0], l0[1], l1[1], xl.x, xl.y);
        mma_bf16(acc[j], l0[2], l1[2], l0[3], l1[3], xl.z, xl.w);
        mma_bf16(acc[j], h0[0], h1[0], h0[1], h1[1], xh.x, xh.y);
        mma_bf16(acc[j], h0[2], h1[2], h0[3], h1[3], xh.z, xh.w);
      }
    }
  }
};

// Sums: the K = 16 of an MMA has to lie in one group for all lanes, so lane t of a quad takes the eight weights 8 t ..
// of every group (bytes 8 t .. of 32; low nibbles one group, high ones the next).  Every lane decodes the
// scales of its two rows itself: four lanes do the same work, but exchanging them costs more shared-memory
// cycles than the weights.  xs: the sums of the activations of the superblock's groups for tokens 2t, 2t + 1.
template <int TYPE, int NT> struct Sums {
  static_assert(TYPE == kQ4_K || TYPE == kQ5_K, "groups of 32 with a minimum");
  static constexpr bool kSums = true;
  __device__ static __forceinline__ int x_place(int c) { return c; }
  __device__ static __forceinline__ void item(const uint8_t *row0, const uint8_t *row1, int, int,
                                              const uint8_t *const (&x)[NT], const uint8_t *xs, int t, float (&acc)[NT][4]) {
    constexpr int kQuants = TYPE == kQ5_K ? 48 : 16;
    RowScales sc;
    sc.fetch(row0, row1);
    uint2 fifth[2];  // Q5_K: the fifth bits of the lane's eight weights of every group, bit s for group s
    if (TYPE == kQ5_K) {
      fifth[0] = lds64(row0 + 16 + 8 * t);
      fifth[1] = lds64(row1 + 16 + 8 * t);
    }
#pragma unroll
    for (int pair = 0; pair < 4; pair++) {
      const uint2 q[2] = {lds64(row0 + kQuants + 32 * pair + 8 * t), lds64(row1 + kQuants + 32 * pair + 8 * t)};
#pragma unroll
      for (int hi = 0; hi < 2; hi++) {
        const int s = 2 * pair + hi;
        uint32_t a[2][4];
        float d[2], c[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const uint32_t w[2] = {q[h].x, q[h].y};
#pragma unroll
          for (int e = 0; e < 2; e++) {
            uint32_t v = (hi ? w[e] >> 4 : w[e]) & 0x0f0f0f0fu;
            if constexpr (TYPE == kQ5_K) {
              const uint32_t f = e ? fifth[h].y : fifth[h].x;
              v |= (s < 4 ? f << (4 - s) : f >> (s - 4)) & 0x10101010u;
            }
            bytes_plus128(v, a[h][2 * e], a[h][2 * e + 1]);
          }
        }
        sc.group(s, d, c);
#pragma unroll
        for (int j = 0; j < NT; j++) {
          const uint4 v = lds128(x[j] + 64 * s);
          const uint2 n = lds64(xs + (s * 8 * NT + 8 * j) * 4);
          float sum[4];
          mma_bf16_zero(sum, a[0][0], a[1][0], a[0][1], a[1][1], v.x, v.y);
          mma_bf16(sum, a[0][2], a[1][2], a[0][3], a[1][3], v.z, v.w);
          acc[j][0] = fmaf(d[0], sum[0], fmaf(c[0], __uint_as_float(n.x), acc[j][0]));
          acc[j][1] = fmaf(d[0], sum[1], fmaf(c[0], __uint_as_float(n.y), acc[j][1]));
          acc[j][2] = fmaf(d[1], sum[2], fmaf(c[1], __uint_as_float(n.x), acc[j][2]));
          acc[j][3] = fmaf(d[1], sum[3], fmaf(c[1], __uint_as_float(n.y), acc[j][3]));
        }
      }
    }
  }
};

template <int TYPE, int NT, bool GLU, class ITEM>
__global__ void __launch_bounds__(kStreamThreads, 1)
    rows_stream_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_up,
                       const __grid_constant__ StreamParams sp) {
  using Cfg = RowCfg<TYPE>;
  const RowsParams &p = sp.r;
  constexpr int kTokens = 8 * NT, kOuts = GLU ? 8 : 16, kS = box_sbs<TYPE>(), kRow = box_row<TYPE>(), kBox = 16 * kRow;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const uint32_t bars = smem_u32(smem) + 8 * kStreamStages * warp;  // the warp's barriers, before the activations
  uint8_t *x0 = smem + 8 * kStreamStages * kStreamWarps;
  uint8_t *ring = smem + sp.off_ring + warp * sp.stages * kBox;
  const int tile0 = blockIdx.x * sp.tiles_per_cta, tiles = min(sp.tiles_per_cta, sp.tiles - tile0);
  const int nsb = p.nsb, items = tiles * nsb, per_tile = (nsb + kS - 1) / kS;  // boxes along a tile
  const int first = warp * items / kStreamWarps, last = (warp + 1) * items / kStreamWarps;

  auto out_of = [&](int tile) { return (tile0 + tile) * kOuts; };  // the first output of a tile
  // the first superblock of box b of a tile (two at a time: the last box of an odd number starts one earlier)
  auto box_start = [&](int b) { return min(kS * b, nsb - kS); };
  // byte in the row where the box at superblock s starts
  auto box_byte = [&](int s) { return TYPE == kQ6_K ? min((Cfg::SB * s) & ~15, (int)p.row_bytes - kRow) : Cfg::SB * s; };

  // the warp's boxes: from that of its first item to that of its last; the next one that is not yet under way
  const int tile_a = first / nsb, box_a = (first - tile_a * nsb) / kS;
  const int tile_z = (last - 1) / nsb, box_z = (last - 1 - tile_z * nsb) / kS;
  int boxes = first < last ? (tile_z - tile_a) * per_tile + box_z - box_a + 1 : 0;
  int next_tile = tile_a, next_box = box_a;
  auto issue = [&](int s) {  // into slot s of the ring
    if (boxes > 0 && lane == 0) {
      const uint32_t full = bars + 8 * s, dst = smem_u32(ring) + s * kBox;
      // kept inside the matrix: rows past its end are copies of the last one, whose sums are not stored
      const int at = box_byte(box_start(next_box)) >> 2, from = min(out_of(next_tile), p.n_out - p.box_rows);
      mbar_arrive_expect_tx(full, (GLU ? 2 : 1) * p.box_rows * kRow);
      tma_load_2d(dst, &tmap_w, at, from, full);  // 4-byte elements, 16-byte boundaries
      if constexpr (GLU) tma_load_2d(dst + 8 * kRow, &tmap_up, at, from, full);
    }
    boxes--;
    if (++next_box == per_tile) {
      next_box = 0;
      next_tile++;
    }
  };

  if (lane < sp.stages) mbar_init(bars + 8 * lane, 1);
  mbar_fence_init();
  __syncwarp();
  pdl_launch_dependents();
  if (!p.resident) pdl_wait_prior_grid();
  for (int s = 0; s < sp.stages; s++) issue(s);
  if (p.resident) pdl_wait_prior_grid();
  for (int i = tid; i < p.m_rows * nsb * 32; i += kStreamThreads) {
    const int token = i / (nsb * 32), c = i - token * nsb * 32;
    cp_async16(smem_u32(x0) + token * sp.x_stride + 512 * (c >> 5) + 16 * ITEM::x_place(c & 31), p.x + token * p.x_stride + 8 * c);
  }
  cp_async_commit();
  cp_async_wait<0>();
  __syncthreads();
  const uint8_t *x_lane[NT];
#pragma unroll
  for (int j = 0; j < NT; j++) x_lane[j] = x0 + min(8 * j + g, p.m_rows - 1) * sp.x_stride + 16 * t;
  if constexpr (ITEM::kSums) {
    // the sums of the activations, [superblock][group][token], by MMAs with a matrix of ones
    const uint32_t ones = 0x3f803f80u;
    for (int i = warp; i < 8 * nsb; i += kStreamWarps) {
#pragma unroll
      for (int j = 0; j < NT; j++) {
        const uint4 v = lds128(x_lane[j] + 64 * i);
        float s[4];
        mma_bf16_zero(s, ones, ones, ones, ones, v.x, v.y);
        mma_bf16(s, ones, ones, ones, ones, v.z, v.w);
        if (g == 0) *reinterpret_cast<float2 *>(smem + sp.off_sums + (i * kTokens + 8 * j + 2 * t) * 4) = make_float2(s[0], s[1]);
      }
    }
    __syncthreads();
  }
  float acc[NT][4] = {};
  float *part = reinterpret_cast<float *>(smem + sp.off_part);
  int tile = tile_a, sb = first - tile_a * nsb, slot = 0, phase = 0;
  bool ok = true;
#pragma unroll 1
  for (int i = first; i < last;) {
    ok &= mbar_wait(bars + 8 * slot, phase);
    // the box's items that are in the run
    const int n0 = out_of(tile), from = min(n0, p.n_out - p.box_rows);
    const int start = box_start(sb / kS), end = min((sb / kS + 1) * kS, nsb);
    auto stage_row = [&](int r) { return min(n0 + (GLU ? r & 7 : r) - from, p.box_rows - 1) + (GLU && r >= 8 ? 8 : 0); };
    const uint8_t *row0 = ring + slot * kBox + stage_row(g) * kRow, *row1 = ring + slot * kBox + stage_row(g + 8) * kRow;
#pragma unroll 1
    for (; sb < end && i < last; sb++, i++) {
      const uint8_t *x[NT];
#pragma unroll
      for (int j = 0; j < NT; j++) x[j] = x_lane[j] + 512 * sb;
      // Q6_K: the block's place in its window
      const int off = TYPE == kQ6_K ? Cfg::SB * sb - box_byte(start) : 0, in_box = TYPE == kQ6_K ? 0 : Cfg::SB * (sb - start);
      ITEM::item(row0 + in_box, row1 + in_box, off, off, x, smem + sp.off_sums + sb * 8 * kTokens * 4 + 8 * t, t, acc);
    }
    __syncwarp();  // the box has been read
    issue(slot);
    if (++slot == sp.stages) {
      slot = 0;
      phase ^= 1;
    }
    if (sb == nsb || i == last) {
      // part warp + tile: (warp, tile) grows along the list of items, so no two of them meet
      float *to = part + (warp + tile) * 16 * kTokens;
#pragma unroll
      for (int j = 0; j < NT; j++) {
        float *at_token = to + (8 * j + 2 * t) * 16 + g;
        at_token[0] = acc[j][0];
        at_token[16] = acc[j][1];
        at_token[8] = acc[j][2];
        at_token[24] = acc[j][3];
        acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
      }
      sb = 0;
      tile++;
    }
  }
  if (!ok) drain_copies_in_flight();
  __syncthreads();

  // every output from the parts of its tile: the warps whose runs meet items tile nsb .. (tile + 1) nsb - 1
  constexpr int kQuads = kOuts / 4;
  for (int i = tid; i < tiles * kQuads * p.m_rows; i += kStreamThreads) {
    const int token = i / (tiles * kQuads), q = i - token * tiles * kQuads, tl = q / kQuads, o = 4 * (q % kQuads);
    const int w0 = (kStreamWarps * (tl * nsb + 1) - 1) / items, w1 = (kStreamWarps * (tl + 1) * nsb - 1) / items;
    float a[4] = {}, b[4] = {};
    for (int w = w0; w <= w1; w++) {
      if (items < kStreamWarps && w * items / kStreamWarps == (w + 1) * items / kStreamWarps) continue;  // a warp without items
      const float *from = part + (w + tl) * 16 * kTokens + token * 16 + o;
#pragma unroll
      for (int k = 0; k < 4; k++) {
        a[k] += from[k];
        if (GLU) b[k] += from[8 + k];
      }
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
      a[k] *= p.gain;
      b[k] *= p.gain;
    }
    if constexpr (GLU) glu_store4(p.epi, a, b, token, out_of(tl) + o, p.n_out);
    else epilogue_store4(p.epi, a, token, out_of(tl) + o, p.n_out);
  }
}

// Shared memory of a launch; false if the activations leave no room for a ring of two.
template <int TYPE, int NT, bool SUMS> bool stream_layout(StreamParams &sp, int &bytes) {
  constexpr int kMax = 227 * 1024, kStage = kStreamWarps * 16 * box_row<TYPE>();
  sp.x_stride = sp.r.nsb * 512 + 64;  // consecutive tokens half a bank cycle apart
  const long long x = 8 * kStreamStages * kStreamWarps + (long long)sp.r.m_rows * sp.x_stride;
  const long long sums = SUMS ? (long long)sp.r.nsb * 8 * 8 * NT * 4 : 0;
  const long long part = (long long)(kStreamWarps + sp.tiles_per_cta - 1) * 16 * 8 * NT * 4;
  const long long left = kMax - (x + 127) / 128 * 128 - sums - part;
  if (left < 2 * kStage) return false;
  sp.stages = (int)(left / kStage < kStreamStages ? left / kStage : kStreamStages);
  sp.off_ring = (int)((x + 127) / 128 * 128);
  sp.off_sums = sp.off_ring + sp.stages * kStage;
  sp.off_part = (int)(sp.off_sums + sums);
  bytes = (int)(sp.off_part + part);
  return true;
}

constexpr int kNotTaken = -1;  // the shape is another kernel's

template <int TYPE, int NT, bool GLU, class ITEM> int launch_stream(const RowsCall &c, cudaStream_t s) {
  StreamParams sp;
  constexpr int outs = GLU ? 8 : 16;
  static RowsOnce once;
  auto kernel = rows_stream_kernel<TYPE, NT, GLU, ITEM>;
  int sms = 0, bytes = 0;
  int st = rows_configure(once, reinterpret_cast<const void *>(kernel), 227 * 1024, sms);
  if (st) return st;
  sp.r.nsb = c.k_in / 256;
  if (sp.r.nsb < box_sbs<TYPE>() || (TYPE == kQ6_K && c.k_in % 2048 != 0)) return kNotTaken;
  sp.r.m_rows = c.m_rows;
  sp.tiles = (c.n_out + outs - 1) / outs;
  sp.tiles_per_cta = (sp.tiles + sms - 1) / sms;
  if (!stream_layout<TYPE, NT, ITEM::kSums>(sp, bytes)) return kNotTaken;
  CUtensorMap maps[2] = {};
  st = rows_params<TYPE, GLU>(c, box_row<TYPE>(), outs, sp.r, maps);
  if (st) return st;
  sp.r.per = sp.r.nsb;
  const int run = (sp.tiles_per_cta * sp.r.nsb + kStreamWarps - 1) / kStreamWarps;  // items of a warp, of a tile at most nsb
  sp.r.gain = ITEM::kSums ? 1.f : rows_gain(run < sp.r.nsb ? run : sp.r.nsb);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((sp.tiles + sp.tiles_per_cta - 1) / sp.tiles_per_cta);
  cfg.blockDim = dim3(kStreamThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, kernel, maps[0], maps[1], sp);
}

template <int TYPE, bool GLU> int launch_stream_typed(const RowsCall &c, cudaStream_t s) {
  if constexpr (GLU && (TYPE == kQ4_K || TYPE == kQ5_K))
    return c.m_rows <= 8 ? launch_stream<TYPE, 1, GLU, Sums<TYPE, 1>>(c, s) : launch_stream<TYPE, 2, GLU, Sums<TYPE, 2>>(c, s);
  else
    return c.m_rows <= 8 ? launch_stream<TYPE, 1, GLU, Rounded<TYPE, 1>>(c, s) : launch_stream<TYPE, 2, GLU, Rounded<TYPE, 2>>(c, s);
}

// kNotTaken: more than 16 rows, or activations that do not fit
template <bool GLU> int launch_rows_stream(const RowsCall &c, cudaStream_t s) {
  if (c.m_rows > 16) return kNotTaken;
  switch (c.type) {
    case kQ4_K: return launch_stream_typed<kQ4_K, GLU>(c, s);
    case kQ5_K: return launch_stream_typed<kQ5_K, GLU>(c, s);
    case kQ6_K: return launch_stream_typed<kQ6_K, GLU>(c, s);
    case kQ8_0: return launch_stream_typed<kQ8_0, GLU>(c, s);
    case kIQ4_NL: return launch_stream_typed<kIQ4_NL, GLU>(c, s);
    default: return COGNI_QMM_ERR_TYPE;
  }
}

}  // namespace
}  // namespace cogni
