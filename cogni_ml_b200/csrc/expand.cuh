// Pieces of the expansion of quants to bf16, shared by the products that round their weights
// (gemm_prefill.cuh, gemm_rows.cuh).
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

namespace cogni {
namespace {

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t *>(&v);
}
// Packed pairs of f32 (sm_100 has two-wide f32 add / mul / fma: same IEEE results per element, half
// the instructions in the expansion, which is what the dequant warps are bound by).
__device__ __forceinline__ uint64_t f2_pack(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint32_t f2_to_bf16x2(uint64_t v) {
  float a, b;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
  return pack_bf16(a, b);
}
// bytes (i, i+1) of v as the floats 2^23 + b, packed
__device__ __forceinline__ uint64_t bytes2_biased(uint32_t v, int i) {
  return f2_pack(__uint_as_float(__byte_perm(v, 0x4B000000u, 0x7650 + i)),
                 __uint_as_float(__byte_perm(v, 0x4B000000u, 0x7650 + i + 1)));
}
// Four IQ4_NL nibbles (bits 0-15 of hq) as int8 (dequant.cr:11-16): three byte permutes, the table's halves by
// the low three bits, then a choice by the fourth.
__device__ __forceinline__ uint32_t iq4nl_lookup4(uint32_t hq) {
  const uint32_t s7 = hq & 0x7777u;
  const uint32_t lo = __byte_perm(0xBFAD9881u, 0xF6EADDCFu, s7);
  const uint32_t hi = __byte_perm(0x26190D01u, 0x71594535u, s7);
  return __byte_perm(lo, hi, 0x3210u | ((hq >> 1) & 0x4444u));
}

}  // namespace
}  // namespace cogni
