// Warp-level matrix products and fragment helpers shared by the decoding kernels.  These kernels are bound by reading 8-bit keys and values
// or expert weights, which bulk copies bring to a ring of each warp in shared memory.  From there a lane takes its fragments to registers,
// where codes become fp16, and eight query rows or tokens ride on every weight: the tensor pipe is 9 to 18 % busy.  A tcgen05 tile would need
// the converted operand back in shared memory and 128 rows of it before the first product.
//
// m16n8k16, lane = 4 g + c:  A: a0 (row g, k 2c..), a1 (row g + 8, k 2c..), a2 (row g, k 2c + 8..), a3 (row g + 8, k 2c + 8..)
//                            B: b0 (k 2c.., column g), b1 (k 2c + 8.., column g);  C: c0 c1 (row g, columns 2c 2c+1), c2 c3 (row g + 8)
// The order of k is free as long as A and B agree, which is what lets a lane take 8 or 16 adjacent elements per load.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace mts {

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same with the sum begun at zero.
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f), "f"(0.f), "f"(0.f), "f"(0.f));
}
// Transpose of an 8 x 8 matrix of 16-bit values held as fragments (row = lane / 4, columns 2c, 2c + 1).
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_bf162(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Four excess-128 codes to two pairs of fp16 integers: a byte below the byte 0x64 reads 1024 + the byte, and the subtraction of 1152 is
// exact.  (Leaving it out and starting the sums from -1152 times the sum of the other factor saves half of the instructions but
// costs precision where sums cancel: 8e-4 of an output over 131k tokens, 1e-3 in a logit of some hundreds.)
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t l = __byte_perm(w, 0x64646464u, 0x4140), h = __byte_perm(w, 0x64646464u, 0x4342);
  const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
  const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&l), bias), b = __hsub2(*reinterpret_cast<const __half2*>(&h), bias);
  lo = *reinterpret_cast<const uint32_t*>(&a);
  hi = *reinterpret_cast<const uint32_t*>(&b);
}

}  // namespace mts
