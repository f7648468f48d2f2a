// 16-bit matrix instructions of the expert kernels (gfx950), and fp32 operands as sums of bf16 ones.
#pragma once
#include "numeric.hpp"

namespace dimo {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// D = A B + C over 16 values of k.  Lane l holds A[i = l % 32][k = 8 (l / 32) ..+ 7] and B[k = 8 (l / 32) ..+ 7][j = l % 32]
// (eight 16-bit values in ascending k); register r of lane l is D[i = 8 (r / 4) + 4 (l / 32) + r % 4][j = l % 32].
__device__ __forceinline__ f32x16 mfma_32x32x16(BF16, uint4 a, uint4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma_32x32x16(F16, uint4 a, uint4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Sixteen bytes per lane from memory straight into LDS: lane l's land at S + 16 l bytes (S: the wave's, the same in every
// lane).  Done when vmcnt has counted it down, as for any load.
__device__ __forceinline__ void load_to_lds(const void *from, uint16_t *S) {
  __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void *)from,
                                   (__attribute__((address_space(3))) void *)S, 16, 0, 0);
}
// Sixteen bytes from device memory by an address that may be a constant's: said to be global, or the compiler loads it as
// "flat", which counts as an LDS access too.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint4 load_global(const void *p) {
  return __builtin_bit_cast(uint4, *(const __attribute__((address_space(1))) u32x4 *)p);
}
__device__ __forceinline__ int32_t load_global(const int32_t *p) { return *(const __attribute__((address_space(1))) int32_t *)p; }
// Eight bytes per lane from LDS, transposed among 16 lanes: lane j of them names four 16-bit values of row j / 4 (columns
// 4 (j % 4) ..+ 3 of a 4 x 16 block) and gets column j of the block, rows 0 .. 3.
typedef short s16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint2 read_transposed(const uint16_t *S) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)S));
}

// D = A B + C over 64 values of k in microscaled 4-bit form: lane l holds the block of 32 codes of A's row i = l % 32 at
// k = 32 (l / 32) ..+ 31 (sixteen bytes, ascending k, low four bits first) with its scale byte, B's column j = l % 32
// likewise.  D as above.
// BYTE: which byte of the lane's scale words counts.
typedef int i32x8 __attribute__((ext_vector_type(8)));
template <int BYTE>
__device__ __forceinline__ f32x16 mfma_mx4_32x32x64(uint4 a, uint32_t scale_a, uint4 b, uint32_t scale_b, f32x16 c) {
  const i32x8 av = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0}, bv = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, c, 4, 4, BYTE, (int)scale_a, BYTE, (int)scale_b);  // (4: e2m1)
}

// fp32 = three bf16 pieces: the top eight significant bits (cut, so that no finite value becomes infinite), what is left
// rounded to eight bits, and the rest, which eight bits hold exactly -- 24 bits in all.  Of the nine products of two
// such sums the three smallest are left out (two of up to 2^-7 2^-16 of the product and one far below: 2^-22 in all, of random
// sign), at 6 / 16 of an fp32 matrix instruction's issue time.  With the roundings of the sums a single product is off by up
// to 6.1 x 2^-24 of it (measured: 4.9 at most, 0.44 in the middle), where an fp32 multiplication is off by 1.  From 2^-110
// down the lowest piece leaves bf16's range (2^-133), and an operand is off by up to 2^-134.
// An infinite value leaves NaN (inf - inf) and so shows up as NaN in its row of outputs.
struct Split3 {
  uint16_t hi, mid, lo;
};
__device__ __forceinline__ Split3 split3(float v) {
  Split3 s;
  s.hi = (uint16_t)(__builtin_bit_cast(uint32_t, v) >> 16);
  const float r = v - BF16::load(s.hi);
  s.mid = BF16::save(r);
  s.lo = BF16::save(r - BF16::load(s.mid));
  return s;
}

}  // namespace dimo
