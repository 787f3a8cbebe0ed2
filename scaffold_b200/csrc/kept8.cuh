// The 8-bit copy of an activation. 16 consecutive elements of the tensor's memory share a step 2^e, the smallest one
// (e >= -126) with max |x| < 126.5 * 2^e; each is kept as q = rint(x / 2^e), so |q| <= 126 and one whole number is left
// on either side (GroupNorm uses it to keep a value on its side of the ReLU). A power of two makes every operation on
// the way in and out exact but that one rounding: the copy does not depend on the order or the kind of arithmetic.
// Error: half a step, which is at most max|x| / 126 of the block (2^-7 * max|x| on average over the mantissa); 2^-127 where
// e is held at -126 (max|x| below 63.25 * 2^-126, a block below 2^-127 comes back as zeros); less than a step in the
// blocks of the last line.
//
// Memory: int8 q[blocks][16], then one byte e + 127 per block (1..249; 255: the block held an infinity or a NaN and is
// restored as NaN, its q are zeros, so that 0 * 2^(255-127) = 0 * inf is the NaN). The last block is padded with zeros.
// Blocks whose 64 * 2^e is beyond the type's largest number keep |q| <= 63: a restored value is finite when x was.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace sb {

constexpr int KEPT_BLOCK = 16;
constexpr float KEPT_MAGIC = 12582912.f;  // 1.5 * 2^23: x + KEPT_MAGIC rounds x to a whole number, ties to even
constexpr uint32_t KEPT_TOP_BF16 = 249;   // exponent bytes from which 64 steps are beyond the type (bf16 and fp32; fp16)
constexpr uint32_t KEPT_TOP_FP16 = 137;

// exponent byte of a block whose largest magnitude has the fp32 bits `amax`. 126.5 = 1.9765625 * 64, so e is the
// exponent of amax less 6, and one more from the significand 1.9765625 = 1 + 0x7D0000 / 2^23 on.
__device__ __forceinline__ uint32_t kept_exponent(uint32_t amax) {
  if (amax >= 0x7F800000u) return 255u;
  const int b = (int)((amax + 0x30000u) >> 23) - 6;
  return b < 1 ? 1u : (uint32_t)b;
}
__device__ __forceinline__ float kept_step(uint32_t b) { return __uint_as_float(b << 23); }          // 2^e; 255: inf
__device__ __forceinline__ float kept_inv(uint32_t b) { return __uint_as_float((254u - b) << 23); }  // 2^-e, b <= 249
// the low byte of each of four rounded numbers (x + KEPT_MAGIC), first one lowest
__device__ __forceinline__ uint32_t kept_pack4(float a, float b, float c, float d) {
  const uint32_t ab = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040);
  const uint32_t cd = __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040);
  return __byte_perm(ab, cd, 0x5410);
}
// rounded numbers of a block at the top of the type's range
__device__ __forceinline__ float kept_cap(float t) { return fminf(fmaxf(t, KEPT_MAGIC - 63.f), KEPT_MAGIC + 63.f); }
// four kept numbers as floats: the byte q + 128 becomes the float 2^23 + q + 128 (no conversion instruction)
__device__ __forceinline__ void kept_unpack4(uint32_t w, float (&f)[4]) {
  w ^= 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7540 + i)) - 8388736.f;
}

// the larger magnitude of each half of two pairs of bf16 (a NaN is the largest); the signs mean nothing
__device__ __forceinline__ uint32_t kept_max2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

}  // namespace sb
