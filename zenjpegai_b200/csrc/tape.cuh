// 8-bit activation tapes: element types of the training operators, and the group format.
//
// A map's channel row (one picture, one channel, P = h w positions) is cut into groups of 32
// consecutive positions, the last one short when 32 does not divide P. A group holds one exponent
// byte e and a signed code per position; the value is code 2^e, with
//   e = clamp(floor(log2 max|x|) - 6, -126, 121), code = clamp(rint(x 2^-e), -127, 127),
// and e = 127 (codes 0) for a group with an infinity or a NaN, which then stands for NaN.
// The scale is a power of two rather than max|x| / 127 (up to one bit coarser) because scaling is
// then exact: a code has at most 7 bits, so the value is exact in bf16 and the tensor cores take
// taped activations without a rounding, and the codes do not depend on how a kernel divides.
// Saturating at 127 keeps |value| below the next power of two above max|x|: nothing overflows, in
// f16 either.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace zjai {

constexpr int kTapeGroup = 32;
constexpr int kTapeNan = 127;

__host__ __device__ inline long long tape_groups(long long p) {
  return (p + kTapeGroup - 1) / kTapeGroup;
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// Exponent of a group from the largest |x| as the bits of a float (bits of non-negative floats
// order like integers, a NaN above infinity).
__device__ __forceinline__ int tape_exp(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return kTapeNan;
  return max((int)(amax_bits >> 23) - 133, -126);
}
// 2^e of an exponent byte; e = 127 gives NaN, so a marked group's values come out as NaN
__device__ __forceinline__ float tape_scale(int e) {
  return e == kTapeNan ? __uint_as_float(0x7fc00000u)
                       : __uint_as_float((uint32_t)(max(e, -126) + 127) << 23);
}
// 2^-e of a finite group (e <= 121)
__device__ __forceinline__ float tape_inv_scale(int e) {
  return __uint_as_float((uint32_t)(127 - e) << 23);
}
// rint(x 2^-e) saturated, as a float around the constant 1.5 * 2^23 whose low byte is the code:
// the product is exact (a power of two), so the FMA's one rounding is the rint.
__device__ __forceinline__ uint32_t tape_code_bits(float x, float inv) {
  const float magic = 12582912.f;
  return __float_as_uint(fminf(fmaxf(fmaf(x, inv, magic), magic - 127.f), magic + 127.f));
}
}  // namespace zjai
