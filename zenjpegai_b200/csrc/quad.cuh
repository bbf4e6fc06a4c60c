// Four neighbouring positions of planar rows: loads, stores, packed f32x2 arithmetic, and their part
// of an 8-bit tape. Vector accesses where rows are multiples of four positions on aligned bases
// (kVec: a lane's four are then all in a row or all behind its end), else one by one.
#pragma once
#include <type_traits>

#include "../../include/zjai.h"
#include "tape.cuh"

namespace zjai {

// Four neighbouring positions, as two packed pairs.
struct F4 {
  float2 a, b;
};
__device__ __forceinline__ F4 operator+(F4 x, F4 y) {
  return {__fadd2_rn(x.a, y.a), __fadd2_rn(x.b, y.b)};
}
__device__ __forceinline__ F4 operator*(F4 x, F4 y) {
  return {__fmul2_rn(x.a, y.a), __fmul2_rn(x.b, y.b)};
}
__device__ __forceinline__ F4 fma4(F4 x, F4 y, F4 z) {
  return {__ffma2_rn(x.a, y.a, z.a), __ffma2_rn(x.b, y.b, z.b)};
}
__device__ __forceinline__ F4 all(float v) {
  return {make_float2(v, v), make_float2(v, v)};
}
// one exact product and one rounding, as a subtraction (packed operands take no sign)
__device__ __forceinline__ F4 operator-(F4 x, F4 y) { return fma4(y, all(-1.f), x); }
__device__ __forceinline__ F4 make4(float4 v) {
  return {make_float2(v.x, v.y), make_float2(v.z, v.w)};
}
__device__ __forceinline__ float4 flat(F4 v) { return make_float4(v.a.x, v.a.y, v.b.x, v.b.y); }

// four halves in two words, and back
template <class T>
__device__ __forceinline__ F4 halves4(uint2 w) {
  if constexpr (std::is_same<T, __half>::value)
    return {__half22float2(reinterpret_cast<const __half2&>(w.x)),
            __half22float2(reinterpret_cast<const __half2&>(w.y))};
  else
    return {make_float2(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u)),
            make_float2(__uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u))};
}
template <class T>
__device__ __forceinline__ uint2 words2(F4 v) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 x = __float22half2_rn(v.a), y = __float22half2_rn(v.b);
    return make_uint2(reinterpret_cast<const uint32_t&>(x), reinterpret_cast<const uint32_t&>(y));
  } else {
    const __nv_bfloat162 x = __float22bfloat162_rn(v.a), y = __float22bfloat162_rn(v.b);
    return make_uint2(reinterpret_cast<const uint32_t&>(x), reinterpret_cast<const uint32_t&>(y));
  }
}

// four positions from row pointer + at, zeros behind the row's end; kVec: all in or out, aligned
template <bool kVec, class T>
__device__ __forceinline__ F4 load4(const T* row, int at, int p) {
  if constexpr (kVec) {
    if (at >= p) return all(0.f);
    if constexpr (sizeof(T) == 4) {
      return make4(__ldg(reinterpret_cast<const float4*>(row + at)));
    } else {
      return halves4<T>(__ldg(reinterpret_cast<const uint2*>(row + at)));
    }
  } else {
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = at + i < p ? to_f32(row[at + i]) : 0.f;
    return {make_float2(v[0], v[1]), make_float2(v[2], v[3])};
  }
}
// four positions at q, aligned
template <class T>
__device__ __forceinline__ void store4_in(T* q, F4 v) {
  if constexpr (sizeof(T) == 4)
    *reinterpret_cast<float4*>(q) = flat(v);
  else
    *reinterpret_cast<uint2*>(q) = words2<T>(v);
}
template <bool kVec, class T>
__device__ __forceinline__ void store4(T* row, int at, int p, F4 v) {
  if constexpr (kVec) {
    if (at < p) store4_in(row + at, v);
  } else {
    const float f[4] = {v.a.x, v.a.y, v.b.x, v.b.y};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + i < p) row[at + i] = from_f32<T>(f[i]);
  }
}
// codes of four positions as a word
template <bool kVec>
__device__ __forceinline__ uint32_t load_codes(const int8_t* row, int at, int p) {
  if constexpr (kVec) return at < p ? __ldg(reinterpret_cast<const uint32_t*>(row + at)) : 0u;
  uint32_t w = 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (at + i < p) w |= (uint32_t)(uint8_t)__ldg(row + at + i) << (8 * i);
  return w;
}
// and back to values code 2^e: a code with its sign bit flipped becomes the low bits of 2^23 + 128 +
// code, and an exact subtraction takes the offset off (before the scale: 2^23 times a large scale
// would overflow). Four times the rate of the integer conversion.
__device__ __forceinline__ F4 taped4(uint32_t codes, int e) {
  const uint32_t w = codes ^ 0x80808080u;
  const F4 off = all(-8388736.f);
  const F4 v = {make_float2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440)),
                            __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7441))),
                make_float2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7442)),
                            __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7443)))};
  return (v + off) * all(tape_scale(e));
}

__device__ __forceinline__ float sum4(F4 v) {
  const float2 t = __fadd2_rn(v.a, v.b);
  return t.x + t.y;
}

__device__ __forceinline__ float dot4(F4 x, F4 y) {
  const float2 t = __ffma2_rn(x.a, y.a, __fmul2_rn(x.b, y.b));
  return t.x + t.y;
}

// largest magnitude of four positions, as the bits of a float (a NaN is the largest)
__device__ __forceinline__ uint32_t amax4(F4 v) {
  const uint32_t k = 0x7fffffffu;
  return max(max(__float_as_uint(v.a.x) & k, __float_as_uint(v.a.y) & k),
             max(__float_as_uint(v.b.x) & k, __float_as_uint(v.b.y) & k));
}
// Codes of four positions in a group whose largest magnitude is m; whole warps call. Only the
// largest 1 / 128 of magnitudes can round to 128, and a marked group has no codes: a warp that has
// neither (one of 30 or so has) saves the clamps.
__device__ __forceinline__ uint32_t codes4(F4 v, uint32_t m) {
  const float inv = tape_inv_scale(max((int)(m >> 23) - 133, -126));
  F4 c = fma4(v, all(inv), all(12582912.f));  // see tape_code_bits
  if (__any_sync(0xffffffffu, (m & 0x7fffffu) >= 0x7f0000u || m >= 0x7f800000u)) {
    const float none = m >= 0x7f800000u ? 0.f : inv;
    const auto code = [&](float x) {
      return m >= 0x7f800000u ? 0.f : __uint_as_float(tape_code_bits(x, none));
    };
    c = {make_float2(code(v.a.x), code(v.a.y)), make_float2(code(v.b.x), code(v.b.y))};
  }
  return __byte_perm(__byte_perm(__float_as_uint(c.a.x), __float_as_uint(c.a.y), 0x0040),
                     __byte_perm(__float_as_uint(c.b.x), __float_as_uint(c.b.y), 0x0040), 0x5410);
}
// Hold four positions of a row (zeros behind its end) as part of a tape's group; the row's eight
// lanes call together, whole warps (`on`: the row exists). e0: the row's first element, ge: the
// group's place among the exponents.
template <bool kVec>
__device__ __forceinline__ void tape_store4(const zjai_tape& t, long long e0, long long ge, int at,
                                            int p, F4 v, bool on) {
  uint32_t m = amax4(v);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  const uint32_t w = codes4(v, m);
  if (!on) return;
  int8_t* codes = t.codes + e0;
  if constexpr (kVec) {
    if (at < p) *reinterpret_cast<uint32_t*>(codes + at) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + i < p) codes[at + i] = (int8_t)(w >> (8 * i) & 0xffu);
  }
  if ((threadIdx.x & 7) == 0) t.exps[ge] = (int8_t)tape_exp(m);
}
// value of positions behind the row's end set to zero
template <bool kVec>
__device__ __forceinline__ F4 clip4(F4 v, int at, int p) {
  if (kVec) return at < p ? v : all(0.f);
  return {make_float2(at < p ? v.a.x : 0.f, at + 1 < p ? v.a.y : 0.f),
          make_float2(at + 2 < p ? v.b.x : 0.f, at + 3 < p ? v.b.y : 0.f)};
}

}  // namespace zjai
