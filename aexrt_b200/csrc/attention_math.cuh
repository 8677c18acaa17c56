// Arithmetic that the attention kernels share: 2^x, packing to 16 bits, and non-finite values of V.
#pragma once
#include "attention_common.cuh"

namespace aexrt {

// A row's maximum may run ahead of the reference that its probabilities are taken against by 2^8: they
// stay below 2^8, far inside fp16, and most tiles need no rescaling of the accumulators.
constexpr float kLazyLog2 = 8.f;

// 2^x on the special-function unit (subnormal results flush to 0).
__device__ __forceinline__ float exp2_sfu(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack16<__half>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <>
__device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// A word of two 16-bit values with an infinity or NaN among them: the exponent field of all ones
// carries into the sign bit.
template <typename T>
__device__ __forceinline__ uint32_t non_finite_bits(uint32_t w) {
  return __is_same(T, __nv_bfloat16) ? ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u
                                     : ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
}

// Kind of a non-finite 16-bit value: 0 +inf, 1 -inf, 2 NaN.
template <typename T>
__device__ __forceinline__ int non_finite_kind(uint32_t h) {
  const uint32_t mantissa = __is_same(T, __nv_bfloat16) ? h & 0x7fu : h & 0x3ffu;
  return mantissa ? 2 : static_cast<int>(h >> 15) & 1;
}

// Takes the non-finite values out of 16 bytes of a V tile (values of columns d0 .. d0 + 7 of key
// `key`): zeros in their place, and the first such key of each column and kind in fix.
template <typename T>
__device__ __noinline__ uint4 take_non_finite(uint4 x, int key, int d0, int* fix) {
  uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = non_finite_bits<T>(w[i]);
    if (b & 0x8000u) {
      atomicMin(fix + non_finite_kind<T>(w[i] & 0xffffu) * 128 + d0 + 2 * i, key);
      w[i] &= 0xffff0000u;
    }
    if (b & 0x80000000u) {
      atomicMin(fix + non_finite_kind<T>(w[i] >> 16) * 128 + d0 + 2 * i + 1, key);
      w[i] &= 0xffffu;
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// What a row that sees keys 0 .. seen - 1 gets in a column from values that were taken out.
__device__ __forceinline__ float put_back(float o, const int* fix, int col, int seen) {
  const bool up = fix[col] < seen, down = fix[128 + col] < seen, nan = fix[256 + col] < seen;
  if (nan || (up && down)) return __int_as_float(0x7fffffff);
  return up ? INFINITY : (down ? -INFINITY : o);
}

}  // namespace aexrt
