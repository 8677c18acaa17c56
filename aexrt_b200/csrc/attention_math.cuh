// Arithmetic that the attention kernels share: 2^x, packing to 16 bits, and non-finite values of V.
#pragma once
#include "attention_common.cuh"

namespace aexrt {

// A row's maximum may run ahead of the reference that its probabilities are taken against by 2^8, so that most tiles need
// no rescaling of the accumulators.
constexpr float kLazyLog2 = 8.f;

// P is held in the tensors' 16-bit type, as the tensor cores take it; the normaliser is summed from the unrounded values.
// In fp16 it is taken 2^7 times larger (up to 2^15 with the above): its steps end at 2^-24, and many keys of 2^-25 of the
// largest probability, which round to 0 there, may count together.  bf16 has fp32's range.
template <typename T>
constexpr float kProbLog2 = __is_same(T, __half) ? 7.f : 0.f;
template <typename T>
constexpr float kProbUnit = __is_same(T, __half) ? 1.f / 128 : 1.f;

// s * c - m * c as one multiply-add carries the rounding of m * c, half a step of its own magnitude: 2^-12 here.
// Beyond, s - m is taken first (exact for the scores that count), so that scores as large as fp32 holds still
// give finite probabilities.
constexpr float kLargeLog2 = 4096.f;

// Keys that one accumulator of a tensor-core product takes.  Such a sum cuts every product to 2^-25 of what is summed
// so far before it adds it (measured: ones are lost from 2^26 on, products below 2^-10 beside 65504), so n keys can
// lose n * 2^-25 of sum |p v|: 2^-11 of it here, half a step of fp16.  Then the sums go to fp32 ones, which round.
constexpr int kSumKeys = 16384;

// 2^x on the special-function unit (subnormal results flush to 0).
__device__ __forceinline__ float exp2_sfu(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Sums that were taken against the maximum `from` count this much against `to`, which is not below it (equal ones,
// infinite ones too: 1).
__device__ __forceinline__ float moved(float from, float to, float sl2) { return from == to ? 1.f : exp2_sfu((from - to) * sl2); }

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
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

// An output as its type holds it.  It is an average of finite values, or infinite because one of them is: the
// probabilities' rounding may take an fp16 average of up to 65504 past 65520, which would round to infinity.
template <typename T>
__device__ __forceinline__ float in_range(float o) {
  if constexpr (__is_same(T, __half)) return fabsf(o) < 66000.f ? fminf(fmaxf(o, -65504.f), 65504.f) : o;
  return o;
}
template <typename T>
__device__ __forceinline__ uint32_t pack_out(float lo, float hi) { return pack16<T>(in_range<T>(lo), in_range<T>(hi)); }

// A word of two 16-bit values with an infinity or NaN among them: the exponent field of all ones
// carries into the sign bit.
template <typename T>
__device__ __forceinline__ uint32_t non_finite_bits(uint32_t w) {
  return __is_same(T, __nv_bfloat16) ? ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u
                                     : ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
}

// Notes a non-finite value (bits h) of column `col` of key `key`: fix[col] has the first key with +inf or
// NaN, fix[128 + col] the first with -inf or NaN.
template <typename T>
__device__ __forceinline__ void note_non_finite(uint32_t h, int key, int col, int* fix) {
  const bool nan = (h & (__is_same(T, __nv_bfloat16) ? 0x7fu : 0x3ffu)) != 0, down = (h >> 15) & 1;
  if (nan || !down) atomicMin(fix + col, key);
  if (nan || down) atomicMin(fix + 128 + col, key);
}

// Takes the non-finite values out of 16 bytes of a V tile (values of columns d0 .. d0 + 7 of key
// `key`): zeros in their place, and a note of them.
template <typename T>
__device__ __forceinline__ uint4 take_non_finite(uint4 x, int key, int d0, int* fix) {
  uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = non_finite_bits<T>(w[i]);
    if (b & 0x8000u) {
      note_non_finite<T>(w[i] & 0xffffu, key, d0 + 2 * i, fix);
      w[i] &= 0xffff0000u;
    }
    if (b & 0x80000000u) {
      note_non_finite<T>(w[i] >> 16, key, d0 + 2 * i + 1, fix);
      w[i] &= 0xffffu;
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// A row's output o in a column, with the values added that were taken out and that it sees (keys 0 .. seen - 1).  Sums:
// what the other keys gave may be infinite or NaN itself.
__device__ __forceinline__ float put_back(float o, const int* fix, int col, int seen) {
  const bool up = fix[col] < seen, down = fix[128 + col] < seen;
  return o + (up ? (down ? __int_as_float(0x7fffffff) : INFINITY) : (down ? -INFINITY : 0.f));
}
constexpr int kFixInts = 2 * 128;

}  // namespace aexrt
