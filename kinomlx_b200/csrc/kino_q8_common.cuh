// Shared pieces of the 8-bit serving kernels: the two code formats, their scales, and the
// conversions between codes and floating values.
//
// A group of values (a token's row, a weight's output channel, the tokens of one cache block and
// head) is held as codes times one fp32 scale, amax / top (top 127 for int8, 448 for e4m3):
//   code = x * top / amax, rounded to fp32 and then to the code grid, to nearest even both times.
// The quotient's first rounding is exact to 2^-48 (see Q8Factor), so a value that lies on the
// border of two codes, which bf16 values often do (amax / 2 in int8), goes to the even one and
// not where the rounding of a reciprocal happens to push it. A group whose scale would fall below
// 2^-126 (1 / scale would overflow) is a group of zeros with scale 0; one that holds an infinity
// or a NaN gets the scale NaN and codes 0, so that it reads back as NaN wherever it is used and no
// code is ever a NaN pattern.
#pragma once
#include <cuda_fp8.h>

#include "kino_common.cuh"

namespace kino {

constexpr int Q8_INT8 = 0;
constexpr int Q8_E4M3 = 1;
constexpr float Q8_LEAST_SCALE = 1.1754943508222875e-38f;  // 2^-126

template <int FMT>
__device__ __forceinline__ float q8_top() {
  return FMT == Q8_INT8 ? 127.0f : 448.0f;
}

// Records an error for kino_device_status; the first one stays.
__device__ __forceinline__ void q8_flag(int code) { atomicCAS(&g_device_error, 0, code); }

// Scale of a group from the bit pattern of its largest magnitude. Patterns of non-negative floats
// order like the floats, with NaN above infinity, so an integer maximum keeps what is not finite.
template <int FMT>
__device__ __forceinline__ float q8_scale(uint32_t amax_bits) {
  if (amax_bits >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
  const float s = __fdiv_rn(__uint_as_float(amax_bits), q8_top<FMT>());
  return s < Q8_LEAST_SCALE ? 0.0f : s;
}

// A factor of about 48 bits: x * (hi + lo) as fma(x, hi, x * lo) has one rounding that counts.
struct Q8Factor {
  float hi, lo;
  __device__ __forceinline__ float times(float x) const { return fmaf(x, hi, x * lo); }
};

// a / b (b > 0 and the quotient in range).
__device__ __forceinline__ Q8Factor q8_quotient(float a, float b) {
  Q8Factor f;
  f.hi = __fdiv_rn(a, b);
  f.lo = __fdiv_rn(fmaf(-f.hi, b, a), b);
  return f;
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// Four codes, lowest byte first, of quotients within the code range (a group with scale 0 or NaN
// gets zeros from the caller). int8: 1.5 * 2^23 + x has the integer nearest to x, ties to even, in
// its low bits, two's complement (a conversion to integer runs at a quarter of an addition's rate).
template <int FMT>
__device__ __forceinline__ uint32_t q8_encode4(float a, float b, float c, float d) {
  if constexpr (FMT == Q8_INT8) {
    constexpr float kShift = 12582912.0f;
    const uint32_t ia = __float_as_uint(a + kShift), ib = __float_as_uint(b + kShift);
    const uint32_t ic = __float_as_uint(c + kShift), id = __float_as_uint(d + kShift);
    return __byte_perm(__byte_perm(ia, ib, 0x0040), __byte_perm(ic, id, 0x0040), 0x5410);
  } else {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  }
}

// Two codes as exact bf16 values, from a register that holds them in the byte positions given
// below; the other two bytes may hold anything.
//
// int8, codes in the low byte of each half: with u = the low 7 bits, 0x4300 | u is the bf16
// 128 + u, and 0x4300 | sign bit is 128 or 256 (the sign bit is the exponent's lowest), so their
// difference is u - 128 * sign, the code.
// e4m3, codes in the high byte of each half: sign, exponent and mantissa moved to their bf16
// places are the value times 2^(7 - 127), subnormals included; times 2^120 restores it. (The NaN
// pattern, which no kernel here writes, reads as 480.)
__device__ __forceinline__ uint32_t q8_int8_pair(uint32_t spread) {
  const uint32_t lo = (spread & 0x007F007Fu) | 0x43004300u;
  const uint32_t hi = (spread & 0x00800080u) | 0x43004300u;
  uint32_t r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ uint32_t q8_e4m3_pair(uint32_t spread) {
  const uint32_t t = ((spread >> 4) & 0x07F007F0u) | (spread & 0x80008000u);
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(t), "r"(0x7B807B80u));  // 2^120
  return r;
}

// Bytes i and j (0..3 of a, 4..7 of b) as a bf16 pair (i low).
template <int FMT>
__device__ __forceinline__ uint32_t q8_pair(uint32_t a, uint32_t b, int i, int j) {
  if constexpr (FMT == Q8_INT8) {
    return q8_int8_pair(__byte_perm(a, b, i | (j << 8)));
  } else {
    return q8_e4m3_pair(__byte_perm(a, b, (i << 4) | (j << 12)));
  }
}

// The same as exact f16 pairs. int8: 0x64 in front of code + 128 is the f16 1024 + code + 128.
// e4m3: the value times 2^(7 - 15), subnormals included; q8_f16_unit restores it.
template <int FMT>
__device__ __forceinline__ uint32_t q8_f16_bias(uint32_t w) {  // once for four codes
  return FMT == Q8_INT8 ? w ^ 0x80808080u : w;
}
template <int FMT>
__device__ __forceinline__ uint32_t q8_f16_of(uint32_t spread) {
  uint32_t r;
  if constexpr (FMT == Q8_INT8) {
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(spread), "r"(0x64806480u));  // 1152
  } else {
    r = ((spread >> 1) & 0x3F803F80u) | (spread & 0x80008000u);
  }
  return r;
}
// Bytes 2 h, 2 h + 1 of a biased word.
template <int FMT>
__device__ __forceinline__ uint32_t q8_f16_pair(uint32_t w, int h) {
  if constexpr (FMT == Q8_INT8)
    return q8_f16_of<FMT>(__byte_perm(w, 0x64646464u, h ? 0x4342 : 0x4140));
  else
    return q8_f16_of<FMT>(__byte_perm(w, 0u, h ? 0x3424 : 0x1404));
}
template <int FMT>
__device__ __forceinline__ constexpr float q8_f16_unit() {
  return FMT == Q8_INT8 ? 1.0f : 256.0f;
}

// Four consecutive codes as fp32 values.
template <int FMT>
__device__ __forceinline__ void q8_decode4(uint32_t w, float (&f)[4]) {
  const float2 lo = unpack_bf16x2(q8_pair<FMT>(w, 0u, 0, 1));
  const float2 hi = unpack_bf16x2(q8_pair<FMT>(w, 0u, 2, 3));
  f[0] = lo.x;
  f[1] = lo.y;
  f[2] = hi.x;
  f[3] = hi.y;
}

// Where sequence b's rows are: given starts, or the same number for each.
struct Q8Rows {
  const int32_t* starts;  // [batch + 1] or null
  int each;
  int64_t rows;
  __device__ __forceinline__ void of(int b, int64_t& first, int& count) const {
    if (starts != nullptr) {
      const int s0 = starts[b], s1 = starts[b + 1];
      first = s0;
      count = s1 - s0;
      if (s0 < 0 || s1 < s0 || s1 > rows) {  // not the rows of this call: nothing to do
        count = 0;
        q8_flag(1);
      }
    } else {
      first = static_cast<int64_t>(b) * each;
      count = each;
    }
  }
};

}  // namespace kino
