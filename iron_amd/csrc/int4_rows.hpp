// Rows of a 4-bit KV cache: a head's D keys or values at one position in
// D / 2 + 16 bytes. D / 2 bytes of codes, then four pairs (s, b) of fp16, one for
// each quarter of the row (D / 4 consecutive values): value = b + s (16 + code).
// A word of codes holds eight consecutive values, the even ones in the nibbles of
// its low half, the odd ones in those of its high half: two neighbours come out as
// a packed pair. 16 + code as fp16 is the code in bits 6 .. 9 under the bits of 16,
// so two values cost a shift, an and-or and one packed fma; with b + s code the
// conversion would cost a subtraction more.
#pragma once

#include "iron_common.hpp"

namespace iron {

typedef _Float16 i4_f16x2 __attribute__((ext_vector_type(2)));

template <int D>
constexpr int kInt4Row = D / 2 + 16;  // bytes

// (x & mask) | bits in one instruction, which takes one scalar operand only: the compiler makes two of it.
__device__ __forceinline__ unsigned i4_pick(unsigned x, unsigned bits) {
  unsigned r;
  asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "s"(0x03c003c0u), "v"(bits));
  return r;
}

// The fp16 pairs (0, 1), (2, 3), (4, 5), (6, 7) of a word of codes, each value
// rounded once: half a step of fp16, an eighth of bf16's.
__device__ __forceinline__ void int4_unpack8(unsigned codes, i4_f16x2 s, i4_f16x2 b, unsigned (&out)[4]) {
  constexpr unsigned kSixteen = 0x4c004c00u;
  const unsigned x[4] = {codes << 6, codes << 2, codes >> 2, codes >> 6};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    out[i] = __builtin_bit_cast(unsigned, __builtin_elementwise_fma(__builtin_bit_cast(i4_f16x2, i4_pick(x[i], kSixteen)), s, b));
}

// The same as sums of two fp16 numbers and b, without rounding: s has 11 bits and
// 16 + code has 5, so s is cut behind its sixth, and (16 + code) / 2 times either part
// fits fp16 (halved, the largest s does too; below 2^-13 the lower part may lose
// its last bit, 2^-25). high + low + b / 2 is half the value.
__device__ __forceinline__ void int4_split8(unsigned codes, i4_f16x2 s_high, i4_f16x2 s_low, unsigned (&high)[4], unsigned (&low)[4]) {
  constexpr unsigned kEight = 0x48004800u;
  const unsigned x[4] = {codes << 6, codes << 2, codes >> 2, codes >> 6};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const i4_f16x2 y = __builtin_bit_cast(i4_f16x2, i4_pick(x[i], kEight));
    high[i] = __builtin_bit_cast(unsigned, y * s_high);
    low[i] = __builtin_bit_cast(unsigned, y * s_low);
  }
}

// s and b of a pair, twice each.
__device__ __forceinline__ i4_f16x2 int4_scale(unsigned pair) {
  const _Float16 s = __builtin_bit_cast(_Float16, static_cast<uint16_t>(pair & 0xffffu));
  return i4_f16x2{s, s};
}
__device__ __forceinline__ i4_f16x2 int4_base(unsigned pair) {
  const _Float16 b = __builtin_bit_cast(_Float16, static_cast<uint16_t>(pair >> 16));
  return i4_f16x2{b, b};
}

__device__ __forceinline__ int int4_code(unsigned word, int i) { return word >> (4 * (i >> 1) + 16 * (i & 1)) & 15; }

// Value code of a pair in fp32 (the product is exact).
__device__ __forceinline__ float int4_dequant(unsigned pair, int code) {
  return fmaf(static_cast<float>(int4_scale(pair)[0]), static_cast<float>(16 + code), static_cast<float>(int4_base(pair)[0]));
}

// Value d of the row at `row`.
template <int D>
__device__ __forceinline__ float int4_value(const void* row, int d) {
  const unsigned* words = static_cast<const unsigned*>(row);
  return int4_dequant(words[D / 8 + d / (D / 4)], int4_code(words[d >> 3], d & 7));
}

// Half the largest range of a quarter whose b stays in fp16: b >= -(1 + 32 / 15) times it.
constexpr float kInt4Most = 20480.f;

// The smallest, the largest of three numbers; the compiler's own makes quiet NaN of its operands first, at an instruction each.
__device__ __forceinline__ float i4_min3(float a, float b, float c) {
  float r;
  asm("v_min3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
__device__ __forceinline__ float i4_max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// A lane's neighbour's number (quad_perm [1,0,3,2]), and that of the other pair of four ([2,3,0,1]).
__device__ __forceinline__ float i4_beside(float x) { return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0xb1, 0xf, 0xf, false)); }
__device__ __forceinline__ float i4_across(float x) { return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x4e, 0xf, 0xf, false)); }

// Quantizes a quarter of 8 G values (of a 16-bit type), eight in each of G lanes: the
// codes of the lane's eight in a word, and the pair. s is the range by 15 and b the
// least value less 16 s, each rounded to fp16; a code is the nearest for those, of two
// equally near ones the upper: how many of the borders b + (k + 16.5) s, k = 0 .. 14, lie
// at or below x. The product is off by less than half a code (by 2^-8: a range of 16-bit
// values is 2^-11 of them or more), and one comparison with the border next to it, which
// fp32 holds exactly, decides. Values are cut to +-20480; a NaN makes the quarter NaN.
// All lanes of a quarter are active. 13 instructions a value.
template <int G>
__device__ __forceinline__ unsigned int4_quantize(float (&x)[8], unsigned& codes) {
  bool nan = false;
#pragma unroll
  for (int i = 0; i < 8; i += 2) nan |= __builtin_isunordered(x[i], x[i + 1]);
  float lo = i4_min3(x[0], x[1], x[2]), hi = i4_max3(x[0], x[1], x[2]);
  lo = i4_min3(i4_min3(lo, x[3], x[4]), i4_min3(x[5], x[6], x[7]), lo);
  hi = i4_max3(i4_max3(hi, x[3], x[4]), i4_max3(x[5], x[6], x[7]), hi);
  lo = i4_min3(lo, i4_beside(lo), lo);
  hi = i4_max3(hi, i4_beside(hi), hi);
  if constexpr (G == 4) {
    lo = i4_min3(lo, i4_across(lo), lo);
    hi = i4_max3(hi, i4_across(hi), hi);
  }
  // lanes of the wave with a NaN; those of this lane's quarter
  const unsigned long long odd = __ballot(nan);
  nan = (threadIdx.x & 32 ? static_cast<unsigned>(odd >> 32) : static_cast<unsigned>(odd)) >> (threadIdx.x & 31 & ~(G - 1)) & ((1u << G) - 1);
  if (__ballot(!(lo >= -kInt4Most && hi <= kInt4Most))) {
    auto cut = [](float y) { return fminf(fmaxf(y, -kInt4Most), kInt4Most); };
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = cut(x[i]);
    lo = cut(lo);
    hi = cut(hi);
  }
  const _Float16 sh = static_cast<_Float16>((hi - lo) / 15.f);
  const float s = static_cast<float>(sh);
  const _Float16 bh = static_cast<_Float16>((lo - 16.f * s) + 0.f);  // of zeros of both signs, +0
  const float b = static_cast<float>(bh), inv = s > 0.f ? 1.f / s : 0.f, first = -16.f - b * inv;
  const float step = s > 0.f ? s : INFINITY;  // without a range every border is out of reach
  codes = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float k = __builtin_amdgcn_fmed3f(floorf(fmaf(x[i], inv, first)), 0.f, 14.f);  // the border above code k
    const int code = static_cast<int>(k) + (x[i] >= fmaf(k + 16.5f, step, b) ? 1 : 0);
    codes |= static_cast<unsigned>(code) << (4 * (i >> 1) + 16 * (i & 1));
  }
  if (nan) codes = 0;
  return nan ? 0x7e000000u : __builtin_bit_cast(uint16_t, sh) | static_cast<unsigned>(__builtin_bit_cast(uint16_t, bh)) << 16;
}

}  // namespace iron
