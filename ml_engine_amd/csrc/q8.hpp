// Activations in 8 bits: one power-of-two step per 32 consecutive values of a
// row.  A group's step is 2^k, k the smallest exponent in [-126, 121] for which
// its largest magnitude is below 127.5 steps; a value is kept as the nearest
// whole number of steps (ties to even), q in [-127, 127], and the step as the
// byte e = k + 127.  q 2^k is off by at most half a step (magnitudes above
// 127.5 * 2^121, whose nearest multiple would be 2^128, by less than one); every
// operation is exact, so the same tensor always gives the same codes.
//
// A power of two costs up to one bit against a free scale, and buys that q 2^k
// is a bf16 number: the matrix cores read a kept activation as it is, in one
// bf16 plane.
//
// A group with an infinity or a NaN has e = 255 and the codes +1 for +inf, -1
// for -inf, 0 for the rest: the byte as a float's exponent is infinity, so its
// infinities come back as they were and all other values of the group as NaN.
#pragma once
#include "common.hpp"

namespace q8 {

constexpr int kGroup = 32;

inline int groups(int cols) { return cols / kGroup + (cols % kGroup != 0); }

// The value of a group's step.
__device__ __forceinline__ float step_of(unsigned e) { return __builtin_bit_cast(float, e << 23); }

// e of a group whose largest magnitude has the bits `top` (NaN above infinity).
__device__ __forceinline__ unsigned exponent_of(unsigned top) {
  if (top >= 0x7f800000u) return 255u;
  const unsigned e = (top >> 23) + ((top & 0x7fffffu) >= 0x7f0000u ? 1u : 0u);
  return e > 7u ? (e < 254u ? e - 6u : 248u) : 1u;
}

// The code of x under e, from inv = inverse_of(e).
__device__ __forceinline__ float inverse_of(unsigned e) { return __builtin_bit_cast(float, (254u - e) << 23); }
__device__ __forceinline__ int code_of(float x, unsigned e, float inv) {
  if (e == 255u) return __builtin_isinf(x) ? (x > 0.f ? 1 : -1) : 0;
  return (int)fminf(fmaxf(rintf(x * inv), -127.f), 127.f);
}

__device__ __forceinline__ unsigned magnitude(float x) { return __builtin_bit_cast(unsigned, x) & 0x7fffffffu; }

// The larger of a value over the four lanes 4 i .. 4 i + 3.
__device__ __forceinline__ unsigned quad_max(unsigned v) {
  const unsigned a = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false);  // lanes 1 0 3 2
  v = v > a ? v : a;
  const unsigned b = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false);  // lanes 2 3 0 1
  return v > b ? v : b;
}

// Eight values of a row, four lanes to a group: their codes in two words, and
// the group's e.  All four lanes of a group run this together (values past
// the row's end given as 0).
__device__ __forceinline__ unsigned quantize8(const float (&x)[8], uint2& code) {
  unsigned top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const unsigned m = magnitude(x[j]);
    top = top > m ? top : m;
  }
  const unsigned e = exponent_of(quad_max(top));
  const float inv = inverse_of(e);
  unsigned w[2] = {0u, 0u};
#pragma unroll
  for (int j = 0; j < 8; ++j) w[j >> 2] |= ((unsigned)code_of(x[j], e, inv) & 0xffu) << (8 * (j & 3));
  code = make_uint2(w[0], w[1]);
  return e;
}

// The values of eight codes under a step.
__device__ __forceinline__ void values8(uint2 code, float step, float (&x)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const unsigned w = j < 4 ? code.x : code.y;
    x[j] = (float)(int)(signed char)(w >> (8 * (j & 3))) * step;
  }
}

// Rows start at any address of their type: loads and stores of several values at once
// are of that alignment, which costs them little (16384 x 4093 norm, both directions and
// the codes read back: 565 us, of 4096 columns 493; element by element 1300).  What is
// left of a row, n < 8 values, is four at once where there are as many, and up to three
// single ones.
struct Left {
  bool four;
  int single;  // after the four
  __device__ __forceinline__ explicit Left(int n) : four((n & 4) != 0), single(n & 3) {}
};

// a or b, by value: a plain choice between two elements of an array becomes one
// element at an address, and the array memory.
__device__ __forceinline__ float pick(bool first, float a, float b) {
  const unsigned m = first ? ~0u : 0u;
  return __builtin_bit_cast(float, (__builtin_bit_cast(unsigned, a) & m) | (__builtin_bit_cast(unsigned, b) & ~m));
}

// n <= 8 codes at p, the rest 0.
__device__ __forceinline__ uint2 load_codes(const int8_t* __restrict__ p, int n) {
  uint2 w = make_uint2(0u, 0u);
  if (n == 8) {
    __builtin_memcpy(&w, p, 8);
    return w;
  }
  const Left l(n);
  unsigned a = 0u, b = 0u;
  if (l.four) __builtin_memcpy(&a, p, 4);
  const int8_t* s = p + (n & 4);
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (j < l.single) b |= (unsigned)(unsigned char)s[j] << (8 * j);
  return l.four ? make_uint2(a, b) : make_uint2(b, 0u);
}
__device__ __forceinline__ void store_codes(int8_t* __restrict__ p, uint2 c, int n) {
  if (n == 8) {
    __builtin_memcpy(p, &c, 8);
    return;
  }
  const Left l(n);
  if (l.four) __builtin_memcpy(p, &c.x, 4);
  const unsigned b = l.four ? c.y : c.x;
  int8_t* s = p + (n & 4);
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (j < l.single) s[j] = (int8_t)(b >> (8 * j));
}

// n <= 8 floats at p, the rest 0.
__device__ __forceinline__ void load_row8(const float* __restrict__ p, int n, float (&x)[8]) {
  if (n == 8) {
    const f32x4u a = reinterpret_cast<const f32x4u*>(p)[0], b = reinterpret_cast<const f32x4u*>(p)[1];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = a[j];
      x[4 + j] = b[j];
    }
    return;
  }
  const Left l(n);
  f32x4u a = {0.f, 0.f, 0.f, 0.f};
  float b[4] = {};
  if (l.four) a = *reinterpret_cast<const f32x4u*>(p);
  const float* s = p + (n & 4);
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (j < l.single) b[j] = s[j];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[j] = l.four ? a[j] : b[j];
    x[4 + j] = l.four ? b[j] : 0.f;
  }
}
__device__ __forceinline__ void store_row8(float* __restrict__ p, const float (&x)[8], int n) {
  if (n == 8) {
    reinterpret_cast<f32x4u*>(p)[0] = f32x4u{x[0], x[1], x[2], x[3]};
    reinterpret_cast<f32x4u*>(p)[1] = f32x4u{x[4], x[5], x[6], x[7]};
    return;
  }
  const Left l(n);
  if (l.four) *reinterpret_cast<f32x4u*>(p) = f32x4u{x[0], x[1], x[2], x[3]};
  float* s = p + (n & 4);
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (j < l.single) s[j] = pick(l.four, x[4 + j], x[j]);
}

inline int check_shape(const char* who, int rows, int cols, const void* q, int64_t ldq, const void* e, int64_t lde) {
  MLE_CHECK_ARG(rows >= 0 && cols > 0 && cols <= (1 << 30), "%s: bad shape %d x %d", who, rows, cols);
  MLE_CHECK_ARG(rows == 0 || (q && e), "%s: null pointer", who);
  MLE_CHECK_ARG(ldq >= cols && lde >= groups(cols), "%s: ldq %lld < %d or lde %lld < %d", who, (long long)ldq, cols,
                (long long)lde, groups(cols));
  return MLE_OK;
}

}  // namespace q8
