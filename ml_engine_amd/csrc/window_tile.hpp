// Tiles of 64 rows for the attention kernels, and products of them on the matrix
// cores with fp32 accuracy.
//
// Products.  An fp32 value x, scaled by a power of two so that its tile's largest is in
// [2^14, 2^15), is held as two fp16 parts, hi = fp16(x) and lo = fp16(x - hi): 22 bits of
// every value down to 2^-18 of the largest, and 2^-40 of the largest below (the matrix
// cores keep fp16's subnormals).  A product is hi hi + hi lo + lo hi, three
// v_mfma_f32_32x32x16_f16, where three bf16 parts (split_core.hpp) take six.
// What is not finite stays so in hi, and shows in the sums.
//
// Layout.  A tile lies in LDS row by row, 128 or 256 bytes of fp16 to a row and plane,
// the lo plane after the hi plane.  The 16-byte units of a row are permuted by an
// exclusive or with bits of the row, in reverse order, so that both ways of reading
// spread over all banks:
//   frag_row: rows as the index that a product keeps (16 bytes of 32 rows);
//   frag_col: rows as the index that it sums over: ds_read_b64_tr_b16 hands 16 lanes 4
//     consecutive rows each of their 16 columns.
// One copy serves both, so a tile of K is split once for K Q^T and for K^T dS^T.
//
// The sum's order.  A block of scores leaves the accumulators with 16 rows to a lane,
// 8 (r / 4) + 4 (lane / 32) + r % 4 for r = 0 .. 15; the next product sums over them in
// that order, eight r at a time, so probabilities go from the accumulators to the
// operand without leaving the lane (frag_col reads the same order).
#pragma once
#include "window_attention.hpp"

namespace wattn {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int TR = 64;      // rows of a tile
constexpr int kTop = 14;    // exponent of a tile's largest value
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// DP: columns, the head's dimension rounded up to 64, 96 or 128.
template <int DP>
struct Tile {
  static constexpr int UNITS = DP / 8, PITCH = DP <= 64 ? 128 : 256, PLANE = TR * PITCH, BYTES = 2 * PLANE;
  static constexpr int KS = DP / 16, DB = DP / 32;  // steps over the columns; blocks of 32 columns
};

template <int DP>
__device__ __forceinline__ int swizzle(int row) {
  return DP <= 64 ? ((row & 2) << 1) | ((row & 4) >> 1) | ((row & 8) >> 3)
                  : ((row & 1) << 3) | ((row & 2) << 1) | ((row & 4) >> 1) | ((row & 8) >> 3);
}

struct Frag {
  f16x8 hi, lo;
};

__device__ __forceinline__ f32x16 mma(const f16x8& a, const f16x8& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ void mma3(const Frag& a, const Frag& b, f32x16& c) {
  c = mma(a.lo, b.hi, c);
  c = mma(a.hi, b.lo, c);
  c = mma(a.hi, b.hi, c);
}

__device__ __forceinline__ Frag split8(const float (&x)[8]) {
  Frag f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    f.hi[j] = (_Float16)x[j];
    f.lo[j] = (_Float16)(x[j] - (float)f.hi[j]);
  }
  return f;
}

// Eight of a block's 16 rows as an operand.
__device__ __forceinline__ Frag split_rows(const f32x16& x, int s) {
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = x[8 * s + j];
  return split8(v);
}

// A lane's places in a tile.
template <int DP>
struct Places {
  int row[Tile<DP>::KS];  // of frag_row: row lane % 32, columns 16 s + 8 (lane / 32) ..
  int col[Tile<DP>::DB];  // of frag_col
  __device__ __forceinline__ Places(int lane) {
    const int c = lane & 31, h = lane >> 5, i = lane & 15, g = (lane >> 4) & 1;
#pragma unroll
    for (int s = 0; s < Tile<DP>::KS; ++s) row[s] = c * Tile<DP>::PITCH + (((2 * s + h) ^ swizzle<DP>(c)) << 4);
    const int r = 4 * h + (i >> 2);
#pragma unroll
    for (int d = 0; d < Tile<DP>::DB; ++d)
      col[d] = r * Tile<DP>::PITCH + (((4 * d + 2 * g + ((i & 3) >> 1)) ^ swizzle<DP>(r)) << 4) + 8 * (i & 1);
  }
};

// Rows 32 b + lane % 32, columns of step s.
template <int DP>
__device__ __forceinline__ Frag frag_row(const char* t, const Places<DP>& p, int b, int s) {
  const char* at = t + p.row[s] + 32 * b * Tile<DP>::PITCH;
  Frag f;
  f.hi = *reinterpret_cast<const f16x8*>(at);
  f.lo = *reinterpret_cast<const f16x8*>(at + Tile<DP>::PLANE);
  return f;
}

__device__ __forceinline__ s16x4 read_tr(const char* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p));
}

// Columns 32 d + lane % 32, the 16 rows of step s in the accumulators' order.
template <int DP>
__device__ __forceinline__ Frag frag_col(const char* t, const Places<DP>& p, int s, int d) {
  const char* a = t + p.col[d] + 16 * s * Tile<DP>::PITCH;
  const char* b = t + (p.col[d] ^ 16) + (16 * s + 8) * Tile<DP>::PITCH;  // 8 rows on: the swizzle's last bit
  Frag f;
  const f16x4 h0 = __builtin_bit_cast(f16x4, read_tr(a)), h1 = __builtin_bit_cast(f16x4, read_tr(b));
  const f16x4 l0 = __builtin_bit_cast(f16x4, read_tr(a + Tile<DP>::PLANE)),
              l1 = __builtin_bit_cast(f16x4, read_tr(b + Tile<DP>::PLANE));
  f.hi = __builtin_shufflevector(h0, h1, 0, 1, 2, 3, 4, 5, 6, 7);
  f.lo = __builtin_shufflevector(l0, l1, 0, 1, 2, 3, 4, 5, 6, 7);
  return f;
}

// Eight columns from 8 u of a row, zeros past `dim` and of a row that is not there.
__device__ __forceinline__ void load8(const float* __restrict__ row, int u, int dim, bool there, float (&x)[8]) {
  const int n = there ? dim - 8 * u : 0;
  const float* p = row + 8 * u;
  if (n >= 8) {
    const f32x4u a = reinterpret_cast<const f32x4u*>(p)[0], b = reinterpret_cast<const f32x4u*>(p)[1];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = a[j];
      x[4 + j] = b[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = 0.f;
    if (n > 0) {
#pragma unroll
      for (int j = 0; j < 7; ++j)
        if (j < n) x[j] = p[j];
    }
  }
}

__device__ __forceinline__ float top8(const float (&x)[8]) {
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(x[j]));
  return m;
}

// The largest over 16 lanes, in each of them.
__device__ __forceinline__ float row16_max(float v) {
  auto dpp = [](float x, auto ctrl) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xF, 0xF, true));
  };
  v = fmaxf(v, dpp(v, std::integral_constant<int, 0xB1>{}));   // lanes 1 0 3 2
  v = fmaxf(v, dpp(v, std::integral_constant<int, 0x4E>{}));   // lanes 2 3 0 1
  v = fmaxf(v, dpp(v, std::integral_constant<int, 0x124>{}));  // four lanes round
  v = fmaxf(v, dpp(v, std::integral_constant<int, 0x128>{}));  // eight
  return v;
}
__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, 64); }

// floor(log2) of a magnitude (0 and subnormals as 2^-127, infinity as the largest number).
__device__ __forceinline__ int exponent(float m) {
  const int e = (int)(__builtin_bit_cast(unsigned, m) >> 23);
  return min(e, 254) - 127;
}

// A thread's share of a tile of NT threads: N chunks of eight columns.
template <int DP, int NT>
struct Share {
  static constexpr int ALL = TR * Tile<DP>::UNITS, N = (ALL + NT - 1) / NT;
  float x[N][8];
  static __device__ __forceinline__ int unit(int c) { return c * NT + (int)threadIdx.x; }
  static constexpr bool whole = ALL % NT == 0;
  // Rows r0 .. r0 + 63 of a tensor from `base`, those in [r0, end).
  __device__ __forceinline__ void load(const float* __restrict__ base, int64_t ld, int r0, int end, int dim) {
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const int id = unit(c), row = id / Tile<DP>::UNITS, u = id % Tile<DP>::UNITS;
      const bool there = (whole || id < ALL) && r0 + row < end;
      load8(base + (int64_t)(there ? r0 + row : 0) * ld, u, dim, there, x[c]);
    }
  }
  __device__ __forceinline__ float top() const {
    float m = 0.f;
#pragma unroll
    for (int c = 0; c < N; ++c) m = fmaxf(m, top8(x[c]));
    return m;
  }
  // Split at 2^shift into a tile; put_rows: at 2^(kTop - ex) of each row.
  __device__ __forceinline__ void put(char* t, int shift) const {
    put_with(t, [=](int) { return shift; });
  }
  __device__ __forceinline__ void put_rows(char* t, const int* ex) const {
    put_with(t, [=](int row) { return kTop - ex[row]; });
  }
  template <class F>
  __device__ __forceinline__ void put_with(char* t, F shift_of) const {
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const int id = unit(c), row = id / Tile<DP>::UNITS, u = id % Tile<DP>::UNITS;
      if (!whole && id >= ALL) break;
      const int shift = shift_of(row);
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __builtin_amdgcn_ldexpf(x[c][j], shift);
      const Frag f = split8(v);
      char* at = t + row * Tile<DP>::PITCH + ((u ^ swizzle<DP>(row)) << 4);
      *reinterpret_cast<f16x8*>(at) = f.hi;
      *reinterpret_cast<f16x8*>(at + Tile<DP>::PLANE) = f.lo;
    }
  }
};

// The largest magnitudes of coming tiles: slot t of four takes tile t's, a wave at a time.
struct Tops {
  unsigned v[4][2];
};
__device__ __forceinline__ void add_top(unsigned* slot, float m) {
  m = row16_max(m);
  if ((threadIdx.x & 15) == 0) atomicMax(slot, __builtin_bit_cast(unsigned, m));
}

// The tiles that rows at positions first .. last (0 <= first <= last) see: sinks before the window, then the window.
struct Tiles {
  int before, low, count;
  __device__ __forceinline__ Tiles(const Args& a, int first, int last) {
    low = max(first - a.window + 1, 0) / TR;
    before = min((a.sinks + TR - 1) / TR, low);
    count = before + last / TR + 1 - low;
  }
  __device__ __forceinline__ int row(int t) const { return TR * (t < before ? t : low + t - before); }
};

}  // namespace wattn
