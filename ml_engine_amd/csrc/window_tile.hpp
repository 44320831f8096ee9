// Tiles of 64 or 32 rows for the attention kernels, and products of them on the matrix
// cores with fp32 accuracy.
//
// Products.  An fp32 value x, scaled by a power of two so that its tile's largest is in
// [2^14, 2^15), is held as two fp16 parts, hi its first 11 bits and lo the next 11 and a sign:
// off by at most 2^-23 of x, or by 2^-39 of the tile's largest where that is more (the matrix
// cores keep fp16's subnormals).  A product is hi hi + hi lo + lo hi, three
// v_mfma_f32_32x32x16_f16, where three bf16 parts (split_core.hpp) take six; lo lo is at most
// 2^-22 of it.  What is not finite stays so in hi, and shows in the sums.
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

#include <type_traits>

namespace wattn {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kTop = 14;    // exponent of a tile's largest value
constexpr float kLog2e = 1.44269504088896340736f;

// DP: columns, the head's dimension rounded up to 64, 96 or 128; R rows.
template <int DP_, int R_>
struct Tile {
  static constexpr int DP = DP_, R = R_, NB = R / 32;  // blocks of 32 rows
  static constexpr int UNITS = DP / 8, PITCH = DP <= 64 ? 128 : 256, PLANE = R * PITCH, BYTES = 2 * PLANE;
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

// x times a power of two s in two parts: hi is x s rounded to fp16, lo what hi as it is held leaves of it,
// rounded.  (A hi below 2^-14 has fewer than 11 bits; what it drops is lo's too.)  FUSED: lo from hi by
// v_fma_mix_f32, four instructions for two values, else by conversions, six.  Staged tiles take the
// first, a wave's own rows the second, and so do rows from the accumulators in the forward: with the first
// there too 2 x 16 heads of 4096 x 128 under a window of 1024 take 261 us forward instead of 253.
template <bool FUSED>
__device__ __forceinline__ Frag split8(const float (&x)[8], float s) {
  f16x2 h[4], l[4];
  float minus = -1.f;
  if (FUSED) asm("" : "+s"(minus));  // (a product that the compiler keeps)
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = x[2 * j] * s, b = x[2 * j + 1] * s;
    unsigned u = __builtin_bit_cast(unsigned, f16x2{(_Float16)a, (_Float16)b});
    asm("" : "+v"(u));  // (one conversion for both values and both uses)
    h[j] = __builtin_bit_cast(f16x2, u);
    const float a0 = (float)h[j][0], b0 = (float)h[j][1];
    l[j] = FUSED ? f16x2{(_Float16)fmaf(a0, minus, a), (_Float16)fmaf(b0, minus, b)} : f16x2{(_Float16)(a - a0), (_Float16)(b - b0)};
  }
  return Frag{__builtin_shufflevector(__builtin_shufflevector(h[0], h[1], 0, 1, 2, 3),
                                      __builtin_shufflevector(h[2], h[3], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7),
              __builtin_shufflevector(__builtin_shufflevector(l[0], l[1], 0, 1, 2, 3),
                                      __builtin_shufflevector(l[2], l[3], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7)};
}

// Eight of a block's 16 rows as an operand.
template <bool FUSED>
__device__ __forceinline__ Frag split_rows(const f32x16& x, int s, float scale) {
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = x[8 * s + j];
  return split8<FUSED>(v, scale);
}

// A lane's places in a tile: of frag_row's first step and of frag_col's first columns.  Later
// ones differ in bits that the swizzle only flips.
template <class T>
struct Places {
  int row, col;
  __device__ __forceinline__ Places(int lane) {
    const int c = lane & 31, h = lane >> 5, i = lane & 15, g = (lane >> 4) & 1, r = 4 * h + (i >> 2);
    row = c * T::PITCH + ((h ^ swizzle<T::DP>(c)) << 4);  // row c, columns 16 s + 8 h ..
    col = r * T::PITCH + (((2 * g + ((i & 3) >> 1)) ^ swizzle<T::DP>(r)) << 4) + 8 * (i & 1);
  }
};

// Row 32 b + lane % 32, columns of step s.
template <class T>
__device__ __forceinline__ Frag frag_row(const char* t, const Places<T>& p, int b, int s) {
  const char* at = t + (p.row ^ (s << 5)) + 32 * b * T::PITCH;
  Frag f;
  f.hi = *reinterpret_cast<const f16x8*>(at);
  f.lo = *reinterpret_cast<const f16x8*>(at + T::PLANE);
  return f;
}

__device__ __forceinline__ s16x4 read_tr(const char* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p));
}

// Columns 32 d + lane % 32, the 16 rows of step s in the accumulators' order.
template <class T>
__device__ __forceinline__ Frag frag_col(const char* t, const Places<T>& p, int s, int d) {
  const int c = p.col ^ (d << 6);
  const char* a = t + c + 16 * s * T::PITCH;
  const char* b = t + (c ^ 16) + (16 * s + 8) * T::PITCH;  // 8 rows on: the swizzle's last bit
  Frag f;
  const f16x4 h0 = __builtin_bit_cast(f16x4, read_tr(a)), h1 = __builtin_bit_cast(f16x4, read_tr(b));
  const f16x4 l0 = __builtin_bit_cast(f16x4, read_tr(a + T::PLANE)),
              l1 = __builtin_bit_cast(f16x4, read_tr(b + T::PLANE));
  f.hi = __builtin_shufflevector(h0, h1, 0, 1, 2, 3, 4, 5, 6, 7);
  f.lo = __builtin_shufflevector(l0, l1, 0, 1, 2, 3, 4, 5, 6, 7);
  return f;
}

__device__ __forceinline__ float top8(const float (&x)[8]) {
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(x[j]));
  return m;
}

// The largest of a wave's values, all at least 0, in lane 63.
__device__ __forceinline__ float wave_top(float v) {
  auto step = [](float x, auto ctrl, auto rows) {
    return fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value,
                                                                          decltype(rows)::value, 0xF, false)));
  };
  typedef std::integral_constant<int, 0xF> All;
  v = step(v, std::integral_constant<int, 0xB1>{}, All{});   // lanes 1 0 3 2
  v = step(v, std::integral_constant<int, 0x4E>{}, All{});   // lanes 2 3 0 1
  v = step(v, std::integral_constant<int, 0x124>{}, All{});  // four lanes round
  v = step(v, std::integral_constant<int, 0x128>{}, All{});  // eight: a row of 16
  v = step(v, std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});  // rows 0, 2 to 1, 3
  return step(v, std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});  // half to half
}
__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, 64); }

// floor(log2) of a magnitude, within what scale() can raise (smaller ones, 0 among them, as
// 2^-112; infinity as the largest number).
__device__ __forceinline__ int exponent(float m) {
  const int e = (int)(__builtin_bit_cast(unsigned, m) >> 23);
  return min(max(e, 15), 254) - 127;
}
// The power of two that brings values of this exponent to [2^kTop, 2^(kTop + 1)).
__device__ __forceinline__ float scale(int e) { return __builtin_bit_cast(float, (unsigned)(kTop - e + 127) << 23); }

// Eight values read as four from column col and four from col + 4 of n that are there (by now
// or never), where four that reach past the end were read as the last four.
// (FOURS: a way of its own for whole fours, which the widest kernels have no registers for.)
template <bool FOURS>
__device__ __forceinline__ void cut8(float (&x)[8], int n, int cut) {
  if (FOURS && cut == 0) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = n > j ? x[j] : 0.f;
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; k += 4) {
    const float v[4] = {x[k], x[k + 1], x[k + 2], x[k + 3]};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float late = cut == 3 ? v[min(j + 1, 3)] : cut == 2 ? v[min(j + 2, 3)] : v[3];
      x[k + j] = n - k >= 4 ? v[j] : j < n - k ? late : 0.f;
    }
  }
}

// A row of a wave's own operand (dim >= 4; zeros of one that is not there, p being one that
// is), columns 16 s + 8 half .. of step s; the largest magnitude.  All loads before any use.
template <int KS>
__device__ __forceinline__ float load_row(const float* __restrict__ p, int half, int dim, bool there, float (&x)[KS][8]) {
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int c = 16 * s + 8 * half;
    const f32x4u v0 = *reinterpret_cast<const f32x4u*>(p + min(c, dim - 4)),
                 v1 = *reinterpret_cast<const f32x4u*>(p + min(c + 4, dim - 4));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[s][j] = v0[j];
      x[s][4 + j] = v1[j];
    }
  }
  if (dim < 16 * KS || !__all(there)) {
#pragma unroll
    for (int s = 0; s < KS; ++s) cut8<(KS < 8)>(x[s], there ? dim - 16 * s - 8 * half : 0, dim & 3);
  }
  float m = 0.f;
#pragma unroll
  for (int s = 0; s < KS; ++s) m = fmaxf(m, top8(x[s]));
  return m;
}

// An operand's exponent from a tile on whose largest magnitude is `top`, the sums being at the
// largest exponent so far.  A tile far below that would lose bits that rows need which no
// longer see the large one: `odd`, then (fp32 products).
__device__ __forceinline__ int raised(int so_far, float top, bool& odd) {
  const int e = exponent(top);
  odd |= top > 0.f && so_far - e > 16;
  return max(so_far, e);
}

// A thread's share of two tensors' tiles among NT threads: N chunks of eight columns, the
// first tensor's tile and then the second's.  A wave's chunk is of one tensor.
template <class T, int NT>
struct Share {
  static constexpr int ALL = T::R * T::UNITS, N = (2 * ALL + NT - 1) / NT;
  static_assert(ALL % 64 == 0 && NT % 64 == 0, "whole waves");
  float x[N][8];
  // (a chunk past the last is the last, read again and not put)
  static __device__ __forceinline__ int unit(int c) {
    const int id = c * NT + (int)threadIdx.x;
    return (2 * ALL) % NT == 0 ? id : min(id, 2 * ALL - 1);
  }
  static __device__ __forceinline__ bool has(int c) { return (2 * ALL) % NT == 0 || c * NT + (int)threadIdx.x < 2 * ALL; }
  // Of the second tensor?  (the same for all of a wave)
  static __device__ __forceinline__ bool second(int c) {
    if ((c + 1) * NT <= ALL) return false;
    if (c * NT >= ALL) return true;
    return c * NT + __builtin_amdgcn_readfirstlane((int)threadIdx.x) >= ALL;
  }
  static __device__ __forceinline__ int row(int c) { return (unit(c) - (second(c) ? ALL : 0)) / T::UNITS; }
  static __device__ __forceinline__ int col(int c) { return 8 * ((unit(c) - (second(c) ? ALL : 0)) % T::UNITS); }
  // Rows r0 .. r0 + R - 1 (r0 < end) of both, dim >= 4.  What is not there is read at a place that
  // is, and put right by clear() once it has come: two ways of loading would meet in a copy of
  // the registers, which waits for the loads.
  __device__ __forceinline__ void load(const float* __restrict__ base0, int64_t ld0, const float* __restrict__ base1,
                                       int64_t ld1, int r0, int end, int dim) {
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const bool s = second(c);
      const float* p = (s ? base1 : base0) + (int64_t)min(r0 + row(c), end - 1) * (s ? ld1 : ld0);
      const f32x4u v0 = *reinterpret_cast<const f32x4u*>(p + min(col(c), dim - 4)),
                   v1 = *reinterpret_cast<const f32x4u*>(p + min(col(c) + 4, dim - 4));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[c][j] = v0[j];
        x[c][4 + j] = v1[j];
      }
    }
  }
  // Zeros from row `end` and column `dim` on, and in rows h0 .. h1 - 1; four values that reach past
  // dim have been read as the last four.
  __device__ __forceinline__ void clear(int r0, int end, int dim, int h0 = 0, int h1 = 0) {
    if (r0 + T::R <= end && dim == T::DP && (r0 >= h1 || r0 + T::R <= h0)) return;
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const int r = r0 + row(c);
      cut8<(T::DP < 128)>(x[c], (r < end) & ((r < h0) | (r >= h1)) ? dim - col(c) : 0, dim & 3);
    }
  }
  // The largest magnitude of the first (second) tensor's chunks.
  __device__ __forceinline__ float top(bool of_second) const {
    float m = 0.f;
#pragma unroll
    for (int c = 0; c < N; ++c) m = fmaxf(m, second(c) == of_second ? top8(x[c]) : 0.f);
    return m;
  }
  // Split into the two tiles, at the scales that scale_of(second tensor?, row) gives.
  template <class F>
  __device__ __forceinline__ void put(char* t0, char* t1, F scale_of) const {
#pragma unroll
    for (int c = 0; c < N; ++c) {
      if (!has(c)) break;
      const bool s = second(c);
      const int r = row(c), u = col(c) / 8;
      const Frag f = split8<true>(x[c], scale_of(s, r));
      char* at = (s ? t1 : t0) + r * T::PITCH + ((u ^ swizzle<T::DP>(r)) << 4);
      *reinterpret_cast<f16x8*>(at) = f.hi;
      *reinterpret_cast<f16x8*>(at + T::PLANE) = f.lo;
    }
  }
};

// The largest magnitudes of coming tiles of two tensors: slot t of four takes tile t's, a value
// from each wave.  (Not an atomic maximum: the compiler makes a loop over lanes of it, some 700
// cycles a tile.)
template <int NW>
struct Tops {
  float v[2][4][NW];
  __device__ __forceinline__ void add(int tensor, int t, float m) {
    m = wave_top(m);
    if ((threadIdx.x & 63) == 63) v[tensor][t & 3][threadIdx.x >> 6] = m;
  }
  __device__ __forceinline__ float get(int tensor, int t) const {
    float m = 0.f;
#pragma unroll
    for (int w = 0; w < NW; w += 4) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(&v[tensor][t & 3][w]);
      m = fmaxf(fmaxf(fmaxf(m, x[0]), fmaxf(x[1], x[2])), x[3]);
    }
    return m;
  }
};

// N steps, each using a fragment that has been read from LDS AHEAD steps before.  The barriers hold
// the scheduler to it: left to itself it waits for every read where it is used, which
// costs a step more than its three products.
template <int N, int AHEAD, class Load, class Use>
__device__ __forceinline__ void steps(Load load, Use use) {
  Frag f[AHEAD + 1];
#pragma unroll
  for (int i = 0; i < AHEAD && i < N; ++i) f[i] = load(i);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i + AHEAD < N) f[(i + AHEAD) % (AHEAD + 1)] = load(i + AHEAD);
    __builtin_amdgcn_sched_barrier(0);
    use(i, f[i % (AHEAD + 1)]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// A block's scores set to minus infinity where a row does not see a key, one unsigned comparison
// for both ends of the window.  Rows in lanes: `base` is the row's position less the block's first
// key and 4 (lane / 32) (negative: not there); `sinks` those from that key on, of use if `some`.
__device__ __forceinline__ void hide_keys(f32x16& x, int base, int window, int sinks, bool some) {
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int c = 8 * (r >> 2) + (r & 3);
    const unsigned most = some && c < sinks ? 0x7fffffffu : (unsigned)window;
    x[r] = (unsigned)(base - c) < most ? x[r] : -INFINITY;
  }
}
// Keys in lanes: `base` is the block's first row and 4 (lane / 32) less the key's position, `most`
// how far from a row on it is seen (0: not there).
__device__ __forceinline__ void hide_rows(f32x16& x, int base, unsigned most) {
#pragma unroll
  for (int r = 0; r < 16; ++r) x[r] = (unsigned)(base + 8 * (r >> 2) + (r & 3)) < most ? x[r] : -INFINITY;
}

// The tiles of R keys that rows at positions first .. last (0 <= first <= last) see: sinks before
// the window, then the window.
template <int R>
struct Tiles {
  int before, low, count;
  __device__ __forceinline__ Tiles(const Args& a, int first, int last) {
    low = max(first - a.window + 1, 0) / R;
    before = min((a.sinks + R - 1) / R, low);
    count = before + last / R + 1 - low;
  }
  __device__ __forceinline__ int row(int t) const { return R * (t < before ? t : low + t - before); }
};

}  // namespace wattn
