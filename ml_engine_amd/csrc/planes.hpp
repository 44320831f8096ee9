// Products of operands that are kept as 16-bit planes, C = A B^T on the
// matrix cores.
//
// An operand [rows, k] is split once, by the kernel that makes it, into planes
// of bf16 or fp16 whose sum it is; the product's main loop then only moves
// bytes and multiplies, where one that splits fp32 as it goes
// (split_core.hpp) spends most of its vector instructions on that.
//
// Layout of a packed operand: units of 1 KB, [k / 32][16-row block][plane], each
// the fragment of one 16 x 16 x 32 MFMA as the 64 lanes hold it: lane l has
// row l % 16 of the block and k values 8 (l / 16) .. + 7, 16 bytes.  A tile's
// stage of 32 k is one contiguous run, copied to LDS by global_load_lds a KB per
// wave and instruction; a fragment is one ds_read_b128 of consecutive lanes,
// free of bank conflicts without a swizzle.  The 64 rows of a group lie in its
// four blocks by row % 4, so that a lane ends with 4 x 4 neighbours of C:
// accumulator (i, n, r) of lane (lr, q) of a wave is row 16 q + 4 r + i, column
// 4 lr + n of its 64 x 64 part.
//
// Rows are padded with zeros to whole tiles and k to whole stages by whoever
// packs, so the loop has no bounds: it reads blocks [tile * 4 CM, + 4 CM) of A and
// [tile * 4 CN, + 4 CN) of B for every k block.
#pragma once
#include "common.hpp"

namespace planes {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int kUnit = 1024;  // bytes
constexpr int kK = 32;       // k of a stage

struct Fp16 {
  static __device__ __forceinline__ f32x4 mma(const u32x4& a, const u32x4& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
struct Bf16 {
  static __device__ __forceinline__ f32x4 mma(const u32x4& a, const u32x4& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
  }
};

// A workgroup of CM x CN waves, each 64 x 64 of C; PA, PB planes of the operands.
template <class T_, int CM_, int CN_, int PA_, int PB_>
struct Shape {
  using T = T_;
  static constexpr int CM = CM_, CN = CN_, PA = PA_, PB = PB_;
  static constexpr int TM = 64 * CM, TN = 64 * CN, NW = CM * CN, NTH = 64 * NW;
  static constexpr int UA = 4 * CM * PA, UB = 4 * CN * PB;  // units of a stage
  static constexpr int STAGE = (UA + UB) * kUnit, LDS = 2 * STAGE;
  static_assert((UA + UB) % NW == 0, "units per wave");
};

struct Operand {
  const char* p;
  int64_t kstride;  // bytes from one k block to the next: blocks * planes * kUnit
};

// Byte offset of the 16 bytes with row `row`, k values 8 (k / 8) .. + 7, in a
// packed operand of `blocks` 16-row blocks and P planes (plane 0).
template <int P>
__device__ __forceinline__ int64_t chunk_at(int64_t blocks, int64_t row, int64_t k) {
  const int64_t blk = (row >> 6) * 4 + (row & 3);
  const int pos = (int)(row & 63) >> 2;
  return (((k >> 5) * blocks + blk) * P) * kUnit + (((int)k >> 3) & 3) * 256 + pos * 16;
}

// A wave's place in the workgroup and a lane's in the wave.
template <class S>
struct Lane {
  int lane, lr, q, wm, wn;
  __device__ __forceinline__ Lane() {
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    lane = threadIdx.x & 63;
    lr = lane & 15;
    q = lane >> 4;
    wm = wave % S::CM;
    wn = wave / S::CM;
  }
  // Within the workgroup's tile.
  __device__ __forceinline__ int row(int i, int r) const { return 64 * wm + 16 * q + 4 * r + i; }
  __device__ __forceinline__ int col() const { return 64 * wn + 4 * lr; }
};

// Starts the copy of a stage of tile (tm, tn) into `buf`.
template <class S>
__device__ __forceinline__ void stage_load(const Operand& A, const Operand& B, int tm, int tn, int kb, char* buf) {
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const char* a = A.p + (int64_t)kb * A.kstride + (int64_t)tm * S::UA * kUnit;
  const char* b = B.p + (int64_t)kb * B.kstride + (int64_t)tn * S::UB * kUnit;
#pragma unroll
  for (int j = 0; j < (S::UA + S::UB) / S::NW; ++j) {
    const int u = wave + j * S::NW;  // (uniform)
    const char* src = u < S::UA ? a + u * kUnit : b + (u - S::UA) * kUnit;
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src + lane * 16),
                                     (__attribute__((address_space(3))) void*)(buf + u * kUnit), 16, 0, 0);
  }
}

// Fragments of a stage for one wave, and their products into its sums.
// hi takes the first planes' products, lo those of a first plane with a later one.
template <class S>
__device__ __forceinline__ void stage_mma(const char* buf, const Lane<S>& w, f32x4 (&hi)[4][4], f32x4 (&lo)[4][4]) {
  using T = typename S::T;
  constexpr int PA = S::PA, PB = S::PB;
  const char* a = buf + (w.wm * 4 * PA) * kUnit + w.lane * 16;
  const char* b = buf + (S::UA + w.wn * 4 * PB) * kUnit + w.lane * 16;
  u32x4 fb[4][PB];
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int p = 0; p < PB; ++p) fb[n][p] = *reinterpret_cast<const u32x4*>(b + (n * PB + p) * kUnit);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    u32x4 fa[PA];
#pragma unroll
    for (int p = 0; p < PA; ++p) fa[p] = *reinterpret_cast<const u32x4*>(a + (i * PA + p) * kUnit);
#pragma unroll
    for (int n = 0; n < 4; ++n) hi[i][n] = T::mma(fa[0], fb[n][0], hi[i][n]);
#pragma unroll
    for (int p = 1; p < PB; ++p)
#pragma unroll
      for (int n = 0; n < 4; ++n) lo[i][n] = T::mma(fa[0], fb[n][p], lo[i][n]);
#pragma unroll
    for (int p = 1; p < PA; ++p)
#pragma unroll
      for (int n = 0; n < 4; ++n) lo[i][n] = T::mma(fa[p], fb[n][0], lo[i][n]);
  }
}

template <class S>
__device__ __forceinline__ void multiply(const Operand& A, const Operand& B, int tm, int tn, int k0, int k1, char* lds,
                                         const Lane<S>& w, f32x4 (&hi)[4][4], f32x4 (&lo)[4][4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int n = 0; n < 4; ++n) hi[i][n] = lo[i][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (k0 < k1) stage_load<S>(A, B, tm, tn, k0, lds);
  for (int k = k0; k < k1; ++k) {
    char* cur = lds + ((k - k0) & 1) * S::STAGE;
    char* nxt = lds + (((k - k0) & 1) ^ 1) * S::STAGE;
    __syncthreads();  // this stage has arrived, and nobody reads the last one any more
    if (k + 1 < k1) stage_load<S>(A, B, tm, tn, k + 1, nxt);
    stage_mma<S>(cur, w, hi, lo);
  }
}

}  // namespace planes
