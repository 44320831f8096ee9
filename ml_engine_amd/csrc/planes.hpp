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

// The high halves of two words side by side: `b` above `a`.
__device__ __forceinline__ unsigned high_halves(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }
__device__ __forceinline__ unsigned bits(float x) { return __builtin_bit_cast(unsigned, x); }
// x with its last 16 bits cleared: a bf16 number, exact for any x.
__device__ __forceinline__ float top8(float x) { return __builtin_bit_cast(float, bits(x) & 0xffff0000u); }

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

// The same with the sums cleared every `run` stages: begin(first stage of the run) is
// called before the run, whose loads are then there at its end, and end() after it, to
// add the sums to what the caller keeps.
template <class S, class F, class G>
__device__ __forceinline__ void multiply_runs(const Operand& A, const Operand& B, int tm, int tn, int k0, int k1, int run,
                                              char* lds, const Lane<S>& w, f32x4 (&hi)[4][4], f32x4 (&lo)[4][4], F begin,
                                              G end) {
  if (k0 < k1) stage_load<S>(A, B, tm, tn, k0, lds);
  for (int kr = k0; kr < k1; kr += run) {
    begin(kr);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int n = 0; n < 4; ++n) hi[i][n] = lo[i][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int ke = min(k1, kr + run);
    for (int k = kr; k < ke; ++k) {
      char* cur = lds + ((k - k0) & 1) * S::STAGE;
      char* nxt = lds + (((k - k0) & 1) ^ 1) * S::STAGE;
      __syncthreads();
      if (k + 1 < k1) stage_load<S>(A, B, tm, tn, k + 1, nxt);
      stage_mma<S>(cur, w, hi, lo);
    }
    end();
  }
}

// ------------------------------------------------------------- fp16 operands
// A scaled value v in two fp16 planes, h + 2^-LO l: with |v| < 2^15 the pair holds 22
// bits of every value down to 2^-(LO + 3) and 2^-(24 + LO) of the smaller ones.
template <int LO>
__device__ __forceinline__ void put16(char* p, const float (&v)[8]) {
  f16x8 h, l;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    h[j] = (_Float16)v[j];
    l[j] = (_Float16)((v[j] - (float)h[j]) * (float)(1 << LO));
  }
  *reinterpret_cast<f16x8*>(p) = h;
  *reinterpret_cast<f16x8*>(p + kUnit) = l;
}
// The same of x 2^e; what is not finite stays in the first plane.
template <int LO>
__device__ __forceinline__ void put16(char* p, const float (&x)[8], const int (&e)[8]) {
  f16x8 h, l;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float v = __builtin_ldexpf(x[j], e[j]);
    h[j] = (_Float16)v;
    l[j] = __builtin_isfinite(v) ? (_Float16)((v - (float)h[j]) * (float)(1 << LO)) : (_Float16)0.f;
  }
  *reinterpret_cast<f16x8*>(p) = h;
  *reinterpret_cast<f16x8*>(p + kUnit) = l;
}

struct PackArgs {
  const float* src;
  int64_t ld;
  int rows, k;          // of the operand; rest zeros
  int blocks, kblocks;  // of the packed operand
  const int* ex;        // exponents by k or by row
  // What is left out, zeros whatever it holds (nullable): pack_cols: k with keys < 0;
  // rows (pack_cols) or k (pack_rows) with a bias of -infinity.
  const int* keys;
  const float* bias;
  char* out;
  // Blocks of 256 threads that pack it.
  __host__ __device__ int64_t rows_blocks() const { return ((int64_t)blocks * kblocks + 3) / 4; }
  __host__ __device__ int64_t cols_blocks() const { return ((int64_t)(blocks / 4) * kblocks + 3) / 4; }
};

// Operands whose k runs along the source's rows (element (row, k) at row * ld + k): a
// wave per unit, 128 contiguous bytes of 16 rows; 256 threads to a block.
template <bool EX_BY_K, int LO>
__device__ __forceinline__ void pack_rows(const PackArgs& a, int64_t block) {
  const int64_t u = block * 4 + (threadIdx.x >> 6);
  if (u >= (int64_t)a.blocks * a.kblocks) return;
  const int lane = threadIdx.x & 63;
  const int kb = (int)(u / a.blocks), blk = (int)(u - (int64_t)kb * a.blocks);
  const int row = (blk >> 2) * 64 + 4 * (lane & 15) + (blk & 3), k = kb * 32 + 8 * (lane >> 4);
  float x[8];
  int e[8];
  const int n = row < a.rows ? min(max(a.k - k, 0), 8) : 0;
  const float* p = a.src + (int64_t)row * a.ld + k;
  if (n == 8) {
    const f32x4 v0 = reinterpret_cast<const f32x4u*>(p)[0], v1 = reinterpret_cast<const f32x4u*>(p)[1];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = v0[j];
      x[4 + j] = v1[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = j < n ? p[j] : 0.f;
  }
  if (a.bias) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (a.bias[min(k + j, a.k - 1)] == -INFINITY) x[j] = 0.f;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) e[j] = EX_BY_K ? a.ex[min(k + j, a.k - 1)] : a.ex[min(row, a.rows - 1)];
  put16<LO>(a.out + u * 2 * kUnit + lane * 16, x, e);
}

// Operands whose rows run along the source's (element (row, k) at k * ld + row): a
// wave per 64-row group and k block, 256 contiguous bytes of 32 source rows; the
// 4 x 8 values of a lane are transposed in its registers.
template <bool EX_BY_K, int LO>
__device__ __forceinline__ void pack_cols(const PackArgs& a, int64_t block) {
  const int groups = a.blocks >> 2;
  const int64_t u = block * 4 + (threadIdx.x >> 6);
  if (u >= (int64_t)groups * a.kblocks) return;
  const int lane = threadIdx.x & 63;
  const int kb = (int)(u / groups), g = (int)(u - (int64_t)kb * groups);
  const int row = g * 64 + 4 * (lane & 15), k = kb * 32 + 8 * (lane >> 4);
  f32x4 x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const bool live = k + j < a.k && (!a.keys || a.keys[k + j] >= 0);
    const float* p = a.src + (int64_t)(k + j) * a.ld + row;
    x[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (live && row + 3 < a.rows) {
      x[j] = *reinterpret_cast<const f32x4u*>(p);
    } else if (live) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (row + i < a.rows) x[j][i] = p[i];
    }
  }
  int e[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) e[j] = EX_BY_K ? a.ex[min(k + j, a.k - 1)] : 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float v[8];
    const bool out = a.bias && a.bias[min(row + i, a.rows - 1)] == -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = out ? 0.f : x[j][i];
      if (!EX_BY_K) e[j] = a.ex[min(row + i, a.rows - 1)];
    }
    put16<LO>(a.out + ((int64_t)kb * a.blocks + g * 4 + i) * 2 * kUnit + lane * 16, v, e);
  }
}

}  // namespace planes
