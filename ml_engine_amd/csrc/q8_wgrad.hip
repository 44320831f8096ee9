// A Linear's weight gradient from an input kept in 8 bits (q8.hpp):
//   dW [in, out] (+)= X^T dY,  db (+)= column sums of dY,  X the kept values.
//
// A kept value q 2^k is a bf16 number, and dY is the exact sum of three bf16 planes
// (the top 8 bits of its magnitude, the next 8, the last 8), so three MFMAs make
// the products exactly, where fp32 operands take six and drop terms.  The first
// plane's products go to one accumulator, the others' to a second.  The later
// planes hold 2^24 times their bits: those of values under 2^-110, which long
// training meets, would otherwise lie below the smallest bf16 and be lost (a relative
// 7e-5 at 2^-120, all towards zero).  Where the second accumulator overflows (sums of
// 2^111 or more) and the first does not, fp32 products take those elements' place.
//
// A tile of 64 CM x 64 CN of dW, 32 rows of X and dY to a stage, double-buffered in
// LDS in the unit layout of planes.hpp.  While a stage is multiplied, the next one's
// raw codes and floats, loaded a stage earlier, are turned into planes and written to
// the other buffer.  Rows are shared between workgroups where the tiles alone
// would leave CUs idle; the partial sums are joined in order.  Bound by the matrix cores
// and the conversion beside them (busy 41 % of the time): 8192 x 1024 x 4096 in 207 us, 1.0
// PFLOP/s of 16 bits (9 us more to join two row splits; with the later planes unscaled 4 less).
#include "gemm_args.hpp"
#include "planes.hpp"
#include "q8.hpp"

#include <algorithm>
#include <cmath>

using namespace mle;

namespace {

using planes::kUnit;
using planes::u32x4;
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

template <int CM, int CN>
using Shape = planes::Shape<planes::Bf16, CM, CN, 1, 3>;

struct WgradArgs {
  const int8_t* q;
  int64_t ldq;
  const uint8_t* e;
  int64_t lde;
  const float* dY;
  int64_t lddy;
  float* dW;
  int64_t lddw;
  float* db;
  int rows, in, out, accumulate;
  int gx, gy, splits, per;  // tiles; K splits and the stages of each
  float* part;              // [split][in][out], then [split][out] of db, where splits > 1
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, (int)bytes, 0x00020000);
}

// The raw values of one thread's part of a stage.
//   X:  4 columns x 4 rows of codes and the rows' exponent bytes, per task.  Rows past
//       the last read it again: dY's zeros meet them.
//   dY: 8 rows of a column, per task; rows past the last read as zero.
// Columns past the matrix only feed outputs that are not stored.
template <class S>
struct Raw {
  static constexpr int NA = S::TM * 2 / S::NTH, NB = S::TN * 4 / S::NTH;
  static_assert(NA + NB <= 4, "a row of products for each conversion");
  unsigned code[NA][4];
  unsigned exp[NA][4];
  float y[NB][8];
};

// NARROW: fewer than 4 columns of X.
template <class S, bool NARROW>
__device__ __forceinline__ void load_stage(const WgradArgs& a, int m0, int n0, int row0, int rows, Raw<S>& x) {
  using R = Raw<S>;
  const int t = threadIdx.x, n = min(rows - row0, planes::kK);  // n <= 0: nothing
#pragma unroll
  for (int c = 0; c < R::NA; ++c) {
    const int u = t + c * S::NTH, m = m0 + 4 * (u % (S::TM / 4)), k = row0 + 4 * (u / (S::TM / 4));
    // four codes at any alignment; at the row's end the last four, moved down
    const int at = NARROW ? 0 : min(m, a.in - 4), down = NARROW ? 0 : 8 * min(m - at, 3), grp = min(m, a.in - 1) / q8::kGroup;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t row = min(k + j, rows - 1);
      const int8_t* q = a.q + row * a.ldq + at;
      unsigned v = 0;
      if (!NARROW) {
        __builtin_memcpy(&v, q, 4);
        v >>= down;
      } else {
        for (int i = 0; i < 3; ++i) v |= (unsigned)(unsigned char)q[min(i, a.in - 1)] << (8 * i);
      }
      x.code[c][j] = v;
      x.exp[c][j] = a.e[row * a.lde + grp];
    }
  }
  const uint32_t ldy = (uint32_t)a.lddy * 4u;
  const auto ry = rsrc(a.dY + (n > 0 ? row0 : 0) * a.lddy, n > 0 ? (n - 1) * ldy + a.out * 4u : 0u);
#pragma unroll
  for (int c = 0; c < R::NB; ++c) {
    // a wave: 64 columns of one eight of rows, its lanes in the order that the
    // units hold them
    const int u = t + c * S::NTH, lane = u & 63, g = (u >> 6) % S::CN, k = 8 * ((u >> 6) / S::CN);
    const int col = n0 + 64 * g + 4 * (lane & 15) + (lane >> 4);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      x.y[c][j] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(ry, (int)((k + j) * ldy + col * 4u), 0, 0));
  }
}

using planes::bits;
using planes::high_halves;
using planes::top8;
constexpr float kLater = 0x1p24f;  // what the second and third plane are scaled by

// Codes to bf16: exact, so the low half of the product is zero.
template <class S>
__device__ __forceinline__ void put_codes(char* lds, const Raw<S>& x, int c) {
  const int u = threadIdx.x + c * S::NTH, m = 4 * (u % (S::TM / 4)), k = 4 * (u / (S::TM / 4));
  float step[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) step[j] = q8::step_of(x.exp[c][j]);
  char* p = lds + (m >> 6) * 4 * kUnit + (k >> 3) * 256 + ((m & 63) >> 2) * 16 + (k & 4) * 2;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    unsigned v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = bits((float)(int)(signed char)(x.code[c][j] >> (8 * i)) * step[j]);
    *reinterpret_cast<u32x2*>(p + i * kUnit) = u32x2{high_halves(v[0], v[1]), high_halves(v[2], v[3])};
  }
}
// A column's eight floats to their three planes.  (An infinity's remainders are
// NaN, and so are its products.  The remainders' scale is exact; beyond 2^111 it
// makes infinities.)
template <class S>
__device__ __forceinline__ void put_floats(char* lds, const Raw<S>& x, int c) {
  const int u = threadIdx.x + c * S::NTH, lane = u & 63, g = (u >> 6) % S::CN, k8 = (u >> 6) / S::CN;
  char* p = lds + S::UA * kUnit + (g * 4 + (lane >> 4)) * 3 * kUnit + k8 * 256 + (lane & 15) * 16;
  u32x4 h, m, l;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = x.y[c][2 * j], b = x.y[c][2 * j + 1];
    const float ra = (a - top8(a)) * kLater, rb = (b - top8(b)) * kLater;
    h[j] = high_halves(bits(a), bits(b));
    m[j] = high_halves(bits(ra), bits(rb));
    l[j] = high_halves(bits(ra - top8(ra)), bits(rb - top8(rb)));
  }
  *reinterpret_cast<u32x4*>(p) = h;
  *reinterpret_cast<u32x4*>(p + kUnit) = m;
  *reinterpret_cast<u32x4*>(p + 2 * kUnit) = l;
}

// The two sums to one, in hi.  Elements whose later planes overflowed are summed again
// from fp32 products over rows [r0, r1), four of a lane's sixteen rows of dW at a time;
// c0 is its first column, m0 the tile's first row.
template <class S>
__device__ __forceinline__ void join_planes(const WgradArgs& a, const planes::Lane<S>& w, int m0, int c0, int r0, int r1,
                                            f32x4 (&hi)[4][4], const f32x4 (&lo)[4][4]) {
  float finite = 0.f;  // stays zero while every sum is
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) finite = fmaf(lo[i][n][r], 0.f, finite);
  unsigned over[4] = {};  // by r: bit 4 i + n
  if (finite != 0.f) {  // (what lies past dY's columns may be anything: those are not stored)
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int n = 0; n < 4; ++n)
          if ((c0 + n < a.out) & __builtin_isfinite(hi[i][n][r]) & !__builtin_isfinite(lo[i][n][r])) over[r] |= 1u << (4 * i + n);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int n = 0; n < 4; ++n) hi[i][n] += lo[i][n] * (1.f / kLater);
  if ((over[0] | over[1] | over[2] | over[3]) == 0) return;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    f32x4 sum[4] = {};
#pragma unroll 1
    for (int row = r0; row < r1; ++row) {
      const float* dy = a.dY + row * a.lddy;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int m = min(m0 + w.row(i, r), a.in - 1);
        const float x = (float)a.q[row * a.ldq + m] * q8::step_of(a.e[row * a.lde + m / q8::kGroup]);
#pragma unroll
        for (int n = 0; n < 4; ++n) sum[i][n] = fmaf(x, dy[min(c0 + n, a.out - 1)], sum[i][n]);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int n = 0; n < 4; ++n)
        if ((over[r] >> (4 * i + n)) & 1) hi[i][n][r] = sum[i][n];
  }
}

template <class S, bool NARROW>
__global__ __launch_bounds__(S::NTH, 2) void q8_wgrad_kernel(WgradArgs a) {
  using R = Raw<S>;
  __shared__ __attribute__((aligned(16))) char lds[S::LDS];
  const planes::Lane<S> w;
  int tm, tn, z;
  gemm::item_tile(blockIdx.x, a.gx * a.gy * a.splits, a.gx, a.gy, tm, tn, z);
  const int m0 = tm * S::TM, n0 = tn * S::TN;
  const int r0 = z * a.per * planes::kK, r1 = (int)min((int64_t)a.rows, (int64_t)r0 + (int64_t)a.per * planes::kK);
  const int nk = (r1 - r0 + planes::kK - 1) / planes::kK;
  const bool sums = a.db && tm == 0;
  f32x4 hi[4][4], lo[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int n = 0; n < 4; ++n) hi[i][n] = lo[i][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  double col[R::NB] = {};
  R x;  // the raw stage on its way (two of them: 8192 x 1024 x 4096 247 -> 266 us)
  auto add = [&]() {
    if (sums)
#pragma unroll
      for (int c = 0; c < R::NB; ++c)
        col[c] += ((x.y[c][0] + x.y[c][1]) + (x.y[c][2] + x.y[c][3])) + ((x.y[c][4] + x.y[c][5]) + (x.y[c][6] + x.y[c][7]));
  };
  load_stage<S, NARROW>(a, m0, n0, r0, r1, x);
#pragma unroll
  for (int c = 0; c < R::NA; ++c) put_codes<S>(lds, x, c);
#pragma unroll
  for (int c = 0; c < R::NB; ++c) put_floats<S>(lds, x, c);
  add();
  load_stage<S, NARROW>(a, m0, n0, r0 + planes::kK, r1, x);
  for (int k = 0; k < nk; ++k) {
    const char* cur = lds + (k & 1) * S::STAGE;
    char* nxt = lds + ((k & 1) ^ 1) * S::STAGE;
    __syncthreads();  // this stage is written, and nobody reads the other buffer any more
    const char* pa = cur + (w.wm * 4) * kUnit + w.lane * 16;
    const char* pb = cur + (S::UA + w.wn * 12) * kUnit + w.lane * 16;
    u32x4 fb[4][3], fa[2];
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int p = 0; p < 3; ++p) fb[n][p] = *reinterpret_cast<const u32x4*>(pb + (n * 3 + p) * kUnit);
    fa[0] = *reinterpret_cast<const u32x4*>(pa);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // (the small tile's loads want the whole of this order; the large one is
      // faster as the compiler mixes it: 16384 x 2048 x 2048 471 against 570 us)
      if (S::NW <= 4) __builtin_amdgcn_sched_barrier(0);
      if (i < 3) fa[(i + 1) & 1] = *reinterpret_cast<const u32x4*>(pa + (i + 1) * kUnit);
#pragma unroll
      for (int p = 2; p > 0; --p)
#pragma unroll
        for (int n = 0; n < 4; ++n) lo[i][n] = planes::Bf16::mma(fa[i & 1], fb[n][p], lo[i][n]);
#pragma unroll
      for (int n = 0; n < 4; ++n) hi[i][n] = planes::Bf16::mma(fa[i & 1], fb[n][0], hi[i][n]);
      // the next stage's conversion beside the last rows' products, so that its
      // loads have most of a stage to arrive
#pragma unroll
      for (int c = 0; c < R::NA + R::NB; ++c)
        if (c + 4 - (R::NA + R::NB) == i) {
          if (c < R::NA) put_codes<S>(nxt, x, c);
          else put_floats<S>(nxt, x, c - R::NA);
        }
    }
    add();
    load_stage<S, NARROW>(a, m0, n0, r0 + (k + 2) * planes::kK, r1, x);
  }

  if (sums) {  // the eights of rows of each column, in order
    double* red = reinterpret_cast<double*>(lds);
    __syncthreads();
#pragma unroll
    for (int c = 0; c < R::NB; ++c) {
      const int u = threadIdx.x + c * S::NTH, lane = u & 63, g = (u >> 6) % S::CN, k8 = (u >> 6) / S::CN;
      red[k8 * S::TN + 64 * g + 4 * (lane & 15) + (lane >> 4)] = col[c];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < S::TN; c += S::NTH) {
      if (n0 + c >= a.out) continue;
      const float s = (float)(((red[c] + red[S::TN + c]) + red[2 * S::TN + c]) + red[3 * S::TN + c]);
      if (a.splits > 1) a.part[(int64_t)a.splits * a.in * a.out + (int64_t)z * a.out + n0 + c] = s;
      else a.db[n0 + c] = a.accumulate ? a.db[n0 + c] + s : s;
    }
  }
  const bool whole = a.splits == 1;
  float* out = whole ? a.dW : a.part + (int64_t)z * a.in * a.out;
  const int64_t ld = whole ? a.lddw : a.out;
  const bool old = whole && a.accumulate;
  const int c0 = n0 + w.col();
  join_planes<S>(a, w, m0, c0, r0, r1, hi, lo);
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = m0 + w.row(i, r);
      if (row >= a.in || c0 >= a.out) continue;
      float* p = out + row * ld + c0;
      f32x4 v;
#pragma unroll
      for (int n = 0; n < 4; ++n) v[n] = hi[i][n][r];
      if (c0 + 3 < a.out) {
        if (old) v += *reinterpret_cast<const f32x4u*>(p);
        *reinterpret_cast<f32x4u*>(p) = v;
      } else {
#pragma unroll
        for (int n = 0; n < 4; ++n)
          if (c0 + n < a.out) p[n] = old ? p[n] + v[n] : v[n];
      }
    }
}

// The splits' sums in order, four columns to a thread; the last workgroups take db.
__global__ __launch_bounds__(256) void q8_wgrad_join_kernel(WgradArgs a, unsigned nmain) {
  const int64_t mn = (int64_t)a.in * a.out;
  if (blockIdx.x >= nmain) {
    const int c = (blockIdx.x - nmain) * 256 + threadIdx.x;
    if (c >= a.out) return;
    const float* p = a.part + a.splits * mn + c;
    float s = p[0];
#pragma unroll 8
    for (int z = 1; z < a.splits; ++z) s += p[(int64_t)z * a.out];
    a.db[c] = a.accumulate ? a.db[c] + s : s;
    return;
  }
  const int groups = (a.out + 3) / 4;
  const int64_t total = (int64_t)a.in * groups;
  for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < total; u += (int64_t)nmain * 256) {
    const int64_t row = u / groups;
    const int col = (int)(u - row * groups) * 4;
    const float* p = a.part + row * a.out + col;
    float* d = a.dW + row * a.lddw + col;
    if (col + 3 < a.out) {
      f32x4 s = *reinterpret_cast<const f32x4u*>(p);
#pragma unroll 8
      for (int z = 1; z < a.splits; ++z) s += *reinterpret_cast<const f32x4u*>(p + z * mn);
      if (a.accumulate) s += *reinterpret_cast<const f32x4u*>(d);
      *reinterpret_cast<f32x4u*>(d) = s;
    } else {
      for (int n = 0; n < 4 && col + n < a.out; ++n) {
        float s = p[n];
        for (int z = 1; z < a.splits; ++z) s += p[z * mn + n];
        d[n] = a.accumulate ? d[n] + s : s;
      }
    }
  }
}

// Tile and K splits.  Large tiles (256 x 128) where they fill half the chip or
// more at a split of at least 32 stages, else small ones (128 x 128); then as many
// splits as make one workgroup to a CU of the large, two of the small, of at
// least 8 and 4 stages, and no more than pay for their partial sums (a stage
// takes about 1 us, a byte written and read again 0.5 ps).  A large tile half of which is past
// the matrix loses (16384 x 48 x 4096 127 us against 103), one with a third of it wins
// (8192 x 330 x 4096 124 against 144).
constexpr int kMost = 1 << 30;  // rows, in, out
struct WgradPlan {
  bool large;
  int gx, gy, splits, per;
  size_t bytes;
};
WgradPlan wgrad_plan(int rows, int in, int out) {
  WgradPlan p;
  const int stages = (rows + planes::kK - 1) / planes::kK;
  const int64_t big = (int64_t)((in + 255) / 256) * ((out + 127) / 128);
  p.large = in > 128 && big * std::max(1, stages / 32) >= gemm::kChipCus / 2;
  const int tm = p.large ? 256 : 128;
  p.gx = (out + 127) / 128;
  p.gy = (in + tm - 1) / tm;
  const int64_t tiles = (int64_t)p.gx * p.gy, want = (p.large ? 1 : 2) * gemm::kChipCus / tiles;
  const int64_t pays = (int64_t)std::sqrt(stages * 5e5 / ((double)in * out));
  const int n = (int)std::max<int64_t>(1, std::min<int64_t>(std::min(want, pays), stages / (p.large ? 8 : 4)));
  p.per = std::max(1, (stages + n - 1) / n);
  p.splits = std::max(1, (stages + p.per - 1) / p.per);
  p.bytes = p.splits > 1 ? (size_t)p.splits * ((size_t)in * out + out) * sizeof(float) : 0;
  return p;
}

}  // namespace

extern "C" {

size_t mle_q8_linear_wgrad_ws_bytes(int rows, int in, int out) {
  return rows <= 0 || in <= 0 || out <= 0 || rows > kMost || in > kMost || out > kMost ? 0 : std::max<size_t>(wgrad_plan(rows, in, out).bytes, 16);
}

int mle_q8_linear_wgrad(mle_stream stream, int rows, int in, int out, const int8_t* q, int64_t ldq, const uint8_t* e,
                        int64_t lde, const float* dY, int64_t lddy, float* dW, int64_t lddw, float* db, int accumulate,
                        void* ws, size_t ws_bytes) {
  const int rc = q8::check_shape("mle_q8_linear_wgrad", rows, in, q, ldq, e, lde);
  if (rc) return rc;
  MLE_CHECK_ARG(rows <= kMost && out > 0 && out <= kMost && dW && (dY || rows == 0) && lddy >= out && lddw >= out,
                "mle_q8_linear_wgrad: bad argument (rows %d, out %d, lddy %lld, lddw %lld)", rows, out, (long long)lddy,
                (long long)lddw);
  // a stage's 32 rows lie within the 31-bit offsets of buffer loads
  if (lddy > 0xffffff) return set_error(MLE_ERR_UNSUPPORTED, "mle_q8_linear_wgrad: lddy %lld above 2^24", (long long)lddy);
  if (rows == 0) {
    if (accumulate) return MLE_OK;
    if (db) {
      const int z = mle_fill(stream, db, 0.f, (size_t)out);
      if (z) return z;
    }
    return mle_gemm_ex(stream, 1, 0, in, out, 0, 1.f, nullptr, in, 0, nullptr, out, 0, 0.f, dW, lddw, 0, 1, nullptr, nullptr,
                       nullptr, 0);  // (a product over nothing)
  }
  const size_t need = mle_q8_linear_wgrad_ws_bytes(rows, in, out);
  if (need && (!ws || !aligned16(ws) || ws_bytes < need))
    return set_error(MLE_ERR_WORKSPACE, "mle_q8_linear_wgrad: workspace of %zu bytes, 16-byte aligned, needed", need);
  const WgradPlan p = wgrad_plan(rows, in, out);
  MLE_CHECK_ARG((int64_t)p.gx * p.gy * p.splits * (p.large ? 512 : 256) < (1LL << 32), "mle_q8_linear_wgrad: grid too large");
  const WgradArgs a{q, ldq, e, lde, dY, lddy, dW, lddw, db, rows, in, out, accumulate, p.gx, p.gy, p.splits, p.per,
              static_cast<float*>(ws)};
  hipStream_t s = as_stream(stream);
  const unsigned grid = (unsigned)(p.gx * p.gy * p.splits);
  ProbeScope probe("q8_wgrad", s, 2.0 * rows * (double)in * out, rows * (double)in + 4.0 * ((double)rows * out + (double)in * out));
  if (p.large) mle::launch(q8_wgrad_kernel<Shape<4, 2>, false>, grid, 512, 0, s, a);
  else if (in >= 4) mle::launch(q8_wgrad_kernel<Shape<2, 2>, false>, grid, 256, 0, s, a);
  else mle::launch(q8_wgrad_kernel<Shape<2, 2>, true>, grid, 256, 0, s, a);
  if (p.splits > 1) {
    const unsigned nmain = stream_grid((size_t)in * ((out + 3) / 4), 256, 4096);
    mle::launch(q8_wgrad_join_kernel, nmain + (db ? (unsigned)((out + 255) / 256) : 0u), 256, 0, s, a, nmain);
  }
  return check_launch("mle_q8_linear_wgrad");
}

}  // extern "C"
