// The vocabulary's output projection with its softmax cross entropy, without
// keeping the logits.
//
//   l = X W + b,  lse_r = log sum_v exp l_rv
//   row_loss_r = lse_r - l_r,key(r) where key(r) is in [0, vocab), else 0
//   P_rv = s (exp(l_rv - lse_r) - [v = key(r)]), 0 for the other rows
//   dX = P W^T,  dW = X^T P,  db = column sums of P
//
// The logits are formed piece by piece of the vocabulary, once in the forward
// and once more in the backward: 8 rows d vocab operations where keeping
// rows x vocab logits would take 6.
//
// Few logits: the library's product writes a piece's logits to the workspace and
// small kernels walk them.  More: products of fp16 planes (planes.hpp), in which
// no logit is ever stored.
//
//   An fp32 value scaled into fp16's range is the sum of two fp16 values to 22
//   bits, and three MFMAs (h h, h l, l h) make a product where three bf16 planes
//   (split_core.hpp) need six.  The error per product, 2^-22 and random, is that
//   of fp32 products summed over a long k.  Scales are powers of two, one per index
//   wherever the sum allows it:
//     logits  X by feature (its largest magnitude to 2^15), W by the same feature
//             inversely and one factor per piece: a feature's share of a logit
//             keeps its bits however the two sides divide it
//     dX      W by feature; P as it is, |P| <= 1
//     dW      X by feature; P by column and 64 rows, whose partial sums are
//             scaled back one by one
//   so that a small gradient of a column or feature is as exact as a large one.  Within
//   a scale, values down to 2^-28 of the largest keep their 22 bits (the second plane
//   holds 2^11 times the remainder; without that 2^-17, and a column's small
//   probabilities were lost beside a target's), and smaller ones are held to 2^-50 of it.
//
//   P leaves the tile that forms it in both orders, packed for the two products
//   that read it; db's column sums are taken from the same registers.
#include "gemm_args.hpp"
#include "planes.hpp"
#include "split_core.hpp"

#include <float.h>

#include <algorithm>

using namespace mle;

namespace {

constexpr int NT = 256;

struct Rows {
  const int32_t* keys;
  int clen, max_clen, vocab;
  int r0;  // the call's row that is row 0 here
  __device__ __forceinline__ int key(int64_t r) const {
    r += r0;
    const int k = keys[clen == max_clen ? r : r / clen * max_clen + r % clen];
    return k >= 0 && k < vocab ? k : -1;
  }
};

// What a row has of the vocabulary's pieces so far.
struct RowState {
  float max, sum, target, pad;  // sum of exp(l - max)
};

// A stored logit x of a piece's column c: -infinity where the bias (the piece's, or
// null) takes the entry out, also if its weights' product is infinite or a NaN.
__device__ __forceinline__ float logit(float x, const float* bias, int c) {
  return x != x && bias && bias[c] == -INFINITY ? -INFINITY : x;
}

// A row of a piece to L threads: its maximum and sum join the row's.  A wave to a row
// of few columns (8192 x 300: 36 us with a workgroup to it, 5.6 so).
template <int L>
__global__ __launch_bounds__(L < NT ? NT : L) void xent_stats_kernel(const float* __restrict__ l, int nrows, int cols, int v0,
                                                                     const float* __restrict__ bias, Rows rows,
                                                                     RowState* __restrict__ state, int first) {
  __shared__ float red[L / 64];
  const int64_t r = L < NT ? (int64_t)blockIdx.x * (NT / L) + threadIdx.x / L : blockIdx.x;
  const int t = threadIdx.x % L;
  if (r >= nrows) return;  // (a whole wave)
  const float* x = l + r * cols;
  float m = -FLT_MAX;
#pragma unroll 4
  for (int c = t; c < cols; c += L) m = fmaxf(m, x[c]);  // (not of a NaN)
  m = L == 64 ? wave_max(m) : block_max<L>(m, red);
  float s = 0.f;
#pragma unroll 4
  for (int c = t; c < cols; c += L) s += expf(x[c] - m);
  s = L == 64 ? wave_sum(s) : block_sum<L>(s, red);
  if (s != s && bias) {  // a NaN: those of entries that the bias takes out do not count
    s = 0.f;
    for (int c = t; c < cols; c += L) s += expf(logit(x[c], bias, c) - m);
    s = L == 64 ? wave_sum(s) : block_sum<L>(s, red);
  }
  if (t != 0) return;
  RowState n{m, s, 0.f, 0.f};
  if (!first) {
    const RowState o = state[r];
    n.max = fmaxf(o.max, m);
    n.sum = o.sum * expf(o.max - n.max) + s * expf(m - n.max);
    n.target = o.target;
  }
  const int k = rows.key(r);
  if (k >= v0 && k < v0 + cols) n.target = logit(x[k - v0], bias, k - v0);
  state[r] = n;
}

// lse, the row losses and their scaled sum; one workgroup.
__global__ __launch_bounds__(1024) void xent_finish_kernel(const RowState* __restrict__ state, int nrows, Rows rows,
                                                           float scale, float* __restrict__ lse,
                                                           float* __restrict__ row_loss, float* __restrict__ loss, int add) {
  __shared__ double red[16];
  double sum = 0.0;
  for (int64_t r = threadIdx.x; r < nrows; r += 1024) {
    const RowState t = state[r];
    const float z = t.max + logf(t.sum);
    const float one = rows.key(r) >= 0 ? z - t.target : 0.f;
    lse[r] = z;
    if (row_loss) row_loss[r] = one;
    sum += (double)one;
  }
  sum = block_sum<1024>(sum, red);
  if (threadIdx.x == 0) loss[0] = (float)(sum * (double)scale) + (add ? loss[0] : 0.f);
}

// A piece's logits to P, in place: 1024 of them, in the matrix's order, to a workgroup.
// Those past the first `blocks` take the rows of X that take part, the others as zeros,
// for dW: what a row that takes no part holds, NaN included, must not reach it.
// db (nullable) is cleared for the product that adds to it.
__global__ __launch_bounds__(NT) void xent_grad_kernel(float* l, int nrows, int cols, int v0, Rows rows,
                                                       const float* __restrict__ lse, const float* __restrict__ upstream,
                                                       float scale, unsigned blocks, const float* __restrict__ X, int64_t ldx,
                                                       int d, float* __restrict__ out, float* __restrict__ db,
                                                       const float* __restrict__ bias) {
  const bool logits = blockIdx.x < blocks;
  const unsigned n = logits ? cols : d;
  const int64_t e0 = (int64_t)(logits ? blockIdx.x : blockIdx.x - blocks) * (4 * NT);
  const int64_t r0 = e0 / n;
  const unsigned c0 = (unsigned)(e0 - r0 * n);
  const float g = upstream ? upstream[0] * scale : scale;
  int key[4];
  float x[4], z[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // (every load on its way before the first is used; past the end: the last row's)
    const unsigned at = c0 + i * NT + threadIdx.x, down = at / n, c = at - down * n;
    const int64_t r = min(r0 + down, (int64_t)nrows - 1);
    key[i] = rows.key(r);
    z[i] = logits ? lse[r] : 0.f;
    x[i] = logits ? l[r * cols + c] : X[r * ldx + c];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned at = c0 + i * NT + threadIdx.x, down = at / n, c = at - down * n;
    const int64_t r = r0 + down;
    if (r >= nrows) continue;
    if (logits) {
      if (db && r == 0) db[v0 + c] = 0.f;
      l[r * cols + c] = key[i] >= 0 ? g * (expf(logit(x[i], bias, (int)c) - z[i]) - ((int)c + v0 == key[i] ? 1.f : 0.f)) : 0.f;
    } else {
      out[r * d + c] = key[i] >= 0 ? x[i] : 0.f;
    }
  }
}

// dX (+)= the slices' sums in order, and the products of P's columns from `k0` on.
__global__ __launch_bounds__(NT) void xent_slices_kernel(const float* __restrict__ part, int slices, int64_t total, int d,
                                                         const float* __restrict__ P, int cols, int k0,
                                                         const float* __restrict__ W, int64_t ldw, float* __restrict__ dX,
                                                         int64_t lddx, int accumulate) {
  const int64_t u = (int64_t)blockIdx.x * NT + threadIdx.x;
  if (u >= total) return;
  const int64_t r = u / d;
  const int c = (int)(u - r * d);
  float s = part[u];
  for (int z = 1; z < slices; ++z) s += part[z * total + u];
  for (int k = k0; k < cols; ++k) s = fmaf(P[r * cols + k], W[(int64_t)c * ldw + k], s);
  float* p = dX + r * lddx + c;
  *p = accumulate ? *p + s : s;
}

// dW (+)= xs^T P and db (+)= column sums of P for few rows, where a product's tile has
// only a stage or a few: 128 x 128 of dW to a workgroup, 64 x 64 to a wave, the
// operands' fragments straight from memory (four neighbouring columns of eight rows to
// a lane, transposed in its registers, as planes.hpp orders them), without LDS or
// barriers, so that waves of different progress share a CU.  The products are
// split_core.hpp's: three bf16 planes of 2^24 times an fp32 value, six MFMAs.  Elements
// that this scale makes infinite (values from 2^104, sums from 2^80) are summed again
// from fp32 products.  32 x 876 -> 26839 30 us, 3.2 TB/s written (the library's product
// 68); 64 x 1024 -> 32000 56 us (75).
using planes::u32x4;
struct DwArgs {
  const float* X;  // [rows][d]
  const float* P;  // [rows][cols]
  int rows, d, cols, gx, gy, accumulate;
  float* dW;
  int64_t lddw;
  float* db;
};
__device__ __forceinline__ f32x4 four_of(const float* p, int c, int n) {
  if (c + 3 < n) return *reinterpret_cast<const f32x4u*>(p + c);
  return f32x4{p[min(c, n - 1)], p[min(c + 1, n - 1)], p[min(c + 2, n - 1)], p[min(c + 3, n - 1)]};
}
__global__ __launch_bounds__(NT, 2) void xent_dw_kernel(DwArgs a) {
  using T = planes::Bf16;
  const int lane = threadIdx.x & 63, lr = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), wm = wave & 1, wn = wave >> 1;
  int tm, tn, z;
  gemm::item_tile(blockIdx.x, a.gx * a.gy, a.gx, a.gy, tm, tn, z);
  const int m0 = tm * 128 + 64 * wm, c0 = tn * 128 + 64 * wn + 4 * lr;
  if (m0 >= a.d || tn * 128 + 64 * wn >= a.cols) return;  // (a whole wave; there are no barriers)
  f32x4 hi[4][4], lo[4][4];
  float sum[4] = {};
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int n = 0; n < 4; ++n) hi[i][n] = lo[i][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int r0 = 0; r0 < a.rows; r0 += 32) {
    f32x4 x[8], p[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {  // (past the last row its values again, and P as zeros)
      const int64_t r = min(r0 + 8 * q + j, a.rows - 1);
      p[j] = four_of(a.P + r * a.cols, c0, a.cols);
      x[j] = four_of(a.X + r * a.d, m0 + 4 * lr, a.d);
    }
    u32x4 b[4][3];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float one = r0 + 8 * q + j < a.rows ? p[j][n] : 0.f;
        sum[n] += one;
        v[j] = one * split::kScale;
      }
      split::split8(v, b[n][0], b[n][1], b[n][2]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = x[j][i] * split::kScale;
      u32x4 h, m, l;
      split::split8(v, h, m, l);
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        lo[i][n] = T::mma(l, b[n][0], lo[i][n]);
        lo[i][n] = T::mma(h, b[n][2], lo[i][n]);
        lo[i][n] = T::mma(m, b[n][1], lo[i][n]);
        lo[i][n] = T::mma(m, b[n][0], lo[i][n]);
        lo[i][n] = T::mma(h, b[n][1], lo[i][n]);
        hi[i][n] = T::mma(h, b[n][0], hi[i][n]);
      }
    }
  }
  float finite = 0.f;  // stays zero while every sum is
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      hi[i][n] = (hi[i][n] + lo[i][n]) * split::kUnscale;
#pragma unroll
      for (int r = 0; r < 4; ++r) finite = fmaf(hi[i][n][r], 0.f, finite);
    }
  if (finite != 0.f) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      f32x4 again[4] = {};
#pragma unroll 1
      for (int k = 0; k < a.rows; ++k) {
        const f32x4 p = four_of(a.P + (int64_t)k * a.cols, c0, a.cols);
        const f32x4 x = four_of(a.X + (int64_t)k * a.d, m0 + 16 * q + 4 * r, a.d);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int n = 0; n < 4; ++n) again[i][n] = fmaf(x[i], p[n], again[i][n]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int n = 0; n < 4; ++n)
          if (!__builtin_isfinite(hi[i][n][r])) hi[i][n][r] = again[i][n];
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = m0 + 16 * q + 4 * r + i;
      if (row >= a.d || c0 >= a.cols) continue;
      float* w = a.dW + (int64_t)row * a.lddw + c0;
      f32x4 v;
#pragma unroll
      for (int n = 0; n < 4; ++n) v[n] = hi[i][n][r];
      if (c0 + 3 < a.cols) {
        if (a.accumulate) v += *reinterpret_cast<const f32x4u*>(w);
        *reinterpret_cast<f32x4u*>(w) = v;
      } else {
#pragma unroll
        for (int n = 0; n < 4; ++n)
          if (c0 + n < a.cols) w[n] = a.accumulate ? w[n] + v[n] : v[n];
      }
    }
  if (!a.db || m0 > 0) return;
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    sum[n] += __shfl_xor(sum[n], 16, 64);
    sum[n] += __shfl_xor(sum[n], 32, 64);
    if (q == 0 && c0 + n < a.cols) a.db[c0 + n] = a.accumulate ? a.db[c0 + n] + sum[n] : sum[n];
  }
}

// ---------------------------------------------------------------- fp16 planes
using planes::Operand;
using S = planes::Shape<planes::Fp16, 2, 2, 2, 2>;  // 128 x 128 of C, two workgroups to a CU
constexpr int kTile = 128;
constexpr int kLo = 11;      // the second plane's scale against the first
constexpr int kTop = 15;     // scaled magnitudes are below 2^kTop
constexpr int kNone = -400;  // exponent of a feature that is zero everywhere
constexpr float kLog2e = 1.44269504088896340736f;

// ceil(log2) of the finite magnitudes seen: every one of them is below 2^this.
__device__ __forceinline__ int exponent_above(unsigned bits) {
  return bits == 0 ? kNone : max((int)(bits >> 23), 1) - 126;
}
__device__ __forceinline__ unsigned finite_bits(float x) {
  const unsigned b = __builtin_bit_cast(unsigned, x) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}

constexpr int kRowsAtOnce = 32768;  // rows of a chunk
constexpr int kSlabs = 64;          // of them, at most
constexpr int kFeatures = 4;        // of W to a workgroup,
constexpr int kChunk = 4 * NT;      // and columns

struct AmaxArgs {
  const float* X;
  int64_t ldx;
  const float* W;
  int64_t ldw;
  int rows, d, vocab, piece, chunks;  // chunks: of kChunk columns, per piece
  int slabs, slab_rows, xblocks;      // X: blocks of 256 columns x slabs
  const float* bias;
  unsigned* xpart;                    // [2][slabs][d]: of rows that take part, of the others
  unsigned* wpart;                    // [pieces][chunks][d]
  int padded, kblocks;                // rows: blocks of 256
  unsigned* done;                     // workgroups that have finished a later sum: 0
  const float* lse;                   // backward
  int* key;
  float* z;
};

// The largest finite magnitude of each feature: of X over slabs of rows, of W over
// chunks of a piece's columns (those that a bias of -infinity takes out left out:
// their weights may be anything).  And each row's id (-1: takes no part) with, for the
// backward, its log-sum; padded rows take no part.
__global__ __launch_bounds__(NT) void xent_amax_kernel(AmaxArgs a, Rows rows) {
  __shared__ unsigned red[kFeatures][NT / 64];
  __shared__ __attribute__((aligned(16))) unsigned part[2 * 4 * NT];
  const int tid = threadIdx.x;
  if ((int)blockIdx.x < a.kblocks) {
    const int r = blockIdx.x * NT + tid;
    if (r == 0) *a.done = 0;
    if (r >= a.padded) return;
    a.key[r] = r < a.rows ? rows.key(r) : -1;
    if (a.lse) a.z[r] = r < a.rows ? a.lse[r] : 0.f;
    return;
  }
  const int bx = blockIdx.x - a.kblocks;
  if (bx < a.xblocks) {
    // 256 features of a slab: four to a lane, a quarter of the rows to a wave
    const int tiles = (a.d + NT - 1) / NT, lane = tid & 63, wave = tid >> 6;
    const int slab = bx / tiles, k = (bx % tiles) * NT + 4 * lane;
    const int r0 = slab * a.slab_rows, n = min(a.rows - r0, a.slab_rows);
    const int at = min(k, max(a.d - 4, 0)), per = (n + 3) / 4, b1 = min(n, (wave + 1) * per);
    unsigned m[4] = {}, other[4] = {};
    for (int b0 = wave * per; b0 < b1; b0 += 64) {
      const unsigned long long live = __ballot(b0 + lane < b1 && rows.key(r0 + min(b0 + lane, n - 1)) >= 0);
      const float* x = a.X + (int64_t)(r0 + b0) * a.ldx + at;
      const int nb = min(b1 - b0, 64);
#pragma unroll 8
      for (int r = 0; r < nb; ++r) {
        f32x4 v;
        if (a.d >= 4) v = *reinterpret_cast<const f32x4u*>(x + (int64_t)r * a.ldx);
        else v = f32x4{x[(int64_t)r * a.ldx], x[(int64_t)r * a.ldx + min(1, a.d - 1)], x[(int64_t)r * a.ldx + min(2, a.d - 1)],
                       x[(int64_t)r * a.ldx + min(3, a.d - 1)]};
        const unsigned keep = (live >> r) & 1 ? 0xffffffffu : 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          m[j] = max(m[j], finite_bits(v[j]) & keep);
          other[j] = max(other[j], finite_bits(v[j]) & ~keep);
        }
      }
    }
    uint4* mine = reinterpret_cast<uint4*>(part) + tid;
    mine[0] = make_uint4(m[0], m[1], m[2], m[3]);
    mine[NT] = make_uint4(other[0], other[1], other[2], other[3]);
    __syncthreads();
    // thread c: feature c of the 256, its maxima over the waves
    const int f = (bx % tiles) * NT + tid;
    if (f >= a.d) return;
    // (at the matrix's end a lane holds the last four features)
    const int home = (tid >> 2) * 4 + (bx % tiles) * NT, shift = home - min(home, max(a.d - 4, 0)), j = (tid & 3) + shift;
    unsigned w = 0, o = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w = max(w, part[(64 * i + (tid >> 2)) * 4 + j]);
      o = max(o, part[4 * NT + (64 * i + (tid >> 2)) * 4 + j]);
    }
    a.xpart[(int64_t)slab * a.d + f] = w;
    a.xpart[(int64_t)(a.slabs + slab) * a.d + f] = o;
    return;
  }
  const int fblocks = (a.d + kFeatures - 1) / kFeatures, b = bx - a.xblocks;
  const int k0 = b % fblocks * kFeatures, c = b / fblocks;
  const int v0 = c / a.chunks * a.piece + c % a.chunks * kChunk;
  const int v1 = min(min(v0 + kChunk, (c / a.chunks + 1) * a.piece), a.vocab);
  unsigned m[kFeatures] = {};
  const float* w = a.W + (int64_t)k0 * a.ldw;
  const float* bias = a.bias ? a.bias : w;  // (loaded either way: a branch would part the loads)
#pragma unroll
  for (int i = 0; i < kChunk / NT; ++i) {
    const int v = min(v0 + i * NT + tid, v1 - 1);  // (the last column again past the end)
    const unsigned keep = ((bias[v] == -INFINITY) & (a.bias != nullptr)) ? 0u : 0xffffffffu;
#pragma unroll
    for (int f = 0; f < kFeatures; ++f)
      m[f] = max(m[f], finite_bits(w[(int64_t)min(f, a.d - 1 - k0) * a.ldw + v]) & keep);
  }
#pragma unroll
  for (int f = 0; f < kFeatures; ++f) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m[f] = max(m[f], (unsigned)__shfl_xor((int)m[f], o, 64));
    if ((tid & 63) == 0) red[f][tid >> 6] = m[f];
  }
  __syncthreads();
  if (tid < kFeatures && k0 + tid < a.d)
    a.wpart[(int64_t)c * a.d + k0 + tid] = max(max(red[tid][0], red[tid][1]), max(red[tid][2], red[tid][3]));
}

// Exponents: ex[k] of X; for piece p, el[p][k] of W in the logits, en[p][k] of W in dX,
// scale[p]: a logit is its sum times 2^scale.  A workgroup per piece.
//
// Rows that take no part have a log-sum too, but what they hold must not cost the
// others their bits: their values raise a feature's scale, and the piece's, by
// 2^kRoom at most.  (A row beyond that overflows, by itself.)
constexpr int kRoom = 12;
__global__ __launch_bounds__(1024) void xent_scales_kernel(AmaxArgs a, int* __restrict__ ex, int* __restrict__ el,
                                                           int* __restrict__ en, int* __restrict__ scale) {
  __shared__ int red[2][1024 / 64];
  const int p = blockIdx.x, tid = threadIdx.x;
  int top = 2 * kNone, all = 2 * kNone;
  for (int k = tid; k < a.d; k += 1024) {
    unsigned x = 0, o = 0, w = 0;
#pragma unroll 8
    for (int s = 0; s < a.slabs; ++s) {
      x = max(x, a.xpart[(int64_t)s * a.d + k]);
      o = max(o, a.xpart[(int64_t)(a.slabs + s) * a.d + k]);
    }
#pragma unroll 4
    for (int c = 0; c < a.chunks; ++c) w = max(w, a.wpart[((int64_t)p * a.chunks + c) * a.d + k]);
    const int live = exponent_above(x), other = exponent_above(o), lw = exponent_above(w);
    const int lx = live == kNone ? other : max(live, min(other, live + kRoom));
    if (p == 0) ex[k] = kTop - lx;
    en[(int64_t)p * a.d + k] = kTop - lw;
    el[(int64_t)p * a.d + k] = lx;  // completed below
    top = max(top, live == kNone ? 2 * kNone : live + lw);
    all = max(all, lx + lw);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    top = max(top, __shfl_xor(top, o, 64));
    all = max(all, __shfl_xor(all, o, 64));
  }
  if ((tid & 63) == 0) {
    red[0][tid >> 6] = top;
    red[1][tid >> 6] = all;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 1024 / 64; ++i) {
    top = max(top, red[0][i]);
    all = max(all, red[1][i]);
  }
  top = top == 2 * kNone ? all : max(top, min(all, top + kRoom));
  // (a feature that only those rows have stays below 2^kTop on W's side too)
  for (int k = tid; k < a.d; k += 1024)
    el[(int64_t)p * a.d + k] = min(el[(int64_t)p * a.d + k] + kTop - top, en[(int64_t)p * a.d + k]);
  if (tid == 0) scale[p] = top - 2 * kTop;
}

// X as the logits' first operand and, in the backward, as dW's; a piece of W as the
// logits' second and dX's.  Blocks of each, in that order.
struct PackAll {
  planes::PackArgs xl, xt, wl, wn;
  unsigned nxl, nxt, nwl, nwn;
};
__global__ __launch_bounds__(256) void xent_pack_kernel(PackAll a) {
  unsigned b = blockIdx.x;
  if (b < a.nxl) return planes::pack_rows<true, kLo>(a.xl, b);
  b -= a.nxl;
  if (b < a.nxt) return planes::pack_cols<false, kLo>(a.xt, b);
  b -= a.nxt;
  if (b < a.nwl) return planes::pack_cols<true, kLo>(a.wl, b);
  planes::pack_rows<false, kLo>(a.wn, b - a.nwl);
}

struct TileArgs {
  Operand A, B;
  int nk, gx, gy;
  int cols, v0;         // columns of the piece, its first id
  const float* bias;    // the piece's, or null
  const int* scale;
  const int* key;
  int64_t padded;       // rows
  int64_t pcols;        // padded columns of the piece
  float2* part;         // forward: [64-column block][padded rows] maximum, sum of exp
  float* target;
  const float* lse;     // backward
  char* prow;           // P packed for dX (rows, k = columns)
  char* pcol;           // and for dW (columns, k = rows)
  float* cfac;          // [64-row block][pcols] what a column's sum over the block is scaled back by
  float* csum;          // [64-row block][all columns] column sums of P, the piece's first
  int64_t all;
};

// The sum or maximum over the 16 lanes of a row.
template <int CTRL>
__device__ __forceinline__ float rotated(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ float row_max(float x) {
  x = fmaxf(x, rotated<0x128>(x));
  x = fmaxf(x, rotated<0x124>(x));
  x = fmaxf(x, rotated<0x122>(x));
  return fmaxf(x, rotated<0x121>(x));
}
__device__ __forceinline__ float row_add(float x) {
  x += rotated<0x128>(x);
  x += rotated<0x124>(x);
  x += rotated<0x122>(x);
  return x + rotated<0x121>(x);
}

// A tile of logits, and from them the rows' statistics or P.  Bound by the products' loop,
// matrix cores 54 and 46 % busy at 2.03-2.1 GHz (128 x 128 tiles keep two workgroups of
// 64 KB to a CU, so that one's epilogue runs beside the other's products): 8192 x 1024 ->
// 4096 182 us with the statistics, 1.13 PFLOP/s of 16 bits; 208 us with P, whose two
// packed copies are 268 MB written.
// Exponentials are the hardware's, exp2 of the logit less its maximum or log-sum, times
// log2 e: that product's rounding is no larger than the difference's own.
template <bool GRAD>
__global__ __launch_bounds__(S::NTH, 2) void xent_tile_kernel(TileArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[S::LDS];
  const planes::Lane<S> w;
  int tm, tn, z;
  gemm::item_tile(blockIdx.x, a.gx * a.gy, a.gx, a.gy, tm, tn, z);
  f32x4 l[4][4], lo[4][4];
  planes::multiply<S>(a.A, a.B, tm, tn, 0, a.nk, lds, w, l, lo);

  const int64_t row0 = (int64_t)tm * kTile + 64 * w.wm + 16 * w.q;  // this lane's rows row0 + 4 r + i
  const int c0 = tn * kTile + w.col();                              // and columns c0 + n
  const int sc = a.scale[0];
  float bias[4];
#pragma unroll
  for (int n = 0; n < 4; ++n) bias[n] = a.bias && c0 + n < a.cols ? a.bias[c0 + n] : 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        l[i][n][r] = __builtin_ldexpf(fmaf(lo[i][n][r], 1.f / (1 << kLo), l[i][n][r]), sc) + bias[n];
  int key[4][4];  // [r][i]: this lane's column of the row's id, if 0 .. 3
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int4 k = *reinterpret_cast<const int4*>(a.key + row0 + 4 * r);
    key[r][0] = k.x;
    key[r][1] = k.y;
    key[r][2] = k.z;
    key[r][3] = k.w;
  }
  const int v = a.v0 + c0;

  if (!GRAD) {
    float m_mine = 0.f, s_mine = 0.f;  // of row row0 + lr
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = key[r][i] - v;
#pragma unroll
        for (int n = 0; n < 4; ++n)
          if (c == n && key[r][i] >= 0) a.target[row0 + 4 * r + i] = l[i][n][r];
        float x[4], m = -FLT_MAX, s = 0.f;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          x[n] = c0 + n < a.cols ? l[i][n][r] : -INFINITY;
          m = fmaxf(m, x[n]);
        }
        m = row_max(m);
#pragma unroll
        for (int n = 0; n < 4; ++n) s += __builtin_amdgcn_exp2f((x[n] - m) * kLog2e);
        s = row_add(s);
        if (w.lr == 4 * r + i) {
          m_mine = m;
          s_mine = s;
        }
      }
    a.part[(int64_t)(tn * 2 + w.wn) * a.padded + row0 + w.lr] = make_float2(m_mine, s_mine);
    return;
  }

  float cmax[4] = {0.f, 0.f, 0.f, 0.f}, csum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const f32x4 z4 = *reinterpret_cast<const f32x4*>(a.lse + row0 + 4 * r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = key[r][i] - v;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        float p = __builtin_amdgcn_exp2f((l[i][n][r] - z4[i]) * kLog2e);
        if (c == n) p -= 1.f;
        p = key[r][i] >= 0 && c0 + n < a.cols ? p : 0.f;
        l[i][n][r] = p;
        cmax[n] = fmaxf(cmax[n], fabsf(p));
        csum[n] += p;
      }
    }
  }
  int ec[4];  // exponents of the columns over these 64 rows
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    cmax[n] = fmaxf(cmax[n], __shfl_xor(cmax[n], 16, 64));
    cmax[n] = fmaxf(cmax[n], __shfl_xor(cmax[n], 32, 64));
    csum[n] += __shfl_xor(csum[n], 16, 64);
    csum[n] += __shfl_xor(csum[n], 32, 64);
    ec[n] = min(kTop - exponent_above(__builtin_bit_cast(unsigned, cmax[n])), 126);
  }
  if (w.q == 0) {
    const int64_t blk = (int64_t)tm * 2 + w.wm;
    f32x4 f;
#pragma unroll
    for (int n = 0; n < 4; ++n) f[n] = __builtin_bit_cast(float, (unsigned)(127 - ec[n]) << 23);
    *reinterpret_cast<f32x4*>(a.cfac + blk * a.pcols + c0) = f;
    *reinterpret_cast<f32x4*>(a.csum + blk * a.all + c0) = f32x4{csum[0], csum[1], csum[2], csum[3]};
  }
  // by column: this lane has 16 consecutive rows of each of its columns
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = __builtin_ldexpf(l[j & 3][n][2 * h + (j >> 2)], ec[n]);
      planes::put16<kLo>(a.pcol + planes::chunk_at<2>(a.pcols / 16, c0 + n, row0 + 8 * h), x);
    }
  // by row: lanes 2 j and 2 j + 1 have 8 consecutive columns together; the even one
  // takes rows i = 0, 1, the odd one 2, 3.  Rows lie in a block by 4 r + q here (q + 4 r
  // elsewhere), so that the four lane groups write 64 contiguous bytes; dX's rows
  // come out accordingly.
  const bool odd = w.lr & 1;
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float x[8];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const float own = odd ? l[2 + j][n][r] : l[j][n][r], give = odd ? l[j][n][r] : l[2 + j][n][r];
        const float got = rotated<0xB1>(give);  // the other lane of the pair
        x[n] = (odd ? got : own) * (float)(1 << kTop);
        x[4 + n] = (odd ? own : got) * (float)(1 << kTop);
      }
      const int64_t row = (int64_t)tm * kTile + 64 * w.wm + 16 * r + 4 * w.q + (odd ? 2 + j : j);
      planes::put16<kLo>(a.prow + planes::chunk_at<2>(a.padded / 16, row, c0 & ~7), x);
    }
}

// lse and the row losses from the blocks' statistics, 64 rows to a workgroup whose
// waves take every 16th block, and the sum of the workgroup's row losses; the
// workgroup that finishes last adds those up, in order.
__global__ __launch_bounds__(1024) void xent_join_kernel(const float2* __restrict__ part, int blocks, int64_t padded, int nrows,
                                                         const float* __restrict__ target, const int* __restrict__ key,
                                                         float* __restrict__ lse, float* __restrict__ row_loss,
                                                         double* __restrict__ sums, unsigned* __restrict__ done, float scale,
                                                         float* __restrict__ loss, int add) {
  __shared__ float2 red[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int r = blockIdx.x * 64 + lane;  // (< padded)
  float m = -FLT_MAX, s = 0.f;
  for (int b0 = w; b0 < blocks; b0 += 128) {
    float2 x[8];
    float top = m;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = b0 + 16 * j < blocks ? part[(int64_t)(b0 + 16 * j) * padded + r] : make_float2(-FLT_MAX, 0.f);
      top = fmaxf(top, x[j].x);
    }
    s *= expf(m - top);
#pragma unroll
    for (int j = 0; j < 8; ++j) s += x[j].y * expf(x[j].x - top);
    m = top;
  }
  red[w][lane] = make_float2(m, s);
  __syncthreads();
  if (w != 0) return;
#pragma unroll
  for (int j = 1; j < 16; ++j) m = fmaxf(m, red[j][lane].x);
  s = 0.f;
#pragma unroll
  for (int j = 0; j < 16; ++j) s += red[j][lane].y * expf(red[j][lane].x - m);
  const float z = m + logf(s);
  double one = 0.0;
  if (r < nrows) {
    const float v = key[r] >= 0 ? z - target[r] : 0.f;
    lse[r] = z;
    if (row_loss) row_loss[r] = v;
    one = (double)v;
  }
  one = wave_sum(one);
  unsigned before = 0;
  if (lane == 0) {
    __hip_atomic_store(&sums[blockIdx.x], one, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    before = __hip_atomic_fetch_add(done, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (__shfl(before, 0, 64) + 1 != gridDim.x) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  double total = 0.0;
  for (unsigned i = lane; i < gridDim.x; i += 64)
    total += __hip_atomic_load(&sums[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  total = wave_sum(total);
  if (lane == 0) loss[0] = (float)(total * (double)scale) + (add ? loss[0] : 0.f);
}

// What finishes a product: C (+)= 2^(exponent of its row or column) g sum.
struct OutArgs {
  float* C;
  int64_t ldc;
  int rows, cols, accumulate;
  const int* ex;
  int ex_by_row, add;  // the exponent is add - ex[row or column]
  float scale;
  const float* upstream;
  __device__ __forceinline__ float g() const { return upstream ? upstream[0] * scale : scale; }
  // Columns col .. col + 3 of a row (those of the matrix).
  __device__ __forceinline__ void put(int64_t row, int col, f32x4 v, float gg) const {
    if (row >= rows || col >= cols) return;
    float* p = C + row * ldc + col;
#pragma unroll
    for (int n = 0; n < 4; ++n) v[n] = __builtin_ldexpf(v[n], add - ex[ex_by_row ? row : min(col + n, cols - 1)]) * gg;
    if (col + 3 < cols) {
      if (accumulate) v += *reinterpret_cast<const f32x4u*>(p);
      *reinterpret_cast<f32x4u*>(p) = v;
    } else {
#pragma unroll
      for (int n = 0; n < 4; ++n)
        if (col + n < cols) p[n] = accumulate ? p[n] + v[n] : v[n];
    }
  }
};

struct ProductArgs {
  Operand A, B;
  int nk, gx, gy, splits, per;  // stages; per split
  int items;                    // workgroups
  const float* cfac;            // dW: [64-row block][pcols]
  int64_t pcols;
  OutArgs out;
  float* part;                  // [split][padded rows][padded cols] where splits > 1
};

// COLS false: dX = P W^T, whose rows lie in their blocks as the tile kernel left
// them.  true: dW = X^T P, whose sums over each 64 rows (two stages) are joined and scaled
// back column by column (192 sums to a lane, 244 registers; all three cross entropy
// sizes of 1000 rows and more take 2 % longer than with one sum for both planes,
// which needs them on one scale).
template <bool COLS>
__device__ __forceinline__ void xent_product(const ProductArgs& a, int item, char* lds) {
  const planes::Lane<S> w;
  int tm, tn, z;
  gemm::item_tile(item, a.items, a.gx, a.gy, tm, tn, z);
  const int k0 = z * a.per, k1 = min(a.nk, k0 + a.per);
  f32x4 sum[4][4], hi[4][4], lo[4][4];
  if (COLS) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int n = 0; n < 4; ++n) sum[i][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    const float* fac = a.cfac + (int64_t)tn * kTile + w.col();
    f32x4 f;
    planes::multiply_runs<S>(
        a.A, a.B, tm, tn, k0, k1, 2, lds, w, hi, lo,
        [&](int k) { f = *reinterpret_cast<const f32x4*>(fac + (int64_t)(k >> 1) * a.pcols); },
        [&]() {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int n = 0; n < 4; ++n) sum[i][n] += f[n] * (hi[i][n] + lo[i][n] * (1.f / (1 << kLo)));
        });
  } else {
    planes::multiply<S>(a.A, a.B, tm, tn, k0, k1, lds, w, sum, lo);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int n = 0; n < 4; ++n) sum[i][n] += lo[i][n] * (1.f / (1 << kLo));
  }
  const int64_t row0 = (int64_t)tm * kTile + 64 * w.wm + (COLS ? 16 : 4) * w.q;
  const int c0 = tn * kTile + w.col();
  auto row_of = [&](int r, int i) { return row0 + (COLS ? 4 : 16) * r + i; };
  auto value = [&](int r, int i) { return f32x4{sum[i][0][r], sum[i][1][r], sum[i][2][r], sum[i][3][r]}; };
  if (a.splits > 1) {
    const int64_t ld = (int64_t)a.gx * kTile;
    float* p = a.part + (int64_t)z * a.gy * kTile * ld + c0;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<f32x4*>(p + row_of(r, i) * ld) = value(r, i);
    return;
  }
  // (OutArgs::put, with every load on its way before the first store; past the last row
  // that row again)
  const OutArgs& o = a.out;
  const float g = o.g();
  const bool whole = c0 + 3 < o.cols;
  int e[4][4];
  f32x4 old[4][4];
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t row = min(row_of(r, i), (int64_t)o.rows - 1);
      e[r][i] = COLS ? o.ex[row] : o.ex[min(c0 + i, o.cols - 1)];  // of the row, or of column c0 + i
      old[r][i] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (o.accumulate && whole) old[r][i] = *reinterpret_cast<const f32x4u*>(o.C + row * o.ldc + c0);
    }
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t row = row_of(r, i);
      f32x4 v = value(r, i);
#pragma unroll
      for (int n = 0; n < 4; ++n) v[n] = __builtin_ldexpf(v[n], o.add - (COLS ? e[r][i] : e[0][n])) * g;
      if (row >= o.rows) continue;
      float* p = o.C + row * o.ldc + c0;
      if (whole) {
        *reinterpret_cast<f32x4u*>(p) = o.accumulate ? v + old[r][i] : v;
      } else {
#pragma unroll
        for (int n = 0; n < 4; ++n)
          if (c0 + n < o.cols) p[n] = o.accumulate ? p[n] + v[n] : v[n];
      }
    }
}

// Both products of a piece in one launch, dW's items first (they are the longer
// ones, or equal), so that the chip stays full to the end of the second.  Bound by the
// products' loop (matrix cores 53 % busy at 2.05 GHz): 8192 x 1024 -> 4096 375 us, 1.10
// PFLOP/s of 16 bits; with the loads of dX's old values and of the exponents ahead of
// the stores all eight pieces take 2 % less.
__global__ __launch_bounds__(S::NTH, 2) void xent_products_kernel(ProductArgs w, ProductArgs x, int start) {
  __shared__ __attribute__((aligned(16))) char lds[S::LDS];
  const int b = blockIdx.x;
  if (b < w.items) xent_product<true>(w, b, lds);
  else if (b >= start) xent_product<false>(x, b - start, lds);
}

// The splits' sums in order: blocks [0, nw) of dW, then nx of dX.  The rest, after the
// last piece: db (+)= g times the 64-row blocks' column sums, 64 columns to a
// workgroup, whose waves take every fourth block; their sums in order.
__device__ __forceinline__ void xent_reduce(const ProductArgs& a, unsigned block, unsigned blocks) {
  const int64_t ld = (int64_t)a.gx * kTile, total = (int64_t)a.out.rows * (ld / 4), step = (int64_t)a.gy * kTile * ld;
  const float g = a.out.g();
  for (int64_t u = (int64_t)block * NT + threadIdx.x; u < total; u += (int64_t)blocks * NT) {
    const int64_t row = u / (ld / 4);
    const int col = (int)(u - row * (ld / 4)) * 4;
    if (col >= a.out.cols) continue;
    const float* p = a.part + row * ld + col;
    f32x4 s = *reinterpret_cast<const f32x4*>(p);
#pragma unroll 4
    for (int z = 1; z < a.splits; ++z) s += *reinterpret_cast<const f32x4*>(p + z * step);
    a.out.put(row, col, s, g);
  }
}
struct BiasArgs {
  const float* csum;
  int blocks, vocab, accumulate;
  int64_t all;
  float* db;
  float scale;
  const float* upstream;
};
__global__ __launch_bounds__(NT) void xent_reduce_kernel(ProductArgs w, unsigned nw, ProductArgs x, unsigned nx, BiasArgs a) {
  __shared__ float red[4][64];
  const unsigned block = blockIdx.x;
  if (block < nw) return xent_reduce(w, block, nw);
  if (block < nw + nx) return xent_reduce(x, block - nw, nx);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = (int)(block - nw - nx) * 64 + lane;
  float s = 0.f;
  if (c < a.vocab) {
#pragma unroll 8
    for (int b = wave; b < a.blocks; b += 4) s += a.csum[(int64_t)b * a.all + c];
  }
  red[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || c >= a.vocab) return;
  s = ((red[0][lane] + red[1][lane]) + red[2][lane]) + red[3][lane];
  s *= a.upstream ? a.upstream[0] * a.scale : a.scale;
  a.db[c] = a.accumulate ? a.db[c] + s : s;
}

constexpr int kMost = 1 << 30;  // rows, d, vocab
size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

// ----------------------------------------------------------------------- plans
// Few logits: columns of a piece, and the workspace's parts.
struct SmallPlan {
  int piece;
  size_t logits, rows, state, slices, gemm;  // bytes
  size_t total() const { return logits + rows + state + slices + gemm; }
};
constexpr size_t kPieceBytes = (size_t)128 << 20;
// dX of few rows and features over up to 4096 columns is a product that the library
// leaves to one workgroup per 16 x 16 of it; it is cut into slices of about 1024
// columns (64 x 256 over 4096: 18 -> 10.3 us with their sum).
int dx_slices(int rows, int d, int n) {
  const int64_t tiles = (int64_t)((rows + 15) / 16) * ((d + 15) / 16);
  return n >= 1536 && n <= 4096 && tiles <= 128 ? (n + 1023) / 1024 : 1;
}
SmallPlan small_plan(int rows, int d, int vocab) {
  SmallPlan p;
  const size_t cols = kPieceBytes / sizeof(float) / (size_t)rows / 256 * 256;
  p.piece = (int)std::min<size_t>((size_t)vocab, std::max<size_t>(cols, 256));
  p.logits = round256((size_t)rows * p.piece * sizeof(float));
  p.rows = round256((size_t)rows * d * sizeof(float));
  p.state = round256((size_t)rows * sizeof(RowState));
  const int last = vocab % p.piece ? vocab % p.piece : p.piece;
  p.gemm = p.slices = 0;
  for (int v : {p.piece, last}) {
    const int n = dx_slices(rows, d, v);
    if (n > 1) p.slices = std::max(p.slices, round256((size_t)n * rows * d * sizeof(float)));
    p.gemm = std::max(p.gemm, std::max(mle_gemm_ws_bytes(rows, v, d, 1),
                                       std::max(mle_gemm_ws_bytes(rows, d, v, 1), mle_gemm_ws_bytes(d, v, rows, 1))));
  }
  if (p.piece == vocab) p.gemm = std::max(p.gemm, mle_linear_bwd_ws_bytes(rows, d, vocab, 1));
  p.gemm = round256(p.gemm);
  return p;
}

// Where the products of fp16 planes run: from 192 rows (a tile and a half) and a size
// whose faster products pay for three launches more and two passes over the operands.
// Measured at both, forward and backward, planes against stored pieces, us:
//   small  256 x 256 -> 4096 82 / 67, 1000 x 128 -> 1000 76 / 48, 512 x 1024 -> 2000
//          131 / 109, 512 x 256 -> 4096 89 / 86, 1000 x 64 -> 2500 79 / 71
//   large  1000 x 512 -> 2000 106 / 124, 512 x 1024 -> 4096 147 / 161, 1000 x 64 ->
//          4000 81 / 87, 512 x 512 -> 8000 124 / 156, 8192 x 256 -> 1000 136 / 174
//   rows   128 x 512 -> 32000 215 / 181, 256 x 64 -> 16000 81 / 79
bool use_planes(int rows, int d, int vocab) {
  return rows >= 192 && (double)rows * vocab * (900.0 + d) >= 2.8e9;
}

// Few logits: where dW's own kernel runs, a stage or two of rows and tiles enough to hide
// its loads (both sides, forward and backward, own kernel / library product, us: 32 x
// 876 -> 26839 156 / 191, 64 x 1023 -> 32001 204 / 243, 1 x 512 -> 32000 102 / 116; 95 x
// 800 -> 7067 94 / 96, 191 x 1024 -> 16000 245 / 235, 64 x 256 -> 4096 46 / 42).
bool short_dw(int rows, int d, int n) {
  const int64_t tiles = ((int64_t)d + 127) / 128 * (((int64_t)n + 127) / 128);
  return rows <= 64 && tiles >= 512 && tiles < (1 << 23);
}

// The two products of a piece share a grid of two workgroups to a CU.  A product
// whose workgroups would each take more than 5/4 of a CU slot's share of the
// stages has its K split, into at least 16 stages each (an even number: the column
// factors cover two).
struct Split {
  int splits, per;
};
Split split_of(int stages, int64_t share) {
  int n = (int)std::max<int64_t>(1, std::min<int64_t>((stages + share * 5 / 4 - 1) / std::max<int64_t>(share * 5 / 4, 1), stages / 16));
  const int per = ((stages + n - 1) / n + 1) / 2 * 2;
  return Split{(stages + per - 1) / per, per};
}
struct PairSplit {
  Split w, x;
  size_t wbytes, xbytes;  // of partial sums
};
PairSplit pair_split(int padded, int dp, int pcols, bool has_w, bool has_x) {
  const int64_t tw = has_w ? (int64_t)(dp / kTile) * (pcols / kTile) : 0, tx = has_x ? (int64_t)(padded / kTile) * (dp / kTile) : 0;
  const int sw = padded / 32, sx = pcols / 32;
  const int64_t share = (tw * sw + tx * sx + 2 * gemm::kChipCus - 1) / (2 * gemm::kChipCus);
  PairSplit p{split_of(sw, share), split_of(sx, share), 0, 0};
  if (has_w && p.w.splits > 1) p.wbytes = (size_t)p.w.splits * dp * pcols * 4;
  if (has_x && p.x.splits > 1) p.xbytes = (size_t)p.x.splits * padded * dp * 4;
  return p;
}

// The planes' plan: rows are taken kRowsAtOnce at a time (rows of a chunk, padded to
// whole tiles), the vocabulary in pieces that keep both packed P within
// kPlaneBytes.
constexpr size_t kPlaneBytes = (size_t)256 << 20;
struct PlanePlan {
  int rows, d, vocab;
  int padded, dk, dp, piece, pieces, chunks, slabs, slab_rows;
  // offsets into the workspace
  size_t xpart, wpart, ex, el, en, scale, key, z, target, sums, done, xl, wl;
  size_t part;                                         // forward
  size_t xt, wn, prow, pcol, cfac, csum, wsplit, xsplit;  // backward, at the same place
  size_t total;
};
PlanePlan plane_plan(int all_rows, int d, int vocab) {
  PlanePlan p;
  p.rows = std::min(all_rows, kRowsAtOnce);
  p.d = d;
  p.vocab = vocab;
  p.padded = (p.rows + kTile - 1) / kTile * kTile;
  p.dk = (d + 31) / 32;
  p.dp = (d + kTile - 1) / kTile * kTile;
  const int64_t most = std::max<int64_t>(kTile, (int64_t)(kPlaneBytes / 8 / p.padded) / kTile * kTile);
  p.pieces = (int)((vocab + most - 1) / most);
  p.piece = ((vocab + p.pieces - 1) / p.pieces + kTile - 1) / kTile * kTile;
  p.pieces = (vocab + p.piece - 1) / p.piece;
  p.chunks = (p.piece + kChunk - 1) / kChunk;
  p.slabs = std::min(kSlabs, (p.rows + 31) / 32);
  p.slab_rows = (p.rows + p.slabs - 1) / p.slabs;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += round256(bytes);
    return o;
  };
  const size_t padded = p.padded, piece = p.piece, all = (size_t)p.pieces * p.piece;
  p.xpart = take((size_t)2 * p.slabs * d * 4);
  p.wpart = take((size_t)p.pieces * p.chunks * d * 4);
  p.ex = take((size_t)d * 4);
  p.el = take((size_t)p.pieces * d * 4);
  p.en = take((size_t)p.pieces * d * 4);
  p.scale = take((size_t)p.pieces * 4);
  p.key = take(padded * 4);
  p.z = take(padded * 4);
  p.target = take(padded * 4);
  p.sums = take(padded / 64 * 8);
  p.done = take(4);
  p.xl = take(padded * p.dk * 32 * 4);
  p.wl = take(piece * p.dk * 32 * 4);
  const size_t both = at;
  p.part = take(padded * (all / 64) * sizeof(float2));
  const size_t fwd = at;
  at = both;
  p.xt = take(padded * p.dp * 4);
  p.wn = take(piece * p.dp * 4);
  p.prow = take(padded * piece * 4);
  p.pcol = take(padded * piece * 4);
  p.cfac = take(padded / 64 * piece * 4);
  p.csum = take(padded / 64 * all * 4);
  // partial sums, whichever products a call has and of whichever piece and chunk
  const int last_cols = (int)(vocab - (size_t)(p.pieces - 1) * piece + kTile - 1) / kTile * kTile;
  const int last_rows = ((all_rows - 1) % p.rows + kTile) / kTile * kTile;
  size_t wbytes = 0, xbytes = 0;
  for (int cols : {p.piece, last_cols})
    for (int rows : {p.padded, last_rows})
      for (int has : {1, 2, 3}) {
        const PairSplit s = pair_split(rows, p.dp, cols, has & 1, has & 2);
        wbytes = std::max(wbytes, s.wbytes);
        xbytes = std::max(xbytes, s.xbytes);
      }
  p.wsplit = take(wbytes);
  p.xsplit = take(xbytes);
  p.total = std::max(at, fwd);
  return p;
}

int check(const char* who, int rows, int d, int vocab, const float* X, int64_t ldx, const float* W, int64_t ldw,
          const int32_t* keys, int clen, int max_clen) {
  MLE_CHECK_ARG(rows >= 0 && d > 0 && vocab > 0 && rows <= kMost && d <= kMost && vocab <= kMost, "%s: bad shape (rows %d, d %d, vocab %d)", who, rows, d, vocab);
  MLE_CHECK_ARG(W && (rows == 0 || (X && keys)), "%s: null pointer", who);
  MLE_CHECK_ARG(ldx >= d && ldw >= vocab, "%s: ldx %lld < %d or ldw %lld < %d", who, (long long)ldx, d, (long long)ldw,
                vocab);
  MLE_CHECK_ARG(clen > 0 && max_clen >= clen, "%s: clen %d, max_clen %d", who, clen, max_clen);
  return MLE_OK;
}
// The planes' launches number (feature, chunk of columns) pairs in 31 bits.
int check_planes(const char* who, int rows, int d, int vocab) {
  if (rows <= 0 || !use_planes(rows, d, vocab)) return MLE_OK;
  const PlanePlan p = plane_plan(rows, d, vocab);
  if ((double)p.pieces * p.chunks * d >= 1073741824.0 || p.dk > (1 << 26))
    return set_error(MLE_ERR_UNSUPPORTED, "%s: d %d with a vocabulary of %d is too large", who, d, vocab);
  return MLE_OK;
}
int check_ws(const char* who, size_t need, const void* ws, size_t ws_bytes) {
  if (need && (!ws || !aligned16(ws) || ws_bytes < need))
    return set_error(MLE_ERR_WORKSPACE, "%s: workspace of %zu bytes, 16-byte aligned, needed", who, need);
  return MLE_OK;
}

size_t ws_need(int rows, int d, int vocab) {
  return use_planes(rows, d, vocab) ? plane_plan(rows, d, vocab).total : small_plan(rows, d, vocab).total();
}

#define TRY(call)                  \
  do {                             \
    const int rc_ = (call);        \
    if (rc_ != MLE_OK) return rc_; \
  } while (0)

// The part of a call that the planes' forward and backward share: exponents, ids and
// X for the logits, over one chunk of rows.
struct Chunk {
  PlanePlan p;
  char* ws;
  hipStream_t s;
  const float* X;
  int64_t ldx;
  const float* W;
  int64_t ldw;
  const float* bias;
  int rows, padded;
  template <class T = char>
  T* at(size_t o) const {
    return reinterpret_cast<T*>(ws + o);
  }

  // Exponents and ids.
  void begin(const Rows& rw, const float* lse) const {
    AmaxArgs a{};
    a.X = X;
    a.ldx = ldx;
    a.W = W;
    a.ldw = ldw;
    a.rows = rows;
    a.d = p.d;
    a.vocab = p.vocab;
    a.piece = p.piece;
    a.chunks = p.chunks;
    a.slabs = p.slabs;
    a.slab_rows = p.slab_rows;
    a.xblocks = (p.d + NT - 1) / NT * p.slabs;
    a.xpart = at<unsigned>(p.xpart);
    a.wpart = at<unsigned>(p.wpart);
    a.padded = padded;
    a.kblocks = (padded + NT - 1) / NT;
    a.bias = bias;
    a.done = at<unsigned>(p.done);
    a.lse = lse;
    a.key = at<int>(p.key);
    a.z = at<float>(p.z);
    mle::launch(xent_amax_kernel, (unsigned)(a.kblocks + a.xblocks + p.pieces * p.chunks * ((p.d + kFeatures - 1) / kFeatures)), NT, 0, s, a, rw);
    mle::launch(xent_scales_kernel, (unsigned)p.pieces, 1024, 0, s, a, at<int>(p.ex), at<int>(p.el), at<int>(p.en), at<int>(p.scale));
  }
  int cols(int i) const { return std::min(p.piece, p.vocab - i * p.piece); }
  int pcols(int i) const { return (cols(i) + kTile - 1) / kTile * kTile; }
  // Piece i of W for the logits, and for dX where `inputs`; with the first piece, X for
  // the logits, and for dW where `weights`.
  void pack(int i, bool inputs, bool weights) const {
    const float* w = W + (int64_t)i * p.piece;
    const float* b = bias ? bias + (int64_t)i * p.piece : nullptr;
    PackAll a{{X, ldx, rows, p.d, padded / 16, p.dk, at<int>(p.ex), nullptr, nullptr, at(p.xl)},
              {X, ldx, p.d, rows, p.dp / 16, padded / 32, at<int>(p.ex), at<int>(p.key), nullptr, at(p.xt)},
              {w, ldw, cols(i), p.d, pcols(i) / 16, p.dk, at<int>(p.el) + (int64_t)i * p.d, nullptr, b, at(p.wl)},
              {w, ldw, p.d, cols(i), p.dp / 16, pcols(i) / 32, at<int>(p.en) + (int64_t)i * p.d, nullptr, b, at(p.wn)},
              0, 0, 0, 0};
    a.nxl = i == 0 ? (unsigned)a.xl.rows_blocks() : 0u;
    a.nxt = i == 0 && weights ? (unsigned)a.xt.cols_blocks() : 0u;
    a.nwl = (unsigned)a.wl.cols_blocks();
    a.nwn = inputs ? (unsigned)a.wn.rows_blocks() : 0u;
    mle::launch(xent_pack_kernel, a.nxl + a.nxt + a.nwl + a.nwn, 256, 0, s, a);
  }
  Operand operand(size_t o, int padded_rows) const { return Operand{at(o), (int64_t)padded_rows / 16 * 2 * planes::kUnit}; }
  TileArgs tile(int i) const {
    TileArgs a{};
    a.A = operand(p.xl, padded);
    a.B = operand(p.wl, pcols(i));
    a.nk = p.dk;
    a.gx = pcols(i) / kTile;
    a.gy = padded / kTile;
    a.cols = cols(i);
    a.v0 = i * p.piece;
    a.bias = bias ? bias + a.v0 : nullptr;
    a.scale = at<int>(p.scale) + i;
    a.key = at<int>(p.key);
    a.padded = padded;
    a.pcols = pcols(i);
    return a;
  }
  // The products of piece i, and what finishes them; a null matrix leaves its product
  // out, a null db the bias gradient.
  void products(int i, OutArgs ow, OutArgs ox, const BiasArgs& bias_grad) const {
    const PairSplit ps = pair_split(padded, p.dp, pcols(i), ow.C != nullptr, ox.C != nullptr);
    auto product = [&](Operand A, Operand B, int stages, int gx, int gy, Split sp, const OutArgs& out, size_t part) {
      ProductArgs a{};
      a.A = A;
      a.B = B;
      a.nk = stages;
      a.gx = gx;
      a.gy = gy;
      a.splits = sp.splits;
      a.per = sp.per;
      a.items = out.C ? gx * gy * sp.splits : 0;
      a.cfac = at<float>(p.cfac);
      a.pcols = pcols(i);
      a.out = out;
      a.part = at<float>(part);
      return a;
    };
    const ProductArgs w = product(operand(p.xt, p.dp), operand(p.pcol, pcols(i)), padded / 32, pcols(i) / kTile, p.dp / kTile,
                                  ps.w, ow, p.wsplit);
    const ProductArgs x = product(operand(p.prow, padded), operand(p.wn, p.dp), pcols(i) / 32, p.dp / kTile, padded / kTile,
                                  ps.x, ox, p.xsplit);
    const int start = (w.items + gemm::kXcds - 1) / gemm::kXcds * gemm::kXcds;  // (item 0 of dX on XCD 0 again)
    mle::launch(xent_products_kernel, (unsigned)(start + x.items), S::NTH, 0, s, w, x, start);
    auto blocks = [](const ProductArgs& a) {
      return a.items && a.splits > 1 ? stream_grid((size_t)a.out.rows * a.gx * (kTile / 4), NT, 4096) : 0u;
    };
    const unsigned nw = blocks(w), nx = blocks(x), nb = bias_grad.db ? (unsigned)((bias_grad.vocab + 63) / 64) : 0u;
    if (nw + nx + nb) mle::launch(xent_reduce_kernel, nw + nx + nb, NT, 0, s, w, nw, x, nx, bias_grad);
  }
};

// Rows [r0, ..) of a call.
Chunk chunk_of(const PlanePlan& p, void* ws, hipStream_t s, int r0, int all_rows, const float* X, int64_t ldx,
               const float* W, int64_t ldw, const float* bias) {
  const int rows = std::min(p.rows, all_rows - r0);
  return Chunk{p, static_cast<char*>(ws), s, X + (int64_t)r0 * ldx, ldx, W, ldw, bias, rows, (rows + kTile - 1) / kTile * kTile};
}

int planes_fwd(mle_stream stream, int rows, int d, int vocab, const float* X, int64_t ldx, const float* W, int64_t ldw,
               const float* bias, Rows rw, float loss_scale, float* lse, float* row_loss, float* loss, void* ws) {
  const PlanePlan p = plane_plan(rows, d, vocab);
  hipStream_t s = as_stream(stream);
  for (int r0 = 0; r0 < rows; r0 += p.rows) {
    const Chunk c = chunk_of(p, ws, s, r0, rows, X, ldx, W, ldw, bias);
    rw.r0 = r0;
    c.begin(rw, nullptr);
    int blocks = 0;
    for (int i = 0; i < p.pieces; ++i) {
      c.pack(i, false, false);
      TileArgs a = c.tile(i);
      a.part = c.at<float2>(p.part) + (int64_t)blocks * c.padded;
      a.target = c.at<float>(p.target);
      mle::launch(xent_tile_kernel<false>, (unsigned)(a.gx * a.gy), S::NTH, 0, s, a);
      blocks += 2 * a.gx;
    }
    const int groups = c.padded / 64;
    mle::launch(xent_join_kernel, (unsigned)groups, 1024, 0, s, c.at<float2>(p.part), blocks, (int64_t)c.padded, c.rows,
                c.at<float>(p.target), c.at<int>(p.key), lse + r0, row_loss ? row_loss + r0 : nullptr, c.at<double>(p.sums),
                c.at<unsigned>(p.done), loss_scale, loss, r0 > 0 ? 1 : 0);
  }
  return check_launch("mle_vocab_xent_fwd");
}

int planes_bwd(mle_stream stream, int rows, int d, int vocab, const float* X, int64_t ldx, const float* W, int64_t ldw,
               const float* bias, Rows rw, const float* lse, const float* upstream, float grad_scale, float* dX,
               int64_t lddx, int accumulate_dx, float* dW, int64_t lddw, float* db, int accumulate_dw, void* ws) {
  const PlanePlan p = plane_plan(rows, d, vocab);
  hipStream_t s = as_stream(stream);
  for (int r0 = 0; r0 < rows; r0 += p.rows) {
    const Chunk c = chunk_of(p, ws, s, r0, rows, X, ldx, W, ldw, bias);
    rw.r0 = r0;
    c.begin(rw, lse + r0);
    const int add = accumulate_dw || r0 > 0;
    const int64_t all = (int64_t)p.pieces * p.piece;
    for (int i = 0; i < p.pieces; ++i) {
      const int64_t v0 = (int64_t)i * p.piece;
      c.pack(i, dX != nullptr, dW != nullptr);
      TileArgs a = c.tile(i);
      a.lse = c.at<float>(p.z);
      a.prow = c.at(p.prow);
      a.pcol = c.at(p.pcol);
      a.cfac = c.at<float>(p.cfac);
      a.csum = c.at<float>(p.csum) + v0;
      a.all = all;
      mle::launch(xent_tile_kernel<true>, (unsigned)(a.gx * a.gy), S::NTH, 0, s, a);
      OutArgs ow{}, ox{};
      if (dW) ow = OutArgs{dW + v0, lddw, d, c.cols(i), add, c.at<int>(p.ex), 1, 0, grad_scale, upstream};
      if (dX)
        ox = OutArgs{dX + (int64_t)r0 * lddx, lddx, c.rows, d, accumulate_dx || i > 0, c.at<int>(p.en) + (int64_t)i * d, 0, -kTop,
                     grad_scale, upstream};
      BiasArgs bias_grad{};
      if (db && i == p.pieces - 1)
        bias_grad = BiasArgs{c.at<float>(p.csum), c.padded / 64, vocab, add, all, db, grad_scale, upstream};
      c.products(i, ow, ox, bias_grad);
    }
  }
  return check_launch("mle_vocab_xent_bwd");
}

}  // namespace

extern "C" {

size_t mle_vocab_xent_ws_bytes(int rows, int d, int vocab) {
  return rows <= 0 || d <= 0 || vocab <= 0 || rows > kMost || d > kMost || vocab > kMost ? 0 : ws_need(rows, d, vocab);
}

int mle_vocab_xent_fwd(mle_stream stream, int rows, int d, int vocab, const float* X, int64_t ldx, const float* W,
                       int64_t ldw, const float* bias, const int32_t* keys, int clen, int max_clen, float loss_scale,
                       float* lse, float* row_loss, float* loss, void* ws, size_t ws_bytes) {
  TRY(check("mle_vocab_xent_fwd", rows, d, vocab, X, ldx, W, ldw, keys, clen, max_clen));
  MLE_CHECK_ARG(loss && (lse || rows == 0), "mle_vocab_xent_fwd: null pointer");
  if (rows == 0) return mle_fill(stream, loss, 0.f, 1);
  TRY(check_planes("mle_vocab_xent_fwd", rows, d, vocab));
  TRY(check_ws("mle_vocab_xent_fwd", ws_need(rows, d, vocab), ws, ws_bytes));
  if (use_planes(rows, d, vocab))
    return planes_fwd(stream, rows, d, vocab, X, ldx, W, ldw, bias, Rows{keys, clen, max_clen, vocab, 0}, loss_scale, lse,
                      row_loss, loss, ws);
  const SmallPlan p = small_plan(rows, d, vocab);
  hipStream_t s = as_stream(stream);
  const Rows rw{keys, clen, max_clen, vocab, 0};
  float* l = static_cast<float*>(ws);
  RowState* state = reinterpret_cast<RowState*>(static_cast<char*>(ws) + p.logits + p.rows);
  void* gws = reinterpret_cast<char*>(state) + p.state + p.slices;
  for (int v0 = 0; v0 < vocab; v0 += p.piece) {
    const int n = std::min(p.piece, vocab - v0), first = v0 == 0 ? 1 : 0;
    const float* b = bias ? bias + v0 : nullptr;
    TRY(mle_gemm_ex(stream, 0, 0, rows, n, d, 1.f, X, ldx, 0, W + v0, ldw, 0, 0.f, l, n, 0, 1, nullptr, b, gws, p.gemm));
    // (with many rows a wave to each is enough to fill the chip)
    if (n <= 1024 || rows >= 2048)
      mle::launch(xent_stats_kernel<64>, (unsigned)(((int64_t)rows + 3) / 4), NT, 0, s, l, rows, n, v0, b, rw, state, first);
    else mle::launch(xent_stats_kernel<1024>, (unsigned)rows, 1024, 0, s, l, rows, n, v0, b, rw, state, first);
  }
  mle::launch(xent_finish_kernel, 1u, 1024, 0, s, state, rows, rw, loss_scale, lse, row_loss, loss, 0);
  return check_launch("mle_vocab_xent_fwd");
}

int mle_vocab_xent_bwd(mle_stream stream, int rows, int d, int vocab, const float* X, int64_t ldx, const float* W,
                       int64_t ldw, const float* bias, const int32_t* keys, int clen, int max_clen, const float* lse,
                       const float* upstream, float grad_scale, float* dX, int64_t lddx, int accumulate_dx, float* dW,
                       int64_t lddw, float* db, int accumulate_dw, void* ws, size_t ws_bytes) {
  TRY(check("mle_vocab_xent_bwd", rows, d, vocab, X, ldx, W, ldw, keys, clen, max_clen));
  MLE_CHECK_ARG((lse || rows == 0) && (!dX || lddx >= d) && (!dW || lddw >= vocab),
                "mle_vocab_xent_bwd: null pointer, or lddx %lld < %d or lddw %lld < %d", (long long)lddx, d,
                (long long)lddw, vocab);
  MLE_CHECK_ARG(dW || !db, "mle_vocab_xent_bwd: db without dW");
  TRY(check_planes("mle_vocab_xent_bwd", rows, d, vocab));
  if (rows > 0) TRY(check_ws("mle_vocab_xent_bwd", ws_need(rows, d, vocab), ws, ws_bytes));
  if (rows > 0 && use_planes(rows, d, vocab))
    return !dX && !dW ? MLE_OK
                      : planes_bwd(stream, rows, d, vocab, X, ldx, W, ldw, bias, Rows{keys, clen, max_clen, vocab, 0}, lse,
                                   upstream, grad_scale, dX, lddx, accumulate_dx, dW, lddw, db, accumulate_dw, ws);
  if (rows == 0) {
    if (db && !accumulate_dw) TRY(mle_fill(stream, db, 0.f, (size_t)vocab));
    if (dW && !accumulate_dw)
      TRY(mle_gemm_ex(stream, 1, 0, d, vocab, 0, 1.f, nullptr, d, 0, nullptr, vocab, 0, 0.f, dW, lddw, 0, 1, nullptr, nullptr,
                      nullptr, 0));
    return MLE_OK;
  }
  if (!dX && !dW) return MLE_OK;
  const SmallPlan p = small_plan(rows, d, vocab);
  hipStream_t s = as_stream(stream);
  const Rows rw{keys, clen, max_clen, vocab, 0};
  float* l = static_cast<float*>(ws);
  float* xs = reinterpret_cast<float*>(static_cast<char*>(ws) + p.logits);
  float* part = reinterpret_cast<float*>(static_cast<char*>(ws) + p.logits + p.rows + p.state);
  void* gws = reinterpret_cast<char*>(part) + p.slices;
  // The Linear backward's own launches where its matrices are dense.
  const bool own_dw = dW && short_dw(rows, d, p.piece);
  const bool dense = dX && dW && !own_dw && p.piece == vocab && dx_slices(rows, d, vocab) == 1 && ldw == vocab && lddw == vocab && lddx == d;
  for (int v0 = 0; v0 < vocab; v0 += p.piece) {
    const int n = std::min(p.piece, vocab - v0), slices = dX ? dx_slices(rows, d, n) : 1;
    auto groups = [&](int cols) { return (unsigned)(((int64_t)rows * cols + 4 * NT - 1) / (4 * NT)); };
    TRY(mle_gemm_ex(stream, 0, 0, rows, n, d, 1.f, X, ldx, 0, W + v0, ldw, 0, 0.f, l, n, 0, 1, nullptr,
                    bias ? bias + v0 : nullptr, gws, p.gemm));
    mle::launch(xent_grad_kernel, groups(n) + (dW && v0 == 0 ? groups(d) : 0u), NT, 0, s, l, rows, n, v0, rw, lse, upstream,
                grad_scale, groups(n), X, ldx, d, xs, db && !accumulate_dw && !dense && !own_dw ? db : nullptr, bias ? bias + v0 : nullptr);
    if (dense) {
      TRY(mle_linear_bwd_ex(stream, rows, d, vocab, 1, xs, l, 0, W, 0, dX, accumulate_dx, dW, db, 0, accumulate_dw, gws, p.gemm));
      break;
    }
    const int acc = accumulate_dx || v0 > 0;
    if (slices > 1) {
      const int q = n / slices / 4 * 4;
      const int64_t total = (int64_t)rows * d;
      TRY(mle_gemm_ex(stream, 0, 1, rows, d, q, 1.f, l, n, q, W + v0, ldw, q, 0.f, part, d, total, slices, nullptr, nullptr, gws,
                      p.gemm));
      mle::launch(xent_slices_kernel, (unsigned)((total + NT - 1) / NT), NT, 0, s, part, slices, total, d, l, n, slices * q,
                  W + v0, ldw, dX, lddx, acc);
    } else if (dX) {
      TRY(mle_gemm_ex(stream, 0, 1, rows, d, n, 1.f, l, n, 0, W + v0, ldw, 0, acc ? 1.f : 0.f, dX, lddx, 0, 1,
                      nullptr, nullptr, gws, p.gemm));
    }
    if (own_dw) {
      const DwArgs a{xs, l, rows, d, n, (n + 127) / 128, (d + 127) / 128, accumulate_dw, dW + v0, lddw, db ? db + v0 : nullptr};
      mle::launch(xent_dw_kernel, (unsigned)(a.gx * a.gy), NT, 0, s, a);
    } else if (dW) {
      TRY(mle_gemm_ex(stream, 1, 0, d, n, rows, 1.f, xs, d, 0, l, n, 0, accumulate_dw ? 1.f : 0.f, dW + v0, lddw, 0, 1,
                      db ? db + v0 : nullptr, nullptr, gws, p.gemm));
    }
  }
  return check_launch("mle_vocab_xent_bwd");
}

}  // extern "C"
