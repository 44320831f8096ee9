// The residual Add and the layer norm that reads it, with a learned weight and
// bias, and the backward of both.
//
//   h = x + r,  u = (h - mean) rstd,  rstd = 1 / sqrt(mean of (h - mean)^2 + eps),  y = u w + b
//   g = dy w:  dh = dres + rstd (g - mean(g) - u mean(g u)),  dw = sum over rows of dy u,  db = sum of dy
//
// One pass over a row: T lanes of a wave, or a workgroup of T threads, hold it
// in registers, eight consecutive values to a thread and chunk.  The variance is
// that of the centred values, so a mean far above the spread costs no bits; the
// row's sums are in 64 bits.  The backward, which has the mean in 32 bits, takes what
// that lacks from the row (rest_of).  The weight's and the bias's gradients are summed per
// workgroup in registers and joined in order.  Bound by memory, each tensor passed once: 16384 x
// 4096 take 204 us forward (5.3 TB/s) and 213 + 7.5 us backward (5.0 TB/s), 8192 x 512 with
// three launches 35 us in all, 64 x 256 3.8 + 4.7 us.
#include "q8.hpp"

#include <algorithm>

using namespace mle;

namespace {

constexpr int NT = 256;
constexpr int kMaxParts = 512;          // partial weight gradients: workgroups of the backward
constexpr int kFewRows = 256;           // up to which the backward is one launch
constexpr int kRestRows = 8;            // of a workgroup of layernorm_rest_kernel
constexpr int kWidest = 8192;           // columns of a row in registers
constexpr int kColsOfJoin = 1 << 25;    // of a launch of 64 threads to a column: fewer than 2^32 threads
constexpr int kRowsOfLaunch = 1 << 21;  // of a launch of one workgroup to a row: fewer than 2^32 threads

struct LnArgs {
  int rows, cols;
  const float* x;
  const float* r;
  const float* w;
  const float* b;
  float* h;
  float* y;
  float* mean;
  float* rstd;
  float eps;
};

struct LnBwdArgs {
  int rows, cols;
  const float* h;
  const float* w;
  const float* mean;
  const float* rstd;
  const float* dy;
  const float* dres;
  float* dh;
  int acc_dh;
  float* part;  // [workgroups][2][cols], dw's and db's; null: neither
};

// The sums of a and b over a row's T threads, in every one of them.
template <int T>
__device__ __forceinline__ double2 row_sums(double a, double b, double (*red)[2]) {
#pragma unroll
  for (int o = (T < 64 ? T : 64) / 2; o > 0; o >>= 1) {
    a += __shfl_xor(a, o, 64);
    b += __shfl_xor(b, o, 64);
  }
  if (T <= 64) return make_double2(a, b);
  __syncthreads();  // the last sums have been read
  if ((threadIdx.x & 63) == 0) {
    red[threadIdx.x >> 6][0] = a;
    red[threadIdx.x >> 6][1] = b;
  }
  __syncthreads();
  a = b = 0.0;
#pragma unroll
  for (int i = 0; i < T / 64; ++i) {
    a += red[i][0];
    b += red[i][1];
  }
  return make_double2(a, b);
}

// The backward's u = ((h - mean) - rest) rstd.  The mean's rounding moves u by at most 2^-24 |mean|
// rstd; below 2^-22 that is left (rest 0, exactly), above it the rest of the mean is the mean of
// h - mean, which costs such a row one sum more.
__device__ __forceinline__ bool is_far(float mean, float rstd) { return fabsf(mean) * rstd > 4.f; }

// That sum: eight consecutive differences in 32 bits (exact in rows far enough from zero, 3 roundings of
// them in others), these in 64 and rounded to 2^-27 of the mean's power of two 2^k.  A far row's differences
// add up to less than cols 2^(k - 1), so that up to 2^27 columns every sum of such is exact: the same
// in any order, whatever the kernel's form.
struct Rest {
  float mean;
  double grid;  // adding it leaves what is above 2^(k - 27)
  double sum = 0.0;
  __device__ __forceinline__ explicit Rest(float m) : mean(m) {
    const int k = (int)((__builtin_bit_cast(unsigned, m) >> 23) & 255u) - 127;
    grid = ldexp(1.5, k - 27 + 52);
  }
  // The first n of eight values (none where n is below 1).
  __device__ __forceinline__ void add(const float (&h)[8], int n) {
    float d[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) d[j] = j < n ? h[j] - mean : 0.f;
    sum += ((double)(((d[0] + d[1]) + (d[2] + d[3])) + ((d[4] + d[5]) + (d[6] + d[7]))) + grid) - grid;
  }
};

__device__ __forceinline__ void load_sum8(const LnArgs& a, int64_t at, int n, float (&h)[8]) {
  q8::load_row8(a.x + at, n, h);
  if (a.r) {
    float r[8];
    q8::load_row8(a.r + at, n, r);
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] += r[j];
  }
}

// T threads to a row, C chunks of 8 values each (T * 8 * C >= cols); C == 0: any
// width, the row read three times.
template <int T, int C>
__global__ __launch_bounds__(T < NT ? NT : T) void layernorm_fwd_kernel(LnArgs a) {
  constexpr int B = T < NT ? NT : T, R = B / T;  // rows of a workgroup
  __shared__ double red[B / 64][2];
  const int t = threadIdx.x % T;
  const int64_t row = (int64_t)blockIdx.x * R + threadIdx.x / T;
  if (row >= a.rows) return;  // (T < B: whole waves; T == B: the workgroup)
  const int64_t base = row * a.cols;
  const int chunks = C > 0 ? C : (a.cols + 8 * T - 1) / (8 * T);
  float keep[C > 0 ? C : 1][8];
  double s = 0.0;
#pragma unroll C > 0 ? C : 1
  for (int c = 0; c < chunks; ++c) {
    float(&h)[8] = keep[C > 0 ? c : 0];
    const int col = (c * T + t) * 8, n = min(max(a.cols - col, 0), 8);
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = 0.f;
    if (n == 0) continue;
    load_sum8(a, base + col, n, h);
#pragma unroll
    for (int j = 0; j < 8; ++j) s += (double)h[j];
  }
  const double mean = row_sums<T>(s, 0.0, red).x / a.cols;
  s = 0.0;
#pragma unroll C > 0 ? C : 1
  for (int c = 0; c < chunks; ++c) {
    float(&h)[8] = keep[C > 0 ? c : 0];
    const int col = (c * T + t) * 8, n = min(max(a.cols - col, 0), 8);
    if (n == 0) continue;
    if (C == 0) load_sum8(a, base + col, n, h);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float d = (float)((double)h[j] - mean);
      s += j < n ? (double)d * (double)d : 0.0;
    }
  }
  const double rstd = 1.0 / sqrt(row_sums<T>(s, 0.0, red).x / a.cols + (double)a.eps);
  if (t == 0) {
    a.mean[row] = (float)mean;
    a.rstd[row] = (float)rstd;
  }
#pragma unroll C > 0 ? C : 1
  for (int c = 0; c < chunks; ++c) {
    float(&h)[8] = keep[C > 0 ? c : 0];
    const int col = (c * T + t) * 8, n = min(max(a.cols - col, 0), 8);
    if (n == 0) continue;
    if (C == 0) load_sum8(a, base + col, n, h);
    if (a.h) q8::store_row8(a.h + base + col, h, n);
    if (!a.y) continue;
    float w[8], b[8], y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = 1.f, b[j] = 0.f;
    if (a.w) q8::load_row8(a.w + col, n, w);
    if (a.b) q8::load_row8(a.b + col, n, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = fmaf((float)(((double)h[j] - mean) * rstd), w[j], b[j]);
    q8::store_row8(a.y + base + col, y, n);
  }
}

// Workgroup `block` takes rows block * R + i * blocks * R and keeps its
// threads' columns of dw and db in registers; the R rows that it walks at a time
// add theirs through LDS at the end.
template <int T, int C>
__device__ __forceinline__ void bwd_rows(const LnBwdArgs& a, int block, int blocks) {
  constexpr int B = T < NT ? NT : T, R = B / T;
  __shared__ double red[B / 64][2];
  __shared__ float cols_red[R > 1 ? 8 * B : 1];
  const int t = threadIdx.x % T, k = threadIdx.x / T;
  float dw[C][8], db[C][8], w[C][8];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int col = (c * T + t) * 8, n = min(max(a.cols - col, 0), 8);
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[c][j] = db[c][j] = 0.f, w[c][j] = 1.f;
    if (a.w && n > 0) q8::load_row8(a.w + col, n, w[c]);
  }
  for (int64_t r0 = (int64_t)block * R; r0 < a.rows; r0 += (int64_t)blocks * R) {
    const int64_t row = r0 + k;
    const bool live = row < a.rows;
    const int64_t base = (live ? row : a.rows - 1) * a.cols;
    const float rstd = live ? a.rstd[row] : 0.f, mean = live ? a.mean[row] : 0.f;
    float u[C][8], g[C][8], rest = 0.f;
    double s1 = 0.0, s2 = 0.0;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * T + t) * 8, n = live ? min(max(a.cols - col, 0), 8) : 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) u[c][j] = g[c][j] = 0.f;
      if (n == 0) continue;
      q8::load_row8(a.h + base + col, n, u[c]);
      q8::load_row8(a.dy + base + col, n, g[c]);  // (0 past the row's end, whatever u is there)
    }
    if (is_far(mean, rstd)) {  // (the same for all of a row's threads)
      Rest r(mean);
#pragma unroll
      for (int c = 0; c < C; ++c) r.add(u[c], a.cols - (c * T + t) * 8);
      rest = (float)(row_sums<T>(r.sum, 0.0, red).x / a.cols);
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * T + t) * 8, n = live ? min(max(a.cols - col, 0), 8) : 0;
      if (n == 0) continue;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        u[c][j] = ((u[c][j] - mean) - rest) * rstd;
        dw[c][j] += g[c][j] * u[c][j];
        db[c][j] += g[c][j];
        g[c][j] *= w[c][j];
        s1 += (double)g[c][j];
        s2 += (double)(g[c][j] * u[c][j]);
      }
    }
    const double2 m = row_sums<T>(s1, s2, red);
    const float m1 = (float)(m.x / a.cols), m2 = (float)(m.y / a.cols);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * T + t) * 8, n = live ? min(max(a.cols - col, 0), 8) : 0;
      if (n == 0) continue;
      float old[8] = {}, dres[8] = {}, v[8];
      if (a.dres) q8::load_row8(a.dres + base + col, n, dres);
      if (a.acc_dh) q8::load_row8(a.dh + base + col, n, old);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = old[j] + (dres[j] + rstd * ((g[c][j] - m1) - u[c][j] * m2));
      q8::store_row8(a.dh + base + col, v, n);
    }
  }
  if (!a.part) return;
  float* part = a.part + (int64_t)block * 2 * a.cols;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    float(&sum)[C][8] = p ? db : dw;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * T + t) * 8, n = min(max(a.cols - col, 0), 8);
      if (R > 1) {  // the rows' sums in order
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) cols_red[8 * threadIdx.x + j] = sum[c][j];
        __syncthreads();
        if (k > 0) continue;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          for (int i = 1; i < R; ++i) sum[c][j] += cols_red[8 * (i * T + t) + j];
      }
      if (n > 0) q8::store_row8(part + (int64_t)p * a.cols + col, sum[c], n);
    }
  }
}

template <int T, int C>
__global__ __launch_bounds__(T < NT ? NT : T) void layernorm_bwd_kernel(LnBwdArgs a) {
  bwd_rows<T, C>(a, blockIdx.x, gridDim.x);
}

// A column's sum from those of up to 64 groups of rows in LDS, red[group][column of 16], by 64
// threads: a quarter of the groups to each of four lanes, then the quarters; in lane `column`.
__device__ __forceinline__ float join64(const float (*red)[17]) {
  const int c = threadIdx.x & 15, q = threadIdx.x >> 4;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) s += red[16 * q + i][c];
  const float x0 = __shfl(s, c, 64), x1 = __shfl(s, 16 + c, 64), x2 = __shfl(s, 32 + c, 64), x3 = __shfl(s, 48 + c, 64);
  return ((x0 + x1) + x2) + x3;
}

// Few rows, where launches are the time (256 x 512: 5.0 us against 7.2 in two, 64 x 256: 4.1 against
// 6.1): both in one launch, the first `row_blocks` workgroups the rows and the others 16
// columns of dw and db each, from dy and h once more; the same additions as in two launches.  Where
// rows are far from zero each of these workgroups needs their rests, so all of h: 64 x 256 of only
// such rows 7.8 us, 256 x 512 22, 256 x 2048 43 (and 6.0 of none).
template <int T, int C>
__global__ __launch_bounds__(NT) void layernorm_bwd_small_kernel(LnBwdArgs a, float* __restrict__ dw, float* __restrict__ db,
                                                                 int accumulate, int row_blocks) {
  if ((int)blockIdx.x < row_blocks) {
    bwd_rows<T, C>(a, blockIdx.x, row_blocks);
    return;
  }
  __shared__ float red[2][64][17];
  __shared__ float rest[NT];
  __shared__ int some[NT / 64];
  static_assert(kFewRows <= NT, "a row to a thread");
  const int any = __any((int)threadIdx.x < a.rows && is_far(a.mean[threadIdx.x], a.rstd[threadIdx.x]));
  if ((threadIdx.x & 63) == 0) some[threadIdx.x >> 6] = any;
  const int c = threadIdx.x & 15, col = ((int)blockIdx.x - row_blocks) * 16 + c;
  const auto sums = [&](bool with_rest) {
    for (int g = threadIdx.x >> 4; g < 64; g += NT / 16) {
      float u[4], d[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
#pragma clang fp contract(off)
        const int r = 4 * g + k;
        const bool there = r < a.rows && col < a.cols;
        const int64_t at = there ? (int64_t)r * a.cols + col : 0;
        const int row = there ? r : 0;
        d[k] = there ? a.dy[at] : 0.f;
        const float h = a.h[at] - a.mean[row];
        u[k] = there ? d[k] * ((with_rest ? h - rest[row] : h) * a.rstd[row]) : 0.f;
      }
      red[0][g][c] = ((u[0] + u[1]) + u[2]) + u[3];
      red[1][g][c] = ((d[0] + d[1]) + d[2]) + d[3];
    }
  };
  sums(false);
  __syncthreads();
  if (some[0] | some[1] | some[2] | some[3]) {  // once more with the rests of such rows: 16 lanes to four rows
    const int lane = threadIdx.x & 15;
    for (int r0 = threadIdx.x >> 4; r0 < a.rows; r0 += NT / 4) {
      Rest v[4] = {Rest(a.mean[r0]), Rest(a.mean[min(r0 + 16, a.rows - 1)]), Rest(a.mean[min(r0 + 32, a.rows - 1)]),
                   Rest(a.mean[min(r0 + 48, a.rows - 1)])};
#pragma unroll 2
      for (int at = 8 * lane; at < a.cols; at += 128) {
        const int n = min(a.cols - at, 8);
        float h[4][8];
#pragma unroll
        for (int k = 0; k < 4; ++k) q8::load_row8(a.h + (int64_t)min(r0 + 16 * k, a.rows - 1) * a.cols + at, n, h[k]);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k].add(h[k], n);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) v[k].sum += __shfl_xor(v[k].sum, o, 64);
        const int r = r0 + 16 * k;
        if (lane == 0 && r < a.rows) rest[r] = is_far(v[k].mean, a.rstd[r]) ? (float)(v[k].sum / a.cols) : 0.f;
      }
    }
    __syncthreads();
    sums(true);
    __syncthreads();
  }
  if (threadIdx.x >= 64) return;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float* out = k ? db : dw;
    const float v = join64(red[k]);
    if (out && threadIdx.x < 16 && col < a.cols) out[col] = accumulate ? out[col] + v : v;
  }
}

// The rest of a row's mean, 0 of a row that is not far; by a workgroup of 1024.
__device__ __forceinline__ float rest_of(const LnBwdArgs& a, int64_t row, float mean, float rstd, double (*red)[2]) {
  if (!is_far(mean, rstd)) return 0.f;
  Rest v(mean);
  for (int at = 8 * threadIdx.x; at < a.cols; at += 8192) {
    float h[8];
    const int n = min(a.cols - at, 8);
    q8::load_row8(a.h + row * a.cols + at, n, h);
    v.add(h, n);
  }
  return (float)(row_sums<1024>(v.sum, 0.0, red).x / a.cols);
}
__global__ __launch_bounds__(1024) void layernorm_rest_kernel(LnBwdArgs a, float* __restrict__ rest) {
  __shared__ double red[16][2];
  const int64_t r0 = (int64_t)blockIdx.x * kRestRows;
#pragma unroll
  for (int k = 0; k < kRestRows; ++k) {
    if (r0 + k >= a.rows) return;  // (the workgroup)
    const float v = rest_of(a, r0 + k, a.mean[r0 + k], a.rstd[r0 + k], red);
    if (threadIdx.x == 0) rest[r0 + k] = v;
  }
}

// Rows wider than the register kernels take: h and dy read twice; the weight's and the
// bias's gradients in a pass of their own (layernorm_dw_kernel).
__global__ __launch_bounds__(1024) void layernorm_bwd_wide_kernel(LnBwdArgs a, const float* __restrict__ rests) {
  __shared__ double red[16][2];
  const int64_t base = (int64_t)blockIdx.x * a.cols;
  const float rstd = a.rstd[blockIdx.x], mean = a.mean[blockIdx.x];
  const float rest = rests ? rests[blockIdx.x] : rest_of(a, blockIdx.x, mean, rstd, red);
  double s1 = 0.0, s2 = 0.0;
  for (int i = threadIdx.x; i < a.cols; i += 1024) {
    const float g = a.dy[base + i] * (a.w ? a.w[i] : 1.f), u = ((a.h[base + i] - mean) - rest) * rstd;
    s1 += (double)g;
    s2 += (double)(g * u);
  }
  const double2 m = row_sums<1024>(s1, s2, red);
  const float m1 = (float)(m.x / a.cols), m2 = (float)(m.y / a.cols);
  for (int i = threadIdx.x; i < a.cols; i += 1024) {
    const float g = a.dy[base + i] * (a.w ? a.w[i] : 1.f), u = ((a.h[base + i] - mean) - rest) * rstd;
    const float v = (a.dres ? a.dres[base + i] : 0.f) + rstd * ((g - m1) - u * m2);
    a.dh[base + i] = (a.acc_dh ? a.dh[base + i] : 0.f) + v;
  }
}
// part[block y][.][col] = sums over rows y, y + gridDim.y, ...
__global__ __launch_bounds__(NT) void layernorm_dw_kernel(LnBwdArgs a, const float* __restrict__ rest) {
  const int col = blockIdx.x * NT + threadIdx.x;
  if (col >= a.cols) return;
  float s = 0.f, b = 0.f;
  for (int64_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
    const float dy = a.dy[r * a.cols + col];
    s += dy * (((a.h[r * a.cols + col] - a.mean[r]) - rest[r]) * a.rstd[r]);
    b += dy;
  }
  float* part = a.part + (int64_t)blockIdx.y * 2 * a.cols;
  part[col] = s;
  part[a.cols + col] = b;
}

// dw (+)= and db (+)= the partial sums: 16 columns of one of them to a workgroup, 64
// threads to a column, each adding every 64th part, and the threads' sums in order.  From
// column col0 on.
__global__ __launch_bounds__(1024) void layernorm_join_kernel(const float* __restrict__ part, int parts, int cols, int col0,
                                                              float* __restrict__ dw, float* __restrict__ db,
                                                              int accumulate) {
  __shared__ float red[64][17];
  float* out = blockIdx.y ? db : dw;
  if (!out) return;
  const int c = threadIdx.x & 15, g = threadIdx.x >> 4;
  const int col = col0 + (int)blockIdx.x * 16 + c;
  float s = 0.f;
  if (col < cols) {
#pragma unroll 8
    for (int p = g; p < parts; p += 64) s += part[((int64_t)p * 2 + blockIdx.y) * cols + col];
  }
  red[g][c] = s;
  __syncthreads();
  if (threadIdx.x >= 64) return;
  const float v = join64(red);
  if (threadIdx.x < 16 && col < cols) out[col] = accumulate ? out[col] + v : v;
}

// Workgroups of the backward, each with partial gradients: a function of the shape alone.
int parts_of(int rows, int cols) {
  const int rows_of_wg = cols <= 2048 ? 4 : 1;
  return std::max(1, std::min(kMaxParts, (rows - 1) / rows_of_wg + 1));
}

size_t parts_floats(int rows, int cols) { return (size_t)parts_of(rows, cols) * 2 * cols; }

int check(const char* who, int rows, int cols) {
  MLE_CHECK_ARG(rows >= 0 && cols > 0 && cols <= (1 << 30), "%s: bad shape %d x %d", who, rows, cols);
  return MLE_OK;
}

}  // namespace

extern "C" {

int mle_add_layernorm_fwd(mle_stream stream, int rows, int cols, const float* x, const float* r, const float* w,
                          const float* b, float eps, float* h, float* y, float* mean, float* rstd) {
  const int rc = check("mle_add_layernorm_fwd", rows, cols);
  if (rc) return rc;
  MLE_CHECK_ARG(rows == 0 || (x && mean && rstd), "mle_add_layernorm_fwd: null pointer");
  MLE_CHECK_ARG(eps >= 0.f, "mle_add_layernorm_fwd: eps %g", (double)eps);
  if (rows == 0) return MLE_OK;
  hipStream_t s = as_stream(stream);
  for (int64_t r0 = 0; r0 < rows; r0 += kRowsOfLaunch) {
    const int n = (int)std::min<int64_t>(rows - r0, kRowsOfLaunch);
    const int64_t at = r0 * cols;
    const LnArgs a{n, cols, x + at, r ? r + at : r, w, b, h ? h + at : h, y ? y + at : y, mean + r0, rstd + r0, eps};
    const unsigned by4 = (unsigned)((n + 3) / 4);
    if (cols <= 512) mle::launch(layernorm_fwd_kernel<64, 1>, by4, NT, 0, s, a);
    else if (cols <= 1024) mle::launch(layernorm_fwd_kernel<64, 2>, by4, NT, 0, s, a);
    else if (cols <= 2048) mle::launch(layernorm_fwd_kernel<64, 4>, by4, NT, 0, s, a);
    else if (cols <= 4096) mle::launch(layernorm_fwd_kernel<256, 2>, (unsigned)n, NT, 0, s, a);
    else if (cols <= kWidest) mle::launch(layernorm_fwd_kernel<256, 4>, (unsigned)n, NT, 0, s, a);
    else mle::launch(layernorm_fwd_kernel<1024, 0>, (unsigned)n, 1024, 0, s, a);
  }
  return check_launch("mle_add_layernorm_fwd");
}

size_t mle_add_layernorm_ws_bytes(int rows, int cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return (parts_floats(rows, cols) + (cols > kWidest ? rows : 0)) * sizeof(float);  // (there, the rests of the means)
}

int mle_add_layernorm_bwd(mle_stream stream, int rows, int cols, const float* h, const float* w, const float* mean,
                          const float* rstd, const float* dy, const float* dres, float* dh, int accumulate_dh,
                          float* dw, float* db, int accumulate_dw, void* ws, size_t ws_bytes) {
  const int rc = check("mle_add_layernorm_bwd", rows, cols);
  if (rc) return rc;
  MLE_CHECK_ARG(rows == 0 || (h && mean && rstd && dy && dh), "mle_add_layernorm_bwd: null pointer");
  if (rows == 0) {
    if (accumulate_dw) return MLE_OK;
    if (dw) {
      const int e = mle_fill(stream, dw, 0.f, (size_t)cols);
      if (e) return e;
    }
    return db ? mle_fill(stream, db, 0.f, (size_t)cols) : MLE_OK;
  }
  const bool sums = dw || db;
  if (sums && (!ws || !aligned16(ws) || ws_bytes < mle_add_layernorm_ws_bytes(rows, cols)))
    return set_error(MLE_ERR_WORKSPACE, "mle_add_layernorm_bwd: workspace of %zu bytes, 16-byte aligned, needed",
                     mle_add_layernorm_ws_bytes(rows, cols));
  const int parts = parts_of(rows, cols);
  LnBwdArgs a{rows, cols, h, w, mean, rstd, dy, dres, dh, accumulate_dh, sums ? static_cast<float*>(ws) : nullptr};
  hipStream_t s = as_stream(stream);
  if (sums && rows <= kFewRows && cols <= 2048 && dh != dy && dh != h) {
    a.part = nullptr;
    const unsigned grid = (unsigned)(parts + (cols + 15) / 16);
    if (cols <= 512) mle::launch(layernorm_bwd_small_kernel<64, 1>, grid, NT, 0, s, a, dw, db, accumulate_dw, parts);
    else if (cols <= 1024) mle::launch(layernorm_bwd_small_kernel<64, 2>, grid, NT, 0, s, a, dw, db, accumulate_dw, parts);
    else mle::launch(layernorm_bwd_small_kernel<64, 4>, grid, NT, 0, s, a, dw, db, accumulate_dw, parts);
    return check_launch("mle_add_layernorm_bwd");
  }
  if (cols <= 512) mle::launch(layernorm_bwd_kernel<64, 1>, (unsigned)parts, NT, 0, s, a);
  else if (cols <= 1024) mle::launch(layernorm_bwd_kernel<64, 2>, (unsigned)parts, NT, 0, s, a);
  else if (cols <= 2048) mle::launch(layernorm_bwd_kernel<64, 4>, (unsigned)parts, NT, 0, s, a);
  else if (cols <= 4096) mle::launch(layernorm_bwd_kernel<256, 2>, (unsigned)parts, NT, 0, s, a);
  else if (cols <= kWidest) mle::launch(layernorm_bwd_kernel<256, 4>, (unsigned)parts, NT, 0, s, a);
  else {
    // the weight's sums first: dh may be dy's or h's buffer
    float* rest = sums ? static_cast<float*>(ws) + parts_floats(rows, cols) : nullptr;
    if (sums) {
      mle::launch(layernorm_rest_kernel, (unsigned)((rows - 1) / kRestRows + 1), 1024, 0, s, a, rest);
      mle::launch(layernorm_dw_kernel, dim3((unsigned)((cols + NT - 1) / NT), (unsigned)parts), NT, 0, s, a,
                  static_cast<const float*>(rest));
    }
    for (int64_t r0 = 0; r0 < rows; r0 += kRowsOfLaunch) {
      const int n = (int)std::min<int64_t>(rows - r0, kRowsOfLaunch);
      const int64_t at = r0 * cols;
      const LnBwdArgs b{n, cols, h + at, w, mean + r0, rstd + r0, dy + at, dres ? dres + at : dres, dh + at, accumulate_dh,
                        nullptr};
      mle::launch(layernorm_bwd_wide_kernel, (unsigned)n, 1024, 0, s, b, static_cast<const float*>(rest ? rest + r0 : rest));
    }
  }
  for (int64_t c0 = 0; sums && c0 < cols; c0 += kColsOfJoin)
    mle::launch(layernorm_join_kernel, dim3((unsigned)((std::min<int64_t>(cols - c0, kColsOfJoin) + 15) / 16), 2), 1024, 0, s,
                static_cast<const float*>(ws), parts, cols, (int)c0, dw, db, accumulate_dw);
  return check_launch("mle_add_layernorm_bwd");
}

}  // extern "C"
