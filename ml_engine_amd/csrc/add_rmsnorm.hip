// The residual Add and the root-mean-square norm that reads it, with the
// output also kept in 8 bits (q8.hpp), and the backward of both.
//
//   h = x + r,  rstd = 1 / sqrt(mean(h^2) + eps),  y = h rstd w  along each row
//   u = h rstd, g = dy w:  dh = dres + rstd (g - u mean(g u)),  dw = sum over rows of dy u
//
// One pass over a row: T lanes of a wave, or a workgroup of T threads, hold it
// in registers, eight consecutive values to a thread and chunk (four threads
// to a group of 32, whose step is found within the quad).  y is formed in 64
// bits and rounded once to 32, and the 8 bits are those of that y: a mean
// summed in another order would otherwise move values across the border of two
// codes, and one in some hundred thousand would differ by a whole step.
#include "q8.hpp"

#include <algorithm>

using namespace mle;

namespace {

constexpr int NT = 256;
constexpr int kMaxParts = 512;  // partial weight gradients: workgroups of the backward
constexpr int kRowsOfLaunch = 1 << 21;  // of the forward: a launch has fewer than 2^32 threads

struct NormArgs {
  int rows, cols;
  const float* x;
  const float* r;
  const float* w;
  float* h;
  float* y;
  float* rstd;
  int8_t* q;
  int64_t ldq;
  uint8_t* e;
  int64_t lde;
  float eps;
};

struct NormBwdArgs {
  int rows, cols;
  const float* h;
  const float* w;
  const float* rstd;
  const float* dy;
  const float* dres;
  float* dh;
  int acc_dh;
  float* part;  // [workgroups][cols]; null: no weight gradient
};

// The sum of v over a row's T threads, in every one of them.
template <int T>
__device__ __forceinline__ double row_sum(double v, double* red) {
  if (T <= 64) {
#pragma unroll
    for (int o = T / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
  }
  return block_sum<T < 64 ? 64 : T, double>(v, red);
}

// T threads to a row, C chunks of 8 values each (T * 8 * C >= cols); C == 0:
// any width, h read a second time.  Bound by memory: 8192 x 512 15.6 us (4.6 TB/s),
// 16384 x 4096 210 us (5.4 TB/s).
template <int T, int C>
__global__ __launch_bounds__(T < NT ? NT : T) void rmsnorm_q8_fwd_kernel(NormArgs a) {
  constexpr int B = T < NT ? NT : T, R = B / T;  // rows of a workgroup
  __shared__ double red[B / 64];
  const int t = threadIdx.x % T;
  const int64_t row = (int64_t)blockIdx.x * R + threadIdx.x / T;
  if (row >= a.rows) return;  // (T < B: whole quads and whole rows; T == B: the workgroup)
  const int64_t base = row * a.cols;
  const int chunks = C > 0 ? C : (a.cols + 8 * T - 1) / (8 * T);
  float keep[C > 0 ? C : 1][8];
  double s = 0.0;
#pragma unroll C > 0 ? C : 1
  for (int c = 0; c < chunks; ++c) {
    float(&h)[8] = keep[C > 0 ? c : 0];
    const int col = (c * T + t) * 8, n = min(max(a.cols - col, 0), 8);
    if (n == 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] = 0.f;
      continue;
    }
    q8::load_row8(a.x + base + col, n, h);
    if (a.r) {
      float r[8];
      q8::load_row8(a.r + base + col, n, r);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] += r[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) s += (double)h[j] * (double)h[j];
  }
  s = row_sum<T>(s, red);
  const double rstd = 1.0 / sqrt(s / a.cols + (double)a.eps);
  if (t == 0) a.rstd[row] = (float)rstd;
#pragma unroll C > 0 ? C : 1
  for (int c = 0; c < chunks; ++c) {
    float(&h)[8] = keep[C > 0 ? c : 0];
    const int col = (c * T + t) * 8, n = min(max(a.cols - col, 0), 8);
    if ((c * T + (t & ~3)) * 8 >= a.cols) continue;  // no value of this quad's group
    if (C == 0) {
      q8::load_row8(a.x + base + col, n, h);
      if (a.r) {
        float r[8];
        q8::load_row8(a.r + base + col, n, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] += r[j];
      }
    }
    if (a.h) q8::store_row8(a.h + base + col, h, n);
    float y[8], w[8];
    if (a.w) q8::load_row8(a.w + col, n, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const double u = (double)h[j] * rstd;
      y[j] = j < n ? (float)(a.w ? u * (double)w[j] : u) : 0.f;
    }
    if (a.y) q8::store_row8(a.y + base + col, y, n);
    if (a.q) {
      uint2 code;
      const unsigned e = q8::quantize8(y, code);
      q8::store_codes(a.q + row * a.ldq + col, code, n);
      if ((t & 3) == 0) a.e[row * a.lde + col / q8::kGroup] = (uint8_t)e;
    }
  }
}

// A workgroup takes rows blockIdx.x * R + i * gridDim.x * R and keeps its
// threads' columns of dw in registers; the R rows that it walks at a time add
// theirs through LDS at the end.  8192 x 512 13.2 us, 16384 x 4096 211 us (5.1 TB/s each).
template <int T, int C>
__global__ __launch_bounds__(T < NT ? NT : T) void rmsnorm_bwd_kernel(NormBwdArgs a) {
  constexpr int B = T < NT ? NT : T, R = B / T;
  __shared__ double red[B / 64];
  __shared__ float cols_red[R > 1 ? 8 * B : 1];
  const int t = threadIdx.x % T, k = threadIdx.x / T;
  float dw[C][8], w[C][8];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int col = (c * T + t) * 8, n = min(max(a.cols - col, 0), 8);
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[c][j] = 0.f, w[c][j] = 1.f;
    if (a.w && n > 0) q8::load_row8(a.w + col, n, w[c]);
  }
  for (int64_t r0 = (int64_t)blockIdx.x * R; r0 < a.rows; r0 += (int64_t)gridDim.x * R) {
    const int64_t row = r0 + k;
    const bool live = row < a.rows;
    const int64_t base = (live ? row : a.rows - 1) * a.cols;
    const float rstd = live ? a.rstd[row] : 0.f;
    float u[C][8], g[C][8];
    double s = 0.0;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * T + t) * 8, n = live ? min(max(a.cols - col, 0), 8) : 0;
      if (n == 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) u[c][j] = g[c][j] = 0.f;
        continue;
      }
      q8::load_row8(a.h + base + col, n, u[c]);
      q8::load_row8(a.dy + base + col, n, g[c]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        u[c][j] *= rstd;
        dw[c][j] += g[c][j] * u[c][j];
        g[c][j] *= w[c][j];
        s += (double)(g[c][j] * u[c][j]);
      }
    }
    const float m = (float)(row_sum<T>(s, red) / a.cols);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * T + t) * 8, n = live ? min(max(a.cols - col, 0), 8) : 0;
      if (n == 0) continue;
      float old[8] = {}, dres[8] = {}, v[8];
      if (a.dres) q8::load_row8(a.dres + base + col, n, dres);
      if (a.acc_dh) q8::load_row8(a.dh + base + col, n, old);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = old[j] + (dres[j] + rstd * (g[c][j] - u[c][j] * m));
      q8::store_row8(a.dh + base + col, v, n);
    }
  }
  if (!a.part) return;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int col = (c * T + t) * 8, n = min(max(a.cols - col, 0), 8);
    if (R > 1) {  // the rows' sums in order
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) cols_red[8 * threadIdx.x + j] = dw[c][j];
      __syncthreads();
      if (k > 0) continue;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        for (int i = 1; i < R; ++i) dw[c][j] += cols_red[8 * (i * T + t) + j];
    }
    if (n > 0) q8::store_row8(a.part + (int64_t)blockIdx.x * a.cols + col, dw[c], n);
  }
}

// Rows wider than the register kernels take: h and dy read twice; the weight
// gradient in a pass of its own (rmsnorm_dw_kernel).
__global__ __launch_bounds__(1024) void rmsnorm_bwd_wide_kernel(NormBwdArgs a) {
  __shared__ double red[16];
  const int64_t base = (int64_t)blockIdx.x * a.cols;
  const float rstd = a.rstd[blockIdx.x];
  double s = 0.0;
  for (int i = threadIdx.x; i < a.cols; i += 1024)
    s += (double)((a.dy[base + i] * (a.w ? a.w[i] : 1.f)) * (a.h[base + i] * rstd));
  const float m = (float)(block_sum<1024>(s, red) / a.cols);
  for (int i = threadIdx.x; i < a.cols; i += 1024) {
    const float g = a.dy[base + i] * (a.w ? a.w[i] : 1.f), u = a.h[base + i] * rstd;
    const float v = (a.dres ? a.dres[base + i] : 0.f) + rstd * (g - u * m);
    a.dh[base + i] = (a.acc_dh ? a.dh[base + i] : 0.f) + v;
  }
}
// part[block y][col] = sum of dy u over rows y, y + gridDim.y, ...
__global__ __launch_bounds__(NT) void rmsnorm_dw_kernel(NormBwdArgs a) {
  const int col = blockIdx.x * NT + threadIdx.x;
  if (col >= a.cols) return;
  float s = 0.f;
  for (int64_t r = blockIdx.y; r < a.rows; r += gridDim.y) s += a.dy[r * a.cols + col] * (a.h[r * a.cols + col] * a.rstd[r]);
  a.part[(int64_t)blockIdx.y * a.cols + col] = s;
}

// dw (+)= the partial sums: 16 columns to a workgroup, 64 threads to a column, each
// adding every 64th part, and the threads' sums in order.
__global__ __launch_bounds__(1024) void rmsnorm_join_kernel(const float* __restrict__ part, int parts, int cols,
                                                            float* __restrict__ dw, int accumulate) {
  __shared__ float red[64][17];
  const int c = threadIdx.x & 15, g = threadIdx.x >> 4;
  const int col = blockIdx.x * 16 + c;
  float s = 0.f;
  if (col < cols) {
#pragma unroll 8
    for (int p = g; p < parts; p += 64) s += part[(int64_t)p * cols + col];
  }
  red[g][c] = s;
  __syncthreads();
  if (threadIdx.x >= 64) return;
  // a quarter of the threads' sums to each of four lanes, then the quarters
  s = 0.f;
  const int q = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 16; ++i) s += red[16 * q + i][c];
  const float a = __shfl(s, c, 64), b = __shfl(s, 16 + c, 64), d = __shfl(s, 32 + c, 64), e = __shfl(s, 48 + c, 64);
  if (q != 0 || col >= cols) return;
  const float v = ((a + b) + d) + e;
  dw[col] = accumulate ? dw[col] + v : v;
}

// Workgroups of the backward, each with a partial weight gradient: a function of the shape alone.
int parts_of(int rows, int cols) {
  const int rows_of_wg = cols <= 2048 ? 4 : 1;
  return std::max(1, std::min(kMaxParts, (rows - 1) / rows_of_wg + 1));
}

int check(const char* who, int rows, int cols) {
  MLE_CHECK_ARG(rows >= 0 && cols > 0 && cols <= (1 << 30), "%s: bad shape %d x %d", who, rows, cols);
  return MLE_OK;
}

}  // namespace

extern "C" {

int mle_add_rmsnorm_q8_fwd(mle_stream stream, int rows, int cols, const float* x, const float* r, const float* w,
                           float eps, float* h, float* y, float* rstd, int8_t* q, int64_t ldq, uint8_t* e,
                           int64_t lde) {
  const int rc = check("mle_add_rmsnorm_q8_fwd", rows, cols);
  if (rc) return rc;
  MLE_CHECK_ARG(rows == 0 || (x && rstd), "mle_add_rmsnorm_q8_fwd: null pointer");
  MLE_CHECK_ARG((q == nullptr) == (e == nullptr), "mle_add_rmsnorm_q8_fwd: q and e come together");
  MLE_CHECK_ARG(!q || (ldq >= cols && lde >= q8::groups(cols)), "mle_add_rmsnorm_q8_fwd: ldq %lld < %d or lde %lld < %d",
                (long long)ldq, cols, (long long)lde, q8::groups(cols));
  MLE_CHECK_ARG(eps >= 0.f, "mle_add_rmsnorm_q8_fwd: eps %g", (double)eps);
  if (rows == 0) return MLE_OK;
  hipStream_t s = as_stream(stream);
  for (int64_t r0 = 0; r0 < rows; r0 += kRowsOfLaunch) {
    const int n = (int)std::min<int64_t>(rows - r0, kRowsOfLaunch);
    const int64_t at = r0 * cols;
    const NormArgs a{n, cols, x + at, r ? r + at : r, w, h ? h + at : h, y ? y + at : y, rstd + r0, q ? q + r0 * ldq : q, ldq,
                     e ? e + r0 * lde : e, lde, eps};
    const unsigned by4 = (unsigned)((n + 3) / 4);
    if (cols <= 512) mle::launch(rmsnorm_q8_fwd_kernel<64, 1>, by4, NT, 0, s, a);
    else if (cols <= 1024) mle::launch(rmsnorm_q8_fwd_kernel<64, 2>, by4, NT, 0, s, a);
    else if (cols <= 2048) mle::launch(rmsnorm_q8_fwd_kernel<64, 4>, by4, NT, 0, s, a);
    else if (cols <= 4096) mle::launch(rmsnorm_q8_fwd_kernel<256, 2>, (unsigned)n, NT, 0, s, a);
    else if (cols <= 8192) mle::launch(rmsnorm_q8_fwd_kernel<256, 4>, (unsigned)n, NT, 0, s, a);
    else mle::launch(rmsnorm_q8_fwd_kernel<1024, 0>, (unsigned)n, 1024, 0, s, a);
  }
  return check_launch("mle_add_rmsnorm_q8_fwd");
}

size_t mle_add_rmsnorm_ws_bytes(int rows, int cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return (size_t)parts_of(rows, cols) * cols * sizeof(float);
}

int mle_add_rmsnorm_bwd(mle_stream stream, int rows, int cols, const float* h, const float* w, const float* rstd,
                        const float* dy, const float* dres, float* dh, int accumulate_dh, float* dw, int accumulate_dw,
                        void* ws, size_t ws_bytes) {
  const int rc = check("mle_add_rmsnorm_bwd", rows, cols);
  if (rc) return rc;
  MLE_CHECK_ARG(rows == 0 || (h && rstd && dy && dh), "mle_add_rmsnorm_bwd: null pointer");
  if (rows == 0) return dw && !accumulate_dw ? mle_fill(stream, dw, 0.f, (size_t)cols) : MLE_OK;
  if (dw && (!ws || !aligned16(ws) || ws_bytes < mle_add_rmsnorm_ws_bytes(rows, cols)))
    return set_error(MLE_ERR_WORKSPACE, "mle_add_rmsnorm_bwd: workspace of %zu bytes, 16-byte aligned, needed",
                     mle_add_rmsnorm_ws_bytes(rows, cols));
  const int parts = parts_of(rows, cols);
  const NormBwdArgs a{rows, cols, h, w, rstd, dy, dres, dh, accumulate_dh, dw ? static_cast<float*>(ws) : nullptr};
  hipStream_t s = as_stream(stream);
  if (cols <= 512) mle::launch(rmsnorm_bwd_kernel<64, 1>, (unsigned)parts, NT, 0, s, a);
  else if (cols <= 1024) mle::launch(rmsnorm_bwd_kernel<64, 2>, (unsigned)parts, NT, 0, s, a);
  else if (cols <= 2048) mle::launch(rmsnorm_bwd_kernel<64, 4>, (unsigned)parts, NT, 0, s, a);
  else if (cols <= 4096) mle::launch(rmsnorm_bwd_kernel<256, 2>, (unsigned)parts, NT, 0, s, a);
  else if (cols <= 8192) mle::launch(rmsnorm_bwd_kernel<256, 4>, (unsigned)parts, NT, 0, s, a);
  else {
    // dw first: dh may be dy's or h's buffer
    if (dw) mle::launch(rmsnorm_dw_kernel, dim3((unsigned)((cols + NT - 1) / NT), (unsigned)parts), NT, 0, s, a);
    mle::launch(rmsnorm_bwd_wide_kernel, (unsigned)rows, 1024, 0, s, a);
  }
  if (dw)
    mle::launch(rmsnorm_join_kernel, (unsigned)((cols + 15) / 16), 1024, 0, s, static_cast<const float*>(ws), parts, cols, dw,
                accumulate_dw);
  return check_launch("mle_add_rmsnorm_bwd");
}

}  // extern "C"
