// Activations kept in 8 bits for the backward pass (q8.hpp has the format):
// quantising, reading back, and the activation functions around it.  A Linear's weight
// gradient from a kept input is in q8_wgrad.hip.
#include "activation.hpp"
#include "q8.hpp"

#include <algorithm>

using namespace mle;
using namespace q8;

namespace {

constexpr int NT = 256;

// The elementwise kernels walk units of eight values of a row, four lanes to a
// group of 32: units of a row are numbered to whole groups, so a group's lanes
// always run together.
struct Q8Args {
  int rows, cols, units;  // units of a row: 4 per group
  const float* x;
  int64_t ldx;
  float* y;
  int64_t ldy;
  int8_t* q;
  int64_t ldq;
  uint8_t* e;
  int64_t lde;
  float* dx;
  int64_t lddx;
  int accumulate;
};

// Calls f(row, column, values left of the row (0 .. 8), lane's place in the
// group) for every unit.
template <class F>
__device__ __forceinline__ void each_unit(const Q8Args& a, F f) {
  const int64_t total = (int64_t)a.rows * a.units;
  const int64_t stride = (int64_t)gridDim.x * NT;
  for (int64_t u = (int64_t)blockIdx.x * NT + threadIdx.x; u < total; u += stride) {
    const int64_t row = total <= 0xffffffffLL ? (int64_t)((uint32_t)u / (uint32_t)a.units) : u / a.units;
    const int col = (int)(u - row * a.units) * 8;
    f(row, col, min(max(a.cols - col, 0), 8));
  }
}

// q, e = the 8 bits of x; with KIND >= 0 also y = act(x) from the same read.  Bound by
// memory: 8192 x 1024 8.8 us (4.8 TB/s), 8192 x 2048 with GELU 30 us (5.0 TB/s).
template <int KIND>
__global__ __launch_bounds__(NT) void q8_quantize_kernel(Q8Args a) {
  each_unit(a, [&](int64_t row, int col, int n) {
    float x[8];
    load_row8(a.x + row * a.ldx + col, n, x);
    uint2 code;
    const unsigned e = quantize8(x, code);
    if (n > 0) store_codes(a.q + row * a.ldq + col, code, n);
    if ((threadIdx.x & 3) == 0) a.e[row * a.lde + col / q8::kGroup] = (uint8_t)e;
    if (KIND >= 0) {
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = act_f<KIND < 0 ? 0 : KIND>(x[j]);
      if (n > 0) store_row8(a.y + row * a.ldy + col, y, n);
    }
  });
}

// y = the values of q, e.  8192 x 512: 6.0 us (3.5 TB/s; 2 us of it are the launch).
__global__ __launch_bounds__(NT) void q8_dequantize_kernel(Q8Args a) {
  each_unit(a, [&](int64_t row, int col, int n) {
    if (n == 0) return;
    float y[8];
    values8(load_codes(a.q + row * a.ldq + col, n), q8::step_of(a.e[row * a.lde + col / q8::kGroup]), y);
    store_row8(a.y + row * a.ldy + col, y, n);
  });
}

// dx (+)= act'(the kept x) * dy (a.x), as the elementwise activation backward forms it.
// 8192 x 2048, GELU: 28 us (5.3 TB/s).
template <int KIND>
__global__ __launch_bounds__(NT) void q8_act_bwd_kernel(Q8Args a) {
  each_unit(a, [&](int64_t row, int col, int n) {
    if (n == 0) return;
    float v[8], dy[8], old[8] = {};
    values8(load_codes(a.q + row * a.ldq + col, n), q8::step_of(a.e[row * a.lde + col / q8::kGroup]), v);
    load_row8(a.x + row * a.ldx + col, n, dy);
    float* p = a.dx + row * a.lddx + col;
    if (a.accumulate) load_row8(p, n, old);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = act_bwd_k<KIND>(v[j], dy[j], old[j], a.accumulate != 0);
    store_row8(p, v, n);
  });
}

unsigned grid_of(const Q8Args& a) { return stream_grid((size_t)a.rows * a.units, NT, 16384); }

#define Q8_LAUNCH_ACT(kernel, kind, a, s)                                                    \
  switch (kind) {                                                                            \
    case MLE_RELU: mle::launch(kernel<MLE_RELU>, grid_of(a), NT, 0, s, a); break;            \
    case MLE_GELU: mle::launch(kernel<MLE_GELU>, grid_of(a), NT, 0, s, a); break;            \
    case MLE_SILU: mle::launch(kernel<MLE_SILU>, grid_of(a), NT, 0, s, a); break;            \
    case MLE_TANH: mle::launch(kernel<MLE_TANH>, grid_of(a), NT, 0, s, a); break;            \
    case MLE_SIGMOID: mle::launch(kernel<MLE_SIGMOID>, grid_of(a), NT, 0, s, a); break;      \
    default: mle::launch(kernel<MLE_LEAKY_RELU>, grid_of(a), NT, 0, s, a); break;            \
  }

}  // namespace

extern "C" {

int mle_q8_quantize(mle_stream stream, int rows, int cols, const float* x, int64_t ldx, int8_t* q, int64_t ldq,
                    uint8_t* e, int64_t lde) {
  const int rc = check_shape("mle_q8_quantize", rows, cols, q, ldq, e, lde);
  if (rc) return rc;
  MLE_CHECK_ARG((x || rows == 0) && ldx >= cols, "mle_q8_quantize: null pointer or ldx %lld < %d", (long long)ldx, cols);
  if (rows == 0) return MLE_OK;
  const Q8Args a{rows, cols, 4 * q8::groups(cols), x, ldx, nullptr, 0, q, ldq, e, lde, nullptr, 0, 0};
  mle::launch(q8_quantize_kernel<-1>, grid_of(a), NT, 0, as_stream(stream), a);
  return check_launch("mle_q8_quantize");
}

int mle_q8_dequantize(mle_stream stream, int rows, int cols, const int8_t* q, int64_t ldq, const uint8_t* e,
                      int64_t lde, float* y, int64_t ldy) {
  const int rc = check_shape("mle_q8_dequantize", rows, cols, q, ldq, e, lde);
  if (rc) return rc;
  MLE_CHECK_ARG((y || rows == 0) && ldy >= cols, "mle_q8_dequantize: null pointer or ldy %lld < %d", (long long)ldy, cols);
  if (rows == 0) return MLE_OK;
  const Q8Args a{rows, cols, 4 * q8::groups(cols), nullptr, 0, y, ldy, const_cast<int8_t*>(q), ldq, const_cast<uint8_t*>(e),
           lde, nullptr, 0, 0};
  mle::launch(q8_dequantize_kernel, grid_of(a), NT, 0, as_stream(stream), a);
  return check_launch("mle_q8_dequantize");
}

int mle_q8_act_fwd(mle_stream stream, int kind, int rows, int cols, const float* x, int64_t ldx, float* y, int64_t ldy,
                   int8_t* q, int64_t ldq, uint8_t* e, int64_t lde) {
  const int rc = check_shape("mle_q8_act_fwd", rows, cols, q, ldq, e, lde);
  if (rc) return rc;
  MLE_CHECK_ARG(kind >= MLE_RELU && kind <= MLE_LEAKY_RELU, "mle_q8_act_fwd: activation %d", kind);
  MLE_CHECK_ARG(((x && y) || rows == 0) && ldx >= cols && ldy >= cols,
                "mle_q8_act_fwd: null pointer or a leading dimension below %d", cols);
  if (rows == 0) return MLE_OK;
  const Q8Args a{rows, cols, 4 * q8::groups(cols), x, ldx, y, ldy, q, ldq, e, lde, nullptr, 0, 0};
  Q8_LAUNCH_ACT(q8_quantize_kernel, kind, a, as_stream(stream));
  return check_launch("mle_q8_act_fwd");
}

int mle_q8_act_bwd(mle_stream stream, int kind, int rows, int cols, const int8_t* q, int64_t ldq, const uint8_t* e,
                   int64_t lde, const float* dy, int64_t lddy, float* dx, int64_t lddx, int accumulate) {
  const int rc = check_shape("mle_q8_act_bwd", rows, cols, q, ldq, e, lde);
  if (rc) return rc;
  MLE_CHECK_ARG(kind >= MLE_RELU && kind <= MLE_LEAKY_RELU, "mle_q8_act_bwd: activation %d", kind);
  MLE_CHECK_ARG(((dy && dx) || rows == 0) && lddy >= cols && lddx >= cols,
                "mle_q8_act_bwd: null pointer or a leading dimension below %d", cols);
  if (rows == 0) return MLE_OK;
  const Q8Args a{rows, cols, 4 * q8::groups(cols), dy, lddy, nullptr, 0, const_cast<int8_t*>(q), ldq, const_cast<uint8_t*>(e),
           lde, dx, lddx, accumulate};
  Q8_LAUNCH_ACT(q8_act_bwd_kernel, kind, a, as_stream(stream));
  return check_launch("mle_q8_act_bwd");
}

}  // extern "C"
