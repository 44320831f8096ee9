// Rotary positions with several axes: every pair (a, b) of a head's values is
// turned by its own angle, a position times the pair's frequency,
//   (a cos - b sin, a sin + b cos);
// turning back (inverse) is the transpose, the gradient.
//
// An angle is formed and brought to [-pi/4, pi/4] in 64 bits, where sine and
// cosine are their Taylor polynomials; in 32 bits a position up to a million times a
// frequency of 0.9 is off by up to 2.9 degrees.
//
// A wave takes the heads of a row: a lane keeps the angles of its V pairs (V = 4, 16
// bytes of each half) and walks over the row's heads with them, 64 / (pairs / V)
// heads at a time, so that an angle is formed once for several heads and the loads
// run on without LDS or barriers.  Bound by memory: 32768 rows of 16 + 4 heads of 128
// take 123 us a direction (5.5 TB/s); 32 rows of 32 + 8 heads take 3.6 us, a launch.
#include "common.hpp"

#include <math.h>
#include <algorithm>

using namespace mle;

namespace {

constexpr int kPairs = 128, kAxes = 8;
constexpr int kRowsOfLaunch = 1 << 24;  // a launch has fewer than 2^32 threads

struct RotaryArgs {
  const float* x[2];  // q and k
  float* y[2];
  int64_t ldx[2], ldy[2];
  int heads[2];
  const int32_t* positions;
  int64_t rows, stride;  // of this launch; positions of an axis
  int dim, pairs;
  int inverse, accumulate;
  int split;  // waves that share a row's heads
  unsigned char axis[kPairs];
  double freq[kPairs];  // over 2 pi: turns a position into whole turns
};

// cos and sin of 2 pi t.
__device__ __forceinline__ float2 turn(double t) {
  t -= rint(t);                       // [-1/2, 1/2], exact
  const double q = rint(4.0 * t);     // quarter turns
  const double x = (t - 0.25 * q) * 6.283185307179586476925;  // [-pi/4, pi/4]
  const double z = x * x;
  // what is left out is below 2^-28 (sine) and 2^-32 (cosine) of the result
  const float s = (float)(x * (1.0 + z * (-1.0 / 6 + z * (1.0 / 120 + z * (-1.0 / 5040 + z * (1.0 / 362880))))));
  const float c = (float)(1.0 + z * (-0.5 + z * (1.0 / 24 + z * (-1.0 / 720 + z * (1.0 / 40320 + z * (-1.0 / 3628800))))));
  const int k = (int)q & 3;
  const float cc = k & 1 ? s : c, ss = k & 1 ? c : s;
  return make_float2(k == 1 || k == 2 ? -cc : cc, k & 2 ? -ss : ss);
}

template <int V>
struct Vec {
  typedef f32x4u type;
};
template <>
struct Vec<1> {
  typedef float type;
};

// V consecutive values from p.
template <int V>
__device__ __forceinline__ void load(const float* p, float (&x)[V]) {
  const typename Vec<V>::type v = *reinterpret_cast<const typename Vec<V>::type*>(p);
  __builtin_memcpy(x, &v, sizeof(v));
}
template <int V>
__device__ __forceinline__ void store(float* p, const float (&x)[V]) {
  typename Vec<V>::type v;
  __builtin_memcpy(&v, x, sizeof(v));
  *reinterpret_cast<typename Vec<V>::type*>(p) = v;
}

// V pairs to a lane (V divides pairs); NEIGHBOURS: a pair is two consecutive values.
template <int V, bool NEIGHBOURS>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t wave = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int64_t row = wave / a.split;
  const int part = (int)(wave - row * a.split);
  if (row >= a.rows) return;
  const int n = a.pairs / V;              // lanes of a head
  const int at_once = n < 64 ? 64 / n : 1;  // heads
  const int sub = n < 64 ? lane / n : 0, first = n < 64 ? lane - sub * n : lane;
  const int P = a.pairs, all = a.heads[0] + a.heads[1];
  if (sub < at_once) {
    for (int i = first; i < n; i += 64) {
      float c[V], s[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int p = i * V + j;
        const float2 t = turn((double)a.positions[a.axis[p] * a.stride + row] * a.freq[p]);
        c[j] = t.x;
        s[j] = a.inverse ? -t.y : t.y;
      }
      const int oa = (NEIGHBOURS ? 2 : 1) * i * V, ob = NEIGHBOURS ? oa + V : oa + P;
#pragma unroll 2
      for (int h = part * at_once + sub; h < all; h += a.split * at_once) {
        const int w = h < a.heads[0] ? 0 : 1;
        const int64_t col = (int64_t)(w ? h - a.heads[0] : h) * a.dim;
        const float* x = a.x[w] + row * a.ldx[w] + col;
        float* y = a.y[w] + row * a.ldy[w] + col;
        float u[V], v[V], old[2][V], r[2][V];
        load<V>(x + oa, u);
        load<V>(x + ob, v);
#pragma unroll
        for (int j = 0; j < V; ++j) old[0][j] = old[1][j] = 0.f;
        if (a.accumulate) {
          load<V>(y + oa, old[0]);
          load<V>(y + ob, old[1]);
        }
        if (NEIGHBOURS && V > 1) {  // pairs lie one after the other
          float b[2 * V];
#pragma unroll
          for (int j = 0; j < V; ++j) b[j] = u[j], b[V + j] = v[j];
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float e = b[2 * j], f = b[2 * j + 1];
            b[2 * j] = e * c[j] - f * s[j];
            b[2 * j + 1] = e * s[j] + f * c[j];
          }
#pragma unroll
          for (int j = 0; j < V; ++j) r[0][j] = b[j], r[1][j] = b[V + j];
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            r[0][j] = u[j] * c[j] - v[j] * s[j];
            r[1][j] = u[j] * s[j] + v[j] * c[j];
          }
        }
        if (a.accumulate) {
#pragma unroll
          for (int j = 0; j < V; ++j) r[0][j] += old[0][j], r[1][j] += old[1][j];
        }
        store<V>(y + oa, r[0]);
        store<V>(y + ob, r[1]);
      }
    }
  }
  // the values that are not turned
  const int rest = a.dim - 2 * P;
  if (rest == 0) return;
  for (int h = part; h < all; h += a.split) {
    const int w = h < a.heads[0] ? 0 : 1;
    const int64_t col = (int64_t)(w ? h - a.heads[0] : h) * a.dim + 2 * P;
    const float* x = a.x[w] + row * a.ldx[w] + col;
    float* y = a.y[w] + row * a.ldy[w] + col;
    for (int j = lane; j < rest; j += 64) y[j] = a.accumulate ? y[j] + x[j] : x[j];
  }
}

}  // namespace

extern "C" int mle_rotary(mle_stream stream, int rows, int head_dim, const float* q, int64_t ldq, float* q_out, int64_t ldqo,
                          int heads, const float* k, int64_t ldk, float* k_out, int64_t ldko, int kv_heads,
                          const int32_t* positions, int axes, const int* sections, double base, int flags, int inverse,
                          int accumulate) {
  MLE_CHECK_ARG(rows >= 0 && head_dim > 0 && head_dim <= (1 << 20) && heads > 0 && kv_heads >= 0 && heads <= (1 << 20) &&
                    kv_heads <= (1 << 20),
                "mle_rotary: bad shape, %d rows of %d and %d heads of %d", rows, heads, kv_heads, head_dim);
  MLE_CHECK_ARG(axes > 0 && axes <= kAxes && sections, "mle_rotary: %d axes (1 to %d), sections %p", axes, kAxes,
                (const void*)sections);
  MLE_CHECK_ARG((flags & ~(MLE_ROTARY_NEIGHBOURS | MLE_ROTARY_BY_AXIS)) == 0, "mle_rotary: flags %d", flags);
  MLE_CHECK_ARG(base > 0.0 && base <= 1e300, "mle_rotary: base %g", base);
  int64_t pairs = 0;
  for (int i = 0; i < axes; ++i) {
    MLE_CHECK_ARG(sections[i] >= 0, "mle_rotary: section %d is %d", i, sections[i]);
    pairs += sections[i];
  }
  MLE_CHECK_ARG(pairs > 0 && 2 * pairs <= head_dim, "mle_rotary: %lld pairs of a head of %d", (long long)pairs, head_dim);
  if (pairs > kPairs) return set_error(MLE_ERR_UNSUPPORTED, "mle_rotary: %lld pairs, at most %d", (long long)pairs, kPairs);
  const int64_t wq = (int64_t)heads * head_dim, wk = (int64_t)kv_heads * head_dim;
  MLE_CHECK_ARG(ldq >= wq && ldqo >= wq, "mle_rotary: ldq %lld or ldqo %lld < %lld", (long long)ldq, (long long)ldqo,
                (long long)wq);
  MLE_CHECK_ARG(kv_heads == 0 || (ldk >= wk && ldko >= wk), "mle_rotary: ldk %lld or ldko %lld < %lld", (long long)ldk,
                (long long)ldko, (long long)wk);
  MLE_CHECK_ARG(rows == 0 || (q && q_out && positions && (kv_heads == 0 || (k && k_out))), "mle_rotary: null pointer");
  if (rows == 0) return MLE_OK;
  RotaryArgs a{};
  a.ldx[0] = ldq, a.ldx[1] = ldk, a.ldy[0] = ldqo, a.ldy[1] = ldko;
  a.heads[0] = heads, a.heads[1] = kv_heads;
  a.stride = rows;
  a.dim = head_dim, a.pairs = (int)pairs;
  a.inverse = inverse != 0, a.accumulate = accumulate != 0;
  int p = 0;
  for (int i = 0; i < axes; ++i)
    for (int j = 0; j < sections[i]; ++j, ++p) {
      const bool by_axis = (flags & MLE_ROTARY_BY_AXIS) != 0;
      a.axis[p] = (unsigned char)i;
      a.freq[p] = pow(base, by_axis ? -(double)j / sections[i] : -(double)p / (double)pairs) / 6.283185307179586476925;
    }
  const bool neighbours = (flags & MLE_ROTARY_NEIGHBOURS) != 0, by4 = pairs % 4 == 0;
  // a row's heads over more waves while there are too few rows to fill the chip
  const int n = (int)pairs / (by4 ? 4 : 1), steps = (heads + kv_heads + (n < 64 ? 64 / n : 1) - 1) / (n < 64 ? 64 / n : 1);
  a.split = (int)std::max<int64_t>(1, std::min<int64_t>(steps, 2048 / rows));
  hipStream_t s = as_stream(stream);
  for (int64_t r0 = 0; r0 < rows; r0 += kRowsOfLaunch) {
    a.rows = std::min<int64_t>(rows - r0, kRowsOfLaunch);
    a.positions = positions + r0;
    for (int w = 0; w < (kv_heads ? 2 : 1); ++w) {
      a.x[w] = (w ? k : q) + r0 * a.ldx[w];
      a.y[w] = (w ? k_out : q_out) + r0 * a.ldy[w];
    }
    const unsigned grid = (unsigned)((a.rows * a.split + 3) / 4);
    if (by4 && neighbours) mle::launch(rotary_kernel<4, true>, grid, 256, 0, s, a);
    else if (by4) mle::launch(rotary_kernel<4, false>, grid, 256, 0, s, a);
    else if (neighbours) mle::launch(rotary_kernel<1, true>, grid, 256, 0, s, a);
    else mle::launch(rotary_kernel<1, false>, grid, 256, 0, s, a);
  }
  return check_launch("mle_rotary");
}
