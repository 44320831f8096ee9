// Windowed attention of the newest tokens over a cache: bound by reading the visible
// keys and values once.
//
// The rows of a group of heads that share keys (heads of the group times tokens) are the
// 16 columns of fp32 matrix products (v_mfma_f32_16x16x4_f32), so a key is read once for
// all of them.  A wave walks over blocks of 16 visible keys with loads straight from memory
// to the operands, the next block's in flight; both products sum in an order that lets
// every lane load 16 bytes:
//   S^T = K Q^T:  lane (key, q) holds columns 16 t + 4 q .. + 3 of its key,
//   O^T += V^T P^T:  lane (m, q) holds columns 64 u + 4 m .. + 3 of key 4 q + r, and P
//     leaves the accumulators with the keys 4 q + r of a row, as the product reads it.
// At 128 columns a block is 64 products of 32 cycles for 16 KB, 30 % of the matrix cores at
// the memory's rate.  Eight waves of a workgroup take every eighth block and join in order
// through LDS; where there are too few sequences and heads to fill the chip the keys are
// split over workgroups too, which leave (maximum, sum, O) to a second launch.  32 sequences of
// 8 heads of 4100 keys take 184 us (5.7 TB/s), one of 32768 keys 57 us (4.7 TB/s).
#include "window_kernels.hpp"

using namespace mle;

namespace wattn {
namespace {

constexpr int kRows = 16, kKeys = 16, kStepWaves = 8;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLazy = 10.f;  // how far a score may pass the maximum in use (log2)

// Four values from column `col` of a row of `dim`, zeros past it.
template <bool FULL>
__device__ __forceinline__ f32x4 load4(const float* __restrict__ row, int col, int dim) {
  if (FULL || col + 4 <= dim) return *reinterpret_cast<const f32x4u*>(row + col);
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (col + j < dim) x[j] = row[col + j];
  return x;
}

// A partial row: [dim] values, then the maximum (log2 units) and the sum.
__device__ __forceinline__ int part_size(const Args& a) { return a.dim + 2; }

// Rows of a group: head r / tokens, token r % tokens.
// DU: columns in 64s; FULL: the head has all of them.
template <int DU, bool FULL>
__global__ __launch_bounds__(64 * kStepWaves, 2) void step_kernel(Args a, StepWork wk, int64_t first) {
  constexpr int KT = 4 * DU, PAD = 64 * DU + 4;
  __shared__ __attribute__((aligned(16))) float sum_o[kStepWaves][kRows][PAD];
  __shared__ float sum_m[kStepWaves][kRows], sum_l[kStepWaves][kRows];
  const int64_t id = first + blockIdx.x;
  const int split = (int)(id % wk.splits);
  const int64_t rest = id / wk.splits;
  const int rb = (int)(rest % wk.row_blocks);
  const int64_t group = rest / wk.row_blocks;
  const int b = (int)(group / a.kv_heads), e = (int)(group % a.kv_heads);
  const Seq seq(a, b);
  const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  const int all_rows = a.group * a.rows;
  const int r = rb * kRows + c, token = r % a.rows, h = e * a.group + r / a.rows;
  const int p = seq.first + token;
  const bool live = r < all_rows && p >= 0 && p < seq.len;
  // the keys that any token sees, in blocks; those of this workgroup
  const int pf = max(seq.first, 0), pl = seq.len - 1;
  const int low = max(pf - a.window + 1, 0), before = min(a.sinks, low), count = pl >= pf ? before + pl + 1 - low : 0;
  const int blocks = (count + kKeys - 1) / kKeys, per = (blocks + wk.splits - 1) / wk.splits;
  const int b0 = split * per, b1 = min(b0 + per, blocks);
  const float* K = a.k + (int64_t)b * a.keys * a.ldk + (int64_t)e * a.dim;
  const float* V = a.v + (int64_t)b * a.keys * a.ldv + (int64_t)e * a.dim;
  const auto key_of = [&](int t) { return t < before ? t : low + t - before; };

  struct Block16 {
    f32x4 k[KT], v[4][DU];
  };
  auto load = [&](Block16& x, int blk) {
    const int tk = min(blk * kKeys + c, count - 1);
    const float* row = K + (int64_t)key_of(tk) * a.ldk;
#pragma unroll
    for (int t = 0; t < KT; ++t) x.k[t] = load4<FULL>(row, 16 * t + 4 * q, a.dim);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int tv = blk * kKeys + 4 * q + n;
      const float* vr = V + (int64_t)key_of(min(tv, count - 1)) * a.ldv;
#pragma unroll
      for (int u = 0; u < DU; ++u) {
        x.v[n][u] = load4<FULL>(vr, 64 * u + 4 * c, a.dim);
        if (tv >= count) x.v[n][u] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
  };
  f32x4 qf[KT];
  {
    const float* Q = a.q + ((int64_t)b * a.rows + (live ? token : 0)) * a.ldq + (int64_t)(live ? h : 0) * a.dim;
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      qf[t] = live ? load4<FULL>(Q, 16 * t + 4 * q, a.dim) : f32x4{0.f, 0.f, 0.f, 0.f};
      qf[t] *= a.scale * kLog2e;
    }
  }
  f32x4 o[DU][4];
#pragma unroll
  for (int u = 0; u < DU; ++u)
#pragma unroll
    for (int n = 0; n < 4; ++n) o[u][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -3e38f, l = 0.f;
  auto use = [&](const Block16& x, int blk) {
    f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int n = 0; n < 4; ++n) s[n & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.k[t][n], qf[t][n], s[n & 1], 0, 0, 0);
    s[0] += s[1];
    float x4[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int t = blk * kKeys + 4 * q + n;
      const bool seen = (t < count) & ((a.rows == 1) | sees(a, p, key_of(t)));
      x4[n] = seen ? s[0][n] : -INFINITY;
    }
    float mx = fmaxf(fmaxf(x4[0], x4[1]), fmaxf(x4[2], x4[3]));
    if (__any(mx > m + kLazy)) {
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(fmaxf(mx, __shfl_xor(mx, 32, 64)), m);
      const float f = __builtin_amdgcn_exp2f(m - mx);
      m = mx;
      l *= f;
#pragma unroll
      for (int u = 0; u < DU; ++u)
#pragma unroll
        for (int n = 0; n < 4; ++n) o[u][n] *= f;
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const float pn = __builtin_amdgcn_exp2f(x4[n] - m);
      l += pn;
#pragma unroll
      for (int u = 0; u < DU; ++u)
#pragma unroll
        for (int d = 0; d < 4; ++d) o[u][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.v[n][u][d], pn, o[u][d], 0, 0, 0);
    }
  };
  {
    Block16 x, y;
    int blk = b0 + w;
    if (blk < b1) load(x, blk);
    while (blk < b1) {
      if (blk + kStepWaves < b1) load(y, blk + kStepWaves);
      use(x, blk);
      blk += kStepWaves;
      if (blk >= b1) break;
      if (blk + kStepWaves < b1) load(x, blk + kStepWaves);
      use(y, blk);
      blk += kStepWaves;
    }
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (q == 0) {
    sum_m[w][c] = m;
    sum_l[w][c] = l;
  }
#pragma unroll
  for (int u = 0; u < DU; ++u)
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int d = 64 * u + 16 * q + 4 * n;  // columns d .. d + 3: accumulator n of the four products
      *reinterpret_cast<f32x4*>(&sum_o[w][c][d]) = f32x4{o[u][0][n], o[u][1][n], o[u][2][n], o[u][3][n]};
    }
  __syncthreads();
  // the waves' sums in order: two rows to a wave
#pragma unroll
  for (int k = 0; k < kRows / kStepWaves; ++k) {
    const int row = w * (kRows / kStepWaves) + k, g = rb * kRows + row;
    if (g >= all_rows) continue;
    float mm = sum_m[0][row];
#pragma unroll
    for (int i = 1; i < kStepWaves; ++i) mm = fmaxf(mm, sum_m[i][row]);
    float f[kStepWaves], ll = 0.f;
#pragma unroll
    for (int i = 0; i < kStepWaves; ++i) {
      f[i] = __builtin_amdgcn_exp2f(sum_m[i][row] - mm);
      ll += f[i] * sum_l[i][row];
    }
    const int tok = g % a.rows, pos = seq.first + tok;
    const bool there = pos >= 0 && pos < seq.len;
    float* out = wk.splits > 1 ? wk.part + ((rest * wk.splits + split) * kRows + row) * part_size(a)
                               : a.out + ((int64_t)b * a.rows + tok) * a.ldo + (int64_t)(e * a.group + g / a.rows) * a.dim;
    bool bad = false;
    for (int d = lane; d < a.dim; d += 64) {
      float x = 0.f;
#pragma unroll
      for (int i = 0; i < kStepWaves; ++i) x = fmaf(f[i], sum_o[i][row][d], x);
      if (wk.splits == 1) x = there ? x / ll : 0.f;
      bad |= !(fabsf(x) < INFINITY);
      out[d] = x;
    }
    if (wk.splits > 1) {
      if (lane == 0) {
        out[a.dim] = mm;
        out[a.dim + 1] = ll;
      }
    } else if (a.rows > 1 && __any(bad)) {
      // A token does not see all keys of the block: what one of them holds that is not finite
      // has reached it all the same.
      plain_row(a, b, e * a.group + g / a.rows, tok);
    }
  }
}

// Joins the splits of a row: a quarter of them to each of four waves, eight at a time (one after
// the other, 64 splits were 36 us of 88 at 32 heads over 32768 keys), then the quarters in order.
__global__ __launch_bounds__(256) void step_join_kernel(Args a, StepWork wk, int64_t first) {
  __shared__ float quarter[4][kMaxDim];
  const int64_t id = first + blockIdx.x;
  const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, all_rows = a.group * a.rows;
  const int64_t group = id / all_rows;
  const int g = (int)(id - group * all_rows);
  const int b = (int)(group / a.kv_heads), h = (int)(group % a.kv_heads) * a.group + g / a.rows, tok = g % a.rows;
  const Seq seq(a, b);
  const int pos = seq.first + tok, n = part_size(a);
  const bool there = pos >= 0 && pos < seq.len;
  const int64_t stride = (int64_t)kRows * n;
  const float* p = wk.part + ((group * wk.row_blocks + g / kRows) * wk.splits * kRows + g % kRows) * n;
  // lane s: split s
  float m = -3e38f, l = 0.f;
  if (lane < wk.splits) {
    m = p[lane * stride + a.dim];
    l = p[lane * stride + a.dim + 1];
  }
  const int per = (wk.splits + 3) / 4, s0 = w * per, s1 = min(s0 + per, wk.splits);
  const int d0 = min(lane, a.dim - 1), d1 = min(lane + 64, a.dim - 1);
  const float f = __builtin_amdgcn_exp2f(m - wave_max(m));
  l = wave_sum(l * f);
  float x[2] = {0.f, 0.f};
  for (int s = s0; s < s1; s += 8) {
    float v[8][2];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float* r = p + min(s + k, s1 - 1) * stride;
      v[k][0] = r[d0];
      v[k][1] = r[d1];
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const bool is = s + k < s1;
      const float fs = __shfl(f, is ? s + k : 0, 64);
      x[0] = is ? fmaf(fs, v[k][0], x[0]) : x[0];
      x[1] = is ? fmaf(fs, v[k][1], x[1]) : x[1];
    }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (lane + 64 * k < a.dim) quarter[w][lane + 64 * k] = x[k];
  __syncthreads();
  if (w != 0) return;
  float* out = a.out + ((int64_t)b * a.rows + tok) * a.ldo + (int64_t)h * a.dim;
  bool bad = false;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int d = lane + 64 * k;
    if (d < a.dim) {
      const float y = there ? (quarter[0][d] + quarter[1][d] + quarter[2][d] + quarter[3][d]) / l : 0.f;
      bad |= !(fabsf(y) < INFINITY);
      out[d] = y;
    }
  }
  if (a.rows > 1 && __any(bad)) plain_row(a, b, h, tok);
}

}  // namespace

void step_forward(const Args& a, const StepWork& wk, hipStream_t s) {
  const int64_t all = (int64_t)a.batch * a.kv_heads * wk.row_blocks * wk.splits;
  constexpr int64_t kBlocks = 1 << 22;  // a launch has fewer than 2^32 threads
  for (int64_t f = 0; f < all; f += kBlocks) {
    const unsigned n = (unsigned)std::min(all - f, kBlocks);
    if (a.dim == 64) mle::launch(step_kernel<1, true>, n, 64 * kStepWaves, 0, s, a, wk, f);
    else if (a.dim < 64) mle::launch(step_kernel<1, false>, n, 64 * kStepWaves, 0, s, a, wk, f);
    else if (a.dim == 128) mle::launch(step_kernel<2, true>, n, 64 * kStepWaves, 0, s, a, wk, f);
    else mle::launch(step_kernel<2, false>, n, 64 * kStepWaves, 0, s, a, wk, f);
  }
  if (wk.splits == 1) return;
  const int64_t rows = (int64_t)a.batch * a.heads * a.rows;
  for (int64_t f = 0; f < rows; f += kBlocks)
    mle::launch(step_join_kernel, (unsigned)std::min(rows - f, kBlocks), 256, 0, s, a, wk, f);
}

}  // namespace wattn
