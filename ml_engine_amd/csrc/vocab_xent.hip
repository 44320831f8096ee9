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
#include "common.hpp"

#include <float.h>

#include <algorithm>

using namespace mle;

namespace {

constexpr int NT = 256;

struct Rows {
  const int32_t* keys;
  int clen, max_clen, vocab;
  __device__ __forceinline__ int key(int64_t r) const {
    const int k = keys[clen == max_clen ? r : r / clen * max_clen + r % clen];
    return k >= 0 && k < vocab ? k : -1;
  }
};

// What a row has of the vocabulary's pieces so far.
struct RowState {
  float max, sum, target, pad;  // sum of exp(l - max)
};

// One row of a piece to a workgroup: its maximum and sum join the row's.
__global__ __launch_bounds__(NT) void xent_stats_kernel(const float* __restrict__ l, int cols, int v0, Rows rows,
                                                        RowState* __restrict__ state, int first) {
  __shared__ float red[NT / 64];
  const int64_t r = blockIdx.x;
  const float* x = l + r * cols;
  float m = -FLT_MAX;
  for (int c = threadIdx.x; c < cols; c += NT) m = fmaxf(m, x[c]);
  m = block_max<NT>(m, red);
  float s = 0.f;
  for (int c = threadIdx.x; c < cols; c += NT) s += expf(x[c] - m);
  s = block_sum<NT>(s, red);
  if (threadIdx.x != 0) return;
  RowState t{m, s, 0.f, 0.f};
  if (!first) {
    const RowState o = state[r];
    t.max = fmaxf(o.max, m);
    t.sum = o.sum * expf(o.max - t.max) + s * expf(m - t.max);
    t.target = o.target;
  }
  const int k = rows.key(r);
  if (k >= v0 && k < v0 + cols) t.target = x[k - v0];
  state[r] = t;
}

// lse, the row losses and their scaled sum; one workgroup.
__global__ __launch_bounds__(1024) void xent_finish_kernel(const RowState* __restrict__ state, int nrows, Rows rows,
                                                           float scale, float* __restrict__ lse,
                                                           float* __restrict__ row_loss, float* __restrict__ loss) {
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
  if (threadIdx.x == 0) loss[0] = (float)(sum * (double)scale);
}

// The rows of X that take part, the others as zeros: what a row that takes no
// part holds, NaN included, must not reach dW.
__global__ __launch_bounds__(NT) void xent_rows_kernel(const float* __restrict__ X, int64_t ldx, int d, Rows rows,
                                                       float* __restrict__ out) {
  const int64_t r = blockIdx.x;
  const bool live = rows.key(r) >= 0;
  for (int c = threadIdx.x; c < d; c += NT) out[r * d + c] = live ? X[r * ldx + c] : 0.f;
}

// A piece's logits to P, in place.
__global__ __launch_bounds__(NT) void xent_grad_kernel(float* __restrict__ l, int cols, int v0, Rows rows,
                                                       const float* __restrict__ lse, const float* __restrict__ upstream,
                                                       float scale) {
  const int64_t r = blockIdx.x;
  float* x = l + r * cols;
  const int k = rows.key(r);
  const float z = lse[r], g = upstream ? upstream[0] * scale : scale;
  for (int c = threadIdx.x; c < cols; c += NT) x[c] = k >= 0 ? g * (expf(x[c] - z) - (c + v0 == k ? 1.f : 0.f)) : 0.f;
}

size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

// Columns of a piece, and the workspace's parts.
struct Plan {
  int piece;
  size_t logits, rows, state, gemm;  // bytes
  size_t total() const { return logits + rows + state + gemm; }
};
constexpr size_t kPieceBytes = (size_t)128 << 20;
Plan plan_of(int rows, int d, int vocab) {
  Plan p;
  const size_t cols = kPieceBytes / sizeof(float) / (size_t)rows / 256 * 256;
  p.piece = (int)std::min<size_t>((size_t)vocab, std::max<size_t>(cols, 256));
  p.logits = round256((size_t)rows * p.piece * sizeof(float));
  p.rows = round256((size_t)rows * d * sizeof(float));
  p.state = round256((size_t)rows * sizeof(RowState));
  const int last = vocab % p.piece ? vocab % p.piece : p.piece;
  p.gemm = 0;
  for (int v : {p.piece, last})
    p.gemm = std::max(p.gemm, std::max(mle_gemm_ws_bytes(rows, v, d, 1),
                                       std::max(mle_gemm_ws_bytes(rows, d, v, 1), mle_gemm_ws_bytes(d, v, rows, 1))));
  p.gemm = round256(p.gemm);
  return p;
}

int check(const char* who, int rows, int d, int vocab, const float* X, int64_t ldx, const float* W, int64_t ldw,
          const int32_t* keys, int clen, int max_clen) {
  MLE_CHECK_ARG(rows >= 0 && d > 0 && vocab > 0, "%s: bad shape (rows %d, d %d, vocab %d)", who, rows, d, vocab);
  MLE_CHECK_ARG(W && (rows == 0 || (X && keys)), "%s: null pointer", who);
  MLE_CHECK_ARG(ldx >= d && ldw >= vocab, "%s: ldx %lld < %d or ldw %lld < %d", who, (long long)ldx, d, (long long)ldw,
                vocab);
  MLE_CHECK_ARG(clen > 0 && max_clen >= clen, "%s: clen %d, max_clen %d", who, clen, max_clen);
  return MLE_OK;
}
int check_ws(const char* who, size_t need, const void* ws, size_t ws_bytes) {
  if (need && (!ws || !aligned16(ws) || ws_bytes < need))
    return set_error(MLE_ERR_WORKSPACE, "%s: workspace of %zu bytes, 16-byte aligned, needed", who, need);
  return MLE_OK;
}

#define TRY(call)                  \
  do {                             \
    const int rc_ = (call);        \
    if (rc_ != MLE_OK) return rc_; \
  } while (0)

}  // namespace

extern "C" {

size_t mle_vocab_xent_ws_bytes(int rows, int d, int vocab) {
  return rows <= 0 || d <= 0 || vocab <= 0 ? 0 : plan_of(rows, d, vocab).total();
}

int mle_vocab_xent_fwd(mle_stream stream, int rows, int d, int vocab, const float* X, int64_t ldx, const float* W,
                       int64_t ldw, const float* bias, const int32_t* keys, int clen, int max_clen, float loss_scale,
                       float* lse, float* row_loss, float* loss, void* ws, size_t ws_bytes) {
  TRY(check("mle_vocab_xent_fwd", rows, d, vocab, X, ldx, W, ldw, keys, clen, max_clen));
  MLE_CHECK_ARG(loss && (lse || rows == 0), "mle_vocab_xent_fwd: null pointer");
  if (rows == 0) return mle_fill(stream, loss, 0.f, 1);
  const Plan p = plan_of(rows, d, vocab);
  TRY(check_ws("mle_vocab_xent_fwd", p.total(), ws, ws_bytes));
  hipStream_t s = as_stream(stream);
  const Rows rw{keys, clen, max_clen, vocab};
  float* l = static_cast<float*>(ws);
  RowState* state = reinterpret_cast<RowState*>(static_cast<char*>(ws) + p.logits + p.rows);
  void* gws = reinterpret_cast<char*>(state) + p.state;
  for (int v0 = 0; v0 < vocab; v0 += p.piece) {
    const int n = std::min(p.piece, vocab - v0);
    TRY(mle_gemm_ex(stream, 0, 0, rows, n, d, 1.f, X, ldx, 0, W + v0, ldw, 0, 0.f, l, n, 0, 1, nullptr,
                    bias ? bias + v0 : nullptr, gws, p.gemm));
    mle::launch(xent_stats_kernel, (unsigned)rows, NT, 0, s, l, n, v0, rw, state, v0 == 0 ? 1 : 0);
  }
  mle::launch(xent_finish_kernel, 1u, 1024, 0, s, state, rows, rw, loss_scale, lse, row_loss, loss);
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
  const Plan p = rows > 0 ? plan_of(rows, d, vocab) : Plan{};
  if (rows > 0) TRY(check_ws("mle_vocab_xent_bwd", p.total(), ws, ws_bytes));
  if (db && !accumulate_dw) TRY(mle_fill(stream, db, 0.f, (size_t)vocab));
  if (rows == 0) {
    if (dW && !accumulate_dw)
      TRY(mle_gemm_ex(stream, 1, 0, d, vocab, 0, 1.f, nullptr, d, 0, nullptr, vocab, 0, 0.f, dW, lddw, 0, 1, nullptr, nullptr,
                      nullptr, 0));
    return MLE_OK;
  }
  if (!dX && !dW) return MLE_OK;
  hipStream_t s = as_stream(stream);
  const Rows rw{keys, clen, max_clen, vocab};
  float* l = static_cast<float*>(ws);
  float* xs = reinterpret_cast<float*>(static_cast<char*>(ws) + p.logits);
  void* gws = static_cast<char*>(ws) + p.logits + p.rows + p.state;
  if (dW) mle::launch(xent_rows_kernel, (unsigned)rows, NT, 0, s, X, ldx, d, rw, xs);
  for (int v0 = 0; v0 < vocab; v0 += p.piece) {
    const int n = std::min(p.piece, vocab - v0);
    TRY(mle_gemm_ex(stream, 0, 0, rows, n, d, 1.f, X, ldx, 0, W + v0, ldw, 0, 0.f, l, n, 0, 1, nullptr,
                    bias ? bias + v0 : nullptr, gws, p.gemm));
    mle::launch(xent_grad_kernel, (unsigned)rows, NT, 0, s, l, n, v0, rw, lse, upstream, grad_scale);
    if (dX)
      TRY(mle_gemm_ex(stream, 0, 1, rows, d, n, 1.f, l, n, 0, W + v0, ldw, 0, accumulate_dx || v0 > 0 ? 1.f : 0.f, dX,
                      lddx, 0, 1, nullptr, nullptr, gws, p.gemm));
    if (dW)
      TRY(mle_gemm_ex(stream, 1, 0, d, n, rows, 1.f, xs, d, 0, l, n, 0, accumulate_dw ? 1.f : 0.f, dW + v0, lddw, 0, 1,
                      db ? db + v0 : nullptr, nullptr, gws, p.gemm));
  }
  return check_launch("mle_vocab_xent_bwd");
}

}  // extern "C"
