// The entry points of the windowed attention: checks, workspaces, and which kernels run.
#include "window_attention.hpp"
#include "window_kernels.hpp"

#include <math.h>
#include <algorithm>

using namespace mle;
using namespace wattn;

namespace {

int check(const char* who, int batch, int rows, int keys, int heads, int kv_heads, int dim, float scale, int window,
          int sinks) {
  MLE_CHECK_ARG(batch >= 0 && batch <= (1 << 24) && rows >= 0 && keys >= 0 && rows <= (1 << 30) && keys <= (1 << 30),
                "%s: bad shape, %d sequences of %d rows and %d keys", who, batch, rows, keys);
  MLE_CHECK_ARG(heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && heads <= (1 << 16), "%s: %d heads on %d of keys", who,
                heads, kv_heads);
  MLE_CHECK_ARG(dim > 0, "%s: head_dim %d", who, dim);
  MLE_CHECK_ARG(window >= 1 && sinks >= 0, "%s: window %d (at least 1), sinks %d (at least 0)", who, window, sinks);
  MLE_CHECK_ARG((double)batch * heads * std::max(rows, keys) <= 1e12, "%s: %d sequences of %d rows, %d heads", who, batch, rows,
                heads);
  MLE_CHECK_ARG(isfinite(scale), "%s: scale %g", who, (double)scale);
  if (dim > kMaxDim) return set_error(MLE_ERR_UNSUPPORTED, "%s: head_dim %d, at most %d", who, dim, kMaxDim);
  return MLE_OK;
}

// Are these sizes that check() passes?  (The workspace queries answer 0 for others, and compute
// with none of them.)
bool takes(int batch, int rows, int keys, int heads, int kv_heads, int dim) {
  return batch > 0 && batch <= (1 << 24) && rows > 0 && rows <= (1 << 30) && keys > 0 && keys <= (1 << 30) && heads > 0 &&
         heads <= (1 << 16) && kv_heads > 0 && heads % kv_heads == 0 && dim > 0 && dim <= kMaxDim &&
         (double)batch * heads * std::max(rows, keys) <= 1e12;
}

int check_ld(const char* who, const char* name, int64_t ld, int heads, int dim) {
  MLE_CHECK_ARG(ld >= (int64_t)heads * dim && ld <= ((int64_t)1 << 32), "%s: %s %lld for %d heads of %d", who, name,
                (long long)ld, heads, dim);
  return MLE_OK;
}

Args make_args(const float* q, int64_t ldq, const float* k, int64_t ldk, const float* v, int64_t ldv, int64_t ldo,
               const int32_t* lengths, int batch, int rows, int keys, int heads, int kv_heads, int dim, float scale,
               int window, int sinks) {
  Args a{};
  a.q = q, a.k = k, a.v = v;
  a.ldq = ldq, a.ldk = ldk, a.ldv = ldv, a.ldo = ldo;
  a.lengths = lengths;
  a.batch = batch, a.rows = rows, a.keys = keys;
  a.heads = heads, a.kv_heads = kv_heads, a.group = heads / kv_heads, a.dim = dim;
  a.window = std::min(window, std::max(keys, 1)), a.sinks = std::min(sinks, keys);
  a.scale = scale;
  return a;
}

}  // namespace

extern "C" {

int mle_window_attention_fwd(mle_stream stream, const float* q, int64_t ldq, const float* k, int64_t ldk,
                             const float* v, int64_t ldv, float* out, int64_t ldo, float* lse, const int32_t* lengths,
                             int batch, int seq, int heads, int kv_heads, int head_dim, float scale, int window,
                             int sinks) {
  const char* who = "mle_window_attention_fwd";
  int rc = check(who, batch, seq, seq, heads, kv_heads, head_dim, scale, window, sinks);
  if (!rc) rc = check_ld(who, "ldq", ldq, heads, head_dim);
  if (!rc) rc = check_ld(who, "ldk", ldk, kv_heads, head_dim);
  if (!rc) rc = check_ld(who, "ldv", ldv, kv_heads, head_dim);
  if (!rc) rc = check_ld(who, "ldo", ldo, heads, head_dim);
  if (rc) return rc;
  if (batch == 0 || seq == 0) return MLE_OK;
  MLE_CHECK_ARG(q && k && v && out, "%s: null pointer", who);
  Args a = make_args(q, ldq, k, ldk, v, ldv, ldo, lengths, batch, seq, seq, heads, kv_heads, head_dim, scale, window, sinks);
  a.out = out;
  a.lse = lse;
  tile_forward(a, as_stream(stream));
  return check_launch(who);
}

size_t mle_window_attention_ws_bytes(int batch, int seq, int heads, int kv_heads, int head_dim, int window, int sinks) {
  if (!takes(batch, seq, seq, heads, kv_heads, head_dim)) return 0;
  Args a = make_args(nullptr, 0, nullptr, 0, nullptr, 0, 0, nullptr, batch, seq, seq, heads, kv_heads, head_dim, 1.f,
                     std::max(window, 1), std::max(sinks, 0));
  return BwdWork(a).place(a, nullptr);
}

int mle_window_attention_bwd(mle_stream stream, const float* q, int64_t ldq, const float* k, int64_t ldk,
                             const float* v, int64_t ldv, const float* out, int64_t ldo, const float* lse,
                             const float* dout, int64_t lddo, float* dq, int64_t lddq, int acc_q, float* dk,
                             int64_t lddk, int acc_k, float* dv, int64_t lddv, int acc_v, const int32_t* lengths,
                             int batch, int seq, int heads, int kv_heads, int head_dim, float scale, int window,
                             int sinks, void* ws, size_t ws_bytes) {
  const char* who = "mle_window_attention_bwd";
  int rc = check(who, batch, seq, seq, heads, kv_heads, head_dim, scale, window, sinks);
  if (!rc) rc = check_ld(who, "ldq", ldq, heads, head_dim);
  if (!rc) rc = check_ld(who, "ldk", ldk, kv_heads, head_dim);
  if (!rc) rc = check_ld(who, "ldv", ldv, kv_heads, head_dim);
  if (!rc) rc = check_ld(who, "ldo", ldo, heads, head_dim);
  if (!rc) rc = check_ld(who, "lddo", lddo, heads, head_dim);
  if (!rc) rc = check_ld(who, "lddq", lddq, heads, head_dim);
  if (!rc) rc = check_ld(who, "lddk", lddk, kv_heads, head_dim);
  if (!rc) rc = check_ld(who, "lddv", lddv, kv_heads, head_dim);
  if (rc) return rc;
  if (batch == 0 || seq == 0) return MLE_OK;
  MLE_CHECK_ARG(q && k && v && out && lse && dout && dq && dk && dv, "%s: null pointer", who);
  const size_t need = mle_window_attention_ws_bytes(batch, seq, heads, kv_heads, head_dim, window, sinks);
  if (!ws || !aligned16(ws) || ws_bytes < need)
    return set_error(MLE_ERR_WORKSPACE, "%s: workspace of %zu bytes, 16-byte aligned, needed", who, need);
  Args a = make_args(q, ldq, k, ldk, v, ldv, ldo, lengths, batch, seq, seq, heads, kv_heads, head_dim, scale, window, sinks);
  a.out_in = out, a.lse_in = lse, a.dout = dout, a.lddo = lddo;
  a.dq = dq, a.dk = dk, a.dv = dv;
  a.lddq = lddq, a.lddk = lddk, a.lddv = lddv;
  a.acc_q = acc_q != 0, a.acc_k = acc_k != 0, a.acc_v = acc_v != 0;
  BwdWork w(a);
  w.place(a, ws);
  tile_backward(a, w, as_stream(stream));
  return check_launch(who);
}

size_t mle_window_attention_step_ws_bytes(int batch, int tokens, int capacity, int heads, int kv_heads, int head_dim,
                                          int window, int sinks) {
  if (!takes(batch, tokens, capacity, heads, kv_heads, head_dim)) return 0;
  const Args a = make_args(nullptr, 0, nullptr, 0, nullptr, 0, 0, nullptr, batch, tokens, capacity, heads, kv_heads, head_dim,
                           1.f, std::max(window, 1), std::max(sinks, 0));
  return StepWork::few(tokens) ? StepWork(a).bytes(a) : 0;
}

int mle_window_attention_step(mle_stream stream, const float* q, int64_t ldq, const float* k, int64_t ldk,
                              const float* v, int64_t ldv, float* out, int64_t ldo, const int32_t* lengths, int batch,
                              int tokens, int capacity, int heads, int kv_heads, int head_dim, float scale, int window,
                              int sinks, void* ws, size_t ws_bytes) {
  const char* who = "mle_window_attention_step";
  int rc = check(who, batch, tokens, capacity, heads, kv_heads, head_dim, scale, window, sinks);
  if (!rc) rc = check_ld(who, "ldq", ldq, heads, head_dim);
  if (!rc) rc = check_ld(who, "ldk", ldk, kv_heads, head_dim);
  if (!rc) rc = check_ld(who, "ldv", ldv, kv_heads, head_dim);
  if (!rc) rc = check_ld(who, "ldo", ldo, heads, head_dim);
  if (rc) return rc;
  if (batch == 0 || tokens == 0) return MLE_OK;
  MLE_CHECK_ARG(q && out && lengths && (capacity == 0 || (k && v)), "%s: null pointer", who);
  Args a = make_args(q, ldq, k, ldk, v, ldv, ldo, lengths, batch, tokens, capacity, heads, kv_heads, head_dim, scale, window,
                     sinks);
  a.out = out;
  a.at_end = 1;
  if (!StepWork::few(tokens)) {
    tile_forward(a, as_stream(stream));
    return check_launch(who);
  }
  StepWork w(a);
  const size_t need = w.bytes(a);
  if (need > 0 && (!ws || !aligned16(ws) || ws_bytes < need))
    return set_error(MLE_ERR_WORKSPACE, "%s: workspace of %zu bytes, 16-byte aligned, needed", who, need);
  w.part = static_cast<float*>(ws);
  step_forward(a, w, as_stream(stream));
  return check_launch(who);
}

}  // extern "C"
