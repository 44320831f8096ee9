// Attention over the keys that a causal sliding window and a few first positions
// (sinks) leave visible: what its kernels share, and the plain forms of a row.
//
//   S = scale q k^T,  P = exp(S - lse),  out = P v        along the visible keys
//   D = <dout, out>,  dS = P (dout v^T - D)
//   dq = scale dS k,  dk = scale dS^T q,  dv = P^T dout   (dk, dv over a group's heads)
#pragma once
#include "common.hpp"

namespace wattn {

constexpr int kMaxDim = 128;

struct Args {
  const float *q, *k, *v, *out_in, *dout;  // out_in: the forward's, read by the backward
  float *out, *lse;
  const float* lse_in;
  float *dq, *dk, *dv;
  float* delta;  // D, [batch, heads, rows]
  int64_t ldq, ldk, ldv, ldo, lddo, lddq, lddk, lddv;
  const int32_t* lengths;
  int batch, rows, keys;   // rows of q and keys of k of a sequence
  int heads, kv_heads, group, dim;
  int window, sinks;       // at most `keys` each
  int at_end;              // row i is at position length - rows + i (else at i)
  int acc_q, acc_k, acc_v;
  float scale;
};

// A sequence: its length and the position of its first row.
struct Seq {
  int len, first;
  __device__ __forceinline__ Seq(const Args& a, int b) {
    len = a.lengths ? min(max(a.lengths[b], 0), a.keys) : a.keys;
    first = a.at_end ? len - a.rows : 0;
  }
};

// Key number t of the `count` that position p sees, in order: the sinks before the
// window, then the window.
struct Seen {
  int before, low, count;
  __device__ __forceinline__ Seen(const Args& a, int p) {
    low = max(p - a.window + 1, 0);
    before = min(a.sinks, low);
    count = before + p + 1 - low;
  }
  __device__ __forceinline__ int key(int t) const { return t < before ? t : low + t - before; }
};

// (Without branches, and its users choose values by it: a vector's element set to minus
// infinity under a condition has been compiled into a copy that some lanes skip.)
__device__ __forceinline__ bool sees(const Args& a, int p, int j) {
  return (j <= p) & ((p - j < a.window) | (j < a.sinks));
}

// ---------------------------------------------------------------- plain forms
// A row (or a key) to a wave, with fp32 products, visible pairs only: what holds
// for infinities and NaN, which a product of tiles would carry to rows that do not
// see them.  The fast kernels run these for their rows where a sum is not finite.

__device__ __forceinline__ float dot(const float* __restrict__ x, const float* __restrict__ y, int n) {
  float s = 0.f;
  for (int d = 0; d < n; ++d) s = fmaf(x[d], y[d], s);
  return s;
}

// Row i of sequence b and head h: out and lse.
static __device__ void plain_row(const Args& a, int b, int h, int i) {
  const int lane = threadIdx.x & 63;
  const Seq s(a, b);
  const int p = s.first + i, e = h / a.group;
  float* out = a.out + ((int64_t)b * a.rows + i) * a.ldo + (int64_t)h * a.dim;
  float* lse = a.lse ? a.lse + ((int64_t)b * a.heads + h) * a.rows + i : nullptr;
  if (p < 0 || p >= s.len) {
    for (int d = lane; d < a.dim; d += 64) out[d] = 0.f;
    if (lse && lane == 0) *lse = -INFINITY;
    return;
  }
  const float* q = a.q + ((int64_t)b * a.rows + i) * a.ldq + (int64_t)h * a.dim;
  const float* k = a.k + (int64_t)b * a.keys * a.ldk + (int64_t)e * a.dim;
  const float* v = a.v + (int64_t)b * a.keys * a.ldv + (int64_t)e * a.dim;
  const Seen seen(a, p);
  float m = -INFINITY;
  bool nan = false;
  for (int t = lane; t < seen.count; t += 64) {
    const float x = a.scale * dot(q, k + seen.key(t) * a.ldk, a.dim);
    nan |= x != x;
    m = fmaxf(m, x);
  }
  m = wave_max(m);
  if (__any(nan)) m = NAN;
  float l = 0.f, o[2] = {0.f, 0.f};
  for (int t0 = 0; t0 < seen.count; t0 += 64) {
    const int n = min(seen.count - t0, 64), j = seen.key(min(t0 + lane, seen.count - 1));
    const float x = a.scale * dot(q, k + j * a.ldk, a.dim);
    const float w = lane < n ? expf(x - m) : 0.f;
    l += w;
    float c[2] = {0.f, 0.f};
    for (int u = 0; u < n; ++u) {
      const float wu = __shfl(w, u, 64);
      const float* row = v + (int64_t)__shfl(j, u, 64) * a.ldv;
#pragma unroll
      for (int r = 0; r < 2; ++r)
        if (lane + 64 * r < a.dim) c[r] = fmaf(wu, row[lane + 64 * r], c[r]);
    }
    o[0] += c[0];
    o[1] += c[1];
  }
  l = wave_sum(l);
#pragma unroll
  for (int r = 0; r < 2; ++r)
    if (lane + 64 * r < a.dim) out[lane + 64 * r] = o[r] / l;
  if (lse && lane == 0) *lse = m + logf(l);
}

// P and dS / scale of row i at key j, from their rows.
__device__ __forceinline__ void pair(const Args& a, const float* q, const float* k, const float* v, const float* dout,
                                     float lse, float delta, float& p, float& ds) {
  p = expf(a.scale * dot(q, k, a.dim) - lse);
  ds = p * (dot(dout, v, a.dim) - delta);
}

// dq of row i of sequence b and head h (delta filled).
static __device__ void plain_dq(const Args& a, int b, int h, int i) {
  const int lane = threadIdx.x & 63;
  const Seq s(a, b);
  const int e = h / a.group;
  const int64_t at = (int64_t)b * a.rows + i, st = ((int64_t)b * a.heads + h) * a.rows + i;
  float* dq = a.dq + at * a.lddq + (int64_t)h * a.dim;
  float o[2] = {0.f, 0.f};
  if (i < s.len) {
    const float* q = a.q + at * a.ldq + (int64_t)h * a.dim;
    const float* g = a.dout + at * a.lddo + (int64_t)h * a.dim;
    const float* k = a.k + (int64_t)b * a.keys * a.ldk + (int64_t)e * a.dim;
    const float* v = a.v + (int64_t)b * a.keys * a.ldv + (int64_t)e * a.dim;
    const Seen seen(a, i);
    for (int t0 = 0; t0 < seen.count; t0 += 64) {
      const int n = min(seen.count - t0, 64), j = seen.key(min(t0 + lane, seen.count - 1));
      float p, ds, c[2] = {0.f, 0.f};
      pair(a, q, k + j * a.ldk, v + j * a.ldv, g, a.lse_in[st], a.delta[st], p, ds);
      for (int u = 0; u < n; ++u) {
        const float du = __shfl(ds, u, 64);
        const float* row = k + (int64_t)__shfl(j, u, 64) * a.ldk;
#pragma unroll
        for (int r = 0; r < 2; ++r)
          if (lane + 64 * r < a.dim) c[r] = fmaf(du, row[lane + 64 * r], c[r]);
      }
      o[0] += c[0];
      o[1] += c[1];
    }
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int d = lane + 64 * r;
    if (d < a.dim) dq[d] = (a.acc_q ? dq[d] : 0.f) + a.scale * o[r];
  }
}

// Sums over queries [i0, i1) of head h that see key j of sequence b: ds q (times scale) and p dout.
static __device__ void plain_kv_sums(const Args& a, int b, int h, int j, int i0, int i1, float (&sk)[2], float (&sv)[2]) {
  const int lane = threadIdx.x & 63, e = h / a.group;
  const float* k = a.k + ((int64_t)b * a.keys + j) * a.ldk + (int64_t)e * a.dim;
  const float* v = a.v + ((int64_t)b * a.keys + j) * a.ldv + (int64_t)e * a.dim;
  const float* q = a.q + (int64_t)b * a.rows * a.ldq + (int64_t)h * a.dim;
  const float* g = a.dout + (int64_t)b * a.rows * a.lddo + (int64_t)h * a.dim;
  const int64_t st = ((int64_t)b * a.heads + h) * a.rows;
  for (int t0 = i0; t0 < i1; t0 += 64) {
    const int n = min(i1 - t0, 64), i = min(t0 + lane, i1 - 1);
    float p, ds, ck[2] = {0.f, 0.f}, cv[2] = {0.f, 0.f};
    pair(a, q + i * a.ldq, k, v, g + i * a.lddo, a.lse_in[st + i], a.delta[st + i], p, ds);
    for (int u = 0; u < n; ++u) {
      const float pu = __shfl(p, u, 64), du = __shfl(ds, u, 64);
#pragma unroll
      for (int r = 0; r < 2; ++r)
        if (lane + 64 * r < a.dim) {
          ck[r] = fmaf(du, q[(t0 + u) * a.ldq + lane + 64 * r], ck[r]);
          cv[r] = fmaf(pu, g[(t0 + u) * a.lddo + lane + 64 * r], cv[r]);
        }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      sk[r] = fmaf(a.scale, ck[r], sk[r]);
      sv[r] += cv[r];
    }
  }
}

}  // namespace wattn
