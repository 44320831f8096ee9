// What the backward's passes share (window_bwd.hip, window_bwd_wide.hip).
#pragma once
#include "window_tile.hpp"
#include "window_kernels.hpp"

namespace wattn {

constexpr int kOdd = 1 << 20;   // in place of a row's exponent: something in it is not finite
constexpr int kNone = -(1 << 20);
constexpr int kTileRows = 64;   // of wk.tile_ex
constexpr int kUnit = -10;  // dP and D of a row are taken times 2^(kUnit - exponent of its dout), at most V's largest

// Where a column's largest is brought to when it has grown out of an operand, 2^15 (log2): what
// lies below is off by at most 2^-25, 2^-37 of that largest.  (8 in place of 12: 1 to 2 % less time
// at 2 x 16 heads of 4096 x 128, 16 times the error of the smallest.)
constexpr int kHeld = 12;

// A column's operand held at 2^t: where its largest, mx of a lane and of the lane's other
// half, would reach 2^15, t is lowered to bring it to [2^kHeld, 2^(kHeld + 1)), and the sums follow.
template <int N>
__device__ __forceinline__ void rescale(float mx, int& t, f32x16 (&sums)[N]) {
  if (!__any(exponent(mx) + t > 14 || t > 120)) return;
  const int e = exponent(fmaxf(mx, other_half(mx)));
  const bool over = e + t > 14 || t > 120;
  const int to = over ? min(kHeld - e, 120) : t;
#pragma unroll
  for (int d = 0; d < N; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) sums[d][r] = __builtin_amdgcn_ldexpf(sums[d][r], to - t);
  t = to;
}

// Four of a row's values from column `col`, added to `old` where that is not null.
__device__ __forceinline__ void store4(float* out, const float* old, int col, int dim, float (&x)[4]) {
  if (col + 4 <= dim) {
    f32x4u v = {x[0], x[1], x[2], x[3]};
    if (old) v += *reinterpret_cast<const f32x4u*>(old + col);
    *reinterpret_cast<f32x4u*>(out + col) = v;
  } else {
#pragma unroll
    for (int n = 0; n < 4; ++n)
      if (col + n < dim) out[col + n] = old ? old[col + n] + x[n] : x[n];
  }
}

// One of a key's two sums as plain_kv_sums leaves them in a wave, to dk (dv) or (part) to the
// workgroup's share.
__device__ __forceinline__ void store_plain(const Args& a, float* part, int b, int e, int key, int local, bool dk,
                                            const float (&sum)[2]) {
  const int lane = threadIdx.x & 63;
  float* out = part ? part + ((dk ? 0 : kKeyBlock) + local) * a.dim
             : dk ? a.dk + ((int64_t)b * a.keys + key) * a.lddk + (int64_t)e * a.dim
                  : a.dv + ((int64_t)b * a.keys + key) * a.lddv + (int64_t)e * a.dim;
  const bool add = !part && (dk ? a.acc_k : a.acc_v);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int d = lane + 64 * r;
    if (d < a.dim) out[d] = (add ? out[d] : 0.f) + sum[r];
  }
}

// A row's part in the kv pass, by row of a tile.  (Read four rows at a time from arrays of these.)
template <int R>
struct alignas(16) Rows {
  static_assert(R % 4 == 0, "delta on 16 bytes");
  float lse[R];    // its log-sum less its exponent (log2 units); infinity: not there
  float delta[R];  // D in the units of dP
  int ex[R];
  unsigned odd;    // set where one is not finite
  // From a row's log-sum, D and exponent, each of the first 64 threads having one (R = 32: two
  // the same).
  __device__ __forceinline__ void put(int r0, int end, int ex0, float r_lse, float r_delta, int r_ex) {
    if (threadIdx.x >= 64) return;
    const int n = threadIdx.x % R;
    const bool there = r0 + n < end, bad = there && r_ex == kOdd;
    const int x = there && !bad ? r_ex : 0;
    ex[n] = x;
    lse[n] = there ? r_lse * kLog2e - (float)(x - ex0) : INFINITY;
    delta[n] = there ? __builtin_amdgcn_ldexpf(r_delta, kUnit - x) : 0.f;
    const unsigned any = __any(bad) ? 1u : 0u;
    if (threadIdx.x == 0) odd = any;
  }
};

// A workgroup's part of the kv pass: kKeyBlock keys, and rows of every head of the group.
struct KvJob {
  int b, e, k0, i_begin, i_end;
  float* part;  // where its sums go, or null: to dk and dv
  __device__ __forceinline__ KvJob(const Args& a, const BwdWork& wk, const Place& p) {
    b = (int)(p.group / a.kv_heads), e = (int)(p.group % a.kv_heads);
    const int len = Seq(a, b).len, fi = p.item - wk.key_blocks * wk.nears;  // (the far ones last: they are short)
    const int64_t size = 2 * (int64_t)kKeyBlock * a.dim;
    if (fi < 0) {
      const int blk = p.item / wk.nears, chunk = p.item % wk.nears;
      k0 = blk * kKeyBlock;
      i_begin = k0 + chunk * wk.near_rows;
      i_end = min(min(i_begin + wk.near_rows, wk.near_end(a, k0)), len);
      part = wk.nears > 1 ? wk.near + ((p.group * wk.key_blocks + blk) * wk.nears + chunk) * size : nullptr;
    } else {
      const int blk = fi / wk.fars, chunk = fi % wk.fars;
      k0 = blk * kKeyBlock;
      i_begin = wk.near_end(a, k0) + chunk * wk.far_rows;
      i_end = min(i_begin + wk.far_rows, len);
      part = wk.far + ((p.group * wk.sink_blocks + blk) * wk.fars + chunk) * size;
    }
  }
  // The largest exponent of its rows of dout, in ex[wave].
  __device__ __forceinline__ void largest(const Args& a, const BwdWork& wk, int* ex) const {
    int m = kNone;
    const int n = (i_end - i_begin + kTileRows - 1) / kTileRows;
    for (int t = threadIdx.x; t < n * a.group; t += blockDim.x) {
      const int64_t bh = (int64_t)b * a.heads + e * a.group + t / n;
      m = max(m, wk.tile_ex[bh * wk.tiles + i_begin / kTileRows + t % n]);
    }
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) m = max(m, __shfl_xor(m, x, 64));
    if ((threadIdx.x & 63) == 0) ex[threadIdx.x >> 6] = m;
  }
  // Sums of 32 keys from kw on with fp32 products, by one wave.
  __device__ __forceinline__ void plain(const Args& a, int kw, bool dk, bool dv) const {
    const int len = Seq(a, b).len;
    for (int key = kw; key < min(kw + 32, a.keys); ++key) {
      float sk[2] = {0.f, 0.f}, sv[2] = {0.f, 0.f};
      const int end = key < a.sinks ? i_end : (int)min((int64_t)i_end, (int64_t)key + a.window);
      if (key < len)
        for (int q = 0; q < a.group; ++q) plain_kv_sums(a, b, e * a.group + q, key, max(key, i_begin), end, sk, sv);
      if (dk) store_plain(a, part, b, e, key, key - k0, true, sk);
      if (dv) store_plain(a, part, b, e, key, key - k0, false, sv);
    }
  }
};

// The tiles of R rows of each head in turn; past the last comes the last once more (loads of it go
// unused: no branches around loads).
template <int R>
struct Walk {
  int h, r0, h_end, begin, end;
  __device__ __forceinline__ Walk(const Args& a, const KvJob& job)
      : h(job.e * a.group), r0(job.i_begin), h_end(h + a.group), begin(r0), end(job.i_end) {}
  __device__ __forceinline__ void next() {
    const bool more = r0 + R < end;
    r0 = more ? r0 + R : h + 1 < h_end ? begin : r0;
    h = more ? h : min(h + 1, h_end - 1);
  }
};

void launch_wide(const Args& a, const BwdWork& w, hipStream_t s);

}  // namespace wattn
