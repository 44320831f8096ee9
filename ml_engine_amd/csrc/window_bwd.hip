// Backward of the windowed attention, in passes that each write their own gradients, so
// that no sum depends on timing:
//   prepare   D and the exponent of each row of dout
//   kv        dk and dv of 32 keys to a wave, over the tiles of rows that see them
//   q         dq of 32 rows to a wave, over the tiles of keys that they see
//   join      sinks: the sums over rows past their own window, added in order
// S and dP = dout v^T are computed again in both.
//
// Sinks are seen by every later row.  Blocks of keys with sinks take the rows up to their
// window like all others ("near"); the rows after it ("far") are shared out over workgroups
// whose sums lie in the workspace.
//
// Scales.  A product sums over rows (kv) or keys (q) whose probabilities and gradients may be
// of very unlike size, so the operands that are made here are held at powers of two of their
// own column, a lane's: a key's P and dS (kv), a row's dS (q) have the largest seen so far
// between 2^8 and 2^15, and a larger one rescales the lane's sums.  Rows of dout are at powers
// of two of their own too; P takes those up in its exponent.
#include "window_tile.hpp"
#include "window_kernels.hpp"

using namespace mle;

namespace wattn {
namespace {

constexpr int kOdd = 1 << 20;   // in place of a row's exponent: something in it is not finite
constexpr int kNone = -(1 << 20);
constexpr int kTileRows = 64;   // of wk.tile_ex
constexpr int kUnit = -10;  // dP and D of a row are taken times 2^(kUnit - exponents of its dout and of V): below 1

// D, and the exponents, of 64 rows of a head; four lanes to a row.
__global__ __launch_bounds__(256) void prepare_kernel(Args a, BwdWork wk, int64_t first) {
  __shared__ int red[4];
  const int64_t id = first + blockIdx.x;
  const int tile = (int)(id % wk.tiles);
  const int64_t bh = id / wk.tiles;
  const int b = (int)(bh / a.heads), h = (int)(bh % a.heads);
  const int sub = threadIdx.x & 3, i = tile * kTileRows + (threadIdx.x >> 2);
  const Seq seq(a, b);
  float s = 0.f, m = 0.f;
  if (i < seq.len) {
    const float* g = a.dout + ((int64_t)b * a.rows + i) * a.lddo + (int64_t)h * a.dim;
    const float* o = a.out_in + ((int64_t)b * a.rows + i) * a.ldo + (int64_t)h * a.dim;
    for (int c = 4 * sub; c < a.dim; c += 16) {
      if (c + 4 <= a.dim) {
        const f32x4u x = *reinterpret_cast<const f32x4u*>(g + c), y = *reinterpret_cast<const f32x4u*>(o + c);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s = fmaf(x[j], y[j], s);
          m = fmaxf(m, fabsf(x[j]));
        }
      } else {
        for (int j = c; j < a.dim; ++j) {
          s = fmaf(g[j], o[j], s);
          m = fmaxf(m, fabsf(g[j]));
        }
      }
    }
  }
#pragma unroll
  for (int x = 1; x < 4; x <<= 1) {
    s += __shfl_xor(s, x, 64);
    m = fmaxf(m, __shfl_xor(m, x, 64));
  }
  int ex = kNone;
  if (i < seq.len) {
    const int64_t at = bh * a.rows + i;
    // (a NaN in dout is one in D)
    const bool odd = !(m < INFINITY) || !(fabsf(s) < INFINITY) || !(fabsf(a.lse_in[at]) < INFINITY);
    if (!odd) ex = exponent(m);
    if (sub == 0) {
      a.delta[at] = s;
      wk.ex[at] = odd ? kOdd : ex;
    }
  }
#pragma unroll
  for (int x = 4; x < 64; x <<= 1) ex = max(ex, __shfl_xor(ex, x, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = ex;
  __syncthreads();
  if (threadIdx.x == 0) wk.tile_ex[id] = max(max(red[0], red[1]), max(red[2], red[3]));
}

// A column's operand held at 2^t: where its largest, mx of a lane and of the lane's other
// half, would reach 2^15, t is lowered to bring it to 2^8 .. 2^9, and the sums follow.
template <int N>
__device__ __forceinline__ void rescale(float mx, int& t, f32x16 (&sums)[N]) {
  mx = fmaxf(mx, other_half(mx));
  const int e = exponent(mx);
  const bool over = e + t > 14 || t > 120;
  if (!__any(over)) return;
  const int to = over ? min(8 - e, 120) : t;
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

// A key's sums as plain_kv_sums leaves them in a wave, to its gradients or (part) to the
// workgroup's share of far sums.
__device__ __forceinline__ void store_plain(const Args& a, float* part, int kb, int b, int e, int key, int local,
                                            const float (&sk)[2], const float (&sv)[2]) {
  const int lane = threadIdx.x & 63;
  float* ok = part ? part + local * a.dim : a.dk + ((int64_t)b * a.keys + key) * a.lddk + (int64_t)e * a.dim;
  float* ov = part ? part + (kb + local) * a.dim : a.dv + ((int64_t)b * a.keys + key) * a.lddv + (int64_t)e * a.dim;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int d = lane + 64 * r;
    if (d >= a.dim) continue;
    ok[d] = (a.acc_k && !part ? ok[d] : 0.f) + sk[r];
    ov[d] = (a.acc_v && !part ? ov[d] : 0.f) + sv[r];
  }
}

// A row's part in the kv pass, by row of a tile.
template <int R>
struct Rows {
  float lse[R];    // its log-sum less its exponent (log2 units); infinity: not there
  float delta[R];  // D in the units of dP
  int ex[R];
  unsigned odd;    // set where one is not finite
};

template <int DP, int NW>
__global__ __launch_bounds__(64 * NW, DP <= 64 ? 2 : 1) void kv_kernel(Args a, BwdWork wk, Grid g) {
  using T = Tile<DP>;
  constexpr int NT = 64 * NW, KB = 32 * NW, R = T::R, AHEAD = 1;
  __shared__ __attribute__((aligned(16))) char lds[2][2][T::BYTES];  // [buffer][Q, dout]
  __shared__ __attribute__((aligned(16))) Rows<R> rows[4];
  __shared__ __attribute__((aligned(16))) Tops<NW> tops;
  __shared__ int shared_ex[NW], shared_ev[NW];
  const Place pl = g.place();
  const int b = (int)(pl.group / a.kv_heads), e = (int)(pl.group % a.kv_heads);
  const Seq seq(a, b);
  const int fi = pl.item - wk.key_blocks;  // (the far blocks last: they are short)
  const bool far = fi >= 0;
  const int kb = far ? fi / wk.fars : pl.item, chunk = far ? fi % wk.fars : 0;
  const int k0 = kb * KB;
  const int near_end = wk.near_end(a, k0, KB);
  const int i_begin = far ? near_end + chunk * wk.far_rows : k0;
  const int i_end = min(far ? i_begin + wk.far_rows : near_end, seq.len);
  const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 31, half = lane >> 5;
  const int kw = k0 + 32 * w, j = kw + c;  // of this wave, of this lane
  const bool live = j < seq.len;
  const int per_head = i_begin < i_end ? (i_end - i_begin + R - 1) / R : 0;
  const int count = per_head * a.group;
  float* part = far ? wk.part + ((pl.group * wk.sink_blocks + kb) * wk.fars + chunk) * 2 * KB * a.dim : nullptr;
  // This wave's keys with fp32 products.
  const auto plain = [&]() {
    for (int r = 0; r < 32; ++r) {
      const int key = kw + r;
      if (key >= a.keys) break;
      float sk[2] = {0.f, 0.f}, sv[2] = {0.f, 0.f};
      const int end = key < a.sinks ? i_end : (int)min((int64_t)i_end, (int64_t)key + a.window);
      if (key < seq.len)
        for (int q = 0; q < a.group; ++q) plain_kv_sums(a, b, e * a.group + q, key, max(key, i_begin), end, sk, sv);
      store_plain(a, part, KB, b, e, key, key - k0, sk, sv);
    }
  };
  if (count == 0 || a.dim < 4) {  // (the workgroup) nobody sees them, or rows too short to load
    plain();
    return;
  }
  const Places<DP> at(lane);

  // The largest exponent of the rows of dout to come.
  int ex0 = kNone;
  {
    const int n = (i_end - i_begin + kTileRows - 1) / kTileRows;
    for (int t = threadIdx.x; t < n * a.group; t += NT) {
      const int64_t bh = (int64_t)b * a.heads + e * a.group + t / n;
      ex0 = max(ex0, wk.tile_ex[bh * wk.tiles + i_begin / kTileRows + t % n]);
    }
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) ex0 = max(ex0, __shfl_xor(ex0, x, 64));
    if (lane == 0) shared_ex[w] = ex0;
  }
  // this lane's rows of K, at a power of two of its own, and of V, at the workgroup's
  Frag kf[T::KS], vf[T::KS];
  int ek;
  bool odd = false;
  {
    float x[T::KS][8], m = 0.f;
    const float* K = a.k + ((int64_t)b * a.keys + (live ? j : 0)) * a.ldk + (int64_t)e * a.dim;
#pragma unroll
    for (int s = 0; s < T::KS; ++s) {
      load8(K, 2 * s + half, a.dim, live, x[s]);
      m = fmaxf(m, top8(x[s]));
    }
    m = fmaxf(m, other_half(m));
    odd |= !(m < INFINITY);
    const int ex = exponent(m);
#pragma unroll
    for (int s = 0; s < T::KS; ++s) kf[s] = split8(x[s], scale(ex));
    ek = ex;
  }
  int ev;
  {
    float x[T::KS][8], m = 0.f;
    const float* V = a.v + ((int64_t)b * a.keys + (live ? j : 0)) * a.ldv + (int64_t)e * a.dim;
#pragma unroll
    for (int s = 0; s < T::KS; ++s) {
      load8(V, 2 * s + half, a.dim, live, x[s]);
      m = fmaxf(m, top8(x[s]));
    }
    odd |= !(m < INFINITY);
    m = wave_top(m);
    if (lane == 63) shared_ev[w] = exponent(m);
    __syncthreads();
    ev = shared_ev[0], ex0 = shared_ex[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) ev = max(ev, shared_ev[i]), ex0 = max(ex0, shared_ex[i]);
#pragma unroll
    for (int s = 0; s < T::KS; ++s) vf[s] = split8(x[s], scale(ev));
  }
  Share<DP, NT> rq, rg;
  float r_lse = 0.f, r_delta = 0.f;  // of row threadIdx.x of the tile to come
  int r_ex = 0;
  // Tiles past the last are the last once more, which nobody reads: no branches around loads.
  struct At {
    int h, r0;
  };
  const auto at_tile = [&](int t) {
    t = min(t, count - 1);
    return At{e * a.group + t / per_head, i_begin + R * (t % per_head)};
  };
  auto fetch = [&](int t) {
    const At x = at_tile(t);
    rq.load(a.q + (int64_t)b * a.rows * a.ldq + (int64_t)x.h * a.dim, a.ldq, x.r0, i_end, a.dim);
    rg.load(a.dout + (int64_t)b * a.rows * a.lddo + (int64_t)x.h * a.dim, a.lddo, x.r0, i_end, a.dim);
    const int64_t st = ((int64_t)b * a.heads + x.h) * a.rows + min(x.r0 + (int)threadIdx.x % R, i_end - 1);
    r_lse = a.lse_in[st];
    r_delta = a.delta[st];
    r_ex = wk.ex[st];
  };
  // The tile's largest of Q, and what its rows are scaled by: one step ahead of put().
  auto tell = [&](int t) {
    const At x = at_tile(t);
    rq.clear(x.r0, i_end, a.dim);
    rg.clear(x.r0, i_end, a.dim);
    tops.add(0, t, rq.top());
    if (threadIdx.x < 64) {
      Rows<R>& r = rows[t & 3];
      const int n = threadIdx.x % R;
      const bool there = x.r0 + n < i_end, bad = there && r_ex == kOdd;
      const int ex = there && !bad ? r_ex : 0;
      r.ex[n] = ex;
      r.lse[n] = there ? r_lse * kLog2e - (float)(ex - ex0) : INFINITY;
      r.delta[n] = there ? __builtin_amdgcn_ldexpf(r_delta, kUnit - ex - ev) : 0.f;
      const unsigned any = __any(bad) ? 1u : 0u;
      if (threadIdx.x == 0) r.odd = any;
    }
  };
  int eq = kNone, eq_next = kNone;
  auto put = [&](int t) {
    const float mq = tops.get(0, t);
    odd |= !(mq < INFINITY) || rows[t & 3].odd != 0u;
    eq_next = max(eq_next, exponent(mq));
    rq.put(lds[t & 1][0], eq_next);
    rg.put_rows(lds[t & 1][1], rows[t & 3].ex);
  };
  f32x16 dk[T::DB], dv[T::DB];
#pragma unroll
  for (int d = 0; d < T::DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) dk[d][r] = dv[d][r] = 0.f;
  // this key's P is held at 2^sj (times its row's power of two), its dS at 2^(sj + tj)
  float sj = 100.f;
  int tj = 100;
  fetch(0);
  tell(0);
  __syncthreads();
  put(0);
  fetch(1);
  tell(1);
  for (int t = 0; t < count; ++t) {
    __syncthreads();  // tile t lies in its buffer, nobody reads the other, tile t + 1 is announced
    const int eqt = eq_next;
    put(t + 1);
    fetch(t + 2);
    const char *tq = lds[t & 1][0], *tg = lds[t & 1][1];
    const Rows<R>& rw = rows[t & 3];
    const int r0 = at_tile(t).r0;
    if (eqt != eq) {  // Q's operand has a larger power of two from here on
#pragma unroll
      for (int d = 0; d < T::DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) dk[d][r] = __builtin_amdgcn_ldexpf(dk[d][r], eq - eqt);
      eq = eqt;
    }
    const float ct = __builtin_amdgcn_ldexpf(a.scale * kLog2e, ek + eqt - 2 * kTop);
#pragma unroll
    for (int n = 0; n < T::NB; ++n) {
      const int i0 = r0 + 32 * n;  // rows of this block
      // some pair of it visible?
      if (i0 >= i_end || kw >= seq.len || i0 + 31 < kw || (i0 - (kw + 31) >= a.window && kw >= a.sinks)) continue;
      f32x16 s, x;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = x[r] = 0.f;
      steps<2 * T::KS, AHEAD>([&](int i) { return frag_row<DP>(i & 1 ? tg : tq, at, n, i >> 1); },
                              [&](int i, const Frag& f) {
                                if (i & 1) mma3(f, vf[i >> 1], x);
                                else mma3(f, kf[i >> 1], s);
                              });
      const bool all = kw + 31 <= i0 && (i0 + 31 - kw < a.window || kw + 31 < a.sinks) && kw + 32 <= seq.len;
      f32x4 lse[4], delta[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        lse[q] = *reinterpret_cast<const f32x4*>(&rw.lse[32 * n + 8 * q + 4 * half]);
        delta[q] = *reinterpret_cast<const f32x4*>(&rw.delta[32 * n + 8 * q + 4 * half]);
      }
      float mx = -INFINITY;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = fmaf(s[r], ct, -lse[r >> 2][r & 3]);
        if (!all) {
          const int i = i0 + 8 * (r >> 2) + 4 * half + (r & 3);
          s[r] = (live & sees(a, i, j)) ? s[r] : -INFINITY;
        }
        mx = fmaxf(mx, s[r]);
      }
      mx = fmaxf(mx, other_half(mx));
      if (__any(mx + sj > 15.f)) {
        const float to = mx + sj > 15.f ? floorf(8.f - mx) : sj;
        const int by = (int)(to - sj);
#pragma unroll
        for (int d = 0; d < T::DB; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) dv[d][r] = __builtin_amdgcn_ldexpf(dv[d][r], by);
        sj = to;
        tj -= by;
      }
      mx = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = __builtin_amdgcn_exp2f(s[r] + sj);
        x[r] = s[r] * fmaf(x[r], 0x1p-38f, -delta[r >> 2][r & 3]);
        mx = fmaxf(mx, fabsf(x[r]));
      }
      rescale(mx, tj, dk);
      const float ft = __builtin_amdgcn_ldexpf(1.f, tj);
      const Frag pf[2] = {split_rows(s, 0), split_rows(s, 1)}, df[2] = {split_rows(x, 0, ft), split_rows(x, 1, ft)};
      steps<4 * T::DB, AHEAD>([&](int i) { return frag_col<DP>(i & 1 ? tq : tg, at, 2 * n + i / (2 * T::DB), (i >> 1) % T::DB); },
                              [&](int i, const Frag& f) {
                                const int k = i / (2 * T::DB), d = (i >> 1) % T::DB;
                                if (i & 1) mma3(f, df[k], dk[d]);
                                else mma3(f, pf[k], dv[d]);
                              });
    }
    tell(t + 2);
  }
  float mark = 0.f;
#pragma unroll
  for (int d = 0; d < T::DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) mark = fmaf(0.f, dk[d][r], fmaf(0.f, dv[d][r], mark));
  if (__any(odd || mark != 0.f)) {  // (mark is 0 or NaN)
    plain();
    return;
  }
  if (j >= a.keys) return;
  const float* old_k = a.acc_k && !far ? a.dk + ((int64_t)b * a.keys + j) * a.lddk + (int64_t)e * a.dim : nullptr;
  const float* old_v = a.acc_v && !far ? a.dv + ((int64_t)b * a.keys + j) * a.lddv + (int64_t)e * a.dim : nullptr;
  float* out_k = far ? part + (j - k0) * a.dim : a.dk + ((int64_t)b * a.keys + j) * a.lddk + (int64_t)e * a.dim;
  float* out_v = far ? part + (KB + j - k0) * a.dim : a.dv + ((int64_t)b * a.keys + j) * a.lddv + (int64_t)e * a.dim;
  const int sh_v = live ? -(int)sj + ex0 - kTop : 0;
  const int sh_k = live ? -(int)sj - tj + ex0 + ev - kUnit + eq - kTop : 0;
#pragma unroll
  for (int d = 0; d < T::DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int col = 32 * d + 8 * (r >> 2) + 4 * half;
      float vk[4], vv[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        vk[n] = __builtin_amdgcn_ldexpf(dk[d][r + n] * a.scale, sh_k);
        vv[n] = __builtin_amdgcn_ldexpf(dv[d][r + n], sh_v);
      }
      store4(out_k, old_k, col, a.dim, vk);
      store4(out_v, old_v, col, a.dim, vv);
    }
}

// dq of 32 rows to a wave; rows to lanes, as in the forward.
template <int DP, int NW>
__global__ __launch_bounds__(64 * NW, DP <= 64 ? 2 : 1) void q_kernel(Args a, BwdWork wk, Grid g) {
  using T = Tile<DP>;
  constexpr int NT = 64 * NW, R = T::R, AHEAD = 1;
  __shared__ __attribute__((aligned(16))) char lds[2][2][T::BYTES];  // [buffer][K, V]
  __shared__ __attribute__((aligned(16))) Tops<NW> tops;
  const Block blk = g.block(a, 32 * NW);
  const int b = blk.b, h = blk.h, e = h / a.group;
  const Seq seq(a, b);
  const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 31, half = lane >> 5;
  const int row0 = blk.row + 32 * w, i = row0 + c;
  const bool live = i < seq.len;
  const int first = blk.row, last = min(blk.row + 32 * NW, seq.len) - 1;
  const int wlast = min(row0 + 32, seq.len) - 1;
  const bool any = first <= last;
  const Tiles<R> tiles(a, first, last);
  const int count = any ? tiles.count : 0;
  const auto plain = [&]() {  // this wave's rows with fp32 products
    for (int r = 0; r < 32; ++r)
      if (row0 + r < a.rows) plain_dq(a, b, h, row0 + r);
  };
  if (count == 0 || a.dim < 4) {  // (the workgroup) nothing to see, or rows too short to load
    plain();
    return;
  }
  const float* K = a.k + (int64_t)b * a.keys * a.ldk + (int64_t)e * a.dim;
  const float* V = a.v + (int64_t)b * a.keys * a.ldv + (int64_t)e * a.dim;
  const Places<DP> at(lane);

  Share<DP, NT> rk, rv;
  // Tiles past the last are the last once more, which nobody reads: no branches around loads.
  auto row_of = [&](int t) { return tiles.row(min(t, count - 1)); };
  auto fetch = [&](int t) {
    rk.load(K, a.ldk, row_of(t), seq.len, a.dim);
    rv.load(V, a.ldv, row_of(t), seq.len, a.dim);
  };
  auto tell = [&](int t) {
    rk.clear(row_of(t), seq.len, a.dim);
    rv.clear(row_of(t), seq.len, a.dim);
    tops.add(0, t, rk.top());
    tops.add(1, t, rv.top());
  };
  fetch(0);
  Frag q[T::KS], go[T::KS];
  int eq, eg;
  bool odd = false;
  {
    const float* Q = a.q + ((int64_t)b * a.rows + (live ? i : 0)) * a.ldq + (int64_t)h * a.dim;
    float x[T::KS][8], m = 0.f;
#pragma unroll
    for (int s = 0; s < T::KS; ++s) {
      load8(Q, 2 * s + half, a.dim, live, x[s]);
      m = fmaxf(m, top8(x[s]));
    }
    m = fmaxf(m, other_half(m));
    odd |= !(m < INFINITY);
    const int ex = exponent(m);
#pragma unroll
    for (int s = 0; s < T::KS; ++s) q[s] = split8(x[s], scale(ex));
    eq = ex;
  }
  {
    const float* G = a.dout + ((int64_t)b * a.rows + (live ? i : 0)) * a.lddo + (int64_t)h * a.dim;
    float x[T::KS][8], m = 0.f;
#pragma unroll
    for (int s = 0; s < T::KS; ++s) {
      load8(G, 2 * s + half, a.dim, live, x[s]);
      m = fmaxf(m, top8(x[s]));
    }
    m = fmaxf(m, other_half(m));
    odd |= !(m < INFINITY);
    eg = exponent(m);
#pragma unroll
    for (int s = 0; s < T::KS; ++s) go[s] = split8(x[s], scale(eg));
  }
  const int64_t st = ((int64_t)b * a.heads + h) * a.rows + (live ? i : 0);
  const float delta = live ? a.delta[st] : 0.f, lse = live ? a.lse_in[st] * kLog2e : 0.f;
  odd |= !(fabsf(delta) < INFINITY) || !(fabsf(lse) < INFINITY);
  int ek = kNone, ek_next = kNone, ev = 0;
  auto put = [&](int t) {
    const float mk = tops.get(0, t), mv = tops.get(1, t);
    odd |= !(fmaxf(mk, mv) < INFINITY);
    ek_next = max(ek_next, exponent(mk));
    ev = exponent(mv);
    rk.put(lds[t & 1][0], ek_next);
    rv.put(lds[t & 1][1], ev);
  };
  tell(0);
  __syncthreads();
  f32x16 dq[T::DB];
#pragma unroll
  for (int d = 0; d < T::DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) dq[d][r] = 0.f;
  int ti = 100;  // this row's dS is held at 2^ti (and below)
  const float dd = __builtin_amdgcn_ldexpf(delta, -eg);
  put(0);
  fetch(1);
  tell(1);
  for (int t = 0; t < count; ++t) {
    __syncthreads();
    const int ekt = ek_next, evt = ev;
    put(t + 1);
    fetch(t + 2);
    const char *tk = lds[t & 1][0], *tv = lds[t & 1][1];
    const int j0 = tiles.row(t);
    if (ekt != ek) {  // K's operand has a larger power of two from here on
#pragma unroll
      for (int d = 0; d < T::DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) dq[d][r] = __builtin_amdgcn_ldexpf(dq[d][r], ek - ekt);
      ek = ekt;
    }
    const float ct = __builtin_amdgcn_ldexpf(a.scale * kLog2e, eq + ekt - 2 * kTop);
    const float cd = __builtin_amdgcn_ldexpf(1.f, evt - 2 * kTop);  // dP - D at 2^-eg
#pragma unroll
    for (int n = 0; n < T::NB; ++n) {
      const int jb = j0 + 32 * n;
      if (row0 > wlast || jb > wlast || (row0 - (jb + 31) >= a.window && jb >= a.sinks)) continue;
      f32x16 s, x;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = x[r] = 0.f;
      steps<2 * T::KS, AHEAD>([&](int i) { return frag_row<DP>(i & 1 ? tv : tk, at, n, i >> 1); },
                              [&](int i, const Frag& f) {
                                if (i & 1) mma3(f, go[i >> 1], x);
                                else mma3(f, q[i >> 1], s);
                              });
      const bool all = jb + 31 <= row0 && (wlast - jb < a.window || jb + 31 < a.sinks) && row0 + 32 <= seq.len;
      float mx = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float p = fmaf(s[r], ct, -lse);
        if (!all) {
          const int j = jb + 8 * (r >> 2) + 4 * half + (r & 3);
          p = (live & sees(a, i, j)) ? p : -INFINITY;
        }
        x[r] = __builtin_amdgcn_exp2f(p) * fmaf(x[r], cd, -dd);
        mx = fmaxf(mx, fabsf(x[r]));
      }
      rescale(mx, ti, dq);
      const float ft = __builtin_amdgcn_ldexpf(1.f, ti);
      const Frag df[2] = {split_rows(x, 0, ft), split_rows(x, 1, ft)};
      steps<2 * T::DB, AHEAD>([&](int i) { return frag_col<DP>(tk, at, 2 * n + i / T::DB, i % T::DB); },
                              [&](int i, const Frag& f) { mma3(f, df[i / T::DB], dq[i % T::DB]); });
    }
    tell(t + 2);
  }
  float mark = 0.f;
#pragma unroll
  for (int d = 0; d < T::DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) mark = fmaf(0.f, dq[d][r], mark);
  if (__any(odd || mark != 0.f)) {
    plain();
    return;
  }
  if (i >= a.rows) return;
  float* out = a.dq + ((int64_t)b * a.rows + i) * a.lddq + (int64_t)h * a.dim;
  const int sh = live ? eg - ti + ek - kTop : 0;
#pragma unroll
  for (int d = 0; d < T::DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int col = 32 * d + 8 * (r >> 2) + 4 * half;
      float x[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) x[n] = __builtin_amdgcn_ldexpf(dq[d][r + n] * a.scale, sh);
      store4(out, a.acc_q ? out : nullptr, col, a.dim, x);
    }
}

// Adds the far sums of the sinks, chunk by chunk: a thread to a value.
__global__ __launch_bounds__(256) void join_kernel(Args a, BwdWork wk, int64_t first) {
  const int64_t id = (first + blockIdx.x) * 256 + threadIdx.x;
  const int64_t n = (int64_t)a.sinks * a.dim, group = id / n;  // of a head
  if (group >= (int64_t)a.batch * a.kv_heads) return;
  const int at = (int)(id - group * n), j = at / a.dim, d = at - j * a.dim, blk = j / kKeyBlock;
  const int b = (int)(group / a.kv_heads), e = (int)(group % a.kv_heads);
  const Seq seq(a, b);
  const int begin = wk.near_end(a, blk * kKeyBlock, kKeyBlock);
  if (j >= seq.len || begin >= seq.len) return;
  float sk = 0.f, sv = 0.f;
  const float* p = wk.part + ((group * wk.sink_blocks + blk) * wk.fars) * 2 * kKeyBlock * a.dim + (j - blk * kKeyBlock) * a.dim + d;
  for (int i = begin; i < seq.len; i += wk.far_rows, p += 2 * kKeyBlock * a.dim) {
    sk += p[0];
    sv += p[kKeyBlock * a.dim];
  }
  a.dk[((int64_t)b * a.keys + j) * a.lddk + (int64_t)e * a.dim + d] += sk;
  a.dv[((int64_t)b * a.keys + j) * a.lddv + (int64_t)e * a.dim + d] += sv;
}

constexpr int kWaves = kKeyBlock / 32;  // of a workgroup

template <int DP>
void launch_dim(const Args& a, const BwdWork& wk, hipStream_t s) {
  launch_blocks(kv_kernel<DP, kWaves>, Grid(a, a.kv_heads, wk.key_blocks + wk.sink_blocks * wk.fars), 64 * kWaves, s, a, wk);
  launch_blocks(q_kernel<DP, kWaves>, Grid(a, a.heads, (a.rows + 32 * kWaves - 1) / (32 * kWaves)), 64 * kWaves, s, a, wk);
}

}  // namespace

void tile_backward(const Args& a, const BwdWork& wk, hipStream_t s) {
  const int64_t tiles = (int64_t)a.batch * a.heads * wk.tiles;
  constexpr int64_t kBlocks = 1 << 23;
  for (int64_t f = 0; f < tiles; f += kBlocks)
    mle::launch(prepare_kernel, (unsigned)std::min(tiles - f, kBlocks), 256, 0, s, a, wk, f);
  if (a.dim <= 64) launch_dim<64>(a, wk, s);
  else if (a.dim <= 96) launch_dim<96>(a, wk, s);
  else launch_dim<128>(a, wk, s);
  if (wk.fars == 0) return;
  const int64_t joins = ((int64_t)a.batch * a.kv_heads * a.sinks * a.dim + 255) / 256;
  for (int64_t f = 0; f < joins; f += kBlocks)
    mle::launch(join_kernel, (unsigned)std::min(joins - f, kBlocks), 256, 0, s, a, wk, f);
}

}  // namespace wattn
