// Backward of the windowed attention, in passes that each write their own gradients, so
// that no sum depends on timing:
//   prepare   D and the exponent of each row of dout
//   kv        dk and dv of 32 keys to a wave, over the tiles of rows that see them
//   q         dq of 32 rows to a wave, over the tiles of keys that they see
//   join      the parts of sums over rows, added in order
// S and dP = dout v^T are computed again in both; kv and q are one launch.
//
// Sinks are seen by every later row.  Blocks of keys with sinks take the rows up to their
// window like all others ("near"); the rows after it ("far") are shared out over workgroups
// whose sums lie in the workspace.
//
// Scales.  A product sums over rows (kv) or keys (q) whose probabilities and gradients may be
// of very unlike size, so the operands that are made here are held at powers of two of their
// own column, a lane's: a key's P and dS (kv), a row's dS (q) have the largest seen so far
// between 2^12 and 2^15, and a larger one rescales the lane's sums.  Rows of dout are at powers
// of two of their own too; P takes those up in its exponent.
//
// Here for heads of up to 64, a wave with 32 keys (rows) to itself: two workgroups of four waves
// to a CU, out of step.  Tiles of 32 rows in the kv pass, whose staging then fits beside the
// sums (64-row tiles spilled, and every reload waited for the loads under way: 555 us against
// 523 at 4 x 8 heads of 4096, window 1024); 64 keys in the q pass (528 with 32).  That
// case takes 424 us now (fp32 products at 178 TFLOP/s), 32 x 8 heads of 256 under a window of 128
// 72 us, prepare's 9 among them.
#include "window_bwd.hpp"

using namespace mle;

namespace wattn {
namespace {

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

template <int DP, int NW>
struct Shared {
  alignas(16) char lds[2][2][Tile<DP, 64>::BYTES];  // [buffer][Q, dout or K, V]
  Rows<32> rows[4];
  alignas(16) Tops<NW> tops;
  int ex[NW];
};

// dk and dv of 32 keys to a wave.
template <int DP, int NW>
__device__ __forceinline__ void kv_rows(const Args& a, const BwdWork& wk, const Place& place, Shared<DP, NW>& m) {
  using T = Tile<DP, 32>;
  constexpr int NT = 64 * NW, KB = 32 * NW, R = T::R, AHEAD = 1;
  static_assert(KB == kKeyBlock, "keys of a workgroup");
  const KvJob job(a, wk, place);
  const int b = job.b, e = job.e, k0 = job.k0, i_end = job.i_end;
  const Seq seq(a, b);
  const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 31, half = lane >> 5;
  const int kw = k0 + 32 * w, j = kw + c;  // of this wave, of this lane
  const bool live = j < seq.len;
  const int per_head = job.i_begin < i_end ? (i_end - job.i_begin + R - 1) / R : 0;
  const int count = per_head * a.group;
  if (count == 0 || a.dim < 4) {  // (the workgroup) nobody sees them, or rows too short to load
    job.plain(a, kw, true, true);
    return;
  }
  const Places<T> at(lane);
  typedef Share<T, NT> Part;
  struct In {  // of Q and dout, and of row threadIdx.x % 32 of them
    Part x;
    float lse, delta;
    int ex;
  } in0, in;  // tile 0's, and the others'
  Walk<R> ahead(a, job), here(a, job);
  auto fetch = [&](In& in) {
    in.x.load(a.q + (int64_t)b * a.rows * a.ldq + (int64_t)ahead.h * a.dim, a.ldq,
              a.dout + (int64_t)b * a.rows * a.lddo + (int64_t)ahead.h * a.dim, a.lddo, ahead.r0, i_end, a.dim);
    const int64_t st = ((int64_t)b * a.heads + ahead.h) * a.rows + min(ahead.r0 + (int)threadIdx.x % R, i_end - 1);
    in.lse = a.lse_in[st];
    in.delta = a.delta[st];
    in.ex = wk.ex[st];
  };
  fetch(in0);
  const int first_row = ahead.r0;
  ahead.next();
  fetch(in);
  job.largest(a, wk, m.ex);
  // this lane's rows of K and V, each at a power of two of its own
  Frag kf[T::KS], vf[T::KS];
  int ek, ev;
  bool odd = false;
  {
    float x[T::KS][8];
    const float top = load_row<T::KS>(a.k + ((int64_t)b * a.keys + (live ? j : 0)) * a.ldk + (int64_t)e * a.dim, half, a.dim, live, x);
    odd |= !(top < INFINITY);
    ek = exponent(fmaxf(top, other_half(top)));
#pragma unroll
    for (int s = 0; s < T::KS; ++s) kf[s] = split8<false>(x[s], scale(ek));
  }
  {
    float x[T::KS][8];
    const float top = load_row<T::KS>(a.v + ((int64_t)b * a.keys + (live ? j : 0)) * a.ldv + (int64_t)e * a.dim, half, a.dim, live, x);
    odd |= !(top < INFINITY);
    ev = exponent(fmaxf(top, other_half(top)));
#pragma unroll
    for (int s = 0; s < T::KS; ++s) vf[s] = split8<false>(x[s], scale(ev));
  }
  const float cd = __builtin_amdgcn_ldexpf(1.f, ev + kUnit - 2 * kTop);
  __syncthreads();
  int ex0 = m.ex[0];
#pragma unroll
  for (int i = 1; i < NW; ++i) ex0 = max(ex0, m.ex[i]);
  // The largest of Q in tile t from row r0, and what its rows are scaled by: one step ahead of put().
  auto tell = [&](In& in, int t, int r0) {
    in.x.clear(r0, i_end, a.dim);
    m.tops.add(0, t, in.x.top(false));
    m.rows[t & 3].put(r0, i_end, ex0, in.lse, in.delta, in.ex);
  };
  int eq = kNone, eq_next = kNone;  // the exponent of Q's operand, that dk is at and of the tile to come
  auto put = [&](const Part& x, int t) {
    const float mq = m.tops.get(0, t);
    const Rows<R>& r = m.rows[t & 3];
    odd |= !(mq < INFINITY) || r.odd != 0u;
    eq_next = raised(eq_next, mq, odd);
    const float sq = scale(eq_next);
    x.put(m.lds[t & 1][0], m.lds[t & 1][1], [&](bool g, int row) { return g ? scale(r.ex[row]) : sq; });
  };
  f32x16 dk[T::DB], dv[T::DB];
#pragma unroll
  for (int d = 0; d < T::DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) dk[d][r] = dv[d][r] = 0.f;
  // this key's P is held at 2^sj (times its row's power of two), its dS at 2^(sj + tj)
  float sj = 100.f;
  int tj = 100;
  const unsigned most = !live ? 0u : j < a.sinks ? 0x7fffffffu : (unsigned)a.window;  // how far its rows go
  tell(in0, 0, first_row);
  tell(in, 1, ahead.r0);
  ahead.next();
  __syncthreads();
  put(in0.x, 0);
  for (int t = 0; t < count; ++t) {
    __syncthreads();  // tile t lies in its buffer, nobody reads the other, tile t + 1 is announced
    const int eqt = eq_next;
    if (t + 1 < count) put(in.x, t + 1);
    fetch(in);
    const char *tq = m.lds[t & 1][0], *tg = m.lds[t & 1][1];
    const Rows<R>& rw = m.rows[t & 3];
    const int r0 = here.r0;
    here.next();
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
      steps<2 * T::KS, AHEAD>([&](int i) { return frag_row<T>(i & 1 ? tg : tq, at, n, i >> 1); },
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
      }
      if (!all) hide_rows(s, i0 + 4 * half - j, most);
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[r]);
      if (__any(mx + sj > 15.f)) {
        mx = fmaxf(mx, other_half(mx));
        const float to = mx + sj > 15.f ? floorf(kHeld + 1 - mx) : sj;
        const int by = (int)(to - sj);
#pragma unroll
        for (int d = 0; d < T::DB; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) dv[d][r] = __builtin_amdgcn_ldexpf(dv[d][r], by);
        sj = to;
        tj -= by;
      }
      const float held = __builtin_amdgcn_ldexpf(1.f, (int)sj);  // (as a factor: in the exponent it would cost P's last bits)
      mx = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = __builtin_amdgcn_exp2f(s[r]) * held;
        x[r] = s[r] * fmaf(x[r], cd, -delta[r >> 2][r & 3]);
        mx = fmaxf(mx, fabsf(x[r]));
      }
      rescale(mx, tj, dk);
      const float ft = __builtin_amdgcn_ldexpf(1.f, tj);
      const Frag pf[2] = {split_rows<true>(s, 0, 1.f), split_rows<true>(s, 1, 1.f)}, df[2] = {split_rows<true>(x, 0, ft), split_rows<true>(x, 1, ft)};
      steps<4 * T::DB, AHEAD>([&](int i) { return frag_col<T>(i & 1 ? tq : tg, at, 2 * n + i / (2 * T::DB), (i >> 1) % T::DB); },
                              [&](int i, const Frag& f) {
                                const int k = i / (2 * T::DB), d = (i >> 1) % T::DB;
                                if (i & 1) mma3(f, df[k], dk[d]);
                                else mma3(f, pf[k], dv[d]);
                              });
    }
    if (t + 2 < count) {
      tell(in, t + 2, ahead.r0);
      ahead.next();
    }
  }
  float mark = 0.f;
#pragma unroll
  for (int d = 0; d < T::DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) mark = fmaf(0.f, dk[d][r], fmaf(0.f, dv[d][r], mark));
  if (__any(odd || mark != 0.f)) {  // (mark is 0 or NaN)
    job.plain(a, kw, true, true);
    return;
  }
  if (j >= a.keys) return;
  const float* old_k = a.acc_k && !job.part ? a.dk + ((int64_t)b * a.keys + j) * a.lddk + (int64_t)e * a.dim : nullptr;
  const float* old_v = a.acc_v && !job.part ? a.dv + ((int64_t)b * a.keys + j) * a.lddv + (int64_t)e * a.dim : nullptr;
  float* out_k = job.part ? job.part + (j - k0) * a.dim : a.dk + ((int64_t)b * a.keys + j) * a.lddk + (int64_t)e * a.dim;
  float* out_v = job.part ? job.part + (KB + j - k0) * a.dim : a.dv + ((int64_t)b * a.keys + j) * a.lddv + (int64_t)e * a.dim;
  const int sh_v = live ? -(int)sj + ex0 - kTop : 0;
  const int sh_k = live ? -(int)sj - tj + ex0 - kUnit + eq - kTop : 0;
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
__device__ __forceinline__ void q_rows(const Args& a, const Block& blk, Shared<DP, NW>& m) {
  using T = Tile<DP, 64>;
  constexpr int NT = 64 * NW, R = T::R, AHEAD = 1;
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
  const Places<T> at(lane);

  typedef Share<T, NT> Part;
  Part kv0, kv;  // tile 0's registers, and the others'
  // Loads past the last tile are of the last once more and go unused: no branches around loads.
  auto row_of = [&](int t) { return tiles.row(min(t, count - 1)); };
  auto fetch = [&](Part& x, int t) { x.load(K, a.ldk, V, a.ldv, row_of(t), seq.len, a.dim); };
  auto tell = [&](Part& x, int t) {
    x.clear(row_of(t), seq.len, a.dim);
    m.tops.add(0, t, x.top(false));
    m.tops.add(1, t, x.top(true));
  };
  fetch(kv0, 0);
  fetch(kv, 1);
  Frag q[T::KS], go[T::KS];
  bool odd = false;
  auto own = [&](const float* p, Frag (&f)[T::KS]) {  // a row at a power of two of its own
    float x[T::KS][8];
    float top = load_row<T::KS>(p, half, a.dim, live, x);
    top = fmaxf(top, other_half(top));
    odd |= !(top < INFINITY);
#pragma unroll
    for (int s = 0; s < T::KS; ++s) f[s] = split8<false>(x[s], scale(exponent(top)));
    return exponent(top);
  };
  const int64_t row = (int64_t)b * a.rows + (live ? i : 0);
  const int eq = own(a.q + row * a.ldq + (int64_t)h * a.dim, q), eg = own(a.dout + row * a.lddo + (int64_t)h * a.dim, go);
  const int64_t st = ((int64_t)b * a.heads + h) * a.rows + (live ? i : 0);
  const float delta = live ? a.delta[st] : 0.f, lse = live ? a.lse_in[st] * kLog2e : 0.f;
  odd |= !(fabsf(delta) < INFINITY) || !(fabsf(lse) < INFINITY);
  int ek = kNone, ek_next = kNone, ev = 0;
  auto put = [&](const Part& x, int t) {
    const float mk = m.tops.get(0, t), mv = m.tops.get(1, t);
    odd |= !(fmaxf(mk, mv) < INFINITY);
    ek_next = raised(ek_next, mk, odd);
    ev = exponent(mv);
    const float sk = scale(ek_next), sv = scale(ev);
    x.put(m.lds[t & 1][0], m.lds[t & 1][1], [=](bool v, int) { return v ? sv : sk; });
  };
  tell(kv0, 0);
  tell(kv, 1);
  __syncthreads();
  f32x16 dq[T::DB];
#pragma unroll
  for (int d = 0; d < T::DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) dq[d][r] = 0.f;
  int ti = 100;  // this row's dS is held at 2^ti (and below)
  const float dd = __builtin_amdgcn_ldexpf(delta, -eg);
  put(kv0, 0);
  for (int t = 0; t < count; ++t) {
    __syncthreads();
    const int ekt = ek_next, evt = ev;
    if (t + 1 < count) put(kv, t + 1);
    fetch(kv, t + 2);
    const char *tk = m.lds[t & 1][0], *tv = m.lds[t & 1][1];
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
      steps<2 * T::KS, AHEAD>([&](int i) { return frag_row<T>(i & 1 ? tv : tk, at, n, i >> 1); },
                              [&](int i, const Frag& f) {
                                if (i & 1) mma3(f, go[i >> 1], x);
                                else mma3(f, q[i >> 1], s);
                              });
      const bool all = jb + 31 <= row0 && (wlast - jb < a.window || jb + 31 < a.sinks) && row0 + 32 <= seq.len;
      float mx = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], ct, -lse);
      if (!all) hide_keys(s, live ? i - jb - 4 * half : -1, a.window, a.sinks - jb - 4 * half, jb < a.sinks);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        x[r] = __builtin_amdgcn_exp2f(s[r]) * fmaf(x[r], cd, -dd);
        mx = fmaxf(mx, fabsf(x[r]));
      }
      rescale(mx, ti, dq);
      const float ft = __builtin_amdgcn_ldexpf(1.f, ti);
      const Frag df[2] = {split_rows<true>(x, 0, ft), split_rows<true>(x, 1, ft)};
      steps<2 * T::DB, AHEAD>([&](int i) { return frag_col<T>(tk, at, 2 * n + i / T::DB, i % T::DB); },
                              [&](int i, const Frag& f) { mma3(f, df[i / T::DB], dq[i % T::DB]); });
    }
    if (t + 2 < count) tell(kv, t + 2);
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

// Both passes in one launch, the longer kv pass first: the one fills in behind the other.
template <int DP, int NW>
__global__ __launch_bounds__(64 * NW, 2) void narrow_kernel(Args a, BwdWork wk, Grid kv, Grid q, int64_t first) {
  __shared__ Shared<DP, NW> m;
  const int64_t id = first + blockIdx.x;
  if (id < kv.total)
    kv_rows<DP, NW>(a, wk, kv.place(id), m);
  else
    q_rows<DP, NW>(a, q.block(a, 32 * NW, id - kv.total), m);
}

// Adds the parts of a key's sums, in order, and to its gradients: a thread to a value.
__global__ __launch_bounds__(256) void join_kernel(Args a, BwdWork wk, int keys, int64_t first) {
  const int64_t id = (first + blockIdx.x) * 256 + threadIdx.x;
  const int64_t n = (int64_t)keys * a.dim, group = id / n;  // of a head
  if (group >= (int64_t)a.batch * a.kv_heads) return;
  const int at = (int)(id - group * n), j = at / a.dim, d = at - j * a.dim, blk = j / kKeyBlock, k0 = blk * kKeyBlock;
  const int b = (int)(group / a.kv_heads), e = (int)(group % a.kv_heads);
  const int len = Seq(a, b).len, size = 2 * kKeyBlock * a.dim, place = (j - k0) * a.dim + d, begin = wk.near_end(a, k0);
  float sk = 0.f, sv = 0.f;
  if (wk.nears > 1 && j < len) {
    const float* p = wk.near + (group * wk.key_blocks + blk) * wk.nears * size + place;
    for (int i = k0; i < min(begin, len); i += wk.near_rows, p += size) {
      sk += p[0];
      sv += p[kKeyBlock * a.dim];
    }
  }
  if (j < a.sinks && j < len) {
    const float* p = wk.far + (group * wk.sink_blocks + blk) * wk.fars * size + place;
    for (int i = begin; i < len; i += wk.far_rows, p += size) {
      sk += p[0];
      sv += p[kKeyBlock * a.dim];
    }
  }
  // (with one near part a sink's gradients hold that part already)
  float* dk = a.dk + ((int64_t)b * a.keys + j) * a.lddk + (int64_t)e * a.dim + d;
  float* dv = a.dv + ((int64_t)b * a.keys + j) * a.lddv + (int64_t)e * a.dim + d;
  *dk = (wk.nears == 1 || a.acc_k ? *dk : 0.f) + sk;
  *dv = (wk.nears == 1 || a.acc_v ? *dv : 0.f) + sv;
}

}  // namespace

void tile_backward(const Args& a, const BwdWork& wk, hipStream_t s) {
  const int64_t tiles = (int64_t)a.batch * a.heads * wk.tiles;
  constexpr int64_t kBlocks = 1 << 23;
  for (int64_t f = 0; f < tiles; f += kBlocks)
    mle::launch(prepare_kernel, (unsigned)std::min(tiles - f, kBlocks), 256, 0, s, a, wk, f);
  if (a.dim <= 64) {
    constexpr int NW = kKeyBlock / 32;
    launch_both(narrow_kernel<64, NW>, Grid(a, a.kv_heads, wk.kv_items(), 1024),
                Grid(a, a.heads, (a.rows + 32 * NW - 1) / (32 * NW), 1024), 64 * NW, s, a, wk);
  } else {
    launch_wide(a, wk, s);
  }
  const int keys = wk.nears > 1 ? a.keys : wk.fars > 0 ? std::min(a.sinks, a.keys) : 0;
  const int64_t joins = ((int64_t)a.batch * a.kv_heads * keys * a.dim + 255) / 256;
  for (int64_t f = 0; f < joins; f += kBlocks)
    mle::launch(join_kernel, (unsigned)std::min(joins - f, kBlocks), 256, 0, s, a, wk, keys, f);
}

}  // namespace wattn
