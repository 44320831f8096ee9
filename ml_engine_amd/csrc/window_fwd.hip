// Forward of the windowed attention: 32 rows to a wave, or (KW 2) to two waves that take half
// of each tile's keys and join at the end, one pass over the tiles of keys that the rows of a
// workgroup see with the running maximum and sum of a softmax.
//
// Scores come out as S^T = K Q^T, rows to lanes, so a row's statistics are a lane's
// (two lanes hold 16 of every 32 keys of a row each), and P^T is the operand of
// O^T += V^T P^T as it lies in the accumulators.  P is held at 2^12 for a row's maximum so
// far, so that a weight is off by at most 2^-23 of it or 2^-37 of the row's largest; the sums are
// rescaled only when a score passes that by 2^3 (at 2^8 and 2^7, small weights beside a large one
// lost 2^-10 of themselves, and the times were the same to 1 %).
//
// Bound by vector instructions beside the products: splitting operands, masks, exponentials.
// 2 x 16 heads of 4096 x 128 under a window of 1024 take 254 us (fp32 products at 237
// TFLOP/s, matrix cores 32 % busy, vector units 38 %), 32 x 8 heads of 256 x 64 under one
// of 128 24 us, where a workgroup's two to four tiles leave both idle most of the time.
//
// Of heads of 128 the form of 4 waves spills 5 vector registers and that of pairs and 8 waves 2; one
// workgroup to a CU, which needs no spills, takes 129 us where two take 89 (8 x 16 heads of 1024
// under a window of 128).
#include "window_tile.hpp"
#include "window_kernels.hpp"

using namespace mle;

namespace wattn {
namespace {

constexpr float kHead = 12.f;  // log2

template <int DP, int NW, int KW>
__global__ __launch_bounds__(64 * NW, DP > 64 && NW / KW == 2 ? 1 : 2) void tile_fwd_kernel(Args a, Grid g) {
  // as many products to a wave and tile of wide heads, half the registers to LDS
  using T = Tile<DP, DP <= 64 || KW == 2 ? 64 : 32>;
  constexpr int NT = 64 * NW, R = T::R, AHEAD = 2;
  constexpr int NB = T::NB / KW;  // a wave's blocks of a tile
  __shared__ __attribute__((aligned(16))) char lds[2][2][T::BYTES];  // [buffer][K, V]
  __shared__ __attribute__((aligned(16))) Tops<NW> tops;
  const Block blk = g.block(a, 32 * NW / KW);
  const int b = blk.b, h = blk.h, e = h / a.group;
  const Seq seq(a, b);
  const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 31, half = lane >> 5;
  const int kw = w % KW, n0 = kw * NB;        // which of the rows' waves, its first block of a tile
  const int row0 = blk.row + 32 * (w / KW);   // of this wave
  const int i = row0 + c, p = seq.first + i;  // of this lane
  const bool live = i < a.rows && p >= 0 && p < seq.len;
  // positions of the workgroup's and the wave's rows that are there
  const int first = max(seq.first + blk.row, 0), last = min(seq.first + min(blk.row + 32 * NW / KW, a.rows), seq.len) - 1;
  const int wfirst = max(seq.first + row0, 0), wlast = min(seq.first + min(row0 + 32, a.rows), seq.len) - 1;
  const bool any = first <= last;
  const Tiles<R> tiles(a, first, last);
  const int count = any ? tiles.count : 0;
  if (count == 0 || a.dim < 4) {  // (the workgroup) nothing to see, or rows too short to load
    for (int r = kw; r < 32; r += KW)
      if (row0 + r < a.rows) plain_row(a, b, h, row0 + r);
    return;
  }
  const float* K = a.k + (int64_t)b * a.keys * a.ldk + (int64_t)e * a.dim;
  const float* V = a.v + (int64_t)b * a.keys * a.ldv + (int64_t)e * a.dim;
  const Places<T> at(lane);

  Share<T, NT> kv;
  // Loads past the last tile are of the last once more and go unused: no branches around loads.
  auto row_of = [&](int t) { return tiles.row(min(t, count - 1)); };
  // Keys that no row of the workgroup sees (after its last, and between the sinks and its first window)
  // are zeros, so that what lies there, in a cache's places that were left for instance, takes no
  // bits from the others of its tile.
  auto fetch = [&](int t) { kv.load(K, a.ldk, V, a.ldv, row_of(t), last + 1, a.dim); };
  auto tell = [&](int t) {
    kv.clear(row_of(t), last + 1, a.dim, a.sinks, first - a.window + 1);
    tops.add(0, t, kv.top(false));
    tops.add(1, t, kv.top(true));
  };
  fetch(0);
  // this lane's row of Q, at a power of two of its own
  Frag q[T::KS];
  int eq;
  bool odd = false;  // an infinity among the rows or the tiles, whose powers of two then say nothing
  {
    const float* Q = a.q + ((int64_t)b * a.rows + (live ? i : 0)) * a.ldq + (int64_t)h * a.dim;
    float x[T::KS][8], m = load_row<T::KS>(Q, half, a.dim, live, x);
    m = fmaxf(m, other_half(m));
    odd = !(m < INFINITY);
    const int ex = exponent(m);
    const float sc = a.scale < 0.f ? -scale(ex) : scale(ex);
#pragma unroll
    for (int s = 0; s < T::KS; ++s) q[s] = split8<false>(x[s], sc);
    eq = ex;
  }
  int ek = 0, ev = -1000, ev_next = -1000;  // exponents: of the tile of K at hand, of V's operand so far
  auto put = [&](int t) {  // tile t from the registers to its buffer
    const float mk = tops.get(0, t), mv = tops.get(1, t);
    odd |= !(fmaxf(mk, mv) < INFINITY);
    ek = exponent(mk);
    ev_next = raised(ev_next, mv, odd);
    const float sk = scale(ek), sv = scale(ev_next);
    kv.put(lds[t & 1][0], lds[t & 1][1], [=](bool v, int) { return v ? sv : sk; });
  };
  tell(0);
  __syncthreads();
  f32x16 o[T::DB];
#pragma unroll
  for (int d = 0; d < T::DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
  float m = -3e38f, l = 0.f;  // log2 units; m is kHead below the maximum
  const auto some = [&](int t) {  // does the wave see any of tile t?
    const int j0 = tiles.row(t) + 32 * n0;
    return wfirst <= wlast && j0 <= wlast && (wfirst - (j0 + 32 * NB - 1) < a.window || j0 < a.sinks);
  };
  Frag pf[2 * NB];  // P of a tile
  // P of tile t, whose K has exponent e.
  const auto weights = [&](int t, int e) {
    const char* tk = lds[t & 1][0];
    const int j0 = tiles.row(t) + 32 * n0;
    f32x16 s[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[n][r] = 0.f;
    steps<T::KS * NB, AHEAD>([&](int i) { return frag_row<T>(tk, at, n0 + i % NB, i / NB); },
                                [&](int i, const Frag& f) { mma3(f, q[i / NB], s[i % NB]); });
    const bool all = j0 + 32 * NB - 1 <= wfirst && (wlast - j0 < a.window || j0 + 32 * NB - 1 < a.sinks) && row0 + 32 <= a.rows &&
                     seq.first + row0 >= 0 && seq.first + row0 + 32 <= seq.len;
    if (!all) {
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int j = j0 + 32 * n + 8 * (r >> 2) + 4 * half + (r & 3);
          s[n][r] = (live & sees(a, p, j)) ? s[n][r] : -INFINITY;
        }
    }
    // (never 0, so that what is hidden stays at minus infinity)
    const float ct = fmaxf(__builtin_amdgcn_ldexpf(fabsf(a.scale) * kLog2e, eq + e - 2 * kTop), 0x1p-126f);
    float mx = s[0][0];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[n][r]);
    mx *= ct;
    if (__any(mx > m + 15.f)) {
      const float mn = fmaxf(m, fmaxf(mx, other_half(mx)) - kHead), f = __builtin_amdgcn_exp2f(m - mn);
      l *= f;
#pragma unroll
      for (int d = 0; d < T::DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= f;
      m = mn;
    }
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[n][r] = __builtin_amdgcn_exp2f(fmaf(s[n][r], ct, -m));
        l += s[n][r];
      }
#pragma unroll
    for (int k = 0; k < 2 * NB; ++k) pf[k] = split_rows<false>(s[k >> 1], k & 1, 1.f);
  };
  // O += P V of tile t, whose operand of V has exponent e.
  const auto values = [&](int t, int e) {
    if (e != ev) {  // V's operand has a larger power of two from here on
#pragma unroll
      for (int d = 0; d < T::DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = __builtin_amdgcn_ldexpf(o[d][r], ev - e);
      ev = e;
    }
    const char* tv = lds[t & 1][1];
    steps<2 * NB * T::DB, AHEAD>([&](int i) { return frag_col<T>(tv, at, 2 * n0 + i / T::DB, i % T::DB); },
                                    [&](int i, const Frag& f) { mma3(f, pf[i / T::DB], o[i % T::DB]); });
  };
  put(0);
  fetch(1);
  tell(1);
  for (int t = 0; t < count; ++t) {
    __syncthreads();  // tile t lies in its buffer, nobody reads the other, tile t + 1's tops are known
    const int ekt = ek, evt = ev_next;
    if (t + 1 < count) put(t + 1);
    fetch(t + 2);
    if (some(t)) {
      weights(t, ekt);
      values(t, evt);
    }
    if (t + 2 < count) tell(t + 2);
  }
  l += other_half(l);
  if constexpr (KW == 2) {
    // the second wave's sums to the first, both at the larger maximum and power of two
    static_assert(NW / 2 * 64 * (4 * T::DB + 1) * sizeof(f32x4) <= sizeof(lds), "room for a wave's sums");
    f32x4* at_lane = reinterpret_cast<f32x4*>(lds) + (w / 2) * 64 * (4 * T::DB + 1) + lane;
    __syncthreads();  // the tiles have been read
    if (kw == 1) {
#pragma unroll
      for (int d = 0; d < T::DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4) at_lane[64 * (4 * d + r / 4)] = f32x4{o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]};
      at_lane[64 * 4 * T::DB] = f32x4{m, l, (float)ev, 0.f};
    }
    __syncthreads();
    if (kw == 1) return;
    const f32x4 other = at_lane[64 * 4 * T::DB];
    const float m1 = other[0], l1 = other[1], mj = fmaxf(m, m1);
    const int ev1 = (int)other[2], evj = max(ev, ev1);
    const float f0 = __builtin_amdgcn_exp2f(m - mj), f1 = __builtin_amdgcn_exp2f(m1 - mj);
    l = fmaf(l, f0, l1 * f1);
#pragma unroll
    for (int d = 0; d < T::DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const f32x4 x = at_lane[64 * (4 * d + r / 4)];
#pragma unroll
        for (int n = 0; n < 4; ++n)
          o[d][r + n] = fmaf(__builtin_amdgcn_ldexpf(o[d][r + n], ev - evj), f0, __builtin_amdgcn_ldexpf(x[n], ev1 - evj) * f1);
      }
    m = mj, ev = evj;
  }
  float mark = l;  // not finite where a score or a sum is not
#pragma unroll
  for (int d = 0; d < T::DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) mark = fmaf(0.f, o[d][r], mark);
  if (__any(odd || !(fabsf(mark) < INFINITY))) {
    for (int r = 0; r < 32; ++r)
      if (row0 + r < a.rows) plain_row(a, b, h, row0 + r);
    return;
  }
  if (i >= a.rows) return;
  const float f = live ? 1.f / l : 0.f;
  float* O = a.out + ((int64_t)b * a.rows + i) * a.ldo + (int64_t)h * a.dim;
#pragma unroll
  for (int d = 0; d < T::DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int col = 32 * d + 8 * (r >> 2) + 4 * half;
      f32x4u x;
#pragma unroll
      for (int n = 0; n < 4; ++n) x[n] = live ? __builtin_amdgcn_ldexpf(o[d][r + n] * f, ev - kTop) : 0.f;
      if (col + 4 <= a.dim) *reinterpret_cast<f32x4u*>(O + col) = x;
      else
#pragma unroll
        for (int n = 0; n < 4; ++n)
          if (col + n < a.dim) O[col + n] = x[n];
    }
  if (a.lse && half == 0) {
    // (in 64 bits from the logarithm of l's fraction on: an error of lse is one of all of the row's P; in 32
    // the gradients of 2 x 4 heads of 64 x 32 were off by 5e-7 of their norm, so by 2.6e-7)
    const double log2l = (double)__builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(l)) + __builtin_amdgcn_frexp_expf(l);
    a.lse[((int64_t)b * a.heads + h) * a.rows + i] = live ? (float)(((double)m + log2l) * 0.693147180559945309417) : -INFINITY;
  }
}

template <int DP>
void launch_dim(const Args& a, hipStream_t s) {
  // 8 waves share a tile, 4 where the window is small: a workgroup walks over window + rows
  // keys, of which a wave computes window + 32.  Where that leaves CUs idle two waves share 32 rows'
  // keys: 64 rows to a workgroup (6 heads of 777 x 80, window 200: 30 us against 40, 4 of 2048 x 64:
  // 25 against 34), or 128 where 64 would be no more workgroups or too many (32 heads of
  // 1024 x 64, all keys: 40 against 46).
  const auto blocks = [&](int rows) { return (int64_t)a.batch * a.heads * ((a.rows + rows - 1) / rows); };
  if (a.window >= 512 && blocks(256) >= 256)
    launch_blocks(tile_fwd_kernel<DP, 8, 1>, Grid(a, a.heads, (a.rows + 255) / 256, 8), 512, s, a);
  else if (blocks(64) <= 256 && blocks(64) > blocks(128))
    launch_blocks(tile_fwd_kernel<DP, 4, 2>, Grid(a, a.heads, (a.rows + 63) / 64, 8), 256, s, a);
  else if (blocks(128) <= 256)
    launch_blocks(tile_fwd_kernel<DP, 8, 2>, Grid(a, a.heads, (a.rows + 127) / 128, 8), 512, s, a);
  else
    launch_blocks(tile_fwd_kernel<DP, 4, 1>, Grid(a, a.heads, (a.rows + 127) / 128, 8), 256, s, a);
}

}  // namespace

void tile_forward(const Args& a, hipStream_t s) {
  if (a.dim <= 64) launch_dim<64>(a, s);
  else if (a.dim <= 96) launch_dim<96>(a, s);
  else launch_dim<128>(a, s);
}

}  // namespace wattn
