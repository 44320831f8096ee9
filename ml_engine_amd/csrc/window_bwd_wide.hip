// Backward of the windowed attention for heads of more than 64 (window_bwd.hip has the plan and
// the scales): two waves to 32 keys, or rows.  One wave's operands and sums of such heads take
// all of a SIMD's registers and then some; half of the work each, two waves of a SIMD fit, and
// one's products run among the other's exponentials: 2 x 16 heads of 4096 x 128 under a window
// of 1024 took 1405 us, preparation and joins among them, with a wave to 32 keys, and take 815 so
// (fp32 products at 185 TFLOP/s, matrix cores 35 % busy, vector units 38 %).  Heads of 64 are better off without:
// 577 us against 705 at 4 x 8 heads of 4096.
#include "window_bwd.hpp"

using namespace mle;

namespace wattn {
namespace {

// What one of a pair of waves hands the other: P of a block, 16 values to a lane in the
// accumulators' order, and the power of two that it is held at.
struct Handed {
  f32x4 p[4][64];
  float at[64];
  __device__ __forceinline__ void put(int lane, const f32x16& x, float s) {
#pragma unroll
    for (int q = 0; q < 4; ++q) p[q][lane] = f32x4{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
    at[lane] = s;
  }
  __device__ __forceinline__ float get(int lane, f32x16& x) const {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4 v = p[q][lane];
#pragma unroll
      for (int r = 0; r < 4; ++r) x[4 * q + r] = v[r];
    }
    return at[lane];
  }
};

template <int DP, int NP>
struct Shared {
  alignas(16) char lds[3][2][Tile<DP, 32>::BYTES];  // [buffer][Q, dout or K, V]
  alignas(16) Handed hand[2][NP];
  Rows<32> rows[4];
  alignas(16) Tops<2 * NP> tops;
  int ex[2 * NP];
};

// dk and dv of 32 keys to a pair of waves, w and w + NP: the first takes S = Q K^T, P and
// dv^T += dout^T P, the second, one tile later, dP = dout V^T, dS and dk^T += Q^T dS, with P
// from the first.
template <int DP, int NP>
__device__ __forceinline__ void kv_pairs(const Args& a, const BwdWork& wk, const Place& place, Shared<DP, NP>& m) {
  using T = Tile<DP, 32>;
  constexpr int NT = 128 * NP, NW = 2 * NP, KB = 32 * NP, R = 32, AHEAD = 2;
  static_assert(KB == kKeyBlock, "keys of a workgroup");
  const KvJob job(a, wk, place);
  const int b = job.b, e = job.e, k0 = job.k0, i_end = job.i_end;
  const Seq seq(a, b);
  const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 31, half = lane >> 5;
  const int pair = w % NP;
  const int kw = k0 + 32 * pair, j = kw + c;  // of this pair, of this lane
  const bool live = j < seq.len;
  const int per_head = job.i_begin < i_end ? (i_end - job.i_begin + R - 1) / R : 0;
  const int count = per_head * a.group;
  if (count == 0 || a.dim < 4) {  // (the workgroup) nobody sees them, or rows too short to load
    job.plain(a, kw, w >= NP, w < NP);
    return;
  }
  const Places<T> at(lane);
  typedef Share<T, NT> Part;
  // Which of the pair this is tells its code: each has the registers to itself.
  const auto pass = [&](auto which) {
    constexpr bool second = decltype(which)::value;
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
    // This lane's row of K or V, at a power of two of its own.
    Frag own[T::KS];
    bool odd = false;
    int eo;
    {
      float x[T::KS][8];
      const float* p = (second ? a.v : a.k) + ((int64_t)b * a.keys + (live ? j : 0)) * (second ? a.ldv : a.ldk) + (int64_t)e * a.dim;
      const float top = load_row<T::KS>(p, half, a.dim, live, x);
      odd |= !(top < INFINITY);
      eo = exponent(fmaxf(top, other_half(top)));
#pragma unroll
      for (int s = 0; s < T::KS; ++s) own[s] = split8<false>(x[s], scale(eo));
    }
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
    int eq_next = kNone;  // the exponent of Q's operand so far
    auto put = [&](const Part& x, int t, char (*buf)[T::BYTES]) {
      const float mq = m.tops.get(0, t);
      const Rows<R>& r = m.rows[t & 3];
      odd |= !(mq < INFINITY) || r.odd != 0u;
      eq_next = raised(eq_next, mq, odd);
      const float sq = scale(eq_next);
      x.put(buf[0], buf[1], [&](bool g, int row) { return g ? scale(r.ex[row]) : sq; });
    };
    f32x16 sum[T::DB];  // dv^T or dk^T
#pragma unroll
    for (int d = 0; d < T::DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) sum[d][r] = 0.f;
    // this key's P is held at 2^sj (times its row's power of two), its dS at 2^(sj + tj)
    float sj = 100.f;
    int tj = 100, eq = kNone;
    const unsigned most = !live ? 0u : j < a.sinks ? 0x7fffffffu : (unsigned)a.window;  // how far its rows go
    // Tile t in buf, Q's exponent there being e.
    const auto block = [&](int t, const char (*buf)[T::BYTES], int e) {
      const Rows<R>& rw = m.rows[t & 3];
      const int i0 = here.r0;
      if (second && e != eq) {  // Q's operand has a larger power of two from here on
#pragma unroll
        for (int d = 0; d < T::DB; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) sum[d][r] = __builtin_amdgcn_ldexpf(sum[d][r], eq - e);
        eq = e;
      }
      // some pair of it visible?
      if (kw >= seq.len || i0 + 31 < kw || (i0 - (kw + 31) >= a.window && kw >= a.sinks)) return;
      f32x16 x;
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = 0.f;
      steps<T::KS, AHEAD>([&](int i) { return frag_row<T>(buf[second], at, 0, i); }, [&](int i, const Frag& f) { mma3(f, own[i], x); });
      Handed& h = m.hand[t & 1][pair];
      Frag op[2];
      if constexpr (!second) {
        const float ct = __builtin_amdgcn_ldexpf(a.scale * kLog2e, eo + e - 2 * kTop);
        const bool all = kw + 31 <= i0 && (i0 + 31 - kw < a.window || kw + 31 < a.sinks) && kw + 32 <= seq.len;
        float mx = -INFINITY;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x4 lse = *reinterpret_cast<const f32x4*>(&rw.lse[8 * q + 4 * half]);
#pragma unroll
          for (int r = 0; r < 4; ++r) x[4 * q + r] = fmaf(x[4 * q + r], ct, -lse[r]);
        }
        if (!all) hide_rows(x, i0 + 4 * half - j, most);
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, x[r]);
        if (__any(mx + sj > 15.f)) {
          mx = fmaxf(mx, other_half(mx));
          const float to = mx + sj > 15.f ? floorf(kHeld + 1 - mx) : sj;
          const int by = (int)(to - sj);
#pragma unroll
          for (int d = 0; d < T::DB; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) sum[d][r] = __builtin_amdgcn_ldexpf(sum[d][r], by);
          sj = to;
        }
        const float held = __builtin_amdgcn_ldexpf(1.f, (int)sj);  // (as a factor: in the exponent it would cost P's last bits)
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = __builtin_amdgcn_exp2f(x[r]) * held;
        h.put(lane, x, sj);
        op[0] = split_rows<true>(x, 0, 1.f), op[1] = split_rows<true>(x, 1, 1.f);
      } else {
        f32x16 p;
        const float s = h.get(lane, p);
        const float cd = __builtin_amdgcn_ldexpf(1.f, eo + kUnit - 2 * kTop);
        tj -= (int)(s - sj);
        sj = s;
        float mx = 0.f;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x4 delta = *reinterpret_cast<const f32x4*>(&rw.delta[8 * q + 4 * half]);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            x[4 * q + r] = p[4 * q + r] * fmaf(x[4 * q + r], cd, -delta[r]);
            mx = fmaxf(mx, fabsf(x[4 * q + r]));
          }
        }
        rescale(mx, tj, sum);
        const float ft = __builtin_amdgcn_ldexpf(1.f, tj);
        op[0] = split_rows<true>(x, 0, ft), op[1] = split_rows<true>(x, 1, ft);
      }
      steps<2 * T::DB, AHEAD>([&](int i) { return frag_col<T>(buf[!second], at, i / T::DB, i % T::DB); },
                              [&](int i, const Frag& f) { mma3(f, op[i / T::DB], sum[i % T::DB]); });
    };
    tell(in0, 0, first_row);
    tell(in, 1, ahead.r0);
    ahead.next();
    __syncthreads();
    put(in0.x, 0, m.lds[0]);
    int e_last = 0, now = 0, old = 2;  // the buffers of tiles t and t - 1
    for (int t = 0; t <= count; ++t) {
      __syncthreads();  // tile t lies in its buffer, nobody reads that of t + 1, which is announced; P of t - 1 is there
      const int et = eq_next, coming = now == 2 ? 0 : now + 1;
      if (t + 1 < count) put(in.x, t + 1, m.lds[coming]);
      fetch(in);
      if (second ? t > 0 : t < count) {
        block(second ? t - 1 : t, m.lds[second ? old : now], second ? e_last : et);
        here.next();
      }
      e_last = et, old = now, now = coming;
      if (t + 2 < count) {
        tell(in, t + 2, ahead.r0);
        ahead.next();
      }
    }
    float mark = 0.f;
#pragma unroll
    for (int d = 0; d < T::DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) mark = fmaf(0.f, sum[d][r], mark);
    if (__any(odd || mark != 0.f)) {  // (mark is 0 or NaN)
      job.plain(a, kw, second, !second);
      return;
    }
    if (j >= a.keys) return;
    float* grad = second ? a.dk + ((int64_t)b * a.keys + j) * a.lddk + (int64_t)e * a.dim
                         : a.dv + ((int64_t)b * a.keys + j) * a.lddv + (int64_t)e * a.dim;
    const float* was = (second ? a.acc_k : a.acc_v) && !job.part ? grad : nullptr;
    float* out = job.part ? job.part + ((second ? 0 : KB) + j - k0) * a.dim : grad;
    const int sh = !live ? 0 : second ? -(int)sj - tj + ex0 - kUnit + eq - kTop : -(int)sj + ex0 - kTop;
    const float factor = second ? a.scale : 1.f;
#pragma unroll
    for (int d = 0; d < T::DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        float x[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) x[n] = __builtin_amdgcn_ldexpf(sum[d][r + n] * factor, sh);
        store4(out, was, 32 * d + 8 * (r >> 2) + 4 * half, a.dim, x);
      }
  };
  if (w >= NP)
    pass(std::true_type{});
  else
    pass(std::false_type{});
}

// dq of 32 rows to a pair of waves, rows to lanes as in the forward: the first takes S^T = K Q^T
// and P, the second, one tile later, dP^T = V dout^T, dS and dq^T += K^T dS^T.
template <int DP, int NP>
__device__ __forceinline__ void q_pairs(const Args& a, const Block& blk, Shared<DP, NP>& m) {
  using T = Tile<DP, 32>;
  constexpr int NT = 128 * NP, R = 32, AHEAD = 2;
  const int b = blk.b, h = blk.h, e = h / a.group;
  const Seq seq(a, b);
  const int w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 31, half = lane >> 5;
  const int pair = w % NP;
  const int row0 = blk.row + 32 * pair, i = row0 + c;
  const bool live = i < seq.len;
  const int first = blk.row, last = min(blk.row + 32 * NP, seq.len) - 1;
  const int wlast = min(row0 + 32, seq.len) - 1;
  const bool any = first <= last;
  const Tiles<R> tiles(a, first, last);
  const int count = any ? tiles.count : 0;
  const auto plain = [&]() {  // this pair's rows with fp32 products
    if (w < NP) return;
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
  // Which of the pair this is tells its code: each has the registers to itself.
  const auto pass = [&](auto which) {
    constexpr bool second = decltype(which)::value;
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
    // this lane's row of Q or of dout, at a power of two of its own
    Frag own[T::KS];
    int eo;
    bool odd = false;
    {
      float x[T::KS][8];
      const float* p = (second ? a.dout : a.q) + ((int64_t)b * a.rows + (live ? i : 0)) * (second ? a.lddo : a.ldq) + (int64_t)h * a.dim;
      float top = load_row<T::KS>(p, half, a.dim, live, x);
      top = fmaxf(top, other_half(top));
      odd |= !(top < INFINITY);
      eo = exponent(top);
#pragma unroll
      for (int s = 0; s < T::KS; ++s) own[s] = split8<false>(x[s], scale(eo));
    }
    const int64_t st = ((int64_t)b * a.heads + h) * a.rows + (live ? i : 0);
    const float delta = live ? a.delta[st] : 0.f, lse = live ? a.lse_in[st] * kLog2e : 0.f;
    odd |= !(fabsf(delta) < INFINITY) || !(fabsf(lse) < INFINITY);
    int ek_next = kNone, ev = 0;
    auto put = [&](const Part& x, int t, char (*buf)[T::BYTES]) {
      const float mk = m.tops.get(0, t), mv = m.tops.get(1, t);
      odd |= !(fmaxf(mk, mv) < INFINITY);
      ek_next = raised(ek_next, mk, odd);
      ev = exponent(mv);
      const float sk = scale(ek_next), sv = scale(ev);
      x.put(buf[0], buf[1], [=](bool v, int) { return v ? sv : sk; });
    };
    f32x16 dq[T::DB];
#pragma unroll
    for (int d = 0; d < T::DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) dq[d][r] = 0.f;
    int ti = 100, ek = kNone;  // this row's dS is held at 2^ti; the exponent of K that dq is at
    const float dd = __builtin_amdgcn_ldexpf(delta, -eo);
    // Tile t in buf, the exponents of K and V there being e and f.
    const auto block = [&](int t, const char (*buf)[T::BYTES], int e, int f) {
      const int j0 = tiles.row(t);
      if (second && e != ek) {  // K's operand has a larger power of two from here on
#pragma unroll
        for (int d = 0; d < T::DB; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) dq[d][r] = __builtin_amdgcn_ldexpf(dq[d][r], ek - e);
        ek = e;
      }
      if (row0 > wlast || j0 > wlast || (row0 - (j0 + 31) >= a.window && j0 >= a.sinks)) return;
      f32x16 x;
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = 0.f;
      steps<T::KS, AHEAD>([&](int i) { return frag_row<T>(buf[second], at, 0, i); }, [&](int i, const Frag& f) { mma3(f, own[i], x); });
      Handed& h = m.hand[t & 1][pair];
      if constexpr (!second) {
        const float ct = __builtin_amdgcn_ldexpf(a.scale * kLog2e, eo + e - 2 * kTop);
        const bool all = j0 + 31 <= row0 && (wlast - j0 < a.window || j0 + 31 < a.sinks) && row0 + 32 <= seq.len;
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = fmaf(x[r], ct, -lse);
        if (!all) hide_keys(x, live ? i - j0 - 4 * half : -1, a.window, a.sinks - j0 - 4 * half, j0 < a.sinks);
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = __builtin_amdgcn_exp2f(x[r]);
        h.put(lane, x, 0.f);
      } else {
        f32x16 p;
        h.get(lane, p);
        const float cd = __builtin_amdgcn_ldexpf(1.f, f - 2 * kTop);  // dP - D at 2^-eo
        float mx = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          x[r] = p[r] * fmaf(x[r], cd, -dd);
          mx = fmaxf(mx, fabsf(x[r]));
        }
        rescale(mx, ti, dq);
        const float ft = __builtin_amdgcn_ldexpf(1.f, ti);
        const Frag op[2] = {split_rows<true>(x, 0, ft), split_rows<true>(x, 1, ft)};
        steps<2 * T::DB, AHEAD>([&](int i) { return frag_col<T>(buf[0], at, i / T::DB, i % T::DB); },
                                [&](int i, const Frag& f) { mma3(f, op[i / T::DB], dq[i % T::DB]); });
      }
    };
    tell(kv0, 0);
    tell(kv, 1);
    __syncthreads();
    put(kv0, 0, m.lds[0]);
    int ek_last = 0, ev_last = 0, now = 0, old = 2;  // the buffers of tiles t and t - 1
    for (int t = 0; t <= count; ++t) {
      __syncthreads();  // tile t lies in its buffer, nobody reads that of t + 1, which is announced; P of t - 1 is there
      const int ekt = ek_next, evt = ev, coming = now == 2 ? 0 : now + 1;
      if (t + 1 < count) put(kv, t + 1, m.lds[coming]);
      fetch(kv, t + 2);
      if (second ? t > 0 : t < count) block(second ? t - 1 : t, m.lds[second ? old : now], second ? ek_last : ekt, ev_last);
      ek_last = ekt, ev_last = evt, old = now, now = coming;
      if (t + 2 < count) tell(kv, t + 2);
    }
    if constexpr (second) {
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
      const int sh = live ? eo - ti + ek - kTop : 0;
#pragma unroll
      for (int d = 0; d < T::DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
          float x[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) x[n] = __builtin_amdgcn_ldexpf(dq[d][r + n] * a.scale, sh);
          store4(out, a.acc_q ? out : nullptr, 32 * d + 8 * (r >> 2) + 4 * half, a.dim, x);
        }
    }
  };
  if (w >= NP)
    pass(std::true_type{});
  else
    pass(std::false_type{});
}

// Both passes in one launch, the longer kv pass first: the one fills in behind the other.
template <int DP, int NP>
__global__ __launch_bounds__(128 * NP, 2) void wide_kernel(Args a, BwdWork wk, Grid kv, Grid q, int64_t first) {
  __shared__ Shared<DP, NP> m;
  const int64_t id = first + blockIdx.x;
  if (id < kv.total)
    kv_pairs<DP, NP>(a, wk, kv.place(id), m);
  else
    q_pairs<DP, NP>(a, q.block(a, 32 * NP, id - kv.total), m);
}

}  // namespace

void launch_wide(const Args& a, const BwdWork& wk, hipStream_t s) {
  constexpr int NP = kKeyBlock / 32;
  const Grid kv(a, a.kv_heads, wk.kv_items(), 1024), q(a, a.heads, (a.rows + 32 * NP - 1) / (32 * NP), 1024);
  if (a.dim <= 96)
    launch_both(wide_kernel<96, NP>, kv, q, 128 * NP, s, a, wk);
  else
    launch_both(wide_kernel<128, NP>, kv, q, 128 * NP, s, a, wk);
}

}  // namespace wattn
