// Embedding lookup with scaling, and the table's gradient by sorted tokens.
//
//   out[t] = scale table[key t],   dtable[v] = scale * sum of dy[t] over the tokens t with key v
//
// The forward also lists the tokens by key, in token order within a key: the
// index that the gradient sums from, so that no two threads add to one element
// and every sum has a fixed order, whatever the vocabulary's size.  Both
// directions are bound by memory (rows of the table and of dy); the index is
// latency that hides behind the lookup's stream, in the same launch.
//
// Index, in ints: head[64] (head[0]: tokens listed), rinfo[vocab] = {start,
// count} of each table row's tokens, list[tokens], skey[tokens] (the row of
// each place in the list).
#include "common.hpp"

#include <algorithm>

using namespace mle;

namespace {

constexpr int IX_NT = 1024;
constexpr int IX_RMAX = 1024;   // table rows of an index workgroup
constexpr int IX_WAVES = IX_NT / 64;
constexpr int IX_PER = 8;      // tokens of a lane, at most, in a chunk that it sorts at a time
constexpr int IX_CHUNK = IX_PER * IX_NT;
constexpr int HEAD = 64;
constexpr int PART = 16;        // places of the list that one partial sum covers

// A row in groups of W = 4 columns (VEC: rows of 4 columns or more, at any address of a
// float) or of one.  The last group of 4 is the row's last four columns, some of which
// belong to the group before it.
template <bool VEC>
struct Cols {
  static constexpr int W = VEC ? 4 : 1;
  typedef float vec __attribute__((ext_vector_type(W)));
  typedef float mem __attribute__((ext_vector_type(W), aligned(4)));  // as it lies in memory
  static __host__ __device__ int groups(int dim) { return (dim + W - 1) / W; }
  static __device__ __forceinline__ int at(int c, int dim) { return VEC ? min(c * 4, dim - 4) : c; }
  static __device__ __forceinline__ vec get(const float* p) { return *reinterpret_cast<const mem*>(p); }
  static __device__ __forceinline__ void put(float* p, vec v) { *reinterpret_cast<mem*>(p) = v; }
};

struct IndexArgs {
  const int32_t* keys;
  int clen, max_clen, ntok, vocab, rows_per_wg;
  int ranges, nix;  // of table rows; index workgroups, a multiple of ranges
  int per;          // tokens of a lane in a chunk
  int32_t* head;
  int2* rinfo;
  int32_t* list;
  int32_t* skey;
};

__device__ __forceinline__ int key_of(const IndexArgs& a, int t) {
  return a.clen == a.max_clen ? a.keys[t] : a.keys[(int64_t)(t / a.clen) * a.max_clen + t % a.clen];
}

struct IndexLds {
  int count[IX_WAVES][IX_RMAX];  // tokens of each row among a wave's, then where they go
  int next[IX_RMAX];             // the row's next place in the list
  int wave[IX_WAVES];
  int smaller;
};

// Exclusive prefix sums of one value per thread over the workgroup; total in `sum`.
__device__ __forceinline__ int exclusive_scan(int v, int* wave, int& sum) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int x = __shfl_up(incl, o, 64);
    if (lane >= o) incl += x;
  }
  __syncthreads();
  if (lane == 63) wave[w] = incl;
  __syncthreads();
  int before = 0;
  sum = 0;
#pragma unroll
  for (int i = 0; i < IX_NT / 64; ++i) {
    if (i < w) before += wave[i];
    sum += wave[i];
  }
  return before + incl - v;
}

// Lists the tokens of table rows [v0, v0 + nrows): every workgroup reads all
// the keys, and counts how many lie below its rows, which is where its part of
// the list starts.  A chunk's tokens are taken in order by the waves (64 * per
// consecutive ones each), 64 at a time.  Lanes with equal rows find each other by a
// ballot per bit of the row, so that a token knows its place among the wave's; the
// waves' counts in order give the rest.  Of many chunks, a range of rows has several
// workgroups: each counts all of them and lists its own (64000 tokens, 256 rows: one
// workgroup to a range 61 us, eight 20).
__device__ void index_rows(const IndexArgs& a, int wg, IndexLds& s) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  int range = wg, part = 0, parts = 1;
  if (a.nix != a.ranges) range = wg % a.ranges, part = wg / a.ranges, parts = a.nix / a.ranges;
  const int v0 = range * a.rows_per_wg, nrows = min(a.rows_per_wg, a.vocab - v0);
  const int rbits = 32 - __clz(max(nrows - 1, 1));
  const int per = a.per, chunk = per * IX_NT;
  // this lane's keys of a chunk, in token order by (wave, k, lane); -1 past the end
  auto load = [&](int c0, int (&key)[IX_PER]) {
    if (a.ntok == 0) return;
    const int t0 = c0 + w * per * 64 + lane;
    if (a.clen == a.max_clen) {  // (all loads on their way before the first is used)
#pragma unroll
      for (int k = 0; k < IX_PER; ++k) key[k] = a.keys[min(t0 + k * 64, a.ntok - 1)];
    } else {
#pragma unroll
      for (int k = 0; k < IX_PER; ++k) key[k] = key_of(a, min(t0 + k * 64, a.ntok - 1));
    }
#pragma unroll
    for (int k = 0; k < IX_PER; ++k)
      if (k >= per || t0 + k * 64 >= a.ntok) key[k] = -1;
  };
  auto clear = [&]() {
    for (int i = tid; i < IX_WAVES * nrows; i += IX_NT) s.count[i / nrows][i % nrows] = 0;
  };
  auto mine_of = [&](int key, unsigned& r) {
    r = (unsigned)key - (unsigned)v0;
    return r < (unsigned)nrows;  // (v0 + nrows <= 2^30: a negative id is past it)
  };
  // rank: the token's place among the wave's of its row
  auto rank_wave = [&](const int (&key)[IX_PER], int (&rank)[IX_PER]) {
#pragma unroll
    for (int k = 0; k < IX_PER; ++k) {
      unsigned r;
      const bool mine = mine_of(key[k], r);
      unsigned long long same = __ballot(mine);
      if (same == 0) continue;
      for (int b = 0; b < rbits; ++b) {
        const bool bit = (r >> b) & 1;
        const unsigned long long m = __ballot(bit);
        same &= bit ? m : ~m;
      }
      if (mine) {
        const int before = __popcll(same & ((1ull << lane) - 1));
        const int base = s.count[w][r];
        rank[k] = base + before;
        if (before == 0) s.count[w][r] = base + __popcll(same);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the wave's next 64 read what these wrote
    }
  };
  const bool single = a.ntok <= chunk;
  int key[IX_PER] = {-1, -1, -1, -1, -1, -1, -1, -1}, rank[IX_PER];
  static_assert(IX_PER == 8, "key");
  if (tid == 0) s.smaller = 0;
  clear();
  __syncthreads();
  // the chunks that this workgroup lists
  int first = 0, end = a.ntok;
  if (parts > 1) {
    const unsigned chunks = ((unsigned)a.ntok + IX_CHUNK - 1) / IX_CHUNK;  // (whole ones: per == IX_PER)
    first = (int)(chunks * part / parts) * IX_CHUNK;
    end = min((int)(chunks * (part + 1) / parts) * IX_CHUNK, a.ntok);
  }
  int below = 0, mine = 0, before = 0;  // the row's tokens: all, and those of chunks before
  auto add_counts = [&]() {
    int n = 0;
    if (tid < nrows)
#pragma unroll
      for (int i = 0; i < IX_WAVES; ++i) n += s.count[i][tid];
    return n;
  };
  if (single) {
    load(0, key);
#pragma unroll
    for (int k = 0; k < IX_PER; ++k) below += key[k] >= 0 && key[k] < v0;
    rank_wave(key, rank);
  } else {
    // Counted in any order: where the ids lie without gaps, four of a lane at a time.
    const bool flat = a.clen == a.max_clen && (reinterpret_cast<uintptr_t>(a.keys) & 15) == 0;
    auto load4 = [&](int c0, int (&key)[IX_PER]) {
      if (!flat || c0 + chunk > a.ntok) return load(c0, key);
#pragma unroll
      for (int k = 0; k < IX_PER; k += 4)
        *reinterpret_cast<int4*>(key + k) = *reinterpret_cast<const int4*>(a.keys + c0 + (w * per + k) * 64 + 4 * lane);
    };
    load4(0, key);
    for (int c0 = 0; c0 < a.ntok; c0 += chunk) {
      if (c0 == first && c0 > 0) {
        __syncthreads();
        before = add_counts();
        __syncthreads();
      }
      int next[IX_PER];
      load4(c0 + chunk, next);
#pragma unroll
      for (int k = 0; k < IX_PER; ++k) {
        below += (unsigned)key[k] < (unsigned)v0;
        unsigned r;
        if (mine_of(key[k], r)) atomicAdd(&s.count[w][r], 1);
      }
#pragma unroll
      for (int k = 0; k < IX_PER; ++k) key[k] = next[k];
    }
  }
  below = wave_sum(below);
  if (lane == 0) atomicAdd(&s.smaller, below);
  __syncthreads();
  mine = add_counts();
  int kept;
  const int start = s.smaller + exclusive_scan(mine, s.wave, kept);
  if (tid < nrows) {
    s.next[tid] = start + before;
    if (part == 0) a.rinfo[v0 + tid] = make_int2(start, mine);
  }
  if (wg == a.ranges - 1 && tid == 0) a.head[0] = s.smaller + kept;
  if (kept == 0) return;
  if (!single) load(first, key);
  for (int c0 = first; c0 < end; c0 += chunk) {
    if (!single) {
      __syncthreads();
      clear();
      __syncthreads();
      rank_wave(key, rank);
    }
    __syncthreads();
    if (tid < nrows) {
      int at = s.next[tid];
#pragma unroll
      for (int i = 0; i < IX_WAVES; ++i) {
        const int n = s.count[i][tid];
        s.count[i][tid] = at;
        at += n;
      }
      s.next[tid] = at;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < IX_PER; ++k) {
      unsigned r;
      if (!mine_of(key[k], r)) continue;
      const int to = s.count[w][r] + rank[k];
      a.list[to] = c0 + (w * per + k) * 64 + lane;
      a.skey[to] = key[k];
    }
    if (c0 + chunk < end) load(c0 + chunk, key);
  }
}

// Workgroups [0, nix) build the index, the rest look rows up.  8192 tokens x 512 with 8000
// ids 10.4 us (the index ends last), 32000 x 1024 with 128000 66-73 us (3.6-4.0 TB/s).
template <bool VEC, typename U>
__global__ __launch_bounds__(IX_NT, 8) void embed_fwd_kernel(IndexArgs a, float* __restrict__ out,
                                                          const float* __restrict__ table, int dim, float scale,
                                                          U units) {
  __shared__ IndexLds lds;
  if ((int)blockIdx.x < a.nix) {
    index_rows(a, blockIdx.x, lds);
    return;
  }
  typedef Cols<VEC> C;
  typedef typename C::vec vec;
  constexpr int UN = 4;
  const U stride = (U)(gridDim.x - a.nix) * IX_NT, per = (U)C::groups(dim);
  for (U u0 = (U)(blockIdx.x - a.nix) * IX_NT + threadIdx.x; u0 < units; u0 += UN * stride) {
    vec v[UN];
    int64_t to[UN];
#pragma unroll
    for (int k = 0; k < UN; ++k) {
      const U u = u0 + k * stride;
      v[k] = vec(0.f);
      if (u < units) {
        const U t = u / per;
        const int key = key_of(a, (int)t), col = C::at((int)(u - t * per), dim);
        to[k] = (int64_t)t * dim + col;
        if (key >= 0 && key < a.vocab) v[k] = scale * C::get(table + (int64_t)key * dim + col);
      }
    }
#pragma unroll
    for (int k = 0; k < UN; ++k) {
      const U u = u0 + k * stride;
      if (u < units) C::put(out + to[k], v[k]);  // (columns of two groups: twice the same)
    }
  }
}

struct GradArgs {
  float* dtable;
  const float* dy;
  const int32_t* head;
  const int2* rinfo;
  const int32_t* list;
  const int32_t* skey;
  float* part;  // [blocks][2][groups of columns]
  int dim, vocab, accumulate, blocks;
  float scale;
};

// The sum of dy's rows list[at .. at + n), column group c, in order.
template <bool VEC>
__device__ __forceinline__ typename Cols<VEC>::vec sum_rows(const GradArgs& a, int at, int n, int c) {
  typedef typename Cols<VEC>::vec vec;
  vec s = vec(0.f);
  const float* dy = a.dy + Cols<VEC>::at(c, a.dim);
  int j = 0;
  for (; j + 4 <= n; j += 4) {
    vec v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = Cols<VEC>::get(dy + (int64_t)a.list[at + j + k] * a.dim);
#pragma unroll
    for (int k = 0; k < 4; ++k) s += v[k];
  }
  for (; j < n; ++j) s += Cols<VEC>::get(dy + (int64_t)a.list[at + j] * a.dim);
  return s;
}
template <bool VEC>
__device__ __forceinline__ void put_row(const GradArgs& a, int row, int c, typename Cols<VEC>::vec s) {
  typedef Cols<VEC> C;
  const int col = C::at(c, a.dim), shared = c * C::W - col;  // columns that the group before has
  float* p = a.dtable + (int64_t)row * a.dim + col;
  s *= a.scale;
  if (shared == 0) {
    C::put(p, a.accumulate ? C::get(p) + s : s);
  } else {
#pragma unroll
    for (int k = 1; k < C::W; ++k)
      if (k >= shared) p[k] = a.accumulate ? p[k] + s[k] : s[k];
  }
}

// A token that occurs often would keep one wave busy for long, so a row with
// more than PART tokens is summed in blocks of PART places of the list: waves
// [0, blocks) write each block's sum of such a row (at most two rows reach
// into a block: one that began before it or at its start, slot 0, and one
// that begins within it, slot 1), and embed_join_kernel adds a row's blocks in
// order.  The other waves take 2^(6 - lw) table rows each, one after another
// by all their lanes' columns.  Bound by memory: a table of 128000 x 1024, 32000 tokens, 127 us
// (5.2 TB/s).
template <bool VEC>
__global__ __launch_bounds__(256) void embed_grad_kernel(GradArgs a, int lw) {
  typedef Cols<VEC> C;
  const int lane = threadIdx.x & 63;
  const int cols = C::groups(a.dim);
  const int64_t w = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  if (w < a.blocks) {
    const int total = a.head[0], p0 = (int)w * PART, n = min(PART, total - p0);
    if (n <= 0) return;
    const int key = lane < n ? a.skey[p0 + lane] : -1;
    const int2 info = lane < n ? a.rinfo[key] : make_int2(0, 0);
    const unsigned long long hot = __ballot(lane < n && info.y > PART);
    if (!hot) return;
#pragma unroll
    for (int slot = 0; slot < 2; ++slot) {
      // slot 0: the row of place p0; slot 1: the first hot row that begins later
      const unsigned long long begins = __ballot(lane < n && info.y > PART && info.x == p0 + lane && lane > 0);
      int b;
      if (slot == 0) {
        if (!(hot & 1)) continue;
        b = 0;
      } else {
        if (!begins) continue;
        b = __ffsll((long long)begins) - 1;
      }
      const int row = __shfl(key, b, 64);
      const int len = __popcll(__ballot(lane < n && key == row));
      for (int c = lane; c < cols; c += 64)
        C::put(a.part + ((w * 2 + slot) * cols + c) * C::W, sum_rows<VEC>(a, p0 + b, len, c));
    }
    return;
  }
  const int64_t row = (w - a.blocks) * (64 >> lw) + (lane >> lw);
  if (row >= a.vocab) return;
  const int2 info = a.rinfo[row];
  if (info.y > PART || (a.accumulate && info.y == 0)) return;
  for (int c = lane & ((1 << lw) - 1); c < cols; c += 1 << lw) put_row<VEC>(a, (int)row, c, sum_rows<VEC>(a, info.x, info.y, c));
}

// One workgroup per block of the list: joins the row that begins in it, if it
// is one of more than PART tokens.  CW threads cover CW column groups, 1024 / CW
// of them take the row's blocks in turn, and their sums are added in order.
template <bool VEC>
__global__ __launch_bounds__(1024) void embed_join_kernel(GradArgs a, int cw) {
  typedef Cols<VEC> C;
  typedef typename C::vec vec;
  __shared__ vec red[1024];
  const int total = a.head[0], p0 = (int)blockIdx.x * PART, n = min(PART, total - p0);
  if (n <= 0) return;
  const int lane = threadIdx.x & 63;
  const int2 info = lane < n ? a.rinfo[a.skey[p0 + lane]] : make_int2(0, 0);
  const unsigned long long begins = __ballot(lane < n && info.y > PART && info.x == p0 + lane);
  if (!begins) return;  // (the same in every wave)
  const int b = __ffsll((long long)begins) - 1;
  const int row = a.skey[p0 + b], count = __shfl(info.y, b, 64);
  const int nblk = (b + count + PART - 1) / PART;
  const int cols = C::groups(a.dim), groups = 1024 / cw, g = threadIdx.x / cw, t = threadIdx.x % cw;
  const int per = (nblk + groups - 1) / groups;  // each group a run of blocks
  for (int c0 = 0; c0 < cols; c0 += cw) {
    const int c = c0 + t;
    vec s = vec(0.f);
    if (c < cols) {
      const int k1 = min(nblk, (g + 1) * per);
      int k = g * per;
      auto at = [&](int i) {
        return a.part + ((((int64_t)blockIdx.x + i) * 2 + (i == 0 && b > 0 ? 1 : 0)) * cols + c) * C::W;
      };
      for (; k + 4 <= k1; k += 4) {
        vec v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = C::get(at(k + i));
#pragma unroll
        for (int i = 0; i < 4; ++i) s += v[i];
      }
      for (; k < k1; ++k) s += C::get(at(k));
    }
    __syncthreads();
    red[threadIdx.x] = s;
    __syncthreads();
    if (g == 0 && c < cols) {
      for (int i = 1; i < groups; ++i) s += red[i * cw + t];
      put_row<VEC>(a, row, c, s);
    }
  }
}

int check(const char* who, int batch, int clen, int dim, int vocab) {
  MLE_CHECK_ARG(batch >= 0 && clen > 0 && dim > 0 && dim <= (1 << 30) && vocab > 0 && vocab <= (1 << 30), "%s: bad shape (batch %d, clen %d, dim %d, vocab %d)", who,
                batch, clen, dim, vocab);
  MLE_CHECK_ARG((long long)batch * clen < 2147483647LL - 2 * IX_CHUNK, "%s: too many tokens", who);
  return MLE_OK;
}

size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

// The smallest power of two >= n, at most most.
int pow2_at_least(int n, int most) {
  int p = 1;
  while (p < n && p < most) p *= 2;
  return p;
}

}  // namespace

extern "C" {

size_t mle_embed_sorted_index_bytes(int batch, int clen, int vocab) {
  if (batch < 0 || clen <= 0 || vocab <= 0) return 0;
  return round256((HEAD + 2 * (size_t)vocab + 2 * (size_t)batch * clen) * sizeof(int32_t));
}

int mle_embed_scaled_fwd(mle_stream stream, float* out, const float* table, const int32_t* keys, int batch, int clen,
                         int max_clen, int dim, int vocab, float scale, void* index, size_t index_bytes) {
  const int rc = check("mle_embed_scaled_fwd", batch, clen, dim, vocab);
  if (rc) return rc;
  MLE_CHECK_ARG(table && max_clen >= clen && (batch == 0 || (out && keys)), "mle_embed_scaled_fwd: bad argument");
  if (index && (!aligned16(index) || index_bytes < mle_embed_sorted_index_bytes(batch, clen, vocab)))
    return set_error(MLE_ERR_WORKSPACE, "mle_embed_scaled_fwd: index of %zu bytes, 16-byte aligned, needed",
                     mle_embed_sorted_index_bytes(batch, clen, vocab));
  const int ntok = batch * clen;
  if (ntok == 0 && !index) return MLE_OK;
  IndexArgs a{keys, clen, max_clen, ntok, vocab, 0, 0, 0, 1, nullptr, nullptr, nullptr, nullptr};
  if (index) {
    a.rows_per_wg = std::min(IX_RMAX, std::max(32, (vocab + 255) / 256));
    a.ranges = (vocab + a.rows_per_wg - 1) / a.rows_per_wg;
    a.per = std::max(1, std::min(IX_PER, (int)(((int64_t)ntok + IX_NT - 1) / IX_NT)));
    // workgroups to list many chunks: up to two to a CU, which delays the lookup; one where
    // that is long (64000 tokens, 32000 rows of 512: 110 us with two, 124 with one; 32000
    // tokens, 128000 rows of 1024: 209 / 200)
    const int chunks = (int)(((int64_t)ntok + IX_CHUNK - 1) / IX_CHUNK);
    a.nix = a.ranges * std::max(1, std::min(chunks, (dim <= 512 ? 512 : 256) / a.ranges));
    a.head = static_cast<int32_t*>(index);
    a.rinfo = reinterpret_cast<int2*>(a.head + HEAD);
    a.list = reinterpret_cast<int32_t*>(a.rinfo + vocab);
    a.skey = a.list + ntok;
  }
  const bool vec = dim >= 4;
  const size_t units = (size_t)ntok * (vec ? Cols<true>::groups(dim) : dim);
  const unsigned grid = (unsigned)a.nix + (ntok ? stream_grid((units + 3) / 4, IX_NT, 2048) : 0u);
  hipStream_t s = as_stream(stream);
  // 32-bit numbering where the unrolled walk stays below 2^32
  const bool small = units < 4000000000u;
  if (vec && small) mle::launch(embed_fwd_kernel<true, uint32_t>, grid, IX_NT, 0, s, a, out, table, dim, scale, (uint32_t)units);
  else if (vec) mle::launch(embed_fwd_kernel<true, uint64_t>, grid, IX_NT, 0, s, a, out, table, dim, scale, (uint64_t)units);
  else if (small) mle::launch(embed_fwd_kernel<false, uint32_t>, grid, IX_NT, 0, s, a, out, table, dim, scale, (uint32_t)units);
  else mle::launch(embed_fwd_kernel<false, uint64_t>, grid, IX_NT, 0, s, a, out, table, dim, scale, (uint64_t)units);
  return check_launch("mle_embed_scaled_fwd");
}

size_t mle_embed_sorted_grad_ws_bytes(int batch, int clen, int dim) {
  if (batch <= 0 || clen <= 0 || dim <= 0) return 0;
  return round256(((size_t)batch * clen + PART - 1) / PART * 2 * (((size_t)dim + 3) / 4 * 4) * sizeof(float));
}

int mle_embed_sorted_grad(mle_stream stream, float* dtable, const float* dy, const void* index, size_t index_bytes,
                          int batch, int clen, int dim, int vocab, float scale, int accumulate, void* ws,
                          size_t ws_bytes) {
  const int rc = check("mle_embed_sorted_grad", batch, clen, dim, vocab);
  if (rc) return rc;
  MLE_CHECK_ARG(dtable && index && (batch == 0 || dy), "mle_embed_sorted_grad: null pointer");
  if (!aligned16(index) || index_bytes < mle_embed_sorted_index_bytes(batch, clen, vocab))
    return set_error(MLE_ERR_WORKSPACE, "mle_embed_sorted_grad: index of %zu bytes, 16-byte aligned, needed",
                     mle_embed_sorted_index_bytes(batch, clen, vocab));
  const size_t need = mle_embed_sorted_grad_ws_bytes(batch, clen, dim);
  if (need && (!ws || !aligned16(ws) || ws_bytes < need))
    return set_error(MLE_ERR_WORKSPACE, "mle_embed_sorted_grad: workspace of %zu bytes, 16-byte aligned, needed", need);
  const int ntok = batch * clen;
  const int32_t* head = static_cast<const int32_t*>(index);
  const int2* rinfo = reinterpret_cast<const int2*>(head + HEAD);
  const int32_t* list = reinterpret_cast<const int32_t*>(rinfo + vocab);
  GradArgs a{dtable, dy, head, rinfo, list, list + ntok, static_cast<float*>(ws), dim, vocab, accumulate,
             (ntok + PART - 1) / PART, scale};
  const bool vec = dim >= 4;
  const int cols = vec ? Cols<true>::groups(dim) : dim;
  int lw = 4;  // lanes of a table row: 16, 32 or 64
  while (lw < 6 && (1 << lw) < cols) ++lw;
  const int64_t waves = a.blocks + ((int64_t)vocab + (64 >> lw) - 1) / (64 >> lw);
  if (waves >= (1 << 26) || a.blocks >= (1 << 22))  // (a launch has fewer than 2^32 threads)
    return set_error(MLE_ERR_UNSUPPORTED, "mle_embed_sorted_grad: %d tokens or a table of %d rows are too many", ntok, vocab);
  hipStream_t s = as_stream(stream);
  const unsigned grid = (unsigned)((waves + 3) / 4);
  if (vec) mle::launch(embed_grad_kernel<true>, grid, 256, 0, s, a, lw);
  else mle::launch(embed_grad_kernel<false>, grid, 256, 0, s, a, lw);
  if (ntok > PART) {
    const int cw = pow2_at_least(cols, 256);
    if (vec) mle::launch(embed_join_kernel<true>, (unsigned)a.blocks, 1024, 0, s, a, cw);
    else mle::launch(embed_join_kernel<false>, (unsigned)a.blocks, 1024, 0, s, a, cw);
  }
  return check_launch("mle_embed_sorted_grad");
}

}  // extern "C"
