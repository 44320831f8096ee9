// The launches of the windowed attention's tiled kernels, and how their workgroups
// are numbered.
#pragma once
#include "window_attention.hpp"

#include <algorithm>

namespace wattn {

constexpr int kKeyBlock = 128;  // keys of a workgroup of the backward

// The backward's workspace, and what follows from the sizes.
struct BwdWork {
  int* ex;        // exponent of each row of dout, [batch, heads, rows]
  int* tile_ex;   // the largest of 64 rows, [batch, heads, tiles]
  float* near;    // parts of the keys' sums, [batch, kv_heads, key_blocks, nears, dk and dv, kKeyBlock, dim]
  float* far;     // far sums of the sinks, [batch, kv_heads, sink_blocks, fars, dk and dv, kKeyBlock, dim]
  int tiles, key_blocks, sink_blocks;
  int nears, near_rows;  // chunks of rows of a block's own and window, and their rows
  int fars, far_rows;    // chunks of rows past that
  // Rows from here on see a block's sinks alone.
  __host__ __device__ int near_end(const Args& a, int k0) const {
    const int64_t n = ((int64_t)k0 + kKeyBlock + a.window + 62) / 64 * 64;
    return (int)(n < tiles * 64ll ? n : tiles * 64ll);
  }
  explicit BwdWork(const Args& a) : ex(nullptr), tile_ex(nullptr), near(nullptr), far(nullptr) {
    tiles = (a.rows + 63) / 64;
    key_blocks = (a.keys + kKeyBlock - 1) / kKeyBlock;
    sink_blocks = (std::min(a.sinks, a.keys) + kKeyBlock - 1) / kKeyBlock;
    // Too few blocks of keys for half of the chip's 256 CUs: their rows in parts, the dq pass
    // taking the other half (4 heads of 2048 x 64, window 512, us: whole 82, in parts for 128
    // CUs 61, for 256 68; 6 heads of 777 x 80: 128, 97, 101).
    const int64_t blocks = (int64_t)a.batch * a.kv_heads * key_blocks;
    const int rows = near_end(a, 0);
    near_rows = rows;
    if (blocks > 0 && blocks < 128) near_rows = (int)std::max<int64_t>(64, (rows * blocks / 128 + 63) / 64 * 64);
    nears = rows > 0 ? (rows + near_rows - 1) / near_rows : 1;
    // short, so that they fill in behind the blocks of keys, no longer than those' parts (18 heads
    // of 777 x 80, us: 92 with twice as long ones, 86 so); longer where sinks are so many that
    // their blocks alone fill the chip, and their parts the memory
    const int after = std::max(a.rows - rows, 0);
    const int64_t sets = (int64_t)a.batch * a.kv_heads * sink_blocks, most = std::max<int64_t>(1, 2048 / std::max<int64_t>(sets, 1));
    far_rows = nears > 1 ? near_rows : std::max(256, a.window / 4);
    far_rows = (int)std::max<int64_t>(far_rows, (after + most - 1) / most);
    far_rows = (far_rows + 63) / 64 * 64;
    fars = sink_blocks > 0 && after > 0 ? (after + far_rows - 1) / far_rows : 0;
  }
  int kv_items() const { return key_blocks * nears + sink_blocks * fars; }  // workgroups of the kv pass to a head
  // Lays it out from `ws` (which may be null) after D; the bytes of all of it.
  size_t place(Args& a, void* ws) {
    char* p = static_cast<char*>(ws);
    size_t n = 0;
    auto take = [&](size_t bytes) {
      char* at = p ? p + n : nullptr;
      n += (bytes + 15) & ~(size_t)15;
      return at;
    };
    const size_t rows = (size_t)a.batch * a.heads * a.rows;
    a.delta = reinterpret_cast<float*>(take(rows * sizeof(float)));
    ex = reinterpret_cast<int*>(take(rows * sizeof(int)));
    tile_ex = reinterpret_cast<int*>(take((size_t)a.batch * a.heads * tiles * sizeof(int)));
    const size_t part = (size_t)a.batch * a.kv_heads * 2 * kKeyBlock * a.dim * sizeof(float);
    if (nears > 1) near = reinterpret_cast<float*>(take(part * key_blocks * nears));
    far = reinterpret_cast<float*>(take(part * sink_blocks * fars));
    return n;
  }
};

// A step's: few rows (heads of a group times tokens) over many keys.
struct StepWork {
  float* part;     // [batch, kv_heads, row_blocks, splits, 16 rows, dim and (maximum, sum)]
  int row_blocks;  // of 16 rows of a group
  int splits;      // of the keys
  // From 32 tokens on their rows fill a wave's 32 in the tiled forward.
  static bool few(int tokens) { return tokens < 32; }
  explicit StepWork(const Args& a) : part(nullptr) {
    row_blocks = (a.group * a.rows + 15) / 16;
    const int64_t groups = (int64_t)a.batch * a.kv_heads * row_blocks;
    const int64_t keys = std::min<int64_t>(a.keys, (int64_t)a.sinks + a.window + a.rows - 1);
    splits = 1;
    if (groups < 200) {
      // enough workgroups for the chip's 256 CUs twice, 128 keys (a block to a wave) or more
      // to each; one launch where a second would cost what it saves
      if (keys > 256)
        splits = (int)std::max<int64_t>(1, std::min<int64_t>({(512 + groups - 1) / groups, (keys + 127) / 128, 64}));
    } else if (row_blocks == 1) {
      // Whole groups, but where CUs would wait for the longest or the last of them (8 heads of keys x
      // 128, us whole and split; with more rows to a group splits only cost: 8 tokens of 32 x 32 heads
      // over 2048 keys 172 and 194).  A window that takes in the whole cache leaves what is read to
      // the lengths, which may be unlike: 32 of 1 to 8192: 261 and 211, one of 16384 among 31 of 500:
      // 426 and 72, 64 of 2048 to 4096: 297 and 277; but 32 of 4100 each: 180 and 199, and below 2560 keys as
      // much is lost (32 of 1 to 1024: 38 and 40).
      if (keys == a.keys) splits = (int)std::max<int64_t>(1, std::min<int64_t>(keys / 1280, 8));
      // Groups for a last round of half the CUs or less: 264 of 4100 keys 287 and 224, 384: 308 and 293, 520 of
      // 2050: 239 and 217, 264 of 1024: 77 and 73; 720 of 2050: 275 and 286, 264 of 512: 44 and 46.
      const int64_t last = groups % 256;
      if (groups > 256 && groups < 1024 && last > 0 && last <= 128)
        splits = std::max(splits, (int)std::max<int64_t>(1, std::min<int64_t>(keys / 512, 3)));
    }
  }
  size_t bytes(const Args& a) const {
    return splits == 1 ? 0 : (size_t)a.batch * a.kv_heads * row_blocks * splits * 16 * (a.dim + 2) * sizeof(float);
  }
};

void tile_forward(const Args& a, hipStream_t s);
void step_forward(const Args& a, const StepWork& w, hipStream_t s);
void tile_backward(const Args& a, const BwdWork& w, hipStream_t s);

struct Block {
  int b, h, row;
};
struct Place {
  int64_t group;
  int item;
};

// Workgroups: sequence, head, block of rows.  The blocks of one sequence and group of heads
// read the same keys and values: where the groups fill the 8 XCDs evenly, each XCD (a
// workgroup's number modulo 8) takes whole groups, so that its L2 holds them.  The last rows,
// which see the most, come first.  In a grid of a round or two (by_item) those of all groups do:
// its last workgroups are short (18 heads of 777 x 80, backward: 86 -> 65 us), and long and
// short ones share the CUs, where in turn they would each have their own (32 x 8 heads of 256
// x 64: 28.5 + 81 -> 25 + 74 us).  With more than `mixed` of them to a group they mix anyway: 4 x 8
// heads of 4096 x 64, 16 to a group forward, 161 us so against 170; backward 483 against 473.
// (A kernel may number a group's items by itself: Place.)
struct Grid {
  int64_t first, total, groups;
  int per_group, per_head, blocks;  // per_head: heads of a group; blocks: of rows
  int xcd, by_item;
  Grid(const Args& a, int heads, int blocks_, int mixed) : first(0) {
    groups = (int64_t)a.batch * a.kv_heads;
    per_head = heads / a.kv_heads;
    blocks = blocks_;
    per_group = per_head * blocks;
    total = groups * per_group;
    xcd = groups % 8 == 0;
    by_item = xcd ? total <= 1024 && per_group <= mixed : total <= 512;
  }
  __host__ __device__ __forceinline__ Place place(int64_t id) const {
    Place p;
    if (xcd) {
      const int64_t k = id >> 3;
      if (by_item) {  // (a small grid: 32 bits)
        const int n = (int)groups >> 3;
        p.item = (int)k / n;
        p.group = (int64_t)((int)k % n) * 8 + (id & 7);
      } else {
        const int64_t hi = k / per_group;
        p.item = (int)(k - hi * per_group);
        p.group = hi * 8 + (id & 7);
      }
    } else if (by_item) {
      p.group = (int)id % (int)groups;
      p.item = (int)id / (int)groups;
    } else {
      p.group = id / per_group;
      p.item = (int)(id - p.group * per_group);
    }
    return p;
  }
  __device__ __forceinline__ Block block(const Args& a, int rows) const { return block(a, rows, first + blockIdx.x); }
  __device__ __forceinline__ Block block(const Args& a, int rows, int64_t id) const {
    const Place p = place(id);
    Block r;
    r.b = (int)(p.group / a.kv_heads);
    r.h = (int)(p.group % a.kv_heads) * per_head + p.item % per_head;
    r.row = (blocks - 1 - p.item / per_head) * rows;
    return r;
  }
};

// All of the grid in launches of fewer than 2^32 threads.
template <class K, class... More>
void launch_blocks(K kernel, Grid g, int threads, hipStream_t s, const Args& a, const More&... more) {
  constexpr int64_t kBlocks = 1 << 22;
  for (; g.first < g.total; g.first += kBlocks)
    mle::launch(kernel, (unsigned)std::min<int64_t>(g.total - g.first, kBlocks), threads, 0, s, a, more..., g);
}

// The same for two grids one after the other.
template <class K>
void launch_both(K kernel, const Grid& g0, const Grid& g1, int threads, hipStream_t s, const Args& a, const BwdWork& wk) {
  constexpr int64_t kBlocks = 1 << 22;
  const int64_t total = g0.total + g1.total;
  for (int64_t f = 0; f < total; f += kBlocks)
    mle::launch(kernel, (unsigned)std::min(total - f, kBlocks), threads, 0, s, a, wk, g0, g1, f);
}

}  // namespace wattn
