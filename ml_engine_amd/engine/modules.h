// Layer compositions used by the benchmark configurations, built only from
// GraphOperations ops: MultiHeadAttention (Includes/transformer.h,
// Engine/transformer.cu:635-661), WindowSelfAttention and the diffusion
// ResidualBlock (Includes/diffusion.h:35-46, Engine/diffusion.cu:109-137).
#pragma once
#include <memory>
#include <vector>

#include "engine.h"

class MultiHeadAttention {
 public:
  int hidden, embed_dim, num_heads, head_dim;
  str name;
  Linear q, k, v, o;
  bool qkv_fused = false;  // set by forward: dX of the Q, K, V projections is one grouped GEMM
  MultiHeadAttention(const int embed_dim, const int hidden, const int num_heads, const str& name = "MHA");
  graph forward(const graph& X, const bool mask = true);
  void save(std::ofstream& f) const;
  void load(std::ifstream& f);
};

// Self-attention with rotary positions over a causal window and sinks, the heads of Q in
// groups that share a head of K and V (no counterpart in the reference, whose
// MultiHeadAttention adds positions to its input and softmaxes whole columns).
class WindowSelfAttention {
 public:
  int embed_dim, num_heads, kv_heads, head_dim, window, sinks;
  str name;
  Linear q, k, v, o;
  WindowSelfAttention(const int embed_dim, const int num_heads, const int kv_heads, const int head_dim,
                      const int window, const int sinks = 0, const str& name = "Window Attention");
  // positions: device ids [sections.size()][batch * seq], sections the pairs of a head that turn
  // by each axis; lengths: device ids [batch] or nullptr.
  graph forward(const graph& X, const int32_t* positions, const std::vector<int>& sections,
                const int32_t* lengths = nullptr, const double base = 10000.0, const int rotary_flags = 0);
  void save(std::ofstream& f) const;
  void load(std::ifstream& f);
};

class ResidualBlock {
 public:
  std::unique_ptr<Convolute2D> conv1, conv2, skipconv;
  std::unique_ptr<Linear> time_mlp;
  int in, out, hidden, stride, groups;
  // `groups` is the GroupNorm group count (the reference always uses the
  // GroupNorm default of 8; the diffusion benchmark block uses 32).
  ResidualBlock(const int in_channels, const int out_channels, const int t_hidden, const int stride = 1,
                const int groups = 8);
  graph forward(const graph& x, const graph& t_emb);
  void save(std::ofstream& f) const;
  void load(std::ifstream& f);
};
