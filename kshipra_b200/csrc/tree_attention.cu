// Attention of drafted tokens over the paged cache.
//
// Sequence s has prefix[s] cached positions and n = q_start[s+1] - q_start[s]
// drafted nodes whose K/V stand in the slots of positions prefix .. prefix +
// n - 1 (node order).  Node i attends every cached position and the nodes
// whose bit is set in its mask (64-bit words; no mask: nodes 0..i):
//     o = sum_j exp(q.k_j / sqrt(D) - m) v_j / sum_j exp(q.k_j / sqrt(D) - m)
// with the running maximum m, rescaled as it rises.  A node that may see no
// key gives zeros.  Keys that a node may not see are never read into its sums
// (a NaN there stays there).

#include <math.h>

#include <algorithm>

#include "common.cuh"

namespace ksh {
namespace {

constexpr int kMaxWords = 4;           // mask words per node: 256 nodes

struct TreeArgs {
  const float* q;               // [total, hq, d]
  const float* pool;            // [nb, L, 2, hkv, bs, d]
  const int32_t* block_tables;  // [S, max_blocks]
  const int32_t* q_start;       // [S + 1]
  const int32_t* prefix;        // [S]
  const uint64_t* mask;         // [total, words] or NULL
  float* out;                   // [total, hq, d]
  int32_t* flags;
  int64_t total, num_blocks, num_layers, layer, hkv, hq, bs, max_blocks;
  int num_seqs, words, g, d, max_nodes;
  float scale;
};

// One warp per (node, head), keys one after the other: any head dimension up
// to 256 and any alignment.
__global__ void __launch_bounds__(32) tree_attn_simple_kernel(TreeArgs a) {
  const int lane = threadIdx.x, i = blockIdx.x, h = blockIdx.y, s = blockIdx.z;
  grid_dep_wait();
  grid_dep_launch();
  const int64_t a0 = a.q_start[s], n = a.q_start[s + 1] - a0;
  if (a0 < 0 || n < 0 || a0 + n > a.total || n > a.max_nodes) {
    if (lane == 0) raise_flag(a.flags, KSH_FLAG_BAD_LENGTH);
  }
  if (i >= n || a0 < 0 || a0 + i >= a.total) return;
  const int d = a.d;
  const int64_t pre = max(a.prefix[s], 0);
  const int64_t cap = a.max_blocks * a.bs;
  if (pre + n > cap && lane == 0) raise_flag(a.flags, KSH_FLAG_BAD_LENGTH);
  const int64_t end = min(pre + n, cap);
  const float* q = a.q + ((a0 + i) * a.hq + h) * d;
  const int hk = h / a.g;
  constexpr int kPer = 8;
  float acc[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) acc[e] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  bool bad = false;
  for (int64_t pos = 0; pos < end; ++pos) {
    if (pos >= pre) {
      const int j = static_cast<int>(pos - pre);
      const bool see = a.mask ? (j < a.words * 64 &&
                                 ((a.mask[(a0 + i) * a.words + (j >> 6)] >> (j & 63)) & 1))
                              : j <= i;
      if (!see) continue;
    }
    const int64_t b = pos / a.bs;
    const int64_t blk = a.block_tables[static_cast<int64_t>(s) * a.max_blocks + b];
    if (blk < 0 || blk >= a.num_blocks) {
      bad = true;
      continue;
    }
    const float* k = a.pool + ((((blk * a.num_layers + a.layer) * 2) * a.hkv + hk) * a.bs +
                               (pos - b * a.bs)) * d;
    const float* v = k + a.hkv * a.bs * d;
    float dot = 0.0f;
    for (int c = lane; c < d; c += 32) dot = fmaf(q[c], k[c], dot);
    const float x = warp_sum(dot) * a.scale;
    const float mn = fmaxf(m, x), ms = mn == -INFINITY ? 0.0f : mn;
    const float p = expf(x - ms), corr = expf(m - ms);
    l = fmaf(l, corr, p);
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int c = lane + 32 * e;
      if (c < d) acc[e] = fmaf(acc[e], corr, p * v[c]);
    }
    m = mn;
  }
  if (bad && lane == 0) raise_flag(a.flags, KSH_FLAG_BAD_BLOCK);
  float* o = a.out + ((a0 + i) * a.hq + h) * d;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int c = lane + 32 * e;
    if (c < d) o[c] = l == 0.0f ? 0.0f : acc[e] / l;
  }
}

}  // namespace
}  // namespace ksh

using namespace ksh;

extern "C" int64_t ksh_tree_attention_workspace_size(int64_t num_seqs, int64_t hq, int64_t hkv,
                                                     int64_t d, int64_t max_nodes) {
  (void)max_nodes;
  if (num_seqs <= 0 || hq <= 0 || hkv <= 0 || hq % hkv != 0 || d <= 0) return 0;
  return 256;
}

extern "C" int ksh_tree_attention(const float* q, int64_t total, int64_t hq, int64_t d,
                                  const float* pool, int64_t num_blocks, int64_t num_layers,
                                  int64_t layer, int64_t hkv, int64_t block_size,
                                  const int32_t* block_tables, int64_t max_blocks,
                                  const int32_t* q_start, const int32_t* prefix_lens,
                                  int64_t num_seqs, const uint64_t* mask, int64_t mask_words,
                                  int64_t max_nodes, int64_t max_total_len, float* out,
                                  void* workspace, int64_t workspace_bytes, int32_t* flags,
                                  void* stream) {
  KSH_CHECK_ARG(hq > 0 && hkv > 0 && hq % hkv == 0 && d > 0 && num_blocks > 0 &&
                num_layers > 0 && layer >= 0 && layer < num_layers && block_size > 0 &&
                max_blocks > 0 && num_seqs >= 0 && num_seqs <= INT32_MAX && total >= 0 &&
                total <= INT32_MAX && max_nodes >= 0 && max_total_len >= 0);
  KSH_CHECK_ARG(!mask || mask_words > 0);
  if (num_seqs == 0 || total == 0 || max_nodes == 0) return KSH_OK;
  KSH_CHECK_ARG(q && pool && block_tables && q_start && prefix_lens && out);
  if (d > 256 || max_nodes > kMaxWords * 64 || (mask && mask_words > kMaxWords))
    return KSH_ERR_UNSUPPORTED;
  TreeArgs a = {};
  a.q = q;
  a.pool = pool;
  a.block_tables = block_tables;
  a.q_start = q_start;
  a.prefix = prefix_lens;
  a.mask = mask;
  a.out = out;
  a.flags = flags;
  a.total = total;
  a.num_blocks = num_blocks;
  a.num_layers = num_layers;
  a.layer = layer;
  a.hkv = hkv;
  a.hq = hq;
  a.bs = block_size;
  a.max_blocks = max_blocks;
  a.num_seqs = static_cast<int>(num_seqs);
  a.words = mask ? static_cast<int>(mask_words) : 0;
  a.g = static_cast<int>(hq / hkv);
  a.d = static_cast<int>(d);
  a.max_nodes = static_cast<int>(max_nodes);
  a.scale = static_cast<float>(1.0 / sqrt(static_cast<double>(d)));
  (void)workspace;
  (void)workspace_bytes;
  if (hq > 65535 || num_seqs > 65535) return KSH_ERR_UNSUPPORTED;
  return launch(tree_attn_simple_kernel,
                dim3(static_cast<unsigned>(max_nodes), static_cast<unsigned>(hq),
                     static_cast<unsigned>(num_seqs)),
                dim3(32), 0, static_cast<cudaStream_t>(stream), a);
}
