// Tables of a batch of drafted trees (or plain chunks) from request lengths,
// and the move of the accepted nodes' K/V to consecutive positions.
//
// tree_tables: sequence s holds prefix[s] cached positions and brings n new
// tokens, node i of which has the parent parents[q_start[s] + i] in its own
// sequence (negative: a root).  With depth(root) = 0 and depth(i) =
// depth(parent) + 1,
//   position(i) = prefix + depth(i)          (prefix + i without parents)
//   slot(i)     = table[(prefix + i) / B] * B + (prefix + i) % B
//   mask(i)     = mask(parent) | 1 << i      (64-bit words)
// Node order is storage order, so two siblings share a position and have
// slots of their own.  Latency bound: one CTA per sequence does all of it,
// the ancestor sets by pointer doubling in shared memory (log2(depth) rounds
// instead of a walk of up to depth dependent loads per node).  256 sequences of
// 64 nodes: 7.3 us on the GPU, one sequence of 8 nodes: 6.2 us; a call takes
// 18 us, which is the host allocating five tensors and launching.
//
// tree_commit: for j < path_len, K/V of node path[j] moves to position
// prefix + j in every layer.  A valid path rises, so path[j] >= j and no
// destination is a later source: loads of several entries are in flight
// before the first store and nothing needs a second buffer.  HBM bound: two
// times the moved bytes; 48 sequences x 32 layers, 8 heads x 128: 84 MB in
// 16 us, 5.2 TB/s, 80 % of measured HBM (a launch this short spends the rest
// on starting and on its tail).

#include "common.cuh"

namespace ksh {
namespace {

constexpr int kTabThreads = 256;
constexpr int kMaxWords = 4;           // 64-bit mask words per node (256 nodes)

struct TabArgs {
  const int32_t* prefix;
  const int32_t* new_lens;
  const int32_t* block_ids;      // ragged; NULL: block_tables is an input
  const int32_t* block_start;    // [S + 1]
  const int32_t* parents;        // [total] or NULL
  int32_t* q_start;              // [S + 1]
  int32_t* block_tables;         // [S, max_blocks]
  int64_t* positions;            // [total]
  int64_t* slots;                // [total]
  uint64_t* mask;                // [total, words] or NULL
  int32_t* flags;
  int64_t total, bs, max_blocks, num_block_ids;
  int num_seqs, words;
};

__device__ __forceinline__ int64_t block_sum_i64(int64_t v, int64_t* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  int64_t t = 0;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) t += red[w];
  return t;
}

__global__ void __launch_bounds__(kTabThreads) tree_tables_kernel(TabArgs a) {
  __shared__ int64_t red[kTabThreads / 32];
  __shared__ uint64_t m_s[kMaxWords][kTabThreads];
  __shared__ int16_t up_s[kTabThreads], dep_s[kTabThreads];
  const int s = blockIdx.x, tid = threadIdx.x;
  grid_dep_wait();
  grid_dep_launch();

  // rows before this sequence (the last CTA also writes the total)
  int64_t before = 0;
  for (int i = tid; i < s; i += kTabThreads) before += max(a.new_lens[i], 0);
  before = block_sum_i64(before, red);
  int raw_n = a.new_lens[s], raw_p = a.prefix[s];
  int64_t b0 = 0, nblk = a.max_blocks;
  bool bad = raw_n < 0 || raw_p < 0;
  if (a.block_ids) {
    b0 = a.block_start[s];
    nblk = a.block_start[s + 1] - b0;
    if (b0 < 0 || nblk < 0 || nblk > a.max_blocks || b0 + nblk > a.num_block_ids) {
      bad = true;
      nblk = 0;
    }
  }
  const int64_t n = max(raw_n, 0), pre = max(raw_p, 0);
  if (tid == 0) {
    a.q_start[s] = static_cast<int32_t>(before);
    if (s == a.num_seqs - 1) a.q_start[s + 1] = static_cast<int32_t>(before + n);
  }
  int32_t* row = a.block_tables + static_cast<int64_t>(s) * a.max_blocks;
  if (a.block_ids)
    for (int64_t j = tid; j < a.max_blocks; j += kTabThreads)
      row[j] = j < nblk ? a.block_ids[b0 + j] : 0;
  const int64_t room = a.total - before;           // rows left in the outputs
  if (n > room || (a.parents && n > static_cast<int64_t>(a.words) * 64)) bad = true;

  for (int64_t i0 = 0; i0 < n; i0 += kTabThreads) {
    const int64_t i = i0 + tid;
    int depth = 0;
    if (a.parents) {                               // one round: n <= 256
      const bool on = i < n && i < room;
      const int p = on ? a.parents[before + i] : -1;
      const bool ok = p >= 0 && p < i;
      if (on && p >= 0 && !ok) raise_flag(a.flags, KSH_FLAG_BAD_PARENT);
      uint64_t m[kMaxWords];
#pragma unroll
      for (int w = 0; w < kMaxWords; ++w) m[w] = (tid >> 6) == w ? 1ull << (tid & 63) : 0ull;
      int up = ok ? p : -1, dep = ok ? 1 : 0;
      // after round k a node holds the 2^k nearest members of its chain
      for (int it = 0; it < 8; ++it) {
        up_s[tid] = static_cast<int16_t>(up);
        dep_s[tid] = static_cast<int16_t>(dep);
#pragma unroll
        for (int w = 0; w < kMaxWords; ++w)
          if (w < a.words) m_s[w][tid] = m[w];
        if (!__syncthreads_or(up >= 0)) break;
        if (up >= 0) {
#pragma unroll
          for (int w = 0; w < kMaxWords; ++w)
            if (w < a.words) m[w] |= m_s[w][up];
          dep += dep_s[up];
          up = up_s[up];
        }
        __syncthreads();
      }
      depth = dep;
      if (on && a.mask) {
#pragma unroll
        for (int w = 0; w < kMaxWords; ++w)
          if (w < a.words) a.mask[(before + i) * a.words + w] = m[w];
      }
    }
    if (i < n && i < room) {
      const int64_t at = pre + i, j = at / a.bs;
      int64_t slot = -1;
      if (j < nblk) {
        const int32_t blk = a.block_ids ? a.block_ids[b0 + j] : row[j];
        slot = static_cast<int64_t>(blk) * a.bs + at % a.bs;
      } else {
        bad = true;
      }
      a.positions[before + i] = a.parents ? pre + depth : at;
      a.slots[before + i] = slot;
    }
    if (a.parents) break;
  }
  // rows past the last sequence (total larger than the lengths say) and nodes
  // past the mask's capacity
  if (s == a.num_seqs - 1 && before + n != a.total) bad = true;
  const int64_t done = a.parents && n > kTabThreads ? before + kTabThreads : before + n;
  const int64_t stop = s == a.num_seqs - 1 ? a.total : min(before + n, a.total);
  for (int64_t r = done + tid; r < stop; r += kTabThreads) {
    a.positions[r] = 0;
    a.slots[r] = -1;
    if (a.mask)
      for (int w = 0; w < a.words; ++w) a.mask[r * a.words + w] = 0;
  }
  if (bad) raise_flag(a.flags, KSH_FLAG_BAD_LENGTH);
}

struct CommitArgs {
  float* pool;
  const int32_t* block_tables;
  const int32_t* prefix;
  const int32_t* path;          // [S, path_stride]
  const int32_t* path_len;
  int32_t* new_lens;            // [S] prefix + path_len, or NULL
  int32_t* flags;
  int64_t num_blocks, num_layers, hkv, bs, d, max_blocks, path_stride;
};

constexpr int kCommitThreads = 256;
constexpr int kMaxMoves = 256;

// One CTA per (layer, sequence); a thread owns one element (V: float4 or
// float) of the 2 * hkv * d floats of a token and walks the moves in batches.
template <typename V>
__global__ void __launch_bounds__(kCommitThreads) tree_commit_kernel(CommitArgs a) {
  __shared__ int64_t src_s[kMaxMoves], dst_s[kMaxMoves];
  __shared__ int n_s;
  const int tid = threadIdx.x;
  const int64_t layer = blockIdx.x, s = blockIdx.y;
  grid_dep_wait();
  grid_dep_launch();
  const int64_t pre = a.prefix[s];
  int64_t len = a.path_len[s];
  const bool first = layer == 0 && tid == 0;
  if (len < 0 || len > a.path_stride || pre < 0) {
    if (first) raise_flag(a.flags, KSH_FLAG_BAD_LENGTH);
    len = 0;
  }
  if (first && a.new_lens) a.new_lens[s] = static_cast<int32_t>(max(pre, int64_t(0)) + len);
  const int32_t* path = a.path + s * a.path_stride;
  const int32_t* table = a.block_tables + s * a.max_blocks;
  // float offset of a token's K row of head 0 in this layer, -1 if it has none
  auto offset = [&](int64_t pos) -> int64_t {
    const int64_t j = pos / a.bs;
    if (j >= a.max_blocks) return -1;
    const int64_t blk = table[j];
    if (blk < 0 || blk >= a.num_blocks) return -1;
    return (((blk * a.num_layers + layer) * 2) * a.hkv * a.bs + pos % a.bs) * a.d;
  };
  for (int64_t j0 = 0; j0 < len; j0 += kMaxMoves) {
    if (tid == 0) n_s = 0;
    __syncthreads();
    // entries that move, in path order
    if (tid < 32) {
      int n = 0;
      for (int64_t j = j0 + tid; j - tid < min(len, j0 + kMaxMoves); j += 32) {
        int64_t so = -1, dp = -1;
        if (j < len) {
          const int64_t p = path[j], q = j > 0 ? path[j - 1] : -1;
          if (p <= q || p < j) {                   // not a rising path: the entry stays
            if (layer == 0) raise_flag(a.flags, KSH_FLAG_BAD_LENGTH);
          } else if (p != j) {
            so = offset(pre + p);
            dp = offset(pre + j);
            if ((so < 0 || dp < 0) && layer == 0) raise_flag(a.flags, KSH_FLAG_BAD_BLOCK);
          }
        }
        const bool on = so >= 0 && dp >= 0;
        const unsigned votes = __ballot_sync(0xffffffffu, on);
        if (on) {
          const int at = n + __popc(votes & ((1u << tid) - 1));
          src_s[at] = so;
          dst_s[at] = dp;
        }
        n += __popc(votes);
      }
      if (tid == 0) n_s = n;
    }
    __syncthreads();
    const int n = n_s;
    constexpr int E = sizeof(V) / 4;
    const int64_t per = a.d / E, rows = 2 * a.hkv;
    for (int64_t x = tid; x < rows * per; x += blockDim.x) {
      const int64_t r = x / per, c = x - r * per;
      const int64_t at = r * a.bs * a.d + c * E;
      for (int k0 = 0; k0 < n; k0 += 8) {
        V v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k0 + k < n) v[k] = *reinterpret_cast<const V*>(a.pool + src_s[k0 + k] + at);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k0 + k < n) *reinterpret_cast<V*>(a.pool + dst_s[k0 + k] + at) = v[k];
      }
    }
    __syncthreads();
  }
}

}  // namespace
}  // namespace ksh

using namespace ksh;

extern "C" int ksh_tree_tables(const int32_t* prefix_lens, const int32_t* new_lens,
                               int64_t num_seqs, int64_t total, int64_t block_size,
                               const int32_t* block_ids, int64_t num_block_ids,
                               const int32_t* block_start, int64_t max_blocks,
                               const int32_t* parents, int64_t mask_words, int32_t* q_start,
                               int32_t* block_tables, int64_t* positions, int64_t* slots,
                               uint64_t* mask, int32_t* flags, void* stream) {
  KSH_CHECK_ARG(num_seqs > 0 && num_seqs <= INT32_MAX && total >= 0 && total <= INT32_MAX &&
                block_size > 0 && max_blocks > 0 && num_block_ids >= 0);
  KSH_CHECK_ARG(prefix_lens && new_lens && q_start && block_tables);
  KSH_CHECK_ARG(total == 0 || (positions && slots));
  KSH_CHECK_ARG((block_ids == nullptr) == (block_start == nullptr));
  if (parents) {
    KSH_CHECK_ARG(mask_words > 0 && (mask || total == 0));
    if (mask_words > kMaxWords) return KSH_ERR_UNSUPPORTED;
  }
  TabArgs a = {};
  a.prefix = prefix_lens;
  a.new_lens = new_lens;
  a.block_ids = block_ids;
  a.block_start = block_start;
  a.parents = parents;
  a.q_start = q_start;
  a.block_tables = block_tables;
  a.positions = positions;
  a.slots = slots;
  a.mask = parents ? mask : nullptr;
  a.flags = flags;
  a.total = total;
  a.bs = block_size;
  a.max_blocks = max_blocks;
  a.num_block_ids = num_block_ids;
  a.num_seqs = static_cast<int>(num_seqs);
  a.words = parents ? static_cast<int>(mask_words) : 0;
  return launch(tree_tables_kernel, dim3(static_cast<unsigned>(num_seqs)), dim3(kTabThreads), 0,
                static_cast<cudaStream_t>(stream), a);
}

extern "C" int ksh_tree_commit(float* pool, int64_t num_blocks, int64_t num_layers, int64_t hkv,
                               int64_t block_size, int64_t d, const int32_t* block_tables,
                               int64_t max_blocks, const int32_t* prefix_lens, int64_t num_seqs,
                               const int32_t* path, int64_t path_stride, const int32_t* path_len,
                               int32_t* new_lens, int32_t* flags, void* stream) {
  KSH_CHECK_ARG(num_blocks > 0 && num_layers > 0 && num_layers <= INT32_MAX && hkv > 0 &&
                block_size > 0 && d > 0 && max_blocks > 0 && num_seqs > 0 && path_stride > 0);
  KSH_CHECK_ARG(pool && block_tables && prefix_lens && path && path_len);
  if (num_seqs > 65535) return KSH_ERR_UNSUPPORTED;
  CommitArgs a = {};
  a.pool = pool;
  a.block_tables = block_tables;
  a.prefix = prefix_lens;
  a.path = path;
  a.path_len = path_len;
  a.new_lens = new_lens;
  a.flags = flags;
  a.num_blocks = num_blocks;
  a.num_layers = num_layers;
  a.hkv = hkv;
  a.bs = block_size;
  a.d = d;
  a.max_blocks = max_blocks;
  a.path_stride = path_stride;
  const dim3 grid(static_cast<unsigned>(num_layers), static_cast<unsigned>(num_seqs));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // More CTAs than eight per SM: half as wide, so that they still run at once
  // (48 sequences x 32 layers, 8 heads x 128: 11.2 us from L2, 13.8 with 256
  // threads).  With few of them the wide ones finish a token sooner (4
  // sequences: 10.2 us cold, 12.3 with 128).
  const dim3 block(num_layers * num_seqs > 8 * static_cast<int64_t>(num_sms()) ? kCommitThreads / 2 : kCommitThreads);
  if (d % 4 == 0 && (reinterpret_cast<uintptr_t>(pool) & 15) == 0)
    return launch(tree_commit_kernel<float4>, grid, block, 0, st, a);
  return launch(tree_commit_kernel<float>, grid, block, 0, st, a);
}
