// Attention of a chunk of new tokens over the 16-bit paged cache.
//
// Sequence s has prefix[s] cached positions and brings n = q_start[s+1] -
// q_start[s] rows whose K/V stand at positions prefix .. prefix + n - 1.  Row i
// attends positions 0 .. prefix + i:
//     o = sum_j exp(q.k_j / sqrt(D) - m) v_j / sum_j exp(q.k_j / sqrt(D) - m)
// with the running maximum m.  q and o are fp32, K and V fp16 or bf16.

#include <cuda_bf16.h>
#include <math.h>

#include <algorithm>

#include "tc_common.cuh"

namespace ksh {
namespace {

using namespace tc;

struct CacheArgs {
  const float* q;               // [total, hq, d]
  const void* pool;             // [nb, L, 2, hkv, bs, d]
  const int32_t* block_tables;  // [S, max_blocks]
  const int32_t* q_start;       // [S + 1]
  const int32_t* prefix;        // [S]
  float* out;                   // [total, hq, d]
  int32_t* flags;
  int64_t total, num_blocks, num_layers, layer, hkv, hq, bs, max_blocks;
  int num_seqs, g, d, max_q;
  float scale;
};

__device__ __forceinline__ float widen(__half x) { return __half2float(x); }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }

// Any head dimension up to 256 and any alignment: one warp per (row, head), keys
// one after the other.
template <typename T>
__global__ void __launch_bounds__(32) cache_attn_simple_kernel(CacheArgs a) {
  const int lane = threadIdx.x, i = blockIdx.x, h = blockIdx.y, s = blockIdx.z;
  grid_dep_wait();
  grid_dep_launch();
  const int64_t a0 = a.q_start[s], n = a.q_start[s + 1] - a0;
  const int64_t pre = max(a.prefix[s], 0);
  const int64_t cap = a.max_blocks * a.bs;
  if (lane == 0 && (a0 < 0 || n < 0 || a0 + n > a.total || n > a.max_q || a.prefix[s] < 0 || pre + n > cap))
    raise_flag(a.flags, KSH_FLAG_BAD_LENGTH);
  if (i >= n || a0 < 0 || a0 + i >= a.total) return;
  const int d = a.d;
  const int64_t end = min(pre + i + 1, cap);
  const float* q = a.q + ((a0 + i) * a.hq + h) * d;
  const int hk = h / a.g;
  const T* pool = static_cast<const T*>(a.pool);
  constexpr int kPer = 8;
  float acc[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) acc[e] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  bool bad = false;
  for (int64_t pos = 0; pos < end; ++pos) {
    const int64_t b = pos / a.bs;
    const int64_t blk = a.block_tables[static_cast<int64_t>(s) * a.max_blocks + b];
    if (blk < 0 || blk >= a.num_blocks) {
      bad = true;
      continue;
    }
    const T* k = pool + ((((blk * a.num_layers + a.layer) * 2) * a.hkv + hk) * a.bs + (pos - b * a.bs)) * d;
    const T* v = k + a.hkv * a.bs * d;
    float dot = 0.0f;
    for (int c = lane; c < d; c += 32) dot = fmaf(q[c], widen(k[c]), dot);
    const float x = warp_sum(dot) * a.scale;
    const float mn = fmaxf(m, x), ms = mn == -INFINITY ? 0.0f : mn;
    const float p = expf(x - ms), corr = expf(m - ms);
    l = fmaf(l, corr, p);
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int c = lane + 32 * e;
      if (c < d) acc[e] = fmaf(acc[e], corr, p * widen(v[c]));
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

extern "C" int64_t ksh_cache_attention_workspace_size(int64_t num_seqs, int64_t hq, int64_t hkv,
                                                      int64_t d, int64_t max_q_len) {
  if (num_seqs <= 0 || hq <= 0 || hkv <= 0 || hq % hkv != 0 || d <= 0 || max_q_len < 0) return 0;
  return 256;
}

extern "C" int ksh_cache_attention(const float* q, int64_t total, int64_t hq, int64_t d,
                                   const void* pool, int pool_type, int64_t num_blocks,
                                   int64_t num_layers, int64_t layer, int64_t hkv,
                                   int64_t block_size, const int32_t* block_tables,
                                   int64_t max_blocks, const int32_t* q_start,
                                   const int32_t* prefix_lens, int64_t num_seqs,
                                   int64_t max_q_len, int64_t max_total_len, float* out,
                                   void* workspace, int64_t workspace_bytes, int32_t* flags,
                                   void* stream) {
  KSH_CHECK_ARG(hq > 0 && hkv > 0 && hq % hkv == 0 && d > 0 && num_blocks > 0 && num_blocks <= INT32_MAX &&
                num_layers > 0 && layer >= 0 && layer < num_layers && block_size > 0 && block_size <= INT32_MAX &&
                max_blocks > 0 && max_blocks <= INT32_MAX && num_seqs >= 0 && num_seqs <= INT32_MAX && total >= 0 &&
                total <= INT32_MAX && max_q_len >= 0 && max_q_len <= INT32_MAX && max_total_len >= 0);
  KSH_CHECK_ARG(pool_type == KSH_TYPE_F16 || pool_type == KSH_TYPE_BF16);
  if (num_seqs == 0 || total == 0 || max_q_len == 0) return KSH_OK;
  KSH_CHECK_ARG(q && pool && block_tables && q_start && prefix_lens && out);
  if (d > 256 || hq > 65535 || num_seqs > 65535) return KSH_ERR_UNSUPPORTED;
  CacheArgs a = {};
  a.q = q;
  a.pool = pool;
  a.block_tables = block_tables;
  a.q_start = q_start;
  a.prefix = prefix_lens;
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
  a.g = static_cast<int>(hq / hkv);
  a.d = static_cast<int>(d);
  a.max_q = static_cast<int>(max_q_len);
  a.scale = static_cast<float>(1.0 / sqrt(static_cast<double>(d)));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(max_q_len), static_cast<unsigned>(hq), static_cast<unsigned>(num_seqs));
  return pool_type == KSH_TYPE_F16 ? launch(cache_attn_simple_kernel<__half>, grid, dim3(32), 0, st, a)
                                   : launch(cache_attn_simple_kernel<__nv_bfloat16>, grid, dim3(32), 0, st, a);
}
