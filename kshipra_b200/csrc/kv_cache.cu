// The paged K/V cache in 16 bits (fp16 or bf16; fp32 too where a type is
// named): the pass that writes it and the operations on its pages.  The
// attention that reads it stands in cache_attention.cu.

#include <cuda_bf16.h>

#include <algorithm>

#include "tc_common.cuh"

namespace ksh {
namespace {

using namespace tc;

// ---------------------------------------------------------------------------
// Norms of q and k per head, position rotation, K/V into the pool
// ---------------------------------------------------------------------------
//   y = w * (x / sqrt(mean(x^2) + eps))      (q and k, where a norm is given)
//   out[j]       = y[j] cos_j - y[j + d/2] sin_j
//   out[j + d/2] = y[j + d/2] cos_j + y[j] sin_j
// Products and the sum are rounded one by one (the bits of ksh_rope_kv_write
// where the pool is fp32 and no norm is given), K and V then once to the pool's
// type, to nearest; a value past the type's range becomes infinite, as torch's
// conversion does.

struct WriteArgs {
  const float* qkv;               // [m, (hq + 2 hkv) d]
  const int64_t* positions;
  const int64_t* slots;
  const float *rcos, *rsin;       // [max_pos, d / 2]
  const float *q_norm, *k_norm;   // [d] or NULL
  float* q_out;                   // [m, hq, d]
  void* pool;
  int32_t* flags;
  int64_t m, max_pos, num_blocks, num_layers, layer, bs;
  int hq, hkv, d;
  float eps;
};

__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__half* p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void put4(float* p, float4 x) { *reinterpret_cast<float4*>(p) = x; }
__device__ __forceinline__ void put4(__half* p, float4 x) {
  __half2 h[2] = {__floats2half2_rn(x.x, x.y), __floats2half2_rn(x.z, x.w)};
  *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(h);
}
__device__ __forceinline__ void put4(__nv_bfloat16* p, float4 x) {
  __nv_bfloat162 h[2] = {__floats2bfloat162_rn(x.x, x.y), __floats2bfloat162_rn(x.z, x.w)};
  *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(h);
}

// Element offset of a slot's K row of head 0 (V: hkv * bs * d further, a head
// bs * d); negative for a slot outside the pool.
__device__ __forceinline__ int64_t slot_offset(const WriteArgs& a, int64_t slot) {
  if (slot < 0) return -1;
  const int64_t blk = static_cast<uint64_t>(slot) >> 32 ? slot / a.bs
                                                        : static_cast<uint32_t>(slot) / static_cast<uint32_t>(a.bs);
  if (blk >= a.num_blocks) return -1;
  return (((blk * a.num_layers + a.layer) * 2) * a.hkv * a.bs + (slot - blk * a.bs)) * a.d;
}

constexpr int kWriteThreads = 128;

// D / 8 threads for each head of a token, four of the first half's elements
// and the four that they rotate with each; a norm's sum by shuffles among them.
// 2048 rows, 32 / 8 heads of 128, bf16, norms (93 MB, 14.5 us of HBM): 21.5 us with other
// inputs in each call, 18.5 replayed over eight sets of them, 16.5 over one that stays in
// L2, so HBM is not what bounds it: a thread makes three trips to memory one after the
// other, for its elements, for the position and its angles, for the slot.  With 256 threads a
// CTA 23.4, 512 28; two or four heads a thread, which share the angles' loads, 21 (at 256
// threads 23 and 26); stores past L2 would save 1 us here and cost the attention, which
// reads q next.
template <int D, typename T>
__global__ void __launch_bounds__(kWriteThreads) rope_write_kernel(WriteArgs a) {
  constexpr int TPH = D / 8, HALF = D / 2;
  const int heads = a.hq + 2 * a.hkv;
  const int64_t unit = (static_cast<int64_t>(blockIdx.x) * kWriteThreads + threadIdx.x) / TPH;
  const int j = static_cast<int>(threadIdx.x % TPH) * 4;
  const bool on = unit < a.m * heads;
  const int64_t t = on ? ((unit >> 32) ? unit / heads : static_cast<uint32_t>(unit) / static_cast<uint32_t>(heads)) : 0;
  const int h = on ? static_cast<int>(unit - t * heads) : 0;
  const bool rot = h < a.hq + a.hkv;
  const float* nw = h < a.hq ? a.q_norm : rot ? a.k_norm : nullptr;
  grid_dep_wait();
  grid_dep_launch();
  float4 w1, w2;
  if (nw) {
    w1 = *reinterpret_cast<const float4*>(nw + j);
    w2 = *reinterpret_cast<const float4*>(nw + HALF + j);
  }
  float4 x1 = make_float4(0.f, 0.f, 0.f, 0.f), x2 = x1;
  if (on) {
    const float* src = a.qkv + (t * heads + h) * D + j;
    x1 = __ldcs(reinterpret_cast<const float4*>(src));          // read once
    x2 = __ldcs(reinterpret_cast<const float4*>(src + HALF));
  }
  if (a.q_norm || a.k_norm) {      // the same for every thread
    float ss = x1.x * x1.x;
    ss = fmaf(x1.y, x1.y, ss), ss = fmaf(x1.z, x1.z, ss), ss = fmaf(x1.w, x1.w, ss);
    ss = fmaf(x2.x, x2.x, ss), ss = fmaf(x2.y, x2.y, ss), ss = fmaf(x2.z, x2.z, ss), ss = fmaf(x2.w, x2.w, ss);
#pragma unroll
    for (int o = TPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (nw) {
      const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, static_cast<float>(D)), a.eps)));
      x1 = make_float4(__fmul_rn(w1.x, __fmul_rn(x1.x, inv)), __fmul_rn(w1.y, __fmul_rn(x1.y, inv)),
                       __fmul_rn(w1.z, __fmul_rn(x1.z, inv)), __fmul_rn(w1.w, __fmul_rn(x1.w, inv)));
      x2 = make_float4(__fmul_rn(w2.x, __fmul_rn(x2.x, inv)), __fmul_rn(w2.y, __fmul_rn(x2.y, inv)),
                       __fmul_rn(w2.z, __fmul_rn(x2.z, inv)), __fmul_rn(w2.w, __fmul_rn(x2.w, inv)));
    }
  }
  if (!on) return;
  if (rot) {
    int64_t pos = a.positions[t];
    if (pos < 0 || pos >= a.max_pos) {
      if (h == 0 && j == 0) raise_flag(a.flags, KSH_FLAG_BAD_POSITION);
      pos = 0;
    }
    const float4 c = *reinterpret_cast<const float4*>(a.rcos + pos * HALF + j);
    const float4 s = *reinterpret_cast<const float4*>(a.rsin + pos * HALF + j);
    const float4 y1 = x1, y2 = x2;
    auto lo = [](float p, float q, float cc, float sn) { return __fadd_rn(__fmul_rn(p, cc), __fmul_rn(-q, sn)); };
    auto hi = [](float p, float q, float cc, float sn) { return __fadd_rn(__fmul_rn(q, cc), __fmul_rn(p, sn)); };
    x1 = make_float4(lo(y1.x, y2.x, c.x, s.x), lo(y1.y, y2.y, c.y, s.y), lo(y1.z, y2.z, c.z, s.z), lo(y1.w, y2.w, c.w, s.w));
    x2 = make_float4(hi(y1.x, y2.x, c.x, s.x), hi(y1.y, y2.y, c.y, s.y), hi(y1.z, y2.z, c.z, s.z), hi(y1.w, y2.w, c.w, s.w));
  }
  if (h < a.hq) {
    float* dst = a.q_out + (t * a.hq + h) * D + j;
    put4(dst, x1);
    put4(dst + HALF, x2);
    return;
  }
  const int64_t at = slot_offset(a, a.slots[t]);
  if (at < 0) {
    if (h == a.hq && j == 0) raise_flag(a.flags, KSH_FLAG_BAD_SLOT);
    return;
  }
  T* dst = static_cast<T*>(a.pool) + at + static_cast<int64_t>(h - a.hq) * a.bs * D + j;   // V heads follow K's
  put4(dst, x1);
  put4(dst + HALF, x2);
}

// Any even head dimension and alignment: a warp per head.
template <typename T>
__global__ void __launch_bounds__(kWriteThreads) rope_write_any_kernel(WriteArgs a) {
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x & 31, heads = a.hq + 2 * a.hkv, d = a.d, half = d / 2;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * (kWriteThreads / 32) + (threadIdx.x >> 5);
  if (unit >= a.m * heads) return;
  const int64_t t = unit / heads;
  const int h = static_cast<int>(unit - t * heads);
  const bool rot = h < a.hq + a.hkv;
  const float* x = a.qkv + unit * d;
  const float* nw = h < a.hq ? a.q_norm : rot ? a.k_norm : nullptr;
  float inv = 1.0f;
  if (nw) {
    float ss = 0.0f;
    for (int j = lane; j < d; j += 32) ss = fmaf(x[j], x[j], ss);
    ss = warp_sum(ss);
    inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, static_cast<float>(d)), a.eps)));
  }
  int64_t pos = 0, at = 0;
  if (rot) {
    pos = a.positions[t];
    if (pos < 0 || pos >= a.max_pos) {
      if (h == 0 && lane == 0) raise_flag(a.flags, KSH_FLAG_BAD_POSITION);
      pos = 0;
    }
  }
  if (h >= a.hq) {
    at = slot_offset(a, a.slots[t]);
    if (at < 0) {
      if (h == a.hq && lane == 0) raise_flag(a.flags, KSH_FLAG_BAD_SLOT);
      return;
    }
    at += static_cast<int64_t>(h - a.hq) * a.bs * d;
  }
  for (int j = lane; j < half; j += 32) {
    float x1 = x[j], x2 = x[j + half];
    if (nw) {
      x1 = __fmul_rn(nw[j], __fmul_rn(x1, inv));
      x2 = __fmul_rn(nw[j + half], __fmul_rn(x2, inv));
    }
    float y1 = x1, y2 = x2;
    if (rot) {
      const float c = a.rcos[pos * half + j], s = a.rsin[pos * half + j];
      y1 = __fadd_rn(__fmul_rn(x1, c), __fmul_rn(-x2, s));
      y2 = __fadd_rn(__fmul_rn(x2, c), __fmul_rn(x1, s));
    }
    if (h < a.hq) {
      float* dst = a.q_out + (t * a.hq + h) * d;
      dst[j] = y1;
      dst[j + half] = y2;
    } else {
      T* dst = static_cast<T*>(a.pool) + at;
      put(dst + j, y1);
      put(dst + j + half, y2);
    }
  }
}

template <typename T>
int launch_write(const WriteArgs& a, cudaStream_t st) {
  const int64_t units = a.m * (a.hq + 2 * a.hkv);
  uintptr_t al = reinterpret_cast<uintptr_t>(a.qkv) | reinterpret_cast<uintptr_t>(a.rcos) |
                 reinterpret_cast<uintptr_t>(a.rsin) | reinterpret_cast<uintptr_t>(a.q_out) |
                 reinterpret_cast<uintptr_t>(a.q_norm) | reinterpret_cast<uintptr_t>(a.k_norm) |
                 reinterpret_cast<uintptr_t>(a.pool);
  auto grid = [&](int64_t threads) { return (units * threads + kWriteThreads - 1) / kWriteThreads; };
  if (grid(32) > INT32_MAX) return KSH_ERR_UNSUPPORTED;
  if ((al & 15) == 0) {
    if (a.d == 64) return launch(rope_write_kernel<64, T>, dim3(static_cast<unsigned>(grid(8))), dim3(kWriteThreads), 0, st, a);
    if (a.d == 128) return launch(rope_write_kernel<128, T>, dim3(static_cast<unsigned>(grid(16))), dim3(kWriteThreads), 0, st, a);
  }
  return launch(rope_write_any_kernel<T>, dim3(static_cast<unsigned>(grid(32))), dim3(kWriteThreads), 0, st, a);
}

// ---------------------------------------------------------------------------
// Pages: fork and compact
// ---------------------------------------------------------------------------
// Tables and counts are a few hundred kilobytes at most and every step needs
// the one before it, so one cluster of eight CTAs makes them, its barrier
// between the steps; the pages are then copied by a launch over all SMs that
// reads what to copy from the scratch.

constexpr int kPageThreads = 512, kPageCtas = 8;
constexpr int kPageWarps = kPageThreads / 32 * kPageCtas;

struct ForkArgs {
  const int32_t *tables, *lens, *parents, *ref;   // [S, M], [S], [N], [nb]
  int32_t *new_tables, *new_lens, *new_ref;       // [N, M], [N], [nb]
  int64_t* slots;                                 // [N]
  int32_t* scratch;                               // first [S], then src, dst, rest [N] each
  int32_t* flags;
  int64_t max_blocks, bs;
  int num_seqs, n, num_blocks;
};

// Exclusive sum over the cluster of one count per warp, in warp order (rank,
// warp), and the total; cnt_s [kPageWarps] lies in every CTA.
__device__ __forceinline__ int cluster_scan(int count, int* cnt_s, int gw, int lane, int* total) {
  if (lane < kPageCtas) {
    const uint32_t at = map_rank(smem_u32(cnt_s + gw), lane);
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(count) : "memory");
  }
  cluster_sync();
  int before = 0, all = 0;
  for (int i = lane; i < kPageWarps; i += 32) {
    const int c = cnt_s[i];
    all += c;
    if (i < gw) before += c;
  }
  *total = static_cast<int>(__reduce_add_sync(0xffffffffu, all));
  return static_cast<int>(__reduce_add_sync(0xffffffffu, before));
}

// Children i = 0 .. n - 1 continue sequences parents[i].  A child's pages
// before the one that its next token goes to are its parent's; that one is the
// parent's for the first of the children that would write into it, where no other
// row holds it, and a fresh one (with the filled rows copied) for the others and
// where a page begins.
__global__ void __cluster_dims__(kPageCtas, 1, 1) __launch_bounds__(kPageThreads) fork_kernel(ForkArgs a) {
  __shared__ int cnt_s[2][kPageWarps];
  const int tid = threadIdx.x, lane = tid & 31;
  const int rank = static_cast<int>(cluster_rank());
  const int gt = rank * kPageThreads + tid, gw = gt >> 5;
  constexpr int kAll = kPageThreads * kPageCtas;
  grid_dep_wait();
  grid_dep_launch();
  int32_t* const first = a.scratch;
  int32_t* const src = first + a.num_seqs;
  int32_t* const dst = src + a.n;
  int32_t* const rest = dst + a.n;
  const int M = static_cast<int>(a.max_blocks), bs = static_cast<int>(a.bs);
  const int64_t cap = static_cast<int64_t>(M) * bs;
  auto length = [&](int s) {
    const int ln = a.lens[s];
    if (ln < 0 || ln > cap) raise_flag(a.flags, KSH_FLAG_BAD_LENGTH);
    return static_cast<int>(min(static_cast<int64_t>(max(ln, 0)), cap));
  };
  auto parent = [&](int i) {
    const int p = a.parents[i];
    if (p >= a.num_seqs) raise_flag(a.flags, KSH_FLAG_BAD_PARENT);
    return p >= a.num_seqs ? -1 : p;
  };
  for (int i = gt; i < a.num_blocks; i += kAll) a.new_ref[i] = a.ref[i];
  for (int i = gt; i < a.num_seqs; i += kAll) first[i] = INT32_MAX;
  cluster_sync();
  // what the old sequences hold goes, what the children share comes; a warp a row
  for (int s = gw; s < a.num_seqs; s += kPageWarps) {
    const int held = (length(s) + bs - 1) / bs;
    for (int j = lane; j < held; j += 32) {
      const int page = a.tables[static_cast<int64_t>(s) * M + j];
      const bool ok = page >= 0 && page < a.num_blocks;
      if (ok) atomicSub(a.new_ref + page, 1);
      if (!ok || a.ref[page] <= 0) raise_flag(a.flags, KSH_FLAG_BAD_BLOCK);
    }
  }
  for (int i = gw; i < a.n; i += kPageWarps) {
    const int p = parent(i);
    const int ln = p < 0 ? 0 : length(p), full = ln / bs;
    for (int j = lane; j < M; j += 32) {
      int page = 0;
      if (j < full) {
        page = a.tables[static_cast<int64_t>(p) * M + j];
        if (page >= 0 && page < a.num_blocks) atomicAdd(a.new_ref + page, 1);
      }
      a.new_tables[static_cast<int64_t>(i) * M + j] = page;
    }
    if (lane == 0) {
      a.new_lens[i] = ln;
      if (p >= 0) atomicMin(first + p, i);
      const int r = ln - full * bs;
      if (p >= 0 && full >= M) raise_flag(a.flags, KSH_FLAG_BAD_LENGTH);
      rest[i] = p < 0 || full >= M ? -1 : r;           // filled rows of the page that the next token goes to
      dst[i] = p >= 0 && full < M && r > 0 ? a.tables[static_cast<int64_t>(p) * M + full] : -1;
    }
  }
  cluster_sync();
  // A warp has a run of children.  A page that is being filled and that nobody holds
  // now goes to the first child whose parent held it: the least of i - n stands in for
  // its count until the child takes it.
  const int per = (a.n + kPageWarps - 1) / kPageWarps;
  for (int i = gw * per + lane; i < min(a.n, (gw + 1) * per); i += 32) {
    const int p = a.parents[i], page = __ldcg(dst + i);
    const bool mine = __ldcg(rest + i) > 0 && __ldcg(first + p) == i, there = page >= 0 && page < a.num_blocks;
    if (mine && there && __ldcg(a.new_ref + page) <= 0) atomicMin(a.new_ref + page, i - a.n);
    src[i] = mine;
  }
  cluster_sync();
  // the page that the next token goes to: kept, or fresh; fresh ones are numbered in
  // the children's order.
  int count = 0;
  for (int i = gw * per + lane; i - lane < min(a.n, (gw + 1) * per); i += 32) {
    bool fresh = false;
    if (i < min(a.n, (gw + 1) * per)) {
      int state = __ldcg(rest + i);                    // -1: no page wanted, -2: settled
      if (state < 0) {
        a.slots[i] = -1;
      } else {
        const int page = __ldcg(dst + i);
        const bool mine = __ldcg(src + i) != 0, there = page >= 0 && page < a.num_blocks;
        const bool keep = mine && there && __ldcg(a.new_ref + page) == i - a.n;
        fresh = !(mine && !there) && !keep;
        if (fresh) {
          a.slots[i] = there ? page : -1;              // what is copied, for now
        } else {
          a.new_tables[static_cast<int64_t>(i) * M + __ldcg(a.new_lens + i) / bs] = page;
          if (keep) a.new_ref[page] = 1;
          a.slots[i] = keep ? static_cast<int64_t>(page) * bs + state : -1;
          rest[i] = keep ? -2 : -1;
        }
      }
    }
    count += __popc(__ballot_sync(0xffffffffu, fresh));
  }
  int wanted, rank_of = cluster_scan(count, cnt_s[0], gw, lane, &wanted);     // its barrier: the counts are complete
  // the lowest free pages, as many as are wanted: a warp has a run of pages
  const int ppw = ((a.num_blocks + kPageWarps - 1) / kPageWarps + 31) / 32 * 32;
  const int p0 = min(a.num_blocks, gw * ppw), p1 = min(a.num_blocks, p0 + ppw);
  int free_here = 0;
  for (int i = p0 + lane; i - lane < p1; i += 32) {
    const int c = i < p1 ? __ldcg(a.new_ref + i) : 1;
    if (c < 0) raise_flag(a.flags, KSH_FLAG_BAD_BLOCK);        // held more often than counted
    free_here += __popc(__ballot_sync(0xffffffffu, c == 0));
  }
  int have, at = cluster_scan(free_here, cnt_s[1], gw, lane, &have);
  for (int i = p0 + lane; i - lane < p1 && at < wanted; i += 32) {
    const bool f = i < p1 && __ldcg(a.new_ref + i) == 0;
    const uint32_t who = __ballot_sync(0xffffffffu, f);
    const int k = at + __popc(who & ((1u << lane) - 1));
    if (f && k < wanted) {
      src[k] = i;                                      // fresh page k, for now
      a.new_ref[i] = 1;
    }
    at += __popc(who);
  }
  cluster_sync();
  for (int i = gw * per + lane; i - lane < min(a.n, (gw + 1) * per); i += 32) {
    const bool here = i < min(a.n, (gw + 1) * per), fresh = here && __ldcg(rest + i) >= 0;
    const uint32_t who = __ballot_sync(0xffffffffu, fresh);
    const int k = rank_of + __popc(who & ((1u << lane) - 1));
    if (here) dst[i] = fresh && k < have ? __ldcg(src + k) : -1;
    rank_of += __popc(who);
  }
  cluster_sync();
  for (int i = gw * per + lane; i < min(a.n, (gw + 1) * per); i += 32) {
    const int r = __ldcg(rest + i), page = __ldcg(dst + i), from = static_cast<int>(__ldcg(a.slots + i));
    src[i] = r >= 0 && page >= 0 ? from : -1;
    if (r < 0) continue;
    if (page < 0) {
      raise_flag(a.flags, KSH_FLAG_NO_PAGE);
      a.slots[i] = -1;
      continue;
    }
    a.new_tables[static_cast<int64_t>(i) * M + __ldcg(a.new_lens + i) / bs] = page;
    a.slots[i] = static_cast<int64_t>(page) * bs + r;
  }
}

// The filled rows of each copied page: a warp takes a (child, layer, K or V,
// head) with `rest` rows of `row` units of U, which stand one after the other.
template <typename U>
__global__ void __launch_bounds__(256) fork_copy_kernel(const int32_t* scratch, int num_seqs, int n, int segs, int64_t seg_units,
                                                        int row_units, U* pool) {
  grid_dep_wait();
  grid_dep_launch();
  const int i = blockIdx.y, lane = threadIdx.x & 31;
  const int32_t* src = scratch + num_seqs;
  const int from = src[i];
  if (from < 0) return;
  const int to = src[n + i], units = src[2 * n + i] * row_units;
  for (int s = blockIdx.x * 8 + (threadIdx.x >> 5); s < segs; s += gridDim.x * 8) {
    const U* x = pool + (static_cast<int64_t>(from) * segs + s) * seg_units;
    U* y = pool + (static_cast<int64_t>(to) * segs + s) * seg_units;
    int k = lane;
    for (; k + 96 < units; k += 128) {
      const U v0 = x[k], v1 = x[k + 32], v2 = x[k + 64], v3 = x[k + 96];
      y[k] = v0, y[k + 32] = v1, y[k + 64] = v2, y[k + 96] = v3;
    }
    for (; k < units; k += 32) y[k] = x[k];
  }
}

struct CompactArgs {
  const int32_t *tables, *ref;                    // [entries], [nb]
  int32_t *new_tables, *new_ref, *map, *used;     // [entries], [nb], [nb], [1]
  int32_t* scratch;                               // moves, then src [nb / 2], dst [nb / 2]
  int64_t entries;
  int num_blocks;
};

// u pages are in use: the k-th used page from u on goes to the k-th free page
// below u, so no move writes what another reads.
__global__ void __cluster_dims__(kPageCtas, 1, 1) __launch_bounds__(kPageThreads) compact_kernel(CompactArgs a) {
  __shared__ int cnt_s[2][kPageWarps];
  const int tid = threadIdx.x, lane = tid & 31;
  const int gt = static_cast<int>(cluster_rank()) * kPageThreads + tid, gw = gt >> 5;
  constexpr int kAll = kPageThreads * kPageCtas;
  grid_dep_wait();
  grid_dep_launch();
  cluster_sync();                                                     // every CTA runs: the scans write into all of them
  const int nb = a.num_blocks;
  const int ppw = ((nb + kPageWarps - 1) / kPageWarps + 31) / 32 * 32;
  const int p0 = min(nb, gw * ppw), p1 = min(nb, p0 + ppw);
  int count = 0, u;
  for (int i = p0 + lane; i - lane < p1; i += 32) count += __popc(__ballot_sync(0xffffffffu, i < p1 && a.ref[i] > 0));
  const int below = cluster_scan(count, cnt_s[0], gw, lane, &u);      // used pages before the run
  int32_t* const src = a.scratch + 1;
  int32_t* const dst = src + nb / 2;
  if (gt == 0) *a.used = u;
  // used pages below u: u - (moves); the moves are numbered from both lists alike
  int holes = 0, moves;
  for (int i = p0 + lane; i - lane < p1; i += 32) holes += __popc(__ballot_sync(0xffffffffu, i < p1 && i < u && a.ref[i] <= 0));
  int hole = cluster_scan(holes, cnt_s[1], gw, lane, &moves);
  if (gt == 0) *a.scratch = moves;
  int mover = p0 < u ? 0 : below - (u - moves);                       // used pages from u up to the run
  for (int i = p0 + lane; i - lane < p1; i += 32) {
    const int r = i < p1 ? a.ref[i] : 0;
    const bool h = i < p1 && i < u && r <= 0, m = i < p1 && i >= u && r > 0;
    const uint32_t hs = __ballot_sync(0xffffffffu, h), ms = __ballot_sync(0xffffffffu, m), low = (1u << lane) - 1;
    if (h) dst[hole + __popc(hs & low)] = i;
    if (m) src[mover + __popc(ms & low)] = i;
    hole += __popc(hs);
    mover += __popc(ms);
    if (i < p1) {
      a.map[i] = i;
      a.new_ref[i] = m || r < 0 ? 0 : r;
    }
  }
  cluster_sync();
  for (int k = gt; k < moves; k += kAll) {
    const int from = __ldcg(src + k), to = __ldcg(dst + k);
    a.map[from] = to;
    a.new_ref[to] = a.ref[from];
  }
  cluster_sync();
  for (int64_t i = gt; i < a.entries; i += kAll) {
    const int page = a.tables[i];
    a.new_tables[i] = page >= 0 && page < nb ? __ldcg(a.map + page) : page;
  }
}

// Whole pages in pieces of 256 x kMoveUnroll units.  HBM bound: 100 pages of 2 MB (400
// MB moved) in 68 us with the tables, 95 % of measured HBM.  Many small CTAs in turn
// rather than eight resident ones an SM with larger pieces (81): a CTA that waits for
// its loads leaves its place to another.
constexpr int kMoveUnroll = 2;

template <typename U>
__global__ void __launch_bounds__(256) compact_move_kernel(const int32_t* scratch, int half, int64_t page_units, int pieces, U* pool) {
  grid_dep_wait();
  grid_dep_launch();
  const int64_t total = static_cast<int64_t>(*scratch) * pieces;
  constexpr int64_t piece = 256 * kMoveUnroll;
  for (int64_t w = blockIdx.x; w < total; w += gridDim.x) {
    const int64_t k = w / pieces, at = (w - k * pieces) * piece + threadIdx.x;
    const U* x = pool + scratch[1 + k] * page_units;
    U* y = pool + scratch[1 + half + k] * page_units;
    U v[kMoveUnroll];
#pragma unroll
    for (int i = 0; i < kMoveUnroll; ++i)
      if (at + 256 * i < page_units) v[i] = x[at + 256 * i];
#pragma unroll
    for (int i = 0; i < kMoveUnroll; ++i)
      if (at + 256 * i < page_units) y[at + 256 * i] = v[i];
  }
}

// Largest unit (16, 8, 4, 2 bytes) that divides both.
int unit_bytes(const void* p, int64_t bytes) {
  const uint64_t all = reinterpret_cast<uintptr_t>(p) | static_cast<uint64_t>(bytes);
  return (all & 15) == 0 ? 16 : (all & 7) == 0 ? 8 : (all & 3) == 0 ? 4 : 2;
}

int type_bytes(int type) { return type == KSH_TYPE_F32 ? 4 : type == KSH_TYPE_F16 || type == KSH_TYPE_BF16 ? 2 : 0; }

}  // namespace
}  // namespace ksh

using namespace ksh;

extern "C" int ksh_rope_cache_write(const float* qkv, int64_t m, int64_t hq, int64_t hkv, int64_t d,
                                    const int64_t* positions, const int64_t* slot_mapping,
                                    const float* rope_cos, const float* rope_sin, int64_t max_pos,
                                    const float* q_norm, const float* k_norm, float eps,
                                    float* q_out, void* pool, int pool_type, int64_t num_blocks,
                                    int64_t num_layers, int64_t layer, int64_t block_size,
                                    int32_t* flags, void* stream) {
  KSH_CHECK_ARG(m >= 0 && m <= INT32_MAX && hq > 0 && hkv > 0 && hq <= 65535 && hkv <= 65535 && d > 0 && d % 2 == 0 &&
                d <= 65536 && max_pos > 0 && num_blocks > 0 && num_layers > 0 && layer >= 0 && layer < num_layers &&
                block_size > 0 && block_size <= INT32_MAX);
  KSH_CHECK_ARG(type_bytes(pool_type) != 0);
  if (m == 0) return KSH_OK;
  KSH_CHECK_ARG(qkv && positions && slot_mapping && rope_cos && rope_sin && q_out && pool);
  WriteArgs a = {};
  a.qkv = qkv;
  a.positions = positions;
  a.slots = slot_mapping;
  a.rcos = rope_cos;
  a.rsin = rope_sin;
  a.q_norm = q_norm;
  a.k_norm = k_norm;
  a.q_out = q_out;
  a.pool = pool;
  a.flags = flags;
  a.m = m;
  a.max_pos = max_pos;
  a.num_blocks = num_blocks;
  a.num_layers = num_layers;
  a.layer = layer;
  a.bs = block_size;
  a.hq = static_cast<int>(hq);
  a.hkv = static_cast<int>(hkv);
  a.d = static_cast<int>(d);
  a.eps = eps;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return pool_type == KSH_TYPE_F32 ? launch_write<float>(a, st)
         : pool_type == KSH_TYPE_F16 ? launch_write<__half>(a, st)
                                     : launch_write<__nv_bfloat16>(a, st);
}

extern "C" int64_t ksh_fork_pages_scratch_ints(int64_t num_seqs, int64_t n) {
  return num_seqs < 0 || n < 0 ? 0 : num_seqs + 3 * n + 1;
}

extern "C" int ksh_fork_pages(void* pool, int pool_type, int64_t num_blocks, int64_t num_layers,
                              int64_t hkv, int64_t block_size, int64_t d, const int32_t* block_tables,
                              int64_t max_blocks, const int32_t* lens, int64_t num_seqs,
                              const int32_t* parents, int64_t n, const int32_t* ref_counts,
                              int32_t* new_tables, int32_t* new_lens, int64_t* slots,
                              int32_t* new_ref, int32_t* scratch, int64_t scratch_ints,
                              int32_t* flags, void* stream) {
  const int eb = type_bytes(pool_type);
  KSH_CHECK_ARG(eb != 0 && num_blocks > 0 && num_blocks <= INT32_MAX / 2 && num_layers > 0 && hkv > 0 && block_size > 0 &&
                block_size <= INT32_MAX && d > 0 && max_blocks > 0 && max_blocks <= INT32_MAX / 64 && num_seqs >= 0 &&
                num_seqs <= INT32_MAX / 8 && n >= 0);
  KSH_CHECK_ARG(pool && ref_counts && new_ref && (num_seqs == 0 || (block_tables && lens)));
  KSH_CHECK_ARG(n == 0 || (parents && new_tables && new_lens && slots));
  if (n > 65535) return KSH_ERR_UNSUPPORTED;
  if (!scratch || scratch_ints < ksh_fork_pages_scratch_ints(num_seqs, n)) return KSH_ERR_WORKSPACE;
  const int64_t segs = num_layers * 2 * hkv;
  if (segs > INT32_MAX / 8 || block_size * d * eb > INT32_MAX) return KSH_ERR_UNSUPPORTED;
  ForkArgs a = {};
  a.tables = block_tables;
  a.lens = lens;
  a.parents = parents;
  a.ref = ref_counts;
  a.new_tables = new_tables;
  a.new_lens = new_lens;
  a.new_ref = new_ref;
  a.slots = slots;
  a.scratch = scratch;
  a.flags = flags;
  a.max_blocks = max_blocks;
  a.bs = block_size;
  a.num_seqs = static_cast<int>(num_seqs);
  a.n = static_cast<int>(n);
  a.num_blocks = static_cast<int>(num_blocks);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int rc = launch(fork_kernel, dim3(kPageCtas), dim3(kPageThreads), 0, st, a);
  if (rc != KSH_OK || n == 0) return rc;
  const int ub = unit_bytes(pool, d * eb);
  const dim3 grid(static_cast<unsigned>((segs + 7) / 8), static_cast<unsigned>(n));
  auto copy = [&](auto* p) {
    using U = std::remove_pointer_t<decltype(p)>;
    return launch(fork_copy_kernel<U>, grid, dim3(256), 0, st, scratch, a.num_seqs, a.n, static_cast<int>(segs),
                  block_size * d * eb / ub, static_cast<int>(d * eb / ub), p);
  };
  return ub == 16 ? copy(static_cast<uint4*>(pool)) : ub == 8 ? copy(static_cast<uint2*>(pool))
         : ub == 4 ? copy(static_cast<uint32_t*>(pool)) : copy(static_cast<uint16_t*>(pool));
}

extern "C" int64_t ksh_compact_pages_scratch_ints(int64_t num_blocks) { return num_blocks < 0 ? 0 : num_blocks + 2; }

extern "C" int ksh_compact_pages(void* pool, int pool_type, int64_t num_blocks, int64_t num_layers,
                                 int64_t hkv, int64_t block_size, int64_t d,
                                 const int32_t* block_tables, int64_t entries,
                                 const int32_t* ref_counts, int32_t* new_tables, int32_t* new_ref,
                                 int32_t* page_map, int32_t* used, int32_t* scratch,
                                 int64_t scratch_ints, void* stream) {
  const int eb = type_bytes(pool_type);
  KSH_CHECK_ARG(eb != 0 && num_blocks > 0 && num_blocks <= INT32_MAX / 2 && num_layers > 0 && hkv > 0 && block_size > 0 &&
                d > 0 && entries >= 0);
  KSH_CHECK_ARG(pool && ref_counts && new_ref && page_map && used && (entries == 0 || (block_tables && new_tables)));
  if (!scratch || scratch_ints < ksh_compact_pages_scratch_ints(num_blocks)) return KSH_ERR_WORKSPACE;
  CompactArgs a = {};
  a.tables = block_tables;
  a.ref = ref_counts;
  a.new_tables = new_tables;
  a.new_ref = new_ref;
  a.map = page_map;
  a.used = used;
  a.scratch = scratch;
  a.entries = entries;
  a.num_blocks = static_cast<int>(num_blocks);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t bytes = num_layers * 2 * hkv * block_size * d * eb;
  const int ub = unit_bytes(pool, bytes);
  const int64_t units = bytes / ub, pieces = (units + 256 * kMoveUnroll - 1) / (256 * kMoveUnroll);
  if (pieces > INT32_MAX) return KSH_ERR_UNSUPPORTED;
  const int rc = launch(compact_kernel, dim3(kPageCtas), dim3(kPageThreads), 0, st, a);
  if (rc != KSH_OK || num_blocks < 2) return rc;
  const int grid = static_cast<int>(std::min<int64_t>(num_blocks / 2 * pieces, 64LL * num_sms()));
  auto move = [&](auto* p) {
    using U = std::remove_pointer_t<decltype(p)>;
    return launch(compact_move_kernel<U>, dim3(static_cast<unsigned>(grid)), dim3(256), 0, st, scratch,
                  static_cast<int>(num_blocks / 2), units, static_cast<int>(pieces), p);
  };
  return ub == 16 ? move(static_cast<uint4*>(pool)) : ub == 8 ? move(static_cast<uint2*>(pool))
         : ub == 4 ? move(static_cast<uint32_t*>(pool)) : move(static_cast<uint16_t*>(pool));
}
