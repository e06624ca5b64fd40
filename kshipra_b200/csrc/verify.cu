// Target probabilities from logits, and verification of drafted tokens.
//
// target_probs: p[r, i] = exp((x[r, i] - max_r) / T_r) / sum, T_r <= 0: one at
// the first maximum.  HBM bound: 8 bytes per element.
//
// verify_tree: nodes of a sequence's tree in node order, node 0 the root.
// With r = P[root], Z = 1, at the current node c the child i (parent(i) = c)
// carrying token t is accepted iff
//     u_i * Z * Q_c(t) < r(t)          (Q := 1 for fixed proposals)
// then c = i, r = P[i], Z = 1; otherwise the mass that the proposal covered is
// taken out of r:
//     r = max(r - Z * Q_c, 0), Z = sum r   (fixed: Z -= r(t), r(t) = 0)
// so that the tokens emitted follow the target's distribution whatever was
// drafted.  At the end the next token is the first t with cumsum(r)[t] >
// u * sum(r).  Sums over the vocabulary are held in 64 bits: the choice is a
// whole number, and a sum that depends on its order in the last bits of 32
// would move it for one sample in a hundred at 128 K tokens.

#include <float.h>
#include <math.h>

#include <algorithm>

#include "tc_common.cuh"

namespace ksh {
namespace {

using namespace tc;

constexpr int kMaxCluster = 8;
// A row's elements are numbered in 32 bits, and loops go one stride past its
// end: rows up to 2^30 leave room for that.
constexpr int64_t kMaxVocab = 1 << 30;

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// 2^x to 2 ulp; the argument's own rounding is the larger part of a term's error
__device__ __forceinline__ float pow2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Scale of (x - max) / t to powers of two.  Finite, so that the maxima of a row
// at a temperature below 2^-127 keep their 0; a temperature of NaN stays NaN.
__device__ __forceinline__ float to_pow2(float t) {
  const float c = 1.44269504088896340736f / t;
  return c > FLT_MAX ? FLT_MAX : c;
}
__device__ __forceinline__ void st_cluster_f64(uint32_t addr, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory");
}
__device__ __forceinline__ void st_cluster_b64(uint32_t addr, uint64_t v) {
  asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
// Every CTA of the cluster runs before another writes into its shared memory:
// joined at the kernel's start, waited for before the first such write.
__device__ __forceinline__ void cluster_join() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_joined() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
// Elements before the first 16-byte boundary of a row.
__device__ __forceinline__ int head_of(const float* row) {
  return static_cast<int>((4 - ((reinterpret_cast<uintptr_t>(row) >> 2) & 3)) & 3);
}

// ---------------------------------------------------------------------------
// One row per cluster: each CTA keeps its part of the row in shared memory,
// so the row is read once and written once; the maximum and the sum cross the
// cluster through distributed shared memory.  512 x 128256: 109 us, 4.8 TB/s,
// 74 % of measured HBM; clusters read, wait for each other and write in waves,
// and three CTAs per SM overlap these.  The part comes by bulk copies (through
// registers, where three CTAs of 384 threads hold two thirds of it in flight:
// 110 us, with half of those 131; CTAs of 416 threads, of which two fit: 149);
// streaming hints on loads and stores cost 2 us; clusters of 16 with parts half
// as large: 115 us.  One CTA per row reading it three times: 23 %.

constexpr int kProbThreads = 384;
constexpr int kProbWarps = kProbThreads / 32;
constexpr int kProbCopy = 1024;            // float4 of one bulk copy
constexpr int kProbSlice = 50 * 1024;      // floats of a part, at most

struct ProbArgs {
  const float* x;
  const float* temperature;
  float* p;
  int64_t x_stride, p_stride;
  int vocab, chunk;             // chunk: floats of a part, a multiple of four
};

// Order-preserving key of (value, first index); -0 == +0; NaN above +inf, as in
// torch.argmax and the tensor-core lm_head.
__device__ __forceinline__ uint64_t top_key(float v, int i) {
  const uint32_t u = __float_as_uint(v + 0.0f);
  const uint32_t k = v == v ? ((u & 0x80000000u) ? ~u : u | 0x80000000u) : 0xffffffffu;
  return (static_cast<uint64_t>(k) << 32) | (0xffffffffu - static_cast<uint32_t>(i));
}

__global__ void __launch_bounds__(kProbThreads) target_probs_kernel(ProbArgs a) {
  extern __shared__ __align__(16) float slice[];
  __shared__ float redf[kProbWarps];
  __shared__ uint64_t redk[kProbWarps];
  __shared__ float redg[kProbWarps];
  __shared__ uint64_t top_s[kMaxCluster];
  __shared__ __align__(8) uint64_t full;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const int64_t r = blockIdx.x / size;
  if (tid == 0) {
    mbar_init(&full, 1);
    fence_barrier_init();
  }
  __syncthreads();
  cluster_join();
  grid_dep_wait();
  grid_dep_launch();
  const float* xr = a.x + r * a.x_stride;
  float* pr = a.p + r * a.p_stride;
  const float t = a.temperature ? a.temperature[r] : 1.0f;
  // this CTA's elements [lo, hi); loads and stores take four at a time from the
  // row's 16-byte boundary a0 on (element i at slice[i - a0 + 4]), the sum goes
  // by index alone: where a row lies does not change its bits
  const int lo = min(a.vocab, static_cast<int>(rank) * a.chunk), hi = min(a.vocab, lo + a.chunk);
  const int a0 = min(lo + head_of(xr + lo), hi), n4 = (hi - a0) / 4, rest = a0 + 4 * n4;
  float* const s = slice + 4 - a0;
  // all of the part on its way at once
  if (tid < 32) {
    if (tid == 0) mbar_arrive_expect_tx(&full, static_cast<uint32_t>(n4) * 16);
    __syncwarp();
    for (int i = tid * kProbCopy; i < n4; i += 32 * kProbCopy)
      asm volatile(
          "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
              smem_u32(s + a0 + 4 * i)),
          "l"(xr + a0 + 4 * i), "r"(min(kProbCopy, n4 - i) * 16), "r"(smem_u32(&full))
          : "memory");
  }
  float m = -INFINITY;
  {
    const int e = tid < a0 - lo ? lo + tid : (tid >= 4 && tid - 4 < hi - rest ? rest + tid - 4 : -1);
    if (e >= 0) {
      s[e] = xr[e];
      m = s[e];
    }
  }
  const bool came = mbar_wait(&full, 0);
  {
    const float4* s4 = reinterpret_cast<const float4*>(s + a0);
#pragma unroll 4
    for (int i = tid; i < n4; i += kProbThreads) {
      const float4 v = s4[i];
      m = fmaxf(m, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)));
    }
  }
  if (!(t <= 0.0f)) {
    // terms against the part's own maximum; its share of the row's sum and the
    // factor that brings them to the row's maximum follow from one exchange
    m = warp_max(m);
    if (lane == 0) redf[warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kProbWarps; ++w) m = fmaxf(m, redf[w]);
    const float ref = m == -INFINITY ? 0.0f : m;    // a part of nothing but -inf
    const float c = to_pow2(t);
    float sum = 0.0f;
#pragma unroll 8
    for (int i = lo + tid; i < hi; i += kProbThreads) {
      const float v = pow2((s[i] - ref) * c);
      s[i] = v;
      sum += v;
    }
    sum = warp_sum(sum);
    if (lane == 0) redg[warp] = sum;
    __syncthreads();
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kProbWarps; ++w) sum += redg[w];
    cluster_joined();
    if (tid < static_cast<int>(size))
      st_cluster_b64(map_rank(smem_u32(&top_s[rank]), tid),
                     (static_cast<uint64_t>(__float_as_uint(sum)) << 32) | __float_as_uint(m));
    cluster_sync();
    float M = -INFINITY;
    for (uint32_t g = 0; g < size; ++g) M = fmaxf(M, __uint_as_float(static_cast<uint32_t>(top_s[g])));
    sum = 0.0f;
    for (uint32_t g = 0; g < size; ++g) {
      const float mg = __uint_as_float(static_cast<uint32_t>(top_s[g]));
      const float sg = __uint_as_float(static_cast<uint32_t>(top_s[g] >> 32));
      sum += sg * pow2((mg - M) * c);
    }
    // a row of nothing but -inf stays NaN
    float inv = m == -INFINITY && M != -INFINITY ? 0.0f : pow2((m - M) * c) / sum;
    if (!came) inv = NAN;
    if (((reinterpret_cast<uintptr_t>(pr) ^ reinterpret_cast<uintptr_t>(xr)) & 15) == 0) {
      float4* p4 = reinterpret_cast<float4*>(pr + a0);
      const float4* s4 = reinterpret_cast<const float4*>(s + a0);
      const int e = tid < a0 - lo ? lo + tid : (tid >= 4 && tid - 4 < hi - rest ? rest + tid - 4 : -1);
#pragma unroll 4
      for (int i = tid; i < n4; i += kProbThreads) {
        const float4 v = s4[i];
        p4[i] = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
      }
      if (e >= 0) pr[e] = s[e] * inv;
    } else {
      for (int i = lo + tid; i < hi; i += kProbThreads) pr[i] = s[i] * inv;
    }
    return;
  }
  // one at the first maximum
  uint64_t key = 0;
  __syncthreads();
  for (int i = lo + tid; i < hi; i += kProbThreads) key = max(key, top_key(s[i], i));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
  if (lane == 0) redk[warp] = key;
  __syncthreads();
  for (int w = 0; w < kProbWarps; ++w) key = max(key, redk[w]);
  cluster_joined();
  if (tid < static_cast<int>(size)) st_cluster_b64(map_rank(smem_u32(&top_s[rank]), tid), key);
  cluster_sync();
  for (uint32_t c = 0; c < size; ++c) key = max(key, top_s[c]);
  const int at = static_cast<int>(0xffffffffu - static_cast<uint32_t>(key));
  for (int i = lo + tid; i < hi; i += kProbThreads) pr[i] = !came ? NAN : i == at ? 1.0f : 0.0f;
}

// Rows too long for a cluster's shared memory: one CTA each, three readings.
__global__ void __launch_bounds__(kProbThreads) target_probs_long_kernel(ProbArgs a) {
  __shared__ float redf[kProbWarps];
  __shared__ double redd[kProbWarps];
  __shared__ uint64_t redk[kProbWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_dep_wait();
  grid_dep_launch();
  const float* xr = a.x + blockIdx.x * a.x_stride;
  float* pr = a.p + blockIdx.x * a.p_stride;
  const float t = a.temperature ? a.temperature[blockIdx.x] : 1.0f;
  float m = -INFINITY;
  uint64_t key = 0;
  for (int i = tid; i < a.vocab; i += kProbThreads) {
    m = fmaxf(m, xr[i]);
    key = max(key, top_key(xr[i], i));
  }
  m = warp_max(m);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
  if (lane == 0) {
    redf[warp] = m;
    redk[warp] = key;
  }
  __syncthreads();
  for (int w = 0; w < kProbWarps; ++w) {
    m = fmaxf(m, redf[w]);
    key = max(key, redk[w]);
  }
  if (t <= 0.0f) {
    const int at = static_cast<int>(0xffffffffu - static_cast<uint32_t>(key));
    for (int i = tid; i < a.vocab; i += kProbThreads) pr[i] = i == at ? 1.0f : 0.0f;
    return;
  }
  const float c = to_pow2(t);
  // thousands of terms a thread: in 32 bits a flat row's sum was off by 1e-5
  double sum = 0.0;
  for (int i = tid; i < a.vocab; i += kProbThreads) sum += static_cast<double>(pow2((xr[i] - m) * c));
  sum = warp_sum_f64(sum);
  if (lane == 0) redd[warp] = sum;
  __syncthreads();
  sum = 0.0;
  for (int w = 0; w < kProbWarps; ++w) sum += redd[w];
  const float inv = static_cast<float>(1.0 / sum);
  for (int i = tid; i < a.vocab; i += kProbThreads) pr[i] = pow2((xr[i] - m) * c) * inv;
}

// ---------------------------------------------------------------------------

constexpr int kMaxNodes = 256;
constexpr int kVerThreads = 256, kSlots = 32;
constexpr int kVerWarps = kVerThreads / 32;
enum { MODE_GREEDY = 0, MODE_FIXED = 1, MODE_DRAWN = 2 };

struct VerArgs {
  const int64_t* tokens;        // [total]
  const int32_t* parents;       // [total]
  const int32_t* q_start;       // [S + 1]
  const float* target;          // [total, vocab], rows p_stride apart
  const float* draft;           // [total, vocab], rows q_stride apart
  const int64_t* greedy;        // [total]
  const float* u_accept;        // [total]
  const float* u_sample;        // [S]
  int32_t* path;                // [S, max_nodes]
  int32_t* path_len;            // [S]
  int64_t* next;                // [S]
  int32_t* flags;
  int64_t total, p_stride, q_stride;
  int vocab, max_nodes, chunk;  // chunk: elements of a warp's piece of a row
};

// What is left of the target's row at the current node.  Taking Z_1 Q, Z_2 Q, ..
// out one after the other, max(.., 0) each time, is max(P - (Z_1 + Z_2 + ..) Q,
// 0) in one step; of fixed proposals the refused tokens are kept.
struct Rest {
  const float* p;
  const float* q;
  const int* gone;
  double a;                     // sum of the Z
  int k;                        // refusals
};

// A cluster per sequence.  Every CTA walks the tree alike from the drafted
// tokens' entries (all gathered at once); sums over the row are shared by the
// cluster's warps, each with a contiguous piece, and the pieces' sums go to
// every CTA through distributed shared memory.  Only the rows that a sum is
// needed of are read, 512 elements of the last one twice.
// 64 sequences x 128256, drawn proposals, 8 nodes: 25 us back to back against
// 10 us for one reading of each final pair of rows: a refusal's sum needs the one
// before it, and each is a pass of about 4 us over the row (now in L2) and the
// cluster.  One sequence x 151936, fixed proposals: 12 us, latency; the call's
// 15 us are the host's, and so are 16 with 64 sequences x 8 nodes and 13.6 with
// greedy tokens.  At 64 registers (four CTAs per SM) the drawn form spills 224
// bytes a thread, the fixed one 64.
template <int MODE>
__global__ void __launch_bounds__(kVerThreads, 4) verify_tree_kernel(VerArgs a) {
  __shared__ int tok_s[kMaxNodes], par_s[kMaxNodes], path_s[kMaxNodes], gone_s[kMaxNodes];
  __shared__ float u_s[kMaxNodes], p_s[kMaxNodes], q_s[kMaxNodes];
  __shared__ double part_s[2][kMaxCluster * kVerWarps], step_s[kVerWarps][kSlots];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const int s = blockIdx.x / size;
  const bool first = rank == 0;
  grid_dep_wait();
  grid_dep_launch();
  const int64_t a0 = a.q_start[s], a1 = a.q_start[s + 1];
  int n = static_cast<int>(min(a1 - a0, static_cast<int64_t>(a.max_nodes)));
  if (a0 < 0 || a1 > a.total || a1 - a0 > a.max_nodes || a1 < a0) {
    if (first && tid == 0) raise_flag(a.flags, KSH_FLAG_BAD_LENGTH);
    if (a0 < 0 || a1 > a.total) n = 0;
  }
  int32_t* path = a.path + static_cast<int64_t>(s) * a.max_nodes;
  if (n <= 0) {
    if (!first) return;
    for (int i = tid; i < a.max_nodes; i += kVerThreads) path[i] = -1;
    if (tid == 0) {
      a.path_len[s] = 0;
      a.next[s] = -1;
    }
    return;
  }
  if (MODE != MODE_GREEDY) cluster_join();
  bool joined = false;
  for (int i = tid; i < n; i += kVerThreads) {
    const int64_t t = a.tokens[a0 + i];
    const int par = a.parents[a0 + i];
    int up = i > 0 && par >= 0 && par < i ? par : -1;
    if (first && i > 0 && (par < 0 || par >= i)) raise_flag(a.flags, KSH_FLAG_BAD_PARENT);
    const bool ok = t >= 0 && t < a.vocab;
    if (first && i > 0 && !ok) raise_flag(a.flags, KSH_FLAG_BAD_TOKEN);
    if (!ok) up = -1;                       // never accepted, takes no mass
    tok_s[i] = ok ? static_cast<int>(t) : -1;
    par_s[i] = up;
    if (up >= 0) {
      if (MODE == MODE_GREEDY) {
        u_s[i] = a.greedy[a0 + up] == t ? 1.0f : 0.0f;
      } else {
        u_s[i] = a.u_accept[a0 + i];
        p_s[i] = a.target[(a0 + up) * a.p_stride + t];
        if (MODE == MODE_DRAWN) q_s[i] = a.draft[(a0 + up) * a.q_stride + t];
      }
    }
  }
  __syncthreads();

  Rest r = {};
  r.gone = gone_s;
  auto row_of = [&](int node) {
    r.p = a.target + (a0 + node) * a.p_stride;
    r.q = MODE == MODE_DRAWN ? a.draft + (a0 + node) * a.q_stride : nullptr;
    r.a = 0.0;
    r.k = 0;
  };
  // Warp g's piece of the row: elements [g * chunk, (g + 1) * chunk).
  auto piece = [&](int g, int* lo, int* hi) {
    *lo = min(a.vocab, g * a.chunk);
    *hi = min(a.vocab, *lo + a.chunk);
  };
  auto aligned = [&]() {
    const uintptr_t at = reinterpret_cast<uintptr_t>(r.p) | (MODE == MODE_DRAWN ? reinterpret_cast<uintptr_t>(r.q) : 0);
    return (at & 15) == 0;
  };
  // The rest at 16 elements of each lane, `step` apart four by four from i on
  // (zeros from hi on): every load is on its way before the first is used.
  auto rest16 = [&](int i, int step, int hi, bool vec, double (&v)[16]) {
    float p[16], q[16];
    const bool both = MODE == MODE_DRAWN && r.k > 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = i + u * step;
      if (vec && j + 3 < hi) {
        *reinterpret_cast<float4*>(p + 4 * u) = *reinterpret_cast<const float4*>(r.p + j);
        if (both) *reinterpret_cast<float4*>(q + 4 * u) = *reinterpret_cast<const float4*>(r.q + j);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[4 * u + e] = j + e < hi ? r.p[j + e] : 0.0f;
          if (both) q[4 * u + e] = j + e < hi ? r.q[j + e] : 0.0f;
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      v[e] = static_cast<double>(p[e]);
      if (both) {
        v[e] = fma(-r.a, static_cast<double>(q[e]), v[e]);
        v[e] = v[e] > 0.0 ? v[e] : 0.0;
      }
    }
    if (MODE == MODE_FIXED)
      for (int k = 0; k < r.k; ++k) {
        const int g = r.gone[k] - i;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (g == u * step + e) v[4 * u + e] = 0.0;
      }
  };
  auto sum16 = [](const double (&v)[16]) {
    return (((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]))) +
           (((v[8] + v[9]) + (v[10] + v[11])) + ((v[12] + v[13]) + (v[14] + v[15])));
  };
  int turn = 0;
  // Sums of every piece into all CTAs' part_s[turn], of the piece's 512-element
  // steps into step_s where the search will need them; the row's sum.
  double cum[4];                            // lane: sums up to its (size / 2) pieces
  const int per_slot = (a.chunk + 512 * kSlots - 1) / (512 * kSlots);   // steps that share a slot
  auto total = [&](bool steps) -> double {
    int lo, hi;
    piece(static_cast<int>(rank) * kVerWarps + warp, &lo, &hi);
    const bool vec = aligned();
    double sum = 0.0, slot = 0.0;
    int n_in = 0, at = 0;
    for (int i = lo; i < hi; i += 512) {
      double v[16];
      rest16(i + 4 * lane, 128, hi, vec, v);
      slot += sum16(v);
      if (steps && (++n_in == per_slot || i + 512 >= hi)) {
        slot = warp_sum_f64(slot);
        if (lane == 0) step_s[warp][at] = slot;
        sum += slot;
        slot = 0.0;
        n_in = 0;
        ++at;
      }
    }
    if (!steps) sum = warp_sum_f64(slot);
    turn ^= 1;
    if (!joined) cluster_joined();
    joined = true;
    if (lane < static_cast<int>(size))
      st_cluster_f64(map_rank(smem_u32(&part_s[turn][rank * kVerWarps + warp]), lane), sum);
    cluster_sync();
    // all pieces in order, the same in every warp: lane l the pieces from
    // l * per on
    const int all = static_cast<int>(size) * kVerWarps, per = (all + 31) / 32;
    double c = 0.0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (e < per && lane * per + e < all) c += part_s[turn][lane * per + e];
      cum[e] = c;
    }
    double inc = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) cum[e] += inc - c;
    return __shfl_sync(0xffffffffu, inc, 31);
  };

  int cur = 0, len = 1;
  double z = 1.0;
  bool stale = false;                       // z waits for a sum over the row
  if (tid == 0) path_s[0] = 0;
  if (MODE != MODE_GREEDY) row_of(0);
  for (int i = 1; i < n; ++i) {             // the same walk in every thread
    if (par_s[i] != cur) continue;
    bool yes;
    if (MODE == MODE_GREEDY) {
      yes = u_s[i] != 0.0f;
    } else {
      if (MODE == MODE_DRAWN && stale) {
        z = total(false);
        stale = false;
      }
      const int t = tok_s[i];
      const double q = MODE == MODE_DRAWN ? static_cast<double>(q_s[i]) : 1.0;
      double rt = static_cast<double>(p_s[i]);
      if (MODE == MODE_DRAWN) {
        rt = fmax(fma(-r.a, q, rt), 0.0);
      } else {
        for (int j = 0; j < r.k; ++j)
          if (gone_s[j] == t) rt = 0.0;
      }
      yes = __dmul_rn(__dmul_rn(static_cast<double>(u_s[i]), z), q) < rt;
      if (!yes && MODE == MODE_DRAWN) {
        r.a += z;
        ++r.k;
        stale = true;
      } else if (!yes) {
        __syncthreads();
        if (tid == 0) gone_s[r.k] = t;
        __syncthreads();
        ++r.k;
        z -= rt;
      }
    }
    if (yes) {
      cur = i;
      if (tid == 0) path_s[len] = i;
      ++len;
      z = 1.0;
      stale = false;
      if (MODE != MODE_GREEDY) row_of(i);
    }
  }
  __syncthreads();
  if (first) {
    for (int i = tid; i < a.max_nodes; i += kVerThreads) path[i] = i < len ? path_s[i] : -1;
    if (tid == 0) a.path_len[s] = len;
  }
  if (MODE == MODE_GREEDY) {
    if (first && tid == 0) a.next[s] = a.greedy[a0 + cur];
    return;
  }
  double sum = total(true);
  if (!(sum > 0.0)) {                       // nothing left: the node's own row
    row_of(cur);
    sum = total(true);
  }
  if (!(sum > 0.0)) {
    if (first && tid == 0) {
      raise_flag(a.flags, KSH_FLAG_BAD_PROBS);
      a.next[s] = 0;
    }
    return;
  }
  const double want = __dmul_rn(static_cast<double>(a.u_sample[s]), sum);
  // the piece that crosses the mark; at the very end the last one with mass
  const int all = static_cast<int>(size) * kVerWarps, per = (all + 31) / 32;
  int mine = -1, some = -1;
  double before = 0.0;
#pragma unroll
  for (int e = 3; e >= 0; --e) {
    const int g = lane * per + e;
    if (e < per && g < all) {
      const double own = part_s[turn][g];
      if (own > 0.0 && some < 0) some = g;
      if (cum[e] > want && own > 0.0) {
        mine = g;
        before = cum[e] - own;
      }
    }
  }
  const unsigned cross = __ballot_sync(0xffffffffu, mine >= 0), mass = __ballot_sync(0xffffffffu, some >= 0);
  if (cross) {
    const int from = __ffs(static_cast<int>(cross)) - 1;
    mine = __shfl_sync(0xffffffffu, mine, from);
    before = __shfl_sync(0xffffffffu, before, from);
  } else {
    mine = __shfl_sync(0xffffffffu, some, 31 - __clz(static_cast<int>(mass)));
    before = INFINITY;                      // no element crosses: the last with mass
  }
  if (mine / kVerWarps != static_cast<int>(rank) || mine % kVerWarps != warp) return;
  int lo, hi;
  piece(mine, &lo, &hi);
  const bool vec = aligned();
  bool seek = before != INFINITY;
  double base = seek ? before : 0.0;
  // the slot that crosses the mark (else the last one with mass)
  const int span = 512 * per_slot, slots = (hi - lo + span - 1) / span;
  int pick = -1, heavy = 0;
  for (int at = 0; at < slots && pick < 0; ++at) {
    const double own = step_s[warp][at];
    if (own > 0.0) heavy = at;
    if (seek && base + own > want && own > 0.0)
      pick = at;
    else
      base += own;
  }
  seek = pick >= 0;
  if (!seek) pick = heavy;
  // its steps: lane l has 16 elements in a row
  int found = -1, last = lo;
  const int end = min(lo + (pick + 1) * span, hi);
  for (int i0 = lo + pick * span; i0 < end && found < 0; i0 += 512) {
    double v[16];
    rest16(i0 + 16 * lane, 4, end, vec, v);
    const double x = sum16(v);
    double c = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, c, o);
      if (lane >= o) c += up;
    }
    double sofar = base + (c - x);
    int here = -1, live = -1;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      sofar += v[e];
      if (v[e] > 0.0) {
        live = i0 + 16 * lane + e;
        if (here < 0 && seek && sofar > want) here = live;
      }
    }
    const unsigned over = __ballot_sync(0xffffffffu, here >= 0), any = __ballot_sync(0xffffffffu, live >= 0);
    if (over) found = __shfl_sync(0xffffffffu, here, __ffs(static_cast<int>(over)) - 1);
    if (any) last = __shfl_sync(0xffffffffu, live, 31 - __clz(static_cast<int>(any)));
    base += __shfl_sync(0xffffffffu, c, 31);
  }
  if (lane == 0) a.next[s] = found >= 0 ? found : last;
}

template <class Args>
int launch_cluster(void (*kern)(Args), int64_t groups, int cluster, int threads, size_t smem,
                   cudaStream_t stream, const Args& a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(groups * cluster));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a);
  if (e != cudaSuccess) return record_cuda_error(e);
  count_launch();
  return KSH_OK;
}

}  // namespace
}  // namespace ksh

using namespace ksh;

extern "C" int ksh_target_probs(const float* logits, int64_t m, int64_t vocab,
                                int64_t logits_stride, const float* temperature, float* probs,
                                int64_t probs_stride, void* stream) {
  KSH_CHECK_ARG(m >= 0 && m <= INT32_MAX && vocab > 0 && vocab <= INT32_MAX &&
                logits_stride >= vocab && probs_stride >= vocab);
  if (m == 0) return KSH_OK;
  KSH_CHECK_ARG(logits && probs);
  if (vocab > kMaxVocab) return KSH_ERR_UNSUPPORTED;
  ProbArgs a = {logits, temperature, probs, logits_stride, probs_stride, static_cast<int>(vocab), 0};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // CTAs per row: parts of at most 80 KB, so that two or three CTAs share an
  // SM and one's reading overlaps another's writing; with few rows more and
  // smaller parts, down to 8 KB
  int cluster = 1;
  while (cluster < kMaxCluster && vocab > 20480LL * cluster) cluster *= 2;
  while (cluster < kMaxCluster && m * cluster < 2LL * num_sms() && vocab > 4096LL * cluster) cluster *= 2;
  const int64_t chunk = ((vocab + cluster - 1) / cluster + 3) / 4 * 4;
  if (chunk > kProbSlice || m * cluster > INT32_MAX)
    return launch(target_probs_long_kernel, dim3(static_cast<unsigned>(m)), dim3(kProbThreads), 0, st, a);
  a.chunk = static_cast<int>(chunk);
  const size_t smem = static_cast<size_t>(chunk + 12) * 4;
  if (set_smem_optin(reinterpret_cast<const void*>(target_probs_kernel), smem) != KSH_OK) return KSH_ERR_CUDA;
  return launch_cluster(target_probs_kernel, m, cluster, kProbThreads, smem, st, a);
}

extern "C" int ksh_verify_tree(const int64_t* tokens, const int32_t* parents,
                               const int32_t* q_start, int64_t num_seqs, int64_t total,
                               int64_t max_nodes, int64_t vocab, const float* target_probs,
                               int64_t target_stride, const float* draft_probs,
                               int64_t draft_stride, const int64_t* target_tokens,
                               const float* u_accept, const float* u_sample, int32_t* path,
                               int32_t* path_len, int64_t* next_tokens, int32_t* flags,
                               void* stream) {
  KSH_CHECK_ARG(num_seqs > 0 && num_seqs <= INT32_MAX && total >= 0 && total <= INT32_MAX &&
                max_nodes > 0 && vocab > 0 && vocab <= INT32_MAX);
  KSH_CHECK_ARG(q_start && path && path_len && next_tokens && (total == 0 || (tokens && parents)));
  KSH_CHECK_ARG((target_probs != nullptr) != (target_tokens != nullptr));
  if (target_probs) {
    KSH_CHECK_ARG(u_accept && u_sample && target_stride >= vocab);
    KSH_CHECK_ARG(!draft_probs || draft_stride >= vocab);
  } else {
    KSH_CHECK_ARG(!draft_probs);
  }
  if (max_nodes > kMaxNodes || vocab > kMaxVocab) return KSH_ERR_UNSUPPORTED;
  VerArgs a = {};
  a.tokens = tokens;
  a.parents = parents;
  a.q_start = q_start;
  a.target = target_probs;
  a.draft = draft_probs;
  a.greedy = target_tokens;
  a.u_accept = u_accept;
  a.u_sample = u_sample;
  a.path = path;
  a.path_len = path_len;
  a.next = next_tokens;
  a.flags = flags;
  a.total = total;
  a.p_stride = target_stride;
  a.q_stride = draft_stride;
  a.vocab = static_cast<int>(vocab);
  a.max_nodes = static_cast<int>(max_nodes);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (target_tokens) return launch_cluster(verify_tree_kernel<MODE_GREEDY>, num_seqs, 1, kVerThreads, 0, st, a);
  // CTAs per sequence: as many as run at once (four per SM), pieces of at least
  // 256 elements a warp.  64 x 128256 drawn: 25.0 us with 8 (more even over the
  // SMs), 27.2 with 4 of 512 threads, 31.8 with 4 of 256.
  int cluster = 1;
  while (cluster < kMaxCluster && num_seqs * cluster <= 2 * num_sms() && vocab >= 4096LL * cluster) cluster *= 2;
  if (num_seqs * cluster > INT32_MAX) return KSH_ERR_UNSUPPORTED;
  a.chunk = static_cast<int>(((vocab + cluster * kVerWarps - 1) / (cluster * kVerWarps) + 3) / 4 * 4);
  if (draft_probs) return launch_cluster(verify_tree_kernel<MODE_DRAWN>, num_seqs, cluster, kVerThreads, 0, st, a);
  return launch_cluster(verify_tree_kernel<MODE_FIXED>, num_seqs, cluster, kVerThreads, 0, st, a);
}
