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

#include <math.h>

#include "common.cuh"

namespace ksh {
namespace {

constexpr int kProbThreads = 512;

__global__ void __launch_bounds__(kProbThreads)
target_probs_kernel(const float* x, int64_t x_stride, const float* temperature, float* p,
                    int64_t p_stride, int64_t vocab) {
  __shared__ float redf[kProbThreads / 32];
  __shared__ int64_t redi[kProbThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_dep_wait();
  grid_dep_launch();
  const float* xr = x + static_cast<int64_t>(blockIdx.x) * x_stride;
  float* pr = p + static_cast<int64_t>(blockIdx.x) * p_stride;
  const float t = temperature ? temperature[blockIdx.x] : 1.0f;
  float m = -INFINITY;
  int64_t at = vocab;
  for (int64_t i = tid; i < vocab; i += kProbThreads) {
    const float v = xr[i];
    if (v > m || (v == m && i < at)) {
      m = v;
      at = i;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, m, o);
    const int64_t oa = __shfl_xor_sync(0xffffffffu, at, o);
    if (om > m || (om == m && oa < at)) {
      m = om;
      at = oa;
    }
  }
  if (lane == 0) {
    redf[warp] = m;
    redi[warp] = at;
  }
  __syncthreads();
  for (int w = 0; w < kProbThreads / 32; ++w)
    if (redf[w] > m || (redf[w] == m && redi[w] < at)) {
      m = redf[w];
      at = redi[w];
    }
  if (t <= 0.0f) {
    for (int64_t i = tid; i < vocab; i += kProbThreads) pr[i] = i == at ? 1.0f : 0.0f;
    return;
  }
  float sum = 0.0f;
  for (int64_t i = tid; i < vocab; i += kProbThreads) sum += expf((xr[i] - m) / t);
  sum = warp_sum(sum);
  __syncthreads();
  if (lane == 0) redf[warp] = sum;
  __syncthreads();
  sum = 0.0f;
  for (int w = 0; w < kProbThreads / 32; ++w) sum += redf[w];
  for (int64_t i = tid; i < vocab; i += kProbThreads) pr[i] = expf((xr[i] - m) / t) / sum;
}

// ---------------------------------------------------------------------------

constexpr int kMaxNodes = 256;
constexpr int kVerThreads = 512;
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
  int vocab, max_nodes;
};

// What is left of the target's row at the current node: the Z of every
// rejected draw, or the tokens of every rejected fixed proposal.
struct Rest {
  const float* p;
  const float* q;
  const double* z;
  const int* gone;
  int k;
};

template <int MODE>
__device__ __forceinline__ double rest_at(const Rest& r, int i) {
  double v = static_cast<double>(r.p[i]);
  if (MODE == MODE_DRAWN) {
    if (r.k > 0) {
      const double q = static_cast<double>(r.q[i]);
      for (int j = 0; j < r.k; ++j) v = fmax(__dsub_rn(v, __dmul_rn(r.z[j], q)), 0.0);
    }
  } else {
    for (int j = 0; j < r.k; ++j)
      if (r.gone[j] == i) v = 0.0;
  }
  return v;
}

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int MODE>
__global__ void __launch_bounds__(kVerThreads) verify_tree_kernel(VerArgs a) {
  __shared__ int tok_s[kMaxNodes], par_s[kMaxNodes], path_s[kMaxNodes], gone_s[kMaxNodes];
  __shared__ float u_s[kMaxNodes], p_s[kMaxNodes], q_s[kMaxNodes];
  __shared__ double z_s[kMaxNodes], part_s[kVerWarps];
  __shared__ int hit_s;
  const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_dep_wait();
  grid_dep_launch();
  const int64_t a0 = a.q_start[s], a1 = a.q_start[s + 1];
  int n = static_cast<int>(min(a1 - a0, static_cast<int64_t>(a.max_nodes)));
  if (a0 < 0 || a1 > a.total || a1 - a0 > a.max_nodes || a1 < a0) {
    if (tid == 0) raise_flag(a.flags, KSH_FLAG_BAD_LENGTH);
    if (a0 < 0 || a1 > a.total) n = 0;
  }
  int32_t* path = a.path + static_cast<int64_t>(s) * a.max_nodes;
  if (n <= 0) {
    for (int i = tid; i < a.max_nodes; i += kVerThreads) path[i] = -1;
    if (tid == 0) {
      a.path_len[s] = 0;
      a.next[s] = -1;
    }
    return;
  }
  for (int i = tid; i < n; i += kVerThreads) {
    const int64_t t = a.tokens[a0 + i];
    const int par = a.parents[a0 + i];
    int up = i > 0 && par >= 0 && par < i ? par : -1;
    if (i > 0 && (par < 0 || par >= i)) raise_flag(a.flags, KSH_FLAG_BAD_PARENT);
    const bool ok = t >= 0 && t < a.vocab;
    if (i > 0 && !ok) raise_flag(a.flags, KSH_FLAG_BAD_TOKEN);
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
  r.z = z_s;
  r.gone = gone_s;
  auto row_of = [&](int node) {
    r.p = a.target + (a0 + node) * a.p_stride;
    r.q = MODE == MODE_DRAWN ? a.draft + (a0 + node) * a.q_stride : nullptr;
    r.k = 0;
  };
  // sum of the rest over the row, the same in every thread; part_s keeps the
  // warps' shares (a warp owns a contiguous piece)
  const int chunk = (a.vocab + kVerWarps - 1) / kVerWarps;
  const int lo = min(warp * chunk, a.vocab), hi = min(lo + chunk, a.vocab);
  auto total = [&]() -> double {
    double v = 0.0;
    for (int i = lo + lane; i < hi; i += 32) v += rest_at<MODE>(r, i);
    v = warp_sum_f64(v);
    __syncthreads();
    if (lane == 0) part_s[warp] = v;
    __syncthreads();
    double t = 0.0;
    for (int w = 0; w < kVerWarps; ++w) t += part_s[w];
    return t;
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
        z = total();
        stale = false;
      }
      const int t = tok_s[i];
      const double q = MODE == MODE_DRAWN ? static_cast<double>(q_s[i]) : 1.0;
      double rt = static_cast<double>(p_s[i]);
      for (int j = 0; j < r.k; ++j) {
        if (MODE == MODE_DRAWN)
          rt = fmax(__dsub_rn(rt, __dmul_rn(z_s[j], q)), 0.0);
        else if (gone_s[j] == t)
          rt = 0.0;
      }
      yes = __dmul_rn(__dmul_rn(static_cast<double>(u_s[i]), z), q) < rt;
      if (!yes) {
        __syncthreads();
        if (tid == 0) {
          if (MODE == MODE_DRAWN) z_s[r.k] = z; else gone_s[r.k] = t;
        }
        __syncthreads();
        ++r.k;
        if (MODE == MODE_DRAWN) stale = true; else z -= rt;
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
  for (int i = tid; i < a.max_nodes; i += kVerThreads) path[i] = i < len ? path_s[i] : -1;
  if (tid == 0) a.path_len[s] = len;
  if (MODE == MODE_GREEDY) {
    if (tid == 0) a.next[s] = a.greedy[a0 + cur];
    return;
  }
  double sum = total();
  if (!(sum > 0.0)) {                       // nothing left: the node's own row
    row_of(cur);
    sum = total();
  }
  const double want = __dmul_rn(static_cast<double>(a.u_sample[s]), sum);
  // the warp whose piece crosses the mark finds the token
  if (tid == 0) hit_s = -1;
  __syncthreads();
  double before = 0.0;
  int mine = -1, last = 0;
  for (int w = 0; w < kVerWarps; ++w) {
    if (part_s[w] > 0.0) last = w;
    if (mine < 0 && before + part_s[w] > want) mine = w;
    if (mine < 0) before += part_s[w];
  }
  if (mine < 0) mine = last;                // the mark at the very end
  if (!(sum > 0.0)) {
    if (tid == 0) {
      raise_flag(a.flags, KSH_FLAG_BAD_PROBS);
      a.next[s] = 0;
    }
    return;
  }
  if (warp != mine) return;
  int found = -1, some = 0;
  double base = before;
  for (int i0 = lo; i0 < hi && found < 0; i0 += 32) {
    const int i = i0 + lane;
    const double v = i < hi ? rest_at<MODE>(r, i) : 0.0;
    double c = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, c, o);
      if (lane >= o) c += up;
    }
    const unsigned over = __ballot_sync(0xffffffffu, v > 0.0 && base + c > want);
    const unsigned any = __ballot_sync(0xffffffffu, v > 0.0);
    if (over) found = i0 + __ffs(over) - 1;
    if (any) some = i0 + 31 - __clz(any);
    base += __shfl_sync(0xffffffffu, c, 31);
  }
  if (lane == 0) a.next[s] = found >= 0 ? found : some;
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
  return launch(target_probs_kernel, dim3(static_cast<unsigned>(m)), dim3(kProbThreads), 0,
                static_cast<cudaStream_t>(stream), logits, logits_stride, temperature, probs,
                probs_stride, vocab);
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
  if (max_nodes > kMaxNodes) return KSH_ERR_UNSUPPORTED;
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
  const dim3 grid(static_cast<unsigned>(num_seqs));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (target_tokens) return launch(verify_tree_kernel<MODE_GREEDY>, grid, dim3(kVerThreads), 0, st, a);
  if (draft_probs) return launch(verify_tree_kernel<MODE_DRAWN>, grid, dim3(kVerThreads), 0, st, a);
  return launch(verify_tree_kernel<MODE_FIXED>, grid, dim3(kVerThreads), 0, st, a);
}
