// Attention of drafted tokens over the paged cache.
//
// Sequence s has prefix[s] cached positions and n = q_start[s+1] - q_start[s]
// drafted nodes whose K/V stand in the slots of positions prefix .. prefix +
// n - 1 (node order).  Node i attends every cached position and the nodes
// whose bit is set in its mask (64-bit words; no mask: nodes 0..i):
//     o = sum_j exp(q.k_j / sqrt(D) - m) v_j / sum_j exp(q.k_j / sqrt(D) - m)
// with the running maximum m, rescaled as it rises.  A node that may see no
// key gives zeros; what a node may not see does not reach its sums, NaN and
// infinity included.
//
// Head dimensions 64 and 128 (tree_attn_tc_kernel): the n * g query rows of a
// kv head share every K/V row, so past about 20 rows CUDA cores would bound
// the kernel (4 R D operations for 8 D bytes); the products go to the tensor
// cores at fp32 accuracy by splitting each operand into two fp16 terms,
// x * 2^e = hi + lo (22 bits; one power of two per row), and taking
// hi*lo + lo*hi + hi*hi.  With 128 query rows on the MMA's M side that is
// 1.6 K tensor cycles per 64 keys of D = 128 against 2.8 K cycles that the
// SM's share of HBM needs for their 64 KB: HBM stays the bound up to 128 rows.
//
// One persistent CTA per SM.  The (sequence, kv head, 128-row tile) items'
// 64-key tiles form one line that is cut into equal pieces, one per CTA, so
// uneven lengths leave no SM idle; an item cut between CTAs leaves its
// (m, l, acc) pieces in the workspace and tree_merge_kernel joins them in key
// order (the same bits in every run).  Warps of a CTA:
//   0..3   rows: thread = query row.  Scores from TMEM, running softmax in
//          32 bits, P split into hi / lo back into TMEM (over the scores), and
//          every tile's P V added into fp32 registers (adding a long context
//          up inside the tensor core would round toward zero at each step)
//   4..11  K/V: global -> registers (one tile ahead) -> scaled hi / lo fp16 in
//          shared memory, 128-byte swizzle; block table per key, any block size
//   12     MMAs: S = Q K^T (A = Q in TMEM, B = K), O = P V (A = P in TMEM, B =
//          V with the keys along K, so no transpose is stored)

#include <math.h>

#include <algorithm>

#include "tc_common.cuh"

namespace ksh {
namespace {

using namespace tc;

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
  struct SplitItem* items;      // [gridDim.x] items cut at the end of a CTA's piece
  float* part;                  // [gridDim.x][2] partial states
  int64_t total, num_blocks, num_layers, layer, hkv, hq, bs, max_blocks;
  int num_seqs, words, g, d, max_nodes;
  float scale;
};

// An item whose first piece CTA `first` holds: joined from pieces first..last.
struct SplitItem {
  int32_t first, last;          // last < first: none
  int32_t row0;                 // q row of the tile's first node's sequence (a0)
  int32_t rbase;                // first query row (node * g + head of the group) of the tile
  int32_t rows;                 // live rows
  int32_t hk;
  int32_t pad[2];
};

constexpr int kTK = 64;                  // keys per tile
constexpr int kRows = 128;               // query rows per tile (MMA M)
constexpr int kRowWarps = 4, kLoadWarps = 8;
constexpr int kTcThreads = 512;          // rows 128, loaders 256, MMA warp + 3 idle
constexpr int kKeysPerWarp = kTK / kLoadWarps;

// floats of one partial state: m [128], l [128], acc [D / 4][128][4]
template <int D>
constexpr int64_t part_floats() { return 2 * kRows + static_cast<int64_t>(D) * kRows; }

template <int D>
struct TreeLayout {
  static constexpr int TERM = kTK * D * 2;           // one fp16 term of a K or V tile
  static constexpr int HALF = kTK * 128;             // 64 columns of it: 128-byte rows
  static constexpr int NST = D == 128 ? 3 : 6;       // stages of K and of V
  static constexpr int K_OFF = 0;
  static constexpr int V_OFF = NST * 2 * TERM;
  static constexpr int META = 2 * V_OFF;             // kinv, vinv [NST][64]
  static constexpr int BITS = META + 2 * NST * kTK * 4;    // valid, kpois, vpois [NST][8] bytes
  static constexpr int BAR = BITS + 3 * NST * 8;
  static constexpr int NBAR = 4 * NST + 2 * 3 + 2;
  static constexpr int MISC = BAR + NBAR * 8;
  static constexpr int BYTES = MISC + 64 + 1024;
  // TMEM columns: Q hi, Q lo (D / 2 each), two S / P buffers, two O buffers
  static constexpr uint32_t Q_COL = 0, S_COL = D, O_COL = D + 2 * kTK;
  static constexpr uint32_t COLS = 512;
  static_assert(O_COL + 2 * D <= COLS, "TMEM columns");
  static_assert(BYTES <= 227 * 1024, "shared memory");
};

// One sequence's share of the work.
struct SeqWork {
  int64_t a0;
  int nq, keys, pre, ntiles, nqt;
  bool bad;                     // lengths that do not fit
  __device__ __forceinline__ int64_t units(int64_t hkv) const {
    return hkv * nqt * static_cast<int64_t>(ntiles);
  }
};

__device__ __forceinline__ SeqWork seq_work(const TreeArgs& a, int s) {
  SeqWork w = {};
  const int64_t a0 = a.q_start[s], n = a.q_start[s + 1] - a0;
  const int pre = a.prefix[s];
  w.a0 = a0;
  w.pre = max(pre, 0);
  w.bad = a0 < 0 || n < 0 || a0 + n > a.total || n > a.max_nodes || pre < 0;
  const int64_t cap = a.max_blocks * a.bs;
  if (w.pre + n > cap) w.bad = true;
  if (a0 < 0 || n <= 0 || a0 >= a.total) return w;
  w.nq = static_cast<int>(min(min(n, static_cast<int64_t>(a.max_nodes)), a.total - a0));
  w.keys = static_cast<int>(min(w.pre + n, min(cap, static_cast<int64_t>(INT32_MAX - kTK))));
  w.ntiles = (w.keys + kTK - 1) / kTK;
  w.nqt = (w.nq * a.g + kRows - 1) / kRows;
  return w;
}

// The pieces of items in one CTA's share [u, u_end) of the line, one after
// the other.  Each warp keeps its own walk in shared memory (registers are
// for the tiles).
struct Walk {
  int64_t u, u_end, base;       // base: first unit of sequence s
  int s;
};
struct Piece {
  int64_t a0;
  int s, hk, qt, t0, t1, nq, keys, pre, ntiles;
};

__device__ __forceinline__ bool next_piece(const TreeArgs& a, Walk* wk, Piece* p) {
  Walk k = *wk;
  if (k.u >= k.u_end) return false;
  SeqWork w = seq_work(a, k.s);
  while (k.u >= k.base + w.units(a.hkv)) {
    k.base += w.units(a.hkv);
    w = seq_work(a, ++k.s);
  }
  const int item = static_cast<int>((k.u - k.base) / w.ntiles);
  p->t0 = static_cast<int>((k.u - k.base) - static_cast<int64_t>(item) * w.ntiles);
  p->t1 = static_cast<int>(min(static_cast<int64_t>(w.ntiles), p->t0 + (k.u_end - k.u)));
  p->hk = item / w.nqt;
  p->qt = item - p->hk * w.nqt;
  p->s = k.s;
  p->a0 = w.a0;
  p->nq = w.nq;
  p->keys = w.keys;
  p->pre = w.pre;
  p->ntiles = w.ntiles;
  k.u += p->t1 - p->t0;
  __syncwarp();
  if ((threadIdx.x & 31) == 0) *wk = k;
  __syncwarp();
  return true;
}

__device__ __forceinline__ float4 ld_stream(const float* p) {
  float4 v;
  asm volatile("ld.global.L1::no_allocate.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// Power of two that brings a row whose largest |x| has these bits into
// [2^14, 2^15), and its inverse.
__device__ __forceinline__ void row_scale(uint32_t bits, float* s, float* inv) {
  const int e = min(268 - static_cast<int>(bits >> 23), 253);
  *s = __uint_as_float(static_cast<uint32_t>(e) << 23);
  *inv = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
// x = hi + lo as fp16 pairs
__device__ __forceinline__ void split2(float x, float y, uint32_t* hi, uint32_t* lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  *hi = h2_bits(h);
  *lo = h2_bits(__floats2half2_rn(x - f.x, y - f.y));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// MN-major operand, 128-byte swizzle: 64 columns of 2 bytes per 128-byte row,
// 8 rows (of the K dimension) per 1024-byte group; `lbo` bytes to the next 64
// columns.
__device__ __forceinline__ uint64_t desc_mn_sw128(uint32_t smem_addr, uint32_t lbo) {
  uint64_t d = desc_k_sw128(smem_addr);
  d &= ~(static_cast<uint64_t>(0x3FFFu) << 16);
  return d | (static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16);
}

template <int N>
__device__ __forceinline__ void set_regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void set_regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Float offset of the K row of a sequence's `pos`, -1 without one.
__device__ __forceinline__ int64_t key_offset(const TreeArgs& a, int s, int hk, int pos, int D) {
  const int64_t j = pos / a.bs;
  const int64_t blk = a.block_tables[static_cast<int64_t>(s) * a.max_blocks + j];
  if (blk < 0 || blk >= a.num_blocks) return -1;
  return ((((blk * a.num_layers + a.layer) * 2) * a.hkv + hk) * a.bs + (pos - j * a.bs)) * D;
}

template <int D>
__global__ void __launch_bounds__(kTcThreads, 1) tree_attn_tc_kernel(TreeArgs a) {
  using L = TreeLayout<D>;
  constexpr int NST = L::NST;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* kinv_s = reinterpret_cast<float*>(smem + L::META);
  float* vinv_s = kinv_s + NST * kTK;
  uint8_t* valid_s = smem + L::BITS;
  uint8_t* kpois_s = valid_s + NST * 8;
  uint8_t* vpois_s = kpois_s + NST * 8;
  uint64_t* kfull = reinterpret_cast<uint64_t*>(smem + L::BAR);
  uint64_t* kempty = kfull + NST;
  uint64_t* vfull = kempty + NST;
  uint64_t* vempty = vfull + NST;
  uint64_t* sfull = vempty + NST;       // [2]
  uint64_t* pready = sfull + 2;         // [2]
  uint64_t* ofull = pready + 2;         // [2]
  uint64_t* qready = ofull + 2;
  uint64_t* drain = qready + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* s0_s = reinterpret_cast<int*>(tmem_slot + 2);
  int64_t* line_s = reinterpret_cast<int64_t*>(tmem_slot + 4);   // U, base of s0
  __shared__ int64_t scan_s[kTcThreads / 32];
  __shared__ Walk walk_s[kTcThreads / 32];
  __shared__ uint64_t rare_s[2][kRows];     // keys with a V that is not finite, per row
  __shared__ SplitItem cut_s;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < NST; ++i) {
      mbar_init(&kfull[i], kLoadWarps);
      mbar_init(&kempty[i], 1 + kRowWarps);      // the MMAs and every row warp
      mbar_init(&vfull[i], kLoadWarps);
      mbar_init(&vempty[i], 1 + kRowWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sfull[i], 1);
      mbar_init(&pready[i], kRowWarps);
      mbar_init(&ofull[i], 1);
    }
    mbar_init(qready, kRowWarps);
    mbar_init(drain, 1);
    *abort_flag = 0;
    *s0_s = 0;
    fence_barrier_init();
  }
  if (warp == 12) {
    tmem_alloc(tmem_slot, L::COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  grid_dep_wait();
  grid_dep_launch();

  // The line of tiles: its length, and the sequence where this CTA's share
  // starts.
  int64_t U = 0, u0 = 0, G = 1;                   // CTAs that get tiles
  for (int pass = 0; pass < 2; ++pass) {
    int64_t carry = 0;
    for (int b = 0; b < a.num_seqs; b += kTcThreads) {
      const int s = b + tid;
      int64_t v = 0;
      if (s < a.num_seqs) {
        const SeqWork w = seq_work(a, s);
        v = w.units(a.hkv);
        if (pass == 0 && blockIdx.x == 0 && w.bad) raise_flag(a.flags, KSH_FLAG_BAD_LENGTH);
      }
      int64_t inc = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
      }
      __syncthreads();
      if (lane == 31) scan_s[warp] = inc;
      __syncthreads();
      int64_t before = carry;
      for (int w = 0; w < kTcThreads / 32; ++w) {
        if (w < warp) before += scan_s[w];
        carry += scan_s[w];
      }
      inc += before;
      if (pass == 1 && v > 0 && u0 >= inc - v && u0 < inc) {
        *s0_s = s;
        line_s[1] = inc - v;
      }
    }
    if (pass == 0) {
      U = carry;
      G = max(min(static_cast<int64_t>(gridDim.x), U), int64_t(1));
      u0 = min(static_cast<int64_t>(blockIdx.x), G) * U / G;
    }
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int64_t u1 = min(static_cast<int64_t>(blockIdx.x) + 1, G) * U / G;
  Walk* const wk = &walk_s[warp];
  if (lane == 0) {
    Walk k = {};
    k.u = u0;
    k.u_end = u1;
    if (u0 < u1) {
      k.s = *s0_s;
      k.base = line_s[1];
    }
    *wk = k;
  }
  if (tid == 0) cut_s.first = 0, cut_s.last = -1;
  __syncwarp();
  Piece pc = {};

  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    bool ok = false;
    for (uint32_t i = 0; i < (1u << 22) && !ok; ++i) {
      ok = mbar_try_wait(bar, parity);
      if (!ok && (i & 63u) == 63u && *abort_flag) break;
    }
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) *abort_flag = 1;
    return ok;
  };

  if (warp >= 12) {
    set_regs_dec<56>();
    if (warp == 12) {
      // ---------------- MMAs ----------------
      constexpr uint32_t id_s = idesc_f16_f32(kRows, kTK);
      constexpr uint32_t id_o = idesc_f16_f32(kRows, D) | (1u << 16);   // B: keys along K
      int n = 0, seg = 0;
      bool ok = true;
      const uint32_t kbase = smem_u32(smem + L::K_OFF), vbase = smem_u32(smem + L::V_OFF);
      auto issue_o = [&](int m) -> bool {            // O = P V of tile m
        const int st = m % NST, b = m & 1;
        if (!wait(&vfull[st], (m / NST) & 1) || !wait(&pready[b], (m >> 1) & 1)) return false;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t d = tmem + L::O_COL + static_cast<uint32_t>(b) * D;
          const uint32_t ph = tmem + L::S_COL + static_cast<uint32_t>(b) * kTK;
          // columns of 16 keys: [hi 8][hi 8][lo 8][lo 8] per 32 keys
          auto pcol = [&](int k, int lo) { return ph + static_cast<uint32_t>((k >> 1) * 32 + lo * 16 + (k & 1) * 8); };
          const uint64_t vh = desc_mn_sw128(vbase + st * 2 * L::TERM, L::HALF);
          const uint64_t vl = desc_mn_sw128(vbase + st * 2 * L::TERM + L::TERM, L::HALF);
          // 16 keys: 8 columns of P, 2048 bytes (128 in the address field) of V
#pragma unroll
          for (int k = 0; k < kTK / 16; ++k) mma_f16_ts(d, pcol(k, 0), vl + 128 * k, id_o, k > 0);
#pragma unroll
          for (int k = 0; k < kTK / 16; ++k) mma_f16_ts(d, pcol(k, 1), vh + 128 * k, id_o, 1u);
#pragma unroll
          for (int k = 0; k < kTK / 16; ++k) mma_f16_ts(d, pcol(k, 0), vh + 128 * k, id_o, 1u);
          mma_commit(&vempty[st]);
          mma_commit(&ofull[b]);
        }
        __syncwarp();
        return true;
      };
      while (ok && next_piece(a, wk, &pc)) {
        if (!(ok = wait(qready, seg & 1))) break;
        ++seg;
        tc_fence_after();
        for (int t = pc.t0; t < pc.t1; ++t, ++n) {
          const int st = n % NST, b = n & 1;
          if (!(ok = wait(&kfull[st], (n / NST) & 1))) break;
          tc_fence_after();
          if (elect_one()) {
            const uint32_t d = tmem + L::S_COL + static_cast<uint32_t>(b) * kTK;
            const uint32_t qh = tmem + L::Q_COL, ql = qh + D / 2;
            const uint32_t kb = kbase + st * 2 * L::TERM;
            // the small terms first: the tensor core cuts low bits off at
            // every step, relative to the sum so far
#pragma unroll
            for (int term = 0; term < 3; ++term) {
              const uint32_t qa = term == 1 ? ql : qh;
              const uint32_t kt = kb + (term == 0 ? L::TERM : 0);
#pragma unroll
              for (int k = 0; k < D / 16; ++k) {
                const uint64_t kd = desc_k_sw128(kt + (k / 4) * L::HALF) + 2 * (k % 4);
                mma_f16_ts(d, qa + 8 * k, kd, id_s, (term > 0 || k > 0) ? 1u : 0u);
              }
            }
            mma_commit(&kempty[st]);
            mma_commit(&sfull[b]);
          }
          __syncwarp();
          if (t > pc.t0 && !(ok = issue_o(n - 1))) break;
        }
        if (ok) ok = issue_o(n - 1);
      }
      // nothing of this CTA's is in flight when its TMEM goes
      if (elect_one()) mma_commit(drain);
      __syncwarp();
      mbar_wait(drain, 0);
    }
  } else if (warp >= kRowWarps) {
    // ---------------- K/V ----------------
    set_regs_dec<120>();
    const int lw = warp - kRowWarps;
    constexpr int RPI = 128 / D;                    // rows per warp-wide load
    constexpr int NLD = kKeysPerWarp / RPI;         // loads of K (and of V) per tile
    const int sub = D == 128 ? 0 : lane >> 4;       // row of the load
    const int ln = D == 128 ? lane : lane & 15;     // float4 column of the row
    const int64_t vstep = a.hkv * a.bs * D;
    const uint32_t half_off = static_cast<uint32_t>(ln >> 4) * L::HALF;
    const uint32_t chunk = static_cast<uint32_t>((ln & 15) >> 1), word = static_cast<uint32_t>(ln & 1) * 8;
    bool have = next_piece(a, wk, &pc);
    int t = pc.t0;
    bool bad = false;
    // offset of key lw * 8 + (lane & 7) of tile t
    auto offset_of = [&]() -> int64_t {
      const int pos = t * kTK + lw * kKeysPerWarp + (lane & 7);
      if (!have || pos >= pc.keys) return -1;
      const int64_t o = key_offset(a, pc.s, pc.hk, pos, D);
      bad |= o < 0;
      return o;
    };
    auto step = [&]() {
      if (++t >= pc.t1) {
        have = next_piece(a, wk, &pc);
        t = pc.t0;
      }
    };
    float4 kr[NLD], vr[NLD];
    auto load = [&](float4 (&r)[NLD], int64_t off, int64_t add) {
#pragma unroll
      for (int i = 0; i < NLD; ++i) {
        const int64_t o = __shfl_sync(0xffffffffu, off, i * RPI + sub);
        r[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (o >= 0) r[i] = ld_stream(a.pool + o + add + 4 * ln);
      }
    };
    // scaled hi / lo terms of the warp's rows into a stage; bits of the rows
    // that hold something not finite (those elements go in as zeros)
    auto store = [&](float4 (&r)[NLD], uint8_t* stage, float* inv_s) -> uint32_t {
      uint32_t pois = 0;
#pragma unroll
      for (int i = 0; i < NLD; ++i) {
        const int key = i * RPI + sub;              // of the warp's eight
        float4 v = r[i];
        uint32_t mx = max(max(abs_bits(v.x), abs_bits(v.y)), max(abs_bits(v.z), abs_bits(v.w)));
        if (__any_sync(0xffffffffu, mx >= 0x7f800000u)) {
          const bool mine = mx >= 0x7f800000u;
          const unsigned who = __ballot_sync(0xffffffffu, mine);
          if (D == 128) {
            pois |= 1u << i;
          } else {
            if (who & 0xffffu) pois |= 1u << (i * RPI);
            if (who >> 16) pois |= 1u << (i * RPI + 1);
          }
          v.x = abs_bits(v.x) >= 0x7f800000u ? 0.f : v.x;
          v.y = abs_bits(v.y) >= 0x7f800000u ? 0.f : v.y;
          v.z = abs_bits(v.z) >= 0x7f800000u ? 0.f : v.z;
          v.w = abs_bits(v.w) >= 0x7f800000u ? 0.f : v.w;
          mx = max(max(abs_bits(v.x), abs_bits(v.y)), max(abs_bits(v.z), abs_bits(v.w)));
        }
        if (D == 128) {
          mx = __reduce_max_sync(0xffffffffu, mx);
        } else {
#pragma unroll
          for (int o = 8; o > 0; o >>= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        }
        float sc, inv;
        row_scale(mx, &sc, &inv);
        uint2 hi, lo;
        split2(v.x * sc, v.y * sc, &hi.x, &lo.x);
        split2(v.z * sc, v.w * sc, &hi.y, &lo.y);
        const int row = lw * kKeysPerWarp + key;
        const uint32_t at = half_off + static_cast<uint32_t>(row) * 128 +
                            ((chunk ^ static_cast<uint32_t>(row & 7)) << 4) + word;
        *reinterpret_cast<uint2*>(stage + at) = hi;
        *reinterpret_cast<uint2*>(stage + L::TERM + at) = lo;
        if (ln == 0) inv_s[row] = inv;
      }
      return pois;
    };
    int64_t off = offset_of();
    if (have) {
      load(kr, off, 0);
      load(vr, off, vstep);
    }
    for (int n = 0; have; ++n) {
      const int st = n % NST;
      const uint32_t ph = ((n / NST) - 1) & 1;
      const unsigned there = __ballot_sync(0xffffffffu, off >= 0) & 0xffu;
      step();
      const int64_t off1 = offset_of();
      if (n >= NST && !wait(&kempty[st], ph)) break;
      uint32_t pois = store(kr, smem + L::K_OFF + st * 2 * L::TERM, kinv_s + st * kTK);
      if (lane == 0) {
        valid_s[st * 8 + lw] = static_cast<uint8_t>(there);
        kpois_s[st * 8 + lw] = static_cast<uint8_t>(pois);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&kfull[st]);
      if (have) load(kr, off1, 0);
      if (n >= NST && !wait(&vempty[st], ph)) break;
      pois = store(vr, smem + L::V_OFF + st * 2 * L::TERM, vinv_s + st * kTK);
      if (lane == 0) vpois_s[st * 8 + lw] = static_cast<uint8_t>(pois);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&vfull[st]);
      if (have) load(vr, off1, vstep);
      off = off1;
    }
    if (bad) raise_flag(a.flags, KSH_FLAG_BAD_BLOCK);
  } else {
    // ---------------- rows ----------------
    set_regs_inc<216>();
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    int n = 0;
    bool ok = true;
    while (ok && next_piece(a, wk, &pc)) {
      const int R = pc.qt * kRows + tid;            // query row of the kv head
      const int node = R / a.g;
      const bool live = node < pc.nq;
      const bool any = pc.qt * kRows + warp * 32 < pc.nq * a.g;   // the warp has live rows
      auto row_at = [&]() -> int64_t {              // the row's place in q and out
        return ((pc.a0 + node) * a.hq + static_cast<int64_t>(pc.hk) * a.g + (R - node * a.g)) * D;
      };
      float acc[D];
      float qs, qinv;
      // Q: hi / lo terms into TMEM
      {
        const float* qp = a.q + row_at();
        uint32_t mx = 0;
#pragma unroll
        for (int c = 0; c < D; c += 4) {
          const float4 v = live ? *reinterpret_cast<const float4*>(qp + c) : make_float4(0.f, 0.f, 0.f, 0.f);
          acc[c] = v.x;
          acc[c + 1] = v.y;
          acc[c + 2] = v.z;
          acc[c + 3] = v.w;
          mx = max(max(mx, max(abs_bits(v.x), abs_bits(v.y))), max(abs_bits(v.z), abs_bits(v.w)));
        }
        row_scale(mx, &qs, &qinv);
#pragma unroll
        for (int c0 = 0; c0 < D; c0 += 64) {
          uint32_t hi[32], lo[32];
#pragma unroll
          for (int c = 0; c < 32; ++c) split2(acc[c0 + 2 * c] * qs, acc[c0 + 2 * c + 1] * qs, &hi[c], &lo[c]);
          tmem_st_32x32b_x32(lanes + L::Q_COL + c0 / 2, hi);
          tmem_st_32x32b_x32(lanes + L::Q_COL + D / 2 + c0 / 2, lo);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(qready);
      }
      auto word = [&](int i) -> uint64_t {          // nodes 64 i .. 64 i + 63 that the row sees
        if (a.mask) return live && i < a.words ? a.mask[(pc.a0 + node) * a.words + i] : 0;
        const int bits = node + 1 - 64 * i;
        return bits <= 0 ? 0 : bits >= 64 ? ~0ull : (1ull << bits) - 1;
      };
      const float cq = qinv * (a.scale * 1.44269504088896340736f);   // to powers of two
      float m = -INFINITY, mref = 0.0f, l = 0.0f;
#pragma unroll
      for (int c = 0; c < D; ++c) acc[c] = 0.0f;
      // of the tile whose P V is still to be added
      float corr_p = 1.0f, vs_p = 0.0f;
      bool rare_p = false;

      auto promote = [&](int mt, int tile) -> bool {
        if (!wait(&ofull[mt & 1], (mt >> 1) & 1)) return false;
        tc_fence_after();
        if (any) {
          const uint32_t o = lanes + L::O_COL + static_cast<uint32_t>(mt & 1) * D;
          if (__any_sync(0xffffffffu, corr_p != 1.0f)) {
#pragma unroll
            for (int c = 0; c < D; ++c) acc[c] *= corr_p;
          }
#pragma unroll
          for (int c0 = 0; c0 < D; c0 += 32) {
            float v[32];
            tmem_ld_32x32b_x32(o + c0, v);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 32; ++c) acc[c0 + c] = fmaf(v[c], vs_p, acc[c0 + c]);
          }
          if (rare_p) {        // V elements that are not finite: to the rows that see them
            for (uint64_t left = live ? rare_s[mt & 1][tid] : 0; left; left &= left - 1) {
              const int pos = tile * kTK + __ffsll(static_cast<long long>(left)) - 1;
              const int64_t at = key_offset(a, pc.s, pc.hk, pos, D);
              if (at < 0) continue;
              const float* vp = a.pool + at + a.hkv * a.bs * D;
#pragma unroll
              for (int c = 0; c < D; ++c) {
                const float x = vp[c];
                if (abs_bits(x) >= 0x7f800000u) acc[c] += x;
              }
            }
          }
          tc_fence_before();
        }
        return true;
      };

      for (int t = pc.t0; t < pc.t1; ++t, ++n) {
        const int st = n % NST, b = n & 1;
        if (!(ok = wait(&sfull[b], (n >> 1) & 1) && wait(&vfull[st], (n / NST) & 1))) break;
        tc_fence_after();
        const uint64_t kpois = *reinterpret_cast<const uint64_t*>(kpois_s + st * 8);
        float corr = 1.0f, vs = 0.0f;
        bool rare = false;
        if (any) {
          const uint32_t sc = lanes + L::S_COL + static_cast<uint32_t>(b) * kTK;
          uint64_t see = *reinterpret_cast<const uint64_t*>(valid_s + st * 8);
          const int n0 = t * kTK - pc.pre;           // node of the tile's first key
          if (n0 + kTK > 0) {                        // the tree's part of the keys
            if (n0 < 0) {
              see &= ((1ull << -n0) - 1) | (word(0) << -n0);
            } else {
              const int i = n0 >> 6, sh = n0 & 63;
              see &= sh ? (word(i) >> sh) | (word(i + 1) << (64 - sh)) : word(i);
            }
          }
          const uint64_t vpois = *reinterpret_cast<const uint64_t*>(vpois_s + st * 8);
          rare = vpois != 0;
          if (rare) rare_s[b][tid] = vpois & see;
          const bool hide = __any_sync(0xffffffffu, see != ~0ull);
          // 32 scores of the row at a time, read twice: registers hold the
          // accumulators
          float x[32];
          auto scores = [&](int h) {
            tmem_ld_32x32b_x32(sc + 32 * h, x);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              const float4 k4 = *reinterpret_cast<const float4*>(kinv_s + st * kTK + 32 * h + j);
              x[j] *= k4.x;
              x[j + 1] *= k4.y;
              x[j + 2] *= k4.z;
              x[j + 3] *= k4.w;
            }
            if (hide || kpois) {
              for (uint32_t left = static_cast<uint32_t>(kpois >> (32 * h)); left && live; left &= left - 1) {
                // K elements that are not finite went in as zeros
                const int j = __ffs(static_cast<int>(left)) - 1;
                const int64_t at = key_offset(a, pc.s, pc.hk, t * kTK + 32 * h + j, D);
                const float* qp = a.q + row_at();
                float add = 0.0f;
                if (at >= 0)
                  for (int c = 0; c < D; ++c) {
                    const float kx = a.pool[at + c];
                    if (abs_bits(kx) >= 0x7f800000u) add += qp[c] * kx;
                  }
#pragma unroll
                for (int e = 0; e < 32; ++e)
                  if (e == j) x[e] += add;
              }
              const uint32_t on = static_cast<uint32_t>(see >> (32 * h));
#pragma unroll
              for (int j = 0; j < 32; ++j) x[j] = (on >> j) & 1 ? x[j] : -INFINITY;
            }
          };
          float m4[4] = {m, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
          for (int h = 0; h < kTK / 32; ++h) {
            scores(h);
#pragma unroll
            for (int j = 0; j < 32; ++j) m4[j & 3] = fmaxf(m4[j & 3], x[j]);
          }
          m = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
          const float ref = m == -INFINITY ? 0.0f : m * cq;
          corr = l > 0.0f ? ex2(mref - ref) : 1.0f;
          mref = ref;
          // P, scaled per key by V's scale relative to the tile's largest
          float vm = fmaxf(vinv_s[st * kTK + lane], vinv_s[st * kTK + 32 + lane]);
          vm = fmaxf(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(vm))), 0x1p-100f);
          const float up = 32768.0f / vm;           // powers of two
          vs = vm * (1.0f / 32768.0f);
          float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
          for (int h = 0; h < kTK / 32; ++h) {
            scores(h);
            uint32_t pt[32];                        // hi pairs, then lo pairs, over the scores
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              const float4 v4 = *reinterpret_cast<const float4*>(vinv_s + st * kTK + 32 * h + j);
              const float p0 = ex2(fmaf(x[j], cq, -ref)), p1 = ex2(fmaf(x[j + 1], cq, -ref));
              const float p2 = ex2(fmaf(x[j + 2], cq, -ref)), p3 = ex2(fmaf(x[j + 3], cq, -ref));
              s4[0] += p0;
              s4[1] += p1;
              s4[2] += p2;
              s4[3] += p3;
              split2(p0 * (v4.x * up), p1 * (v4.y * up), &pt[j / 2], &pt[16 + j / 2]);
              split2(p2 * (v4.z * up), p3 * (v4.w * up), &pt[j / 2 + 1], &pt[16 + j / 2 + 1]);
            }
            tmem_st_32x32b_x32(sc + 32 * h, pt);
          }
          l = fmaf(l, corr, (s4[0] + s4[1]) + (s4[2] + s4[3]));
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&pready[b]);
          mbar_arrive(&kempty[st]);
          mbar_arrive(&vempty[st]);
        }
        if (t > pc.t0 && !(ok = promote(n - 1, t - 1))) break;
        corr_p = corr;
        vs_p = vs;
        rare_p = rare;
      }
      if (!ok || !(ok = promote(n - 1, pc.t1 - 1))) break;

      const bool whole = pc.t0 == 0 && pc.t1 == pc.ntiles;
      if (whole) {
        if (live) {
          const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
          float* op = a.out + row_at();
#pragma unroll
          for (int c = 0; c < D; c += 4) {
            float4 v = make_float4(acc[c] * inv, acc[c + 1] * inv, acc[c + 2] * inv, acc[c + 3] * inv);
            if (l == 0.0f) v = make_float4(0.f, 0.f, 0.f, 0.f);
            *reinterpret_cast<float4*>(op + c) = v;
          }
        }
      } else {
        float* part = a.part + (static_cast<int64_t>(blockIdx.x) * 2 + (pc.t0 > 0 ? 0 : 1)) * part_floats<D>();
        if (live) {
          part[tid] = m == -INFINITY ? -INFINITY : mref;
          part[kRows + tid] = l;
#pragma unroll
          for (int c = 0; c < D; c += 4)
            reinterpret_cast<float4*>(part + 2 * kRows)[(c / 4) * kRows + tid] =
                make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
        }
        if (pc.t0 == 0 && tid == 0) {              // the share's last piece: joined from here on
          const int64_t end = wk->u + (pc.ntiles - pc.t1);       // past the item's last unit
          cut_s.first = static_cast<int>(blockIdx.x);
          cut_s.last = static_cast<int>((end * G - 1) / U);
          cut_s.row0 = static_cast<int>(pc.a0);
          cut_s.rbase = pc.qt * kRows;
          cut_s.rows = min(kRows, pc.nq * a.g - pc.qt * kRows);
          cut_s.hk = pc.hk;
        }
      }
    }
  }
  __syncthreads();
  if (tid == 0) {
    if (*abort_flag) {
      raise_flag(a.flags, KSH_FLAG_TIMEOUT);
      cut_s.last = -1;
    }
    a.items[blockIdx.x] = cut_s;
  }
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, L::COLS);
  }
}

// Joins the pieces of an item cut between CTAs, in key order:
// M = max m, out = sum acc 2^(m - M) / sum l 2^(m - M).
constexpr int kMergeThreads = 256, kMergeChunks = 8;

template <int D>
__global__ void __launch_bounds__(kMergeThreads) tree_merge_kernel(TreeArgs a) {
  grid_dep_wait();
  grid_dep_launch();
  const SplitItem it = a.items[blockIdx.x];
  if (it.last < it.first) return;
  for (int i = blockIdx.y * kMergeThreads + threadIdx.x; i < kRows * (D / 4);
       i += kMergeThreads * kMergeChunks) {
    const int r = i % kRows, c4 = i / kRows;
    if (r >= it.rows) continue;
    const float* p0 = a.part + (static_cast<int64_t>(it.first) * 2 + 1) * part_floats<D>();
    auto piece = [&](int c) {
      return c == it.first ? p0 : a.part + static_cast<int64_t>(c) * 2 * part_floats<D>();
    };
    float M = -INFINITY;
    for (int c = it.first; c <= it.last; ++c) M = fmaxf(M, piece(c)[r]);
    const float ref = M == -INFINITY ? 0.0f : M;
    float L = 0.0f;
    float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = it.first; c <= it.last; ++c) {
      const float* p = piece(c);
      const float w = ex2(p[r] - ref);
      L = fmaf(p[kRows + r], w, L);
      const float4 v = reinterpret_cast<const float4*>(p + 2 * kRows)[c4 * kRows + r];
      A.x = fmaf(v.x, w, A.x);
      A.y = fmaf(v.y, w, A.y);
      A.z = fmaf(v.z, w, A.z);
      A.w = fmaf(v.w, w, A.w);
    }
    const int R = it.rbase + r, node = R / a.g;
    float* op = a.out + ((static_cast<int64_t>(it.row0) + node) * a.hq +
                         static_cast<int64_t>(it.hk) * a.g + (R - node * a.g)) * D;
    const float inv = 1.0f / L;
    float4 v = make_float4(A.x * inv, A.y * inv, A.z * inv, A.w * inv);
    if (L == 0.0f) v = make_float4(0.f, 0.f, 0.f, 0.f);
    reinterpret_cast<float4*>(op)[c4] = v;
  }
}

template <int D>
int launch_tree_tc(const TreeArgs& a, int grid, cudaStream_t st) {
  using L = TreeLayout<D>;
  auto kern = tree_attn_tc_kernel<D>;
  if (set_smem_optin(reinterpret_cast<const void*>(kern), L::BYTES) != KSH_OK) return KSH_ERR_CUDA;
  const int rc = launch(kern, dim3(static_cast<unsigned>(grid)), dim3(kTcThreads), L::BYTES, st, a);
  if (rc != KSH_OK || grid == 1) return rc;
  return launch(tree_merge_kernel<D>, dim3(static_cast<unsigned>(grid - 1), kMergeChunks),
                dim3(kMergeThreads), 0, st, a);
}

int64_t items_bytes() { return (static_cast<int64_t>(num_sms()) * sizeof(SplitItem) + 255) / 256 * 256; }

// Other head dimensions and unaligned tensors: one warp per (node, head), keys one after the other: any head dimension up
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
  if (num_seqs <= 0 || hq <= 0 || hkv <= 0 || hq % hkv != 0 || d <= 0 || max_nodes < 0) return 0;
  if (d != 64 && d != 128) return 256;
  const int64_t part = d == 64 ? part_floats<64>() : part_floats<128>();
  return items_bytes() + 2 * part * 4 * num_sms();
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
  const bool fast = (d == 64 || d == 128) && ((reinterpret_cast<uintptr_t>(pool) |
      reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  if (fast) {
    if (!workspace || workspace_bytes < ksh_tree_attention_workspace_size(num_seqs, hq, hkv, d, max_nodes))
      return KSH_ERR_WORKSPACE;
    if ((reinterpret_cast<uintptr_t>(workspace) & 255) != 0) return KSH_ERR_ALIGN;
    a.items = static_cast<SplitItem*>(workspace);
    a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + items_bytes());
    // no more CTAs than there can be tiles
    const int64_t tiles = std::max<int64_t>(1, (max_total_len + kTK - 1) / kTK);
    const int64_t qtiles = (max_nodes * a.g + kRows - 1) / kRows;
    const int grid = static_cast<int>(std::min<double>(
        num_sms(), static_cast<double>(num_seqs) * static_cast<double>(hkv) * static_cast<double>(qtiles) *
                       static_cast<double>(tiles)));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return d == 64 ? launch_tree_tc<64>(a, grid, st) : launch_tree_tc<128>(a, grid, st);
  }
  if (hq > 65535 || num_seqs > 65535) return KSH_ERR_UNSUPPORTED;
  return launch(tree_attn_simple_kernel,
                dim3(static_cast<unsigned>(max_nodes), static_cast<unsigned>(hq),
                     static_cast<unsigned>(num_seqs)),
                dim3(32), 0, static_cast<cudaStream_t>(stream), a);
}
