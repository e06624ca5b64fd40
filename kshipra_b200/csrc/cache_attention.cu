// Attention of a chunk of new tokens over the 16-bit paged cache.
//
// Sequence s has prefix[s] cached positions and brings n = q_start[s+1] -
// q_start[s] rows whose K/V stand at positions prefix .. prefix + n - 1.  Row i
// attends positions 0 .. prefix + i:
//     o = sum_j exp(q.k_j / sqrt(D) - m) v_j / sum_j exp(q.k_j / sqrt(D) - m)
// with the running maximum m.  q and o are fp32, K and V fp16 or bf16.
//
// Three kernels: calls whose sequences bring at most 16 rows (tokens x heads of a group)
// of head dimension 64 or 128, as decoding does, go to cache_attn_rows_kernel, others of
// these dimensions to cache_attn_tc_kernel, the rest to cache_attn_any_kernel.
//
// Head dimensions 64 and 128 (cache_attn_tc_kernel): K and V go to the tensor cores
// as they stand in the cache, TMA boxes of pool rows straight into the MMAs'
// operand layout.  q and P, which are fp32, go in as sums of 16-bit terms of the
// cache's type (fp16: two of 11 bits, q with a power of two per row; bf16: three of
// 8), so a product costs two or three MMAs and the result has fp32's accuracy
// (relative L2 error against 64 bits 3e-7 to 9e-7; the same in fp32 torch 8e-7 to
// 3.4e-6).  Rounding q and P to one 16-bit term each would cost 2^-9 to 2^-12.
//
// One persistent CTA per SM.  An item is (sequence, row tile of up to 128 rows =
// tokens x heads of a kv head, kv head); its 128-key tiles end at the last token's
// position, so masked tiles are not read.  All items' keys form one line that is cut
// into equal shares, one per CTA, so that uneven lengths leave no SM idle; an item
// cut between CTAs leaves its (m, l, acc) pieces in the workspace and
// cache_merge_kernel joins them in key order (the same bits in every run).  One
// token of a sequence is an item of few rows.  Warps of a CTA:
//   14, 15  K and V tiles into shared memory, and V's rows that not every query row
//           sees cleaned of what may stand in them
//   12, 13  MMAs, one warp for the even tiles and one for the odd: S = Q K^T (A = Q in
//           TMEM), O = P V (A = P in TMEM, over S)
//   0..7    rows: thread = query row and half of the tile's keys (up to 32 rows:
//           an eighth): softmax in 32 bits, P's terms into TMEM
//   8..11   sums: thread = query row: every tile's P V added into fp32 registers (a
//           long context added up inside the tensor core would lose low bits at each
//           step), results and pieces written
//
// What bounds it: with two terms a tile of 128 rows, 128 keys and D = 128 is 2.05 K
// tensor cycles, with three 3.07 K, and 64 KB of K and V, 2.3 to 2.9 K cycles of the
// SM's share of HBM.  Measured (back to back from a graph; in long runs the power limit
// holds the clock at 1.5 GHz and adds 10 to 15 %):
//   2048 tokens behind 4096, 32 / 8 heads of 128, fp16: 287 us, 600 TFLOP/s of attention
//   and twice that of MMAs; tensor pipe 66 % active.
//   3 sequences of up to 31000 keys with chunks of up to 200, bf16: 300 to 345 us; 19 % of
//   the tiles are of two sequences' single tokens, four rows of 128 in each.
//   24 sequences of up to 2000 keys, chunks of up to 301 among single tokens, 14 / 2
//   heads of 64, bf16: 91 to 117 us, of which its tiles' and items' cycles (33 tiles and
//   2.8 items an SM) explain 51 to 67.
//   A chunk of 2048 beside 63 single tokens behind 4096, 32 / 8 heads of 128, fp16: 400 to
//   440 us.
//   All eight of these kernels spill, not in the MMA warps' loops (fp16 52 to 72 bytes
//   stored, bf16 72 at D = 128 and 88 to 96 at D = 64).
//   (Decoding by this kernel, too: 64 sequences x 4096 keys, 32 / 8 heads of 128, 214 us,
//   bf16 265 to 315; tensor pipe 70 % active on rows that are mostly not there.)
// In a tile the longest chain is P V (1.0 K), its sums (1.2 K) and the waits between
// them (0.3 K each: with MMAs in flight an mbarrier's answer takes that long).  No
// faster, for the fp16 cases above: the sums in the row warps (10 % slower), sixteen row
// warps with a quarter each (15 %), one MMA warp (its waits add up to 1.5 K cycles a
// tile, 20 %), one warp for S and one for P V with Q in shared memory (30 %: the MMAs'
// reads then fill it), O in two halves (5 to 10 %); bf16 widened to fp16 in shared memory by
// four more warps and two terms (25 %).

#include <cuda_bf16.h>
#include <math.h>

#include <algorithm>
#include <cstring>
#include <type_traits>

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
  struct SplitItem* items;      // [gridDim.x] items cut at the end of a CTA's share
  float* part;                  // [gridDim.x][2] partial states
  int64_t total, num_blocks, num_layers, layer, hkv, hq, bs, max_blocks;
  int num_seqs, g, d, max_q;
  int npt;                      // rows of q (all heads of the group) per tile of 128
  int box;                      // pool rows per copy
  int item_cost;                // keys that an item's start counts for, beside its own
  float scale;
};

// An item whose first piece CTA `first` holds: joined from pieces first..last.
struct SplitItem {
  int32_t first, last;          // last < first: none
  int32_t row0;                 // q row of the tile's first token
  int32_t rows;                 // live rows
  int32_t hk;
  int32_t pad[3];
};

__device__ __forceinline__ float widen(__half x) { return __half2float(x); }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }

// What the probabilities (at most 1) of keys 0 .. last are scaled down by, and so their
// sum: the power of two that keeps the sum of their products with values as large as
// bf16's within fp32's range (fp16's leave 2^112 of room).  It costs no bits, except that
// products of V below 2^-118 times the number of keys may become subnormal.
template <typename T>
__device__ __forceinline__ float head_room(uint32_t last) {
  if (!std::is_same_v<T, __nv_bfloat16>) return 1.0f;
  return __uint_as_float((95u + static_cast<uint32_t>(__clz(static_cast<int>(last)))) << 23);   // 2^-ceil(log2(last + 1))
}

// Any head dimension up to 256 and any alignment: a CTA per (row, head), whose warps
// take 16 keys at a time each, four of them in flight, and join their states at the
// end.  VEC: elements a load takes, four where dimension and pool allow; PER: elements a
// lane has.  Bound by instructions and, with few rows, by a warp's trips to memory.  16 /
// 4 heads, fp16: one sequence x 540 keys 23 us with D = 96, 32 with D = 256 (a warp for
// all keys, one after the other: 525); 64 x 4096 keys 540 and 1180 (7000 and 7750; bf16 440
// and 1157), four sequences' chunks of 128 behind 1000 655 and 1070.  With two elements a
// load 25, 57, 510 and 3380, 740 and 2650; a group's heads side by side in the grid save
// nothing.  It is no kernel for long chunks, whose rows each read all of K and V: 2048
// tokens behind 4096, 32 / 8 heads, 23 to 25 ms at D = 96 and 43 to 46 at 256 (0.28 by the
// tiles at D = 128).
constexpr int kAnyWarps = 8, kAnyRun = 16, kAnyKeys = 4, kAnyMax = 256;

template <typename T, int VEC, int PER>
__global__ void __launch_bounds__(kAnyWarps * 32) cache_attn_any_kernel(CacheArgs a) {
  using Raw = std::conditional_t<VEC == 4, uint2, uint16_t>;
  constexpr int kLoads = PER / VEC;
  __shared__ float m_s[kAnyWarps], l_s[kAnyWarps], acc_s[kAnyWarps][kAnyMax];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int h = blockIdx.y;
  const int64_t row = blockIdx.x;
  grid_dep_wait();
  grid_dep_launch();
  const int64_t cap = a.max_blocks * a.bs;
  if (row == 0 && h == 0) {
    for (int s = tid; s < a.num_seqs; s += kAnyWarps * 32) {
      const int64_t a0 = a.q_start[s], n = a.q_start[s + 1] - a0;
      if (a0 < 0 || n < 0 || a0 + n > a.total || n > a.max_q || a.prefix[s] < 0 || max(a.prefix[s], 0) + max(n, int64_t(0)) > cap)
        raise_flag(a.flags, KSH_FLAG_BAD_LENGTH);
    }
  }
  int s = 0, past = a.num_seqs;                   // the last sequence that starts at or before the row
  while (past - s > 1) {
    const int mid = s + (past - s) / 2;
    if (a.q_start[mid] <= row)
      s = mid;
    else
      past = mid;
  }
  const int64_t i = row - a.q_start[s];
  if (i < 0 || i >= a.max_q || row >= a.q_start[s + 1]) return;
  const int d = a.d, hk = h / a.g;
  const int64_t end = min(static_cast<int64_t>(max(a.prefix[s], 0)) + i + 1, cap);
  const int32_t* const table = a.block_tables + static_cast<int64_t>(s) * a.max_blocks;
  const uint32_t bs = static_cast<uint32_t>(a.bs);
  const float* const q = a.q + (row * a.hq + h) * d;
  const T* const kpool = static_cast<const T*>(a.pool) + ((a.layer * 2) * a.hkv + hk) * a.bs * d + lane * VEC;
  const int64_t page = a.num_layers * 2 * a.hkv * a.bs * d, to_v = a.hkv * a.bs * d;
  float qv[PER], acc[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int c = (e / VEC * 32 + lane) * VEC + e % VEC;
    qv[e] = c < d ? q[c] * a.scale : 0.0f;
    acc[e] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  float room = head_room<T>(static_cast<uint32_t>(end - 1));
  bool bad = false;
  auto value = [](Raw r, int e) {
    uint16_t b;
    if constexpr (VEC == 4)
      b = static_cast<uint16_t>((e % 4 < 2 ? r.x : r.y) >> (e % 2 * 16));
    else
      b = r;
    T t;
    memcpy(&t, &b, 2);
    return widen(t);
  };
  for (int64_t p0 = warp * kAnyRun; p0 < end; p0 += kAnyWarps * kAnyRun) {
    // a lane finds one key's place
    int64_t mine = -1;
    if (lane < kAnyRun && p0 + lane < end) {
      const uint32_t pos = static_cast<uint32_t>(p0 + lane), b = pos / bs;   // below 2^32: two int32 lengths
      const int64_t blk = table[b];
      if (blk >= 0 && blk < a.num_blocks)
        mine = blk * page + static_cast<int64_t>(pos - b * bs) * d;
      else
        bad = true;
    }
    const int run = static_cast<int>(min(end - p0, static_cast<int64_t>(kAnyRun)));
#pragma unroll 1
    for (int u0 = 0; u0 < run; u0 += kAnyKeys) {
      Raw k[kAnyKeys][kLoads], v[kAnyKeys][kLoads];
      bool on[kAnyKeys];
#pragma unroll
      for (int u = 0; u < kAnyKeys; ++u) {
        const int64_t at = __shfl_sync(0xffffffffu, mine, u0 + u);
        on[u] = at >= 0;
#pragma unroll
        for (int e = 0; e < kLoads; ++e) {
          const bool there = on[u] && (e * 32 + lane) * VEC < d;
          k[u][e] = there ? *reinterpret_cast<const Raw*>(kpool + at + e * 32 * VEC) : Raw{};
          v[u][e] = there ? *reinterpret_cast<const Raw*>(kpool + at + to_v + e * 32 * VEC) : Raw{};
        }
      }
      float x[kAnyKeys];
#pragma unroll
      for (int u = 0; u < kAnyKeys; ++u) {
        x[u] = 0.0f;
#pragma unroll
        for (int e = 0; e < PER; ++e) x[u] = fmaf(qv[e], value(k[u][e / VEC], e), x[u]);
      }
      // four sums over the warp at once: a lane ends with that of key lane >> 3
      float y = lane & 16 ? x[2] : x[0], z = lane & 16 ? x[3] : x[1];
      y += __shfl_xor_sync(0xffffffffu, lane & 16 ? x[0] : x[2], 16);
      z += __shfl_xor_sync(0xffffffffu, lane & 16 ? x[1] : x[3], 16);
      const float w = __shfl_xor_sync(0xffffffffu, lane & 8 ? y : z, 8);
      y = (lane & 8 ? z : y) + w;
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
      float top = m;
#pragma unroll
      for (int u = 0; u < kAnyKeys; ++u) {
        x[u] = __shfl_sync(0xffffffffu, y, 8 * u);
        if (!on[u]) x[u] = -INFINITY;
        top = fmaxf(top, x[u]);
      }
      const float ref = top == -INFINITY ? 0.0f : top;
      if constexpr (PER == 8 && std::is_same_v<T, __nv_bfloat16>) {
        // made anew, as there is no register for it (64 x 4096 keys of 256 1157 us, held 1350)
        uint32_t last = static_cast<uint32_t>(end) - 1;
        asm volatile("" : "+r"(last));
        room = head_room<T>(last);
      }
      if (top > m) {
        const float corr = expf(m - ref);
        m = top;
        l *= corr;
#pragma unroll
        for (int e = 0; e < PER; ++e) acc[e] *= corr;
      }
#pragma unroll
      for (int u = 0; u < kAnyKeys; ++u) {
        x[u] = expf(x[u] - ref) * room;
        l += x[u];
      }
#pragma unroll
      for (int u = 0; u < kAnyKeys; ++u)
#pragma unroll
        for (int e = 0; e < PER; ++e) acc[e] = fmaf(x[u], value(v[u][e / VEC], e), acc[e]);
    }
  }
  if (bad) raise_flag(a.flags, KSH_FLAG_BAD_BLOCK);
  if (lane == 0) m_s[warp] = m, l_s[warp] = l;
#pragma unroll
  for (int e = 0; e < PER; ++e) acc_s[warp][(e / VEC * 32 + lane) * VEC + e % VEC] = acc[e];
  __syncthreads();
  if (tid >= d) return;
  float top = -INFINITY, sum = 0.0f, o = 0.0f;
#pragma unroll
  for (int w = 0; w < kAnyWarps; ++w) top = fmaxf(top, m_s[w]);
  const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
  for (int w = 0; w < kAnyWarps; ++w) {
    const float f = expf(m_s[w] - ref);
    sum = fmaf(l_s[w], f, sum);
    o = fmaf(acc_s[w][tid], f, o);
  }
  a.out[(row * a.hq + h) * d + tid] = sum == 0.0f ? 0.0f : o / sum;
}

template <typename T>
int launch_cache_any(const CacheArgs& a, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(a.total), static_cast<unsigned>(a.hq)), block(kAnyWarps * 32);
  auto go = [&](auto kern) { return launch(kern, grid, block, 0, st, a); };
  if (a.d % 4 == 0 && (reinterpret_cast<uintptr_t>(a.pool) & 7) == 0)
    return a.d <= 128 ? go(cache_attn_any_kernel<T, 4, 4>) : go(cache_attn_any_kernel<T, 4, 8>);
  return a.d <= 128 ? go(cache_attn_any_kernel<T, 1, 4>) : go(cache_attn_any_kernel<T, 1, 8>);
}

// ---------------------------------------------------------------------------
// Tensor cores
// ---------------------------------------------------------------------------

constexpr int kTK = 128;                 // keys per tile
constexpr int kRows = 128;               // query rows per tile (MMA M)
constexpr int kRowWarps = 8, kSumWarp = kRowWarps, kSumWarps = 4;
constexpr int kMmaWarp = kSumWarp + kSumWarps, kCopyWarp = kMmaWarp + 2;     // even and odd tiles; K and V
constexpr int kThreads = 32 * (kCopyWarp + 2);
// registers a thread, of 128 at launch: rows, sums, the other roles (the sums spill
// below 176, which costs 50 %)
constexpr int kRowRegs = 120, kSumRegs = 192, kRegs = 80;
// An item's start (its Q, an empty pipeline) takes about four tiles' time; counted so
// in the line, the CTAs with more items are not the last ones.  24 sequences of
// chunks and single tokens, D = 64, bf16: 91 us, 160 with 128 keys, 122 with 1024; counted
// and not, D = 128, fp16: a chunk of 2048 beside 63 single tokens behind 4096 400 to 440 us
// and 1010, one of 256 beside seven behind 8000 84 to 102 and 352.  It is left out of calls
// with fewer than four tiles an SM, by the host's bound (sequences x longest chunk x longest
// context, which a padded or captured call exceeds); measured there it would gain, too:
// 4 x 1000 keys with chunks of 30 16.4 us (left out 20.3), 4000 keys with a chunk of 20 22
// (27.6), eight chunks of 128 30 (57.7).
constexpr int kItemCost = 512;
constexpr int kMeta = 16;                // tiles whose notes are kept: more than the stages let run apart
// Tiles (pieces) that the row warps can be ahead of the sum warps, and more
constexpr int kRing = 4;
// floats of one partial state: m [128], l [128], acc [D / 4][128][4]
template <int D>
constexpr int64_t part_floats() { return 2 * kRows + static_cast<int64_t>(D) * kRows; }

// 16-bit terms of a query and of a probability: two of 11 bits, three of 8
template <typename T>
struct Kind {
  static constexpr bool kBf16 = false;
  static constexpr int TERMS = 2;
};
template <>
struct Kind<__nv_bfloat16> {
  static constexpr bool kBf16 = true;
  static constexpr int TERMS = 3;
};

template <int D, typename T>
struct CacheLayout {
  static constexpr bool LOW = Kind<T>::TERMS == 3;   // third terms stand in shared memory
  static constexpr int HALF = kTK * 128;             // bytes of 64 columns of a tile
  static constexpr int TILE = kTK * D * 2;
  // stages of K and of V; the third terms of Q and P (128 rows x D, 128 rows x 128 keys)
  static constexpr int NST = D == 128 ? (LOW ? 2 : 3) : (LOW ? 4 : 6);
  static constexpr int K_OFF = 0, V_OFF = NST * TILE, QLOW = V_OFF + NST * TILE, PLOW = QLOW + (LOW ? TILE : 0);
  // notes on a tile: range, four words of keys that are there, four of keys whose
  // V is not finite
  static constexpr int META = PLOW + (LOW ? 2 * HALF : 0), META_WORDS = 9;
  static constexpr int MAX = META + kMeta * META_WORDS * 4;       // row maxima of the halves [2][2][128]
  static constexpr int CORR = MAX + 4 * kRows * 4;                // what the sums are rescaled by [kRing][128]
  static constexpr int FIN = CORR + kRing * kRows * 4;            // a piece's reference and the halves' sums [kRing][3][128]
  static constexpr int FOLD = FIN + kRing * 3 * kRows * 4;        // 32 rows of O on their way to another warp
  static constexpr int BAR = FOLD + 32 * D * 4;
  static constexpr int NBAR = 5 * NST + 5 * 2 + 1;
  static constexpr int MISC = BAR + NBAR * 8;
  static constexpr int BYTES = MISC + 64 + 1024;
  // TMEM columns: two S, whose place P takes (16 keys: eight columns of hi and
  // eight of lo pairs), O, Q hi and lo (D / 2 each)
  static constexpr uint32_t S_COL = 0, O_COL = 2 * kTK, Q_COL = O_COL + D, COLS = 512;
  static_assert(Q_COL + D <= COLS, "TMEM columns");
  static_assert(BYTES <= 222 * 1024, "shared memory");
};
// words of a tile's notes
constexpr int kRange = 0, kThere = 1, kPois = 5;
// the range word: keys that all rows see | keys that are read << 8, and whether pages
// are missing
constexpr uint32_t kMissing = 1u << 16;

// One sequence's share of the work.
struct SeqWork {
  int64_t a0;
  int nq, pre, nqt;
  bool bad;                     // lengths that do not fit
};

__device__ __forceinline__ SeqWork seq_work(const CacheArgs& a, int s) {
  SeqWork w = {};
  const int64_t a0 = a.q_start[s], n = a.q_start[s + 1] - a0;
  const int pre = a.prefix[s];
  const int64_t cap = min(a.max_blocks * a.bs, static_cast<int64_t>(INT32_MAX - 2 * kTK - kItemCost));
  w.a0 = a0;
  w.bad = a0 < 0 || n < 0 || a0 + n > a.total || n > a.max_q || pre < 0 || max(pre, 0) + max(n, int64_t(0)) > cap;
  if (a0 < 0 || n <= 0 || a0 >= a.total) return w;
  w.nq = static_cast<int>(min(min(n, static_cast<int64_t>(a.max_q)), min(a.total - a0, cap)));
  w.pre = static_cast<int>(min(static_cast<int64_t>(max(pre, 0)), cap - w.nq));
  w.nqt = (w.nq + a.npt - 1) / a.npt;
  return w;
}
// The line's units are keys: an item counts those that its last row sees, and
// item_cost.  Units of the items of row tiles 0 .. qt - 1, and of all.
__device__ __forceinline__ int64_t units_before(const CacheArgs& a, const SeqWork& w, int qt) {
  return a.hkv * (static_cast<int64_t>(qt) * (w.pre + a.item_cost) + static_cast<int64_t>(a.npt) * qt * (qt + 1) / 2);
}
__device__ __forceinline__ int64_t units_of(const CacheArgs& a, const SeqWork& w) {
  return w.nqt == 0 ? 0 : units_before(a, w, w.nqt - 1) + a.hkv * (static_cast<int64_t>(w.pre) + w.nq + a.item_cost);
}

// (Out of line, as what is called from several roles or seldom: with all of it inline
// the code is 180 KB, and a role that comes to an item's start waits for instructions.)
// The items of one CTA's share [u0, u1) of the line, one after the other; tile t of
// the item that starts at u belongs to the share that holds u + t * kTK.  Each warp
// keeps its own walk in shared memory (registers are for the tiles).
struct Walk {
  SeqWork w;                    // of sequence s
  int64_t u, u0, u1;            // u: where the next item starts
  int s, qt, hk;
};
struct Piece {
  int64_t a0, u;                // of the sequence, of the item
  int s, hk, t0, t1, nq, pre, ntiles;
  int node0, keys, kmin;        // first token of the row tile; keys that any row sees, that all see
};

__device__ __forceinline__ bool next_piece(const CacheArgs& a, Walk* wk, Piece* p) {
  Walk k = *wk;
  bool found = false;
  while (!found && k.u < k.u1) {
    const int keys = k.w.pre + min(k.w.nq, (k.qt + 1) * a.npt);
    p->ntiles = (keys + kTK - 1) / kTK;
    p->t0 = k.u0 > k.u ? static_cast<int>((k.u0 - k.u + kTK - 1) / kTK) : 0;
    const int64_t to = (k.u1 - k.u + kTK - 1) / kTK;
    p->t1 = static_cast<int>(min(to, static_cast<int64_t>(p->ntiles)));
    p->a0 = k.w.a0;
    p->u = k.u;
    p->s = k.s;
    p->hk = k.hk;
    p->nq = k.w.nq;
    p->pre = k.w.pre;
    p->node0 = k.qt * a.npt;
    p->keys = keys;
    p->kmin = k.w.pre + p->node0 + 1;
    found = p->t0 < p->t1;
    k.u += keys + a.item_cost;
    if (++k.hk == static_cast<int>(a.hkv)) {
      k.hk = 0;
      if (++k.qt == k.w.nqt) {
        k.qt = 0;
        do {
          if (++k.s >= a.num_seqs) {
            k.u = k.u1;
            break;
          }
          k.w = seq_work(a, k.s);
        } while (k.w.nqt == 0);
      }
    }
  }
  __syncwarp();
  if ((threadIdx.x & 31) == 0) *wk = k;
  __syncwarp();
  return found;
}

// Up to 64 polls of an mbarrier's phase, as few instructions as a poll takes
// (the waiting warps share their schedulers with working ones).
__device__ __forceinline__ bool mbar_poll64(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u32 k;\n\t"
      "mov.u32 k, 64;\n\t"
      "POLL:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra DONE;\n\t"
      "sub.u32 k, k, 1;\n\t"
      "setp.ne.u32 q, k, 0;\n\t"
      "@q bra POLL;\n\t"
      "DONE:\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Whether a phase is over, without waiting: the answer is used some way on (a
// wait that need not wait takes 150 to 250 cycles).
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Of four barriers at once, a bit each.
__device__ __forceinline__ uint32_t mbar_test4(uint64_t* b0, uint32_t p0, uint64_t* b1, uint32_t p1, uint64_t* b2, uint32_t p2,
                                               uint64_t* b3, uint32_t p3) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q, r, s;\n\t.reg .u32 x;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 q, [%3], %4;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 r, [%5], %6;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 s, [%7], %8;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "selp.u32 x, 2, 0, q;\n\t"
      "or.b32 %0, %0, x;\n\t"
      "selp.u32 x, 4, 0, r;\n\t"
      "or.b32 %0, %0, x;\n\t"
      "selp.u32 x, 8, 0, s;\n\t"
      "or.b32 %0, %0, x;\n\t}"
      : "=&r"(r)
      : "r"(smem_u32(b0)), "r"(p0), "r"(smem_u32(b1)), "r"(p1), "r"(smem_u32(b2)), "r"(p2), "r"(smem_u32(b3)), "r"(p3)
      : "memory");
  return r;
}
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// largest |x|; NaN wins
__device__ __forceinline__ float amax3(float a, float b, float c) {
  float m;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(fabsf(a)), "f"(fabsf(b)), "f"(fabsf(c)));
  return m;
}
// Power of two that brings values up to `top` into [2^14, 2^15), and its
// inverse.
__device__ __forceinline__ void pow2_scale(float top, float* s, float* inv) {
  const int e = min(268 - static_cast<int>(abs_bits(top) >> 23), 253);
  *s = __uint_as_float(static_cast<uint32_t>(e) << 23);
  *inv = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
}
// two floats in one register pair: one instruction for both
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 f2(float x, float y) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpack(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
// x as a sum of pairs of 16-bit terms: fp16 hi (the leading 11 bits) + lo (the next
// 11), bf16 hi + lo + low (eight each).
template <typename T>
__device__ __forceinline__ void split(F2 xy, uint32_t* hi, uint32_t* lo, uint32_t* low) {
  constexpr uint32_t kKeep = Kind<T>::kBf16 ? 0xffff0000u : 0xffffe000u;
  auto cut = [](float2 f) {
    return make_float2(__uint_as_float(__float_as_uint(f.x) & kKeep), __uint_as_float(__float_as_uint(f.y) & kKeep));
  };
  auto less = [](F2 a, float2 b) { return fma2(f2(b.x, b.y), f2(-1.0f, -1.0f), a); };
  const float2 h = cut(unpack(xy));
  const F2 r = less(xy, h);
  if constexpr (Kind<T>::kBf16) {
    const float2 m = cut(unpack(r)), t = unpack(less(r, m));
    *hi = __byte_perm(__float_as_uint(h.x), __float_as_uint(h.y), 0x7632);
    *lo = __byte_perm(__float_as_uint(m.x), __float_as_uint(m.y), 0x7632);
    const __nv_bfloat162 b = __floats2bfloat162_rn(t.x, t.y);
    *low = *reinterpret_cast<const uint32_t*>(&b);
  } else {
    const float2 t = unpack(r);
    *hi = h2_bits(__floats2half2_rn(h.x, h.y));
    *lo = h2_bits(__floats2half2_rn(t.x, t.y));
  }
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float m;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The loads of v have arrived (v as operands: no use may move above this).
__device__ __forceinline__ void tmem_wait_ld(float (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]),
                 "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]),
                 "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]),
                 "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]),
                 "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]),
                 "+f"(v[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_wait_ld(float (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]),
                 "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]),
                 "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// Four lanes with element k of row i each (i = 0..3 in x[i], k = lane & 3) change
// to row k's elements in each lane.  Its own inverse.
__device__ __forceinline__ void exchange4(float4 (&x)[4], int lane) {
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (!(i & o)) {
        const bool up = lane & o;
        float4 s = up ? x[i] : x[i + o];
        s.x = __shfl_xor_sync(0xffffffffu, s.x, o);
        s.y = __shfl_xor_sync(0xffffffffu, s.y, o);
        s.z = __shfl_xor_sync(0xffffffffu, s.z, o);
        s.w = __shfl_xor_sync(0xffffffffu, s.w, o);
        if (up)
          x[i] = s;
        else
          x[i + o] = s;
      }
}
// Operand descriptor of V, 128-byte swizzle: a 128-byte row holds 64 of the N
// columns, 1024 bytes from eight keys to the next eight, HALF to the next 64
// columns.
__device__ __forceinline__ uint64_t desc_v(uint32_t smem_addr, uint32_t half) {
  return static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(half >> 4) << 16) |
         (static_cast<uint64_t>(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
template <int N>
__device__ __forceinline__ void set_regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void set_regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ void tmem_st_32x32b_x8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// The warps of the sums meet.
__device__ __forceinline__ void sums_sync() { asm volatile("bar.sync 5, 128;" ::: "memory"); }
// The two warps of 32 query rows (halves of the keys) meet.
__device__ __forceinline__ void pair_sync(int warp) {
  asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// Element offset of the K row of a sequence's `pos`, -1 without one.
__device__ __forceinline__ int64_t key_offset(const CacheArgs& a, int s, int hk, int pos, int D) {
  const int bs = static_cast<int>(a.bs), j = pos / bs;
  const int64_t blk = a.block_tables[static_cast<int64_t>(s) * a.max_blocks + j];
  if (blk < 0 || blk >= a.num_blocks) return -1;
  return ((((blk * a.num_layers + a.layer) * 2) * a.hkv + hk) * a.bs + (pos - j * bs)) * D;
}

// Byte of a tile's 16-byte chunk c (of D / 8) of a key's row.
template <int D>
__device__ __forceinline__ uint32_t tile_byte(int key, int c) {
  return (D == 128 ? static_cast<uint32_t>(c >> 3) * CacheLayout<D, __half>::HALF : 0u) + static_cast<uint32_t>(key) * 128 +
         (static_cast<uint32_t>((c & 7) ^ (key & 7)) << 4);
}

// A pair of 16-bit values: ones in the exponent, as sign bits.
template <typename T>
__device__ __forceinline__ uint32_t not_finite2(uint32_t w) {
  constexpr uint32_t e = Kind<T>::kBf16 ? 0x7f807f80u : 0x7c007c00u, one = Kind<T>::kBf16 ? 0x00800080u : 0x04000400u;
  return ((w & e) + one) & 0x80008000u;
}

// V rows that not every query row sees: those that are not there become zeros (a
// probability of 0 times what happens to stand in them must be 0), and so do
// elements that are not finite, whose keys are noted for the rows that see them.
template <int D, typename T>
__device__ __noinline__ void clean_v(uint8_t* tile, uint32_t* note, int lane) {
  constexpr int CPR = D / 8;
  const uint32_t range = note[kRange];
  const int hi = static_cast<int>((range >> 8) & 0xff), from = (range & kMissing) ? 0 : static_cast<int>(range & 0xff);
  if (lane < 4) note[kPois + lane] = 0;
  __syncwarp();
  for (int i = from * CPR + lane; i < kTK * CPR; i += 32) {
    const int key = i / CPR;
    uint4* at = reinterpret_cast<uint4*>(tile + tile_byte<D>(key, i % CPR));
    if (key >= hi || !((note[kThere + (key >> 5)] >> (key & 31)) & 1)) {
      *at = make_uint4(0, 0, 0, 0);
      continue;
    }
    uint4 v = *at;
    const uint32_t bx = not_finite2<T>(v.x), by = not_finite2<T>(v.y), bz = not_finite2<T>(v.z), bw = not_finite2<T>(v.w);
    if (bx | by | bz | bw) {
      auto keep = [](uint32_t w, uint32_t b) {
        return w & ~((b & 0x8000u ? 0xffffu : 0u) | (b & 0x80000000u ? 0xffff0000u : 0u));
      };
      *at = make_uint4(keep(v.x, bx), keep(v.y, by), keep(v.z, bz), keep(v.w, bw));
      atomicOr(note + kPois + (key >> 5), 1u << (key & 31));
    }
  }
  __syncwarp();
}

// Adds the elements that are not finite of tile t's noted V rows (keys from .. cnt - 1
// are a row's) to O, 16 columns at a time.
template <int D, typename T>
__device__ __forceinline__ void add_rare(const CacheArgs& a, const Piece& p, uint32_t oc, const uint32_t* note, int t, int from,
                                         int cnt) {
#pragma unroll 1
  for (int c0 = 0; c0 < D; c0 += 16) {
    float v[16];
    tmem_ld_32x32b_x16(oc + c0, v);
    tmem_wait_ld(v);
#pragma unroll 1
    for (int k = from; k < cnt; ++k) {
      if (!((note[kPois + (k >> 5)] >> (k & 31)) & 1)) continue;
      const int64_t at = key_offset(a, p.s, p.hk, t * kTK + k, D);
      if (at < 0) continue;
      const T* vp = static_cast<const T*>(a.pool) + at + a.hkv * a.bs * D + c0;
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        const float x = widen(vp[c]);
        v[c] += isfinite(x) ? 0.0f : x;
      }
    }
    uint32_t bits[16];
#pragma unroll
    for (int c = 0; c < 16; ++c) bits[c] = __float_as_uint(v[c]);
    __syncwarp();
    tmem_st_32x32b_x16(oc + c0, bits);
  }
  tmem_wait_st();
}

// BOX: copies by TMA, `box` pool rows each (block sizes that are multiples of
// eight); otherwise row by row.
template <int D, typename T, bool BOX>
__global__ void __launch_bounds__(kThreads, 1)
cache_attn_tc_kernel(CacheArgs a, const __grid_constant__ CUtensorMap map) {
  using L = CacheLayout<D, T>;
  constexpr int NST = L::NST;
  constexpr bool kBf16 = Kind<T>::kBf16;
  extern __shared__ uint8_t smem_raw[];
  // aligned by an offset, so that the compiler still sees shared memory (a
  // pointer rounded as an integer makes every access a generic one)
  uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint32_t* const notes = reinterpret_cast<uint32_t*>(smem + L::META);
  float* const max_s = reinterpret_cast<float*>(smem + L::MAX);
  float* const corr_s = reinterpret_cast<float*>(smem + L::CORR);
  float* const fin_s = reinterpret_cast<float*>(smem + L::FIN);
  float4* const fold_s = reinterpret_cast<float4*>(smem + L::FOLD);
  uint64_t* kraw = reinterpret_cast<uint64_t*>(smem + L::BAR);
  uint64_t* vraw = kraw + NST;
  uint64_t* vfull = vraw + NST;         // cleaned, or as it came
  uint64_t* kempty = vfull + NST;
  uint64_t* vempty = kempty + NST;
  uint64_t* sfull = vempty + NST;       // [2]
  uint64_t* pready = sfull + 2;         // [2]
  uint64_t* oempty = pready + 2;        // [2]: the MMA warps' tiles alternate
  uint64_t* qready = oempty + 2;        // [2]
  uint64_t* ofull = qready + 2;
  uint64_t* drain = ofull + 1;          // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  __shared__ int64_t scan_s[kThreads / 32];
  __shared__ Walk walk_s[kThreads / 32], start_s;
  __shared__ SplitItem cut_s;
  __shared__ Piece piece_s[kRowWarps + kSumWarps];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < NST; ++i) {
      mbar_init(&kraw[i], 1);
      mbar_init(&vraw[i], 1);
      mbar_init(&vfull[i], 1);
      mbar_init(&kempty[i], 1);
      mbar_init(&vempty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sfull[i], 1);
      mbar_init(&pready[i], kRowWarps);
      mbar_init(&oempty[i], kSumWarps);
      mbar_init(&qready[i], kRowWarps);
      mbar_init(&drain[i], 1);
    }
    mbar_init(ofull, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, L::COLS);
    tmem_relinquish();
  }
  if (BOX && warp == kCopyWarp && lane == 0) prefetch_tmap(&map);
  tc_fence_before();
  grid_dep_wait();

  // Q into L2 while the memory is idle: behind the K/V copies a row takes
  // thousands of cycles
  {
    const int64_t bytes = a.total * a.hq * D * 4, each = (bytes / gridDim.x + 15) & ~int64_t(15);
    const int64_t lo = each * blockIdx.x;
    if (lo < bytes)
      prefetch_range_l2(reinterpret_cast<const uint8_t*>(a.q) + lo,
                        static_cast<size_t>(min(each, bytes - lo)), tid, kThreads);
  }

  // The line: its length, and the place where this CTA's share starts.
  int64_t u0 = 0, q = 0, r = 0;                   // q units a CTA, one more for the first r
  {
    SeqWork w = {};
    int64_t v = 0, inc = 0, carry = 0;
    auto scan = [&](int b, bool first) {          // of kThreads sequences from b on
      w = {};
      v = 0;
      if (b + tid < a.num_seqs) {
        w = seq_work(a, b + tid);
        v = units_of(a, w);
        if (first && blockIdx.x == 0 && w.bad) raise_flag(a.flags, KSH_FLAG_BAD_LENGTH);
      }
      inc = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
      }
      __syncthreads();
      if (lane == 31) scan_s[warp] = inc;
      __syncthreads();
      const int warps = min(kThreads / 32, (a.num_seqs - b + 31) / 32);
      int64_t before = carry;
      for (int i = 0; i < warps; ++i) {
        if (i < warp) before += scan_s[i];
        carry += scan_s[i];
      }
      inc += before;
    };
    auto find = [&](int b) {
      if (v > 0 && u0 >= inc - v && u0 < inc) {
        const int64_t rel = u0 - (inc - v);
        int lo = 0, hi = w.nqt - 1;               // the last row tile that starts at or before rel
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (units_before(a, w, mid) <= rel)
            lo = mid;
          else
            hi = mid - 1;
        }
        const int64_t in = rel - units_before(a, w, lo);
        const int len = w.pre + min(w.nq, (lo + 1) * a.npt) + a.item_cost;
        const int hk = static_cast<int>((in >> 32) ? in / len : static_cast<uint32_t>(in) / static_cast<uint32_t>(len));
        start_s.w = w;
        start_s.s = b + tid;
        start_s.qt = lo;
        start_s.hk = hk;
        start_s.u = u0 - (in - static_cast<int64_t>(hk) * len);
        start_s.u0 = u0;
        start_s.u1 = u0 + q + (blockIdx.x < r ? 1 : 0);
      }
    };
    if (tid == 0) start_s.u = start_s.u1 = 0;
    for (int b = 0; b < a.num_seqs; b += kThreads) scan(b, true);
    // a share is a tile at least, so that every CTA between an item's first and last
    // has a piece of it
    const int64_t U = carry, G = max(min(static_cast<int64_t>(gridDim.x), U / kTK), int64_t(1));
    q = (U >> 32) ? U / G : static_cast<uint32_t>(U) / static_cast<uint32_t>(G);
    r = U - q * G;
    u0 = blockIdx.x * q + min(static_cast<int64_t>(blockIdx.x), r);
    if (blockIdx.x < G) {
      if (a.num_seqs <= kThreads) {
        find(0);
      } else {
        carry = 0;
        for (int b = 0; b < a.num_seqs; b += kThreads) scan(b, false), find(b);
      }
    }
  }
  __syncthreads();
  // the next kernel's CTAs may take TMEM before they wait for this one: not
  // before this CTA has its own
  grid_dep_launch();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  Walk* const wk = &walk_s[warp];
  // a row's token in the tile (rows are few: exact)
  const float per = 1.0f / static_cast<float>(a.g);
  auto token_of = [&](int R) { return static_cast<int>((static_cast<float>(R) + 0.5f) * per); };
  if (lane == 0) *wk = start_s;
  if (tid == 0) cut_s.first = 0, cut_s.last = -1;
  __syncwarp();
  Piece pc = {};

  // Bounded wait of the whole warp; gives up for all roles together, and from then on
  // at once: the row and sum warps go through their steps to the end all the same,
  // because they meet in them.
  bool dead = false;
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    if (dead) return false;
    bool ok = false;
    for (uint32_t i = 0; i < (1u << 16); ++i) {
      ok = mbar_poll64(bar, parity);
      if (ok || *abort_flag) break;
    }
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) {
      *abort_flag = 1;
      dead = true;
    }
    return ok;
  };

  // The same for three barriers, whose answers come together; *fourth: whether that
  // one's phase is over, too.
  auto wait3 = [&](uint64_t* b0, uint32_t p0, uint64_t* b1, uint32_t p1, uint64_t* b2, uint32_t p2, uint64_t* b3, uint32_t p3,
                   bool* fourth) -> bool {
    if (dead) return false;
    bool ok = false;
    uint32_t all = 0;
    for (uint32_t i = 0; i < (1u << 22); ++i) {
      all = mbar_test4(b0, p0, b1, p1, b2, p2, b3, p3);
      ok = (all & 7) == 7;
      if (ok || ((i & 63) == 63 && *abort_flag)) break;
    }
    ok = __all_sync(0xffffffffu, ok);
    *fourth = __all_sync(0xffffffffu, all & 8);
    if (!ok) {
      *abort_flag = 1;
      dead = true;
    }
    return ok;
  };

  if (warp >= kMmaWarp) {
  set_regs_dec<kRegs>();
  if (warp < kCopyWarp) {
    // ---------------- MMAs ----------------
    // One warp for the even tiles and one for the odd: a wait takes 300 cycles beside
    // MMAs even where there is nothing to wait for, and now the other warp's run
    // meanwhile.  S and P of a tile are one warp's, so they follow one another.
    constexpr uint32_t kType = kBf16 ? (1u << 7) | (1u << 10) : 0u;
    constexpr uint32_t id_s = idesc_f16_f32(kRows, kTK) | kType;
    constexpr uint32_t id_o = idesc_f16_f32(kRows, D) | kType | (1u << 16);   // B: keys along K
    const uint32_t kbase = smem_u32(smem + L::K_OFF), vbase = smem_u32(smem + L::V_OFF);
    const int b = warp - kMmaWarp;
    const uint32_t sp = tmem + L::S_COL + static_cast<uint32_t>(b) * kTK;
    int n = 0, seg = 0;
    bool ok = true;
    auto scores = [&](int m) {                      // S of tile m
      const int st = m % NST;
      if (elect_one()) {
        const uint64_t kd = desc_k_sw128(kbase + st * L::TILE);
        // the small terms first: the tensor core cuts low bits off at every step,
        // relative to the sum so far
        if (L::LOW) {
          const uint64_t qd = desc_k_sw128(smem_u32(smem + L::QLOW));
#pragma unroll 8
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t at = (k / 4) * (L::HALF / 16) + 2 * (k % 4);
            mma_f16(sp, qd + at, kd + at, id_s, k > 0 ? 1u : 0u);
          }
        }
        // (loops, not 32 instructions in a row: with as many descriptors in registers
        // the warp spills, and issues late)
#pragma unroll 1
        for (int term = 1; term >= 0; --term)
#pragma unroll 8
          for (int k = 0; k < D / 16; ++k)
            mma_f16_ts(sp, tmem + L::Q_COL + term * (D / 2) + 8 * k, kd + (k / 4) * (L::HALF / 16) + 2 * (k % 4), id_s,
                       (L::LOW || term == 0 || k > 0) ? 1u : 0u);
        mma_commit(&kempty[st]);
        mma_commit(&sfull[b]);
      }
      __syncwarp();
    };
    while (ok && next_piece(a, wk, &pc)) {
      const int first = n + ((n & 1) ^ b);          // the piece's first tile of this warp
      n += pc.t1 - pc.t0;
      if (first >= n) continue;
      if (!(ok = wait(&qready[b], seg & 1) && wait(&kraw[first % NST], (first / NST) & 1))) break;
      ++seg;
      tc_fence_after();
      scores(first);
#pragma unroll 1
      for (int m = first; m < n; m += 2) {
        const int st = m % NST;
        const bool more = m + 2 < n;
        uint64_t* const k2 = &kraw[(m + 2) % NST];
        const uint32_t k2p = ((m + 2) / NST) & 1;
        bool k_there;
        // m == 0: O is free, pready twice
        if (!(ok = wait3(&pready[b], (m >> 1) & 1, &vfull[st], (m / NST) & 1, m == 0 ? &pready[b] : &oempty[b ^ 1],
                         m == 0 ? 0 : ((m - 1) >> 1) & 1, k2, k2p, &k_there)))
          break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t vd = desc_v(vbase + st * L::TILE, L::HALF);
          if (L::LOW) {
            const uint64_t pd = desc_k_sw128(smem_u32(smem + L::PLOW));
#pragma unroll 8
            for (int k = 0; k < kTK / 16; ++k)
              mma_f16(tmem + L::O_COL, pd + (k / 4) * (L::HALF / 16) + 2 * (k % 4), vd + k * (2048 / 16), id_o, k > 0 ? 1u : 0u);
          }
#pragma unroll 1
          for (int term = 1; term >= 0; --term)
#pragma unroll 8
            for (int k = 0; k < kTK / 16; ++k)
              mma_f16_ts(tmem + L::O_COL, sp + 16 * k + 8 * term, vd + k * (2048 / 16), id_o,
                         (L::LOW || term == 0 || k > 0) ? 1u : 0u);
          mma_commit(&vempty[st]);
          mma_commit(ofull);
        }
        __syncwarp();
        // over P of this tile, which the products before it in the pipe have read
        if (more) {
          if (!k_there && !(ok = wait(k2, k2p))) break;
          tc_fence_after();
          scores(m + 2);
        }
      }
    }
    // nothing of this CTA's is in flight when its TMEM goes
    if (elect_one()) mma_commit(&drain[b]);
    __syncwarp();
    mbar_wait(&drain[b], 0);
  } else {
    // ---------------- K (one warp) / V (the next) rows into shared memory ----------------
    const int kv = warp - kCopyWarp;
    uint64_t* const freed = kv ? vempty : kempty;
    uint64_t* const raw = kv ? vraw : kraw;
    // V's tiles that every query row sees need no more than to arrive
    const bool clean = kv != 0;
    // A lane has the boxes lane & 15 of a tile (of the columns 64 (lane >> 4) on), or
    // its keys lane + 32 h: table column, place in the block and table entry, the
    // entry fetched one tile ahead.  A tile's lookups are additions.
    constexpr int NH = BOX ? 1 : 4;
    constexpr int kLag = NST > 2 ? 2 : 1;         // row by row: tiles on their way behind the one announced
    const int bs = static_cast<int>(a.bs), dj = kTK / bs, dr = kTK - dj * bs;
    const int box = BOX ? a.box : 1, nbox = kTK / box;
    const int mine = BOX ? (lane & 15) : lane;
    const bool use = !BOX || (mine < nbox && lane < D / 4);
    const uint32_t rows_per_block = static_cast<uint32_t>(a.num_layers * 2 * a.hkv * a.bs);
    bool have = next_piece(a, wk, &pc), bad = false;
    uint32_t cleans = 0;
    int t = 0, done = 0, sent = 0;                // sent: row by row, tiles that are announced
    uint32_t row0 = 0;                            // of the piece's layer and head in block 0
    const int32_t* table = nullptr;
    int col[NH], rest[NH], blk[NH];
    auto begin = [&]() {
      t = pc.t0;
      row0 = static_cast<uint32_t>(((a.layer * 2 + kv) * a.hkv + pc.hk) * a.bs);
      table = a.block_tables + static_cast<int64_t>(pc.s) * a.max_blocks;
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const int pos = t * kTK + (mine + 32 * h) * box;
        col[h] = pos / bs;
        rest[h] = pos - col[h] * bs;
      }
    };
    auto fetch = [&]() {
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        blk[h] = -1;
        if (have && use && t * kTK + (mine + 32 * h) * box < pc.keys) {
          blk[h] = table[col[h]];
          if (blk[h] < 0) blk[h] = INT32_MAX;
        }
      }
    };
    // V with rows that not every query row sees, once it has landed
    auto cleaned = [&](int i) {
      uint32_t* const note = notes + (i % kMeta) * L::META_WORDS;
      if ((note[kRange] & 0xff) < kTK || (note[kRange] & kMissing)) clean_v<D, T>(smem + L::V_OFF + (i % NST) * L::TILE, note, lane);
    };
    auto announce = [&]() {                       // row by row: a tile's copies have landed
      if (clean) cleaned(sent);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive((clean ? vfull : raw) + sent % NST);
      ++sent;
    };
    if (have) begin();
    fetch();
    while (have) {
      uint32_t row[NH], there[NH];
      bool lost = false;
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const bool on = blk[h] >= 0 && blk[h] < a.num_blocks;
        lost = lost || (blk[h] >= 0 && !on);
        row[h] = on ? static_cast<uint32_t>(blk[h]) * rows_per_block + row0 + static_cast<uint32_t>(rest[h]) : 0xffffffffu;
        there[h] = __ballot_sync(0xffffffffu, on);
      }
      lost = __any_sync(0xffffffffu, lost);
      bad = bad || lost;
      const int lo = min(max(pc.kmin - t * kTK, 0), kTK), hi = min(max(pc.keys - t * kTK, 0), kTK);
      if (++t < pc.t1) {
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          col[h] += dj;
          rest[h] += dr;
          if (rest[h] >= bs) rest[h] -= bs, ++col[h];
        }
      } else {
        have = next_piece(a, wk, &pc);
        if (have) begin();
      }
      fetch();
      const int st = done % NST;
      uint32_t* const note = notes + (done % kMeta) * L::META_WORDS;
      if (done >= NST && !wait(freed + st, ((done / NST) - 1) & 1)) break;
      // both warps the same
      uint32_t word = 0xffffffffu;
      if (BOX) {
        if (lost && lane < 4) {
          word = 0;
          for (int i = 0; i < 32; ++i) word |= ((there[0] >> ((32 * lane + i) / box)) & 1u) << i;
        }
      } else {
        word = lane == 0 ? there[0] : lane == 1 ? there[NH > 1 ? 1 : 0] : lane == 2 ? there[NH > 2 ? 2 : 0] : there[NH > 3 ? 3 : 0];
      }
      if (lane < 4) note[kThere + lane] = word;
      if (lane == 0) note[kRange] = static_cast<uint32_t>(lo) | static_cast<uint32_t>(hi) << 8 | (lost ? kMissing : 0);
      __syncwarp();
      uint8_t* const tile = smem + (kv ? L::V_OFF : L::K_OFF) + st * L::TILE;
      if (BOX) {
        const bool whole = lo == kTK && !lost;
        uint64_t* const bar = (clean && whole ? vfull : raw) + st;
        if (lane == 0) mbar_arrive_expect_tx(bar, static_cast<uint32_t>(__popc(there[0]) * box) * 128u);
        __syncwarp();
        if (row[0] != 0xffffffffu)
          tma_load_2d(tile + (lane >> 4) * L::HALF + mine * box * 128, &map, bar, (lane >> 4) * 64, static_cast<int32_t>(row[0]));
        if (clean && !whole) {
          // (vraw's phases count these tiles alone)
          mbar_wait(vraw + st, (cleans >> st) & 1);
          cleans ^= 1u << st;
          cleaned(done);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(vfull + st);
        }
      } else {
        constexpr int CPR = D / 8, RPI = 32 / CPR;    // rows an instruction covers
        const uint32_t dst = smem_u32(tile);
        const T* const src = static_cast<const T*>(a.pool);
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll 4
          for (int i = 0; i < 32 / RPI; ++i) {
            const int k = i * RPI + lane / CPR, c = lane % CPR;
            const uint32_t at = __shfl_sync(0xffffffffu, row[h], k);
            if (at != 0xffffffffu) copy16(dst + tile_byte<D>(32 * h + k, c), src + static_cast<int64_t>(at) * D + c * 8);
          }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (done - sent == kLag) {
          asm volatile("cp.async.wait_group %0;" ::"n"(kLag) : "memory");
          announce();
        }
      }
      ++done;
    }
    if (BOX) {
      // after an abort, let the copies still in flight land before the CTA exits
      if (*abort_flag)
        for (int i = max(0, done - NST); i < done; ++i) mbar_wait((clean ? vfull : raw) + i % NST, (i / NST) & 1);
    } else {
      asm volatile("cp.async.wait_all;" ::: "memory");
      while (sent < done) announce();
    }
    if (bad && lane == 0) raise_flag(a.flags, KSH_FLAG_BAD_BLOCK);
  }
  } else if (warp < kRowWarps) {
    // ---------------- rows ----------------
    set_regs_dec<kRowRegs>();
    const int hw = warp >> 2, row = (warp & 3) * 32 + lane;      // half, query row
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    constexpr int DH = D / 2;                       // columns of Q per half
    constexpr float kRefShift = kBf16 ? 8.0f : -6.0f;
    int n = 0, seg = 0;
    const Piece& ps = piece_s[warp];                // of the rare paths
    while (next_piece(a, wk, &pc)) {
      __syncwarp();
      if (lane == 0) piece_s[warp] = pc;
      __syncwarp();
      const int t0 = pc.t0, t1 = pc.t1;
      const int rows = min(a.npt, pc.nq - pc.node0) * a.g;       // live ones of the tile
      // Up to 32 rows (decoding) stand in the lanes four times, a quarter of the keys
      // each with its own softmax state: the chain of a tile is a quarter as long.
      const bool fold = rows <= 32;
      const int qrow = fold ? lane : row;
      const bool live = qrow < rows;
      // the row's place in q and out
      auto row_at = [&](int R) -> int64_t {
        const int node = token_of(R);
        return ((ps.a0 + ps.node0 + node) * a.hq + static_cast<int64_t>(ps.hk) * a.g + (R - node * a.g)) * D;
      };
      const bool some = fold || (warp & 3) * 32 < rows;
      float qinv = 1.0f;
      // Q: the half's columns as terms into TMEM (zeros for rows that are not live).
      // Four lanes load 64 bytes of a row, for the rows of the four, and exchange
      // them: one trip to memory, 1500 cycles beside the copies.
      {
        float4 v[DH / 4];
#pragma unroll
        for (int c = 0; c < DH / 4; ++c) v[c] = make_float4(0.f, 0.f, 0.f, 0.f);
        float qs = 1.0f;
        if (some) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int R = (qrow & ~3) + k;
            if (R < rows) {
              const float* qp = a.q + row_at(R) + hw * DH + (lane & 3) * 4;
#pragma unroll
              for (int c = 0; c < DH / 16; ++c) v[4 * c + k] = *reinterpret_cast<const float4*>(qp + 16 * c);
            }
          }
          float top = 0.0f;
#pragma unroll
          for (int c = 0; c < DH / 4; c += 4) {
            float4 x[4] = {v[c], v[c + 1], v[c + 2], v[c + 3]};
            exchange4(x, lane);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if (!kBf16) top = amax3(amax3(top, x[k].x, x[k].y), x[k].z, x[k].w);
              v[c + k] = x[k];
            }
          }
          if (!kBf16) {                              // the halves' maxima
            float* const mx = max_s + (n & 1) * 2 * kRows + row;
            mx[hw * kRows] = top;
            pair_sync(warp);
            pow2_scale(amax3(top, mx[(hw ^ 1) * kRows], 0.0f), &qs, &qinv);
            pair_sync(warp);
          }
        }
#pragma unroll
        for (int c = 0; c < DH / 4; c += 4) {
          uint32_t hi[8], lo[8], low[8];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            split<T>(mul2(f2(v[c + k].x, v[c + k].y), f2(qs, qs)), &hi[2 * k], &lo[2 * k], &low[2 * k]);
            split<T>(mul2(f2(v[c + k].z, v[c + k].w), f2(qs, qs)), &hi[2 * k + 1], &lo[2 * k + 1], &low[2 * k + 1]);
          }
          const int at = hw * DH + 4 * c;            // column
          if (L::LOW) {
            *reinterpret_cast<uint4*>(smem + L::QLOW + tile_byte<D>(row, at / 8)) = make_uint4(low[0], low[1], low[2], low[3]);
            *reinterpret_cast<uint4*>(smem + L::QLOW + tile_byte<D>(row, at / 8 + 1)) = make_uint4(low[4], low[5], low[6], low[7]);
          }
          tmem_st_32x32b_x8(lanes + L::Q_COL + at / 2, hi);
          tmem_st_32x32b_x8(lanes + L::Q_COL + (D + at) / 2, lo);
        }
        tmem_wait_st();
        if (L::LOW) fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {                            // to the MMA warps that have tiles of the piece
          mbar_arrive(&qready[n & 1]);
          if (t1 - t0 > 1) mbar_arrive(&qready[(n & 1) ^ 1]);
        }
      }
      const float cq = qinv * (a.scale * 1.44269504088896340736f);   // to powers of two
      if (!some) {
        // no row of the warp's is live (Q, and so S and P, are zeros): it only keeps step
#pragma unroll 1
        for (int t = t0; t < t1; ++t, ++n) {
          wait(&sfull[n & 1], (n >> 1) & 1);
          // (bf16: in step with O, as the warps with rows are)
          if (L::LOW && n > 0) wait(ofull, (n - 1) & 1);
          if (lane == 0) mbar_arrive(&pready[n & 1]);
        }
        ++seg;
        continue;
      }
      const int limit = live ? pc.pre + pc.node0 + token_of(qrow) : -1;   // the last key that the row sees
      // running state: the reference that the sums stand at (in powers of two;
      // it follows the maximum once that is 2^8 above it, so most tiles
      // rescale nothing), the half's sum
      float mref = -INFINITY, l = 0.0f;
      const float room = head_room<T>(static_cast<uint32_t>(pc.keys - 1));      // the same for all pieces of an item
      bool s_there = false;                         // seen a tile ahead
      if (fold) {
        const int part = warp & 3;                   // the keys 32 part on are the pair's
#pragma unroll 1
        for (int t = t0; t < t1; ++t, ++n) {
          const int b = n & 1;
          if (!__all_sync(0xffffffffu, s_there)) wait(&sfull[b], (n >> 1) & 1);
          tc_fence_after();
          const uint32_t sb = lanes + L::S_COL + static_cast<uint32_t>(b) * kTK, own = sb + 32 * part + 16 * hw;
          float x[16];
          tmem_ld_32x32b_x16(own, x);
          float corr = 1.0f;
          const uint32_t* const note = notes + (n % kMeta) * L::META_WORDS;
          const bool special = (t + 1) * kTK > pc.kmin || (*const_cast<const volatile uint32_t*>(note + kRange) & kMissing);
          tmem_wait_ld(x);
          if (__builtin_expect(special, 0)) {
            const int k = limit + 1 - t * kTK - 32 * part;
            const uint32_t seen = (note[kThere + part] & (k >= 32 ? 0xffffffffu : k <= 0 ? 0u : (1u << k) - 1)) >> (16 * hw);
#pragma unroll
            for (int j = 0; j < 16; ++j) x[j] = (seen >> j) & 1 ? x[j] : -INFINITY;
          }
          float m = max3(x[0], x[1], x[2]);
#pragma unroll
          for (int j = 3; j + 1 < 16; j += 2) m = max3(m, x[j], x[j + 1]);
          float* const mx = max_s + (n & 1) * 2 * kRows + row;
          mx[hw * kRows] = fmaxf(m, x[15]);
          pair_sync(warp);
          const float mc = fmaxf(mx[0], mx[kRows]) * cq;
          if (mc > mref + 8.0f) {
            corr = ex2(mref - mc);
            mref = mc;
          }
          const float ref = mref == -INFINITY ? 0.0f : mref + kRefShift;
          const F2 nref = f2(-ref, -ref), c2 = f2(cq, cq);
          F2 s2 = f2(0.f, 0.f);
          if (hw == 0) corr_s[(n % kRing) * kRows + row] = corr;
          const bool low_free = L::LOW && n > 0 && mbar_test(ofull, (n - 1) & 1);
          s_there = t + 1 < t1 && mbar_test(&sfull[b ^ 1], ((n + 1) >> 1) & 1);
          uint32_t pt[16], low[8];
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            const float2 e = unpack(fma2(f2(x[j], x[j + 1]), c2, nref));
            F2 p = f2(ex2(e.x), ex2(e.y));
            if (kBf16) p = mul2(p, f2(room, room));
            s2 = add2(s2, p);
            split<T>(p, &pt[j / 2], &pt[j / 2 + 8], &low[j / 2]);
          }
          tmem_st_32x32b_x16(own, pt);
          // zeros for the other quarters' keys
#pragma unroll
          for (int j = 0; j < 16; ++j) pt[j] = 0;
#pragma unroll 1
          for (int g = 4 * hw; g < 4 * hw + 4; ++g)
            if ((g >> 1) != part) tmem_st_32x32b_x16(sb + 16 * g, pt);
          const float2 sum = unpack(s2);
          l = fmaf(l, corr, sum.x + sum.y);
          if (t + 1 == t1) {
            float* const fin = fin_s + (seg % kRing) * 3 * kRows + row;
            fin[hw * kRows] = l;
            if (hw == 0) fin[2 * kRows] = mref;
          }
          if constexpr (L::LOW) {
            if (n > 0 && !__all_sync(0xffffffffu, low_free)) wait(ofull, (n - 1) & 1);
            uint8_t* const ps = smem + L::PLOW;
            if (t == t0)                             // they stay zeros for the rest of the piece
              for (int c = 8 * hw; c < 8 * hw + 8; ++c)
                if ((c >> 2) != part) *reinterpret_cast<uint4*>(ps + tile_byte<kTK>(row, c)) = make_uint4(0, 0, 0, 0);
            const int c = 4 * part + 2 * hw;
            *reinterpret_cast<uint4*>(ps + tile_byte<kTK>(row, c)) = make_uint4(low[0], low[1], low[2], low[3]);
            *reinterpret_cast<uint4*>(ps + tile_byte<kTK>(row, c + 1)) = make_uint4(low[4], low[5], low[6], low[7]);
            fence_proxy_async_smem();
          }
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&pready[b]);
        }
        ++seg;
        continue;
      }
#pragma unroll 1
      for (int t = t0; t < t1; ++t, ++n) {
        const int b = n & 1;
        if (!__all_sync(0xffffffffu, s_there)) wait(&sfull[b], (n >> 1) & 1);
        tc_fence_after();
        const uint32_t sc = lanes + L::S_COL + static_cast<uint32_t>(b) * kTK + 64 * hw;   // the half's scores
        float xa[32], xb[32];
        tmem_ld_32x32b_x32(sc, xa);
        tmem_ld_32x32b_x32(sc + 32, xb);
        float corr = 1.0f;
        const uint32_t* const note = notes + (n % kMeta) * L::META_WORDS;
        const bool special = (t + 1) * kTK > pc.kmin || (*const_cast<const volatile uint32_t*>(note + kRange) & kMissing);
        tmem_wait_ld(xa);
        tmem_wait_ld(xb);
        if (__builtin_expect(special, 0)) {
          const int cnt = limit + 1 - t * kTK;     // keys of the tile that come before the row's end
          auto seen = [&](int i) -> uint32_t {
            const int k = cnt - 32 * i;
            return note[kThere + i] & (k >= 32 ? 0xffffffffu : k <= 0 ? 0u : (1u << k) - 1);
          };
          const uint32_t wa = seen(2 * hw), wb = seen(2 * hw + 1);
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            xa[j] = (wa >> j) & 1 ? xa[j] : -INFINITY;
            xb[j] = (wb >> j) & 1 ? xb[j] : -INFINITY;
          }
        }
        float m0 = max3(xa[0], xa[1], xa[2]), m1 = max3(xb[0], xb[1], xb[2]);
#pragma unroll
        for (int j = 3; j + 1 < 32; j += 2) {
          m0 = max3(m0, xa[j], xa[j + 1]);
          m1 = max3(m1, xb[j], xb[j + 1]);
        }
        const float m = max3(m0, m1, fmaxf(xa[31], xb[31]));
        // both halves take the whole row's maximum
        float* const mx = max_s + (n & 1) * 2 * kRows + row;
        mx[hw * kRows] = m;
        pair_sync(warp);
        const float mc = fmaxf(m, mx[(hw ^ 1) * kRows]) * cq;
        if (mc > mref + 8.0f) {
          corr = ex2(mref - mc);
          mref = mc;
        }
        // P = 2^(x c - ref): up to 2^14 in fp16 terms, which keeps them above fp16's
        // smallest; up to 1 in bf16, times head_room, as V may be as large as fp32
        const float ref = mref == -INFINITY ? 0.0f : mref + kRefShift;
        const F2 nref = f2(-ref, -ref), c2 = f2(cq, cq);
        F2 s2[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
        uint32_t low[L::LOW ? 32 : 1];
        const bool low_free = L::LOW && n > 0 && mbar_test(ofull, (n - 1) & 1);
        auto probs = [&](const float (&x)[32], int j0, int group) {    // 16 keys
          uint32_t pt[16];
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            const float2 e = unpack(fma2(f2(x[j0 + j], x[j0 + j + 1]), c2, nref));
            F2 p = f2(ex2(e.x), ex2(e.y));
            if (kBf16) p = mul2(p, f2(room, room));
            s2[(j >> 1) & 1] = add2(s2[(j >> 1) & 1], p);
            split<T>(p, &pt[j / 2], &pt[j / 2 + 8], &low[L::LOW ? 8 * group + j / 2 : 0]);
          }
          tmem_st_32x32b_x16(sc + 16 * group, pt);
        };
        if (hw == 0) corr_s[(n % kRing) * kRows + row] = corr;
        probs(xa, 0, 0);
        probs(xa, 16, 1);
        probs(xb, 0, 2);
        s_there = t + 1 < t1 && mbar_test(&sfull[b ^ 1], ((n + 1) >> 1) & 1);
        probs(xb, 16, 3);
        const float2 sa = unpack(s2[0]), sb = unpack(s2[1]);
        l = fmaf(l, corr, (sa.x + sa.y) + (sb.x + sb.y));
        if (t + 1 == t1) {
          float* const fin = fin_s + (seg % kRing) * 3 * kRows + row;
          fin[hw * kRows] = l;
          if (hw == 0) fin[2 * kRows] = mref;
        }
        if constexpr (L::LOW) {                      // where the tile before's third terms have been read
          if (n > 0 && !__all_sync(0xffffffffu, low_free)) wait(ofull, (n - 1) & 1);
#pragma unroll
          for (int c = 0; c < 8; ++c)
            *reinterpret_cast<uint4*>(smem + L::PLOW + tile_byte<kTK>(row, 8 * hw + c)) =
                make_uint4(low[4 * c], low[4 * c + 1], low[4 * c + 2], low[4 * c + 3]);
          fence_proxy_async_smem();
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&pready[b]);
      }
      ++seg;
    }
  } else {
    // ---------------- sums ----------------
    // Every tile's P V added into fp32 registers (a long context added up inside the
    // tensor core would lose low bits at each step); a thread has a row.
    set_regs_inc<kSumRegs>();
    const int row = (warp & 3) * 32 + lane;
    const uint32_t oc = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + L::O_COL;
    int n = 0, seg = 0;
    const Piece& ps = piece_s[kRowWarps + (warp & 3)];
    while (next_piece(a, wk, &pc)) {
      __syncwarp();
      if (lane == 0) piece_s[kRowWarps + (warp & 3)] = pc;
      __syncwarp();
      const int t0 = pc.t0, t1 = pc.t1;
      const int rows = min(a.npt, pc.nq - pc.node0) * a.g;
      const bool fold = rows <= 32;
      const int part = warp & 3, qrow = fold ? lane : row;
      const bool live = qrow < rows, some = fold || part * 32 < rows;
      auto row_at = [&](int R) -> int64_t {
        const int node = token_of(R);
        return ((ps.a0 + ps.node0 + node) * a.hq + static_cast<int64_t>(ps.hk) * a.g + (R - node * a.g)) * D;
      };
      F2 acc[D / 2];
#pragma unroll
      for (int c = 0; c < D / 2; ++c) acc[c] = f2(0.f, 0.f);
#pragma unroll 1
      for (int t = t0; t < t1; ++t, ++n) {
        wait(ofull, n & 1);
        const uint32_t* const note = notes + (n % kMeta) * L::META_WORDS;
        if (some) {
          tc_fence_after();
          const float corr = corr_s[(n % kRing) * kRows + row];
          if (__builtin_expect((t + 1) * kTK > pc.kmin || (note[kRange] & kMissing), 0)) {
            // V elements that are not finite went in as zeros: to the rows that see them
            if (note[kPois] | note[kPois + 1] | note[kPois + 2] | note[kPois + 3])
              add_rare<D, T>(a, ps, oc, note, t, fold ? 32 * part : 0,
                             live ? min(pc.pre + pc.node0 + token_of(qrow) + 1 - t * kTK, fold ? 32 * part + 32 : kTK) : 0);
          }
          if (__any_sync(0xffffffffu, corr != 1.0f)) {
#pragma unroll
            for (int c = 0; c < D / 2; ++c) acc[c] = mul2(acc[c], f2(corr, corr));
          }
          constexpr int C = 32;                      // columns a load, as registers allow
          float v[C];
#pragma unroll
          for (int i = 0; i < D; i += C) {
            tmem_ld_32x32b_x32(oc + i, v);
            tmem_wait_ld(v);
#pragma unroll
            for (int c = 0; c < C / 2; ++c) {
              const F2 x = f2(v[2 * c], v[2 * c + 1]);
              acc[i / 2 + c] = add2(acc[i / 2 + c], x);
            }
          }
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&oempty[n & 1]);
      }
      const float* const fin = fin_s + (seg % kRing) * 3 * kRows + row;
      ++seg;
      if (!some) continue;
      float l = fin[0] + fin[kRows], ref = fin[2 * kRows];
      if (fold) {
        // the quarters' states, joined like an item's pieces
        const float* const all = fin - row + lane;
        float top = all[2 * kRows];
#pragma unroll
        for (int k = 1; k < 4; ++k) top = fmaxf(top, all[2 * kRows + 32 * k]);
        const float at = top == -INFINITY ? 0.0f : top, mine = ex2(ref - at);
        l = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) l = fmaf(all[32 * k] + all[kRows + 32 * k], ex2(all[2 * kRows + 32 * k] - at), l);
        ref = top;
#pragma unroll
        for (int c = 0; c < D / 2; ++c) acc[c] = mul2(acc[c], f2(mine, mine));
#pragma unroll 1
        for (int k = 1; k < 4; ++k) {
          if (part == k) {
#pragma unroll
            for (int c = 0; c < D / 4; ++c) {
              const float2 p = unpack(acc[2 * c]), u = unpack(acc[2 * c + 1]);
              fold_s[c * 32 + lane] = make_float4(p.x, p.y, u.x, u.y);
            }
          }
          sums_sync();
          if (part == 0) {
#pragma unroll
            for (int c = 0; c < D / 4; ++c) {
              const float4 v = fold_s[c * 32 + lane];
              acc[2 * c] = add2(acc[2 * c], f2(v.x, v.y));
              acc[2 * c + 1] = add2(acc[2 * c + 1], f2(v.z, v.w));
            }
          }
          sums_sync();
        }
        if (part != 0) continue;
      }
      if (t0 == 0 && t1 == ps.ntiles) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        if (live) {
          float* op = a.out + row_at(qrow);
#pragma unroll
          for (int c = 0; c < D; c += 4) {
            const float2 p = unpack(mul2(acc[c / 2], f2(inv, inv))), u = unpack(mul2(acc[c / 2 + 1], f2(inv, inv)));
            *reinterpret_cast<float4*>(op + c) = make_float4(p.x, p.y, u.x, u.y);
          }
        }
      } else {
        float* state = a.part + (static_cast<int64_t>(blockIdx.x) * 2 + (t0 > 0 ? 0 : 1)) * part_floats<D>();
        if (live) {
          state[qrow] = ref;
          state[kRows + qrow] = l;
#pragma unroll
          for (int c = 0; c < D; c += 4) {
            const float2 p = unpack(acc[c / 2]), u = unpack(acc[c / 2 + 1]);
            reinterpret_cast<float4*>(state + 2 * kRows)[c / 4 * kRows + qrow] = make_float4(p.x, p.y, u.x, u.y);
          }
        }
        if (t0 == 0 && warp == kSumWarp && lane == 0) {                 // the share's last piece: joined from here on
          const int64_t x = ps.u + static_cast<int64_t>(ps.ntiles - 1) * kTK;   // the item's last tile
          cut_s.first = static_cast<int>(blockIdx.x);
          cut_s.last = static_cast<int>(x < r * (q + 1) ? x / (q + 1) : r + (x - r * (q + 1)) / q);
          cut_s.row0 = static_cast<int>(ps.a0 + ps.node0);
          cut_s.rows = rows;
          cut_s.hk = ps.hk;
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
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, L::COLS);
  }
}

// Joins the pieces of an item cut between CTAs, in key order:
// M = max m, out = sum acc 2^(m - M) / sum l 2^(m - M), in one pass over the
// pieces with the running M, two at a time.
constexpr int kMergeThreads = 256, kMergeChunks = 16, kMergePieces = 2;

template <int D>
__global__ void __launch_bounds__(kMergeThreads) cache_merge_kernel(CacheArgs a) {
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
    float M = -INFINITY, L = 0.0f;
    float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c0 = it.first; c0 <= it.last; c0 += kMergePieces) {
      float m[kMergePieces], l[kMergePieces];
      float4 v[kMergePieces];
#pragma unroll
      for (int u = 0; u < kMergePieces; ++u) {
        const float* p = piece(min(c0 + u, it.last));
        m[u] = p[r];
        l[u] = p[kRows + r];
        v[u] = reinterpret_cast<const float4*>(p + 2 * kRows)[c4 * kRows + r];
      }
      float top = M;
#pragma unroll
      for (int u = 0; u < kMergePieces; ++u) top = fmaxf(top, m[u]);
      const float ref = top == -INFINITY ? 0.0f : top;
      const float w0 = ex2(M - ref);
      M = top;
      L *= w0;
      A = make_float4(A.x * w0, A.y * w0, A.z * w0, A.w * w0);
#pragma unroll
      for (int u = 0; u < kMergePieces; ++u) {
        if (c0 + u > it.last) break;
        const float w = ex2(m[u] - ref);
        L = fmaf(l[u], w, L);
        A.x = fmaf(v[u].x, w, A.x);
        A.y = fmaf(v[u].y, w, A.y);
        A.z = fmaf(v[u].z, w, A.z);
        A.w = fmaf(v[u].w, w, A.w);
      }
    }
    const int node = r / a.g;
    float* op = a.out + ((static_cast<int64_t>(it.row0) + node) * a.hq +
                         static_cast<int64_t>(it.hk) * a.g + (r - node * a.g)) * D;
    const float inv = 1.0f / L;
    float4 v = make_float4(A.x * inv, A.y * inv, A.z * inv, A.w * inv);
    if (L == 0.0f) v = make_float4(0.f, 0.f, 0.f, 0.f);
    reinterpret_cast<float4*>(op)[c4] = v;
  }
}

template <int D, typename T, bool BOX>
int launch_cache_tc(const CacheArgs& a, const CUtensorMap& map, int grid, cudaStream_t st) {
  using L = CacheLayout<D, T>;
  auto kern = cache_attn_tc_kernel<D, T, BOX>;
  if (set_smem_optin(reinterpret_cast<const void*>(kern), L::BYTES) != KSH_OK) return KSH_ERR_CUDA;
  const int rc = launch(kern, dim3(static_cast<unsigned>(grid)), dim3(kThreads), L::BYTES, st, a, map);
  if (rc != KSH_OK || grid == 1) return rc;
  return launch(cache_merge_kernel<D>, dim3(static_cast<unsigned>(grid - 1), kMergeChunks),
                dim3(kMergeThreads), 0, st, a);
}

template <int D, typename T>
int launch_cache_tc(CacheArgs& a, int grid, cudaStream_t st) {
  CUtensorMap map = {};
  if (a.bs % 8 != 0) return launch_cache_tc<D, T, false>(a, map, grid, st);
  a.box = 8;
  while (a.box < kTK && a.bs % (2 * a.box) == 0) a.box *= 2;
  const uint64_t rows = static_cast<uint64_t>(a.num_blocks) * a.num_layers * 2 * a.hkv * a.bs;
  if (!make_tensor_map_2d(&map, CU_TENSOR_MAP_DATA_TYPE_UINT16, a.pool, D, rows, D * 2, 64, static_cast<uint32_t>(a.box),
                          CU_TENSOR_MAP_SWIZZLE_128B))
    return KSH_ERR_CUDA;
  return launch_cache_tc<D, T, true>(a, map, grid, st);
}

// ---------------------------------------------------------------------------
// Few rows (decoding): up to 16 rows of q, all heads of a group, a sequence
// ---------------------------------------------------------------------------
// The tiles above do their products for 128 rows, however few there are.  Here a warp
// works alone: 16 keys of a (sequence, kv head) a step, K and V by cp.async into its own
// ring in shared memory, S^T = K Q^T and O^T = V^T P^T as 16 x 8 x 16 products of eight
// rows (q's terms in registers, P's transposed by movmatrix), each step's P V added in
// fp32.  No warp waits for another.  The line of all items' steps is cut into equal
// shares, one per warp, and cache_rows_merge_kernel joins the pieces in key order.
// HBM bound where many sequences of 128 decode.  us, and by cache_attn_tc_kernel: 64
// sequences x 4096 keys, 32 / 8 heads of 128, fp16 (1.08 GB) 172 (214), 97 % of measured HBM,
// tensor pipe 20 % active; bf16 170 (294); 128 / 8 heads 201 (248), four tokens each 199 (233;
// bf16 247), pages of ten tokens 170 (422); 256 sequences x 300 keys 65 (158), 4 x 1000 15 (27).
// Not HBM bound: 64 x 4096, 14 / 2 heads of 64 (134 MB, 21 us of HBM) 38 to 40 (60): a step
// is 4 KB, and its table entries are there one step ahead only; 1 x 30000, 32 / 8 heads of
// 128 (123 MB, 19 us) 44 to 47 (49): some 149 pieces of each kv head are joined by one CTA;
// 1 x 540, 14 / 2 heads of 64, 11.1 (15.4): start and two launches.  The kernel of bf16 at D =
// 128 with 9 to 16 rows spills 134 bytes, the others nothing.  With the rows as the first
// operand (16, half of them not there) 193 and 240: these products are issued at a
// fraction of the tile kernel's rate.

constexpr int kFewRows = 16, kFewKeys = 16, kFewWarps = 8;
// Steps that a share has at least: with fewer more pieces are joined, with more fewer
// warps work (1 x 540 keys: 1 24.5 us, 2 16.1, 4 13.5, 8 15.7).
constexpr int kFewShare = 4;
template <int D>
constexpr int kFewStages = 3 * 128 / D;
template <int D>
constexpr int kFewStage = kFewKeys * D * 2 * 2;                  // bytes of K and V
template <int D>
constexpr int64_t few_floats() { return 2 * kFewRows + static_cast<int64_t>(D) * kFewRows; }

template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (Kind<T>::kBf16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool TRANS>
__device__ __forceinline__ void load_8x8x4(uint32_t (&r)[4], uint32_t addr) {
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// 16 bytes, zeros where there is nothing to copy.
__device__ __forceinline__ void copy16_or_zero(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

// NT: eights of rows.
template <int D, typename T, int NT>
__global__ void __launch_bounds__(kFewWarps * 32, 1) cache_attn_rows_kernel(CacheArgs a) {
  constexpr int NST = kFewStages<D>, KS = D / 16, TERMS = Kind<T>::TERMS;
  constexpr int CPR = D / 8, RPI = 32 / CPR;                      // 16-byte chunks of a row, rows an instruction copies
  constexpr float kRefShift = Kind<T>::kBf16 ? 8.0f : -6.0f;
  extern __shared__ __align__(128) uint8_t few_smem[];
  __shared__ int64_t scan_s[kFewWarps];
  __shared__ int start_s[kFewWarps][3];
  __shared__ uint32_t there_s[kFewWarps][NST];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int hkv = static_cast<int>(a.hkv), g = a.g;
  grid_dep_wait();
  grid_dep_launch();

  // ---- the line, and where the warps' shares start ----
  const int64_t me = static_cast<int64_t>(warp) * gridDim.x + blockIdx.x;    // few shares: one an SM
  int64_t v = 0, inc = 0, carry = 0, q = 0, r = 0, G = 1;
  auto scan = [&](int b, bool flag) {
    v = 0;
    if (b + tid < a.num_seqs) {
      const SeqWork w = seq_work(a, b + tid);
      if (flag && blockIdx.x == 0 && w.bad) raise_flag(a.flags, KSH_FLAG_BAD_LENGTH);
      if (w.nq > 0) v = static_cast<int64_t>(hkv) * ((w.pre + w.nq + kFewKeys - 1) / kFewKeys);
    }
    inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    __syncthreads();
    if (lane == 31) scan_s[warp] = inc;
    __syncthreads();
    int64_t before = carry;
#pragma unroll
    for (int i = 0; i < kFewWarps; ++i) {
      if (i < warp) before += scan_s[i];
      carry += scan_s[i];
    }
    inc += before;
  };
  auto start_of = [&](int64_t i) { return i * q + min(i, r); };
  auto find = [&](int b) {
    if (v == 0) return;
    const int64_t per = v / hkv;
#pragma unroll 1
    for (int w = 0; w < kFewWarps; ++w) {
      const int64_t i = static_cast<int64_t>(w) * gridDim.x + blockIdx.x, at = start_of(i) - (inc - v);
      if (i >= G || at < 0 || at >= v) continue;
      start_s[w][0] = b + tid;
      start_s[w][1] = static_cast<int>(at / per);
      start_s[w][2] = static_cast<int>(at % per);
    }
  };
  for (int b = 0; b < a.num_seqs; b += kFewWarps * 32) scan(b, true);
  const int64_t U = carry;
  G = max(min(static_cast<int64_t>(gridDim.x) * kFewWarps, U / kFewShare), int64_t(1));
  q = U / G;
  r = U - q * G;
  if (a.num_seqs <= kFewWarps * 32) {
    find(0);
  } else {
    carry = 0;
    for (int b = 0; b < a.num_seqs; b += kFewWarps * 32) scan(b, false), find(b);
  }
  __syncthreads();
  SplitItem cut = {};
  cut.last = -1;
  int64_t left = me < G ? start_of(me + 1) - start_of(me) : 0;     // steps still to be computed
  if (left > 0) {
    // ---- copies: the place that is copied next, and its table entries ----
    const uint32_t bs = static_cast<uint32_t>(a.bs);
    const uint32_t rows_per_block = static_cast<uint32_t>(a.num_layers * 2 * a.hkv * a.bs);
    const int64_t to_v = a.hkv * a.bs * D;
    const uint32_t ring = smem_u32(few_smem) + static_cast<uint32_t>(warp) * NST * kFewStage<D>;
    const int chunk = lane % CPR, sub = lane / CPR;
    int ls = start_s[warp][0], lhk = start_s[warp][1], lt = start_s[warp][2];
    int64_t lleft = left;
    int lkeys;
    {
      const SeqWork w = seq_work(a, ls);
      lkeys = w.pre + w.nq;
    }
    int blk = -1;                                 // of key lane & 15: -1 behind the end
    uint32_t rest = 0;
    bool bad = false;
    auto fetch = [&]() {
      const int pos = lt * kFewKeys + (lane & 15);
      blk = -1;
      if (lleft > 0 && pos < lkeys) {
        const uint32_t j = static_cast<uint32_t>(pos) / bs;
        rest = static_cast<uint32_t>(pos) - j * bs;
        blk = a.block_tables[static_cast<int64_t>(ls) * a.max_blocks + j];
        if (blk < 0) blk = INT32_MAX;
      }
    };
    auto issue = [&](int st) {
      if (lleft > 0) {
        const bool on = blk >= 0 && blk < a.num_blocks;
        bad = bad || (blk >= 0 && !on);
        const uint32_t row = on ? static_cast<uint32_t>(blk) * rows_per_block + rest +
                                      static_cast<uint32_t>((a.layer * 2 * hkv + lhk) * a.bs)
                                : 0xffffffffu;
        const uint32_t there = __ballot_sync(0xffffffffu, on) & 0xffffu;
        if (lane == 0) there_s[warp][st] = there;
        const uint32_t kd = ring + static_cast<uint32_t>(st) * kFewStage<D>;
#pragma unroll
        for (int i = 0; i < kFewKeys / RPI; ++i) {
          const int key = i * RPI + sub;
          const uint32_t at = __shfl_sync(0xffffffffu, row, key);
          const bool is = at != 0xffffffffu;
          const T* src = static_cast<const T*>(a.pool) + (is ? static_cast<int64_t>(at) * D + chunk * 8 : 0);
          const uint32_t dst = kd + static_cast<uint32_t>(key) * (D * 2) + (static_cast<uint32_t>(chunk ^ (key & 7)) << 4);
          copy16_or_zero(dst, src, is);
          copy16_or_zero(dst + kFewKeys * D * 2, is ? src + to_v : src, is);
        }
        --lleft;
        if (++lt * kFewKeys >= lkeys) {
          lt = 0;
          if (++lhk == hkv) {
            lhk = 0;
            if (lleft > 0) {
              SeqWork w;
              do w = seq_work(a, ++ls);
              while (w.nq == 0 && ls + 1 < a.num_seqs);
              lkeys = w.pre + w.nq;
            }
          }
        }
        fetch();
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    fetch();
#pragma unroll 1
    for (int i = 0; i < NST - 1; ++i) issue(i);

    // ---- products ----
    int s = start_s[warp][0], hk = start_s[warp][1], t = start_s[warp][2];
    SeqWork w = seq_work(a, s);
    int st = 0, rows = 0, steps = 0, t0 = 0;
    // a lane's place in a product: row of eight, and columns c0 and c0 + 1 of eight
    const int r0 = lane >> 2, c0 = (lane & 3) * 2;
    constexpr int PAR = 2 / NT;                   // chains of a term's sums
    uint32_t qb[TERMS][KS][NT][2];
    float acc[D / 16][NT][4], m[NT][2], l[NT][2], cq[NT][2];     // (d, rows), by columns: rows 8 n + c0, 8 n + c0 + 1
    int lim[NT][2];
    float room = 1.0f;
    auto row_at = [&](int R) -> int64_t {
      const int node = R / g;
      return ((w.a0 + node) * a.hq + static_cast<int64_t>(hk) * g + (R - node * g)) * D;
    };
    bool fresh = true;
    for (; left > 0; --left) {
      if (fresh) {                                // an item begins, or the share inside one
        fresh = false;
        rows = w.nq * g;
        steps = (w.pre + w.nq + kFewKeys - 1) / kFewKeys;
        room = head_room<T>(static_cast<uint32_t>(w.pre + w.nq - 1));
        t0 = t;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int R = 8 * n + r0;
          float2 x[KS][2];
          const float* const p = a.q + (R < rows ? row_at(R) : 0) + c0;
#pragma unroll
          for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              x[k][e] = R < rows ? *reinterpret_cast<const float2*>(p + 16 * k + 8 * e) : make_float2(0.f, 0.f);
          float sc = 1.0f, inv = 1.0f;
          if constexpr (!Kind<T>::kBf16) {
            float top = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; ++k) top = amax3(amax3(top, x[k][0].x, x[k][0].y), x[k][1].x, x[k][1].y);
#pragma unroll
            for (int o = 1; o <= 2; o <<= 1) top = amax3(top, __shfl_xor_sync(0xffffffffu, top, o), 0.0f);
            pow2_scale(top, &sc, &inv);
          }
          inv *= a.scale * 1.44269504088896340736f;                // to powers of two
#pragma unroll
          for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              uint32_t low;
              split<T>(mul2(f2(x[k][e].x, x[k][e].y), f2(sc, sc)), &qb[0][k][n][e], &qb[1][k][n][e], &low);
              if constexpr (TERMS == 3) qb[2][k][n][e] = low;
            }
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            cq[n][j] = __shfl_sync(0xffffffffu, inv, (c0 + j) * 4);
            lim[n][j] = 8 * n + c0 + j < rows ? w.pre + (8 * n + c0 + j) / g : -1;    // the last key that the row sees
            m[n][j] = -INFINITY;
            l[n][j] = 0.0f;
          }
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][n][e] = 0.0f;
        }
      }
      asm volatile("cp.async.wait_group %0;" ::"n"(NST - 2) : "memory");
      __syncwarp();
      issue(st == 0 ? NST - 1 : st - 1);          // the stage of the step before
      const uint32_t kd = ring + static_cast<uint32_t>(st) * kFewStage<D>, vd = kd + kFewKeys * D * 2;
      const uint32_t there = there_s[warp][st];
      const int octet = lane >> 3, in8 = lane & 7;
      float sc[TERMS][PAR][NT][4];
#pragma unroll
      for (int i = 0; i < TERMS * PAR * NT * 4; ++i) (&sc[0][0][0][0])[i] = 0.0f;
      {
        const uint32_t at = kd + static_cast<uint32_t>((octet & 1) * 8 + in8) * (D * 2);
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          uint32_t ka[4];
          load_8x8x4<false>(ka, at + (static_cast<uint32_t>((2 * k + (octet >> 1)) ^ in8) << 4));
#pragma unroll
          for (int i = 0; i < TERMS; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_16816<T>(sc[i][k % PAR][n], ka, qb[i][k][n][0], qb[i][k][n][1]);
        }
      }
      const bool some_hidden = (t + 1) * kFewKeys > w.pre + 1, special = some_hidden || there != 0xffffu;
      float x[NT][4];                             // keys r0 (+ 8 from element 2 on) of 16, rows 8 n + c0 (+ 1)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float y[TERMS];
#pragma unroll
          for (int i = 0; i < TERMS; ++i) y[i] = PAR == 2 ? sc[i][0][n][e] + sc[i][PAR - 1][n][e] : sc[i][0][n][e];
          if constexpr (TERMS == 3) y[1] += y[2];
          x[n][e] = y[0] + y[1];
        }
      if (special) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int k = r0 + (e >> 1) * 8;
            if (!((there >> k) & 1) || t * kFewKeys + k > lim[n][e & 1]) x[n][e] = -INFINITY;
          }
      }
      // the reference follows the maximum once that is 2^8 above it
      bool up = false;
      float mc[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float top = fmaxf(x[n][j], x[n][2 + j]);
#pragma unroll
          for (int o = 4; o <= 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          mc[n][j] = top * cq[n][j];
          up = up || mc[n][j] > m[n][j] + 8.0f;
        }
      if (__any_sync(0xffffffffu, up)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            if (!(mc[n][j] > m[n][j] + 8.0f)) continue;
            const float f = ex2(m[n][j] - mc[n][j]);
            m[n][j] = mc[n][j];
            l[n][j] *= f;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              acc[i][n][j] *= f;
              acc[i][n][2 + j] *= f;
            }
          }
      }
      uint32_t pb[TERMS][NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float ra = m[n][0] == -INFINITY ? 0.0f : m[n][0] + kRefShift, rb = m[n][1] == -INFINITY ? 0.0f : m[n][1] + kRefShift;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[n][e] = ex2(fmaf(x[n][e], cq[n][e & 1], e & 1 ? -rb : -ra));
          if (Kind<T>::kBf16) x[n][e] *= room;
        }
        l[n][0] += x[n][0] + x[n][2];
        l[n][1] += x[n][1] + x[n][3];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t hi, lo, low;
          split<T>(f2(x[n][2 * h], x[n][2 * h + 1]), &hi, &lo, &low);
          pb[0][n][h] = transpose_8x8(hi);
          pb[1][n][h] = transpose_8x8(lo);
          if constexpr (TERMS == 3) pb[2][n][h] = transpose_8x8(low);
        }
      }
      // V that some row does not see and that is not finite must not meet that row's 0
      bool rare = false;
      if (some_hidden && w.nq > 1) {
        uint32_t f = 0;
        for (int i = lane; i < kFewKeys * CPR; i += 32) {
          uint4 y;
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(y.x), "=r"(y.y), "=r"(y.z), "=r"(y.w) : "r"(vd + 16 * i));
          f |= not_finite2<T>(y.x) | not_finite2<T>(y.y) | not_finite2<T>(y.z) | not_finite2<T>(y.w);
        }
        rare = __any_sync(0xffffffffu, f != 0);
      }
      if (!rare) {
        const uint32_t at = vd + static_cast<uint32_t>((octet >> 1) * 8 + in8) * (D * 2);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          uint32_t va[4];
          load_8x8x4<true>(va, at + (static_cast<uint32_t>((2 * i + (octet & 1)) ^ in8) << 4));
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = TERMS - 1; k >= 0; --k) mma_16816<T>(o, va, pb[k][n][0], pb[k][n][1]);   // the small terms first
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][n][e] += o[e];
          }
        }
      } else {
#pragma unroll
        for (int k = 0; k < kFewKeys; ++k) {
          const int pos = t * kFewKeys + k;
          const bool on = (there >> k) & 1;
          float pr[NT][2];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) pr[n][j] = __shfl_sync(0xffffffffu, x[n][k / 8 * 2 + j], k % 8 * 4 + (lane & 3));
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint16_t b;
              asm volatile("ld.shared.u16 %0, [%1];"
                           : "=h"(b)
                           : "r"(vd + k * (D * 2) + (((2 * i + (e >> 1)) ^ (k & 7)) << 4) + r0 * 2));
              T y;
              memcpy(&y, &b, 2);
#pragma unroll
              for (int n = 0; n < NT; ++n)
                if (on && pos <= lim[n][e & 1]) acc[i][n][e] = fmaf(pr[n][e & 1], widen(y), acc[i][n][e]);
            }
        }
      }
      st = st + 1 == NST ? 0 : st + 1;
      ++t;
      if (t < steps && left > 1) continue;
      // ---- the piece t0 .. t - 1 of the item is done ----
      const bool whole = t0 == 0 && t == steps;
      float* const part = a.part + (me * 2 + (t0 > 0 ? 0 : 1)) * few_floats<D>();
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int o = 4; o <= 16; o <<= 1) l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], o);
          const int R = 8 * n + c0 + j;
          if (R >= rows) continue;
          const float inv = !whole ? 1.0f : l[n][j] == 0.0f ? 0.0f : 1.0f / l[n][j];
          float* const to = (whole ? a.out + row_at(R) : part + 2 * kFewRows + R * D) + r0;
          if (!whole && r0 == 0) part[R] = m[n][j], part[kFewRows + R] = l[n][j];
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            to[16 * i] = acc[i][n][j] * inv;
            to[16 * i + 8] = acc[i][n][2 + j] * inv;
          }
        }
      if (!whole && t0 == 0) {                    // the share's last piece: joined from here on
        const int64_t at = start_of(me + 1) - 1 + (steps - t);     // the item's last step
        cut.first = static_cast<int>(me);
        cut.last = static_cast<int>(at < r * (q + 1) ? at / (q + 1) : r + (at - r * (q + 1)) / q);
        cut.row0 = static_cast<int>(w.a0);
        cut.rows = rows;
        cut.hk = hk;
      }
      fresh = true;
      t = 0;
      if (++hk == hkv) {
        hk = 0;
        if (left > 1) {
          do w = seq_work(a, ++s);
          while (w.nq == 0 && s + 1 < a.num_seqs);
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (bad) raise_flag(a.flags, KSH_FLAG_BAD_BLOCK);
  }
  if (lane == 0) a.items[me] = cut;
}

// Joins the pieces of an item cut between warps, in key order: a CTA an item, its
// threads in groups that take runs of the pieces (one long sequence has over a hundred).
constexpr int kJoinThreads = 256;

template <int D>
__global__ void __launch_bounds__(kJoinThreads) cache_rows_merge_kernel(CacheArgs a) {
  __shared__ float m_s[kJoinThreads], l_s[kJoinThreads];
  __shared__ float4 a_s[kJoinThreads];
  grid_dep_wait();
  grid_dep_launch();
  const SplitItem it = a.items[blockIdx.x];
  if (it.last < it.first) return;
  constexpr int kPieces = 4;
  const int units = it.rows * (D / 4), groups = max(1, kJoinThreads / units), tid = threadIdx.x;
  const int all = it.last - it.first + 1, per = (all + groups - 1) / groups, grp = tid / units;
  for (int i = groups > 1 ? tid % units : tid; i < units; i += kJoinThreads) {    // (one trip where there are groups)
    const int row = i / (D / 4), c = i % (D / 4);
    const int from = groups > 1 ? it.first + grp * per : it.first;
    const int to = groups > 1 ? (grp < groups ? min(it.last, from + per - 1) : from - 1) : it.last;
    float M = -INFINITY, L = 0.0f;
    float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](const float* m, const float* l, const float4* v, int n) {
      float top = M;
#pragma unroll
      for (int u = 0; u < kPieces; ++u)
        if (u < n) top = fmaxf(top, m[u]);
      const float ref = top == -INFINITY ? 0.0f : top, w0 = ex2(M - ref);
      M = top;
      L *= w0;
      A = make_float4(A.x * w0, A.y * w0, A.z * w0, A.w * w0);
#pragma unroll
      for (int u = 0; u < kPieces; ++u) {
        if (u >= n) break;
        const float w = ex2(m[u] - ref);
        L = fmaf(l[u], w, L);
        A = make_float4(fmaf(v[u].x, w, A.x), fmaf(v[u].y, w, A.y), fmaf(v[u].z, w, A.z), fmaf(v[u].w, w, A.w));
      }
    };
    for (int p0 = from; p0 <= to; p0 += kPieces) {
      float m[kPieces], l[kPieces];
      float4 v[kPieces];
#pragma unroll
      for (int u = 0; u < kPieces; ++u) {
        if (p0 + u > to) break;
        const float* part = a.part + (static_cast<int64_t>(p0 + u) * 2 + (p0 + u == it.first ? 1 : 0)) * few_floats<D>();
        m[u] = part[row];
        l[u] = part[kFewRows + row];
        v[u] = reinterpret_cast<const float4*>(part + 2 * kFewRows + row * D)[c];
      }
      add(m, l, v, to - p0 + 1);
    }
    if (groups > 1) {
      m_s[tid] = M, l_s[tid] = L, a_s[tid] = A;
      __syncthreads();
      if (grp > 0) return;
      for (int k = 1; k < groups; ++k) {
        const float m[kPieces] = {m_s[k * units + i]}, l[kPieces] = {l_s[k * units + i]};
        const float4 v[kPieces] = {a_s[k * units + i]};
        add(m, l, v, 1);
      }
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    const int node = row / a.g;
    float* out = a.out + ((static_cast<int64_t>(it.row0) + node) * a.hq + static_cast<int64_t>(it.hk) * a.g + (row - node * a.g)) * D;
    reinterpret_cast<float4*>(out)[c] = make_float4(A.x * inv, A.y * inv, A.z * inv, A.w * inv);
  }
}

template <int D, typename T>
int launch_cache_rows(const CacheArgs& a, int grid, cudaStream_t st) {
  constexpr int kBytes = kFewWarps * kFewStages<D> * kFewStage<D>;
  auto go = [&](auto kern) -> int {
    if (set_smem_optin(reinterpret_cast<const void*>(kern), kBytes) != KSH_OK) return KSH_ERR_CUDA;
    return launch(kern, dim3(static_cast<unsigned>(grid)), dim3(kFewWarps * 32), kBytes, st, a);
  };
  const int rc = static_cast<int64_t>(a.max_q) * a.g <= 8 ? go(cache_attn_rows_kernel<D, T, 1>) : go(cache_attn_rows_kernel<D, T, 2>);
  if (rc != KSH_OK) return rc;
  return launch(cache_rows_merge_kernel<D>, dim3(static_cast<unsigned>(grid * kFewWarps - 1)), dim3(kJoinThreads), 0, st, a);
}

static_assert(few_floats<64>() * kFewWarps == part_floats<64>() && few_floats<128>() * kFewWarps == part_floats<128>(), "workspace");

int64_t items_bytes() { return (static_cast<int64_t>(num_sms()) * kFewWarps * sizeof(SplitItem) + 255) / 256 * 256; }

}  // namespace
}  // namespace ksh

using namespace ksh;

extern "C" int64_t ksh_cache_attention_workspace_size(int64_t num_seqs, int64_t hq, int64_t hkv,
                                                      int64_t d, int64_t max_q_len) {
  if (num_seqs <= 0 || hq <= 0 || hkv <= 0 || hq % hkv != 0 || d <= 0 || max_q_len < 0) return 0;
  if (d != 64 && d != 128) return 256;
  return items_bytes() + 2 * (d == 64 ? part_floats<64>() : part_floats<128>()) * 4 * num_sms();
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
  if (d > 256) return KSH_ERR_UNSUPPORTED;
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
  // Tensor cores: rows of the pool are numbered in 32 bits (2^31 rows of 64
  // halves are 256 GB), a tile holds the heads of at least one token
  const bool fast = (d == 64 || d == 128) && a.g <= kRows &&
      ((reinterpret_cast<uintptr_t>(pool) | reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) == 0 &&
      static_cast<double>(num_blocks) * 2.0 * static_cast<double>(num_layers) * static_cast<double>(hkv) *
              static_cast<double>(block_size) <= static_cast<double>(INT32_MAX);
  if (fast) {
    if (!workspace || workspace_bytes < ksh_cache_attention_workspace_size(num_seqs, hq, hkv, d, max_q_len))
      return KSH_ERR_WORKSPACE;
    if ((reinterpret_cast<uintptr_t>(workspace) & 255) != 0) return KSH_ERR_ALIGN;
    a.items = static_cast<SplitItem*>(workspace);
    a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + items_bytes());
    a.npt = kRows / a.g;
    if (max_q_len * a.g <= kFewRows) {
      const double shares = static_cast<double>(num_seqs) * static_cast<double>(hkv) *
                            static_cast<double>(std::max<int64_t>(1, (max_total_len + kFewKeys * kFewShare - 1) / (kFewKeys * kFewShare)));
      const int grid = static_cast<int>(std::min<double>(num_sms(), shares));
      if (pool_type == KSH_TYPE_F16)
        return d == 64 ? launch_cache_rows<64, __half>(a, grid, st) : launch_cache_rows<128, __half>(a, grid, st);
      return d == 64 ? launch_cache_rows<64, __nv_bfloat16>(a, grid, st) : launch_cache_rows<128, __nv_bfloat16>(a, grid, st);
    }
    // No more CTAs than there can be tiles; an item's start counts only where there
    // are several tiles a CTA.
    const double tiles = static_cast<double>(num_seqs) * static_cast<double>(hkv) *
                         static_cast<double>((std::min(max_q_len, total) + a.npt - 1) / a.npt) *
                         static_cast<double>(std::max<int64_t>(1, (max_total_len + kTK - 1) / kTK));
    const int grid = static_cast<int>(std::min<double>(num_sms(), tiles));
    a.item_cost = tiles >= 4.0 * num_sms() ? kItemCost : 0;
    if (pool_type == KSH_TYPE_F16)
      return d == 64 ? launch_cache_tc<64, __half>(a, grid, st) : launch_cache_tc<128, __half>(a, grid, st);
    return d == 64 ? launch_cache_tc<64, __nv_bfloat16>(a, grid, st) : launch_cache_tc<128, __nv_bfloat16>(a, grid, st);
  }
  // (the grid numbers heads in 16 bits; the limit on sequences is the entry's, stated in its header)
  if (hq > 65535 || num_seqs > 65535) return KSH_ERR_UNSUPPORTED;
  return pool_type == KSH_TYPE_F16 ? launch_cache_any<__half>(a, st) : launch_cache_any<__nv_bfloat16>(a, st);
}
