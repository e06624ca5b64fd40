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
// hi*lo + lo*hi + hi*hi.  P goes in relative to the largest V row that the
// query row sees in a tile, so an output is held to 2^-22 of its weighted values
// and, beside that, to about 2^-32 of that V row whatever its weight (a cached row
// 2^16 times its neighbours, with no weight: 1.5e-5).  With 128 query rows on
// the MMA's M side that is 1.6 K tensor cycles per 64 keys of D = 128, while the
// SM's share of HBM takes 2.5 K cycles to bring their 64 KB.
//
// One persistent CTA per SM.  The (sequence, kv head, 128-row tile) items'
// 64-key tiles form one line that is cut into equal pieces, one per CTA, so
// uneven lengths leave no SM idle; an item cut between CTAs leaves its
// (m, l, acc) pieces in the workspace and tree_merge_kernel joins them in key
// order (the same bits in every run).  Warps of a CTA:
//   17, 18  block table lookups and bulk copies of K (17) and V (18) rows into
//           shared memory, a copy per run of keys that stand one after the other
//   8..15   widening (four warps for K, four for V): raw rows -> scaled hi / lo
//           fp16, 128-byte swizzle, in place
//   16      MMAs: S = Q K^T (A = Q in TMEM, B = K), O = P V (A = P in TMEM,
//           B = V with the keys along K, so no transpose is stored)
//   0..7    rows: thread = query row, and half of the tile's keys and of D.
//           Scores from TMEM, running softmax in 32 bits, P as hi / lo into
//           TMEM, and every tile's P V added into fp32 registers (a long
//           context added up inside the tensor core would lose low bits at
//           each step).  Both halves take the whole row's maximum, so neither
//           waits for the other.
// Registers decide the split: 128 x 128 accumulators are a quarter of the
// file (the row warps spill 108 bytes a thread at D = 128, 96 at 64), so K / V in
// flight stay in shared memory and the code of each role is kept short (an
// earlier form with the copies in registers spilled more and missed the
// instruction cache; unrolling the widening twice costs 12 %).
//
// Measured, 64 sequences x 4096 keys x 16 nodes, 32 / 8 heads, D = 128: 530 us
// alone (4.1 TB/s, 63 % of measured HBM), 583 to 617 us back to back, where the
// power limit holds the clock at 1.55 GHz.  There the copies by themselves take
// 354 us (they alone reach the limit), and leaving one part out saves: MMAs 150 us,
// rows 70, widening 65.  Inside a tile (3.9 K cycles) the rows are the longest
// chain: 1.9 K softmax, 0.7 K for adding O, the rest waits.  3 x 31000 keys x
// 61 nodes (two row tiles read K and V one after the other, the second time
// from L2): 314 us alone, 360 to 385 back to back.  24 x 3000 x 20 nodes, 14 / 2
// heads, D = 64: 44 us, 2.7 K cycles a tile, of which the rows' chain is 2.3 K.
// No faster: two stages of K and four of V for three and three; S and O issued
// by two warps; one thread instead of a warp waiting and issuing (slower);
// up to 64 rows standing twice in the lanes with half of the keys each; a
// softmax state per half with alternating tiles (slower); at D = 64 sixteen row
// warps, each with a quarter of the keys and of D (24 x 3000: 39 us for 35).

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
  int item_cost;                // units an item's start counts for, beside its tiles
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
constexpr int kRowWarps = 8, kWideWarps = 8;
constexpr int kMmaWarp = kRowWarps + kWideWarps, kCopyWarp = kMmaWarp + 1;
constexpr int kTcThreads = 32 * (kRowWarps + kWideWarps + 4);   // an idle warp fills the last warpgroup
constexpr int kGroup = 8, kGroups = kTK / kGroup;    // keys that share a scale
// An item's start (its Q, an empty pipeline, the state written out) takes about
// four tiles' time; counted so in the line, the CTAs with two items are not the
// last ones.  24 sequences of 20 x 7 rows over up to 3000 keys of D = 64: 44 us,
// 48 with no such count.  Where there are fewer tiles than SMs can share out
// (4 a CTA) it would only put more tiles into some CTAs.
constexpr int kItemCost = 4;
constexpr int kMeta = 16;                // tiles whose scales are kept: more than the stages let run apart

// floats of one partial state: m [128], l [128], acc [D / 4][128][4]
template <int D>
constexpr int64_t part_floats() { return 2 * kRows + static_cast<int64_t>(D) * kRows; }

template <int D>
struct TreeLayout {
  static constexpr int TERM = kTK * D * 2;           // one fp16 term of a K (or V) tile
  static constexpr int NST = D == 128 ? 3 : 6;       // stages of K and of V
  // A stage is first the raw rows, then, in place, their two terms: a widening
  // warp's eight rows (GRP bytes) become its own hi blocks, 64 columns of
  // eight 128-byte rows each, and lo blocks.  The groups' stride goes into the
  // operand descriptors.
  static constexpr int GRP = kGroup * D * 4;
  static constexpr int LO = D / 64 * 1024;           // lo blocks of a group, after the hi blocks
  static constexpr int K_OFF = 0, V_OFF = NST * 2 * TERM;
  // per tile (ring of kMeta): inverse scales of K and V per group of eight
  // keys (1 in tiles with drafted nodes), and per key (in those)
  static constexpr int META = V_OFF + NST * 2 * TERM;    // kinv, vinv [8], krel, vrel [64]
  static constexpr int BITS = META + 2 * kMeta * (kGroups + kTK) * 4;   // valid, kpois, vpois, tile [8]
  static constexpr int BAR = BITS + 4 * kMeta * 8;
  static constexpr int NBAR = 6 * NST + 2 * 2 + 5;
  static constexpr int MISC = BAR + NBAR * 8;
  static constexpr int BYTES = MISC + 64 + 1024;
  // TMEM columns: Q hi, Q lo (D / 2 each), two S, two P buffers, O
  static constexpr uint32_t Q_COL = 0, S_COL = D, P_COL = D + 2 * kTK, O_COL = D + 4 * kTK;
  static constexpr uint32_t COLS = 512;
  static_assert(O_COL + D <= COLS, "TMEM columns");
  static_assert(BYTES <= 220 * 1024, "shared memory");
};

// One sequence's share of the work.
struct SeqWork {
  int64_t a0;
  int nq, keys, pre, ntiles, nqt;
  bool bad;                     // lengths that do not fit
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

// The pieces of items in one CTA's share of the line, one after the other.
// Each warp keeps its own walk in shared memory (registers are for the tiles);
// a step is additions, and loads only where a new sequence begins.
struct Walk {
  SeqWork w;                    // of sequence s
  int64_t left;                 // units of the share still to go
  int s, item, t;               // t: next tile of the item
};
struct Piece {
  int64_t a0;
  int s, hk, qt, t0, t1, nq, keys, pre, ntiles;
};

__device__ __forceinline__ bool next_piece(const TreeArgs& a, Walk* wk, Piece* p) {
  Walk k = *wk;
  if (k.left <= 0) return false;
  if (k.t == k.w.ntiles) {
    k.t = 0;
    ++k.item;
    k.left -= a.item_cost;
    if (k.left <= 0) return false;
    if (k.item == static_cast<int>(a.hkv) * k.w.nqt) {
      k.item = 0;
      do {
        if (++k.s >= a.num_seqs) return false;    // lengths that changed on the way
        k.w = seq_work(a, k.s);
      } while (k.w.nqt == 0);
    }
  }
  p->t0 = k.t;
  p->t1 = k.t = static_cast<int>(min(static_cast<int64_t>(k.w.ntiles), k.t + k.left));
  k.left -= p->t1 - p->t0;
  p->hk = k.w.nqt == 1 ? k.item : k.item / k.w.nqt;
  p->qt = k.item - p->hk * k.w.nqt;
  p->s = k.s;
  p->a0 = k.w.a0;
  p->nq = k.w.nq;
  p->keys = k.w.keys;
  p->pre = k.w.pre;
  p->ntiles = k.w.ntiles;
  __syncwarp();
  if ((threadIdx.x & 31) == 0) *wk = k;
  __syncwarp();
  return true;
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
// Global -> shared copy, 16-byte aligned, completing on an mbarrier.
__device__ __forceinline__ void copy_bulk(void* dst, const float* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ bool not_finite(float x) { return abs_bits(x) >= 0x7f800000u; }
// largest |x|; NaN wins
__device__ __forceinline__ float amax3(float a, float b, float c) {
  float m;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(fabsf(a)), "f"(fabsf(b)), "f"(fabsf(c)));
  return m;
}
__device__ __forceinline__ float warp_amax(float x) {
  float m;
  asm volatile("redux.sync.max.abs.NaN.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(x));
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
// x = hi + lo as fp16 pairs: hi the leading 11 bits, lo the next 11
__device__ __forceinline__ void split2(F2 xy, uint32_t* hi, uint32_t* lo) {
  const float2 f = unpack(xy);
  const float hx = __uint_as_float(__float_as_uint(f.x) & 0xffffe000u);
  const float hy = __uint_as_float(__float_as_uint(f.y) & 0xffffe000u);
  const float2 r = unpack(fma2(f2(hx, hy), f2(-1.0f, -1.0f), xy));
  *hi = h2_bits(__floats2half2_rn(hx, hy));
  *lo = h2_bits(__floats2half2_rn(r.x, r.y));
}
// The loads of v have arrived (v as operands: no use may move above this).
__device__ __forceinline__ void tmem_wait_ld(float (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]),
                 "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]),
                 "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
               :
               : "memory");
}
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
__device__ __forceinline__ float max3(float a, float b, float c) {
  float m;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

// Operand descriptor, 128-byte swizzle, 1024-byte blocks of eight 128-byte
// rows.  K-major (K): `groups` bytes from eight rows to the next eight.
// MN-major (V): a row holds 64 of the N columns; `groups` bytes from eight rows
// (of the K dimension) to the next, 1024 to the next 64 columns.
__device__ __forceinline__ uint64_t desc_blocks(uint32_t smem_addr, uint32_t groups) {
  return static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(1024u >> 4) << 16) |
         (static_cast<uint64_t>(groups >> 4) << 32) | (1ull << 46) | (2ull << 61);
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
  const int bs = static_cast<int>(a.bs), j = pos / bs;
  const int64_t blk = a.block_tables[static_cast<int64_t>(s) * a.max_blocks + j];
  if (blk < 0 || blk >= a.num_blocks) return -1;
  return ((((blk * a.num_layers + a.layer) * 2) * a.hkv + hk) * a.bs + (pos - j * bs)) * D;
}

// The largest of a tile's V scales (with drafted nodes: one per key) that a row
// sees.  Out of line: seldom called, and with the loop in the row warps' code 64 x
// 4096 keys took 0.7 % longer.
__device__ __noinline__ float seen_scale(const float* rel, uint64_t see) {
  float top = 0.0f;
#pragma unroll 1
  for (int j = 0; j < kTK; ++j)
    if ((see >> j) & 1) top = fmaxf(top, rel[j]);
  return top;
}

template <int D>
__global__ void __launch_bounds__(kTcThreads, 1) tree_attn_tc_kernel(TreeArgs a) {
  using L = TreeLayout<D>;
  constexpr int NST = L::NST;
  extern __shared__ uint8_t smem_raw[];
  // aligned by an offset, so that the compiler still sees shared memory (a
  // pointer rounded as an integer makes every access a generic one)
  uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  float* kinv_s = reinterpret_cast<float*>(smem + L::META);    // [kMeta][8]
  float* vinv_s = kinv_s + kMeta * kGroups;
  float* krel_s = vinv_s + kMeta * kGroups;                 // [kMeta][64]
  float* vrel_s = krel_s + kMeta * kTK;
  uint8_t* valid_s = smem + L::BITS;                           // [kMeta][8]: bits of the groups' keys
  uint8_t* kpois_s = valid_s + kMeta * 8;
  uint8_t* vpois_s = kpois_s + kMeta * 8;
  uint8_t* tile_s = vpois_s + kMeta * 8;                   // 1: drafted nodes, 2: the CTA's last
  uint64_t* rkfull = reinterpret_cast<uint64_t*>(smem + L::BAR);
  uint64_t* rvfull = rkfull + NST;
  uint64_t* kfull = rvfull + NST;
  uint64_t* vfull = kfull + NST;
  uint64_t* kempty = vfull + NST;
  uint64_t* vempty = kempty + NST;
  uint64_t* sfull = vempty + NST;       // [2]
  uint64_t* pready = sfull + 2;         // [2]
  uint64_t* ofull = pready + 2;
  uint64_t* oempty = ofull + 1;
  uint64_t* qready = oempty + 1;
  uint64_t* lready = qready + 1;
  uint64_t* drain = lready + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  __shared__ int64_t scan_s[kTcThreads / 32];
  __shared__ Walk walk_s[kTcThreads / 32], start_s;
  __shared__ float lsum_s[2][2][kRows];     // the halves' sums, by piece parity
  __shared__ SplitItem cut_s;
  __shared__ Piece piece_s[kRowWarps];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < NST; ++i) {
      mbar_init(&rkfull[i], 1);
      mbar_init(&rvfull[i], 1);
      mbar_init(&kfull[i], kWideWarps / 2);
      mbar_init(&vfull[i], kWideWarps / 2);
      mbar_init(&kempty[i], 1);
      mbar_init(&vempty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sfull[i], 1);
      mbar_init(&pready[i], kRowWarps);
    }
    mbar_init(ofull, 1);
    mbar_init(oempty, kRowWarps);
    mbar_init(qready, kRowWarps);
    mbar_init(lready, kRowWarps);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, L::COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  grid_dep_wait();

  // Q into L2 while the memory is idle: behind the K/V copies a row takes
  // thousands of cycles
  {
    const int64_t bytes = a.total * a.hq * D * 4, each = (bytes / gridDim.x + 15) & ~int64_t(15);
    const int64_t lo = each * blockIdx.x;
    if (lo < bytes)
      prefetch_range_l2(reinterpret_cast<const uint8_t*>(a.q) + lo,
                        static_cast<size_t>(min(each, bytes - lo)), tid, kTcThreads);
  }

  // The line of tiles: its length, and the place where this CTA's share
  // starts.  An item's start counts as item_cost units.
  int64_t u0 = 0, q = 0, r = 0;                   // q units a CTA, one more for the first r
  {
    SeqWork w = {};
    int64_t v = 0, inc = 0, carry = 0;
    auto scan = [&](int b, bool first) {          // of kTcThreads sequences from b on
      w = {};
      v = 0;
      if (b + tid < a.num_seqs) {
        w = seq_work(a, b + tid);
        v = a.hkv * w.nqt * (static_cast<int64_t>(w.ntiles) + a.item_cost);
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
      const int warps = min(kTcThreads / 32, (a.num_seqs - b + 31) / 32);
      int64_t before = carry;
      for (int i = 0; i < warps; ++i) {
        if (i < warp) before += scan_s[i];
        carry += scan_s[i];
      }
      inc += before;
    };
    auto find = [&](int b) {
      if (v > 0 && u0 >= inc - v && u0 < inc) {
        const int64_t rel = u0 - (inc - v), len = w.ntiles + a.item_cost;
        const int64_t item = (rel >> 32) ? rel / len : static_cast<uint32_t>(rel) / static_cast<uint32_t>(len);
        const int at = static_cast<int>(rel - item * len) - a.item_cost;
        start_s.w = w;
        start_s.left = q + (blockIdx.x < r ? 1 : 0) + min(at, 0);
        start_s.s = b + tid;
        start_s.item = static_cast<int>(item);
        start_s.t = max(at, 0);
      }
    };
    if (tid == 0) start_s.left = 0;
    for (int b = 0; b < a.num_seqs; b += kTcThreads) scan(b, true);
    const int64_t U = carry, G = max(min(static_cast<int64_t>(gridDim.x), U), int64_t(1));
    q = (U >> 32) ? U / G : static_cast<uint32_t>(U) / static_cast<uint32_t>(G);
    r = U - q * G;
    u0 = blockIdx.x * q + min(static_cast<int64_t>(blockIdx.x), r);
    if (blockIdx.x < G) {
      if (a.num_seqs <= kTcThreads) {
        find(0);
      } else {
        carry = 0;
        for (int b = 0; b < a.num_seqs; b += kTcThreads) scan(b, false), find(b);
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
  if (lane == 0) *wk = start_s;
  if (tid == 0) cut_s.first = 0, cut_s.last = -1;
  __syncwarp();
  Piece pc = {};

  // Bounded wait of the whole warp; gives up for all roles together.
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    bool ok = false;
    for (uint32_t i = 0; i < (1u << 16); ++i) {
      ok = mbar_poll64(bar, parity);
      if (ok || *abort_flag) break;
    }
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) *abort_flag = 1;
    return ok;
  };

  if (warp >= kMmaWarp) {
    set_regs_dec<64>();
    if (warp == kMmaWarp) {
      // ---------------- MMAs ----------------
      constexpr uint32_t id_s = idesc_f16_f32(kRows, kTK);
      constexpr uint32_t id_o = idesc_f16_f32(kRows, D) | (1u << 16);   // B: keys along K
      int n = 0, seg = 0;
      bool ok = true;
      const uint32_t kbase = smem_u32(smem + L::K_OFF), vbase = smem_u32(smem + L::V_OFF);
      while (ok && next_piece(a, wk, &pc)) {
        if (!(ok = wait(qready, seg & 1))) break;
        ++seg;
        tc_fence_after();
        // S of tile t, then O of tile t - 1
#pragma unroll 1
        for (int t = pc.t0; t <= pc.t1; ++t, ++n) {
          if (t < pc.t1) {
            const int st = n % NST, b = n & 1;
            if (!(ok = wait(&kfull[st], (n / NST) & 1))) break;
            tc_fence_after();
            if (elect_one()) {
              const uint32_t d = tmem + L::S_COL + static_cast<uint32_t>(b) * kTK;
              const uint32_t qh = tmem + L::Q_COL, ql = qh + D / 2;
              const uint64_t kh = desc_blocks(kbase + st * 2 * L::TERM, L::GRP);
              // the small terms first: the tensor core cuts low bits off at
              // every step, relative to the sum so far
#pragma unroll
              for (int term = 0; term < 3; ++term) {
                const uint32_t qa = term == 1 ? ql : qh;
                const uint64_t kt = kh + (term == 0 ? L::LO / 16 : 0);
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
                  mma_f16_ts(d, qa + 8 * k, kt + (k / 4) * 64 + 2 * (k % 4), id_s,
                             (term > 0 || k > 0) ? 1u : 0u);
              }
              mma_commit(&kempty[st]);
              mma_commit(&sfull[b]);
            }
            __syncwarp();
          }
          if (t > pc.t0) {
            const int m = n - 1, st = m % NST, b = m & 1;
            if (!(ok = wait(&vfull[st], (m / NST) & 1) && wait(&pready[b], (m >> 1) & 1) &&
                       (m == 0 || wait(oempty, (m - 1) & 1))))
              break;
            tc_fence_after();
            if (elect_one()) {
              const uint32_t d = tmem + L::O_COL;
              const uint32_t p = tmem + L::P_COL + static_cast<uint32_t>(b) * kTK;
              const uint64_t vh = desc_blocks(vbase + st * 2 * L::TERM, L::GRP);
              // 16 keys: eight columns of hi pairs of P and eight of lo pairs,
              // two groups of V
#pragma unroll
              for (int term = 0; term < 3; ++term) {
                const uint32_t pa = p + (term == 1 ? 8 : 0);
                const uint64_t vt = vh + (term == 0 ? L::LO / 16 : 0);
#pragma unroll
                for (int k = 0; k < kTK / 16; ++k)
                  mma_f16_ts(d, pa + 16 * k, vt + 2 * L::GRP / 16 * k, id_o, (term > 0 || k > 0) ? 1u : 0u);
              }
              mma_commit(&vempty[st]);
              mma_commit(ofull);
            }
            __syncwarp();
          }
        }
        --n;                                        // the round after the last tile
      }
      // nothing of this CTA's is in flight when its TMEM goes
      if (elect_one()) mma_commit(drain);
      __syncwarp();
      mbar_wait(drain, 0);
    } else if (warp <= kCopyWarp + 1) {
      // ---------------- K (one warp) / V (the next) rows into shared memory ----------------
      const int kv = warp - kCopyWarp;
      uint64_t* const rfull = kv ? rvfull : rkfull;
      uint64_t* const freed = kv ? vempty : kempty;
      uint8_t* const base = smem + (kv ? L::V_OFF : L::K_OFF);
      const float* const src = a.pool + (kv ? a.hkv * a.bs * D : 0);
      // A lane has the keys lane and 32 + lane of a tile: table column, place in
      // the block and table entry, the entry fetched one tile ahead.  A tile's
      // lookups are kept to additions (rows of the pool as 32-bit numbers; the
      // host checks that they fit): with divisions and 64-bit offsets here the
      // two warps were the slowest roles, 3270 of 4200 cycles a tile.
      const int bs = static_cast<int>(a.bs), dj = kTK / bs, dr = kTK - dj * bs;
      const uint32_t rows_per_block = static_cast<uint32_t>(a.num_layers * 2 * a.hkv * a.bs);
      bool have = next_piece(a, wk, &pc), bad = false;
      int t = 0, done = 0;                          // done: tiles whose copies are on their way
      uint32_t row0 = 0;                            // of the piece's layer and head in block 0
      const int32_t* table = nullptr;
      int col[2], rest[2], blk[2];
      auto begin = [&]() {
        t = pc.t0;
        row0 = static_cast<uint32_t>((a.layer * 2 * a.hkv + pc.hk) * a.bs);
        table = a.block_tables + static_cast<int64_t>(pc.s) * a.max_blocks;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int pos = t * kTK + 32 * h + lane;
          col[h] = pos / bs;
          rest[h] = pos - col[h] * bs;
        }
      };
      auto fetch = [&]() {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          blk[h] = -1;
          if (have && t * kTK + 32 * h + lane < pc.keys) {
            blk[h] = table[col[h]];
            if (blk[h] < 0) blk[h] = INT32_MAX;
          }
        }
      };
      if (have) begin();
      fetch();
      while (have) {
        uint32_t row[2], there[2], len[2];
        // keys that stand one after the other (in a half of the tile) go in
        // one copy, whatever the block size: bytes from this lane's key on,
        // 0 where an earlier lane's copy brings it
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bool on = blk[h] >= 0 && blk[h] < a.num_blocks;
          bad = bad || (blk[h] >= 0 && !on);
          row[h] = static_cast<uint32_t>(blk[h]) * rows_per_block + row0 + static_cast<uint32_t>(rest[h]);
          there[h] = __ballot_sync(0xffffffffu, on);
          const uint32_t before = __shfl_up_sync(0xffffffffu, row[h], 1);
          const bool follows = on && ((there[h] << 1) >> lane & 1) && row[h] == before + 1;
          const uint32_t chain = __ballot_sync(0xffffffffu, follows);
          // the lanes after this one that follow on; none past lane 31
          len[h] = on && !follows ? static_cast<uint32_t>(__ffs(static_cast<int>(~((chain >> lane) >> 1)))) * (D * 4) : 0u;
        }
        const bool tree = (t + 1) * kTK > pc.pre;
        if (++t < pc.t1) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            col[h] += dj;
            rest[h] += dr;
            if (rest[h] >= bs) rest[h] -= bs, ++col[h];
          }
        } else {
          have = next_piece(a, wk, &pc);
          if (have) begin();
        }
        fetch();
        const int st = done % NST, mt = done % kMeta;
        const uint32_t bytes = static_cast<uint32_t>(__popc(there[0]) + __popc(there[1])) * D * 4;
        if (done >= NST && !wait(freed + st, ((done / NST) - 1) & 1)) break;
        if (lane < 8)                               // both warps the same
          valid_s[mt * 8 + lane] = static_cast<uint8_t>((lane < 4 ? there[0] : there[1]) >> (8 * (lane & 3)));
        if (lane == 0) tile_s[mt * 8] = static_cast<uint8_t>((tree ? 1 : 0) | (have ? 0 : 2));
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(rfull + st, bytes);
        __syncwarp();
        uint8_t* dst = base + st * 2 * L::TERM + lane * D * 4;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (len[h]) copy_bulk(dst + 32 * h * D * 4, src + static_cast<int64_t>(row[h]) * D, len[h], rfull + st);
        ++done;
      }
      // after an abort, let the copies still in flight land before the CTA exits
      if (*abort_flag)
        for (int i = max(0, done - NST); i < done; ++i) mbar_wait(rfull + i % NST, (i / NST) & 1);
      if (bad) raise_flag(a.flags, KSH_FLAG_BAD_BLOCK);
    }
  } else if (warp >= kRowWarps) {
    // ---------------- widening ----------------
    set_regs_dec<64>();
    // four warps for K, four for V, two groups of keys each
    const int kv = (warp - kRowWarps) >> 2, w2 = ((warp - kRowWarps) & 3) * 2;
    uint64_t* const rfull = kv ? rvfull : rkfull;
    uint64_t* const full = kv ? vfull : kfull;
    uint8_t* const base = smem + (kv ? L::V_OFF : L::K_OFF);
    float* const inv_s = kv ? vinv_s : kinv_s;
    float* const rel_s = kv ? vrel_s : krel_s;
    uint8_t* const pois_s = kv ? vpois_s : kpois_s;
    constexpr int RPI = 128 / D;                    // rows per warp-wide load
    constexpr int NLD = kGroup / RPI;
    const int sub = D == 128 ? 0 : lane >> 4;       // row of the load
    const int ln = D == 128 ? lane : lane & 15;     // float4 column of the row
    const uint32_t block = static_cast<uint32_t>(ln >> 4) * 1024;
    const uint32_t chunk = static_cast<uint32_t>((ln & 15) >> 1), word = static_cast<uint32_t>(ln & 1) * 8;
    bool more = wk->left > 0;
#pragma unroll 1
    for (int n = 0; more; ++n) {
      const int st = n % NST, mt = n % kMeta;
      if (!wait(rfull + st, (n / NST) & 1)) break;
      more = !(tile_s[mt * 8] & 2);
      const bool tree = tile_s[mt * 8] & 1;
#pragma unroll 1
      for (int ww = w2; ww < w2 + 2; ++ww) {
        const uint32_t valid = valid_s[mt * 8 + ww];
        uint8_t* grp = base + st * 2 * L::TERM + ww * L::GRP;
        float4 r[NLD];
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < NLD; ++i)
          r[i] = *reinterpret_cast<const float4*>(grp + (i * RPI + sub) * (D * 4) + ln * 16);
        __syncwarp();                                 // the terms go over the rows
#pragma unroll
        for (int i = 0; i < NLD; ++i) top = amax3(amax3(r[i].x, r[i].y, r[i].z), r[i].w, top);
        top = warp_amax(top);
        uint32_t pois = 0;
        if (__builtin_expect(valid != 0xffu || not_finite(top), 0)) {
          // rows that are not there, and elements that are not finite, go in as
          // zeros; the bits of the latter's rows are kept
          top = 0.0f;
#pragma unroll
          for (int i = 0; i < NLD; ++i) {
            float4& v = r[i];
            if (!((valid >> (i * RPI + sub)) & 1)) v = make_float4(0.f, 0.f, 0.f, 0.f);
            const unsigned who = __ballot_sync(
                0xffffffffu, not_finite(v.x) || not_finite(v.y) || not_finite(v.z) || not_finite(v.w));
            if (D == 128) {
              if (who) pois |= 1u << i;
            } else {
              if (who & 0xffffu) pois |= 1u << (i * RPI);
              if (who >> 16) pois |= 1u << (i * RPI + 1);
            }
            v.x = not_finite(v.x) ? 0.f : v.x;
            v.y = not_finite(v.y) ? 0.f : v.y;
            v.z = not_finite(v.z) ? 0.f : v.z;
            v.w = not_finite(v.w) ? 0.f : v.w;
            top = amax3(amax3(v.x, v.y, v.z), v.w, top);
          }
          top = warp_amax(top);
        }
        // one power of two for the eight rows: smaller rows keep 22 bits down to
        // 2^-16 of the largest
        float sc, inv;
        pow2_scale(top, &sc, &inv);
        if (lane == 0) {
          inv_s[mt * kGroups + ww] = inv;
          pois_s[mt * 8 + ww] = static_cast<uint8_t>(pois);
        }
        if (__builtin_expect(tree, 0)) {
          // tiles with drafted nodes: a power of two for each row, so that a row few
          // nodes see cannot cost the others bits; the scores and P take them
          // back, P by what each query row sees
          if (lane == 0) inv_s[mt * kGroups + ww] = 1.0f;
#pragma unroll
          for (int i = 0; i < NLD; ++i) {
            float m = amax3(amax3(r[i].x, r[i].y, r[i].z), r[i].w, 0.0f);
#pragma unroll
            for (int o = D / 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            float s1, inv1;
            pow2_scale(m, &s1, &inv1);
            // sc takes inv back below (left out for these tiles there, 64 x 4096 keys
            // took 1.5 % longer); s1 * inv could overflow, values below 2^15 cannot
            r[i].x = r[i].x * s1 * inv;
            r[i].y = r[i].y * s1 * inv;
            r[i].z = r[i].z * s1 * inv;
            r[i].w = r[i].w * s1 * inv;
            if (ln == 0) rel_s[mt * kTK + ww * kGroup + i * RPI + sub] = inv1;
          }
        }
#pragma unroll
        for (int i = 0; i < NLD; ++i) {
          const uint32_t row = i * RPI + sub;
          uint2 hi, lo;
          split2(mul2(f2(r[i].x, r[i].y), f2(sc, sc)), &hi.x, &lo.x);
          split2(mul2(f2(r[i].z, r[i].w), f2(sc, sc)), &hi.y, &lo.y);
          uint8_t* at = grp + block + row * 128 + ((chunk ^ row) << 4) + word;
          *reinterpret_cast<uint2*>(at) = hi;
          *reinterpret_cast<uint2*>(at + L::LO) = lo;
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(full + st);
    }
  } else {
    // ---------------- rows ----------------
    set_regs_inc<144>();
    const int hw = warp >> 2, row = (warp & 3) * 32 + lane;      // half, query row
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    constexpr int DH = D / 2;                       // columns of O per half
    int n = 0, seg = 0;
    bool ok = true;
    const Piece& ps = piece_s[warp];                // of the rare paths
    while (ok && next_piece(a, wk, &pc)) {
      __syncwarp();
      if (lane == 0) piece_s[warp] = pc;
      __syncwarp();
      const int t0 = pc.t0, t1 = pc.t1, pre = pc.pre;
      const bool live = (pc.qt * kRows + row) / a.g < pc.nq;
      auto node_of = [&]() { return (ps.qt * kRows + row) / a.g; };
      auto row_at = [&]() -> int64_t {              // the row's place in q and out
        const int R = ps.qt * kRows + row, node = R / a.g;
        return ((ps.a0 + node) * a.hq + static_cast<int64_t>(ps.hk) * a.g + (R - node * a.g)) * D;
      };
      float qinv;
      // Q: hi / lo terms of the half's columns into TMEM.  Four lanes load 64
      // bytes of a row, for the rows of the four, and exchange them (a row a
      // lane took 32 lines a load, 8 K cycles an item)
      {
        const float* qp[4];
        float m[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int R = pc.qt * kRows + (row & ~3) + k, node = R / a.g;
          qp[k] = node < pc.nq ? a.q + ((pc.a0 + node) * a.hq + static_cast<int64_t>(pc.hk) * a.g + (R - node * a.g)) * D +
                                     (lane & 3) * 4
                               : nullptr;
          m[k] = 0.0f;
        }
        auto quad = [&](int k, int c) {
          return qp[k] ? *reinterpret_cast<const float4*>(qp[k] + c) : make_float4(0.f, 0.f, 0.f, 0.f);
        };
        float4 v[DH / 4];
#pragma unroll
        for (int half = 1; half >= 0; --half) {      // the other half's for the maximum alone
#pragma unroll
          for (int c = 0; c < DH / 4; ++c) v[c] = quad(c & 3, (hw ^ half) * DH + (c >> 2) * 16);
#pragma unroll
          for (int c = 0; c < DH / 4; ++c)
            m[c & 3] = amax3(amax3(m[c & 3], v[c].x, v[c].y), v[c].z, v[c].w);
        }
        // the four lanes' maxima of the lane's row
#pragma unroll
        for (int o = 1; o <= 2; o <<= 1)
#pragma unroll
          for (int k = 0; k < 4; ++k) m[k] = amax3(m[k], __shfl_xor_sync(0xffffffffu, m[k], o), 0.0f);
        const float top = (lane & 2) ? ((lane & 1) ? m[3] : m[2]) : ((lane & 1) ? m[1] : m[0]);
        float qs;
        pow2_scale(top, &qs, &qinv);
#pragma unroll
        for (int c0 = 0; c0 < DH / 4; c0 += 8) {
          uint32_t hi[16], lo[16];
#pragma unroll
          for (int c = c0; c < c0 + 8; c += 4) {
            float4 x[4] = {v[c], v[c + 1], v[c + 2], v[c + 3]};
            exchange4(x, lane);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int at = (c - c0 + k) * 2;
              split2(mul2(f2(x[k].x, x[k].y), f2(qs, qs)), &hi[at], &lo[at]);
              split2(mul2(f2(x[k].z, x[k].w), f2(qs, qs)), &hi[at + 1], &lo[at + 1]);
            }
          }
          tmem_st_32x32b_x16(lanes + L::Q_COL + (hw * DH + c0 * 4) / 2, hi);
          tmem_st_32x32b_x16(lanes + L::Q_COL + DH + (hw * DH + c0 * 4) / 2, lo);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(qready);
      }
      auto word = [&](int i) -> uint64_t {          // nodes 64 i .. 64 i + 63 that the row sees
        const int node = node_of();
        if (a.mask) return live && i < a.words ? a.mask[(ps.a0 + node) * a.words + i] : 0;
        const int bits = node + 1 - 64 * i;
        return bits <= 0 ? 0 : bits >= 64 ? ~0ull : (1ull << bits) - 1;
      };
      const float cq = qinv * (a.scale * 1.44269504088896340736f);   // to powers of two
      if ((pc.qt * kRows + (warp & 3) * 32) / a.g >= pc.nq) {
        // No row of the warp's is live: zeros for P once (multiplying them costs
        // the tensor cores no power, and power bounds long runs), then it only
        // keeps step.
        uint32_t zero[16];
#pragma unroll
        for (int c = 0; c < 16; ++c) zero[c] = 0;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int c = 0; c < 32; c += 16) tmem_st_32x32b_x16(lanes + L::P_COL + b * kTK + 32 * hw + c, zero);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
#pragma unroll 1
        for (int t = t0; t <= t1; ++t, ++n) {
          if (t < t1) {
            if (!(ok = wait(&sfull[n & 1], (n >> 1) & 1))) break;
            if (lane == 0) mbar_arrive(&pready[n & 1]);
          }
          if (t > t0) {
            if (!(ok = wait(ofull, (n - 1) & 1))) break;
            if (lane == 0) mbar_arrive(oempty);
          }
        }
        if (!ok) break;
        --n;
        if (lane == 0) mbar_arrive(lready);
        if (!(ok = wait(lready, seg & 1))) break;
        ++seg;
        continue;
      }
      // running state: the reference that the sums stand at (in powers of two;
      // it follows the maximum once that is 2^8 above it, so most tiles
      // rescale nothing), the half's sum
      float mref = -INFINITY, l = 0.0f;
      F2 acc[DH / 2];
#pragma unroll
      for (int c = 0; c < DH / 2; ++c) acc[c] = f2(0.f, 0.f);
      // of the tile whose P V is still to be added
      float corr_p = 1.0f, vs_p = 0.0f;
      uint64_t rare_p = 0;

      // softmax of tile t, then the addition of tile t - 1's P V
#pragma unroll 1
      for (int t = t0; t <= t1; ++t, ++n) {
        float corr = 1.0f, vs = 0.0f;
        uint64_t rare = 0;
        if (t < t1) {
          const int st = n % NST, b = n & 1, mt = n % kMeta;
          const uint32_t pq = (n >> 1) & 1, pv = (n / NST) & 1;
          if (!__all_sync(0xffffffffu, mbar_test2(&sfull[b], pq, &vfull[st], pv)))
            if (!(ok = wait(&sfull[b], pq) && wait(&vfull[st], pv))) break;
          tc_fence_after();
          {
            const uint64_t kpois = *reinterpret_cast<const uint64_t*>(kpois_s + mt * 8);
            const uint64_t vpois = *reinterpret_cast<const uint64_t*>(vpois_s + mt * 8);
            const uint64_t valid = *reinterpret_cast<const uint64_t*>(valid_s + mt * 8);
            const bool tree = (t + 1) * kTK > pre;
            const float* kg = kinv_s + mt * kGroups;
            const float* vg = vinv_s + mt * kGroups;
            const uint32_t sc = lanes + L::S_COL + static_cast<uint32_t>(b) * kTK;
            const uint32_t pc0 = lanes + L::P_COL + static_cast<uint32_t>(b) * kTK;
            float x[32], m = -INFINITY;
            auto top32 = [&](int h) {                // eight keys share a scale
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                const float* v = x + 8 * g;
                m = fmaxf(m, fmaxf(max3(max3(v[0], v[1], v[2]), v[3], v[4]), max3(v[5], v[6], v[7])) * kg[4 * h + g]);
              }
            };
            uint32_t own = sc + 32 * hw;             // the half's scores
            if (__builtin_expect(!tree && (valid == ~0ull) && ((kpois | vpois) == 0), 1)) {
              tmem_ld_32x32b_x32(sc + 32 * (hw ^ 1), x);      // the other half's, for the maximum
              tmem_wait_ld(x);
              top32(hw ^ 1);
            } else {
              // the tree's part of the keys, keys that are not there
              uint64_t see = valid;
              const int n0 = t * kTK - pre;          // node of the tile's first key
              if (tree) {
                if (n0 < 0) {
                  see &= ((1ull << -n0) - 1) | (word(0) << -n0);
                } else {
                  const int i = n0 >> 6, sh = n0 & 63;
                  see &= sh ? (word(i) >> sh) | (word(i + 1) << (64 - sh)) : word(i);
                }
              }
              rare = live ? vpois & see : 0;
              if (tree) {
                // P goes in relative to the largest V scale of the tile; where its V
                // rows are 2^8 apart, to the largest that the row sees (both halves
                // alike), so that rows of V that it does not see cost it no bits (P of
                // a key that is not seen is 0 times a finite factor)
                const float* rv = vrel_s + mt * kTK;
                const float s0 = rv[lane], s1 = rv[lane + 32];
                const float big = warp_amax(fmaxf(s0, s1)), low = big * 0x1p-8f;
                float mine = big;
                if (__any_sync(0xffffffffu, ((valid >> lane) & 1 && s0 < low) || ((valid >> lane >> 32) & 1 && s1 < low)))
                  mine = seen_scale(rv, see);
                vs = fmaxf(mine, 0x1p-119f);
              }
              __syncwarp();                          // word() loads for live rows only
#pragma unroll 1
              for (int c = 0; c < 4; ++c) {
                float y[16];
                tmem_ld_32x32b_x16(sc + 16 * c, y);
                tmem_wait_ld(y);
                if (tree) {
#pragma unroll
                  for (int j = 0; j < 16; ++j) y[j] *= krel_s[mt * kTK + 16 * c + j];
                }
                // K elements that are not finite went in as zeros
                for (uint32_t left = static_cast<uint32_t>(kpois >> (16 * c)) & 0xffffu; left && live; left &= left - 1) {
                  const int j = __ffs(static_cast<int>(left)) - 1;
                  const int64_t at = key_offset(a, ps.s, ps.hk, t * kTK + 16 * c + j, D);
                  const float* qp = a.q + row_at();
                  float add = 0.0f;
                  if (at >= 0)
#pragma unroll 1
                    for (int e = 0; e < D; ++e) {
                      const float kx = a.pool[at + e];
                      if (not_finite(kx)) add += qp[e] * kx;
                    }
#pragma unroll
                  for (int e = 0; e < 16; ++e)
                    if (e == j) y[e] += add;
                }
                __syncwarp();                        // lanes without a live row skipped the loop
                const uint32_t on = static_cast<uint32_t>(see >> (16 * c));
                const float k0 = kg[2 * c], k1 = kg[2 * c + 1];
                uint32_t bits[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                  y[j] = (on >> j) & 1 ? y[j] : -INFINITY;
                  m = fmaxf(m, y[j] * (j < 8 ? k0 : k1));
                  bits[j] = __float_as_uint(y[j]);
                }
                if ((c >> 1) == hw) tmem_st_32x32b_x16(pc0 + 16 * c, bits);    // P's columns are free
              }
              tmem_wait_st();
              own = pc0 + 32 * hw;
            }
            tmem_ld_32x32b_x32(own, x);
            tmem_wait_ld(x);
            top32(hw);
            const float mc = m * cq;
            if (mc > mref + 8.0f) {
              corr = ex2(mref - mc);
              mref = mc;
            }
            const float ref = mref == -INFINITY ? 0.0f : mref;
            // V's scales relative to the tile's largest; P is up to 2^8, its
            // terms up to 2^15
            float vm = warp_amax(fmaxf(vg[lane & 7], 0x1p-119f));
            vm = vs != 0.0f ? vs : vm;               // a tile with drafted nodes: the row's own
            const float up = __uint_as_float((261u << 23) - (__float_as_uint(vm) & 0x7f800000u));   // 2^7 / vm
            vs = vm * (1.0f / 128.0f);
            // P = 2^(x c - ref)
            F2 s2[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
            const F2 nref = f2(-ref, -ref);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const float c1 = fmaxf(kg[4 * hw + g] * cq, 0x1p-126f);
              const F2 c2 = f2(c1, c1);
#pragma unroll
              for (int j = 8 * g; j < 8 * g + 8; j += 2) {
                const float2 e = unpack(fma2(f2(x[j], x[j + 1]), c2, nref));
                x[j] = ex2(e.x);
                x[j + 1] = ex2(e.y);
                s2[(j >> 1) & 1] = add2(s2[(j >> 1) & 1], f2(x[j], x[j + 1]));
              }
            }
            const float2 sa = unpack(s2[0]), sb = unpack(s2[1]);
            l = fmaf(l, corr, (sa.x + sa.y) + (sb.x + sb.y));
            if (__builtin_expect(tree, 0)) {
#pragma unroll
              for (int j = 0; j < 32; ++j) x[j] *= vrel_s[mt * kTK + 32 * hw + j];
            }
            // its terms: columns of 16 keys, eight of hi pairs and eight of lo
            uint32_t pt[32];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const float f1 = vg[4 * hw + g] * up;
              const F2 w2 = f2(f1, f1);
#pragma unroll
              for (int j = 0; j < 8; j += 2) {
                const int at = (g >> 1) * 16 + (g & 1) * 4 + j / 2;
                split2(mul2(f2(x[8 * g + j], x[8 * g + j + 1]), w2), &pt[at], &pt[at + 8]);
              }
            }
            tmem_st_32x32b_x32(pc0 + 32 * hw, pt);
            tmem_wait_st();
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&pready[b]);
        }
        if (t > t0) {
          const int mt = n - 1;
          if (!(ok = wait(ofull, mt & 1))) break;
          tc_fence_after();
          {
            const uint32_t o = lanes + L::O_COL + hw * DH;
            if (__any_sync(0xffffffffu, corr_p != 1.0f)) {
#pragma unroll
              for (int c = 0; c < DH / 2; ++c) acc[c] = mul2(acc[c], f2(corr_p, corr_p));
            }
            if (__builtin_expect(__any_sync(0xffffffffu, rare_p != 0), 0)) {
              // V elements that are not finite: to the rows that see them
#pragma unroll 1
              for (int c0 = 0; c0 < DH; c0 += 16) {
                float v[16];
                tmem_ld_32x32b_x16(o + c0, v);
                tmem_wait_ld(v);
                for (uint64_t left = rare_p; left; left &= left - 1) {
                  const int pos = (t - 1) * kTK + __ffsll(static_cast<long long>(left)) - 1;
                  const int64_t at = key_offset(a, ps.s, ps.hk, pos, D);
                  if (at < 0) continue;
                  const float* vp = a.pool + at + a.hkv * a.bs * D + hw * DH + c0;
#pragma unroll
                  for (int c = 0; c < 16; ++c)
                    if (not_finite(vp[c])) v[c] += vp[c];
                }
                uint32_t bits[16];
#pragma unroll
                for (int c = 0; c < 16; ++c) bits[c] = __float_as_uint(v[c]);
                __syncwarp();
                tmem_st_32x32b_x16(o + c0, bits);
              }
              tmem_wait_st();
            }
            float v[32];
#pragma unroll
            for (int i = 0; i < DH; i += 32) {
              tmem_ld_32x32b_x32(o + i, v);
              tmem_wait_ld(v);
#pragma unroll
              for (int c = 0; c < 16; ++c)
                acc[i / 2 + c] = fma2(f2(v[2 * c], v[2 * c + 1]), f2(vs_p, vs_p), acc[i / 2 + c]);
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(oempty);
        }
        corr_p = corr;
        vs_p = vs;
        rare_p = rare;
      }
      if (!ok) break;
      --n;                                          // the round after the last tile

      // the halves' sums
      lsum_s[seg & 1][hw][row] = l;
      __syncwarp();
      if (lane == 0) mbar_arrive(lready);
      if (!(ok = wait(lready, seg & 1))) break;
      l = lsum_s[seg & 1][0][row] + lsum_s[seg & 1][1][row];
      ++seg;
      const bool whole = t0 == 0 && t1 == ps.ntiles;
      if (whole) {
        const float inv = 1.0f / l;
        float* op[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int R = ps.qt * kRows + (row & ~3) + k, node = R / a.g;
          op[k] = node < ps.nq ? a.out + ((ps.a0 + node) * a.hq + static_cast<int64_t>(ps.hk) * a.g + (R - node * a.g)) * D +
                                     hw * DH + (lane & 3) * 4
                               : nullptr;
        }
#pragma unroll
        for (int c = 0; c < DH; c += 16) {
          float4 x[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 p = unpack(acc[c / 2 + 2 * k]), u = unpack(acc[c / 2 + 2 * k + 1]);
            x[k] = make_float4(p.x * inv, p.y * inv, u.x * inv, u.y * inv);
            if (l == 0.0f) x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
          }
          exchange4(x, lane);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (op[k]) *reinterpret_cast<float4*>(op[k] + c) = x[k];
        }
      } else {
        float* part = a.part + (static_cast<int64_t>(blockIdx.x) * 2 + (t0 > 0 ? 0 : 1)) * part_floats<D>();
        if (live) {
          if (hw == 0) {
            part[row] = mref;
            part[kRows + row] = l;
          }
#pragma unroll
          for (int c = 0; c < DH; c += 4) {
            const float2 p = unpack(acc[c / 2]), q = unpack(acc[c / 2 + 1]);
            reinterpret_cast<float4*>(part + 2 * kRows)[(hw * DH + c) / 4 * kRows + row] = make_float4(p.x, p.y, q.x, q.y);
          }
        }
        if (t0 == 0 && tid == 0) {                 // the share's last piece: joined from here on
          const int64_t x = u0 + q + (blockIdx.x < r ? 1 : 0) + (ps.ntiles - t1) - 1;   // the item's last unit
          cut_s.first = static_cast<int>(blockIdx.x);
          cut_s.last = static_cast<int>(x < r * (q + 1) ? x / (q + 1) : r + (x - r * (q + 1)) / q);
          cut_s.row0 = static_cast<int>(ps.a0);
          cut_s.rbase = ps.qt * kRows;
          cut_s.rows = min(kRows, ps.nq * a.g - ps.qt * kRows);
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
// pieces with the running M, two at a time.  4 us of a call (latency: most items
// have two or three pieces); all maxima first and then the sums took 0.7 us
// longer with one tile a piece, eight pieces at a time 0.5.
constexpr int kMergeThreads = 256, kMergeChunks = 16, kMergePieces = 2;

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

// Other head dimensions and unaligned tensors: one warp per (node, head), keys
// one after the other, any head dimension up to 256 and any alignment.  Each
// node reads all of K and V (from L2 after the first), so it takes as long as
// its keys' dot products: 64 x 4096 keys x 16 nodes, 32 heads: 41 ms.
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
                block_size <= INT32_MAX && max_blocks > 0 && num_seqs >= 0 && num_seqs <= INT32_MAX && total >= 0 &&
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
    // K/V rows are numbered in 32 bits (2^31 rows of 64 floats are 512 GB)
    if (static_cast<double>(num_blocks) * 2.0 * static_cast<double>(num_layers) * static_cast<double>(hkv) *
            static_cast<double>(block_size) > static_cast<double>(INT32_MAX))
      return KSH_ERR_UNSUPPORTED;
    if (!workspace || workspace_bytes < ksh_tree_attention_workspace_size(num_seqs, hq, hkv, d, max_nodes))
      return KSH_ERR_WORKSPACE;
    if ((reinterpret_cast<uintptr_t>(workspace) & 255) != 0) return KSH_ERR_ALIGN;
    a.items = static_cast<SplitItem*>(workspace);
    a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + items_bytes());
    // No more CTAs than there can be tiles.
    const int64_t tiles = std::max<int64_t>(1, (max_total_len + kTK - 1) / kTK);
    const int64_t qtiles = (max_nodes * a.g + kRows - 1) / kRows;
    const int grid = static_cast<int>(std::min<double>(
        num_sms(), static_cast<double>(num_seqs) * static_cast<double>(hkv) * static_cast<double>(qtiles) *
                       static_cast<double>(tiles)));
    a.item_cost = static_cast<double>(num_seqs) * static_cast<double>(hkv) * static_cast<double>(qtiles) *
                      static_cast<double>(tiles) >= 4.0 * num_sms() ? kItemCost : 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return d == 64 ? launch_tree_tc<64>(a, grid, st) : launch_tree_tc<128>(a, grid, st);
  }
  if (hq > 65535 || num_seqs > 65535) return KSH_ERR_UNSUPPORTED;
  return launch(tree_attn_simple_kernel,
                dim3(static_cast<unsigned>(max_nodes), static_cast<unsigned>(hq),
                     static_cast<unsigned>(num_seqs)),
                dim3(32), 0, static_cast<cudaStream_t>(stream), a);
}
