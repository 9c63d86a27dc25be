// Attention of trees of drafted tokens over a paged bf16 cache (tcgen05 / TMEM), head_dim 64, 128 or 256.
//
//   o_i = sum_k p_ik v_k,  p_i = softmax over the keys k that node i sees of cap(scale q_i . k_k)
//
// A request has a context of c cells and n nodes whose keys and values lie behind it (node j in cell c + j). Node i sees the context and the nodes whose bits are
// set in its mask; of either, if there is a window, only what lies less than `window` before its own position. A node that sees nothing gives zeros.
//
// Bound: a node's G query heads of a kv head share every key and value, so that rows = n G rows of scores read 4 D bytes a key once: with up to
// 256 rows a request the cache's bytes are the floor, above it the products and exponentials. Rows are therefore the 128-row operand (a thread
// owns a row: no sums across threads), keys the other one, and a CTA takes two tiles of rows against each tile of 64 keys, a warpgroup a tile. Where a request has
// only one tile of rows the warpgroups take every second tile of keys instead and are added at the end. Either has two score buffers: the products
// of its next tile run while it works on this one.
//
// Work: the key tiles of all items (request, kv head, two tiles of rows) stand in one line, each CTA (one an SM) takes an equal stretch of it, whatever the
// lengths; an item's start (queries, output) stands in the line as kTreeStart tiles. Parts of items that a stretch's end cuts go to scratch and a
// short kernel joins them, in a fixed order.
//
// What a node does not see does not reach it: hidden scores become -inf before the softmax, and values are inspected in the tiles where nodes
// differ in what they see (the product would multiply an infinity or NaN by 0): what is not finite is taken out there and added at
// the end to the nodes that see it.
//
// head_dim 256 has one accumulator and so one tile of rows: both warpgroups work on each tile of keys, two threads a row, half of its weights and of the
// accumulator's columns each.
//
// Warp roles (384 threads): warps 0..3 / 4..7 softmax and output; warp 8 keys by TMA, and the pieces of the stretch for the others; warp 9 values by TMA; warps
// 10 / 11 MMA of either warpgroup, warp 10 TMEM owner. (One warp for both kinds of loads bounded the kernel by its instructions, 128 requests 300 us; one issuer
// for both warpgroups made each wait for the other's turn.)
//
// Measured (us on the device after a pause, at 1965 MHz; in brackets what the bytes or products take at least; 32-token pages). One tile of rows is bound by memory at that
// clock where heads have 128 dims: 128 requests of 200 to 3800 keys with 32 nodes, 32 heads over 8, 195 to 202 by the card (173), 5.7 TB/s; call after call the power limit takes the clock to
// 1425 MHz: 243, 4.7 TB/s, as many cycles as memory and the softmax warps' chain bound together. 16 of 8000 keys with 4 nodes 91 (80); 256 dims, 20 of 4000 with 16 nodes 119 to 122 (101), with 100 nodes 243 (108). With 64 dims a
// tile is half the bytes and as many exponentials: 33 of 4096 with 20 nodes, 24 heads over 8, 86 (43), soft-capped 139. Two tiles of rows are bound by the chain of a
// warpgroup: one context of 120000 keys with 61 nodes 147 to 156 (75), 64 of 2000 with 60 nodes 171 to 180 (92), tensor pipe and special functions busy in 0.45 of the cycles each. A tile of 64
// keys takes a warpgroup some 2500 cycles: its scores' wait 300 and load 150, the maximum 370, the exponentials 1050 (as many where a warp has the scheduler to itself), the
// rest 400. Slower: turns at the exponentials (155 -> 197 us), tiles of 128 keys with one buffer of scores (174 to 187), weights checked by their own maximum instead of the scores'
// (10 %); an eighth to a third of the exponentials as polynomials made that case 4 % faster and those with one tile of rows 5 to 10 % slower.
#include <limits.h>

#include <algorithm>
#include <type_traits>

#include "api.h"
#include "sm100.cuh"

namespace b200 {

static constexpr int kTreeThreads = 384, kTreeReqs = 8192, kTreeNodes = 1024;       // (the last two: at most)
static constexpr int kTreeKeys = 64;          // keys of a tile
static constexpr int kTreeStart = 4;          // what an item's start costs, in key tiles (48 ragged requests 72.7 us, with 6 74.3; 128 requests 195.3 and 193.8)
static constexpr int kTreeLeast = 5;          // tiles of a stretch at the least (one sequence of 1000 keys: 15.5 us, with 3 16.4, with 2 18.0)
static constexpr int kTreePieces = 4;         // pieces that the TMA warp is ahead
static constexpr float kTreeWideCap = 256.f;  // in log2 units

struct TreeParams {
  const __nv_bfloat16* cache;
  __nv_bfloat16* out;
  long long ldo;
  const int32_t* block_table;
  long long ldt, num_blocks;
  int max_blocks;
  const int32_t *seq_lens, *q_start;
  const int64_t* positions;            // null: no window
  const uint64_t* mask;                // [T][words]
  int words, num_reqs, total_q, Hkv, G, nodes;         // nodes of a tile of rows
  int block_size, window, max_len;
  float scale_log2, cap2;
  float* parts;
  int* status;
};

template <int D>
struct TreeShape {
  static constexpr bool kWide = D == 256;              // one tile of rows, two threads a row
  static constexpr int kParts = D / 64;                // 64-dim pieces of a row
  static constexpr int kSlot = kTreeKeys * D * 2, kPiece = kTreeKeys * 128;
  static constexpr int kKeySlots = D == 64 ? 10 : D == 128 ? 5 : 2, kValueSlots = D == 64 ? 10 : D == 128 ? 5 : 3;
  static constexpr int kQTile = 128 * D * 2, kQTiles = kWide ? 1 : 2;
  static constexpr int kTiles = kQTiles * kQTile + (kKeySlots + kValueSlots) * kSlot;
  static constexpr int kRows = 128 * kQTiles;
  static constexpr long long kPartFloats = (long long)kRows * D + 2 * kRows;          // [D / 4][kRows][4], then the rows' maxima and sums
  // Tensor memory. Two buffers of scores for each warpgroup, their P over them; its accumulator. Wide: one set of buffers, P apart (both threads of a
  // row read all its scores).
  static constexpr int kO = kWide ? 128 : 256, kP = 384;
  // tiles of a piece in which nodes may differ in what they see: those of 1024 nodes, and where a window ends those of 1024 positions
  static constexpr int kOdd = 2 * (kTreeNodes / kTreeKeys + 2);
};

struct TreeReq {
  int n, row0, len, ctx, begin, tiles, pairs, items;   // begin: first key tile; tiles: key tiles; pairs: items of a kv head
};
template <int D>
__device__ __forceinline__ TreeReq tree_req(const TreeParams& p, int start, int end, int len) {
  TreeReq r;
  r.row0 = min(max(start, 0), p.total_q);
  const int rows = max(0, min(end, p.total_q) - r.row0);
  r.n = min(rows, kTreeNodes);         // (more are left out)
  r.len = min(max(len, 0), p.max_len);
  r.ctx = r.len - rows;
  const int low = p.window > 0 ? max(0, r.ctx - p.window + 1) : 0;
  r.begin = min(low, max(r.len - 1, 0)) / kTreeKeys;
  r.tiles = max(1, (r.len + kTreeKeys - 1) / kTreeKeys - r.begin);     // (no keys: a tile that nobody sees)
  const int row_tiles = (r.n + p.nodes - 1) / p.nodes;
  r.pairs = (row_tiles + TreeShape<D>::kQTiles - 1) / TreeShape<D>::kQTiles;
  r.items = r.pairs * p.Hkv;
  return r;
}
template <int D>
__device__ __forceinline__ TreeReq tree_req(const TreeParams& p, int b) { return tree_req<D>(p, p.q_start[b], p.q_start[b + 1], p.seq_lens[b]); }

// A piece of a CTA's stretch: key tiles of an item. nt = 0: no more.
struct TreePiece {
  int b, row0, n, len, ctx;
  int key0, nt;                        // first key, tiles
  int head, node0;                     // kv head, first node
  bool two, cut, whole;                // a second tile of rows; the item began before; the piece is all of it
};
struct TreeStart {
  int req, off, begin, end, len;       // where a stretch starts: request, cells of it that are behind, its nodes and keys
};
template <int D>
struct TreeWalk {
  const TreeParams& p;
  TreeReq r;
  int b, off;                          // request, cells of it that are behind
  long long left;                      // cells of the stretch
  int end, next_end, next_len;         // where the request's nodes end; of the next request, on their way
  __device__ __forceinline__ TreeWalk(const TreeParams& p_, const TreeStart& s, long long left_) : p(p_), b(s.req), off(s.off), left(left_), end(s.end) {
    if (left <= 0) return;
    ahead();
    r = tree_req<D>(p, s.begin, s.end, s.len);
  }
  __device__ __forceinline__ void ahead() {
    const int nb = min(b + 1, p.num_reqs - 1);
    next_end = p.q_start[nb + 1];
    next_len = p.seq_lens[nb];
  }
  __device__ __forceinline__ bool next(TreePiece& w, int& jb) {
    while (left > 0) {
      const int cells = kTreeStart + r.tiles;
      if (off >= r.items * cells) {
        if (++b >= p.num_reqs) return false;
        const int start = end;
        end = next_end;
        r = tree_req<D>(p, start, end, next_len);
        ahead();
        off = 0;
        continue;
      }
      const int item = off / cells, o = off - item * cells;
      const int take = (int)min((long long)(cells - o), left);
      off += take;
      left -= take;
      jb = max(0, o - kTreeStart);
      w.nt = max(0, o + take - kTreeStart) - jb;
      if (w.nt <= 0) continue;
      w.b = b, w.row0 = r.row0, w.n = r.n, w.len = r.len, w.ctx = r.ctx;
      w.key0 = (r.begin + jb) * kTreeKeys;
      w.head = item / r.pairs;
      w.node0 = (item - w.head * r.pairs) * TreeShape<D>::kQTiles * p.nodes;
      w.two = w.node0 + p.nodes < r.n && TreeShape<D>::kQTiles == 2;
      w.cut = jb > 0;
      w.whole = w.nt == r.tiles;
      return true;
    }
    return false;
  }
};

// What the join needs of an item that stretches cut, written by the CTA that has its last part.
struct TreeCut {
  int first;                           // CTA of the first part, its second one; those up to this CTA have their first (below 0: nothing to join)
  int row0, head, rows;                // output row of the first node, kv head, rows (node-major)
};

template <int D>
struct alignas(8) TreeBars {
  uint64_t q_full, q_empty, k_full[TreeShape<D>::kKeySlots], k_empty[TreeShape<D>::kKeySlots];
  uint64_t v_full[TreeShape<D>::kValueSlots], v_empty[TreeShape<D>::kValueSlots];
  uint64_t s_full[2][2], p_full[2][2], pv_done[2], drained[2], o_full, meet;
  uint64_t piece_full[kTreePieces], piece_empty[kTreePieces];
  TreePiece piece[kTreePieces];
  TreeCut cut;
  uint32_t tmem_base;
  TreeStart start;
  union {
    long long sums[kTreeThreads / 32];
    float rows[2][128];                // what the two threads of a row tell one another
  };
  uint32_t odd_any;
  int odd_tile[TreeShape<D>::kOdd];
  uint32_t odd[TreeShape<D>::kOdd][2]; // keys with a value that is not finite
};
template <int D>
constexpr int tree_smem() { return TreeShape<D>::kTiles + 1024 + (int)sizeof(TreeBars<D>); }
static_assert(tree_smem<64>() <= 227 * 1024 && tree_smem<128>() <= 227 * 1024 && tree_smem<256>() <= 227 * 1024, "shared memory of a CTA");

// A ring's slot and the parity of its use.
template <int N>
struct TreeSlot {
  int at = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void next() {
    if (++at == N) at = 0, parity ^= 1;
  }
  // After a wait that ran out: what was loaded last into each slot arrives before the CTA ends. (A slot without a load has the parity that does not wait.)
  __device__ __forceinline__ void drain(uint64_t* full, int* status) const {
    for (int i = 0; i < N; ++i) mbar_wait_warp(full + i, i < at ? parity : parity ^ 1, status);
  }
};
// The rows of the cache's tensor map that hold the tiles of a piece, one tile after the other: a lane holds the first row of each of 32 pages, the next 32 on their way.
// Pages outside the cache give rows behind it, which read as zeros.
struct TreePages {
  const int32_t* table;
  int bs, kv, per, num_blocks, last;   // per: pages of a tile
  int base, off, in_page, now, next;
  __device__ __forceinline__ int rows(int page) const {
    const int blk = table[min(page, last)];
    return ((blk < 0 || blk >= num_blocks ? num_blocks : blk) * 2 + kv) * bs;
  }
  __device__ __forceinline__ TreePages(const TreeParams& p, const TreePiece& w, int kv_)
      : table(p.block_table + w.b * p.ldt), bs(p.block_size), kv(kv_), per(max(1, kTreeKeys / p.block_size)), num_blocks((int)p.num_blocks),
        last(max(0, (w.len - 1) / p.block_size)), base(w.key0 / p.block_size), off(0), in_page(w.key0 - base * p.block_size) {
    const int lane = threadIdx.x & 31;
    now = rows(base + lane);
    next = rows(base + 32 + lane);
  }
  // One tile into `dst`; the whole warp calls it.
  template <int D>
  __device__ __forceinline__ void load(uint8_t* dst, const CUtensorMap* map, uint64_t* full, int head) {
    if (off == 32) {                   // (a tile's pages are a power of two: none passes the end)
      base += 32, off = 0;
      now = next;
      next = rows(base + 32 + (threadIdx.x & 31));
    }
    for (int x = 0; x < per; ++x) {
      const int row = __shfl_sync(0xffffffffu, now, off + x) + in_page;
      if (elect_one()) {
#pragma unroll
        for (int d = 0; d < D / 64; ++d) tma_load_3d(dst + d * TreeShape<D>::kPiece, map, full, d * 64, head, row);
      }
      __syncwarp();
      dst += bs * 128;
    }
    if (bs <= kTreeKeys) {
      off += per;
    } else if ((in_page += kTreeKeys) == bs) {
      in_page = 0;
      ++off;
    }
  }
};

__device__ __forceinline__ float tree_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// cap tanh(x / cap) of four scores in log2 units, y = x / cap: 1 - 2 / (1 + e^(2 y)), where one reciprocal of a product of four does for all (special functions bound
// the capped softmax: 64 dims, windows of 1024, 68 us with a reciprocal each). e^(2 y) stops at 2^30, past which the quotient is less than 2^-29. Off by 2^-21 of the
// cap, which is too much of one far above the scores (WIDE): small y take y - y^3 / 3 + 2 y^5 / 15 there, off by 2^-28 of itself below 1 / 16. A NaN makes all
// four one: hidden scores are 0 before.
template <bool WIDE>
__device__ __forceinline__ void tree_cap(uint32_t* s, float cap2, float to_2y) {
  float t[4], d[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    t[e] = __uint_as_float(s[e]) * to_2y;
    float x;
    asm("min.NaN.f32 %0, %1, 0f41f00000;" : "=f"(x) : "f"(t[e]));
    d[e] = 1.f + tree_ex2(x);
  }
  const float d01 = d[0] * d[1], d23 = d[2] * d[3];
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d01 * d23));
  r *= -2.f * cap2;
  const float r01 = r * d23, r23 = r * d01;
  const float q[4] = {r01 * d[1], r01 * d[0], r23 * d[3], r23 * d[2]};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float c = cap2 + q[e];
    if (WIDE) {
      const float y = t[e] * 0.34657359f, yy = y * y;
      if (fabsf(y) < 0.0625f) c = cap2 * y * fmaf(yy, fmaf(yy, 0.13333333f, -0.33333333f), 1.f);
    }
    s[e] = __float_as_uint(c);
  }
}
// Bits 15 and 31: which of two bf16 is not finite (an exponent of ones and one more passes into the sign's place).
__device__ __forceinline__ uint32_t odd_bf16x2(uint32_t w) { return (w & 0x7f807f80u) + 0x00800080u; }
// Of the four 16-byte pieces x of four neighbouring lanes, lane k gets the k-th of each: x[i] is lane i's.
__device__ __forceinline__ void tree_quads(uint4 (&x)[4]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int bit = 1; bit < 4; bit *= 2) {
    const bool up = lane & bit;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i & bit) continue;
      uint4& a = x[i];
      uint4& b = x[i | bit];
      const uint4 give = up ? a : b;
      uint4 get;
      get.x = __shfl_xor_sync(0xffffffffu, give.x, bit);
      get.y = __shfl_xor_sync(0xffffffffu, give.y, bit);
      get.z = __shfl_xor_sync(0xffffffffu, give.z, bit);
      get.w = __shfl_xor_sync(0xffffffffu, give.w, bit);
      a = up ? get : a;
      b = up ? b : get;
    }
  }
}

// Bits of the keys key .. key + 31 that a row sees. low: the first position in its window (INT_MIN: no window). The context's cells lie at their own positions, the
// nodes of the request at `positions`, behind the context: a window ends among them only where it is shorter than the tree is deep.
__device__ __forceinline__ uint32_t tree_seen(const uint64_t* mask, int words, const int64_t* positions, int key, int ctx, int len, int low) {
  const int rel = key - ctx;
  uint32_t v = 0xffffffffu;
  if (rel > -32) {
    const int from = max(rel, 0), a = from >> 6, sh = from & 63;
    uint64_t w = a < words ? __ldg(mask + a) >> sh : 0;
    if (sh > 32 && a + 1 < words) w |= __ldg(mask + a + 1) << (64 - sh);
    v = rel >= 0 ? (uint32_t)w : (uint32_t)w << -rel | ((1u << -rel) - 1);
  }
  if (len - key < 32) v &= len > key ? (1u << (len - key)) - 1 : 0;
  const int edge = min(low, ctx);
  if (key < edge) v &= edge - key < 32 ? ~((1u << (edge - key)) - 1) : 0;
  if (low > ctx && rel > -32) {        // (all of the context is hidden: what is left are nodes)
#pragma unroll 1
    for (uint32_t left = v; left; left &= left - 1)
      if (positions[rel + __ffs(left) - 1] < low) v &= ~(left & -left);
  }
  return v;
}

// CAP: with capped scores (a kernel of its own: the others lose 2 % to its code)
template <int D, bool CAP>
__global__ void __launch_bounds__(kTreeThreads, 1)
    tree_attn_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmKV, TreeParams p) {
  using Sh = TreeShape<D>;
  constexpr int K = kTreeKeys, kOdd = Sh::kOdd;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t *sK = sQ + Sh::kQTiles * Sh::kQTile, *sV = sK + Sh::kKeySlots * Sh::kSlot;
  TreeBars<D>& bars = *reinterpret_cast<TreeBars<D>*>(smem + Sh::kTiles);
  const int warp = warp_index(), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(&bars.q_full, 1);
    // What the issuers share they both take and both give back, tiles of the other warpgroup's too: a wait for one parity of a barrier is good for the
    // phase after the last one that the waiter has seen, and for no other. (Wide: one issuer gives back twice.)
    mbar_init(&bars.q_empty, 2);
    for (int i = 0; i < Sh::kKeySlots; ++i) {
      mbar_init(&bars.k_full[i], 1);
      mbar_init(&bars.k_empty[i], 2);
    }
    for (int i = 0; i < Sh::kValueSlots; ++i) {
      mbar_init(&bars.v_full[i], 1);
      mbar_init(&bars.v_empty[i], 2);
    }
    for (int t = 0; t < 2; ++t) {
      for (int b = 0; b < 2; ++b) {
        mbar_init(&bars.s_full[t][b], 1);
        mbar_init(&bars.p_full[t][b], Sh::kWide ? 8 : 4);
      }
      mbar_init(&bars.pv_done[t], 1);
      mbar_init(&bars.drained[t], 1);
    }
    mbar_init(&bars.o_full, 2);
    mbar_init(&bars.meet, 8);
    for (int i = 0; i < kTreePieces; ++i) {
      mbar_init(&bars.piece_full[i], 1);
      mbar_init(&bars.piece_empty[i], 11);
    }
    mbar_fence_init();
    bars.odd_any = 0;
    bars.cut.first = -1;
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmKV);
  }
  if (threadIdx.x < kOdd * 2) bars.odd[threadIdx.x >> 1][threadIdx.x & 1] = 0;
  if (warp == 10) {
    tmem_alloc(&bars.tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = bars.tmem_base;
  pdl_wait();
  pdl_launch_dependents();

  // ---- this CTA's stretch of the line
  const int per = (p.num_reqs + kTreeThreads - 1) / kTreeThreads;
  const int b0 = min(p.num_reqs, (int)threadIdx.x * per), b1 = min(p.num_reqs, b0 + per);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) {
    const TreeReq r = tree_req<D>(p, b);
    mine += (long long)r.items * (kTreeStart + r.tiles);
  }
  long long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) bars.sums[warp] = upto;
  __syncthreads();
  long long total = 0;
  for (int i = 0; i < kTreeThreads / 32; ++i) {
    if (i < warp) upto += bars.sums[i];
    total += bars.sums[i];
  }
  const long long stretch = max((total + gridDim.x - 1) / gridDim.x, (long long)kTreeLeast);
  const long long lo = min(total, stretch * blockIdx.x), hi = min(total, lo + stretch);
  if (lo < hi && upto - mine <= lo && lo < upto) {
    long long at = upto - mine;
    for (int b = b0; b < b1; ++b) {
      const TreeStart s{b, (int)(lo - at), p.q_start[b], p.q_start[b + 1], p.seq_lens[b]};
      const TreeReq r = tree_req<D>(p, s.begin, s.end, s.len);
      const long long cells = (long long)r.items * (kTreeStart + r.tiles);
      if (lo < at + cells) {
        bars.start = s;
        break;
      }
      at += cells;
    }
  }
  __syncthreads();

  if (warp == 8) {
    // ---------------- pieces, queries and keys ----------------
    TreeWalk<D> walk(p, bars.start, hi - lo);
    TreeSlot<Sh::kKeySlots> slot;
    uint32_t queries = 0;
    bool ok = true;
    for (uint32_t piece = 0; ok; ++piece) {
      TreePiece w;
      int jb = 0;
      const bool more = walk.next(w, jb);
      if (!more) w.nt = 0;
      const int at = piece % kTreePieces;
      if (piece >= kTreePieces && !(ok = mbar_wait_warp(&bars.piece_empty[at], (piece / kTreePieces - 1) & 1, p.status))) break;
      if (lane == 0) {
        bars.piece[at] = w;
        if (more && w.cut && jb + w.nt == walk.r.tiles) {
          // the last part of an item that began in the stretch of another CTA: of the one that has the line's cell of its first tile
          bars.cut.first = (int)((lo - jb) / stretch);
          bars.cut.row0 = w.row0 + w.node0;
          bars.cut.head = w.head;
          bars.cut.rows = min(w.n - w.node0, p.nodes * (w.two ? 2 : 1)) * p.G;
        }
        mbar_arrive(&bars.piece_full[at]);
      }
      __syncwarp();
      if (!more) break;
      TreePages pages(p, w, 0);
      if (piece > 0 && !(ok = mbar_wait_warp(&bars.q_empty, (piece - 1) & 1, p.status))) break;
      const int row = w.row0 + w.node0, tiles = w.two ? 2 : 1;
      ++queries;
      if (lane == 0) mbar_expect_tx(&bars.q_full, tiles * Sh::kParts * p.nodes * p.G * 128);
      __syncwarp();
      if (lane < tiles * Sh::kParts) {
        const int t = lane / Sh::kParts, part = lane % Sh::kParts;
        tma_load_3d(sQ + t * Sh::kQTile + part * 16384, &tmQ, &bars.q_full, part * 64, w.head * p.G, row + t * p.nodes);
      }
      __syncwarp();
      for (int j = 0; j < w.nt; ++j, slot.next()) {
        if (!(ok = mbar_wait_warp(&bars.k_empty[slot.at], slot.parity ^ 1, p.status))) break;
        if (elect_one()) mbar_expect_tx(&bars.k_full[slot.at], Sh::kSlot);
        __syncwarp();
        pages.load<D>(sK + slot.at * Sh::kSlot, &tmKV, &bars.k_full[slot.at], w.head);
      }
    }
    if (!ok) {
      slot.drain(bars.k_full, p.status);
      if (queries) mbar_wait_warp(&bars.q_full, (queries - 1) & 1, p.status);
    }
  } else if (warp == 9) {
    // ---------------- values ----------------
    TreeSlot<Sh::kValueSlots> slot;
    bool ok = true;
    for (uint32_t piece = 0; ok; ++piece) {
      const int at = piece % kTreePieces;
      if (!(ok = mbar_wait_warp(&bars.piece_full[at], (piece / kTreePieces) & 1, p.status))) break;
      const TreePiece w = bars.piece[at];
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.piece_empty[at]);
      if (w.nt == 0) break;
      TreePages pages(p, w, 1);
      for (int j = 0; j < w.nt; ++j, slot.next()) {
        if (!(ok = mbar_wait_warp(&bars.v_empty[slot.at], slot.parity ^ 1, p.status))) break;
        if (elect_one()) mbar_expect_tx(&bars.v_full[slot.at], Sh::kSlot);
        __syncwarp();
        pages.load<D>(sV + slot.at * Sh::kSlot, &tmKV, &bars.v_full[slot.at], w.head);
      }
    }
    if (!ok) slot.drain(bars.v_full, p.status);
  } else if (warp >= 10) {
    // ---------------- MMA of warpgroup t ----------------
    constexpr uint32_t idesc_qk = umma_idesc_bf16(128, K, 0, 0), idesc_pv = umma_idesc_bf16(128, D, 0, 1);
    // Descriptors of the first operand tiles; the others' lie a constant further (their addresses, in 16 bytes, are the lowest bits).
    const int t = warp - 10;
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t q_desc = umma_desc_k_sw128(smem_u32(sQ), 1024), k_desc = umma_desc_k_sw128(smem_u32(sK), 1024);
    const uint64_t v_desc = umma_desc_mn_sw128(smem_u32(sV), Sh::kPiece, 1024);
    TreeSlot<Sh::kKeySlots> ks;
    TreeSlot<Sh::kValueSlots> vs;
    uint32_t c_k = 0, c_v = 0;         // tiles of this warpgroup: scores issued, products issued
    bool ok = true;
    for (uint32_t piece = 0; ok; ++piece) {
      const int at = piece % kTreePieces;
      if (!(ok = mbar_wait_warp(&bars.piece_full[at], (piece / kTreePieces) & 1, p.status))) break;
      const int nt = __shfl_sync(0xffffffffu, bars.piece[at].nt, 0);
      const bool two = __shfl_sync(0xffffffffu, (int)bars.piece[at].two, 0) != 0;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.piece_empty[at]);
      if (nt == 0) break;
      if (Sh::kWide && t == 1) continue;                           // (there is one accumulator: the other warp has it all)
      const bool both = Sh::kWide || two;                          // every tile for every warpgroup
      const int ahead = both ? 2 : 4, last = both ? nt - 1 : nt - 1 - ((nt - 1 - t) & 1);          // this warpgroup's last tile (below 0: none)
      if (!(ok = mbar_wait_warp(&bars.q_full, piece & 1, p.status))) break;
      if (last < 0) {                  // (for this piece's output, not for one before it that the other issuer is still at)
        if (lane == 0) mbar_arrive(&bars.q_empty);
        if (piece > 0 && !(ok = mbar_wait_warp(&bars.o_full, (piece - 1) & 1, p.status))) break;
        if (lane == 0) mbar_arrive(&bars.o_full);
      }
      const uint64_t q = q_desc + (two ? t : 0) * (Sh::kQTile >> 4);
      const auto qk = [&](int j) {     // scores of tile j
        if (!mbar_wait_warp(&bars.k_full[ks.at], ks.parity, p.status)) return false;
        if (both || (j & 1) == t) {
          tc_fence_after_sync();
          const uint64_t k = k_desc + ks.at * (Sh::kSlot >> 4);
          const uint32_t buf = c_k & 1, s_at = tm + (t * 2 + buf) * K;
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              umma_bf16_ss(s_at, q + (((kk / 4) * 16384 + (kk % 4) * 32) >> 4), k + (((kk / 4) * Sh::kPiece + (kk % 4) * 32) >> 4), idesc_qk, kk != 0);
            umma_commit(&bars.s_full[t][buf]);
            umma_commit(&bars.k_empty[ks.at]);
            if (j == last) umma_commit(&bars.q_empty);
            if (Sh::kWide) {
              umma_commit(&bars.k_empty[ks.at]);
              if (j == last) umma_commit(&bars.q_empty);
            }
          }
          ++c_k;
        } else if (lane == 0) {
          mbar_arrive(&bars.k_empty[ks.at]);
        }
        __syncwarp();
        ks.next();
        return true;
      };
      for (int j = 0; ok && j < min(ahead, nt); ++j) ok = qk(j);
      for (int j = 0; ok && j < nt; ++j, vs.next()) {
        if (!(ok = mbar_wait_warp(&bars.v_full[vs.at], vs.parity, p.status))) break;
        if (both || (j & 1) == t) {
          const uint32_t buf = c_v & 1;
          if (!(ok = mbar_wait_warp(&bars.p_full[t][buf], c_v >> 1 & 1, p.status))) break;
          const bool first = j < (both ? 1 : 2);                   // (the accumulator is free: the weights come from warps that have met at the last output's end)
          tc_fence_after_sync();
          const uint64_t v = v_desc + vs.at * (Sh::kSlot >> 4);
          const uint32_t p_at = Sh::kWide ? tm + Sh::kP + buf * 32 : tm + (t * 2 + buf) * K, o_at = tm + Sh::kO + t * D;
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < K / 16; ++kk) umma_bf16_ts(o_at, p_at + kk * 8, v + kk * (2048 >> 4), idesc_pv, !first || kk != 0);
            umma_commit(&bars.v_empty[vs.at]);
            umma_commit(&bars.pv_done[t]);
            if (j == last) umma_commit(&bars.o_full);
            if (Sh::kWide) {
              umma_commit(&bars.v_empty[vs.at]);
              if (j == last) umma_commit(&bars.o_full);
            }
          }
          ++c_v;
        } else if (lane == 0) {
          mbar_arrive(&bars.v_empty[vs.at]);
        }
        __syncwarp();
        if (j + ahead < nt) ok = qk(j + ahead);                    // (the tile after this warpgroup's next: the same buffer)
      }
    }
    if (!ok) {                         // a wait ran out: nothing of this issuer's is under way when the CTA ends
      if (elect_one()) umma_commit(&bars.drained[t]);
      __syncwarp();
      mbar_wait_warp(&bars.drained[t], 0, p.status);
    }
  } else {
    // ---------------- softmax and output: a thread a row (two where it is wide) ----------------
    const int half = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane, t = Sh::kWide ? 0 : half;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    // scores as they come -> 2 y log2(e); finite, as a score of 0 times it is 0 however small the cap is
    const float cap_in = CAP ? fminf(p.scale_log2 * fminf(2.8853900817779268f / p.cap2, 3.0e38f), 3.0e38f) : 0.f;
    const int row_node = r / p.G, row_head = r - row_node * p.G;
    uint32_t tiles0 = 0, piece = 0, made = 0, met = 0;       // tiles of V in the pieces before
    bool ok = true;
    const auto meet = [&]() {           // both warpgroups
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.meet);
      return __all_sync(0xffffffffu, mbar_wait(&bars.meet, met++ & 1, p.status));
    };
    for (;; ++piece) {
      const int at = piece % kTreePieces;
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(&bars.piece_full[at], (piece / kTreePieces) & 1, p.status)))) break;
      const TreePiece w = bars.piece[at];
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.piece_empty[at]);
      if (w.nt == 0) break;
      const int node = w.node0 + (w.two ? half * p.nodes : 0) + row_node;
      const bool there = row_node < p.nodes && node < w.n;
      const bool idle = !__any_sync(0xffffffffu, there);               // (its rows may hold anything: no other warp reads them)
      const uint64_t* bits = p.mask + (size_t)(w.row0 + (there ? node : 0)) * p.words;
      int low = INT_MIN;
      if (p.window > 0 && there) {     // (a node lies at most n - 1 positions behind the root)
        const long long depth = p.positions[w.row0 + node] - w.ctx;
        low = w.ctx + (int)min(max(depth, 0ll), (long long)w.n - 1) - p.window + 1;
      }
      const auto seen_word = [&](int key) { return there ? tree_seen(bits, p.words, p.positions + w.row0, key, w.ctx, w.len, low) : 0u; };
      // tiles in which the nodes of the request may differ in what they see: up to where a window begins for all of them, and from the context's end on
      const int odd_to = p.window > 0 ? w.ctx - p.window + w.n - w.key0 : INT_MIN, odd_from = w.ctx - w.key0 - K + 1;
      float m = -INFINITY, l = 0.f;
      int odd_n = 0;
      const bool both = Sh::kWide || w.two;
      const int mine = both ? w.nt : (w.nt + 1 - half) / 2;            // tiles of this warpgroup
      for (int i = 0; i < mine; ++i) {
        const int j = both ? i : 2 * i + half, at0 = j * K, kbase = w.key0 + at0;
        const uint32_t c = made + i, buf = c & 1;
        const bool odd_tile = at0 >= odd_from || at0 < odd_to;
        uint32_t seen[2] = {0xffffffffu, 0xffffffffu};
        if (odd_tile) {
          seen[0] = seen_word(kbase);
          seen[1] = seen_word(kbase + 32);
        }
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(&bars.s_full[t][buf], c >> 1 & 1, p.status)))) break;
        if (!idle) {
          tc_fence_after_sync();
          const uint32_t s_addr = tmem + (t * 2 + buf) * K + lanes;
          uint32_t s[64];
          tmem_ld_32x32b_x32(s_addr, s);
          tmem_ld_32x32b_x32(s_addr + 32, s + 32);
          tmem_ld_wait();
          float sc = p.scale_log2;
          if constexpr (CAP) {
            if (odd_tile) {
#pragma unroll
              for (int e = 0; e < 64; ++e)
                if (!(seen[e >> 5] >> (e & 31) & 1)) s[e] = 0;
            }
            if (p.cap2 <= kTreeWideCap) {
#pragma unroll
              for (int e = 0; e < 64; e += 4) tree_cap<false>(s + e, p.cap2, cap_in);
            } else {
#pragma unroll
              for (int e = 0; e < 64; e += 4) tree_cap<true>(s + e, p.cap2, cap_in);
            }
            sc = 1.f;
          }
          if (odd_tile) {
#pragma unroll
            for (int e = 0; e < 64; ++e)
              if (!(seen[e >> 5] >> (e & 31) & 1)) s[e] = 0xff800000u;       // -inf
          }
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int e = 0; e < 64; e += 4)
#pragma unroll
            for (int g = 0; g < 4; ++g) mx[g] = fmaxf(mx[g], __uint_as_float(s[e + g]));
          // m: reference of the row's maximum, raised lazily (by more than 2^8), so that the accumulator is rescaled rarely; P stays below 256
          const float tile_max = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sc;
          float alpha = 1.f;
          bool rescale = false;
          if (tile_max > m + 8.f) {    // also the first finite tile: m == -inf
            if (m != -INFINITY) {
              alpha = tree_ex2(m - tile_max);
              rescale = true;
            }
            m = tile_max;
          }
          const float m_use = m == -INFINITY ? 0.f : m;
          if (__any_sync(0xffffffffu, rescale)) {
            // the product of the tile before may be under way (its successor waits for this tile's weights)
            if (!(ok = __all_sync(0xffffffffu, mbar_wait(&bars.pv_done[t], (c - 1) & 1, p.status)))) break;
            tc_fence_after_sync();
            constexpr int cols = Sh::kWide ? D / 2 : D;
            const uint32_t o_addr = tmem + Sh::kO + half * cols + lanes;
#pragma unroll 1
            for (int x = 0; x < cols / 16; ++x) {
              uint32_t rr[16];
              tmem_ld_32x32b_x16(o_addr + x * 16, rr);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; ++e) rr[e] = __float_as_uint(__uint_as_float(rr[e]) * alpha);
              tmem_st_32x32b_x16(o_addr + x * 16, rr);
            }
          }
          // The sum is that of the rounded values: a row's weights add up to one, and a single key's value comes out as it is.
          const uint64_t sc2 = pack_f32x2(sc, sc), off2 = pack_f32x2(-m_use, -m_use);
          uint64_t sum2[2] = {0, 0};
          constexpr int kMine = Sh::kWide ? 32 : 64;
          uint32_t pk[kMine / 2];
#pragma unroll
          for (int e = 0; e < kMine / 2; ++e) {
            const uint32_t x0 = Sh::kWide && half ? s[(32 + 2 * e) & 63] : s[2 * e], x1 = Sh::kWide && half ? s[(33 + 2 * e) & 63] : s[2 * e + 1];
            float a, b;
            unpack_f32x2(fma_f32x2(pack_b32x2(x0, x1), sc2, off2), a, b);
            pk[e] = pack_bf16x2(tree_ex2(a), tree_ex2(b));
            sum2[e & 1] = add_f32x2(sum2[e & 1], pack_b32x2(pk[e] << 16, pk[e] & 0xffff0000u));
          }
          if constexpr (Sh::kWide) tmem_st_32x32b_x16(tmem + Sh::kP + buf * 32 + half * 16 + lanes, pk);
          else tmem_st_32x32b_x32(s_addr, pk);
          float sum[4];
          unpack_f32x2(sum2[0], sum[0], sum[1]);
          unpack_f32x2(sum2[1], sum[2], sum[3]);
          l = l * alpha + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
        }
        if (odd_tile && (!Sh::kWide || half == 0)) {
          // Values that are not finite: out of the tile, and noted. A thread takes half of a key's dims. (Where both warpgroups take the tile each does all of
          // it ahead of its own product; they write the same.)
          const uint32_t v = tiles0 + j;
          if (!(ok = __all_sync(0xffffffffu, mbar_wait(&bars.v_full[v % Sh::kValueSlots], (v / Sh::kValueSlots) & 1, p.status)))) break;
          const int key = r & 63;
          uint8_t* row = sV + (v % Sh::kValueSlots) * Sh::kSlot + key * 128;
          const auto at16 = [&](int x) {
            const int piece16 = (r >> 6) * (D / 16) + x;
            return reinterpret_cast<uint4*>(row + (piece16 >> 3) * Sh::kPiece + (((piece16 & 7) ^ (key & 7)) << 4));
          };
          uint32_t any = 0;
#pragma unroll
          for (int x = 0; x < D / 16; ++x) {
            const uint4 y = *at16(x);
            any |= odd_bf16x2(y.x) | odd_bf16x2(y.y) | odd_bf16x2(y.z) | odd_bf16x2(y.w);
          }
          const bool odd = (any & 0x80008000u) != 0;
          if (odd) {
#pragma unroll 1
            for (int x = 0; x < D / 16; ++x) {
              const uint4 y = *at16(x);
              uint32_t e[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                if ((e[g] & 0x7f80u) == 0x7f80u) e[g] &= 0xffff0000u;
                if ((e[g] & 0x7f800000u) == 0x7f800000u) e[g] &= 0xffffu;
              }
              *at16(x) = make_uint4(e[0], e[1], e[2], e[3]);
            }
          }
          fence_proxy_async_smem();
          const uint32_t who = __ballot_sync(0xffffffffu, odd);
          const int most = both ? kOdd : kOdd / 2;                     // (notes that there is room for: all, but of requests with nodes that are left out)
          if (who && lane == 0 && odd_n < most) {
            const int note = (both ? 0 : half * most) + odd_n;
            bars.odd_tile[note] = kbase;
            atomicOr(&bars.odd[note][quarter & 1], who);
            atomicOr(&bars.odd_any, 1u);
          }
          ++odd_n;
        }
        tmem_st_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.p_full[t][buf]);
      }
      if (!ok) break;
      tiles0 += w.nt;
      made += mine;
      // ---- output
      const bool other = !both && w.nt > 1;            // both warpgroups have a share of every row
      if (!w.two && half == 1) {
        bars.rows[0][r] = m;
        bars.rows[1][r] = l;
      }
      if (!(ok = meet())) break;
      float a0 = 1.f, a1 = 0.f;        // factors of the two accumulators
      if (!w.two) {
        if (half == 0) {
          const float l1 = bars.rows[1][r];
          if (Sh::kWide) {             // (one accumulator; the row's weights in two sums)
            l += l1;
          } else if (other) {
            const float m0 = m, m1 = bars.rows[0][r];
            m = fmaxf(m0, m1);
            // (a share of which the row sees nothing has sums of 0, or of NaN that stay)
            a0 = m0 == -INFINITY ? 1.f : tree_ex2(m0 - m);
            a1 = m1 == -INFINITY ? 1.f : tree_ex2(m1 - m);
            l = l * a0 + l1 * a1;
          }
          if (w.whole) {
            const float inv = l != 0.f ? 1.f / l : 0.f;
            a0 *= inv;
            a1 *= inv;
          }
          bars.rows[0][r] = a0;
          bars.rows[1][r] = a1;
        }
        if (!(ok = meet())) break;
        a0 = bars.rows[0][r];
        a1 = bars.rows[1][r];
      } else if (w.whole) {
        a0 = l != 0.f ? 1.f / l : 0.f;
      }
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(&bars.o_full, piece & 1, p.status)))) break;
      tc_fence_after_sync();
      const bool odd_any = *(volatile uint32_t*)&bars.odd_any != 0;
      if (!idle) {
        // columns of this thread's: all of its row's, or one half of them
        constexpr int kHalfCols = D / 2;
        const int col0 = w.two ? 0 : half * kHalfCols, cols = w.two ? D : kHalfCols;
        const int part_row = w.two ? half * 128 + r : r;
        const uint32_t o_addr = tmem + Sh::kO + lanes + (w.two ? half * D : 0);
        __nv_bfloat16* dst = p.out + (w.row0 + node) * p.ldo + (w.head * p.G + row_head) * D;
        float* part = p.parts + (2 * blockIdx.x + (w.cut ? 0 : 1)) * Sh::kPartFloats;
        // (four lanes write 64 bytes of a row together: 16 bytes of 32 rows each would take the store unit four times as long)
        __nv_bfloat16* quad[4];
        if (w.whole) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            quad[i] = reinterpret_cast<__nv_bfloat16*>(__shfl_sync(0xffffffffu, there ? reinterpret_cast<unsigned long long>(dst) : 0ull, (lane & 28) + i));
        }
#pragma unroll 1
        for (int x = 0; x < cols; x += 32) {
          uint32_t rr[32], r1[32];
          tmem_ld_32x32b_x32(o_addr + col0 + x, rr);
          if (other) tmem_ld_32x32b_x32(o_addr + D + col0 + x, r1);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const float o = __uint_as_float(rr[e]) * a0;
            rr[e] = __float_as_uint(other ? fmaf(__uint_as_float(r1[e]), a1, o) : o);
          }
          if (odd_any && there) {
            for (int note = 0; note < kOdd; ++note) {
              for (int q = 0; q < 2; ++q) {
                uint32_t who = bars.odd[note][q];
                if (who == 0) continue;
                who &= seen_word(bars.odd_tile[note] + 32 * q);
                while (who) {
                  const int key = bars.odd_tile[note] + 32 * q + __ffs(who) - 1;
                  who &= who - 1;
                  const int blk = p.block_table[w.b * p.ldt + key / p.block_size];
                  if (blk < 0 || blk >= p.num_blocks) continue;
                  const __nv_bfloat16* v = p.cache + ((((long long)blk * 2 + 1) * p.block_size + key % p.block_size) * p.Hkv + w.head) * D + col0 + x;
#pragma unroll
                  for (int e = 0; e < 32; ++e) {
                    const float y = __bfloat162float(v[e]);
                    if (!(fabsf(y) <= 3.4028234e38f)) rr[e] = __float_as_uint(__uint_as_float(rr[e]) + y);
                  }
                }
              }
            }
          }
          if (w.whole) {
            uint4 o[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const uint32_t* e = rr + 8 * g;
              o[g].x = pack_bf16x2(__uint_as_float(e[0]), __uint_as_float(e[1]));
              o[g].y = pack_bf16x2(__uint_as_float(e[2]), __uint_as_float(e[3]));
              o[g].z = pack_bf16x2(__uint_as_float(e[4]), __uint_as_float(e[5]));
              o[g].w = pack_bf16x2(__uint_as_float(e[6]), __uint_as_float(e[7]));
            }
            tree_quads(o);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (quad[i]) *reinterpret_cast<uint4*>(quad[i] + col0 + x + (lane & 3) * 8) = o[i];
          } else if (there) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<uint4*>(part + ((size_t)((col0 + x + e) >> 2) * Sh::kRows + part_row) * 4) = make_uint4(rr[e], rr[e + 1], rr[e + 2], rr[e + 3]);
          }
        }
        if (!w.whole && there && (w.two || half == 0)) {
          part[(size_t)Sh::kRows * D + part_row] = m;
          part[(size_t)Sh::kRows * D + Sh::kRows + part_row] = l;
        }
      }
      tc_fence_before_sync();
      if (odd_any) {                   // everyone has read the notes: they go
        if (!(ok = meet())) break;
        const int x = threadIdx.x;
        if (x < kOdd * 2) bars.odd[x >> 1][x & 1] = 0;
        if (x == 0) bars.odd_any = 0;
      }
      // (what the threads of a row told one another, the notes and the accumulators are written anew when everyone has read them)
      if (!(ok = meet())) break;
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 10) tmem_dealloc(tmem, 512);
  if (threadIdx.x == 0) reinterpret_cast<TreeCut*>(p.parts + 2 * (long long)gridDim.x * Sh::kPartFloats)[blockIdx.x] = bars.cut;
}

// Parts of items that the ends of stretches cut. Block (b, y): 32 rows of the item whose last part is CTA b's, a lane a row, a warp every eighth four columns.
template <int D>
__global__ void __launch_bounds__(256)
    tree_join_kernel(const float* __restrict__ parts, int ctas, __nv_bfloat16* __restrict__ out, long long ldo, int G, int nodes) {
  using Sh = TreeShape<D>;
  constexpr int kQuads = D / 32;
  pdl_wait();
  pdl_launch_dependents();
  const TreeCut cut = reinterpret_cast<const TreeCut*>(parts + 2 * (long long)ctas * Sh::kPartFloats)[blockIdx.x];
  if (cut.first < 0) return;
  const int warp = threadIdx.x >> 5, row = blockIdx.y * 32 + (threadIdx.x & 31), count = (int)blockIdx.x - cut.first + 1;
  const int i = (row >> 7) * nodes * G + (row & 127);          // node-major
  if ((row & 127) >= nodes * G || i >= cut.rows) return;
  const auto part = [&](int c) { return parts + (2ll * (cut.first + c) + (c == 0)) * Sh::kPartFloats; };
  float top = -INFINITY;
#pragma unroll 4
  for (int c = 0; c < count; ++c) top = fmaxf(top, part(c)[(size_t)Sh::kRows * D + row]);
  float4 acc[kQuads] = {};
  float total = 0.f;
#pragma unroll 2
  for (int c = 0; c < count; ++c) {
    const float* at = part(c);
    const float m = at[(size_t)Sh::kRows * D + row], l = at[(size_t)Sh::kRows * D + Sh::kRows + row];
    const float a = m == -INFINITY ? 1.f : tree_ex2(m - top);  // (nothing seen: sums of 0, or of NaN that stay)
    total = fmaf(l, a, total);
#pragma unroll
    for (int k = 0; k < kQuads; ++k) {
      const float4 v = reinterpret_cast<const float4*>(at)[(size_t)(warp + 8 * k) * Sh::kRows + row];
      acc[k].x = fmaf(v.x, a, acc[k].x);
      acc[k].y = fmaf(v.y, a, acc[k].y);
      acc[k].z = fmaf(v.z, a, acc[k].z);
      acc[k].w = fmaf(v.w, a, acc[k].w);
    }
  }
  const float inv = total != 0.f ? 1.f / total : 0.f;
  const int node = i / G, head = i - node * G;
  uint2* dst = reinterpret_cast<uint2*>(out + (cut.row0 + node) * ldo + (cut.head * G + head) * D);
#pragma unroll
  for (int k = 0; k < kQuads; ++k)
    dst[warp + 8 * k] = make_uint2(pack_bf16x2(acc[k].x * inv, acc[k].y * inv), pack_bf16x2(acc[k].z * inv, acc[k].w * inv));
}

template <int D, bool CAP>
static int launch_tree(const CUtensorMap& tmQ, const CUtensorMap& tmKV, const TreeParams& p, int ctas, cudaStream_t stream) {
  static PerDeviceOnce once;
  if (once.first()) cudaFuncSetAttribute(tree_attn_kernel<D, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, tree_smem<D>());
  if (launch_pdl(tree_attn_kernel<D, CAP>, dim3(ctas), dim3(kTreeThreads), tree_smem<D>(), stream, tmQ, tmKV, p) != cudaSuccess) return -2;
  return launch_pdl(tree_join_kernel<D>, dim3(ctas, TreeShape<D>::kRows / 32), dim3(256), 0, stream, (const float*)p.parts, ctas, p.out, p.ldo,
                    p.G, p.nodes) == cudaSuccess ? 0 : -2;
}

}  // namespace b200

using namespace b200;

// What a call takes, as far as sizes say: 0, or -1 (shape) or -4 (counted in 31 bits: key tiles of all items of a request).
extern "C" int b200_tree_attn_takes(const B200TreeAttn* a) {
  const int D = a->D, keys = kTreeKeys;
  if (D != 64 && D != 128 && D != 256) return -1;
  if (a->Hkv <= 0 || a->Hq <= 0 || a->Hq % a->Hkv || a->Hq / a->Hkv > 128 || a->words <= 0 || a->max_blocks <= 0) return -1;
  const int bs = a->block_size;
  if (bs < 8 || bs % 8 || (bs < keys ? keys % bs : bs % keys)) return -1;
  if (a->num_reqs > kTreeReqs || a->words > kTreeNodes / 64) return -4;
  if (a->num_blocks >= (1ll << 31) / (2 * bs) - 1) return -4;
  const int nodes = 128 / (a->Hq / a->Hkv);
  const long long tiles = ((long long)a->max_blocks * bs + keys - 1) / keys + kTreeStart;
  const long long pairs = (std::min(a->total_q, kTreeNodes) + nodes - 1) / nodes + 1;
  return tiles * pairs >= (1ll << 31) / a->Hkv || (long long)a->max_blocks * bs > (1ll << 31) - 4096 ? -4 : 0;
}

extern "C" long long b200_tree_attn_scratch(int D) {
  const long long part = D == 64 ? TreeShape<64>::kPartFloats : D == 128 ? TreeShape<128>::kPartFloats : TreeShape<256>::kPartFloats;
  return 2 * part * b200_num_sms() + (long long)(sizeof(TreeCut) / 4) * b200_num_sms();
}

extern "C" int b200_tree_attn(const B200TreeAttn* a, cudaStream_t stream) {
  const int rc = b200_tree_attn_takes(a);
  if (rc) return rc;
  if (a->num_reqs <= 0 || a->total_q <= 0) return 0;
  const int D = a->D, keys = kTreeKeys, G = a->Hq / a->Hkv, bs = a->block_size;
  TreeParams p;
  p.cache = (const __nv_bfloat16*)a->cache; p.out = (__nv_bfloat16*)a->out; p.ldo = a->ldo;
  p.block_table = (const int32_t*)a->block_table; p.ldt = a->ldt; p.num_blocks = a->num_blocks; p.max_blocks = a->max_blocks;
  p.seq_lens = (const int32_t*)a->seq_lens; p.q_start = (const int32_t*)a->q_start;
  p.positions = (const int64_t*)a->positions; p.mask = (const uint64_t*)a->mask; p.words = a->words;
  p.num_reqs = a->num_reqs; p.total_q = a->total_q; p.Hkv = a->Hkv; p.G = G; p.nodes = 128 / G;
  p.block_size = bs; p.max_len = a->max_blocks * bs;
  p.window = a->positions && a->window <= p.max_len ? a->window : 0;         // (one that holds any context is none)
  p.scale_log2 = a->scale * 1.4426950408889634f; p.cap2 = a->softcap * 1.4426950408889634f;
  if (!(p.scale_log2 > 0.f && p.scale_log2 < INFINITY && p.cap2 >= 0.f && p.cap2 < INFINITY)) return -1;
  p.parts = (float*)a->parts; p.status = device_status_word();
  CUtensorMap tmQ, tmKV;
  if (!encode_tmap_3d(&tmQ, a->q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, (uint64_t)D, (uint64_t)a->Hq, (uint64_t)a->total_q, (uint64_t)D * 2,
                      (uint64_t)a->ldq * 2, 64, (uint32_t)G, (uint32_t)p.nodes, CU_TENSOR_MAP_SWIZZLE_128B))
    return -3;
  if (!encode_tmap_3d(&tmKV, a->cache, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, (uint64_t)D, (uint64_t)a->Hkv, (uint64_t)a->num_blocks * 2 * bs,
                      (uint64_t)D * 2, (uint64_t)a->Hkv * D * 2, 64, 1, (uint32_t)std::min(bs, keys), CU_TENSOR_MAP_SWIZZLE_128B))
    return -3;
  const int ctas = b200_num_sms();
  const auto launch = [&](auto dim) {
    constexpr int kD = decltype(dim)::value;
    return p.cap2 > 0.f ? launch_tree<kD, true>(tmQ, tmKV, p, ctas, stream) : launch_tree<kD, false>(tmQ, tmKV, p, ctas, stream);
  };
  return D == 64 ? launch(std::integral_constant<int, 64>()) : D == 128 ? launch(std::integral_constant<int, 128>()) : launch(std::integral_constant<int, 256>());
}
