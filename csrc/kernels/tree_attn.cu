// Attention of trees of drafted tokens over a paged bf16 cache (tcgen05 / TMEM), head_dim 64, 128 or 256.
//
//   o_i = sum_k p_ik v_k,  p_i = softmax over the keys k that node i sees of cap(scale q_i . k_k)
//
// A request has a context of c cells and n nodes whose keys and values lie behind it (node j at position c + j). Node i sees the context (its last
// `window` positions, if there is a window) and the nodes whose bits are set in its mask. A node that sees nothing gives zeros.
//
// Bound: a node's G query heads of a kv head share every key and value, so that rows = n G rows of scores read 4 D bytes a key once: with up to
// 256 rows a request the cache's bytes are the floor, above it the products and exponentials. Rows are therefore the 128-row operand (a thread
// owns a row: no sums across threads), keys the other one, and a CTA takes two tiles of rows against each tile of keys. Where a request
// has only one tile of rows, its two halves (a warpgroup, a score and an output accumulator each) take every second tile of keys
// instead and are added at the end: the same two chains of products and softmax in flight, with half the bytes' work each.
//
// Work: the key tiles of all items (request, kv head, two tiles of rows) stand in one line, each CTA (one an SM) takes an equal stretch of it, whatever the
// lengths; an item's start (queries, output) stands in the line as kStart tiles. Parts of items that a stretch's end cuts go to scratch and a short
// kernel joins them, in a fixed order.
//
// What a node does not see does not reach it: hidden scores become -inf before the softmax, and values are inspected in the tiles where nodes
// differ in what they see (the product would multiply an infinity or NaN by 0): what is not finite is taken out there and added at
// the end to the nodes that see it.
//
// Warp roles (320 threads): warp 0 TMA, warp 1 MMA + TMEM owner, warps 2..5 / 6..9 softmax and output.
#include <limits.h>

#include <algorithm>
#include <mutex>
#include <unordered_map>

#include "api.h"
#include "sm100.cuh"

namespace b200 {

static constexpr int kTreeThreads = 320, kTreeReqs = 8192, kTreeNodes = 1024;       // (the last two: at most)
static constexpr int kTreeStart = 3;          // what an item's start costs, in key tiles
static constexpr int kTreeLeast = 2;          // tiles of a stretch at the least

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
  static constexpr int kKeys = kWide ? 64 : 128;
  static constexpr int kParts = D / 64;                // 64-dim pieces of a row
  static constexpr int kSlot = kKeys * D * 2, kPiece = kKeys * 128;
  static constexpr int kRing = D == 64 ? 10 : 5;
  static constexpr int kQTile = 128 * D * 2, kQTiles = kWide ? 1 : 2;
  static constexpr int kTiles = kQTiles * kQTile + kRing * kSlot;
  static constexpr int kRows = 128 * kQTiles;
  static constexpr long long kPartFloats = (long long)kRows * D + 2 * kRows;
  // tensor memory: scores of two tiles, accumulators (two; one and the two tiles' P where it is wide)
  static constexpr int kSCols = kKeys, kO = 2 * kKeys, kP = kWide ? 384 : 0;
  // tiles of a piece in which nodes may differ in what they see: those of 1024 nodes, and where a window ends those of 1024 positions
  static constexpr int kOdd = 2 * (kTreeNodes / kKeys + 2), kWords = kKeys / 32;
};

struct TreeReq {
  int n, row0, len, ctx, begin, tiles, pairs, items;   // begin: first key tile; tiles: key tiles; pairs: items of a kv head
};
template <int D>
__device__ __forceinline__ TreeReq tree_req(const TreeParams& p, int b) {
  TreeReq r;
  r.row0 = min(max(p.q_start[b], 0), p.total_q);
  r.n = max(0, min(p.q_start[b + 1], p.total_q) - r.row0);
  r.len = min(max(p.seq_lens[b], 0), p.max_len);
  r.ctx = r.len - r.n;
  const int low = p.window > 0 ? max(0, r.ctx - p.window + 1) : 0;
  constexpr int K = TreeShape<D>::kKeys;
  r.begin = min(low, max(r.len - 1, 0)) / K;
  r.tiles = max(1, (r.len + K - 1) / K - r.begin);     // (no keys: a tile that nobody sees)
  const int row_tiles = (r.n + p.nodes - 1) / p.nodes;
  r.pairs = (row_tiles + TreeShape<D>::kQTiles - 1) / TreeShape<D>::kQTiles;
  r.items = r.pairs * p.Hkv;
  return r;
}

// The pieces of a CTA's stretch, one after the other; every role walks them for itself.
struct TreePiece {
  int head, node0, jb, je;             // kv head, first node, key tiles [jb, je) of the item's
  bool two;                            // a second tile of rows
};
template <int D>
struct TreeWalk {
  const TreeParams& p;
  TreeReq r;
  int b, off;                          // request, cells of it that are behind
  long long left;                      // cells of the stretch
  __device__ __forceinline__ TreeWalk(const TreeParams& p_, int b_, int off_, long long left_) : p(p_), b(b_), off(off_), left(left_) {
    if (left > 0) r = tree_req<D>(p, b);
  }
  __device__ __forceinline__ bool next(TreePiece& w) {
    while (left > 0) {
      const int cells = kTreeStart + r.tiles;
      if (off >= r.items * cells) {
        if (++b >= p.num_reqs) return false;
        r = tree_req<D>(p, b);
        off = 0;
        continue;
      }
      const int item = off / cells, o = off - item * cells;
      const int take = (int)min((long long)(cells - o), left);
      off += take;
      left -= take;
      w.jb = max(0, o - kTreeStart);
      w.je = max(0, o + take - kTreeStart);
      if (w.je <= w.jb) continue;
      w.head = item / r.pairs;
      w.node0 = (item - w.head * r.pairs) * TreeShape<D>::kQTiles * p.nodes;
      w.two = w.node0 + p.nodes < r.n && TreeShape<D>::kQTiles == 2;
      return true;
    }
    return false;
  }
};

// What the join needs of an item that stretches cut, written by the CTA that has its last part.
struct TreeCut {
  int first, last;                     // CTAs; the first's part is its second, the others' their first (first < 0: nothing to join)
  int row0, head, rows;                // output row of the first node, kv head, rows (node-major)
};

template <int D>
struct alignas(8) TreeBars {
  uint64_t q_full, q_empty, kv_full[TreeShape<D>::kRing], kv_empty[TreeShape<D>::kRing];
  uint64_t s_full[2], p_full[2], o_full, o_free, pv_done, meet;
  uint32_t tmem_base;
  int start_req, start_off;
  long long sums[kTreeThreads / 32];
  float rows[2][128];                  // what the two threads of a row tell one another
  uint32_t odd_any;
  int odd_tile[TreeShape<D>::kOdd];
  uint32_t odd[TreeShape<D>::kOdd][TreeShape<D>::kWords];     // keys with a value that is not finite
};
template <int D>
constexpr int tree_smem() { return TreeShape<D>::kTiles + 1024 + (int)sizeof(TreeBars<D>); }
static_assert(tree_smem<64>() <= 227 * 1024 && tree_smem<128>() <= 227 * 1024 && tree_smem<256>() <= 227 * 1024, "shared memory of a CTA");

__device__ __forceinline__ float tree_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// cap tanh(x / cap) in log2 units, y = x / cap: 1 - 2 / (1 + e^(2 y)) is off by 2^-22 of the cap, which is too much of one far above the scores; small y
// take y - y^3 / 3 + 2 y^5 / 15, off by 2^-28 of itself below 1 / 16.
__device__ __forceinline__ float tree_capped(float x, float cap2, float to_2y) {
  const float t = x * to_2y, y = t * 0.34657359f, yy = y * y;
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + tree_ex2(t)));
  return fabsf(y) < 0.0625f ? cap2 * y * fmaf(yy, fmaf(yy, 0.13333333f, -0.33333333f), 1.f) : fmaf(-2.f * cap2, r, cap2);
}
// The registers of a load from tensor memory may be read after this.
__device__ __forceinline__ void tmem_ld_wait_for(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]),
                 "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
                 "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}
__device__ __forceinline__ bool odd_bf16x2(uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; }

// Bits of the keys kbase + 32 q .. + 31 that a row sees.
__device__ __forceinline__ uint32_t tree_seen(const uint64_t* mask, int words, int key, int ctx, int len, int low) {
  const int rel = key - ctx;
  uint32_t v = 0xffffffffu;
  if (rel > -32) {
    const int from = max(rel, 0), a = from >> 6, sh = from & 63;
    uint64_t w = a < words ? __ldg(mask + a) >> sh : 0;
    if (sh > 32 && a + 1 < words) w |= __ldg(mask + a + 1) << (64 - sh);
    v = rel >= 0 ? (uint32_t)w : (uint32_t)w << -rel | ((1u << -rel) - 1);
  }
  if (len - key < 32) v &= len > key ? (1u << (len - key)) - 1 : 0;
  if (key < low) v &= low - key < 32 ? ~((1u << (low - key)) - 1) : 0;
  return v;
}

template <int D>
__global__ void __launch_bounds__(kTreeThreads, 1)
    tree_attn_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmKV, TreeParams p) {
  using Sh = TreeShape<D>;
  constexpr int kRing = Sh::kRing, kKeys = Sh::kKeys, kOdd = Sh::kOdd, kWords = Sh::kWords;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sKV = sQ + Sh::kQTiles * Sh::kQTile;
  TreeBars<D>& bars = *reinterpret_cast<TreeBars<D>*>(smem + Sh::kTiles);
  const int warp = warp_index(), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(&bars.q_full, 1);
    mbar_init(&bars.q_empty, 1);
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&bars.kv_full[i], 1);
      mbar_init(&bars.kv_empty[i], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bars.s_full[t], 1);
      mbar_init(&bars.p_full[t], Sh::kWide ? 8 : 4);
    }
    mbar_init(&bars.o_full, 1);
    mbar_init(&bars.o_free, 8);
    mbar_init(&bars.pv_done, 1);
    mbar_init(&bars.meet, 8);
    mbar_fence_init();
    bars.odd_any = 0;
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmKV);
  }
  if (threadIdx.x < kOdd * kWords) bars.odd[threadIdx.x / kWords][threadIdx.x % kWords] = 0;
  if (warp == 1) {
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
      const TreeReq r = tree_req<D>(p, b);
      const long long cells = (long long)r.items * (kTreeStart + r.tiles);
      if (lo < at + cells) {
        bars.start_req = b;
        bars.start_off = (int)(lo - at);
        break;
      }
      at += cells;
    }
  }
  __syncthreads();
  TreeWalk<D> walk(p, lo < hi ? bars.start_req : 0, lo < hi ? bars.start_off : 0, hi - lo);
  TreePiece w;

  if (warp == 0) {
    // ---------------- TMA ----------------
    const int page_rows = min(p.block_size, kKeys), loads = kKeys / page_rows;       // pages of a tile (at most 16): a lane each
    uint32_t load = 0, piece = 0;                                                    // of the ring; of the stretch
    bool ok = true;
    for (; ok && walk.next(w); ++piece) {
      const TreeReq& r = walk.r;
      if (piece > 0 && !(ok = mbar_wait_warp(&bars.q_empty, (piece - 1) & 1, p.status))) break;
      const int row = r.row0 + w.node0, tiles = w.two ? 2 : 1;
      if (lane == 0) mbar_expect_tx(&bars.q_full, tiles * Sh::kParts * p.nodes * p.G * 128);
      __syncwarp();
      if (lane < tiles * Sh::kParts) {
        const int t = lane / Sh::kParts, part = lane % Sh::kParts;
        tma_load_3d(sQ + t * Sh::kQTile + part * 16384, &tmQ, &bars.q_full, part * 64, w.head * p.G, row + t * p.nodes);
      }
      __syncwarp();
      const int32_t* bt = p.block_table + walk.b * p.ldt;
      const int last_page = max(0, (r.len - 1) / p.block_size);
      const int nt = w.je - w.jb, first_key = (r.begin + w.jb) * kKeys;
      // entries of the table, 32 at a time, the next ones on their way
      int base = first_key / p.block_size, now = bt[min(base + lane, last_page)], next = bt[min(base + 32 + lane, last_page)];
      long long k_row = 0, v_row = 0;
      const auto fetch = [&](int kv, int j) {
        const int key = first_key + j * kKeys, page = key / p.block_size;
        if (kv == 0) {
          if (page >= base + 32) {
            base += 32;
            now = next;
            next = bt[min(base + 32 + lane, last_page)];
          }
          v_row = k_row;
          // (a tile's pages do not pass a multiple of 32 entries from the piece's first: they may begin anywhere in it)
          const int want = page - base + (p.block_size < kKeys ? lane : 0);
          const int e0 = __shfl_sync(0xffffffffu, now, want & 31), e1 = __shfl_sync(0xffffffffu, next, want & 31);
          const int blk = want < 32 ? e0 : e1;
          k_row = (blk < 0 || blk >= p.num_blocks ? p.num_blocks : (long long)blk) * 2 * p.block_size + key % p.block_size;
        }
        const int sl = load % kRing;
        if (!mbar_wait_warp(&bars.kv_empty[sl], ((load / kRing) & 1) ^ 1, p.status)) return false;
        if (lane == 0) mbar_expect_tx(&bars.kv_full[sl], Sh::kSlot);
        __syncwarp();
        if (lane < loads) {
          uint8_t* dst = sKV + sl * Sh::kSlot + lane * page_rows * 128;
          // (of the tile that K is at; V of the tile before it, where K is one ahead)
          const long long at = kv == 0 ? k_row : (w.two || j == nt - 1 ? k_row : v_row) + p.block_size;
#pragma unroll
          for (int d = 0; d < Sh::kParts; ++d) tma_load_3d(dst + d * Sh::kPiece, &tmKV, &bars.kv_full[sl], d * 64, w.head, (int)at);
        }
        __syncwarp();
        ++load;
        return true;
      };
      if (w.two) {
        for (int j = 0; ok && j < nt; ++j) ok = fetch(0, j) && fetch(1, j);
      } else {
        ok = fetch(0, 0);
        for (int j = 0; ok && j < nt; ++j) {
          if (j + 1 < nt) ok = fetch(0, j + 1);
          ok = ok && fetch(1, j);
        }
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA ----------------
    constexpr uint32_t idesc_qk = umma_idesc_bf16(128, kKeys, 0, 0), idesc_pv = umma_idesc_bf16(128, D, 0, 1);
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0), q_addr = smem_u32(sQ);
    uint32_t load0 = 0, piece = 0, made[2] = {0, 0};               // tiles of P seen, of either half
    bool ok = true;
    const auto full = [&](uint32_t i) { return mbar_wait_warp(&bars.kv_full[i % kRing], (i / kRing) & 1, p.status); };
    const auto qk = [&](int t, int qt, uint32_t i, bool release, bool last) {
      const uint32_t k_addr = smem_u32(sKV + (i % kRing) * Sh::kSlot), q = q_addr + qt * Sh::kQTile;
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_bf16_ss(tm + t * Sh::kSCols, umma_desc_k_sw128(q + (kk / 4) * 16384 + (kk % 4) * 32, 1024),
                       umma_desc_k_sw128(k_addr + (kk / 4) * Sh::kPiece + (kk % 4) * 32, 1024), idesc_qk, kk != 0);
        umma_commit(&bars.s_full[t]);
        if (release) umma_commit(&bars.kv_empty[i % kRing]);
        if (last) umma_commit(&bars.q_empty);
      }
      __syncwarp();
    };
    const auto pv = [&](int t, uint32_t i, bool add, bool release, bool last) {
      const uint64_t vd = umma_desc_mn_sw128(smem_u32(sKV + (i % kRing) * Sh::kSlot), Sh::kPiece, 1024);
      const uint32_t p_at = Sh::kWide ? tm + Sh::kP + t * 32 : tm + t * Sh::kSCols, o_at = Sh::kWide ? tm + Sh::kO : tm + Sh::kO + t * D;
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk) umma_bf16_ts(o_at, p_at + kk * 8, vd + kk * (2048 >> 4), idesc_pv, add || kk != 0);
        if (release) umma_commit(&bars.kv_empty[i % kRing]);
        if (Sh::kWide) umma_commit(&bars.pv_done);
        if (last) umma_commit(&bars.o_full);
      }
      __syncwarp();
    };
    for (; ok && walk.next(w); ++piece) {
      const int nt = w.je - w.jb;
      if (!(ok = mbar_wait_warp(&bars.q_full, piece & 1, p.status))) break;
      if (w.two) {                     // tile j: K at 2 j, V at 2 j + 1, for both tiles of rows
        if (!(ok = full(load0))) break;
        tc_fence_after_sync();
        qk(0, 0, load0, false, false);
        qk(1, 1, load0, true, nt == 1);
        for (int j = 0; ok && j < nt; ++j) {
          const uint32_t v = load0 + 2 * j + 1;
          if (!(ok = full(v))) break;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (!(ok = mbar_wait_warp(&bars.p_full[t], made[t] & 1, p.status))) break;
            ++made[t];
            if (j == 0 && t == 0 && piece > 0 && !(ok = mbar_wait_warp(&bars.o_free, (piece - 1) & 1, p.status))) break;
            tc_fence_after_sync();
            pv(t, v, j > 0, t == 1, t == 1 && j == nt - 1);
            if (j + 1 < nt) {
              if (t == 0) {
                if (!(ok = full(v + 1))) break;
                tc_fence_after_sync();
              }
              qk(t, t, v + 1, t == 1, t == 1 && j + 2 == nt);
            }
          }
        }
      } else {                         // K0 K1 V0 K2 V1 .. V(nt - 1)
        const auto k_at = [&](int j) { return load0 + (j == 0 ? 0 : 2 * j - 1); };
        for (int j = 0; ok && j < min(2, nt); ++j) {
          if (!(ok = full(k_at(j)))) break;
          tc_fence_after_sync();
          qk(j, 0, k_at(j), true, j + 1 == nt);
        }
        for (int j = 0; ok && j < nt; ++j) {
          const int t = j & 1;
          const uint32_t v = load0 + (j == nt - 1 ? 2 * nt - 1 : 2 * j + 2);
          if (!(ok = full(v))) break;
          if (!(ok = mbar_wait_warp(&bars.p_full[t], made[t] & 1, p.status))) break;
          ++made[t];
          if (j == 0 && piece > 0 && !(ok = mbar_wait_warp(&bars.o_free, (piece - 1) & 1, p.status))) break;
          tc_fence_after_sync();
          pv(t, v, Sh::kWide ? j > 0 : j > 1, true, j == nt - 1);
          if (j + 2 < nt) {
            if (!(ok = full(k_at(j + 2)))) break;
            tc_fence_after_sync();
            qk(t, 0, k_at(j + 2), true, j + 3 == nt);
          }
        }
      }
      load0 += 2 * nt;
    }
  } else {
    // ---------------- softmax and output: a thread a row (two where it is wide) ----------------
    const int half = (warp - 2) >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const float cap_in = p.cap2 > 0.f ? fminf(2.8853900817779268f / p.cap2, 3.0e38f) : 0.f;
    const int row_node = r / p.G, row_head = r - row_node * p.G;
    uint32_t load0 = 0, piece = 0, seen_s[2] = {0, 0}, met = 0, pvs = 0;
    bool ok = true;
    const auto meet = [&]() {           // both halves
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.meet);
      return __all_sync(0xffffffffu, mbar_wait(&bars.meet, met++ & 1, p.status));
    };
    for (; ok && walk.next(w); ++piece) {
      const TreeReq rq = walk.r;
      const int nt = w.je - w.jb;
      const int node = w.node0 + (w.two ? half * p.nodes : 0) + row_node;
      const bool there = row_node < p.nodes && node < rq.n;
      const uint64_t* bits = p.mask + (size_t)(rq.row0 + (there ? node : 0)) * p.words;
      int low = 0;
      if (p.window > 0 && there) {     // (a node lies at most n - 1 positions behind the root)
        const long long depth = p.positions[rq.row0 + node] - rq.ctx;
        low = min(rq.ctx, rq.ctx + (int)min(max(depth, 0ll), (long long)rq.n - 1) - p.window + 1);
      }
      const auto seen_word = [&](int key) { return there ? tree_seen(bits, p.words, key, rq.ctx, rq.len, low) : 0u; };
      // (the first positions that the nodes of the piece see differ by as much as their positions do)
      const int low_most = p.window > 0 ? __reduce_max_sync(0xffffffffu, there ? low : INT_MIN) : 0;
      float m = -INFINITY, l = 0.f;
      int odd_n = 0;
      // tiles of this half
      const int step = Sh::kWide || w.two ? 1 : 2;
      for (int j = step == 2 ? half : 0; j < nt; j += step) {
        const int t = Sh::kWide ? j & 1 : half, kbase = (rq.begin + w.jb + j) * kKeys;
        // tiles in which the nodes of the request may differ in what they see (need_mask: those of this warp do)
        const bool odd_tile = kbase + kKeys > rq.ctx || (p.window > 0 && kbase < rq.ctx - p.window + rq.n);
        const bool need_mask = kbase + kKeys > rq.ctx || kbase < low_most;
        if (odd_tile && (step == 2 || half == 0)) {
          // values that are not finite: out of the tile, and noted
          const uint32_t v = load0 + (w.two ? 2 * j + 1 : j == nt - 1 ? 2 * nt - 1 : 2 * j + 2);
          ok = __all_sync(0xffffffffu, mbar_wait(&bars.kv_full[v % kRing], (v / kRing) & 1, p.status));
          if (!ok) break;
          const int key = Sh::kWide ? r & 63 : r, d0 = Sh::kWide ? (r >> 6) * 2 : 0;
          uint8_t* row = sKV + (v % kRing) * Sh::kSlot + key * 128;
          bool odd = false;
#pragma unroll
          for (int d = 0; d < (Sh::kWide ? 2 : Sh::kParts); ++d) {
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              uint4* at = reinterpret_cast<uint4*>(row + (d0 + d) * Sh::kPiece + ((c ^ (key & 7)) << 4));
              const uint4 x = *at;
              if (odd_bf16x2(x.x) || odd_bf16x2(x.y) || odd_bf16x2(x.z) || odd_bf16x2(x.w)) {
                uint32_t e[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  if ((e[i] & 0x7f80u) == 0x7f80u) e[i] &= 0xffff0000u;
                  if ((e[i] & 0x7f800000u) == 0x7f800000u) e[i] &= 0xffffu;
                }
                *at = make_uint4(e[0], e[1], e[2], e[3]);
                odd = true;
              }
            }
          }
          fence_proxy_async_smem();
          const uint32_t who = __ballot_sync(0xffffffffu, odd);
          if (who) {
            // (rare: a note in the list that belongs to the half; room for every tile that can be looked at)
            if (lane == 0) {
              const int at = (step == 2 ? half * (kOdd / 2) : 0) + odd_n;
              bars.odd_tile[at] = kbase;
              atomicOr(&bars.odd[at][Sh::kWide ? quarter & 1 : quarter], who);
              atomicOr(&bars.odd_any, 1u);
            }
          }
          ++odd_n;
        }
        ok = __all_sync(0xffffffffu, mbar_wait(&bars.s_full[t], seen_s[t] & 1, p.status));
        if (!ok) break;
        ++seen_s[t];
        tc_fence_after_sync();
        const uint32_t s_addr = tmem + t * Sh::kSCols + lanes;
        // Caps and masks go through tensor memory, 32 scores at a time: the registers of the plain path hold a tile's scores and no more.
        // (Where it is wide the two threads of a row take a half each and wait for one another.)
        if (p.cap2 > 0.f || (Sh::kWide ? odd_tile : need_mask)) {
#pragma unroll 1
          for (int c = Sh::kWide ? half : 0; c < (Sh::kWide ? half + 1 : kWords); ++c) {
            uint32_t x[32];
            tmem_ld_32x32b_x32(s_addr + c * 32, x);
            const uint32_t seen = need_mask ? seen_word(kbase + 32 * c) : 0xffffffffu;
            tmem_ld_wait();
            if (p.cap2 > 0.f) {
#pragma unroll
              for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(tree_capped(__uint_as_float(x[i]) * p.scale_log2, p.cap2, cap_in));
            }
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!(seen >> i & 1)) x[i] = 0xff800000u;                    // -inf
            tmem_st_32x32b_x32(s_addr + c * 32, x);
          }
          tmem_st_wait();
          if (Sh::kWide) {
            tc_fence_before_sync();
            if (!(ok = meet())) break;
            tc_fence_after_sync();
          }
        }
        const float sc = p.cap2 > 0.f ? 1.f : p.scale_log2;
        // Two passes over the tile, 32 scores at a time with the next on their way.
        uint32_t s[2][32];
        tmem_ld_32x32b_x32(s_addr, s[0]);
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < kWords; ++c) {
          tmem_ld_wait_for(s[c & 1]);
          tmem_ld_32x32b_x32(s_addr + (c + 1 < kWords ? c + 1 : Sh::kWide ? half : 0) * 32, s[(c + 1) & 1]);
#pragma unroll
          for (int i = 0; i < 32; i += 4)
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], __uint_as_float(s[c & 1][i + e]));
        }
        tmem_ld_wait_for(s[0]);        // (kWords is even: the second pass begins where the first did)
        // m: reference of the row's maximum, raised lazily (by more than 2^8), so that the accumulator is rescaled rarely; P stays below 256
        const float tile_max = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sc;
        float alpha = 1.f;
        bool rescale = false;
        if (tile_max > m + 8.f) {      // also the first finite tile: m == -inf
          if (m != -INFINITY) {
            alpha = tree_ex2(m - tile_max);
            rescale = true;
          }
          m = tile_max;
        }
        const float m_use = m == -INFINITY ? 0.f : m;
        const int first_of_half = step == 2 ? half : 0;
        if (Sh::kWide) {               // S(j) is issued ahead of P V(j - 1)
          if (__any_sync(0xffffffffu, rescale) && j > first_of_half) {
            ok = __all_sync(0xffffffffu, mbar_wait(&bars.pv_done, (pvs - 1) & 1, p.status));
            if (!ok) break;
            tc_fence_after_sync();
          }
          ++pvs;
        }
        // (not wide: the accumulator is at rest, as S(j) is issued right behind P V of the half's tile before it, by the same lane)
        if (__any_sync(0xffffffffu, rescale) && j > first_of_half) {
          constexpr int cols = Sh::kWide ? D / 2 : D;
          const uint32_t o_addr = tmem + Sh::kO + half * cols + lanes;
#pragma unroll 1
          for (int c = 0; c < cols / 16; ++c) {
            uint32_t rr[16];
            tmem_ld_32x32b_x16(o_addr + c * 16, rr);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) rr[i] = __float_as_uint(__uint_as_float(rr[i]) * alpha);
            tmem_st_32x32b_x16(o_addr + c * 16, rr);
          }
        }
        // The sum is that of the rounded values: a row's weights add up to one, and a single key's value comes out as it is.
        const uint64_t sc2 = pack_f32x2(sc, sc), off2 = pack_f32x2(-m_use, -m_use);
        uint64_t sum2[2] = {0, 0};
        constexpr int n32 = Sh::kWide ? 1 : kKeys / 32;
#pragma unroll
        for (int c = 0; c < n32; ++c) {
          if (c > 0) tmem_ld_wait_for(s[c & 1]);
          if (c + 1 < n32) tmem_ld_32x32b_x32(s_addr + (c + 1) * 32, s[(c + 1) & 1]);
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float a, b;
            unpack_f32x2(fma_f32x2(pack_b32x2(s[c & 1][2 * i], s[c & 1][2 * i + 1]), sc2, off2), a, b);
            pk[i] = pack_bf16x2(tree_ex2(a), tree_ex2(b));
            sum2[i & 1] = add_f32x2(sum2[i & 1], pack_b32x2(pk[i] << 16, pk[i] & 0xffff0000u));
          }
          // (over scores that both passes have read)
          tmem_st_32x32b_x16((Sh::kWide ? tmem + Sh::kP + t * 32 + half * 16 + lanes : s_addr + c * 16), pk);
        }
        float sum[4];
        unpack_f32x2(sum2[0], sum[0], sum[1]);
        unpack_f32x2(sum2[1], sum[2], sum[3]);
        l = l * alpha + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
        tmem_st_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.p_full[t]);
      }
      load0 += 2 * nt;
      if (!ok) break;
      // ---- output
      const bool whole = w.jb == 0 && w.je == rq.tiles, other = step == 2 && nt > 1;       // other: both halves have a share of every row
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
          if (whole) {
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
      } else if (whole) {
        a0 = l != 0.f ? 1.f / l : 0.f;
      }
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(&bars.o_full, piece & 1, p.status)))) break;
      tc_fence_after_sync();
      // columns of this thread's: all of its row's, or one half of them
      constexpr int kHalfCols = D / 2;
      const int col0 = w.two ? 0 : half * kHalfCols, cols = w.two ? D : kHalfCols;
      const int part_row = w.two ? half * 128 + r : r;
      const uint32_t o_addr = tmem + Sh::kO + lanes + (w.two ? half * D : 0);
      __nv_bfloat16* dst = p.out + (rq.row0 + node) * p.ldo + (w.head * p.G + row_head) * D;
      float* part = p.parts + (2 * blockIdx.x + (w.jb > 0 ? 0 : 1)) * Sh::kPartFloats;
      const bool odd_any = *(volatile uint32_t*)&bars.odd_any != 0;
#pragma unroll 1
      for (int c = 0; c < cols; c += 32) {
        uint32_t rr[32], r1[32];
        tmem_ld_32x32b_x32(o_addr + col0 + c, rr);
        if (other) tmem_ld_32x32b_x32(o_addr + D + col0 + c, r1);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float o = __uint_as_float(rr[i]) * a0;
          rr[i] = __float_as_uint(other ? fmaf(__uint_as_float(r1[i]), a1, o) : o);
        }
        if (odd_any && there) {
          for (int e = 0; e < kOdd; ++e) {
            for (int q = 0; q < kWords; ++q) {
              uint32_t who = bars.odd[e][q];
              if (who == 0) continue;
              who &= seen_word(bars.odd_tile[e] + 32 * q);
              while (who) {
                const int key = bars.odd_tile[e] + 32 * q + __ffs(who) - 1;
                who &= who - 1;
                const int blk = p.block_table[walk.b * p.ldt + key / p.block_size];
                if (blk < 0 || blk >= p.num_blocks) continue;
                const __nv_bfloat16* v = p.cache + ((((long long)blk * 2 + 1) * p.block_size + key % p.block_size) * p.Hkv + w.head) * D + col0 + c;
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                  const float x = __bfloat162float(v[i]);
                  if (!(fabsf(x) <= 3.4028234e38f)) rr[i] = __float_as_uint(__uint_as_float(rr[i]) + x);
                }
              }
            }
          }
        }
        if (there) {
          if (whole) {
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              uint4 o;
              o.x = pack_bf16x2(__uint_as_float(rr[i + 0]), __uint_as_float(rr[i + 1]));
              o.y = pack_bf16x2(__uint_as_float(rr[i + 2]), __uint_as_float(rr[i + 3]));
              o.z = pack_bf16x2(__uint_as_float(rr[i + 4]), __uint_as_float(rr[i + 5]));
              o.w = pack_bf16x2(__uint_as_float(rr[i + 6]), __uint_as_float(rr[i + 7]));
              *reinterpret_cast<uint4*>(dst + col0 + c + i) = o;
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<uint4*>(part + (size_t)part_row * D + col0 + c + i) = make_uint4(rr[i], rr[i + 1], rr[i + 2], rr[i + 3]);
          }
        }
      }
      if (!whole && there && (w.two || half == 0)) {
        part[(size_t)Sh::kRows * D + part_row] = m;
        part[(size_t)Sh::kRows * D + Sh::kRows + part_row] = l;
      }
      tc_fence_before_sync();
      if (odd_any) {                   // everyone has read the notes: they go
        if (!(ok = meet())) break;
        const int i = threadIdx.x - 64;
        if (i < kOdd * kWords) bars.odd[i / kWords][i % kWords] = 0;
        if (i == 0) bars.odd_any = 0;
      }
      // (also keeps what the threads of a row told one another, and the notes, from being written before everyone has read them)
      if (!(ok = meet())) break;
      if (lane == 0) mbar_arrive(&bars.o_free);
      if (threadIdx.x == 64) {
        TreeCut* cut = reinterpret_cast<TreeCut*>(p.parts + 2 * (long long)gridDim.x * Sh::kPartFloats) + blockIdx.x;
        if (w.jb > 0 && w.je == rq.tiles) {
          // the line's cell of the item's first tile says which CTA has its first part
          const long long first = lo - w.jb;
          cut->row0 = rq.row0 + w.node0;
          cut->head = w.head;
          cut->rows = min(rq.n - w.node0, p.nodes * (w.two ? 2 : 1)) * p.G;
          cut->first = (int)(first / stretch);
        } else if (piece == 0) {
          cut->first = -1;
        }
      }
    }
    if (piece == 0 && threadIdx.x == 64) {
      TreeCut* cut = reinterpret_cast<TreeCut*>(p.parts + 2 * (long long)gridDim.x * Sh::kPartFloats) + blockIdx.x;
      cut->first = -1;
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// Parts of items that the ends of stretches cut. Block (b, y): the item whose last part is CTA b's, rows y, y + 8 .. in eights.
template <int D>
__global__ void __launch_bounds__(256)
    tree_join_kernel(const float* __restrict__ parts, int ctas, __nv_bfloat16* __restrict__ out, long long ldo, int G, int nodes) {
  using Sh = TreeShape<D>;
  constexpr int kVec = D / 32;
  pdl_wait();
  const TreeCut cut = reinterpret_cast<const TreeCut*>(parts + 2 * (long long)ctas * Sh::kPartFloats)[blockIdx.x];
  if (cut.first < 0) return;
  const int lane = threadIdx.x & 31, count = (int)blockIdx.x - cut.first + 1;
  for (int i = blockIdx.y * 8 + (threadIdx.x >> 5); i < cut.rows; i += gridDim.y * 8) {
    const int node = i / G, head = i - node * G, tile = node / nodes;
    const int row = tile * 128 + (node - tile * nodes) * G + head;
    const auto part = [&](int c) { return parts + (2ll * (cut.first + c) + (c == 0)) * Sh::kPartFloats; };
    float top = -INFINITY;
    for (int c = lane; c < count; c += 32) top = fmaxf(top, part(c)[(size_t)Sh::kRows * D + row]);
    top = warp_max_f32(top);
    float acc[kVec] = {}, total = 0.f;
    for (int c0 = 0; c0 < count; c0 += 32) {
      float weight = 0.f;
      if (c0 + lane < count) {
        const float* at = part(c0 + lane) + (size_t)Sh::kRows * D + row;
        const float m = at[0];
        weight = m == -INFINITY ? 1.f : tree_ex2(m - top);       // (nothing seen: sums of 0, or of NaN that stay)
        total += at[Sh::kRows] * weight;
      }
      const int n = min(32, count - c0);
#pragma unroll 4
      for (int c = 0; c < n; ++c) {
        const float a = __shfl_sync(0xffffffffu, weight, c);
        const float* o = part(c0 + c) + (size_t)row * D + lane * kVec;
        if constexpr (kVec == 2) {
          const float2 v = *reinterpret_cast<const float2*>(o);
          acc[0] = fmaf(v.x, a, acc[0]);
          acc[1] = fmaf(v.y, a, acc[1]);
        } else {
#pragma unroll
          for (int k = 0; k < kVec; k += 4) {
            const float4 v = *reinterpret_cast<const float4*>(o + k);
            acc[k] = fmaf(v.x, a, acc[k]);
            acc[k + 1] = fmaf(v.y, a, acc[k + 1]);
            acc[k + 2] = fmaf(v.z, a, acc[k + 2]);
            acc[k + 3] = fmaf(v.w, a, acc[k + 3]);
          }
        }
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    const float inv = total != 0.f ? 1.f / total : 0.f;
    uint32_t* dst = reinterpret_cast<uint32_t*>(out + (cut.row0 + node) * ldo + (cut.head * G + head) * D) + lane * (kVec / 2);
#pragma unroll
    for (int k = 0; k < kVec / 2; ++k) dst[k] = pack_bf16x2(acc[2 * k] * inv, acc[2 * k + 1] * inv);
  }
}

template <int D>
static int launch_tree(const CUtensorMap& tmQ, const CUtensorMap& tmKV, const TreeParams& p, int ctas, cudaStream_t stream) {
  static PerDeviceOnce once;
  if (once.first()) cudaFuncSetAttribute(tree_attn_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, tree_smem<D>());
  if (launch_pdl(tree_attn_kernel<D>, dim3(ctas), dim3(kTreeThreads), tree_smem<D>(), stream, tmQ, tmKV, p) != cudaSuccess) return -2;
  return launch_pdl(tree_join_kernel<D>, dim3(ctas, TreeShape<D>::kRows / 32), dim3(256), 0, stream, (const float*)p.parts, ctas, p.out, p.ldo,
                    p.G, p.nodes) == cudaSuccess ? 0 : -2;
}

struct TreeMapKey {
  const void* p;
  uint64_t rows;
  int hkv, d, box;
  bool operator==(const TreeMapKey& o) const { return p == o.p && rows == o.rows && hkv == o.hkv && d == o.d && box == o.box; }
};
struct TreeMapHash {
  size_t operator()(const TreeMapKey& k) const {
    return reinterpret_cast<size_t>(k.p) ^ k.rows * 0x9e3779b97f4a7c15ull ^ (size_t)k.hkv << 40 ^ (size_t)k.d << 20 ^ (size_t)k.box;
  }
};

}  // namespace b200

using namespace b200;

// What a call takes, as far as sizes say: 0, or -1 (shape) or -4 (counted in 31 bits: key tiles of all items of a request).
extern "C" int b200_tree_attn_takes(const B200TreeAttn* a) {
  const int D = a->D, keys = D == 256 ? 64 : 128;
  if (D != 64 && D != 128 && D != 256) return -1;
  if (a->Hkv <= 0 || a->Hq <= 0 || a->Hq % a->Hkv || a->Hq / a->Hkv > 128 || a->words <= 0 || a->max_blocks <= 0) return -1;
  const int bs = a->block_size;
  if (bs < 8 || bs % 8 || (bs < keys ? keys % bs : bs % keys)) return -1;
  if (a->num_reqs > kTreeReqs || a->words > kTreeNodes / 64) return -4;
  if (a->num_blocks >= (1ll << 31) / (2 * bs) - 1) return -4;
  const int nodes = 128 / (a->Hq / a->Hkv);
  const long long tiles = ((long long)a->max_blocks * bs + keys - 1) / keys + kTreeStart;
  const long long pairs = (std::min(a->total_q, 64 * a->words) + nodes - 1) / nodes + 1;
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
  const int D = a->D, keys = D == 256 ? 64 : 128, G = a->Hq / a->Hkv, bs = a->block_size;
  TreeParams p;
  p.cache = (const __nv_bfloat16*)a->cache; p.out = (__nv_bfloat16*)a->out; p.ldo = a->ldo;
  p.block_table = (const int32_t*)a->block_table; p.ldt = a->ldt; p.num_blocks = a->num_blocks; p.max_blocks = a->max_blocks;
  p.seq_lens = (const int32_t*)a->seq_lens; p.q_start = (const int32_t*)a->q_start;
  p.positions = (const int64_t*)a->positions; p.mask = (const uint64_t*)a->mask; p.words = a->words;
  p.num_reqs = a->num_reqs; p.total_q = a->total_q; p.Hkv = a->Hkv; p.G = G; p.nodes = 128 / G;
  p.block_size = bs; p.window = a->positions ? a->window : 0; p.max_len = a->max_blocks * bs;
  p.scale_log2 = a->scale * 1.4426950408889634f; p.cap2 = a->softcap * 1.4426950408889634f;
  p.parts = (float*)a->parts; p.status = device_status_word();
  CUtensorMap tmQ, tmKV;
  if (!encode_tmap_3d(&tmQ, a->q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, (uint64_t)D, (uint64_t)a->Hq, (uint64_t)a->total_q, (uint64_t)D * 2,
                      (uint64_t)a->ldq * 2, 64, (uint32_t)G, (uint32_t)p.nodes, CU_TENSOR_MAP_SWIZZLE_128B))
    return -3;
  static std::mutex mu;
  static std::unordered_map<TreeMapKey, CUtensorMap, TreeMapHash> maps;
  const uint64_t rows = (uint64_t)a->num_blocks * 2 * bs;
  const TreeMapKey key{a->cache, rows, a->Hkv, D, std::min(bs, keys)};
  try {
    std::lock_guard<std::mutex> lock(mu);
    auto it = maps.find(key);
    if (it == maps.end()) {
      if (maps.size() > 4096) maps.clear();          // scratch caches come and go
      CUtensorMap m;
      if (!encode_tmap_3d(&m, a->cache, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, (uint64_t)D, (uint64_t)a->Hkv, rows, (uint64_t)D * 2,
                          (uint64_t)a->Hkv * D * 2, 64, 1, (uint32_t)key.box, CU_TENSOR_MAP_SWIZZLE_128B))
        return -3;
      it = maps.emplace(key, m).first;
    }
    tmKV = it->second;
  } catch (...) {
    return -2;
  }
  const int ctas = b200_num_sms();
  return D == 64 ? launch_tree<64>(tmQ, tmKV, p, ctas, stream) : D == 128 ? launch_tree<128>(tmQ, tmKV, p, ctas, stream)
                                                                         : launch_tree<256>(tmQ, tmKV, p, ctas, stream);
}
