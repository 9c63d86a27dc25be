// How attention over the 4-bit cache is shared out, for both of its kernels. An entry (a sequence, or a tile of 128 query tokens) has items (kv head,
// row tile) that all read the same number of cells (here: 32 or 128 neighbouring keys). The cells of all items of all entries stand in one line, each CTA takes an equal stretch of
// it, and the parts of items that the ends of stretches cut are joined afterwards. What an item costs besides its cells (queries, output) stands in
// the line as kStart cells in front of them: without, the CTAs that get the short items (of a causal prompt's beginning, of short sequences) finish
// last.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <mutex>

#include "fp4_cache.cuh"
#include "sm100.cuh"

namespace b200 {

// Division by a number that the host knows: n / d for n d < 2^32 (mul = 2^32 / d rounded up, 0 for d = 1).
struct Fp4Div {
  uint32_t mul;
#ifdef __CUDACC__
  __device__ __forceinline__ int of(int n) const { return mul ? (int)__umulhi((uint32_t)n, mul) : n; }
#endif
};

struct Fp4Attn {
  const __nv_bfloat16* q;
  long long ldq;
  __nv_bfloat16* out;
  long long ldo;
  const uint8_t* cache;
  long long num_blocks;
  const int32_t* block_table;
  long long ldt;               // entries from one sequence's row of the table to the next
  int max_blocks;              // of a sequence
  const int32_t* seq_lens;
  const int32_t* q_start;      // null: one row a sequence
  const int32_t *tile_req, *tile_q0;
  int num_reqs, total_q, num_tiles;
  int Hkv, G, cells_per_page, window, causal;
  int few;                     // sequences of at most so many rows (query tokens x G) are the row kernel's, the others the tile kernel's
  Fp4Div by_group, by_page_cells;
  float scale_log2, softcap2;
  int* status;
};
// h = item / tiles; one division, and none for a single tile
__device__ __forceinline__ int fp4_head(int item, int tiles) { return tiles == 1 ? item : item / tiles; }

__device__ __forceinline__ float ex2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// cvt_e2m1x8 that the compiler may move.
__device__ __forceinline__ void e2m1x8_f16(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}\n"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}
// Scale bytes lo and hi (selectors of __byte_perm) of w -> f16x2.
__device__ __forceinline__ uint32_t scales_f16x2(uint32_t w, int lo, int hi) { return __byte_perm(w, 0, 0x4040 | lo | hi << 8) << 7; }
// Of four scale bytes the ones that are NaN (or infinite): 0x80 each.
__device__ __forceinline__ uint32_t nan_scales(uint32_t w) { return ((w & 0x78787878u) + 0x08080808u) & w & 0x80808080u; }
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Probabilities are 2^(score - m + kUp), m a reference of the running maximum that is raised when a score passes it by 8: at most 2^15 in f16, and
// the smallest ones keep their bits.
static constexpr float kUp = 7.f;

// cap tanh(x / cap) in log2 units: tanh(y) = 1 - 2 / (1 + e^(2 y)). Off by some 2^-22 of the cap, whatever y is; infinities and NaN go through.
__device__ __forceinline__ float fp4_capped(float x, float to_y2, float cap2) {        // to_y2: x -> 2 y log2(e)
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + ex2_of(x * to_y2)));
  return fmaf(-2.f * cap2, r, cap2);
}
// That is too much of a cap far above the scores. Under one past kWideCap |y| < 1 / 16 takes y - y^3 / 3 + 2 y^5 / 15, off by 2^-28 of itself.
static constexpr float kWideCap = 1500.f;
__device__ __forceinline__ float fp4_wide_capped(float x, float to_y2, float cap2) {
  const float y2log2e = x * to_y2, y = y2log2e * 0.34657359f, yy = y * y;
  return fabsf(y) < 0.0625f ? cap2 * y * fmaf(yy, fmaf(yy, 0.13333333f, -0.33333333f), 1.f) : fp4_capped(x, to_y2, cap2);
}
// to_y2 for scores of `to_log2`: finite, as a score of 0 times it is 0 however small the cap is.
__device__ __forceinline__ float fp4_cap_in(float to_log2, float cap2) { return fminf(to_log2 * fminf(2.8853900817779268f / cap2, 3.0e38f), 3.0e38f); }

// lowest position that the query at `pos` sees
__device__ __forceinline__ int fp4_lowest(int window, int pos) {
  return window > 0 ? pos - window + 1 : window < 0 && pos >= 0 ? pos / -window * -window : 0;
}
__device__ __forceinline__ int fp4_lowest(const Fp4Attn& p, int pos) { return fp4_lowest(p.window, pos); }
// Rows of query tokens [q_begin, + q_len) of a sequence with len keys.
struct Fp4Span {
  int len, q_begin, q_len;
  __device__ __forceinline__ Fp4Span(const Fp4Attn& p, int b) {
    q_begin = p.q_start ? min(max(p.q_start[b], 0), p.total_q) : b;
    q_len = p.q_start ? max(min(p.q_start[b + 1], p.total_q) - q_begin, 0) : 1;
    len = min(max(p.seq_lens[b], 0), p.max_blocks * p.cells_per_page * kCellTokens);
  }
};

// An entry's token0 is the query row of its first row, first that one's position, rows = tokens x G.
static constexpr int kPairKeys = 2 * kCellTokens;
// (kStart by measurement: 256 decoding sequences of 200 to 3800 keys took 153 us with 8, 145 with 20, and 4 % more than that with 32; 48 sequences of 8 to
// 24 rows 109 us with 8, 87 with 24 and 28, 3 to 4 % more with 36 and 44.)
template <int ROWS>
struct Fp4Seq {                // pairs of cells, 32 keys; row tiles of ROWS
  static constexpr int kRows = ROWS, kStart = ROWS > 8 ? 28 : 20, kSnap = 8;
  int req, len, token0, rows, first, begin, cells, tiles;       // begin: first pair of the sequence that any row sees
  static __device__ __forceinline__ int count(const Fp4Attn& p) { return p.num_reqs; }
  __device__ __forceinline__ Fp4Seq() {}
  __device__ __forceinline__ Fp4Seq(const Fp4Attn& p, int b) {
    const Fp4Span s(p, b);
    req = b;
    len = s.len;
    token0 = s.q_begin;
    rows = s.q_len * p.G;
    if (rows > p.few) rows = 0;
    first = len - s.q_len;
    begin = max(0, fp4_lowest(p, first)) / kPairKeys;
    cells = kStart + max(1, (len + kPairKeys - 1) / kPairKeys - begin);          // (no keys: one that counts as masked)
    tiles = (rows + ROWS - 1) / ROWS;
  }
};

static constexpr int kTileKeys = 128, kTileTokens = 128;
struct Fp4Tile {               // tiles of 128 keys, row tiles of 256
  static constexpr int kRows = 256, kStart = 3, kSnap = 8;
  int req, len, token0, rows, first, begin, cells, tiles;       // begin: first key tile that any row sees
  static __device__ __forceinline__ int count(const Fp4Attn& p) { return p.num_tiles; }
  __device__ __forceinline__ Fp4Tile() {}
  __device__ __forceinline__ Fp4Tile(const Fp4Attn& p, int i) {
    req = min(max(p.tile_req[i], 0), p.num_reqs - 1);
    const Fp4Span s(p, req);
    const int q0 = max(p.tile_q0[i], 0), tokens = max(0, min(kTileTokens, s.q_len - q0));
    len = s.len;
    token0 = s.q_begin + q0;
    rows = s.q_len * p.G > p.few ? tokens * p.G : 0;
    first = len - s.q_len + q0;
    begin = max(0, fp4_lowest(p, first)) / kTileKeys;
    const int last = min(p.causal ? first + tokens - 1 : len - 1, len - 1);
    cells = kStart + max(1, (last < 0 ? 0 : last / kTileKeys + 1) - begin);
    tiles = (rows + kRows - 1) / kRows;
  }
};

// line[i] = cells in the line in front of entry i (count + 1 values); gives the line's length. All threads of the block take part. Bounds of sequences that
// go back (q_start does not ascend) could make it longer than 31 bits count: then it is empty, and the call does nothing. Those that ascend cannot; the host
// has seen to that.
template <class Entry>
__device__ uint32_t fp4_line(const Fp4Attn& p, uint32_t* line) {
  __shared__ uint32_t warp_sum[32];
  const int n = Entry::count(p), per = (n + blockDim.x - 1) / blockDim.x, b0 = min((int)threadIdx.x * per, n), b1 = min(b0 + per, n);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  uint32_t sum = 0;
  bool past = false;                                           // a sum has passed 32 bits
  for (int b = b0; b < b1; ++b) {
    const Entry e(p, b);
    const uint32_t c = (uint32_t)e.cells * (uint32_t)(e.tiles * p.Hkv);
    line[b + 1] = c;
    sum += c;
    past |= sum < c;
  }
  uint32_t x = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) {
      x += y;
      past |= x < y;
    }
  }
  if (lane == 31) warp_sum[warp] = x;
  __syncthreads();
  uint32_t before = x - sum;
  for (int w = 0; w < warps; ++w) {
    const uint32_t y = w < warp ? warp_sum[w] : 0;
    before += y;
    past |= before < y;
  }
  for (int b = b0; b < b1; ++b) {
    const uint32_t y = line[b + 1];
    before += y;
    past |= before < y || before >> 31;
    line[b + 1] = before;
  }
  if (threadIdx.x == 0) line[0] = 0;
  return __syncthreads_or(past) ? 0 : line[n];
}
__device__ __forceinline__ int fp4_find(const uint32_t* line, int n, uint32_t u) {   // the entry that cell u is of
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (line[mid + 1] > u) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}
// Stretches: CTA i of `ctas` begins at cell total i / ctas; where that falls into an item of at most kSnap cells, at the nearer end of the item, and
// where it falls among the first kStart or on the first cell behind them, at the item's beginning. (Short items are not worth a part in scratch.)
__device__ __forceinline__ uint32_t fp4_ctas(uint32_t total, uint32_t grid, int least) { return max(1u, min(grid, total / least)); }
template <class Entry>
__device__ __forceinline__ uint32_t fp4_begin(const Fp4Attn& p, const uint32_t* line, uint32_t total, uint32_t i, uint32_t ctas) {
  const uint32_t each = total / ctas, u = each * i + (total - each * ctas) * i / ctas;      // total i / ctas, in 32 bits
  if (u == 0 || u >= total) return u;
  const int b = fp4_find(line, Entry::count(p), u);
  const uint32_t n = Entry(p, b).cells, off = (u - line[b]) % n;
  return n <= Entry::kSnap + Entry::kStart ? u - off + (2 * off >= n ? n : 0) : off <= Entry::kStart ? u - off : u;
}

// The CTA's stretch: its two ends by two lanes at once. By whole warps.
template <class Entry>
__device__ __forceinline__ uint2 fp4_stretch(const Fp4Attn& p, const uint32_t* line, uint32_t total, uint32_t ctas) {
  const uint32_t at = blockIdx.x < ctas ? fp4_begin<Entry>(p, line, total, blockIdx.x + (threadIdx.x & 1), ctas) : 0;
  return make_uint2(__shfl_sync(0xffffffffu, at, 0), __shfl_sync(0xffffffffu, at, 1));
}

// A piece of an item: cells [c0, c1) of the e.cells that it has, kStart among them.
template <class Entry>
struct Fp4Piece {
  uint32_t u, u_end;           // in the line: where the piece begins, where the CTA's stretch ends
  int b, item, c0, c1;
  Entry e;
  __device__ __forceinline__ void at(const Fp4Attn& p, const uint32_t* line, uint32_t from, uint32_t to) {
    u = from;
    u_end = to;
    if (u >= u_end) return;
    b = fp4_find(line, Entry::count(p), u);
    e = Entry(p, b);
    const uint32_t local = u - line[b];
    item = (int)(local / (uint32_t)e.cells);
    c0 = (int)(local - (uint32_t)item * e.cells);
    c1 = (int)min((uint32_t)e.cells, c0 + (u_end - u));
  }
  __device__ __forceinline__ void next(const Fp4Attn& p, const uint32_t* line) {
    u += c1 - c0;
    if (u >= u_end) return;
    ++item;
    if (u == line[b + 1]) {
      item = 0;
      do ++b;
      while (line[b + 1] == u);
      e = Entry(p, b);
    }
    c0 = 0;
    c1 = (int)min((uint32_t)e.cells, u_end - u);
  }
  __device__ __forceinline__ bool more() const { return u < u_end; }
  __device__ __forceinline__ int from() const { return max(0, c0 - Entry::kStart); }             // without those
  __device__ __forceinline__ int to() const { return max(0, c1 - Entry::kStart); }
  __device__ __forceinline__ bool whole() const { return c0 == 0 && c1 == e.cells; }
  // Of the two parts that a CTA has in scratch: 1 for an item that it begins, 0 for one that it goes on with.
  __device__ __forceinline__ int part() const { return c0 == 0; }
};

// Scratch of a part: O in pieces of 4 dims (fp4_part_at), then (m, l) of each row; in CTA order, two a CTA. Behind the parts a CTA says what of its last item is to be joined.
template <class Entry, int D>
__host__ __device__ constexpr size_t fp4_part(uint32_t cta, int part) { return ((size_t)cta * 2 + part) * (Entry::kRows * (D + 2)); }
// (The row kernel writes a row's dims side by side, the tile kernel a lane a row.)
template <class Entry, int D>
__host__ __device__ constexpr int fp4_part_at(int row, int d) { return Entry::kRows > 16 ? (d / 4 * Entry::kRows + row) * 4 + d % 4 : row * D + d; }
template <class Entry, int D>
__host__ __device__ constexpr size_t fp4_scratch(uint32_t grid) { return fp4_part<Entry, D>(grid, 0) + (size_t)grid * 8; }
struct alignas(16) Fp4Cut {    // of an item that this CTA begins and CTAs up to `last` go on with; rows 0: none
  int rows, last, token0, head0, row0, pad[3];
};
template <class Entry, int D>
__device__ __forceinline__ Fp4Cut* fp4_cut(float* parts, uint32_t grid, uint32_t cta) {
  return reinterpret_cast<Fp4Cut*>(parts + fp4_part<Entry, D>(grid, 0)) + cta;
}
// The last piece of a CTA's stretch, by one thread; a CTA without work: more() is false.
template <class Entry, int D>
__device__ __forceinline__ void fp4_say_cut(const Fp4Attn& p, const uint32_t* line, uint32_t total, uint32_t ctas, uint32_t from, uint32_t to,
                                            float* parts) {
  Fp4Cut c = {};
  if (from < to) {
    Fp4Piece<Entry> w;
    w.at(p, line, to - 1, to);                                  // the stretch's last cell
    const uint32_t begin = line[w.b] + (uint32_t)w.item * w.e.cells;
    if (w.c1 < w.e.cells && begin >= from) {                    // its item goes on, and begins here
      const int h = fp4_head(w.item, w.e.tiles);
      c.row0 = (w.item - h * w.e.tiles) * Entry::kRows;
      c.rows = min(Entry::kRows, w.e.rows - c.row0);
      c.last = (int)min(((uint64_t)(begin + w.e.cells) * ctas - 1) / total, (uint64_t)ctas - 1);       // the CTA that has the item's last cell
      c.token0 = w.e.token0;
      c.head0 = h * p.G;
    }
  }
  *fp4_cut<Entry, D>(parts, gridDim.x, blockIdx.x) = c;
}

// Joins the parts of the item that CTA i of the kernel before began: part 1 of that CTA, part 0 of those behind. A thread has 4 dims of a row; of more
// than four parts four threads take every fourth each. Eight parts are on their way at a time. `share` of `shares` blocks takes every shares-th lot.
static constexpr int kJoinThreads = 256;
struct Fp4Sum {
  float4 o;
  float m, l;
  __device__ __forceinline__ void add(const float4* v, const float2* ml, int n) {
    float mx = m;
    for (int k = 0; k < n; ++k) mx = fmaxf(mx, ml[k].x);
    const float f0 = m == -INFINITY ? 0.f : ex2_of(m - mx);
    m = mx;
    l *= f0;
    o.x *= f0; o.y *= f0; o.z *= f0; o.w *= f0;
    for (int k = 0; k < n; ++k) {
      const float f = ml[k].x == -INFINITY ? 0.f : ex2_of(ml[k].x - mx);
      l += ml[k].y * f;
      o.x += v[k].x * f; o.y += v[k].y * f; o.z += v[k].z * f; o.w += v[k].w * f;
    }
  }
};
template <class Entry, int D>
__device__ __forceinline__ void fp4_join(const Fp4Attn& p, float* parts, uint32_t grid, int i, int share, int shares) {
  constexpr int kRows = Entry::kRows;
  __shared__ float4 sum_o[kJoinThreads];
  __shared__ float2 sum_ml[kJoinThreads];
  const Fp4Cut cut = *fp4_cut<Entry, D>(parts, grid, i);
  const int turns = cut.last - i >= 4 ? 4 : 1, lot = kJoinThreads / turns;
  const int lane = threadIdx.x & (lot - 1), turn = threadIdx.x / lot;
  constexpr bool kByRow = kRows <= 16;
  for (int x0 = share * lot; x0 < (kByRow ? cut.rows : cut.rows > 0 ? kRows : 0) * (D / 4); x0 += shares * lot) {
    const int x = x0 + lane, r = kByRow ? x / (D / 4) : x % kRows, d = (kByRow ? x % (D / 4) : x / kRows) * 4;
    Fp4Sum sum = {make_float4(0.f, 0.f, 0.f, 0.f), -INFINITY, 0.f};
    if (r < cut.rows) {
      for (int c0 = i + turn; c0 <= cut.last; c0 += 8 * turns) {
        float2 ml[8];
        float4 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int c = c0 + k * turns;
          const float* part = parts + fp4_part<Entry, D>(c, c == i);
          ml[k] = c <= cut.last ? *reinterpret_cast<const float2*>(part + kRows * D + 2 * r) : make_float2(-INFINITY, 0.f);
          v[k] = c <= cut.last ? *reinterpret_cast<const float4*>(part + fp4_part_at<Entry, D>(r, d)) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        sum.add(v, ml, 8);
      }
    }
    if (turns > 1) {
      sum_o[threadIdx.x] = sum.o;
      sum_ml[threadIdx.x] = make_float2(sum.m, sum.l);
      __syncthreads();
      if (turn == 0) {
        float4 v[3];
        float2 ml[3];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          v[k] = sum_o[(k + 1) * lot + lane];
          ml[k] = sum_ml[(k + 1) * lot + lane];
        }
        sum.add(v, ml, 3);
      }
      __syncthreads();
    }
    if (turn == 0 && r < cut.rows) {
      const float inv = sum.l == 0.f ? 0.f : 1.f / sum.l;
      const int token = p.by_group.of(cut.row0 + r), head = cut.head0 + cut.row0 + r - token * p.G;
      *reinterpret_cast<uint2*>(p.out + (long long)(cut.token0 + token) * p.ldo + (long long)head * D + d) =
          make_uint2(pack_bf16x2(sum.o.x * inv, sum.o.y * inv), pack_bf16x2(sum.o.z * inv, sum.o.w * inv));
    }
  }
}

// What a kernel needs set once a device, before its first launch there; a call that comes meanwhile waits.
struct Fp4Once {
  std::mutex lock;
  unsigned long long done = 0;
  template <class Set>
  bool run(Set set) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return false;
    const std::lock_guard<std::mutex> held(lock);
    const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
    if (done & bit) return true;
    if (!set()) return false;
    done |= bit;
    return true;
  }
};

// The tile kernel (fp4_prefill.cu): the grid it runs on, its least cells a CTA, and its launch.
int fp4_tile_grid();
static constexpr int kTileLeast = 1;
int launch_fp4_tiles(const Fp4Attn& p, int D, float* parts, cudaStream_t stream);

}  // namespace b200
