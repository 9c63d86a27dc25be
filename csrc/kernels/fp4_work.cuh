// How attention over the 4-bit cache is shared out, for both of its kernels. An entry (a sequence, or a tile of 128 query tokens) has items (kv head,
// row tile) that all read the same number of key cells. The cells of all items of all entries stand in one line, each CTA takes an equal stretch of
// it, and the parts of items that the ends of stretches cut are joined afterwards. What an item costs besides its cells (queries, output) stands in
// the line as kStart cells in front of them: without, the CTAs that get the short items of a causal prompt's beginning finish last.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fp4_cache.cuh"
#include "sm100.cuh"

namespace b200 {

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
  float scale_log2, softcap2;
  int* status;
};

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
// Scale bytes lo and hi (selectors of __byte_perm) of w -> f16x2.
__device__ __forceinline__ uint32_t scales_f16x2(uint32_t w, int lo, int hi) { return __byte_perm(w, 0, 0x4040 | lo | hi << 8) << 7; }
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Probabilities are 2^(score - m + kUp), m a reference of the running maximum that is raised when a score passes it by 8: at most 2^15 in f16, and
// the smallest ones keep their bits.
static constexpr float kUp = 7.f;

// lowest position that the query at `pos` sees
__device__ __forceinline__ int fp4_lowest(const Fp4Attn& p, int pos) {
  return p.window > 0 ? pos - p.window + 1 : p.window < 0 && pos >= 0 ? pos / -p.window * -p.window : 0;
}
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
template <int ROWS>
struct Fp4Seq {                // cells of 16 keys, row tiles of ROWS
  static constexpr int kRows = ROWS, kStart = 0, kSnap = 0;
  int req, len, token0, rows, first, begin, cells, tiles;       // begin: first cell of the sequence that any row sees
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
    begin = max(0, fp4_lowest(p, first)) / kCellTokens;
    cells = kStart + max(1, (len + kCellTokens - 1) / kCellTokens - begin);          // (no keys: one cell that counts as masked)
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

// line[i] = cells in the line in front of entry i (count + 1 values). All threads of the block take part.
template <class Entry>
__device__ void fp4_line(const Fp4Attn& p, uint32_t* line) {
  __shared__ uint32_t warp_sum[32];
  const int n = Entry::count(p), per = (n + blockDim.x - 1) / blockDim.x, b0 = min((int)threadIdx.x * per, n), b1 = min(b0 + per, n);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  uint32_t sum = 0;
  for (int b = b0; b < b1; ++b) {
    const Entry e(p, b);
    const uint32_t c = (uint32_t)e.cells * (uint32_t)(e.tiles * p.Hkv);
    line[b + 1] = c;
    sum += c;
  }
  uint32_t x = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_sum[warp] = x;
  __syncthreads();
  uint32_t before = x - sum;
  for (int w = 0; w < warps; ++w) before += w < warp ? warp_sum[w] : 0;
  for (int b = b0; b < b1; ++b) {
    before += line[b + 1];
    line[b + 1] = before;
  }
  if (threadIdx.x == 0) line[0] = 0;
  __syncthreads();
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
  const uint32_t u = (uint32_t)((uint64_t)total * i / ctas);
  if (Entry::kSnap == 0 || u == 0 || u >= total) return u;
  const int b = fp4_find(line, Entry::count(p), u);
  const uint32_t n = Entry(p, b).cells, off = (u - line[b]) % n;
  return n <= Entry::kSnap + Entry::kStart ? u - off + (2 * off >= n ? n : 0) : off <= Entry::kStart ? u - off : u;
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

// Scratch of a part: O [rows][D], then (m, l) of each row; in CTA order, two a CTA.
template <class Entry, int D>
__device__ __forceinline__ size_t fp4_part(uint32_t cta, int part) { return ((size_t)cta * 2 + part) * (Entry::kRows * (D + 2)); }

// Joins the parts of cut items. Block i looks at the line where stretch i + 1 begins; the first cut of an item is the one that joins it: part 1 of the
// CTA that begins it, part 0 of those behind. `share` of `shares` blocks takes every shares-th 4 dims.
template <class Entry, int D>
__device__ __forceinline__ void fp4_join(const Fp4Attn& p, const float* parts, uint32_t* line, uint32_t i, uint32_t grid, int least, int share,
                                         int shares) {
  constexpr int kRows = Entry::kRows;
  fp4_line<Entry>(p, line);
  const int entries = Entry::count(p);
  const uint32_t total = line[entries], ctas = fp4_ctas(total, grid, least);
  if (i + 1 >= ctas) return;
  const uint32_t u = fp4_begin<Entry>(p, line, total, i + 1, ctas);
  if (u >= total) return;
  const int b = fp4_find(line, entries, u);
  const Entry e(p, b);
  const uint32_t item = (u - line[b]) / (uint32_t)e.cells, begin = line[b] + item * e.cells;
  if (begin == u || fp4_begin<Entry>(p, line, total, i, ctas) > begin) return;
  const uint32_t last = (uint32_t)(((uint64_t)(begin + e.cells) * ctas - 1) / total);         // the CTA that has the item's last cell
  const int h = item / e.tiles, r0 = (int)(item - h * e.tiles) * kRows, nrows = min(kRows, e.rows - r0);
  for (int x = threadIdx.x + share * blockDim.x; x < nrows * (D / 4); x += shares * blockDim.x) {
    const int r = x / (D / 4), d = x % (D / 4) * 4;
    float mx = -INFINITY;
    for (uint32_t c = i; c <= last; ++c) mx = fmaxf(mx, parts[fp4_part<Entry, D>(c, c == i) + kRows * D + 2 * r]);
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll 4
    for (uint32_t c = i; c <= last; ++c) {
      const float* part = parts + fp4_part<Entry, D>(c, c == i);
      const float2 ml = *reinterpret_cast<const float2*>(part + kRows * D + 2 * r);
      const float4 v = *reinterpret_cast<const float4*>(part + r * D + d);
      const float f = ml.x == -INFINITY ? 0.f : ex2_of(ml.x - mx);
      sum += ml.y * f;
      a.x += v.x * f; a.y += v.y * f; a.z += v.z * f; a.w += v.w * f;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int token = (r0 + r) / p.G, head = r0 + r - token * p.G;
    *reinterpret_cast<uint2*>(p.out + (long long)(e.token0 + token) * p.ldo + (long long)(h * p.G + head) * D + d) =
        make_uint2(pack_bf16x2(a.x * inv, a.y * inv), pack_bf16x2(a.z * inv, a.w * inv));
  }
}

// The tile kernel (fp4_prefill.cu): the grid it runs on, its least cells a CTA, and its launch.
int fp4_tile_grid();
static constexpr int kTileLeast = 1;
int launch_fp4_tiles(const Fp4Attn& p, int D, float* parts, cudaStream_t stream);

}  // namespace b200
