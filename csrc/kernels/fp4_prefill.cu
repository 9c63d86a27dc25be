// Attention over the paged cache held in 4 bits, for many query rows a sequence (prompts and portions of prompts), on tcgen05 / tensor memory.
//
// A CTA works on 256 rows (query tokens x heads of a group: neighbouring rows share their keys, whatever the group) as two halves of 128 over tiles
// of 128 keys:
//   S(t) = Q(t) K^T,   P(t) = 2^(S - m + 7),   O(t) += P(t) V
// Keys and values are expanded to f16 on the way to shared memory, by four warps that read codes and scales straight from the cache's cells and
// write the 128-byte swizzled tiles that the matrix instructions take (keys with dims contiguous, values the same: their operand is MN-major). A tile
// is expanded once for 256 rows. Q is f16 times a power of two per row, which goes back into the softmax scale. While the softmax of one half
// runs, the tensor pipe works on the other, in the order of issue of the bf16 kernel for two heads (attn_prefill.cu):
//   P(t, j) written and V(j) there   ->  O(t) += P(t, j) V(j), then, with K(j+1) there, S(t) = Q(t) K(j+1)^T
// P goes back to tensor memory over its scores. The work of a call is shared out evenly among one CTA an SM (fp4_work.cuh): long and short
// prompts, early and late tiles of a causal prompt, a portion of few tokens after a long context.
//
// Tensor memory (512 columns): S0 | S1 | O0 | O1; P(t) is the first 64 columns of S(t).
// Warps (512 threads): 0 issues MMAs and holds tensor memory; 4..7 and 8..11 softmax and output of half 0 and 1, a thread a row; 12..15 expand, a
// thread a key. Registers move from the first and the last warpgroup to the two of the softmax.
//
// 1999 tokens behind 30000, 32 heads over 8 of 128 dims: 852 us, 1.19 PFLOP/s; a causal prompt of 8192 572 us, 0.96 PFLOP/s (0.72 and 0.58 of
// what a large product reaches). What bounds it: a tile's exponentials, 16 a cycle, and its products take some 2050 cycles each, and mostly one after the
// other: in a prompt of 4096 either unit is busy in 0.45 of the cycles. The masks of the diagonal, the queries and the outputs of a causal prompt's short
// items come on top. A piece costs some 3500 cycles for queries and output, what short prompts pay: 13 of 3 to 211 tokens take 35 us.
//
// Rows differ in what they see of a tile, so a NaN among values does not reach the product: expanders name the keys that have one and put zero, and the
// softmax marks its row's groups where it sees such a key (8192 tokens 562 us without, 572 with it).
#include "api.h"
#include "fp4_work.cuh"

namespace b200 {

static constexpr int kFRing = 4;
static constexpr int kRegsIssue = 40, kRegsSoftmax = 184, kRegsExpand = 96;

__host__ __device__ constexpr uint32_t umma_idesc_f16(int m, int n, int b_mn) {
  return (1u << 4) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
template <int N>
__device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

template <int D>
struct Fp4TileShape {
  static constexpr int kHalves = D / 64;                    // 64-dim halves of an operand tile
  static constexpr int kPlane = 128 * 128;                  // 128 rows of 64 dims
  static constexpr int kSlot = kHalves * kPlane;
  static constexpr int kLine = (2 + kFRing) * kSlot;        // Q of both halves, the ring, then the line
};

struct alignas(8) Fp4TileBars {
  uint64_t q_full[2], kv_full[kFRing], kv_empty[kFRing], s_full[2], p_first[2], p_full[2], pv_done[2];
  uint32_t tmem_base;
};

// What a piece has for its two halves: `rows` of the tile's 256 exist, key tiles [c0, c1) of the item are seen by any of them.
struct Fp4TilePiece {
  int h, r0, rows, halves, k0, n, first;       // k0: first key of the piece's first tile, n: tiles
  __device__ __forceinline__ Fp4TilePiece() {}
  __device__ __forceinline__ Fp4TilePiece(const Fp4Attn& p, const Fp4Piece<Fp4Tile>& w) {
    const Fp4Tile& e = w.e;
    h = fp4_head(w.item, e.tiles);
    r0 = (w.item - h * e.tiles) * Fp4Tile::kRows;
    rows = min(Fp4Tile::kRows, e.rows - r0);
    halves = rows > 128 ? 2 : 1;
    first = e.first;
    const int low = max(0, fp4_lowest(p, first + p.by_group.of(r0))), high = min(p.causal ? first + p.by_group.of(r0 + rows - 1) : e.len - 1, e.len - 1);
    const int t0 = max(e.begin + w.from(), low / kTileKeys), t1 = min(e.begin + w.to(), high < 0 ? 0 : high / kTileKeys + 1);
    k0 = t0 * kTileKeys;
    n = max(0, t1 - t0);
  }
};

// CAP: scores are as they are (0), capped, or capped far above them (2, fp4_wide_capped). A kernel each: what a call does not need is not in its loop.
template <int D, int CAP>
__global__ void __launch_bounds__(512, 1) fp4_tiles_kernel(Fp4Attn p, float* parts) {
  using Cell = Fp4Cell<D>;
  using Shape = Fp4TileShape<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ Fp4TileBars bars;
  __shared__ uint32_t no_page[4][4];                            // key tiles in turn: keys of a warp of expanders that have no page,
  __shared__ uint32_t odd_keys[4][4];                           // those, and the ones with a NaN among their values;
  __shared__ uint8_t nan_groups[4][kTileKeys];                  // of such a key: the groups (16 dims) that are NaN
  __shared__ uint8_t row_nan[Fp4Tile::kRows];                   // the groups of which a row has seen a NaN
  __shared__ Fp4Piece<Fp4Tile> held[16];                        // each warp's piece, out of the registers of its loop over tiles,
  __shared__ Fp4TilePiece held_tile[16];                        // and what it comes to
  uint8_t* sQ = smem;
  uint8_t* ring = smem + 2 * Shape::kSlot;
  uint32_t* line = reinterpret_cast<uint32_t*>(smem + Shape::kLine);
  const int warp = warp_index(), lane = threadIdx.x & 31, group = warp >> 2;
  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bars.q_full[t], 4);
      mbar_init(&bars.s_full[t], 1);
      mbar_init(&bars.p_first[t], 4);
      mbar_init(&bars.p_full[t], 4);
      mbar_init(&bars.pv_done[t], 1);
    }
    for (int i = 0; i < kFRing; ++i) {
      mbar_init(&bars.kv_full[i], 4);
      mbar_init(&bars.kv_empty[i], 1);
    }
    mbar_fence_init();
  }
  if (warp == 0) {
    tmem_alloc(&bars.tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = bars.tmem_base;
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t total = fp4_line<Fp4Tile>(p, line), ctas = fp4_ctas(total, gridDim.x, kTileLeast);
  const uint2 stretch = fp4_stretch<Fp4Tile>(p, line, total, ctas);
  const uint32_t from = stretch.x, to = stretch.y;
  if (threadIdx.x == 32) fp4_say_cut<Fp4Tile, D>(p, line, total, ctas, from, to, parts);        // (of a warp without a part to play)
  Fp4Piece<Fp4Tile>& w = held[warp];
  Fp4TilePiece& x = held_tile[warp];
  const auto hold = [&](const Fp4Piece<Fp4Tile>& now) {
    Fp4TilePiece y;
    if (now.more()) y = Fp4TilePiece(p, now);
    __syncwarp();
    if (lane == 0) {
      w = now;
      x = y;
    }
    __syncwarp();
  };
  const auto begin = [&] {
    Fp4Piece<Fp4Tile> now;
    now.at(p, line, from, to);
    hold(now);
  };
  const auto next = [&] {
    Fp4Piece<Fp4Tile> now = w;
    now.next(p, line);
    hold(now);
  };

  if (group == 0) {
    regs_dec<kRegsIssue>();
    if (warp == 0) {
      constexpr uint32_t idesc_qk = umma_idesc_f16(128, kTileKeys, 0), idesc_pv = umma_idesc_f16(128, D, 1);
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0), q_addr = smem_u32(sQ), ring_addr = smem_u32(ring);
      uint32_t sq = 0, pieces[2] = {0, 0}, count[2] = {0, 0};    // ring items, pieces and tiles of each half so far
      bool ok = true;
      for (begin(); w.more() && ok; next()) {
        const int n = x.n, halves = x.halves;
        if (n == 0) continue;
        const auto qk = [&](int t, uint32_t slot, bool last) {      // S(t) = Q(t) K^T
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              umma_bf16_ss(tm + t * 128, umma_desc_k_sw128(q_addr + t * Shape::kSlot + (kk / 4) * Shape::kPlane + (kk % 4) * 32, 1024),
                           umma_desc_k_sw128(ring_addr + slot * Shape::kSlot + (kk / 4) * Shape::kPlane + (kk % 4) * 32, 1024), idesc_qk, kk != 0);
            umma_commit(&bars.s_full[t]);
            if (last) umma_commit(&bars.kv_empty[slot]);
          }
          __syncwarp();
        };
        const auto wait_kv = [&](uint32_t i) { return mbar_wait_warp(&bars.kv_full[i % kFRing], (i / kFRing) & 1, p.status); };
        if (!(ok = wait_kv(sq))) break;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (t >= halves || !ok) continue;
          if (!(ok = mbar_wait_warp(&bars.q_full[t], pieces[t] & 1, p.status))) continue;
          ++pieces[t];
          tc_fence_after_sync();
          qk(t, sq % kFRing, t == halves - 1);
        }
        for (int j = 0; j < n && ok; ++j) {
          const uint32_t iv = sq + 2 * j + 1, ik = iv + 1, slot = iv % kFRing;
          const uint64_t vd = umma_desc_mn_sw128(ring_addr + slot * Shape::kSlot, Shape::kPlane, 1024);
          if (!(ok = wait_kv(iv))) break;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (t >= halves || !ok) continue;
            const uint32_t phase = count[t] & 1;
            ++count[t];
            if (!(ok = mbar_wait_warp(&bars.p_first[t], phase, p.status))) continue;
            tc_fence_after_sync();
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < kTileKeys / 32; ++kk)
                umma_bf16_ts(tm + 256 + t * 128, tm + t * 128 + kk * 8, vd + kk * (2048 >> 4), idesc_pv, (j | kk) != 0);
            }
            __syncwarp();
            if (!(ok = mbar_wait_warp(&bars.p_full[t], phase, p.status))) continue;
            tc_fence_after_sync();
            if (elect_one()) {
#pragma unroll
              for (int kk = kTileKeys / 32; kk < kTileKeys / 16; ++kk)
                umma_bf16_ts(tm + 256 + t * 128, tm + t * 128 + kk * 8, vd + kk * (2048 >> 4), idesc_pv, 1);
              if (t == halves - 1) umma_commit(&bars.kv_empty[slot]);
              if (j == n - 1) umma_commit(&bars.pv_done[t]);
            }
            __syncwarp();
            if (j + 1 < n) {
              if (t == 0) {
                if (!(ok = wait_kv(ik))) continue;
                tc_fence_after_sync();
              }
              qk(t, ik % kFRing, t == halves - 1);
            }
          }
        }
        sq += 2 * n;
      }
    }
  } else if (group == 3) {
    // ---------------- expanders: thread r has key r of a tile ----------------
    regs_dec<kRegsExpand>();
    const int r = threadIdx.x & 127, token = r % kCellTokens;
    const long long head_bytes = (long long)p.cells_per_page * Cell::kBytes;
    uint32_t sq = 0, tiles = 0;
    bool ok = true;
    for (begin(); w.more() && ok; next()) {
      const int n = x.n, k0 = x.k0, len = w.e.len, h = x.h;
      if (n == 0) continue;
      const int32_t* table = p.block_table + w.e.req * p.ldt;
      const int low = max(0, fp4_lowest(p, x.first + p.by_group.of(x.r0)));
      const auto page_of = [&](int j) {                          // -1: none; -2: not a key that any row sees
        const int pos = k0 + j * kTileKeys + r;
        return pos >= low && pos < len ? max(-1, table[p.by_page_cells.of(pos / kCellTokens)]) : -2;
      };
      const auto cell_of = [&](int j, int page) -> const uint8_t* {
        const int c = (k0 + j * kTileKeys + r) / kCellTokens, cell = c - p.by_page_cells.of(c) * p.cells_per_page;
        return page >= 0 && page < p.num_blocks ? p.cache + ((long long)page * p.Hkv + h) * head_bytes + (long long)cell * Cell::kBytes : nullptr;
      };
      uint4 code[D / 32];
      uint32_t scale[D / 64], value_scale[D / 16];              // (a byte each; those of a key's values come with the key)
      const auto load = [&](const uint8_t* cell, int kv) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) code[i] = make_uint4(0, 0, 0, 0);
        if (!kv) {
#pragma unroll
          for (int i = 0; i < D / 64; ++i) scale[i] = 0;
#pragma unroll
          for (int i = 0; i < D / 16; ++i) value_scale[i] = 0;
        }
        if (!cell) return;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
          code[i] = *reinterpret_cast<const uint4*>(cell + (kv ? Cell::value_at(token, i * 16) : token * Cell::kRow + i * 16));
        if (!kv) {
#pragma unroll
          for (int i = 0; i < D / 64; ++i) scale[i] = reinterpret_cast<const uint32_t*>(cell + Cell::kKeyScales + token * Cell::kScales)[i];
#pragma unroll
          for (int i = 0; i < D / 16; ++i) value_scale[i] = cell[Cell::kValueScales + i * kCellTokens + token];
        }
      };
      int page = page_of(0);
      const uint8_t* cell = cell_of(0, page);
      load(cell, 0);
      for (int i = 0; i < 2 * n; ++i, ++sq) {
        const int j = i >> 1, kv = i & 1;
        const uint32_t slot = sq % kFRing;
        const bool none = page != -2 && cell == nullptr;
        uint4 c[D / 32];
        uint32_t s[D / 64];
#pragma unroll
        for (int k = 0; k < D / 32; ++k) c[k] = code[k];
#pragma unroll
        for (int k = 0; k < D / 64; ++k) {
          s[k] = scale[k];
          // A NaN among values does not go to the product, where 0 times it would reach the rows that do not see its key: their softmax marks the rows
          // that do.
          if (kv) s[k] &= ~((nan_scales(s[k]) >> 7) * 255u);
        }
        // the next item's loads, and in front of a key tile's the page
        if (kv == 0) {
          load(cell, 1);
          if (j + 1 < n) page = page_of(j + 1);
        } else if (j + 1 < n) {
          cell = cell_of(j + 1, page);
          load(cell, 0);
        }
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(&bars.kv_empty[slot], ((sq / kFRing) & 1) ^ 1, p.status)))) break;
        uint8_t* row = ring + slot * Shape::kSlot + r * 128;
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
          const uint32_t word[4] = {c[k].x, c[k].y, c[k].z, c[k].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int g = 2 * k + (e >> 1), piece = 4 * k + e;                   // scale, 16 bytes of the row
            const uint32_t sc = scales_f16x2(s[g / 4], g % 4, g % 4);
            uint32_t v[4];
            e2m1x8_f16(word[e], v);
            *reinterpret_cast<uint4*>(row + (piece / 8) * Shape::kPlane + (((piece % 8) ^ (r & 7)) << 4)) =
                make_uint4(mul_f16x2(v[0], sc), mul_f16x2(v[1], sc), mul_f16x2(v[2], sc), mul_f16x2(v[3], sc));
          }
        }
        if (kv == 0) {
          uint32_t nan = 0;
#pragma unroll
          for (int k = 0; k < D / 64; ++k)
            scale[k] = value_scale[4 * k] | value_scale[4 * k + 1] << 8 | value_scale[4 * k + 2] << 16 | value_scale[4 * k + 3] << 24;
#pragma unroll
          for (int k = 0; k < D / 64; ++k) nan |= ((nan_scales(scale[k]) >> 7) * 0x10204080u >> 28) << (4 * k);
          const uint32_t mask = __ballot_sync(0xffffffffu, none), odd = mask | __ballot_sync(0xffffffffu, nan != 0);
          if (lane == 0) {
            no_page[tiles % 4][warp & 3] = mask;
            odd_keys[tiles % 4][warp & 3] = odd;
          }
          if (odd) nan_groups[tiles % 4][r] = nan;
          ++tiles;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.kv_full[slot]);
      }
    }
  } else {
    // ---------------- softmax and output: thread r has row r of half t ----------------
    regs_inc<kRegsSoftmax>();
    const int t = group - 1, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_addr = tmem + t * 128 + lane_off, o_addr = tmem + 256 + t * 128 + lane_off;
    uint32_t pieces = 0, count = 0, tiles = 0;
    bool ok = true;
    // Queries come and outputs go in whole lines: a warp's 32 rows, kTurnRows of them at a time, a lane 16 bytes. (A lane a row takes a line a lane:
    // the loads and stores of 256 rows were 8000 cycles a piece so.)
    constexpr int kRowLanes = D / 8, kTurnRows = 32 / kRowLanes;
    const int piece16 = lane % kRowLanes, turn_row = lane / kRowLanes, row0 = t * 128 + quarter * 32;
    uint8_t* own = sQ + t * Shape::kSlot + quarter * 32 * 128;   // the warp's rows of Q (in each plane); the outputs pass through there too
    constexpr int kPart = 4096 / (2 * D);                        // rows of D bf16 in the warp's part of a plane
    const auto own_at = [&](int row, int piece) {
      return own + row / kPart * Shape::kPlane + row % kPart * (2 * D) + ((piece ^ (row & 7)) << 4);
    };
    // a value that the compiler takes for new: what follows from it is not kept in registers over the loop of tiles
    const auto here = [](int v) {
      asm volatile("" : "+r"(v));
      return v;
    };
    uint4 raw[kRowLanes];
    const auto rows_from = [&](int r0, long long ld, auto&& each) {      // each(i, offset of the lane's piece of turn i's row)
      const int G = here(p.G), rr = r0 + row0 + here(turn_row), token = p.by_group.of(rr), step_token = p.by_group.of(kTurnRows), step_head = kTurnRows - step_token * G;
      int head = rr - token * G;
      long long at = token * ld + head * D + piece16 * 8;
      const long long step = step_token * ld + step_head * D, wrap = ld - G * D;
#pragma unroll
      for (int i = 0; i < kRowLanes; ++i) {
        each(i, at);
        head += step_head;
        at += step;
        if (head >= G) {
          head -= G;
          at += wrap;
        }
      }
    };
    const auto query = [&] {                                     // the rows' queries of the piece, on their way
      const int left = w.more() && x.n > 0 ? x.rows - row0 - turn_row : 0;       // (raw is set in any case: what it held before is not kept)
      const __nv_bfloat16* q = p.q + (long long)w.e.token0 * p.ldq + (long long)x.h * p.G * D;
      rows_from(x.r0, p.ldq, [&](int i, long long at) {
        raw[i] = i * kTurnRows < left ? *reinterpret_cast<const uint4*>(q + at) : make_uint4(0, 0, 0, 0);
      });
    };
    begin();
    query();
    while (w.more() && ok) {
      if (t >= x.halves) {
        tiles += x.n;
        next();
        query();
        continue;
      }
      const int n = x.n, k0 = x.k0;
      int hi, lo;
      float sc = p.scale_log2, m = -INFINITY, l = 0.f;
      {
        const int token = p.by_group.of(x.r0 + min(t * 128 + r, x.rows - 1)), pos = x.first + token;
        hi = min(p.causal ? pos : w.e.len - 1, w.e.len - 1);
        lo = fp4_lowest(p, pos);
      }
      *const_cast<volatile uint8_t*>(row_nan + t * 128 + r) = 0;
      if (n > 0) {
        // ---- the rows' queries (every product of the piece before is done: its last scores have been read), turned to a lane a row on the way
        const int mine = here(lane), turn = here(turn_row);
#pragma unroll
        for (int i = 0; i < kRowLanes; ++i) *reinterpret_cast<uint4*>(own_at(i * kTurnRows + turn, piece16)) = raw[i];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kRowLanes; ++i) raw[i] = *reinterpret_cast<const uint4*>(own_at(mine, i));
        __syncwarp();
        __nv_bfloat162 most = __float2bfloat162_rn(0.f);
#pragma unroll
        for (int i = 0; i < kRowLanes; ++i) {
          const uint32_t v[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) most = __hmax2(most, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&v[e])));
        }
        const float big = fmaxf(__low2float(most), __high2float(most));
        const int e2 = min(max((int)(__float_as_uint(big) >> 23) - 127, -126), 126);
        const __nv_bfloat162 down = __float2bfloat162_rn(__uint_as_float((uint32_t)(127 - e2) << 23));       // (exact)
        // (never 0, as for queries of zeros and a small scale: a masked score, -infinity, times it would be NaN; so small a factor leaves all scores 0)
        sc = fminf(fmaxf(p.scale_log2 * __uint_as_float((uint32_t)(127 + e2) << 23), 1.2e-38f), 3.0e38f);
#pragma unroll
        for (int i = 0; i < kRowLanes; ++i) {
          const uint32_t v[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
          uint32_t f16[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const __nv_bfloat162 y = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&v[e]), down);
            const float2 f = __bfloat1622float2(y);
            f16[e] = pack_f16x2(f.x, f.y);
          }
          *reinterpret_cast<uint4*>(own + (i / 8) * Shape::kPlane + mine * 128 + (((i % 8) ^ (mine & 7)) << 4)) =
              make_uint4(f16[0], f16[1], f16[2], f16[3]);
        }
        fence_proxy_async_smem();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.q_full[t]);
      }
      for (int j = 0; j < n; ++j, ++count, ++tiles) {
        ok = __all_sync(0xffffffffu, mbar_wait(&bars.s_full[t], count & 1, p.status));
        if (!ok) break;
        tc_fence_after_sync();
        uint32_t s[kTileKeys];
#pragma unroll
        for (int c = 0; c < kTileKeys / 32; ++c) tmem_ld_32x32b_x32(s_addr + c * 32, s + c * 32);
        tmem_ld_wait();
        const int kbase = k0 + j * kTileKeys;
        if constexpr (CAP > 0) {                                 // (scores in log2 units from here on)
          const float in = fp4_cap_in(sc, p.softcap2);
#pragma unroll
          for (int i = 0; i < kTileKeys; ++i) {
            const float x = __uint_as_float(s[i]);
            s[i] = __float_as_uint(CAP == 2 ? fp4_wide_capped(x, in, p.softcap2) : fp4_capped(x, in, p.softcap2));
          }
        }
        const float to_log2 = CAP > 0 ? 1.f : sc;
        if (kbase + kTileKeys - 1 > hi || kbase < lo) {
#pragma unroll
          for (int i = 0; i < kTileKeys; ++i)
            if (kbase + i > hi || kbase + i < lo) s[i] = 0xff800000u;       // -inf
        }
        const volatile uint32_t* odd = odd_keys[tiles % 4];
        if (odd[0] | odd[1] | odd[2] | odd[3]) {
          const volatile uint32_t* gone = no_page[tiles % 4];
          const uint32_t g0 = gone[0], g1 = gone[1], g2 = gone[2], g3 = gone[3];
#pragma unroll
          for (int i = 0; i < kTileKeys; ++i)
            if ((i < 32 ? g0 : i < 64 ? g1 : i < 96 ? g2 : g3) >> (i & 31) & 1) s[i] = 0xff800000u;
          uint32_t seen = 0;                                     // groups that are NaN, of the keys that the row sees (0 for those without a page)
#pragma unroll 1
          for (int k = 0; k < 4; ++k)
            for (uint32_t left = odd[k]; left; left &= left - 1) {
              const int i = k * 32 + __ffs(left) - 1;
              if (kbase + i <= hi && kbase + i >= lo) seen |= nan_groups[tiles % 4][i];
            }
          volatile uint8_t* mine = row_nan + t * 128 + r;
          *mine = *mine | seen;
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < kTileKeys; i += 4)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], __uint_as_float(s[i + e]));
        const float tile_max = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * to_log2;
        float alpha = 1.f;
        bool rescale = false;
        if (tile_max > m + 8.f) {          // also the first finite tile: m == -inf
          if (m != -INFINITY) {
            alpha = ex2_of(m - tile_max);
            rescale = j > 0;
          }
          m = tile_max;
        }
        const float off = m == -INFINITY ? 0.f : kUp - m;
        // O is at rest: S(j) is issued right behind P V(j - 1), by the same elected lane, and a commit covers all that its thread has issued before
        if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            tmem_ld_32x32b_x16(o_addr + c * 16, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st_32x32b_x16(o_addr + c * 16, o);
          }
        }
        const uint64_t sc2 = pack_f32x2(to_log2, to_log2), off2 = pack_f32x2(off, off);
        uint64_t sum2[2] = {0, 0};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float a, b;
            unpack_f32x2(fma_f32x2(pack_b32x2(s[c * 32 + 2 * i], s[c * 32 + 2 * i + 1]), sc2, off2), a, b);
            a = ex2_of(a);
            b = ex2_of(b);
            sum2[i & 1] = add_f32x2(sum2[i & 1], pack_f32x2(a, b));
            pk[i] = pack_f16x2(a, b);
          }
          tmem_st_32x32b_x16(s_addr + c * 16, pk);
          if (c == 1) {                  // P V of the first half of the keys may start
            tmem_st_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.p_first[t]);
          }
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
      if (!ok) break;
      const int left = x.rows - row0, r0 = x.r0, part_of = w.part();
      const bool whole = w.whole();
      const long long out0 = (long long)w.e.token0 * p.ldo + (long long)x.h * p.G * D;
      next();
      query();
      if (n > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(&bars.pv_done[t], pieces & 1, p.status));
        if (!ok) break;
        ++pieces;
        tc_fence_after_sync();
      }
      const uint32_t nan = *const_cast<const volatile uint8_t*>(row_nan + t * 128 + r);
      const auto mark = [&](uint32_t (&o)[32], int c) {          // of 32 dims
        if (__any_sync(0xffffffffu, nan != 0)) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (nan >> (2 * c + i / 16) & 1) o[i] = 0x7fffffffu;
        }
      };
      if (whole) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int mine = here(lane), turn = here(turn_row);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          if (n > 0) {
            tmem_ld_32x32b_x32(o_addr + c * 32, o);   // (whole warp)
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0;
          }
          mark(o, c);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              v[e] = pack_bf16x2(__uint_as_float(o[8 * i + 2 * e]) * inv, __uint_as_float(o[8 * i + 2 * e + 1]) * inv);
            *reinterpret_cast<uint4*>(own_at(mine, c * 4 + i)) = make_uint4(v[0], v[1], v[2], v[3]);
          }
        }
        __syncwarp();
        __nv_bfloat16* out = p.out + out0;
        rows_from(r0, p.ldo, [&](int i, long long at) {
          const uint4 v = *reinterpret_cast<const uint4*>(own_at(turn + i * kTurnRows, piece16));
          if (turn + i * kTurnRows < left) *reinterpret_cast<uint4*>(out + at) = v;
          if (i % 4 == 3) asm volatile("" ::: "memory");         // (few at a time: the next queries hold their registers)
        });
        __syncwarp();
      } else {
        float* part = parts + fp4_part<Fp4Tile, D>(blockIdx.x, part_of);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          if (n > 0) {
            tmem_ld_32x32b_x32(o_addr + c * 32, o);   // (whole warp)
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0;
          }
          mark(o, c);
          if (lane < left) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<uint4*>(part + fp4_part_at<Fp4Tile, D>(t * 128 + r, c * 32 + i)) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
        }
        if (lane < left) *reinterpret_cast<float2*>(part + Fp4Tile::kRows * D + 2 * (t * 128 + r)) = make_float2(m, l);
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

int fp4_tile_grid() { return b200_num_sms(); }

template <int D, int CAP>
static int launch_tiles(const Fp4Attn& p, float* parts, cudaStream_t stream) {
  const size_t smem = 1024 + Fp4TileShape<D>::kLine + (size_t)(p.num_tiles + 1) * 4;
  static Fp4Once once;
  if (!once.run([] {
        cudaFuncAttributes attr;
        // (a warpgroup waits without limit for registers that the launch did not bring)
        return cudaFuncGetAttributes(&attr, fp4_tiles_kernel<D, CAP>) == cudaSuccess && 4 * attr.numRegs >= kRegsIssue + 2 * kRegsSoftmax + kRegsExpand &&
               cudaFuncSetAttribute(fp4_tiles_kernel<D, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, 1024 + Fp4TileShape<D>::kLine + 8001 * 4) == cudaSuccess;
      }))
    return -2;
  return launch_pdl(fp4_tiles_kernel<D, CAP>, dim3(fp4_tile_grid()), dim3(512), smem, stream, p, parts) == cudaSuccess ? 0 : -2;
}
template <int D>
static int launch_tiles(const Fp4Attn& p, float* parts, cudaStream_t stream) {
  return p.softcap2 > kWideCap ? launch_tiles<D, 2>(p, parts, stream) : p.softcap2 > 0.f ? launch_tiles<D, 1>(p, parts, stream) : launch_tiles<D, 0>(p, parts, stream);
}

int launch_fp4_tiles(const Fp4Attn& p, int D, float* parts, cudaStream_t stream) {
  return D == 64 ? launch_tiles<64>(p, parts, stream) : launch_tiles<128>(p, parts, stream);
}

}  // namespace b200
