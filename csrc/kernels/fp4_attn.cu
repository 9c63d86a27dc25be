// Attention over the paged cache held in 4 bits (layout: fp4_cache.cuh), for few query rows a sequence: decode, and the verification of drafts. Also
// the entry point for both kernels; sequences of many rows go to fp4_prefill.cu.
//
//   o[r] = sum_j p[r, j] v_j / sum_j p[r, j],   p[r, j] = 2^(scale log2(e) q_r . k_j - m),   m a running reference of the maximum
//
// The rows of a sequence that share a kv head (query tokens x heads of the group) are cut into tiles of 8 or 16. A warp takes pairs of cells, 32 keys:
//   S^T [16 keys x rows] = K Q^T     A = keys, straight from the cell: codes to f16 (cvt.rn.f16x2.e2m1x2), times their scale, exact
//   O^T [dims x rows]   += V^T P^T   A = values of four keys a lane; codes of two keys are merged before the conversion, so that a pair of
//                                    f16 holds two keys of one dim and one multiplication applies both scales; B = P^T, transposed in
//                                    registers (movmatrix)
// Q is f16 times a power of two per row (its largest magnitude between 1 and 2), which goes back into the softmax scale.
//
// Work is shared out evenly whatever the lengths (fp4_work.cuh). The warps of a CTA take the cells of a piece in turn, fetched ahead by bulk copies
// into a ring of their own. An item that lies in one stretch is finished there; of one that was cut the parts (m, l, O) go to scratch, and a second
// kernel joins them.
//
// mma.sync and not tcgen05: with 8 rows a product of 32 keys is 64 K multiplications a warp, and what takes the time is the 8192 codes in front of
// it, which would pass through shared or tensor memory once more. 256 sequences of 200 to 3800 keys, 32 heads over 8 of 128 dims: 137 us for 596 MB,
// 4.35 TB/s. Some 290 warp instructions a cell (64 conversions, 64 products by scales, 16 matrix products, 16 that merge the codes of two keys). No unit
// is full (96 sequences of 4096 keys): issue 0.64 of the cycles, memory 0.56, the ALU pipe 0.55, FMA 0.36, tensor 0.26; the four warps of a scheduler
// wait as often for a pipe that another has taken as for their own last instruction. One sequence of 1000 keys takes 9 us: 3.8 us until the first cell
// is there (line, table, cell: three loads one behind the other), two of work, and the join.
//
// At 256 dims there is no other kernel: a prompt's rows are tiles of 8 here, each of which expands all that it sees. 8000 tokens of 16 heads over 8 took a
// model of eight layers 76 ms where the bf16 cache takes 27.
#include <type_traits>

#include "api.h"
#include "fp4_work.cuh"

namespace b200 {

static constexpr int kRowStages = 2;
static constexpr int kNoKey = 0x7fffff00;                // first key of a cell that is not there: behind every row

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t low_half2(uint32_t v) {          // (an operand of a multiplication picks the half)
  const __half2 h = __low2half2(*reinterpret_cast<const __half2*>(&v));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t high_half2(uint32_t v) {
  const __half2 h = __high2half2(*reinterpret_cast<const __half2*>(&v));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t low_nibbles_else(uint32_t a, uint32_t b) {     // nibble 0, 2, .. of a, the others of b
  return (a & 0x0f0f0f0fu) | (b & 0xf0f0f0f0u);
}
// The lane that `says` announces `all` bytes and each lane with a source fetches `bytes` of them, without branches.
__device__ __forceinline__ void bulk_pair(uint32_t dst, const uint8_t* src, uint32_t bytes, uint32_t bar, bool says, uint32_t all) {
  asm volatile(
      "{\n\t.reg .pred a, s;\n\t"
      "setp.ne.u32 a, %4, 0;\n\t"
      "setp.ne.u64 s, %1, 0;\n\t"
      "@a mbarrier.arrive.expect_tx.shared::cta.b64 _, [%3], %5;\n\t"
      "@s cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n\t}\n" ::"r"(dst),
      "l"(src), "r"(bytes), "r"(bar), "r"((uint32_t)says), "r"(all)
      : "memory");
}
// What is left of a warp's wait whose first look found nothing.
__device__ __noinline__ bool fp4_wait(uint64_t* bar, uint32_t parity, int* status) { return mbar_wait_warp(bar, parity, status); }

template <int D, int NT>
struct Fp4RowsShape {
  static constexpr int kWarps = 8;
  static constexpr int kRows = 8 * NT, kMT = D / 16;
  static constexpr int kMergeTiles = kMT * NT <= 8 ? kMT : 8 / NT;                   // m-tiles of the merge buffer (32 KB)
  static constexpr int kMergeRow = kMergeTiles * 16 + 8;                             // floats of a row in it
  static constexpr int kRingBytes = kWarps * kRowStages * 2 * Fp4Cell<D>::kBytes;
  static constexpr int kMergeBytes = kWarps * kRows * kMergeRow * 4;
  static constexpr int kFixed = kRingBytes + kMergeBytes + kWarps * kRows * 8 + kWarps * kRowStages * 8;
};

// SEVERAL: a sequence may have several query tokens, so that rows of a tile differ in what they see. CAP: scores are capped.
template <int D, int NT, bool SEVERAL, bool CAP>
__global__ void __launch_bounds__(Fp4RowsShape<D, NT>::kWarps * 32, NT == 1 && D <= 128 ? 2 : 1) fp4_rows_kernel(Fp4Attn p, float* parts) {
  using Cell = Fp4Cell<D>;
  using Shape = Fp4RowsShape<D, NT>;
  using Seq = Fp4Seq<Shape::kRows>;
  constexpr int kRowWarps = Shape::kWarps, kThreads = kRowWarps * 32, kRows = Shape::kRows, kMT = Shape::kMT, kKW = D / 32, kVW = D / 64;   // m-tiles, words of a lane's keys and values
  extern __shared__ __align__(128) uint8_t smem[];
  float* merge = reinterpret_cast<float*>(smem + Shape::kRingBytes);
  float2* top = reinterpret_cast<float2*>(smem + Shape::kRingBytes + Shape::kMergeBytes);    // [warps][rows] m, l
  uint64_t* bars = reinterpret_cast<uint64_t*>(top + kRowWarps * kRows);
  uint32_t* line = reinterpret_cast<uint32_t*>(bars + kRowWarps * kRowStages);
  const int warp = warp_index(), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * kRowStages * 2 * Cell::kBytes;
  uint64_t* full = bars + warp * kRowStages;
  if (lane < kRowStages) mbar_init(&full[lane], 1);
  mbar_fence_init();
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t total = fp4_line<Seq>(p, line), ctas = fp4_ctas(total, gridDim.x, kRowWarps);
  const uint2 stretch = fp4_stretch<Seq>(p, line, total, ctas);
  const uint32_t from = stretch.x, to = stretch.y;
  const auto say_cut = [&] {                     // (the last warp, whose pairs run out first)
    if (threadIdx.x == kThreads - 1) fp4_say_cut<Seq, D>(p, line, total, ctas, from, to, parts);
  };
  if (from >= to) {
    say_cut();
    return;
  }

  // ---- fetching ahead: the warp's pairs of cells in their order, one on its way while another is worked on. Two neighbouring lanes have the
  // addresses of one of the next 16 pairs.
  Fp4Piece<Seq> f;
  f.at(p, line, from, to);
  __shared__ Fp4Piece<Seq> held[kRowWarps];      // each warp's piece, out of the registers of its loop over cells
  Fp4Piece<Seq>& w = held[warp];
  if (lane == 0) w = f;
  __syncwarp();
  int fc = f.from() + warp, fj = 0, fn = 0;         // the next lot's first pair; next of this lot's, how many it has
  const uint8_t* src = nullptr;
  uint32_t have = 0;                            // cells of the lot that there are (behind the keys there is none, nor on a page outside the cache)
  uint32_t cells_at[2] = {0, 0};                // cells (bit 0, bit 1) of the pair that is worked on next, and of the one behind it
  int issued = 0;                               // pairs that were fetched and not waited for
  const uint32_t ring_at = smem_u32(ring) + (lane & 1) * Cell::kBytes, full_at = smem_u32(full);
  const auto fetch = [&](int st) {
    if (fj == fn) {
      while (f.more() && fc >= f.to()) {
        f.next(p, line);
        fc = f.from() + warp;
      }
      if (!f.more()) return;
      const int pair = fc + (lane >> 1) * kRowWarps, c = 2 * (f.e.begin + pair) + (lane & 1), pg = p.by_page_cells.of(c), h = fp4_head(f.item, f.e.tiles);
      const int id = pair < f.to() && c * kCellTokens < f.e.len ? p.block_table[f.b * p.ldt + pg] : -1;
      src = id >= 0 && id < p.num_blocks
                ? p.cache + (((long long)id * p.Hkv + h) * p.cells_per_page + (c - pg * p.cells_per_page)) * Cell::kBytes : nullptr;
      have = __ballot_sync(0xffffffffu, src != nullptr);
      fj = 0;
      fn = min(16, (f.to() - fc + kRowWarps - 1) / kRowWarps);
      fc += fn * kRowWarps;
    }
    const uint32_t two = have & 3u;               // (none: the barrier's phase ends at once)
    have >>= 2;
    cells_at[1] = two;
    const bool mine = (lane >> 1) == fj;
    bulk_pair(ring_at + st * (2 * Cell::kBytes), mine ? src : nullptr, Cell::kBytes, full_at + st * 8, lane == 2 * fj,
              __popc(two) * Cell::kBytes);
    __syncwarp();
    ++issued;
    ++fj;
  };
  fetch(0);
  cells_at[0] = cells_at[1];
  fetch(1);
  say_cut();
  int st = 0;
  uint32_t parity = 0;
  bool ok = true;
  const float cap_in = CAP ? fp4_cap_in(1.f, p.softcap2) : 0.f;

  // queries: lane (g, t) has dims [t D / 4, + D / 4) of row g
  uint4 raw[NT][D / 32];
  const auto query = [&](const Fp4Piece<Seq>& x) {
    const int h = x.more() ? fp4_head(x.item, x.e.tiles) : 0, r0 = x.more() ? (x.item - h * x.e.tiles) * kRows : 0;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = r0 + nt * 8 + g, token = p.by_group.of(r), head = h * p.G + r - token * p.G;
      const __nv_bfloat16* from = p.q + (long long)(x.e.token0 + token) * p.ldq + (long long)head * D + t * (D / 4);
      const bool row = x.more() && r < x.e.rows;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) raw[nt][i] = row ? *reinterpret_cast<const uint4*>(from + i * 8) : make_uint4(0, 0, 0, 0);
    }
  };
  query(w);
  bool first_piece = true;
  while (w.more()) {
    const Seq& s = w.e;
    const int h = fp4_head(w.item, s.tiles), r0 = (w.item - h * s.tiles) * kRows, nrows = min(kRows, s.rows - r0), first = s.first;
    // ---- the tile's queries: B operand
    uint32_t bq[NT][D / 16][2];
    float mul[NT][2];                                                            // of the lane's rows 2t, 2t + 1: scores to log2 units
    int hi[NT][2], lo[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float big = 0.f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const uint32_t v[4] = {raw[nt][i].x, raw[nt][i].y, raw[nt][i].z, raw[nt][i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 x = unpack_bf16x2(v[e]);
          big = fmaxf(big, fmaxf(fabsf(x.x), fabsf(x.y)));
        }
      }
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      const int e2 = min(max((int)(__float_as_uint(big) >> 23) - 127, -126), 126);
      const float down = __uint_as_float((uint32_t)(127 - e2) << 23), up = __uint_as_float((uint32_t)(127 + e2) << 23);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const uint32_t v[4] = {raw[nt][i].x, raw[nt][i].y, raw[nt][i].z, raw[nt][i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 x = unpack_bf16x2(v[e]);
          bq[nt][2 * i + (e >> 1)][e & 1] = pack_f16x2(x.x * down, x.y * down);
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mul[nt][e] = fminf(__shfl_sync(0xffffffffu, up, (2 * t + e) * 4) * p.scale_log2, 3.0e38f);
        const int rr = min(nt * 8 + 2 * t + e, nrows - 1) + r0, pos = first + p.by_group.of(rr);
        hi[nt][e] = p.causal ? pos : s.len - 1;
        lo[nt][e] = fp4_lowest(p, pos);
      }
    }
    const int tok0 = p.by_group.of(r0), tok1 = p.by_group.of(r0 + nrows - 1);                    // the tile's tokens
    const int least_hi = p.causal ? first + tok0 : s.len - 1;
    const int most_lo = fp4_lowest(p, first + tok1), least_lo = fp4_lowest(p, first + tok0);

    // off: what is added to a score in log2 units, kUp less its row's reference
    float o[NT][kMT][4], off[NT][2], l[NT][2];
    const int k0 = 4 * (g >> 1) + (g & 1);                                       // the lane's key of a cell, and two on
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < kMT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.f;
      off[nt][0] = off[nt][1] = INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
    }
    const int c1 = w.to(), begin = s.begin, end = SEVERAL && p.causal ? first + tok1 + 1 : s.len;     // end: behind the last key that any row sees
    const int inner0 = (max(most_lo, 0) + kPairKeys - 1) / kPairKeys, inner1 = (least_hi + 1) / kPairKeys;   // pairs that every row sees all of
    for (int c = w.from() + warp; c < c1 && ok; c += kRowWarps) {
      if (!__all_sync(0xffffffffu, mbar_try_wait(&full[st], parity)) && !fp4_wait(&full[st], parity, p.status)) {
        ok = false;
        break;
      }
      --issued;
      {
        const uint32_t two = cells_at[0];
        const int pair = begin + c, key = pair * kPairKeys;
        const uint8_t* cells[2] = {ring + st * (2 * Cell::kBytes), ring + st * (2 * Cell::kBytes) + Cell::kBytes};
        // S^T: rows g and g + 8 of the tile are keys 4 (g / 2) + g % 2 and two on
        float sc[2][NT][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t kw[2][kKW], ks[2][kKW / 2];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint8_t* row = cells[u] + (k0 + 2 * r) * Cell::kRow + t * (D / 8);
            const uint8_t* sb = cells[u] + Cell::kKeyScales + (k0 + 2 * r) * Cell::kScales + t * (D / 64);
            if constexpr (D == 64) {
              const uint2 x = *reinterpret_cast<const uint2*>(row);
              kw[r][0] = x.x; kw[r][1] = x.y;
              ks[r][0] = *sb * 0x800080u;
            } else {
#pragma unroll
              for (int i = 0; i < kKW / 4; ++i) {
                const uint4 x = *reinterpret_cast<const uint4*>(row + i * 16);
                kw[r][4 * i] = x.x; kw[r][4 * i + 1] = x.y; kw[r][4 * i + 2] = x.z; kw[r][4 * i + 3] = x.w;
                const uint32_t pair = scales_f16x2(*reinterpret_cast<const uint16_t*>(sb + i * 2), 0, 1);
                ks[r][2 * i] = low_half2(pair);
                ks[r][2 * i + 1] = high_half2(pair);
              }
            }
          }
#pragma unroll
          for (int i = 0; i < kKW; ++i) {
            uint32_t x[4], y[4];
            e2m1x8_f16(kw[0][i], x);
            e2m1x8_f16(kw[1][i], y);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              x[e] = mul_f16x2(x[e], ks[0][i >> 1]);
              y[e] = mul_f16x2(y[e], ks[1][i >> 1]);
            }
            const uint32_t a0[4] = {x[0], y[0], x[1], y[1]}, a1[4] = {x[2], y[2], x[3], y[3]};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if (i == 0) mma_f16_first(sc[u][nt], a0, bq[nt][0][0], bq[nt][0][1]);
              else mma_f16(sc[u][nt], a0, bq[nt][2 * i][0], bq[nt][2 * i][1]);
              mma_f16(sc[u][nt], a1, bq[nt][2 * i + 1][0], bq[nt][2 * i + 1][1]);
            }
          }
        }
        const bool edge = two != 3u || pair < inner0 || pair >= inner1;
        const int key0[2] = {two & 1 ? key : kNoKey, two & 2 ? key + kCellTokens : kNoKey};
        uint32_t keep[2] = {0xffffffffu, 0xffffffffu};     // of the scales of the lane's four values
        if (edge) {                  // what no row sees may be anything: NaN times 0 too
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (key0[u] + 4 * t + j >= end || key0[u] + 4 * t + j < least_lo) keep[u] &= ~(0xffu << (8 * j));
        }
        uint32_t bp[2][NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if constexpr (CAP) {                          // (scores in log2 units from here on)
            const float in[2] = {fminf(mul[nt][0] * cap_in, 3.0e38f), fminf(mul[nt][1] * cap_in, 3.0e38f)};
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                sc[u][nt][e] = p.softcap2 > kWideCap ? fp4_wide_capped(sc[u][nt][e], in[e & 1], p.softcap2) : fp4_capped(sc[u][nt][e], in[e & 1], p.softcap2);
          }
          const float m0 = CAP ? 1.f : mul[nt][0], m1 = CAP ? 1.f : mul[nt][1];
          // exponents; the reference is raised when one passes it by 8 (p stays below 2^8 2^kUp), and at the first visible key (off is infinite)
          float x[2][4], over = -INFINITY;
          const auto exponents = [&] {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int e = 0; e < 4; ++e) x[u][e] = fmaf(sc[u][nt][e], e & 1 ? m1 : m0, off[nt][e & 1]);
            if (edge) {
#pragma unroll
              for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const int at = key0[u] + k0 + (e & 2);
                  if (at > hi[nt][e & 1] || at < lo[nt][e & 1]) x[u][e] = -INFINITY;
                }
            }
          };
          exponents();
#pragma unroll
          for (int u = 0; u < 2; ++u) over = fmaxf(over, fmaxf(fmaxf(x[u][0], x[u][1]), fmaxf(x[u][2], x[u][3])));
          if (__any_sync(0xffffffffu, over > 8.f + kUp)) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float top = -INFINITY;
#pragma unroll
              for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = e; i < 4; i += 2)
                  if (x[u][i] != -INFINITY) top = fmaxf(top, sc[u][nt][i] * (e ? m1 : m0));
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
              const float now = kUp - top;                                       // (+infinity where nothing is visible yet)
              if (now < off[nt][e]) {
                const float alpha = off[nt][e] == INFINITY ? 0.f : ex2_of(now - off[nt][e]);
                off[nt][e] = now;
                l[nt][e] *= alpha;
#pragma unroll
                for (int i = 0; i < kMT; ++i) {
                  o[nt][i][e] *= alpha;
                  o[nt][i][e + 2] *= alpha;
                }
              }
            }
            exponents();
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              x[u][e] = ex2_of(x[u][e]);
              l[nt][e & 1] += x[u][e];
            }
            bp[u][nt][0] = transposed(pack_f16x2(x[u][0], x[u][1]));
            bp[u][nt][1] = transposed(pack_f16x2(x[u][2], x[u][3]));
          }
        }
        // Where rows differ in what they see, a NaN among the values is not left to the product: 0 times it would reach the rows that do not see it.
        // A product of its own says which rows do, their outputs become NaN, and its scale in the ring zero. (48 sequences of 2 to 6 drafts: 76 us
        // without, 78 with it. A call of decode has no such rows, and kernels without this: 256 sequences 143 us from a flushed L2, 147 with it.)
        if (SEVERAL && edge && tok0 != tok1) {
          constexpr int kWords = D > 128 ? D / 128 : 1;      // groups of a lane's dims
          const auto word_at = [&](int u, int w) {
            return reinterpret_cast<uint32_t*>(ring + (2 * st + u) * Cell::kBytes + Cell::kValueScales + (g * (D / 8) / 16 + w) * kCellTokens + 4 * t);
          };
          uint32_t odd = 0;
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int w = 0; w < kWords; ++w) odd |= nan_scales(*word_at(u, w) & keep[u]);
          if (__any_sync(0xffffffffu, odd != 0)) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              uint32_t sees[NT][2];
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                float f[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const int at = key0[u] + k0 + (e & 2);
                  f[e] = at <= hi[nt][e & 1] && at >= lo[nt][e & 1] ? 1.f : 0.f;
                }
                sees[nt][0] = transposed(pack_f16x2(f[0], f[1]));
                sees[nt][1] = transposed(pack_f16x2(f[2], f[3]));
              }
#pragma unroll
              for (int w = 0; w < kWords; ++w) {
                const uint32_t scales = *word_at(u, w), bad = nan_scales(scales & keep[u]) >> 7;          // 1 a byte
                const uint32_t n01 = __byte_perm(bad, 0, 0x4140) * 0x3c00u, n23 = __byte_perm(bad, 0, 0x4342) * 0x3c00u;
                const uint32_t a[4] = {n01, n01, n23, n23};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                  float n[4];
                  mma_f16_first(n, a, sees[nt][0], sees[nt][1]);
#pragma unroll
                  for (int i = w * (kMT / kWords); i < (w + 1) * (kMT / kWords); ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                      if (n[e & 1] > 0.f) o[nt][i][e] = __int_as_float(0x7fffffff);
                }
                __syncwarp();
                *word_at(u, w) = scales & ~(bad * 255u);
              }
            }
            fence_proxy_async_smem();                        // (the next copies into the ring follow)
            __syncwarp();
          }
        }
        // O^T: lane (g, t) has keys 4t..4t+3 and dims [g D / 8, + D / 8); the m-tile i is its dims 2i (row g) and 2i + 1 (row g + 8)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t vw[4][kVW];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint8_t* at = cells[u] + Cell::kValues + (((4 * t + j) * Cell::kRow + g * (D / 16)) ^ (32 * t));
            if constexpr (D == 64) {
              vw[j][0] = *reinterpret_cast<const uint32_t*>(at);
            } else if constexpr (D == 128) {
              const uint2 x = *reinterpret_cast<const uint2*>(at);
              vw[j][0] = x.x; vw[j][1] = x.y;
            } else {
              const uint4 x = *reinterpret_cast<const uint4*>(at);
              vw[j][0] = x.x; vw[j][1] = x.y; vw[j][2] = x.z; vw[j][3] = x.w;
            }
          }
#pragma unroll
          for (int i = 0; i < kVW; ++i) {
            const int group = (g * (D / 8) + 8 * i) / 16;
            const uint32_t scales = *reinterpret_cast<const uint32_t*>(cells[u] + Cell::kValueScales + group * kCellTokens + 4 * t) & keep[u];
            const uint32_t s01 = scales_f16x2(scales, 0, 1), s23 = scales_f16x2(scales, 2, 3);
            uint32_t e01[4], d01[4], e23[4], d23[4];             // even dims, odd dims of key pairs
            e2m1x8_f16(low_nibbles_else(vw[0][i], vw[1][i] << 4), e01);
            e2m1x8_f16(low_nibbles_else(vw[0][i] >> 4, vw[1][i]), d01);
            e2m1x8_f16(low_nibbles_else(vw[2][i], vw[3][i] << 4), e23);
            e2m1x8_f16(low_nibbles_else(vw[2][i] >> 4, vw[3][i]), d23);
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const uint32_t a[4] = {mul_f16x2(e01[y], s01), mul_f16x2(d01[y], s01), mul_f16x2(e23[y], s23), mul_f16x2(d23[y], s23)};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma_f16(o[nt][4 * i + y], a, bp[u][nt][0], bp[u][nt][1]);
            }
          }
        }
      }
      __syncwarp();
      cells_at[0] = cells_at[1];
      fetch(st);
      st ^= 1;
      parity ^= st ^ 1;
    }
    // ---- the warps' parts of the piece together; the next piece's queries are on their way meanwhile
    const bool whole = w.whole();
    float* part = parts + fp4_part<Seq, D>(blockIdx.x, w.part());
    const int token0 = s.token0;
    {
      Fp4Piece<Seq> x = w;
      x.next(p, line);
      query(x);
      __syncwarp();
      if (lane == 0) w = x;
      __syncwarp();
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], d);
    constexpr int kMC = Shape::kMergeTiles, kMR = Shape::kMergeRow;
#pragma unroll
    for (int i0 = 0; i0 < kMT; i0 += kMC) {
      // all have read what was there before (they say so, and go on): barrier 1
      if (!first_piece || i0) asm volatile("bar.sync 1, %0;" ::"n"(2 * kThreads) : "memory");
      if (i0 == 0 && g == 0) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) top[warp * kRows + nt * 8 + 2 * t + e] = make_float2(kUp - off[nt][e], l[nt][e]);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (nt * 8 + 2 * t + e < nrows) {
#pragma unroll
            for (int i = 0; i < kMC; ++i)
              *reinterpret_cast<float2*>(merge + (warp * kRows + nt * 8 + 2 * t + e) * kMR + (i * 8 + g) * 2) =
                  make_float2(o[nt][i0 + i][e], o[nt][i0 + i][e + 2]);
          }
      __syncthreads();
      for (int x = threadIdx.x; x < nrows * kMC * 8; x += kThreads) {
        const int i = x % kMC, gg = x / kMC % 8, r = x / (kMC * 8), d = gg * (D / 8) + 2 * (i0 + i);
        float a = 0.f, b = 0.f, mx = -INFINITY, sum = 0.f;
#pragma unroll
        for (int y = 0; y < kRowWarps; ++y) mx = fmaxf(mx, top[y * kRows + r].x);
#pragma unroll
        for (int y = 0; y < kRowWarps; ++y) {
          const float2 ml = top[y * kRows + r], v = *reinterpret_cast<const float2*>(merge + (y * kRows + r) * kMR + (i * 8 + gg) * 2);
          const float f = ml.x == -INFINITY ? 0.f : ex2_of(ml.x - mx);
          a = fmaf(v.x, f, a);
          b = fmaf(v.y, f, b);
          sum = fmaf(ml.y, f, sum);
        }
        if (whole) {
          const int token = p.by_group.of(r0 + r), head = r0 + r - token * p.G;
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          *reinterpret_cast<uint32_t*>(p.out + (long long)(token0 + token) * p.ldo + (long long)(h * p.G + head) * D + d) =
              pack_bf16x2(a * inv, b * inv);
        } else {
          *reinterpret_cast<float2*>(part + r * D + d) = make_float2(a, b);
          if (d == 0) *reinterpret_cast<float2*>(part + kRows * D + 2 * r) = make_float2(mx, sum);
        }
      }
      asm volatile("bar.arrive 1, %0;" ::"n"(2 * kThreads) : "memory");
    }
    first_piece = false;
  }
  if (!first_piece) asm volatile("bar.sync 1, %0;" ::"n"(2 * kThreads) : "memory");      // (nobody leaves while others' arrivals are pending)
  // a wait ran out: what is still on its way to the ring gets the same time again before the CTA gives its memory up
  if (!ok)
    for (int i = 0; i < issued; ++i, st ^= 1, parity ^= st ^ 1) mbar_wait(&full[st], parity, p.status);
}

// Parts of the row kernel's items, each by kRowShares blocks, then those of the tile kernel's: kTileShares shares each, of which a block takes kTurns
// one after another, of items that lie far apart. (One block a share was four waves of blocks, most of them with nothing to do.)
static constexpr int kRowShares = 2, kTileShares = 32, kTurns = 4;
template <int D, int ROWS>
__global__ void __launch_bounds__(kJoinThreads) fp4_join_kernel(Fp4Attn p, float* row_parts, int row_grid, float* tile_parts, int tile_grid) {
  pdl_wait();
  pdl_launch_dependents();
  if ((int)blockIdx.x < row_grid * kRowShares) {
    fp4_join<Fp4Seq<ROWS>, D>(p, row_parts, row_grid, blockIdx.x / kRowShares, blockIdx.x % kRowShares, kRowShares);
  } else if constexpr (D <= 128) {
    const int n = tile_grid * (kTileShares / kTurns);
    uint32_t turns = 0;
#pragma unroll
    for (int k = 0; k < kTurns; ++k)
      if (fp4_cut<Fp4Tile, D>(tile_parts, tile_grid, (blockIdx.x - row_grid * kRowShares + k * n) / kTileShares)->rows > 0) turns |= 1u << k;
#pragma unroll 1
    for (; turns; turns &= turns - 1) {
      const int i = blockIdx.x - row_grid * kRowShares + (__ffs(turns) - 1) * n;
      fp4_join<Fp4Tile, D>(p, tile_parts, tile_grid, i / kTileShares, i % kTileShares, kTileShares);
    }
  }
}

static constexpr int kMostReqs = 8192, kMostTiles = 8000;         // (the line of a step is in shared memory)

template <int D, int NT, bool SEVERAL, bool CAP>
static int launch_rows(const Fp4Attn& p, int grid, float* parts, cudaStream_t stream) {
  using Shape = Fp4RowsShape<D, NT>;
  static Fp4Once once;
  if (!once.run([] {
        return cudaFuncSetAttribute(fp4_rows_kernel<D, NT, SEVERAL, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kFixed + (kMostReqs + 1) * 4) == cudaSuccess;
      }))
    return -2;
  return launch_pdl(fp4_rows_kernel<D, NT, SEVERAL, CAP>, dim3(grid), dim3(Shape::kWarps * 32), Shape::kFixed + (size_t)(p.num_reqs + 1) * 4, stream, p, parts) ==
                 cudaSuccess ? 0 : -2;
}

template <int D, int NT>
static int launch_attn(const Fp4Attn& p, bool rows, bool tiles, float* parts, cudaStream_t stream) {
  using Shape = Fp4RowsShape<D, NT>;
  using Seq = Fp4Seq<Shape::kRows>;
  const int row_grid = rows ? b200_num_sms() * (NT == 1 && D <= 128 ? 2 : 1) : 0, tile_grid = tiles ? fp4_tile_grid() : 0;
  float* tile_parts = parts + fp4_scratch<Seq, D>(row_grid);
  if (rows) {
    const auto form = p.q_start ? (p.softcap2 > 0.f ? launch_rows<D, NT, true, true> : launch_rows<D, NT, true, false>)
                                : (p.softcap2 > 0.f ? launch_rows<D, NT, false, true> : launch_rows<D, NT, false, false>);
    if (const int rc = form(p, row_grid, parts, stream)) return rc;
  }
  if (tiles)
    if (const int rc = launch_fp4_tiles(p, D, tile_parts, stream)) return rc;
  return launch_pdl(fp4_join_kernel<D, Shape::kRows>, dim3(row_grid * kRowShares + tile_grid * (kTileShares / kTurns)), dim3(kJoinThreads), 0, stream, p, parts, row_grid,
                    tile_parts, tile_grid) == cudaSuccess ? 0 : -2;
}

}  // namespace b200

using namespace b200;

// Floats of scratch that b200_fp4_attn needs (B200Fp4Attn.parts).
extern "C" long long b200_fp4_attn_scratch(int D, int prefill) {
  const auto floats = [&](auto d) {
    constexpr int kD = decltype(d)::value;
    const uint32_t sms = b200_num_sms();
    const size_t one = fp4_scratch<Fp4Seq<8>, kD>(2 * sms), two = fp4_scratch<Fp4Seq<16>, kD>(sms);
    return (long long)((one > two ? one : two) + (prefill && kD <= 128 ? fp4_scratch<Fp4Tile, kD>(fp4_tile_grid()) : 0));
  };
  return D == 64 ? floats(std::integral_constant<int, 64>()) : D == 128 ? floats(std::integral_constant<int, 128>())
                                                                        : floats(std::integral_constant<int, 256>());
}

namespace b200 {

// What a call comes to: its kernels, rows of a row tile; rc: refused (-1: no such call, -4: more than is counted in 31 bits).
struct Fp4Plan {
  int rc, few, row_tile;
  bool rows, tiles;
};
static Fp4Plan fp4_plan(const B200Fp4Attn& a) {
  Fp4Plan x = {-1, 0x7fffffff, 8, true, false};
  if ((a.D != 64 && a.D != 128 && a.D != 256) || a.Hkv <= 0 || a.Hq <= 0 || a.Hq % a.Hkv || a.block_size <= 0 || a.block_size % kCellTokens ||
      a.max_blocks <= 0 || a.num_reqs <= 0 || a.total_q <= 0)
    return x;
  x.rc = -4;
  if (a.num_reqs > kMostReqs || (a.q_start && a.num_tiles > kMostTiles)) return x;
  const int G = a.Hq / a.Hkv, cells = a.block_size / kCellTokens;
  const double keys = (double)a.max_blocks * a.block_size, q_rows = (double)a.total_q * G;
  if (keys > 2147479552.0) return x;          // (positions and a tile behind them in 31 bits)
  if (q_rows * G >= 4294967296.0 || (double)a.max_blocks * cells * cells >= 4294967296.0) return x;       // (Fp4Div)
  // Which sequences go to which kernel. Both are launched where the lengths, which only the device knows, may call for both. 24 sequences of 32 heads
  // over 8 of 128 dims, in the row kernel / the tile kernel: 32 rows (8 tokens) behind 4000 keys 94 / 135 us, behind none 28 / 32; 64 rows 167 / 136
  // and 45 / 32; 48 rows lie between.
  static constexpr int kFew = 48;
  const double most_rows = (double)(a.most_q > 0 && a.most_q < a.total_q ? a.most_q : a.total_q) * G;
  x.tiles = a.D <= 128 && a.q_start && a.num_tiles > 0 && most_rows > kFew;
  x.rows = !x.tiles || a.num_reqs > 1;
  if (x.tiles) x.few = x.rows ? kFew : -1;
  // Row tiles of 16 where the sequences have more than 8 rows on average. 48 sequences of 2000 keys, 8 kv heads of 128 dims, in tiles of 8 / of 16: 8 rows
  // 47 / 61 us, 16 rows 71 / 64, 24 rows 95 / 104, 32 rows 120 / 107. (A tile of 16 costs as much as two of 8 do, but for the products by scales and the
  // fetches; one CTA an SM instead of two. At 256 dims its accumulators do not fit.)
  if (a.D <= 128 && q_rows > 8.0 * a.num_reqs) x.row_tile = 16;
  // The longest line of each kernel in 31 bits, for bounds of sequences that ascend: each sequence has one row tile that is not full. (Bounds that go back
  // can make it longer: fp4_line. An item's cells times an entry's items stay in 31 bits even then.)
  const auto up = [](double n, int d) { return (double)(((long long)n + d - 1) / d); };
  if (x.rows) {
    const double seqs = a.num_reqs < a.total_q ? a.num_reqs : a.total_q;
    double items = q_rows / x.row_tile + seqs;
    if (x.tiles) items = min(items, seqs * up(kFew, x.row_tile));
    if ((up(keys, kPairKeys) + Fp4Seq<16>::kStart) * a.Hkv * items > 2147483647.0) return x;
  }
  if (x.tiles) {
    const double items = a.num_tiles * up((double)(a.total_q < kTileTokens ? a.total_q : kTileTokens) * G, Fp4Tile::kRows);
    if ((up(keys, kTileKeys) + Fp4Tile::kStart) * a.Hkv * items > 2147483647.0) return x;
  }
  x.rc = 0;
  return x;
}

}  // namespace b200

// 0 where b200_fp4_attn takes a step of these sizes (pointers are not looked at, but whether there is a q_start); otherwise what it would return.
extern "C" int b200_fp4_attn_takes(const B200Fp4Attn* a) { return a->num_reqs <= 0 || a->total_q <= 0 ? 0 : fp4_plan(*a).rc; }

extern "C" int b200_fp4_attn(const B200Fp4Attn* a, cudaStream_t stream) {
  if (a->num_reqs <= 0 || a->total_q <= 0) return 0;
  if (a->num_blocks <= 0 || !(a->scale > 0.f)) return -1;
  const uintptr_t bits = (uintptr_t)a->q | (uintptr_t)a->out | (uintptr_t)a->cache | (uintptr_t)a->parts | (uintptr_t)((a->ldq | a->ldo) * 2);
  if ((bits & 15) || !a->q || !a->out || !a->cache || !a->block_table || !a->seq_lens || !a->parts || (a->q_start && (!a->tile_req || !a->tile_q0)))
    return -1;
  const Fp4Plan x = fp4_plan(*a);
  if (x.rc) return x.rc;
  const int G = a->Hq / a->Hkv;
  Fp4Attn p;
  p.q = (const __nv_bfloat16*)a->q; p.ldq = a->ldq;
  p.out = (__nv_bfloat16*)a->out; p.ldo = a->ldo;
  p.cache = (const uint8_t*)a->cache; p.num_blocks = a->num_blocks;
  p.block_table = (const int32_t*)a->block_table; p.max_blocks = a->max_blocks; p.ldt = a->ldt;
  p.seq_lens = (const int32_t*)a->seq_lens; p.q_start = (const int32_t*)a->q_start;
  p.tile_req = (const int32_t*)a->tile_req; p.tile_q0 = (const int32_t*)a->tile_q0;
  p.num_reqs = a->num_reqs; p.total_q = a->total_q; p.num_tiles = a->q_start ? a->num_tiles : 0;
  p.Hkv = a->Hkv; p.G = G; p.cells_per_page = a->block_size / kCellTokens;
  p.window = max(-(1 << 30), min(a->window, 1 << 30)); p.causal = a->causal;
  p.few = x.few;
  const auto by = [](int d) { return Fp4Div{d == 1 ? 0u : (uint32_t)(((1ull << 32) + d - 1) / d)}; };
  p.by_group = by(G);
  p.by_page_cells = by(p.cells_per_page);
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.softcap2 = fminf(a->softcap * 1.4426950408889634f, 3.0e38f);
  p.status = device_status_word();
  float* parts = (float*)a->parts;
  const bool two = x.row_tile == 16;
  if (a->D == 64) return two ? launch_attn<64, 2>(p, x.rows, x.tiles, parts, stream) : launch_attn<64, 1>(p, x.rows, x.tiles, parts, stream);
  if (a->D == 128) return two ? launch_attn<128, 2>(p, x.rows, x.tiles, parts, stream) : launch_attn<128, 1>(p, x.rows, x.tiles, parts, stream);
  return launch_attn<256, 1>(p, x.rows, x.tiles, parts, stream);
}
