// Trees of drafted tokens around the attention over them: ancestors' bits and positions before a step, the accepted path's cells after it.
#include "api.h"
#include "sm100.cuh"

namespace b200 {

static constexpr int kCellNodes = 1024;        // of a request

// Row i of a request's n nodes: the bits of i and of the nodes above it, and its position, what lies before the request's nodes plus its depth. A
// thread walks from its node to the root, through shared memory; parents lie below their children, so that a word is whole before the next
// is begun. (An entry that is not below its own node makes it a root: the walk ends whatever the entries are.)
// Bound: the launch and two loads in a chain (bounds, parents). One tree of 60 nodes 2.4 us, 256 trees of 9 to 101 nodes 2.9.
__global__ void __launch_bounds__(128)
    tree_mask_kernel(const int32_t* __restrict__ parents, const int32_t* __restrict__ q_start, const int32_t* __restrict__ seq_lens, int total,
                     int words, uint64_t* __restrict__ bits, int64_t* __restrict__ positions) {
  __shared__ int parent[kCellNodes];
  pdl_wait();
  pdl_launch_dependents();
  const int req = blockIdx.x, row0 = min(max(q_start[req], 0), total), rows = max(0, min(q_start[req + 1], total) - row0);
  const int n = min(rows, kCellNodes);
  const long long context = (long long)seq_lens[req] - rows;
  for (int i = threadIdx.x; i < n; i += blockDim.x) parent[i] = parents[row0 + i];
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    uint64_t* row = bits + (long long)(row0 + i) * words;
    int at = i, word = words - 1, depth = -1;
    uint64_t held = 0;
    while (at >= 0) {
      for (; word > at >> 6; --word) {
        row[word] = held;
        held = 0;
      }
      if (word == at >> 6) held |= 1ull << (at & 63);          // (a node past the words has no bit)
      ++depth;
      const int up = parent[at];
      at = up < at ? up : -1;
    }
    for (; word >= 0; --word) {
      row[word] = held;
      held = 0;
    }
    positions[row0 + i] = context + depth;
  }
}

// Cell context + path[i] of a request goes to cell context + i, i = 1, 2 .., in every cache. A thread moves the same 16 bytes of all cells, in that order
// and several at a time: a source lies behind its own destination and all earlier ones, so that nothing is overwritten that is still to be
// read. A block takes one request's keys or values in one cache. Bound: the chain of bounds, path, table and cells for few paths (one of three drafts in 32 caches 3.0 us,
// 0.16 by its bytes), bytes of scattered cells of 2 KB for many (64 of up to seven drafts in 16 caches 7.7 us, 3.3 TB/s).
static constexpr int kCaches = 64;             // of a launch
struct CompactCaches { uint8_t* at[kCaches]; };
__global__ void __launch_bounds__(256)
    tree_compact_kernel(const __grid_constant__ CompactCaches caches, const int32_t* __restrict__ block_table, long long ldt, int max_blocks,
                        const int32_t* __restrict__ seq_lens, const int32_t* __restrict__ q_start, int total, const int32_t* __restrict__ path,
                        int most, long long num_blocks, int block_size, int cell_vecs) {
  __shared__ long long from[kCellNodes], to[kCellNodes];
  __shared__ int moves;
  pdl_wait();
  pdl_launch_dependents();
  const int req = blockIdx.x;
  const int row0 = min(max(q_start[req], 0), total), rows = max(0, min(q_start[req + 1], total) - row0), n = min(rows, kCellNodes);
  const long long context = (long long)min(max(seq_lens[req], 0), (int)min((long long)max_blocks * block_size, (1ll << 31) - 1)) - rows;
  const int32_t* bt = block_table + req * ldt;
  const auto cell = [&](long long position) {
    const int blk = bt[position / block_size];
    return blk < 0 || blk >= num_blocks ? -1 : ((long long)blk * 2 * block_size + position % block_size) * cell_vecs;
  };
  if (threadIdx.x < 32) {              // the moves, in order
    int found = 0;
    for (int i0 = 1; i0 < min(most, n); i0 += 32) {
      const int i = i0 + threadIdx.x, node = i < min(most, n) ? path[(long long)req * most + i] : -1;
      long long a = -1, b = -1;
      if (node > i && node < n && context + i >= 0) {
        a = cell(context + node);
        b = cell(context + i);
      }
      const bool is = a >= 0 && b >= 0;
      const uint32_t who = __ballot_sync(0xffffffffu, is);
      const int at = found + __popc(who & ((1u << threadIdx.x) - 1));
      if (is) {
        from[at] = a;
        to[at] = b;
      }
      found += __popc(who);
    }
    if (threadIdx.x == 0) moves = found;
  }
  __syncthreads();
  const int count = moves;
  uint4* base = reinterpret_cast<uint4*>(caches.at[blockIdx.y >> 1]) + (long long)(blockIdx.y & 1) * block_size * cell_vecs;
  for (int v = threadIdx.x; v < cell_vecs; v += blockDim.x) {
    uint4* mine = base + v;
    int i = 0;
    for (; i + 4 <= count; i += 4) {
      const uint4 x0 = mine[from[i]], x1 = mine[from[i + 1]], x2 = mine[from[i + 2]], x3 = mine[from[i + 3]];
      mine[to[i]] = x0;
      mine[to[i + 1]] = x1;
      mine[to[i + 2]] = x2;
      mine[to[i + 3]] = x3;
    }
    for (; i < count; ++i) mine[to[i]] = mine[from[i]];
  }
}

}  // namespace b200

using namespace b200;

extern "C" int b200_tree_mask(const void* parents, const void* q_start, const void* seq_lens, int num_reqs, int total, int words, void* bits,
                              void* positions, cudaStream_t stream) {
  if (num_reqs <= 0 || total <= 0) return 0;
  if (words <= 0) return -1;
  if (words > kCellNodes / 64) return -4;
  return launch_pdl(tree_mask_kernel, dim3(num_reqs), dim3(128), 0, stream, (const int32_t*)parents, (const int32_t*)q_start,
                    (const int32_t*)seq_lens, total, words, (uint64_t*)bits, (int64_t*)positions) == cudaSuccess ? 0 : -2;
}

extern "C" int b200_tree_compact(const B200TreeCompact* a, cudaStream_t stream) {
  if (a->num_reqs <= 0 || a->num_caches <= 0 || a->most <= 1 || a->total <= 0) return 0;
  if (a->block_size <= 0 || a->max_blocks <= 0 || a->cell_bytes <= 0 || a->cell_bytes % 16) return -1;
  for (int at = 0; at < a->num_caches; at += kCaches) {
    const int n = a->num_caches - at < kCaches ? a->num_caches - at : kCaches;
    CompactCaches c = {};
    for (int i = 0; i < n; ++i) c.at[i] = (uint8_t*)a->caches[at + i];
    if (launch_pdl(tree_compact_kernel, dim3(a->num_reqs, 2 * n), dim3(256), 0, stream, c, (const int32_t*)a->block_table, a->ldt, a->max_blocks,
                   (const int32_t*)a->seq_lens, (const int32_t*)a->q_start, a->total, (const int32_t*)a->path, a->most, a->num_blocks,
                   a->block_size, (int)(a->cell_bytes / 16)) != cudaSuccess)
      return -2;
  }
  return 0;
}
