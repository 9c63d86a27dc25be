// Verification of drafted tokens against the target's distributions, by given random numbers: chains and trees.
//
// From the root down: at a node with logits l, w_j = e^(l_j - max l), the children x_1, x_2 .. are asked in their order. Drawn from q (the drafter's
// distribution at the node), with b = 0 and Z = sum w at first: x is accepted if u q(x) Z < max(w_x - b q(x), 0); refused, b becomes b + Z and Z
// becomes sum max(w - b q, 0). That is the refusal's residual norm(max(p - q, 0)), one refusal after another, in closed form: each costs one sum over
// the row and no division. Chosen instead (no q): x is accepted if u Z < w_x, and a refused one leaves w; the sums are built up from the tokens that are
// no children's, so that none is a difference. After an accepted child the walk goes on there; where none is accepted the last token is the
// exponential race over what is left of w, with the same numbers as the sampler's draw. Greedy requests accept the argmax.
//
// A cluster of CTAs has a request, each a slice of the columns. A stage brings the rows of `ahead` nodes at once, of the node that the walk is at and of the
// first children below it, by bulk copies into shared memory, takes their largest logits and sums, and walks as far as it gets with them; what is
// left of a refused node's row is drawn from there. One after another the rows would each cost a chain of a load, reductions and a cluster
// barrier. Bound: that chain where there are few requests, the rows' bytes and the draw's random numbers (some 60 instructions a column) where there are
// many (there a stage reads one row: none in vain). Measured: a chain of four drafts, 128256 columns, drawn 17.8 us (0.8 by its rows' bytes; the first row's arrival, a stage's 4 us
// and the draw); 64 chains of one to five over 151936 columns 81 us (33 by the rows that are visited; two waves of 33 clusters, issue 0.52, ALU 0.45); 24 trees of
// 31 to 48 nodes over 128256 columns, chosen 39 us, drawn (up to three children a node) 56. Greedy requests, which have no sum and no draw: one chain 9.4 us, 64 chains 37. Slower: rows streamed through registers a node at a time (one chain 24 to 60 us), q in a slot of its own.
#include <algorithm>
#include <type_traits>

#include "api.h"
#include "row_cluster.cuh"

namespace b200 {

static constexpr int kVerifyThreads = 512, kVerifyNodes = 1024, kVerifyAhead = 4;
static constexpr int kVerifySmem = 190 * 1024;       // of slices
static constexpr int kVerifyMostCols = 778000;      // (sixteen slices)

struct VerifyParams {
  const float* logits;
  long long ldl;
  const float* probs;                // null: drafts were chosen
  long long ldp;
  const int64_t* tokens;
  const int32_t *parents, *q_start;  // parents null: chains
  const float *uniforms, *temperature;
  const uint64_t *seeds, *steps;
  int64_t* out;                      // [num_reqs][most]
  int32_t *path, *count;
  int num_reqs, total, V, most;
  int ahead, slot;                   // rows of a stage, each in a slot of so many bytes of shared memory
  int* status;
};

enum VerifyAction : int { kGoOn, kRefused, kDraw };
struct VerifyShared {
  ArgPair arg[32];
  float sums[32];
  float2 warp_top[kVerifyThreads / 32][kVerifyAhead];      // (largest logit, sum) or (largest logit, its column)
  float2 top[kVerifyAhead];
  int node[kVerifyAhead], first[kVerifyAhead + 1];         // nodes of the stage, their children in `child`
  int taken[kVerifyAhead];                                 // the child that each of them goes on to, or -1
  int nodes, action, at, depth, next;
  uint64_t full[kVerifyAhead];
  int parent[kVerifyNodes], token[kVerifyNodes], child[kVerifyNodes];
  float u[kVerifyNodes], w[kVerifyNodes], q[kVerifyNodes]; // random numbers of the nodes; logits, then weights, and q of the stage's children
};
// Pairs of numbers from every CTA to every CTA: each stores its own into all of them, and they wait for what they are to get (its bytes are counted on a barrier of
// theirs), not for one another. Two buffers in turn: who stores into the one of the last exchange but one has got the last one's numbers from all, who had read
// the buffer before they sent them.
template <int CTAS>
struct VerifyExchange {
  float2 got[2][CTAS][kVerifyAhead];
  uint64_t bar[2];
};
// `mine`: lane 0 .. of the calling warp, number k of this CTA.
template <int CTAS>
__device__ __forceinline__ void send(VerifyExchange<CTAS>& ex, int turn, int k, float2 mine, int rank) {
  const int lane = threadIdx.x & 31;
  if constexpr (CTAS == 1) {
    if (lane == 0) ex.got[turn & 1][0][k] = mine;
  } else if (lane < CTAS) {
    const uint32_t to = mapa_u32(smem_u32(&ex.got[turn & 1][rank][k]), lane), bar = mapa_u32(smem_u32(&ex.bar[turn & 1]), lane);
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(to), "f"(mine.x), "f"(mine.y), "r"(bar) : "memory");
  }
}
// Every thread calls it, after the sends of its CTA where that is the whole cluster.
template <int CTAS>
__device__ __forceinline__ void receive(VerifyExchange<CTAS>& ex, int turn, int numbers, int* status) {
  if constexpr (CTAS == 1) {
    __syncthreads();
  } else {
    if (threadIdx.x == 0) mbar_expect_tx(&ex.bar[turn & 1], CTAS * numbers * 8);
    mbar_wait(&ex.bar[turn & 1], turn >> 1 & 1, status);
  }
}

__device__ __forceinline__ float logit_of(float l) { return fmaxf(l, -INFINITY); }          // (a NaN is -inf)
__device__ __forceinline__ float prob_of(float q) { return fmaxf(q, 0.f); }                 // (a NaN is 0)
__device__ __forceinline__ float verify_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Weights e^(l - m) of a row whose largest logit is m: 0 for -inf and NaN, and 1 for m itself, where it is infinite too. l - m comes first, and near m it is exact: a row's
// weights, and the factors that turn a warp's sum into a CTA's and a cluster's, are the same whatever all its logits have in common. (In log2 units l and m would each carry a
// rounding of 2^-24 of themselves: one fused instruction a column less, and sums off by 2e-4 against the weights at logits of 3000, by 6 % at a million.) The difference
// rounds by 2^-24 of itself, which is 2^-20 of a weight that is 2^-16 of the largest.
struct Weights {
  float m;
  bool far;                            // m is infinite: the others of the row have no weight
  __device__ __forceinline__ Weights(float m_) : m(m_), far(!(fabsf(m_) <= FLT_MAX)) {}
  __device__ __forceinline__ float plain(float l) const { return verify_ex2((l - m) * 1.4426950408889634f); }             // not far, not NaN
  __device__ __forceinline__ float of(float l) const { return plain(logit_of(l)); }
  __device__ __forceinline__ float any(float l) const { return !far ? of(l) : l == m && m > 0.f ? 1.f : 0.f; }
};
__device__ __forceinline__ float weight_of(float l, float m) { return Weights(m).any(l); }

// Columns of a row's slice on their way to a slot of shared memory, by one thread: whole pieces of 16 bytes, of which each holds some of the slice, so that up to three
// columns of its neighbours come along on either side. slice_at: where its first column lies.
__device__ __forceinline__ int slice_shift(const float* x) { return (int)(reinterpret_cast<uintptr_t>(x) >> 2 & 3); }
__device__ __forceinline__ float* slice_at(uint8_t* slot, const float* x) { return reinterpret_cast<float*>(slot) + slice_shift(x); }
__device__ __forceinline__ void fetch_slice(uint8_t* slot, const float* x, int n, uint64_t* bar) {
  const uint32_t bytes = (uint32_t)(slice_shift(x) + n + 3) / 4 * 16;
  mbar_expect_tx(bar, bytes);
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(slot)),
               "l"(reinterpret_cast<uintptr_t>(x) & ~uintptr_t(15)), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
// f(float4) for this thread's share of n pieces of 16 bytes.
template <typename F>
__device__ __forceinline__ void for_pieces(const uint8_t* slot, int n, F f) {
  const float4* x = reinterpret_cast<const float4*>(slot);
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += kVerifyThreads) f(x[i]);
}
// f(column) for this thread's share of n columns, side by side in a warp.
template <typename F>
__device__ __forceinline__ void for_columns(int n, F f) {
#pragma unroll 8
  for (int c = threadIdx.x; c < n; c += kVerifyThreads) f(c);
}

template <int CTAS>
__global__ void __launch_bounds__(kVerifyThreads, 2) tree_verify_kernel(VerifyParams p) {
  extern __shared__ uint4 slots_raw[];
  __shared__ VerifyShared sh;
  __shared__ VerifyExchange<CTAS> ex;
  constexpr int T = kVerifyThreads, W = T / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = row_slice_cols(p.V, CTAS), rank = row_rank<CTAS>(), lo = min(p.V, rank * per), cols = min(p.V, lo + per) - lo;
  const int req = blockIdx.x / CTAS;
  const auto slot = [&](int k) { return reinterpret_cast<uint8_t*>(slots_raw) + k * p.slot; };
  if (threadIdx.x == 0) {
    for (int k = 0; k < p.ahead; ++k) mbar_init(&sh.full[k], 1);
    mbar_init(&ex.bar[0], 1);
    mbar_init(&ex.bar[1], 1);
    mbar_fence_init();
  }
  __syncwarp();
  if constexpr (CTAS > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");      // (waited for ahead of the first store into another CTA)
  pdl_wait();
  pdl_launch_dependents();
  const int row0 = min(max(p.q_start[req], 0), p.total), n = min(max(0, min(p.q_start[req + 1], p.total) - row0), kVerifyNodes);
  const auto logits_of = [&](int node) { return p.logits + (row0 + node) * p.ldl + lo; };
  const auto probs_of = [&](int node) { return p.probs + (row0 + node) * p.ldp + lo; };
  if (threadIdx.x == 0 && n > 0) fetch_slice(slot(0), logits_of(0), cols, &sh.full[0]);
  const bool greedy = p.temperature && p.temperature[req] < kEps, drawn = p.probs != nullptr && !greedy;
  for (int i = threadIdx.x; i < n; i += T) {
    sh.parent[i] = p.parents ? p.parents[row0 + i] : i - 1;
    const int64_t t = p.tokens[row0 + i];
    sh.token[i] = t >= 0 && t < p.V ? (int)t : -1;
    sh.u[i] = p.uniforms[row0 + i];
  }
  int64_t* out = p.out + (long long)req * p.most;
  int32_t* path = p.path + (long long)req * p.most;
  if (rank == 0)
    for (int i = threadIdx.x; i < p.most; i += T) {
      out[i] = -1;
      path[i] = i == 0 && n > 0 ? 0 : -1;
    }
  __syncthreads();
  if (n == 0) {
    if (rank == 0 && threadIdx.x == 0) p.count[req] = 0;
    if constexpr (CTAS > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    return;
  }
  int node = 0, depth = 0, turn = 0;
  uint32_t phase = 0;                  // a bit for each slot
  // (a wait that runs out leaves its mark in the status word; the walk goes on, as others wait for it in the cluster's barriers)
  const auto arrived = [&](int k) {
    mbar_wait(&sh.full[k], phase >> k & 1, p.status);
    phase ^= 1u << k;
  };
  for (int stage = 0;; ++stage) {
    // ---- the nodes of the stage and their children, in order; their rows
    if (warp == 0) {
      int count = 0, found = 0, at = node;
      if (!p.parents) {                // (a chain's node has one child, but for its last, or the last that counts)
        count = min(min(p.ahead, n - node), p.most - depth);
        found = min(count, min(n - node, p.most - depth) - 1);
        if (lane <= count) sh.first[lane] = min(lane, found);
        if (lane < count) sh.node[lane] = node + lane;
        if (lane < found) sh.child[lane] = node + lane + 1;
      } else {
        while (true) {
          if (lane == 0) {
            sh.node[count] = at;
            sh.first[count] = found;
          }
          int below = -1;
          if (depth + count + 1 < p.most)
            for (int base = at + 1; base < n; base += 32) {
              const int j = base + lane;
              const bool is = j < n && sh.parent[j] == at;
              const uint32_t who = __ballot_sync(0xffffffffu, is);
              if (is) sh.child[found + __popc(who & ((1u << lane) - 1))] = j;
              if (below < 0 && who) below = base + __ffs(who) - 1;
              found += __popc(who);
            }
          ++count;
          if (below < 0 || count >= p.ahead) break;
          at = below;
        }
        if (lane == 0) sh.first[count] = found;
      }
      if (lane == 0) sh.nodes = count;
      __syncwarp();
      if (lane < count && (stage > 0 || lane > 0)) fetch_slice(slot(lane), logits_of(sh.node[lane]), cols, &sh.full[lane]);
    }
    __syncthreads();
    const int nodes = sh.nodes, children = sh.first[nodes];
    if (!greedy)
      for (int i = threadIdx.x; i < children; i += T) {
        int k = 0;
        while (i >= sh.first[k + 1]) ++k;
        const int t = sh.token[sh.child[i]];
        sh.w[i] = t < 0 ? -INFINITY : logit_of(__ldg(logits_of(sh.node[k]) - lo + t));
        sh.q[i] = drawn && t >= 0 ? prob_of(__ldg(probs_of(sh.node[k]) - lo + t)) : 0.f;
      }
    if (drawn && p.ahead > 1 && warp == 1) {       // (few requests: what a refusal reads is on its way already)
      for (int k = 0; k < nodes; ++k)
        for (int c = lane * 32; c < cols; c += 1024)
          if (sh.first[k] < sh.first[k + 1]) asm volatile("prefetch.global.L2 [%0];" ::"l"(probs_of(sh.node[k]) + c));
    }
    // chosen drafts stand apart from the row, and what lies beside a slice in its pieces counts for nothing
    const bool beside = ((p.ldl | (int)(reinterpret_cast<uintptr_t>(p.logits) >> 2) | cols) & 3) != 0, chosen = !drawn && children > 0;
    if (!greedy && (beside || chosen)) {
      for (int k = 0; k < nodes; ++k) {
        mbar_wait(&sh.full[k], phase >> k & 1, p.status);
        float* l = slice_at(slot(k), logits_of(sh.node[k]));
        const int shift = slice_shift(logits_of(sh.node[k]));
        if ((int)threadIdx.x < shift) l[-1 - (int)threadIdx.x] = -INFINITY;
        if ((int)threadIdx.x < (-(shift + cols) & 3)) l[cols + threadIdx.x] = -INFINITY;
      }
      if (chosen)
        for (int i = threadIdx.x; i < children; i += T) {
          int k = 0;
          while (i >= sh.first[k + 1]) ++k;
          const int c = sh.token[sh.child[i]] - lo;
          if (c >= 0 && c < cols) slice_at(slot(k), logits_of(sh.node[k]))[c] = -INFINITY;
        }
      __syncthreads();
    }
    // ---- the rows' largest logits, and the sums of the weights or the columns
    for (int k = 0; k < nodes; ++k) {
      const float* l = slice_at(slot(k), logits_of(sh.node[k]));
      arrived(k);
      float2 mine;
      if (greedy) {
        ArgPair best{-FLT_MAX, 0x7fffffff};
        for_columns(cols, [&](int c) {
          if (l[c] >= -FLT_MAX) best = arg_better(best, ArgPair{l[c], lo + c});          // (neither NaN nor -inf)
        });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = arg_better(best, ArgPair{__shfl_xor_sync(~0u, best.v, o), __shfl_xor_sync(~0u, best.i, o)});
        mine = make_float2(best.v, __int_as_float(best.i));
      } else {
        float m = -INFINITY, sum = 0.f;
        const int pieces = (slice_shift(logits_of(sh.node[k])) + cols + 3) / 4;
        for_pieces(slot(k), pieces, [&](float4 v) { m = fmaxf(fmaxf(fmaxf(m, v.x), fmaxf(v.y, v.z)), v.w); });       // (a NaN is passed over)
        m = warp_max_f32(m);
        const Weights w(m);
        float sums[4] = {};
        if (!w.far)
          for_pieces(slot(k), pieces, [&](float4 v) {
            sums[0] += w.plain(v.x), sums[1] += w.plain(v.y), sums[2] += w.plain(v.z), sums[3] += w.plain(v.w);
          });
        sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
        if (w.far || sum != sum) {     // (a NaN among them)
          sum = 0.f;
          for_pieces(slot(k), pieces, [&](float4 v) { sum += (w.any(v.x) + w.any(v.y)) + (w.any(v.z) + w.any(v.w)); });
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
        mine = make_float2(m, sum);
      }
      if (lane == 0) sh.warp_top[warp][k] = mine;
    }
    __syncthreads();
    if constexpr (CTAS > 1)
      if (stage == 0) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (warp < nodes) {                // warp k: node k of the stage
      const float2 x = lane < W ? sh.warp_top[lane][warp] : make_float2(greedy ? -FLT_MAX : -INFINITY, greedy ? __int_as_float(0x7fffffff) : 0.f);
      float2 mine;
      if (greedy) {
        ArgPair a{x.x, __float_as_int(x.y)};
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) a = arg_better(a, ArgPair{__shfl_xor_sync(~0u, a.v, o), __shfl_xor_sync(~0u, a.i, o)});
        mine = make_float2(a.v, __int_as_float(a.i));
      } else {
        mine.x = warp_max_f32(x.x);
        mine.y = x.y * weight_of(x.x, mine.x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mine.y += __shfl_xor_sync(~0u, mine.y, o);
      }
      send<CTAS>(ex, turn, warp, mine, rank);
    }
    receive<CTAS>(ex, turn, nodes, p.status);
    if (warp < nodes) {
      const float2 x = lane < CTAS ? ex.got[turn & 1][lane][warp] : make_float2(greedy ? -FLT_MAX : -INFINITY, greedy ? __int_as_float(0x7fffffff) : 0.f);
      float2 all;
      if (greedy) {
        ArgPair a{x.x, __float_as_int(x.y)};
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) a = arg_better(a, ArgPair{__shfl_xor_sync(~0u, a.v, o), __shfl_xor_sync(~0u, a.i, o)});
        all = make_float2(a.v, __int_as_float(a.i));
      } else {
        all.x = warp_max_f32(x.x);
        if (!drawn)                    // (the chosen drafts are of the row too)
          for (int i = sh.first[warp]; i < sh.first[warp + 1]; ++i) all.x = fmaxf(all.x, sh.w[i]);
        all.y = x.y * weight_of(x.x, all.x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all.y += __shfl_xor_sync(~0u, all.y, o);
      }
      // the child that the walk goes on to from here, if it comes here
      const int begin = sh.first[warp], end = sh.first[warp + 1];
      int taken = -1;
      if (greedy) {
        for (int i = begin; i < end && taken < 0; i += 32) {
          const uint32_t who = __ballot_sync(~0u, i + lane < end && sh.token[sh.child[i + lane]] == __float_as_int(all.y));
          if (who) taken = sh.child[i + __ffs(who) - 1];
        }
      } else if (drawn) {
        // the first child; the others stand against what a refusal leaves
        if (begin < end && sh.u[sh.child[begin]] * sh.q[begin] * all.y < weight_of(sh.w[begin], all.x)) taken = sh.child[begin];
      } else {
        float after = all.y;           // Z at a child: what no child has, and the children from it on
        for (int i0 = begin + ((end - begin - 1) & ~31); i0 >= begin && begin < end; i0 -= 32) {
          const int i = i0 + lane;
          float w = 0.f;
          if (i < end) {
            const int t = sh.token[sh.child[i]];
            bool again = t < 0;        // (of two chosen drafts alike, the second has no weight left)
            for (int e = begin; e < i; ++e) again |= sh.token[sh.child[e]] == t;
            w = again ? 0.f : weight_of(sh.w[i], all.x);
          }
          float z = w;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const float v = __shfl_down_sync(~0u, z, o);
            if (lane + o < 32) z += v;
          }
          z += after;
          const uint32_t who = __ballot_sync(~0u, i < end && sh.u[sh.child[i]] * z < w);
          if (who) taken = sh.child[i0 + __ffs(who) - 1];
          after = __shfl_sync(~0u, z, 0);
        }
      }
      if (lane == 0) {
        sh.top[warp] = all;
        sh.taken[warp] = taken;
      }
    }
    ++turn;
    __syncthreads();
    // ---- as far as it goes
    if (threadIdx.x == 0) {
      int k = 0, action = kGoOn;
      while (true) {
        const int taken = sh.taken[k];
        if (taken < 0) {
          action = drawn && sh.first[k + 1] - sh.first[k] > 1 ? kRefused : kDraw;
          break;
        }
        if (rank == 0) {
          out[depth] = sh.token[taken];
          path[depth + 1] = taken;
        }
        ++depth;
        sh.next = taken;
        if (k + 1 >= nodes || sh.node[k + 1] != taken) break;
        ++k;
      }
      sh.action = action;
      sh.at = k;
      sh.depth = depth;
    }
    __syncthreads();
    const int action = sh.action, k = sh.at, begin = sh.first[k], end = sh.first[k + 1];
    depth = sh.depth;
    if (action == kGoOn) {
      node = sh.next;
      fence_proxy_async_smem();
      __syncthreads();                 // (lists and slices are written anew)
      continue;
    }
    node = sh.node[k];
    const float2 top = sh.top[k];
    const float* l = slice_at(slot(k), logits_of(node));
    const bool refused = drawn && begin < end;
    const float* q = refused ? probs_of(node) : nullptr;
    float b = refused ? top.y : 0.f;
    const Weights weights(top.x);
    const auto left_of = [&](int c, float q) { return fmaxf(fmaf(-b, prob_of(q), weights.any(l[c])), 0.f); };
    // ---- the children after a refused one
    int taken = -1;
    if (action == kRefused) {
      for (int i = begin + 1; i < end && taken < 0; ++i) {
        float part = 0.f;
        for_columns(cols, [&](int c) { part += left_of(c, __ldg(q + c)); });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(~0u, part, o);
        if (lane == 0) sh.sums[warp] = part;
        __syncthreads();
        if (warp == 0) {
          part = lane < W ? sh.sums[lane] : 0.f;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(~0u, part, o);
          send<CTAS>(ex, turn, 0, make_float2(part, 0.f), rank);
        }
        receive<CTAS>(ex, turn, 1, p.status);
        float Z = 0.f;
#pragma unroll
        for (int r = 0; r < CTAS; ++r) Z += ex.got[turn & 1][r][0].x;
        ++turn;
        const int c = sh.child[i];
        if (sh.u[c] * sh.q[i] * Z < fmaxf(fmaf(-b, sh.q[i], weights.any(sh.w[i])), 0.f)) taken = c;
        else b += Z;
      }
    }
    if (taken >= 0) {
      if (rank == 0 && threadIdx.x == 0) {
        out[depth] = sh.token[taken];
        path[depth + 1] = taken;
      }
      node = taken;
      ++depth;
      fence_proxy_async_smem();
      __syncthreads();
      continue;
    }
    // ---- the last token
    int64_t last = __float_as_int(top.y);
    if (!greedy) {
      const uint64_t seed = p.seeds[req], step = p.steps[req];
      ArgPair a{0.f, 0x7fffffff};
      // The race's exponential is -log(1 - v), more than v: what cannot win by the first bits of v is passed over. What may win is weighed in 32 bits, and
      // in the race's own 64 where that does not tell: two candidates of a thread within kSame, and at the end what is within it of the block's best.
      constexpr int kE = 8;
      constexpr float kSame = 1e-5f;
      float least = 0.f, best = 0.f, best_left = 0.f;        // a little below the warp's best time; this thread's best
      int best_c = -1;
      const uint64_t base = step * 0x100000001B3ull + (uint64_t)lo;
      float next[kE];                  // q of the next columns, on its way
      const auto fetch = [&](int c) {
#pragma unroll
        for (int e = 0; e < kE; ++e) next[e] = refused && c + e * T < cols ? __ldg(q + c + e * T) : 0.f;
      };
      const auto group = [&](int c0, auto whole) {           // kE columns of each lane, T apart
        float left[kE], high = 0.f;
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          const int c = c0 + lane + e * T;
          left[e] = 0.f;
          if (whole || c < cols) left[e] = left_of(c, next[e]);
          high = fmaxf(high, left[e]);
        }
        fetch(c0 + lane + kE * T);
        if (!__any_sync(~0u, high > 0.f)) return;
        float rest[kE];                // the first bits of v, and one
#pragma unroll
        for (int e = 0; e < kE; ++e) rest[e] = race_rest(seed, base + (uint64_t)(c0 + lane + e * T));
        if (least == 0.f) {            // (the exponential is less than v / (1 - v))
          high = 0.f;
#pragma unroll
          for (int e = 0; e < kE; ++e) high = fmaxf(high, __fdividef(left[e] * (2.f - kRaceRest - rest[e]), rest[e] - 1.f + kRaceRest));
          least = warp_max_f32(high) * (1.f - 2.f * kSame);
        }
        bool may = false;
#pragma unroll
        for (int e = 0; e < kE; ++e) may |= left[e] >= fmaf(least, rest[e], -least);
        if (!__any_sync(~0u, may)) return;
        uint32_t which = 0;            // (a few of a warp's 256)
#pragma unroll
        for (int e = 0; e < kE; ++e)
          if (left[e] > 0.f && left[e] >= fmaf(least, rest[e], -least)) which |= 1u << e;
        while (which) {
          const int e = __ffs(which) - 1, c = lo + c0 + lane + e * T;
          which &= which - 1;
          float x = left[0];
#pragma unroll
          for (int i = 1; i < kE; ++i) x = i == e ? left[i] : x;
          const float time = __fdividef(x, race_time(seed, step, c));
          bool better = time > best;
          if (fabsf(time - best) <= kSame * best) {
            const ArgPair old{race_key(best_left, seed, step, best_c), best_c}, now{race_key(x, seed, step, c), c};
            better = arg_better(old, now).i == c;
          }
          if (better) {
            best = time;
            best_left = x;
            best_c = c;
          }
        }
        least = fmaxf(least, warp_max_f32(best) * (1.f - 2.f * kSame));
      };
      int c0 = warp * 32;
      fetch(c0 + lane);
      for (; c0 + 32 + (kE - 1) * T <= cols; c0 += kE * T) group(c0, std::true_type());
      if (c0 < cols) group(c0, std::false_type());
      {
        float top_time = warp_max_f32(best);
        if (lane == 0) sh.sums[warp] = top_time;
        __syncthreads();
        top_time = warp_max_f32(lane < W ? sh.sums[lane] : 0.f);
        if (best > 0.f && best >= top_time * (1.f - kSame)) a = ArgPair{race_key(best_left, seed, step, best_c), best_c};
      }
      // the best of the cluster, which is 0 where nothing is left
      const auto best_of = [&](ArgPair a, float nothing) {
        a = block_argmax(a, sh.arg);
        if (warp == 0) send<CTAS>(ex, turn, 0, make_float2(a.v, __int_as_float(a.i)), rank);
        receive<CTAS>(ex, turn, 1, p.status);
        a = ArgPair{nothing, 0x7fffffff};
#pragma unroll
        for (int r = 0; r < CTAS; ++r) a = arg_better(a, ArgPair{ex.got[turn & 1][r][0].x, __float_as_int(ex.got[turn & 1][r][0].y)});
        ++turn;
        return a;
      };
      a = best_of(a, 0.f);
      last = a.i;
      if (!(a.v > 0.f)) {              // (by rounding alone, or in a row of nothing: the likeliest token)
        ArgPair most{-FLT_MAX, 0x7fffffff};
        const float* row = logits_of(node);      // (as it is in memory, with chosen drafts)
        for_columns(cols, [&](int c) {
          if (row[c] >= -FLT_MAX) most = arg_better(most, ArgPair{row[c], lo + c});
        });
        last = best_of(most, -FLT_MAX).i;
      }
    }
    if (rank == 0 && threadIdx.x == 0) {
      out[depth] = last < 0 || last >= p.V ? 0 : last;
      p.count[req] = depth + 1;
    }
    return;
  }
}

template <int CTAS>
static int launch_verify(VerifyParams p, cudaStream_t stream) {
  static PerDeviceOnce once;
  if (once.first()) {
    cudaFuncSetAttribute(tree_verify_kernel<CTAS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kVerifySmem);
    if (CTAS > 8) cudaFuncSetAttribute(tree_verify_kernel<CTAS>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  }
  p.slot = row_slice_cols(p.V, CTAS) * 4 + 16;
  p.ahead = std::min(p.ahead, kVerifySmem / p.slot);
  return launch_cluster_pdl(tree_verify_kernel<CTAS>, dim3(p.num_reqs * CTAS), CTAS, kVerifyThreads, (size_t)p.slot * p.ahead, stream, p) ==
                 cudaSuccess ? 0 : -2;
}

}  // namespace b200

using namespace b200;

extern "C" int b200_tree_verify(const B200TreeVerify* a, cudaStream_t stream) {
  if (a->V <= 0 || a->most <= 0) return -1;
  if (a->V > kVerifyMostCols || a->num_reqs > (1 << 26)) return -4;
  if (a->num_reqs <= 0) return 0;
  VerifyParams p;
  p.logits = (const float*)a->logits; p.ldl = a->ldl; p.probs = (const float*)a->probs; p.ldp = a->ldp;
  p.tokens = (const int64_t*)a->tokens; p.parents = (const int32_t*)a->parents; p.q_start = (const int32_t*)a->q_start;
  p.uniforms = (const float*)a->uniforms; p.temperature = (const float*)a->temperature;
  p.seeds = (const uint64_t*)a->seeds; p.steps = (const uint64_t*)a->steps;
  p.out = (int64_t*)a->out; p.path = (int32_t*)a->path; p.count = (int32_t*)a->count;
  p.num_reqs = a->num_reqs; p.total = a->total; p.V = a->V; p.most = a->most; p.status = device_status_word();
  // CTAs of a request and rows of a stage. Few requests have SMs to spare: sixteen, and rows ahead; many fill the chip with eight, and a row read in vain costs them
  // its time, as do slices that leave room for one CTA an SM. us, 8 CTAs and 1 row / 8 and 2 / 16 and 2 / 16 and 4:
  //   chains of 3 to 6 nodes, 128256 columns: 1 request 20.8 / 20.2 / 15.3 / 13.8, 4: 24.0 / 21.9 / 17.0 / 15.6, 8: 24.3 / 22.4 / 22.2 / 26.9,
  //   16: 32 / 42 / 36 / 46, 64: 76 / 106 / 102 / 148; 32000 columns: 4: 17.8 / 15.4 / 14.8 / 13.3, 16: 19.6 / 17.6 / 26.8 / 25.1, 128: 75 / 69 / 136 / 130;
  //   trees of 20 to 32 nodes, chosen, 128256 columns: 1 request 27.2 / 22.7 / 18.4 / 20.9, 8: 26.7 / 22.5 / 21.4 / 31.1, 64: 67 / 92 / 92 / 160;
  //   drawn, up to three children a node: 1: 29.0 / 27.2 / 21.0 / 19.8, 8: 35 / 37 / 34 / 33, 16: 40 / 53 / 48 / 59, 64: 97 / 132 / 128 / 192;
  //   4000 columns, chains: 1: 12.4 / 10.9 / 10.8 / 9.2, 16: 18.5 / 15.4 / 23.7 / 22.0, 128: 71 / 60 / 116 / 106; drawn trees: 16: 21.2 / 17.8 / 25.9 / 24.6
  // Between the borders, chains of 128256 columns: 5: 23.2 / 22.4 / 17.3 / 15.8, 10: 26.3 / 25.1 / 24.1 / 28.9, 12: 26.2 / 25.3 / 23.8 / 32.8, 13: 29.3 / 27.2 / 24.1 / 30.7, 16: 31.1 / 41.4 / 35.8 / 45.9
  // (from 5 to 8 requests of long rows sixteen CTAs would still be up to 5 us faster; 5 of 4000 columns 14.7 / 11.7 / 11.6 / 10.1, 8 of 32000 15.2 / 13.2 / 15.5 / 14.6)
  const bool few = a->num_reqs <= 4;
  const int ctas = a->V <= 2048 ? 1 : few || row_slice_cols(a->V, 8) * 4 + 16 > kVerifySmem ? 16 : 8;
  const int slot = row_slice_cols(a->V, ctas) * 4 + 16;
  p.ahead = few ? (a->parents ? 2 : 4) : a->num_reqs <= 12 || 2 * slot <= 80 * 1024 ? 2 : 1;
  return ctas == 1 ? launch_verify<1>(p, stream) : ctas == 8 ? launch_verify<8>(p, stream) : launch_verify<16>(p, stream);
}
