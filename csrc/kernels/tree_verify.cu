// Verification of drafted tokens against the target's distributions, by given random numbers: chains and trees.
//
// From the root down: at a node with logits l, w_j = e^(l_j - max l), the children x_1, x_2 .. are asked in their order. Drawn from q (the drafter's
// distribution at the node), with b = 0 and Z = sum w at first: x is accepted if u q(x) Z < max(w_x - b q(x), 0); refused, b becomes b + Z and Z
// becomes sum max(w - b q, 0). That is the refusal's residual norm(max(p - q, 0)), one refusal after another, in closed form: each costs one sum over
// the row and no division. Chosen instead (no q): x is accepted if u Z < w_x, and a refused one leaves w; the sums are built up from the tokens that are
// no children's, so that none is a difference. After an accepted child the walk goes on there; where none is accepted the last token is the
// exponential race over what is left of w, with the same numbers as the sampler's draw. Greedy requests accept the argmax.
//
// Only the rows that the walk visits are read, once each: a node's row (and q's) lies in shared memory, a slice for each CTA of a cluster, for all sums and
// the draw. Bound: a node's chain of loads, reductions and cluster barriers where there are few requests, the rows' bytes where there are many.
#include "api.h"
#include "row_cluster.cuh"

namespace b200 {

static constexpr int kVerifyThreads = 512, kVerifyNodes = 1024;
static constexpr int kVerifySlice = 24576;       // columns of a CTA at the most: two floats each

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
};

struct VerifyShared {
  ArgPair arg[32];
  float sums[32];
  int parent[kVerifyNodes], token[kVerifyNodes], child[kVerifyNodes];
  float u[kVerifyNodes], w[kVerifyNodes], q[kVerifyNodes];       // random numbers of the nodes; weights of the children
  int children, accepted;
};

// Sum over the block, in every thread.
__device__ __forceinline__ float verify_sum(float v, float* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) sh[warp] = v;
  __syncthreads();
  v = lane < kVerifyThreads / 32 ? sh[lane] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  return v;
}
__device__ __forceinline__ float prob_of(float q) { return fminf(fmaxf(q, 0.f), FLT_MAX); }        // (a NaN is 0)
__device__ __forceinline__ float logit_of(float l) { return l != l ? -INFINITY : l; }

template <int CTAS>
__global__ void __launch_bounds__(kVerifyThreads, 1) tree_verify_kernel(VerifyParams p) {
  extern __shared__ float4 slice_raw[];
  __shared__ VerifyShared sh;
  __shared__ RowExchange<CTAS, 3> ex3;
  __shared__ RowExchange<CTAS, 1> ex1;
  constexpr int T = kVerifyThreads;
  const int per = row_slice_cols(p.V, CTAS), rank = row_rank<CTAS>(), lo = min(p.V, rank * per), cols = min(p.V, lo + per) - lo;
  float* w = reinterpret_cast<float*>(slice_raw);
  float* q = w + per;
  const int req = blockIdx.x / CTAS;
  pdl_wait();
  pdl_launch_dependents();
  const int row0 = min(max(p.q_start[req], 0), p.total), n = min(max(0, min(p.q_start[req + 1], p.total) - row0), kVerifyNodes);
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
  row_sync<CTAS>();                    // (every CTA runs, before the first store into another; also a barrier of the CTA)
  if constexpr (CTAS == 1) __syncthreads();
  if (n == 0) {
    if (rank == 0 && threadIdx.x == 0) p.count[req] = 0;
    return;
  }
  int node = 0, depth = 0, turn1 = 0, turn3 = 0;
  int64_t last = 0;
  while (true) {
    const float* l = p.logits + (row0 + node) * p.ldl;
    const float* pq = drawn ? p.probs + (row0 + node) * p.ldp : nullptr;
    // ---- the node's row, its largest logit; its children in their order
    ArgPair top{-FLT_MAX, 0x7fffffff};
    for (int i = threadIdx.x; i < cols; i += T) {
      const float v = logit_of(l[lo + i]);
      w[i] = v;
      if (drawn) q[i] = prob_of(pq[lo + i]);
      top = arg_better(top, ArgPair{v, lo + i});
    }
    if (threadIdx.x < 32) {
      int found = 0;
      if (depth + 1 < p.most)
        for (int base = node + 1; base < n; base += 32) {
          const int j = base + threadIdx.x;
          const bool is = j < n && sh.parent[j] == node;
          const uint32_t who = __ballot_sync(0xffffffffu, is);
          if (is) sh.child[found + __popc(who & ((1u << threadIdx.x) - 1))] = j;
          found += __popc(who);
        }
      if (threadIdx.x == 0) sh.children = found;
    }
    top = block_argmax(top, sh.arg);
    const int children = sh.children;
    if (top.v == -FLT_MAX) {           // (nothing, or nothing above -inf)
      bool any = false;
      for (int i = threadIdx.x; i < cols; i += T) any |= w[i] > -INFINITY;
      if (!__syncthreads_or(any)) top = ArgPair{-INFINITY, 0x7fffffff};
    }
    float sum = 0.f;
    if (!greedy) {
      if (!drawn && children > 0) {    // (chosen drafts stand apart)
        for (int i = threadIdx.x; i < children; i += T) {
          const int c = sh.token[sh.child[i]] - lo;
          if (c >= 0 && c < cols) w[c] = -INFINITY;
        }
        __syncthreads();
      }
      for (int i = threadIdx.x; i < cols; i += T) {
        const float v = w[i], e = v == top.v ? 1.f : expf(v - top.v);       // (an infinity's weight is 1)
        w[i] = v == -INFINITY ? 0.f : e;
        sum += w[i];
      }
      sum = verify_sum(sum, sh.sums);
    }
    float all[CTAS][3];
    row_gather<CTAS, 3>(ex3, turn3++, {top.v, __int_as_float(top.i), sum}, all);
    ArgPair best{-FLT_MAX, 0x7fffffff};
    float m = -INFINITY;
#pragma unroll
    for (int r = 0; r < CTAS; ++r) {
      best = arg_better(best, ArgPair{all[r][0], __float_as_int(all[r][1])});
      m = fmaxf(m, all[r][0]);
    }
    const auto scale_of = [&](float mine) { return mine == m ? 1.f : expf(mine - m); };
    const float factor = top.v == -INFINITY ? 0.f : scale_of(top.v);       // of this CTA's weights
    float Z = 0.f;
#pragma unroll
    for (int r = 0; r < CTAS; ++r) Z += all[r][0] == -INFINITY ? 0.f : all[r][2] * scale_of(all[r][0]);

    // ---- the children
    float b = 0.f;
    int next = -1;
    if (greedy) {
      for (int i = 0; i < children && next < 0; ++i)
        if (sh.token[sh.child[i]] == best.i) next = sh.child[i];
    } else if (children > 0) {
      for (int i = threadIdx.x; i < children; i += T) {
        const int t = sh.token[sh.child[i]];
        const float v = t < 0 ? -INFINITY : logit_of(l[t]);
        bool again = false;            // (of two chosen drafts alike, the second has no weight left)
        if (!drawn)
          for (int k = 0; k < i; ++k) again |= sh.token[sh.child[k]] == t;
        sh.w[i] = v == -INFINITY || again ? 0.f : v == m ? 1.f : expf(v - m);
        sh.q[i] = drawn && t >= 0 ? prob_of(pq[t]) : 0.f;
      }
      __syncthreads();
      if (drawn) {
        for (int i = 0; i < children; ++i) {
          const int c = sh.child[i];
          if (sh.u[c] * sh.q[i] * Z < fmaxf(sh.w[i] - b * sh.q[i], 0.f)) {
            next = c;
            break;
          }
          b += Z;
          float part = 0.f;
          for (int k = threadIdx.x; k < cols; k += T) part += fmaxf(w[k] * factor - b * q[k], 0.f);
          part = verify_sum(part, sh.sums);
          float parts[CTAS][1];
          row_gather<CTAS, 1>(ex1, turn1++, {part}, parts);
          Z = 0.f;
#pragma unroll
          for (int r = 0; r < CTAS; ++r) Z += parts[r][0];
        }
      } else {
        if (threadIdx.x == 0) {        // Z at child i: what no child has, and the children from i on
          float z = Z;
          for (int i = children - 1; i >= 0; --i) {
            z += sh.w[i];
            sh.q[i] = z;
          }
          sh.accepted = -1;
          for (int i = 0; i < children; ++i)
            if (sh.u[sh.child[i]] * sh.q[i] < sh.w[i]) {
              sh.accepted = sh.child[i];
              break;
            }
        }
        __syncthreads();
        next = sh.accepted;
      }
    }
    if (next >= 0) {
      if (rank == 0 && threadIdx.x == 0) {
        out[depth] = p.tokens[row0 + next];
        path[depth + 1] = next;
      }
      node = next;
      ++depth;
      __syncthreads();                 // (lists and slices are written anew)
      continue;
    }
    // ---- the last token
    last = best.i;
    if (!greedy) {
      const uint64_t seed = p.seeds[req], step = p.steps[req];
      ArgPair a{0.f, 0x7fffffff};
      for (int k = threadIdx.x; k < cols; k += T) {
        const float left = drawn ? fmaxf(w[k] * factor - b * q[k], 0.f) : w[k] * factor;
        if (left > 0.f) a = arg_better(a, ArgPair{race_key(left, seed, step, lo + k), lo + k});
      }
      a = block_argmax(a, sh.arg);
      row_gather<CTAS, 3>(ex3, turn3++, {a.v, __int_as_float(a.i), 0.f}, all);
      a = ArgPair{0.f, 0x7fffffff};
#pragma unroll
      for (int r = 0; r < CTAS; ++r) a = arg_better(a, ArgPair{all[r][0], __float_as_int(all[r][1])});
      if (a.v > 0.f) last = a.i;       // (nothing left, which rounding alone can do: the likeliest token)
    }
    break;
  }
  if (rank == 0 && threadIdx.x == 0) {
    out[depth] = last < 0 || last >= p.V ? 0 : last;
    p.count[req] = depth + 1;
  }
}

template <int CTAS>
static int launch_verify(const VerifyParams& p, cudaStream_t stream) {
  static PerDeviceOnce once;
  if (once.first()) {
    cudaFuncSetAttribute(tree_verify_kernel<CTAS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kVerifySlice * 8);
    if (CTAS > 8) cudaFuncSetAttribute(tree_verify_kernel<CTAS>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  }
  const size_t smem = (size_t)row_slice_cols(p.V, CTAS) * (p.probs ? 8 : 4);
  return launch_cluster_pdl(tree_verify_kernel<CTAS>, dim3(p.num_reqs * CTAS), CTAS, kVerifyThreads, smem, stream, p) == cudaSuccess ? 0 : -2;
}

}  // namespace b200

using namespace b200;

extern "C" int b200_tree_verify(const B200TreeVerify* a, cudaStream_t stream) {
  if (a->V <= 0 || a->most <= 0) return -1;
  if (a->V > 16 * kVerifySlice || a->num_reqs > (1 << 26)) return -4;
  if (a->num_reqs <= 0) return 0;
  VerifyParams p;
  p.logits = (const float*)a->logits; p.ldl = a->ldl; p.probs = (const float*)a->probs; p.ldp = a->ldp;
  p.tokens = (const int64_t*)a->tokens; p.parents = (const int32_t*)a->parents; p.q_start = (const int32_t*)a->q_start;
  p.uniforms = (const float*)a->uniforms; p.temperature = (const float*)a->temperature;
  p.seeds = (const uint64_t*)a->seeds; p.steps = (const uint64_t*)a->steps;
  p.out = (int64_t*)a->out; p.path = (int32_t*)a->path; p.count = (int32_t*)a->count;
  p.num_reqs = a->num_reqs; p.total = a->total; p.V = a->V; p.most = a->most;
  if (a->V <= 2048) return launch_verify<1>(p, stream);
  return a->V <= 8 * kVerifySlice ? launch_verify<8>(p, stream) : launch_verify<16>(p, stream);
}
