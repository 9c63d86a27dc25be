// Rows of logits shared by the CTAs of a cluster, and the race of the random draw: what the sampler (sample.cu) and the verification of drafted
// tokens (tree_verify.cu) have in common.
#pragma once
#include <float.h>

#include "sm100.cuh"

namespace b200 {

static constexpr float kEps = 1e-5f;      // temperatures below are greedy

struct ArgPair { float v; int i; };
__device__ __forceinline__ ArgPair arg_better(ArgPair a, ArgPair b) {
  return (b.v > a.v || (b.v == a.v && b.i < a.i)) ? b : a;
}
__device__ __forceinline__ ArgPair block_argmax(ArgPair a, ArgPair* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    ArgPair b;
    b.v = __shfl_xor_sync(0xffffffffu, a.v, o);
    b.i = __shfl_xor_sync(0xffffffffu, a.i, o);
    a = arg_better(a, b);
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  if (lane == 0) sh[warp] = a;
  __syncthreads();
  ArgPair r = (lane < nw) ? sh[lane] : ArgPair{-FLT_MAX, 0x7fffffff};
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    ArgPair b;
    b.v = __shfl_xor_sync(0xffffffffu, r.v, o);
    b.i = __shfl_xor_sync(0xffffffffu, r.i, o);
    r = arg_better(r, b);
  }
  __syncthreads();
  return r;
}

__host__ __device__ __forceinline__ int row_slice_cols(int V, int ctas) { return ((V + ctas - 1) / ctas + 3) & ~3; }
template <int CTAS>
__device__ __forceinline__ int row_rank() {
  if constexpr (CTAS > 1) return (int)cluster_ctarank();
  return 0;
}
template <int CTAS>
__device__ __forceinline__ void row_sync() {
  if constexpr (CTAS > 1) cluster_sync_all();
}
// Exchange of W words per CTA: each CTA stores its own into every CTA of the cluster, and after one cluster barrier all
// threads read them at home. Two buffers in turn, so that one barrier a call is enough.
template <int CTAS, int W>
struct RowExchange {
  float slot[2][CTAS][W];
};
template <int CTAS, int W>
__device__ __forceinline__ void row_gather(RowExchange<CTAS, W>& ex, int turn, const float (&mine)[W], float (&all)[CTAS][W]) {
  if constexpr (CTAS == 1) {
#pragma unroll
    for (int w = 0; w < W; ++w) all[0][w] = mine[w];
    return;
  }
  if (threadIdx.x < CTAS) {
    const uint32_t to = mapa_u32(smem_u32(&ex.slot[turn & 1][cluster_ctarank()][0]), threadIdx.x);
#pragma unroll
    for (int w = 0; w < W; ++w) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4 * w), "f"(mine[w]) : "memory");
  }
  cluster_sync_all();
#pragma unroll
  for (int r = 0; r < CTAS; ++r)
#pragma unroll
    for (int w = 0; w < W; ++w) all[r][w] = ex.slot[turn & 1][r][w];
}

// Exponential race: argmax_i p_i / (-log u_i), u_i of a counter generator.
__host__ __device__ inline uint64_t splitmix64(uint64_t z) {
  z += 0x9E3779B97F4A7C15ull;
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return z ^ (z >> 31);
}
// One and the first 23 bits of 1 - u_i, which is more than they say and at most kRaceRest more; at: step times 0x100000001B3 and the column. (The last step of
// splitmix64 leaves the upper 31 bits as they are.)
static constexpr float kRaceRest = 1.1920929e-7f;
__device__ __forceinline__ float race_rest(uint64_t seed, uint64_t at) {
  uint64_t z = (seed ^ splitmix64(at)) + 0x9E3779B97F4A7C15ull;
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return __uint_as_float((~(uint32_t)(z >> 32) >> 9) | 0x3f800000u);
}
// -log u_i in 32 bits, within 2^-20 of itself: by log1p, whose argument is taken from the number's bits, so that a small one keeps its own.
__device__ __forceinline__ float race_time(uint64_t seed, uint64_t step, int col) {
  const uint64_t z = splitmix64(seed ^ splitmix64(step * 0x100000001B3ull + (uint64_t)col));
  const float rest = ((float)(~z >> 11) + 0.5f) * (1.f / 9007199254740992.f), u = ((float)(z >> 11) + 0.5f) * (1.f / 9007199254740992.f);
  return rest < 0.5f ? -log1pf(-rest) : -logf(u);
}
__device__ __forceinline__ float race_key(float prob, uint64_t seed, uint64_t step, int col) {
  const uint64_t z = splitmix64(seed ^ splitmix64(step * 0x100000001B3ull + (uint64_t)col));
  const double u = ((double)(z >> 11) + 0.5) * (1.0 / 9007199254740992.0);
  const float e = (float)(-log(u));
  return prob / e;
}

}  // namespace b200
