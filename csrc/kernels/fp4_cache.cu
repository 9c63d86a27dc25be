// Keys and values into a paged cache held in 4 bits, and back (layout: fp4_cache.cuh).
//
// append:  y = rope(norm(x)) for q and k heads, v as it is; q goes on in bf16, rounded once; k and v in groups of 16 dims
//            s = max |y| / 6,   code = e2m1(y / s)   (both rounded to nearest, ties to even; s = 0: all codes 0)
//          Sums, rotation and quotients are fp32, and keys are not rounded to bf16 on the way to their codes. Values past 6 * 10240
//          (infinities too) saturate, a NaN makes its group NaN.
// read:    code * s for the given slots, exact in bf16.
//
// Both are passes over memory. At 8192 tokens of 32 + 8 + 8 heads of 128 dims an append takes 48.5 us for 177 MB (3.65 TB/s), a read back 12.3 us for
// 43 MB (3.5 TB/s): instructions bound them (an append issues in 0.64 of the cycles, half of it rotation and quotients), not the 27 and 7 us of the
// bytes. A token or a few take 2.4 us, the latency of position -> angles and slot -> cell.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "api.h"
#include "fp4_cache.cuh"
#include "sm100.cuh"

namespace b200 {

// Eight values -> eight codes, the first in the lowest nibble.
__device__ __forceinline__ uint32_t e2m1_of(const float (&r)[8]) {
  uint32_t w;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}\n"
      : "=r"(w)
      : "f"(r[0]), "f"(r[1]), "f"(r[2]), "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7]));
  return w;
}

__device__ __forceinline__ void unpack_bf16x8(const uint4& v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 f = unpack_bf16x2(w[k]);
    x[2 * k] = f.x;
    x[2 * k + 1] = f.y;
  }
}

// A lane has 8 dims (16 bytes) of a head, so a head is D / 8 lanes and a group of 16 dims two neighbours. A warp takes `passes` times
// the heads that its lanes hold, all of one token, whose position, slot, cos and sin are fetched once behind the first heads' loads.
// Query heads have a loop of their own: two thirds of the work, and half as many instructions as keys and values take.
template <int D, bool MANY>
__global__ void __launch_bounds__(128, MANY ? 8 : 9) fp4_append_kernel(B200Fp4Append p, int parts, int passes) {
  using Cell = Fp4Cell<D>;
  constexpr int kLanes = D / 8, kHeads = 32 / kLanes;
  __shared__ float exchange[4][256];
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane % kLanes, side = lane / kLanes;
  const int nheads = p.Hq + 2 * p.Hkv, v0 = p.Hq + p.Hkv;
  const uint32_t gw = blockIdx.x * 4 + warp;                     // (T * parts < 2^31)
  const int t = (int)(gw / (uint32_t)parts), h0 = (int)(gw - (uint32_t)t * parts) * (kHeads * passes), h1 = min(nheads, h0 + kHeads * passes);
  if (t >= p.T) return;
  const __nv_bfloat16* qrow = (const __nv_bfloat16*)p.q + (size_t)t * p.ldq + l * 8;
  const __nv_bfloat16* krow = (const __nv_bfloat16*)p.k + (size_t)t * p.ldk + l * 8;
  const __nv_bfloat16* vrow = (const __nv_bfloat16*)p.v + (size_t)t * p.ldv + l * 8;
  const auto load = [&](int first) {                            // of the lane's head behind `first`
    const int h = first + side;
    return h >= h1 ? make_uint4(0, 0, 0, 0)
                   : *reinterpret_cast<const uint4*>(h < p.Hq ? qrow + (size_t)h * p.q_head_stride : h < v0 ? krow + (h - p.Hq) * D : vrow + (h - v0) * D);
  };
  uint4 ahead[2] = {load(h0), MANY ? load(h0 + kHeads) : make_uint4(0, 0, 0, 0)};       // two passes on their way
  const int rot = p.cos_sin ? p.rot : 0, half = rot >> 1;
  float c[8], s[8];                                             // y = x c + partner s
#pragma unroll
  for (int e = 0; e < 8; ++e) { c[e] = 1.f; s[e] = 0.f; }
  if (rot && h0 < v0) {
    const int64_t at = ((const int64_t*)p.positions)[t];
    const bool there = at >= 0 && at < p.table_rows;
    const float* cs = (const float*)p.cos_sin + (there ? at : 0) * rot;
    const int d0 = l * 8, j0 = d0 < half ? d0 : d0 - half;
    if (p.neox && !(half & 7) && !(reinterpret_cast<uintptr_t>(p.cos_sin) & 15)) {      // eight angles side by side
      if (d0 < rot) {
#pragma unroll
        for (int k = 0; k < 8; k += 4) {
          const float4 a = *reinterpret_cast<const float4*>(cs + j0 + k), b = *reinterpret_cast<const float4*>(cs + half + j0 + k);
          c[k] = a.x; c[k + 1] = a.y; c[k + 2] = a.z; c[k + 3] = a.w;
          s[k] = b.x; s[k + 1] = b.y; s[k + 2] = b.z; s[k + 3] = b.w;
        }
        if (d0 < half) {
#pragma unroll
          for (int e = 0; e < 8; ++e) s[e] = -s[e];
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = d0 + e;
        if (d < rot) {
          const int j = p.neox ? (d < half ? d : d - half) : d >> 1;
          c[e] = cs[j];
          s[e] = (p.neox ? d < half : !(d & 1)) ? -cs[half + j] : cs[half + j];
        }
      }
    }
    if (!there) {                                               // a position outside the table: NaN
#pragma unroll
      for (int e = 0; e < 8; ++e) c[e] = l * 8 + e < rot ? __int_as_float(0x7fffffff) : 1.f;
    }
  }
  uint8_t* cell = nullptr;                                      // the token's cell of kv head 0
  int token = 0;
  if (h1 > p.Hq) {
    const int64_t slot = ((const int64_t*)p.slots)[t];
    if (slot >= 0 && slot < p.num_blocks * p.block_size) {
      const int64_t blk = (slot >> 31) == 0 ? (int64_t)((uint32_t)slot / (uint32_t)p.block_size) : slot / p.block_size;
      const int off = (int)(slot - blk * p.block_size);
      cell = (uint8_t*)p.cache + (blk * p.Hkv * (p.block_size / kCellTokens) + off / kCellTokens) * Cell::kBytes;
      token = off % kCellTokens;
    }
  }
  const size_t head_bytes = (size_t)(p.block_size / kCellTokens) * Cell::kBytes;
  const float g = p.gemma ? 1.f : 0.f;
  // norm and rotation of a pass's heads; the warp stays together (shuffles)
  const auto turned = [&](int first, const uint4& raw, float (&y)[8]) {
    const int h = first + side;
    float x[8];
    unpack_bf16x8(raw, x);
    const bool is_q = h < p.Hq, is_v = h >= v0;
    if (p.q_norm || p.k_norm) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const __nv_bfloat16* w = (const __nv_bfloat16*)(is_q ? p.q_norm : p.k_norm);
      if (w && !is_v) {
        float wf[8];
        unpack_bf16x8(*reinterpret_cast<const uint4*>(w + l * 8), wf);
        const float inv = rsqrtf(ss / (float)D + p.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = x[e] * inv * (wf[e] + g);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = x[e];
    if (rot && first < v0) {                          // (the same for the warp: a q or k head among its heads)
      float other[8];
      if (!p.neox) {
#pragma unroll
        for (int e = 0; e < 8; ++e) other[e] = x[e ^ 1];
      } else if (!(half & 7)) {
        const int partner = lane + (l * 8 < half ? half / 8 : l * 8 < rot ? -half / 8 : 0);
#pragma unroll
        for (int e = 0; e < 8; ++e) other[e] = __shfl_sync(0xffffffffu, x[e], partner);
      } else {
        float* b = exchange[warp];
        __syncwarp();
#pragma unroll
        for (int e = 0; e < 8; ++e) b[lane * 8 + e] = x[e];
        __syncwarp();
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int d = l * 8 + e;
          other[e] = d < rot ? b[side * D + (d < half ? d + half : d - half)] : 0.f;
        }
      }
      if (p.neox && !(half & 7)) {                              // the lane's dims are all turned, or none is
        if (!is_v && l * 8 < rot) {
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = x[e] * c[e] + other[e] * s[e];
        }
      } else if (!is_v) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = l * 8 + e < rot ? x[e] * c[e] + other[e] * s[e] : x[e];
      }
    }
  };
  const auto query = [&](int h, const float (&y)[8]) {
    __nv_bfloat16* dst = p.q_out ? (__nv_bfloat16*)p.q_out + (size_t)t * p.ldo + h * D
                                 : (__nv_bfloat16*)p.q + (size_t)t * p.ldq + (size_t)h * p.q_head_stride;
    *reinterpret_cast<uint4*>(dst + l * 8) = make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]),
                                                        pack_bf16x2(y[6], y[7]));
  };
  const auto next = [&](int first) {
    const uint4 raw = ahead[0];
    if constexpr (MANY) {
      ahead[0] = ahead[1];
      ahead[1] = load(first + 2 * kHeads);
    }
    return raw;
  };
  int first = h0;
  if constexpr (MANY) {
#pragma unroll 1
    for (; first + kHeads <= min(p.Hq, h1); first += kHeads) {  // passes of query heads only
      float y[8];
      turned(first, next(first), y);
      query(first + side, y);
    }
  }
#pragma unroll 1
  for (; first < h1; first += kHeads) {
    const int h = first + side;
    float y[8];
    turned(first, next(first), y);
    if (!MANY && first + kHeads <= p.Hq) {
      query(h, y);
      return;
    }
    uint32_t top = 0;                                           // of |y|, as bits: a NaN is above infinity
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(y[e]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    if (h >= h1) continue;
    const bool is_q = h < p.Hq, is_v = h >= v0;
    if (is_q) query(h, y);
    if (is_q || !cell) continue;
    const uint8_t scale = fp4_scale_byte(__fdiv_rn(__uint_as_float(top), 6.f));
    const float sf = fp4_scale_value(scale);
    // Quotients by the scale's reciprocal and one correction by the remainder (fma): values of few bits lie exactly between two codes, and there
    // a product with the rounded reciprocal alone decides by its own rounding. With the correction a quotient that fp32 holds exactly, as every
    // border between codes is, comes out exactly. (2048 of these a token of 8 + 8 heads of 128 dims; divisions took twice the kernel's time.)
    float inv, r[8];
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(sf));
    if (sf == 0.f) inv = 0.f;
    if (top >= 0x7f800000u) {                                   // infinities: the largest code
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = fminf(fmaxf(y[e], -3.0e38f), 3.0e38f);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float q = y[e] * inv;
      r[e] = fmaf(fmaf(-q, sf, y[e]), inv, q);
    }
    const uint32_t codes = e2m1_of(r);
    uint8_t* dst = cell + (size_t)(is_v ? h - v0 : h - p.Hq) * head_bytes;
    if (is_v) {
      *reinterpret_cast<uint32_t*>(dst + Cell::value_at(token, l * 4)) = codes;
      if (!(l & 1)) dst[Cell::kValueScales + (l >> 1) * kCellTokens + token] = scale;
    } else {
      *reinterpret_cast<uint32_t*>(dst + token * Cell::kRow + l * 4) = codes;
      if (!(l & 1)) dst[Cell::kKeyScales + token * Cell::kScales + (l >> 1)] = scale;
    }
  }
}

// A lane turns 8 codes into 16 bytes of bf16, of N lots of `tokens` tokens (one, or as many as a block's threads have room for): the same place
// in each, whose loads are all on their way at once.
template <int D, int N>
__global__ void __launch_bounds__(256) fp4_read_kernel(B200Fp4Read p, int tokens) {
  using Cell = Fp4Cell<D>;
  pdl_wait();
  pdl_launch_dependents();
  const int per = 2 * p.Hkv * (D / 8);                          // lanes of a token
  const int local = tokens > 1 ? threadIdx.x / per : 0, first = threadIdx.x - local * per, cells = p.block_size / kCellTokens;
  const long long t0 = (long long)blockIdx.x * tokens * N + local;
  if (local >= tokens) return;
  const uint8_t* cell0[N];                                      // the token's cell of kv head 0; null: none
  int token[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const long long t = t0 + j * tokens;
    const int64_t slot = t < p.n ? ((const int64_t*)p.slots)[t] : -1;
    const int64_t blk = (slot >> 31) == 0 ? (int64_t)((uint32_t)slot / (uint32_t)p.block_size) : slot / p.block_size;
    const int off = (int)(slot - blk * p.block_size);
    token[j] = off % kCellTokens;
    cell0[j] = slot >= 0 && slot < p.num_blocks * p.block_size
                   ? (const uint8_t*)p.cache + (blk * p.Hkv * cells + off / kCellTokens) * Cell::kBytes : nullptr;
  }
  for (int i = first; i < per; i += 256) {
    const int l = i % (D / 8), h2 = i / (D / 8), kv = h2 >= p.Hkv, h = h2 - kv * p.Hkv;
    uint32_t codes[N];
    uint8_t scale[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const uint8_t* cell = cell0[j] + (size_t)h * cells * Cell::kBytes;
      codes[j] = cell0[j] ? *reinterpret_cast<const uint32_t*>(cell + (kv ? Cell::value_at(token[j], l * 4) : token[j] * Cell::kRow + l * 4)) : 0;
      scale[j] = cell0[j] ? cell[kv ? Cell::kValueScales + (l >> 1) * kCellTokens + token[j]
                                    : Cell::kKeyScales + token[j] * Cell::kScales + (l >> 1)] : 0;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float s = fp4_scale_value(scale[j]);
      uint32_t f16[4], o[4];
      cvt_e2m1x8(codes[j], f16);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = __half22float2(*reinterpret_cast<__half2*>(&f16[e]));
        o[e] = pack_bf16x2(f.x * s, f.y * s);
      }
      const long long t = t0 + j * tokens;
      if (t < p.n)
        *reinterpret_cast<uint4*>((__nv_bfloat16*)(kv ? p.v : p.k) + (t * p.Hkv + h) * D + l * 8) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

template <int D>
static int launch_append(const B200Fp4Append& p, cudaStream_t stream) {
  constexpr int kHeads = 32 / (D / 8);
  const int nheads = p.Hq + 2 * p.Hkv;
  const int groups = (nheads + kHeads - 1) / kHeads;
  const auto go = [&](auto kernel, int passes) {
    const int parts = (groups + passes - 1) / passes;
    const long long warps = (long long)p.T * parts;
    if (warps >= (1ll << 31)) return -4;
    return launch_pdl(kernel, dim3((unsigned)((warps + 3) / 4)), dim3(128), 0, stream, p, parts, passes) == cudaSuccess ? 0 : -2;
  };
  // Passes that leave some 8192 warps: more of them than one are worth their own kernel, which fetches two heads ahead and keeps to 64 registers
  // (8192 tokens of 32 + 8 + 8 heads of 128 dims: 48.5 us, one pass a warp 81; 1024 tokens 9.3 and 10.8; 256 tokens are one pass, 4.7).
  const long long each = ((long long)p.T * groups + 8191) / 8192;
  return each > 1 ? go(fp4_append_kernel<D, true>, (int)min(each, (long long)groups)) : go(fp4_append_kernel<D, false>, 1);
}

}  // namespace b200

using namespace b200;

static bool fp4_cache_ok(int D, int block_size, int Hkv, long long num_blocks) {
  return (D == 64 || D == 128 || D == 256) && block_size > 0 && block_size % kCellTokens == 0 && Hkv > 0 && num_blocks > 0;
}

extern "C" int b200_fp4_append(const B200Fp4Append* a, cudaStream_t stream) {
  if (a->T <= 0) return 0;
  if (!fp4_cache_ok(a->D, a->block_size, a->Hkv, a->num_blocks) || a->Hq < 0 || !a->k || !a->v || !a->slots || !a->cache || (a->Hq && !a->q))
    return -1;
  if (a->cos_sin && (!a->positions || a->rot < 0 || a->rot > a->D || (a->rot & 1))) return -1;
  const uintptr_t bits = (uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->q_out | (uintptr_t)a->q_norm |
                         (uintptr_t)a->k_norm | (uintptr_t)a->cache | (uintptr_t)((a->ldq | a->ldk | a->ldv | a->ldo | a->q_head_stride) * 2);
  if (bits & 15) return -1;
  return a->D == 64 ? launch_append<64>(*a, stream) : a->D == 128 ? launch_append<128>(*a, stream) : launch_append<256>(*a, stream);
}

extern "C" int b200_fp4_read(const B200Fp4Read* a, cudaStream_t stream) {
  if (a->n <= 0) return 0;
  if (!fp4_cache_ok(a->D, a->block_size, a->Hkv, a->num_blocks) || (((uintptr_t)a->cache | (uintptr_t)a->k | (uintptr_t)a->v) & 15) || !a->slots ||
      !a->cache || !a->k || !a->v)
    return -1;
  const int per = 2 * a->Hkv * (a->D / 8), tokens = per < 256 ? 256 / per : 1;
  const auto go = [&](auto kernel, long long lot) {
    const long long blocks = (a->n + lot - 1) / lot;
    if (blocks >= (1ll << 31)) return -4;
    return launch_pdl(kernel, dim3((unsigned)blocks), dim3(256), 0, stream, *a, tokens) == cudaSuccess ? 0 : -2;
  };
  // two lots a block where that leaves blocks enough for every SM (8192 tokens of 8 heads of 128 dims: 12.3 us, one lot 14.8, four 12.5)
  const bool many = a->n >= 2ll * tokens * 8 * b200_num_sms();
  const auto by = [&](auto d) {
    constexpr int kD = decltype(d)::value;
    return many ? go(fp4_read_kernel<kD, 2>, 2ll * tokens) : go(fp4_read_kernel<kD, 1>, tokens);
  };
  return a->D == 64 ? by(std::integral_constant<int, 64>()) : a->D == 128 ? by(std::integral_constant<int, 128>()) : by(std::integral_constant<int, 256>());
}
