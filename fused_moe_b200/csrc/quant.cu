// Activation quantiser: bf16 [T, 7168] -> e4m3 [T, 7168] + one fp32 scale per token per 128 columns, stored [56, T].
//
// This is the producer of `hidden_states` / `hidden_states_scale`, which the reference takes as given; its profiling
// script builds them with torch by multiplying with 448 / amax (scripts/yjl_ncu.py:413-416).  The specification here,
// operation for operation in IEEE float32:
//   s = max(amax * (1/448), 1e-12)      inv = 1 / s      q = e4m3_rn_satfinite(x * inv)
// i.e. one reciprocal per 128-column block and one multiplication + conversion per element.  (An earlier version
// reproduced the IEEE QUOTIENT x / s of the synthetic-input generator bit for bit, which needed 21 instructions per
// element and ran at 0.49 of the HBM bandwidth: the generator is a test fixture, not a specification.)
// HBM-bound: 14 336 B read + 7 392 B written per token.  One half-warp per (token, 128-column block): a lane holds 8
// columns (one 16-byte load, one 8-byte store, both fully coalesced), the maximum is one `redux.sync` over 16 lanes.
#include "common.cuh"

namespace b200moe {

__global__ void __launch_bounds__(256)
k_quantize_act(const uint4* x, int T, uint2* q, float* scale) {
  const int lane = threadIdx.x & 31;
  const int sub = lane & 15;        // lane within the half-warp that owns one 128-column block
  const uint32_t half_mask = (lane & 16) ? 0xffff0000u : 0x0000ffffu;
  const long long half_warps = static_cast<long long>(gridDim.x) * (blockDim.x >> 4);
  const long long total = static_cast<long long>(T) * H_BLOCKS;   // 128-column blocks
  pdl_launch_dependents();
  pdl_wait();
  constexpr int UNROLL = 4;   // independent blocks per half-warp and iteration
  for (long long p0 = static_cast<long long>(blockIdx.x) * (blockDim.x >> 4) + (threadIdx.x >> 4); p0 < total;
       p0 += half_warps * UNROLL) {
    uint4 raw[UNROLL];
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      const long long p = p0 + i * half_warps;
      raw[i] = p < total ? ld_dep(x + p * 16 + sub) : make_uint4(0u, 0u, 0u, 0u);   // 8 bf16
    }
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      const long long p = p0 + i * half_warps;
      if (p >= total) break;   // uniform over the half-warp
      const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
      float v[8];
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        // |x| of non-negative floats orders like their bit patterns
        m = max(m, max((w[j] << 16) & 0x7fffffffu, w[j] & 0x7fff0000u));
      }
      const float amax = __uint_as_float(__reduce_max_sync(half_mask, m));
      const float s = fmaxf(__fmul_rn(amax, 1.0f / 448.0f), 1e-12f);
      const float inv = __frcp_rn(s);
      uint2 out;
      out.x = quantize_pair(v[0], v[1], inv) | (quantize_pair(v[2], v[3], inv) << 16);
      out.y = quantize_pair(v[4], v[5], inv) | (quantize_pair(v[6], v[7], inv) << 16);
      q[p * 16 + sub] = out;
      if (sub == 0) {
        const long long t = p / H_BLOCKS;
        const int kb = static_cast<int>(p - t * H_BLOCKS);
        scale[static_cast<size_t>(kb) * T + t] = s;
      }
    }
  }
}

int launch_quantize_act(const void* x, int T, void* q, float* scale, int num_sms, cudaStream_t st) {
  if (T == 0) return B200MOE_OK;
  const long long total = static_cast<long long>(T) * H_BLOCKS;
  long long ctas = (total + 63) / 64;   // 16 half-warps x 4 blocks per CTA and iteration
  // one full wave of resident CTAs (a grid of 8 per SM ran as 1.6 waves of the 5 that fit at 43 registers per thread)
  static int resident = 0;
  if (resident == 0) {
    int n = 0;
    B200MOE_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k_quantize_act, 256, 0));
    resident = n > 0 ? n : 1;
  }
  const long long cap = static_cast<long long>(num_sms) * resident;
  if (ctas > cap) ctas = cap;
  B200MOE_CUDA_TRY(launch_pdl(k_quantize_act, dim3(static_cast<unsigned>(ctas)), dim3(256), 0, st,
                              static_cast<const uint4*>(x), T, static_cast<uint2*>(q), scale));
  return B200MOE_OK;
}

}  // namespace b200moe
