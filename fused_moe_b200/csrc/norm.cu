// Residual addition + RMS norm, in front of the layer.
//
//   r = round(x + residual)      rstd = 1 / sqrt(mean(r^2) + eps)      y = r * rstd * weight
// r is the residual stream that the next block reads, rounded to its own type, and the norm is taken of the rounded values: y
// then depends on nothing but r, so the backward pass needs no other saved tensor.  y leaves in the type of x and / or as e4m3
// with one float32 scale per token per 128 columns, [H / 128, T], as k_quantize_act writes them, from the float32 y.
//
// Backward, with g = dy * weight and n = H columns:
//   dr = rstd * (g - r * rstd^2 * mean(g * r)) + dr_out       dweight = sum over tokens of dy * r * rstd
// rstd is recomputed: sum(r^2) and sum(g * r) are taken in the same pass over the row.
//
// Sums and statistics are float32.  All kernels are bound by the bytes of the rows.
#include <type_traits>

#include "row_vec.cuh"

namespace b200moe {

// Sum over the CTA of N values at once; `s` has 32 * N floats and is not reused before the next barrier.
template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float* s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], d);
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) s[i * 32 + warp] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lane < warps ? s[i * 32 + lane] : 0.f;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], d);
}

// One CTA per token; a thread holds VPT vectors of eight columns, blockDim.x vectors apart, so that a half-warp holds a whole
// 128-column block.
template <typename X, typename R, int VPT>
__global__ void __launch_bounds__(512)
k_add_rms_norm(const uint8_t* x, long long x_pitch, const uint8_t* residual, long long residual_pitch,
               const uint8_t* weight, int weight_type, int T, int n_vec, float eps, uint8_t* stream, uint8_t* y,
               uint8_t* q, float* scale) {
  __shared__ float s_sum[32];
  const int t = blockIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  Vec8<X> xv[VPT];
  Vec8<R> rv[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v >= n_vec) continue;
    xv[i] = load_vec8<X>(x + t * x_pitch, v);
    if (residual) rv[i] = load_vec8<R>(residual + t * residual_pitch, v);
  }
  float r[VPT][8];
  float sum[1] = {0.f};
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[i][j] = 0.f;
    if (v >= n_vec) continue;
    unpack_vec8<X>(xv[i], r[i]);
    if (residual) {
      float a[8];
      unpack_vec8<R>(rv[i], a);
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] += r[i][j];
      const Vec8<R> rounded = pack_vec8<R>(a);
      store_vec8<R>(stream + static_cast<long long>(t) * n_vec * 8 * sizeof(R), v, rounded);
      unpack_vec8<R>(rounded, r[i]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[0] = fmaf(r[i][j], r[i][j], sum[0]);
  }
  block_sum(sum, s_sum);
  const float rstd = __frsqrt_rn(sum[0] / static_cast<float>(n_vec * 8) + eps);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v >= n_vec) continue;
    float w[8];
    load_vec8_any(weight, v, weight_type, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) r[i][j] = r[i][j] * rstd * w[j];
    if (y) store_vec8<X>(y + static_cast<long long>(t) * n_vec * 8 * sizeof(X), v, pack_vec8<X>(r[i]));
    if (q) {   // n_vec is a multiple of 16 here: a half-warp is inside the row or outside as a whole
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(r[i][j]) & 0x7fffffffu);
      // the largest pattern is a NaN where there is one: it then stands in the scale too
      const float amax = __uint_as_float(__reduce_max_sync((threadIdx.x & 16) ? 0xffff0000u : 0x0000ffffu, m));
      float s = __fmul_rn(amax, 1.0f / 448.0f);
      if (s < 1e-12f) s = 1e-12f;
      const float inv = __frcp_rn(s);
      uint2 out;
      out.x = quantize_pair(r[i][0], r[i][1], inv) | (quantize_pair(r[i][2], r[i][3], inv) << 16);
      out.y = quantize_pair(r[i][4], r[i][5], inv) | (quantize_pair(r[i][6], r[i][7], inv) << 16);
      reinterpret_cast<uint2*>(q)[static_cast<long long>(t) * n_vec + v] = out;
      if ((threadIdx.x & 15) == 0) scale[static_cast<long long>(v >> 4) * T + t] = s;
    }
  }
}

// Grid-stride over the tokens: a thread keeps its columns, so dweight accumulates in registers over the CTA's tokens and leaves
// as one float32 row of `partial` per CTA.  Fixed order of every sum: two runs give the same bits.
template <typename X, typename R, int VPT>
__global__ void __launch_bounds__(512)
k_add_rms_norm_backward(const uint8_t* grad_y, long long grad_y_pitch, const uint8_t* grad_stream,
                        long long grad_stream_pitch, const uint8_t* stream, long long stream_pitch, const uint8_t* weight,
                        int weight_type, int T, int n_vec, float eps, uint8_t* grad_x, uint8_t* grad_residual,
                        float* partial) {
  __shared__ float s_sum[2][64];
  pdl_launch_dependents();
  pdl_wait();
  float acc[VPT][8];
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = 0.f;
  int parity = 0;
  for (int t = blockIdx.x; t < T; t += gridDim.x, parity ^= 1) {
    Vec8<X> gv[VPT];
    Vec8<R> rv[VPT], ov[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v >= n_vec) continue;
      gv[i] = load_vec8<X>(grad_y + t * grad_y_pitch, v);
      rv[i] = load_vec8<R>(stream + t * stream_pitch, v);
      if (grad_stream) ov[i] = load_vec8<R>(grad_stream + t * grad_stream_pitch, v);
    }
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v >= n_vec) continue;
      float g[8], r[8], w[8];
      unpack_vec8<X>(gv[i], g);
      unpack_vec8<R>(rv[i], r);
      load_vec8_any(weight, v, weight_type, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sum[0] = fmaf(r[j], r[j], sum[0]);
        sum[1] = fmaf(g[j] * w[j], r[j], sum[1]);
      }
    }
    block_sum(sum, s_sum[parity]);
    const float n = static_cast<float>(n_vec * 8);
    const float rstd = __frsqrt_rn(sum[0] / n + eps);
    const float c = rstd * rstd * (sum[1] / n);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v >= n_vec) continue;
      float g[8], r[8], w[8], d[8];
      unpack_vec8<X>(gv[i], g);
      unpack_vec8<R>(rv[i], r);
      load_vec8_any(weight, v, weight_type, w);
      if (grad_stream) unpack_vec8<R>(ov[i], d);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        acc[i][j] = fmaf(g[j], r[j] * rstd, acc[i][j]);
        const float dr = rstd * (g[j] * w[j] - r[j] * c);
        d[j] = grad_stream ? dr + d[j] : dr;
      }
      if (grad_x) store_vec8<X>(grad_x + static_cast<long long>(t) * n_vec * 8 * sizeof(X), v, pack_vec8<X>(d));
      if (grad_residual)
        store_vec8<R>(grad_residual + static_cast<long long>(t) * n_vec * 8 * sizeof(R), v, pack_vec8<R>(d));
    }
  }
  if (!partial) return;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v < n_vec)
      store_vec8<float>(reinterpret_cast<uint8_t*>(partial + static_cast<long long>(blockIdx.x) * n_vec * 8), v,
                        pack_vec8<float>(acc[i]));
  }
}

// dweight[c] = sum of the rows of `partial`, rounded once: 32 columns per CTA, eight warps a row each in turn.
__global__ void __launch_bounds__(256)
k_norm_weight_grad(const float* partial, int rows, int columns, int type, void* grad_weight) {
  __shared__ float s[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  pdl_launch_dependents();
  pdl_wait();
  float sum = 0.f;
  if (c < columns) {
#pragma unroll 8
    for (int r = warp; r < rows; r += 8) sum += ld_dep(partial + static_cast<long long>(r) * columns + c);
  }
  s[warp][lane] = sum;
  __syncthreads();
  if (warp != 0 || c >= columns) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) sum += s[i][lane];
  if (type == B200MOE_DTYPE_F32) {
    static_cast<float*>(grad_weight)[c] = sum;
  } else if (type == B200MOE_DTYPE_F16) {
    static_cast<__half*>(grad_weight)[c] = __float2half_rn(sum);
  } else {
    static_cast<__nv_bfloat16*>(grad_weight)[c] = __float2bfloat16_rn(sum);
  }
}

struct NormShape {
  int n_vec, vpt, threads;
};
static NormShape norm_shape(int columns) {
  NormShape s;
  s.n_vec = columns / 8;
  s.vpt = s.n_vec > 512 ? 4 : s.n_vec > 256 ? 2 : 1;
  s.threads = ((s.n_vec + s.vpt - 1) / s.vpt + 31) / 32 * 32;
  return s;
}

// Calls f with (X tag, R tag, VPT) of the given types; the residual stream has x's type or float32.
template <typename X, typename R, typename F>
static int with_vpt(int vpt, F&& f) {
  if (vpt == 4) return f(X(), R(), std::integral_constant<int, 4>());
  if (vpt == 2) return f(X(), R(), std::integral_constant<int, 2>());
  return f(X(), R(), std::integral_constant<int, 1>());
}
template <typename F>
static int with_types(int x_type, int stream_type, int vpt, F&& f) {
  if (x_type == B200MOE_DTYPE_F32) return with_vpt<float, float>(vpt, f);
  if (x_type == B200MOE_DTYPE_F16)
    return stream_type == x_type ? with_vpt<__half, __half>(vpt, f) : with_vpt<__half, float>(vpt, f);
  return stream_type == x_type ? with_vpt<__nv_bfloat16, __nv_bfloat16>(vpt, f) : with_vpt<__nv_bfloat16, float>(vpt, f);
}

int launch_add_rms_norm(const void* x, long long x_pitch, int x_type, const void* residual, long long residual_pitch,
                        int residual_type, const void* weight, int weight_type, int T, int columns, float eps,
                        void* stream_out, void* y, void* q, float* scale, int num_sms, cudaStream_t st) {
  const NormShape s = norm_shape(columns);
  return with_types(x_type, residual ? residual_type : x_type, s.vpt, [&](auto xt, auto rt, auto vpt) -> int {
    auto kern = k_add_rms_norm<decltype(xt), decltype(rt), decltype(vpt)::value>;
    B200MOE_CUDA_TRY(launch_pdl(kern, dim3(T), dim3(s.threads), 0, st, static_cast<const uint8_t*>(x), x_pitch,
                                static_cast<const uint8_t*>(residual), residual_pitch,
                                static_cast<const uint8_t*>(weight), weight_type, T, s.n_vec, eps,
                                static_cast<uint8_t*>(stream_out), static_cast<uint8_t*>(y), static_cast<uint8_t*>(q),
                                scale));
    return B200MOE_OK;
  });
}

int launch_add_rms_norm_backward(const void* grad_y, long long grad_y_pitch, int type, const void* grad_stream,
                                 long long grad_stream_pitch, const void* stream, long long stream_pitch, int stream_type,
                                 const void* weight, int weight_type, int T, int columns, float eps, void* grad_x,
                                 void* grad_residual, void* grad_weight, float* partial, int num_sms, cudaStream_t st) {
  const NormShape s = norm_shape(columns);
  int ctas = T < B200MOE_NORM_PARTIAL_ROWS ? T : B200MOE_NORM_PARTIAL_ROWS;
  if (ctas > 2 * num_sms) ctas = 2 * num_sms;
  const int rc = with_types(type, stream_type, s.vpt, [&](auto xt, auto rt, auto vpt) -> int {
    auto kern = k_add_rms_norm_backward<decltype(xt), decltype(rt), decltype(vpt)::value>;
    B200MOE_CUDA_TRY(launch_pdl(kern, dim3(ctas), dim3(s.threads), 0, st, static_cast<const uint8_t*>(grad_y),
                                grad_y_pitch, static_cast<const uint8_t*>(grad_stream), grad_stream_pitch,
                                static_cast<const uint8_t*>(stream), stream_pitch, static_cast<const uint8_t*>(weight),
                                weight_type, T, s.n_vec, eps, static_cast<uint8_t*>(grad_x),
                                static_cast<uint8_t*>(grad_residual), grad_weight ? partial : nullptr));
    return B200MOE_OK;
  });
  if (rc || !grad_weight) return rc;
  B200MOE_CUDA_TRY(launch_pdl(k_norm_weight_grad, dim3((columns + 31) / 32), dim3(256), 0, st,
                              static_cast<const float*>(partial), ctas, columns, weight_type, grad_weight));
  return B200MOE_OK;
}

}  // namespace b200moe
