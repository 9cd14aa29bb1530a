// Residual addition + RMS norm, in front of the layer.
//
//   r = round(x + residual)      rstd = 1 / sqrt(mean(r^2) + eps)      y = r * rstd * weight
// r is the residual stream that the next block reads, rounded to its own type, and the norm is taken of the rounded values: y
// then depends on nothing but r, so the backward pass needs no other saved tensor.  y leaves in the type of x and / or as e4m3
// with one float32 scale per token per 128 columns, [H / 128, T], as k_quantize_act writes them, from the float32 y.
//
// Backward, with g = dy * weight and n = H columns:
//   dr = rstd * (g - r * rstd^2 * mean(g * r)) + dr_out       dweight = sum over tokens of dy * r * rstd
// rstd is recomputed: sum(r^2) and sum(g * r) are taken in the same pass over the row.  The second term is taken as
// (r * rstd) * (rstd * (rstd * mean(g * r))): the first factor is of order 1 and the second of the gradient's own size, so
// neither leaves float32 where the result does not (rstd^3 does, for rows of magnitude 1e14 or 1e-13), and dy * (r * rstd)
// likewise.
//
// Sums and statistics are float32: the squares of a row have to add up to less than 3.4e38 (elements of 1e17 do at 7168
// columns).
//
// Bound by the bytes of the rows once the instructions are out of the way: a first form with one float32 operation per
// instruction, predicated vectors and the weight's type looked up at run time issued 31 (forward, e4m3) and 43 (backward) warp
// instructions per element and lane and ran at 5.5 and 3.7 TB/s; paired operations, types as template arguments and rows of
// whole vectors brought 16384 x 7168 bf16 to 124 us with e4m3 out (826 MB: 6.6 TB/s; 132 - 139 in a long run, where the
// clocks settle lower), 137 us with bf16 out (940 MB) and 144 us backward (940 MB and the partial sums).
#include <type_traits>

#include "row_vec.cuh"

namespace b200moe {

constexpr int MAX_WARPS = 16;   // of a CTA

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
// Two sums over the warp for the price of little more than one: after the first exchange lanes 0..15 hold half sums of `a`
// and lanes 16..31 of `b`.  Returns the half-warp's own sum.
__device__ __forceinline__ float warp_sum_halves(float a, float b) {
  const bool upper = threadIdx.x & 16;
  float v = (upper ? b : a) + __shfl_xor_sync(0xffffffffu, upper ? a : b, 16);
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
// The threads of a row: a warp, or a whole number of warps with a barrier of their own (1 + group; 0 is __syncthreads).
__device__ __forceinline__ void row_barrier(int group, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(threads) : "memory");
}
// Sum over the CTA; `s` has MAX_WARPS floats and is not written again before the next barrier.
__device__ __forceinline__ float block_sum(float v, float* s) {
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  v = warp_sum(v);
  if (lane == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = lane < warps ? s[lane] : 0.f;
#pragma unroll
  for (int d = MAX_WARPS / 2; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d, MAX_WARPS);
  return __shfl_sync(0xffffffffu, v, 0);
}

// Largest magnitude; a NaN where there is one.
__device__ __forceinline__ float max_abs_nan(float m, float a) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(m), "f"(fabsf(a)));
  return d;
}

// One pass: a row is read once, kept in registers across the sum, and written.  What hides the latency of a row's load behind
// other rows' stores is several CTAs per SM, not a pipeline inside one.
//
// A row is VPT vectors of eight columns per thread, as many vectors apart as the row has threads, so that a half-warp holds a
// whole 128-column block.  WARP_ROW, where 32 threads are a row: a warp per token, several tokens per CTA, and no barrier; else
// one CTA per token (8192 x 512 bf16, e4m3 out: 9.2 us with a CTA per token, 5.4 with a warp).
template <typename X, typename R, typename W, int VPT, bool WARP_ROW>
__global__ void __launch_bounds__(MAX_WARPS * 32)
k_add_rms_norm(const uint8_t* x, long long x_pitch, const uint8_t* residual, long long residual_pitch,
               const uint8_t* weight, int T, int n_vec, float eps, uint8_t* stream, uint8_t* y, uint8_t* q, float* scale) {
  __shared__ float s_sum[MAX_WARPS];
  const int tid = WARP_ROW ? threadIdx.x & 31 : threadIdx.x, stride = WARP_ROW ? 32 : blockDim.x;
  const int t = WARP_ROW ? blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  if (WARP_ROW && t >= T) return;
  const uint8_t* x_row = x + t * x_pitch;
  const uint8_t* residual_row = residual + t * residual_pitch;
  const long long row = static_cast<long long>(t) * n_vec;   // in vectors, of the dense rows
  Vec8<X> xv[VPT];
  Vec8<R> rv[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = tid + i * stride;
    if (v >= n_vec) continue;
    xv[i] = load_vec8<X>(x_row, v);
    if (residual) rv[i] = load_vec8<R>(residual_row, v);
  }
  float2 r[VPT][4], sum2 = both(0.f);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = tid + i * stride;
    if (v >= n_vec) continue;
    unpack_vec8<X>(xv[i], r[i]);
    if (residual) {
      float2 a[4];
      unpack_vec8<R>(rv[i], a);
#pragma unroll
      for (int j = 0; j < 4; ++j) a[j] = add2(a[j], r[i][j]);
      const Vec8<R> rounded = pack_vec8<R>(a);
      store_vec8<R>(stream + row * 8 * sizeof(R), v, rounded);
      unpack_vec8<R>(rounded, r[i]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) sum2 = fma2(r[i][j], r[i][j], sum2);
  }
  Vec8<W> wv[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = tid + i * stride;
    if (v < n_vec) wv[i] = load_vec8<W>(weight, v);
  }
  const float sum = WARP_ROW ? warp_sum(sum2.x + sum2.y) : block_sum(sum2.x + sum2.y, s_sum);
  const float2 rstd = both(__frsqrt_rn(sum / static_cast<float>(n_vec * 8) + eps));
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = tid + i * stride;
    if (v >= n_vec) continue;
    float2 w[4];
    unpack_vec8<W>(wv[i], w);
#pragma unroll
    for (int j = 0; j < 4; ++j) r[i][j] = mul2(mul2(r[i][j], rstd), w[j]);
    if (y) store_vec8<X>(y + row * 8 * sizeof(X), v, pack_vec8<X>(r[i]));
    if (q) {   // n_vec is a multiple of 16 here: a half-warp is inside the row or outside as a whole
      float m = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) m = max_abs_nan(max_abs_nan(m, r[i][j].x), r[i][j].y);
      // patterns of non-negative floats order like the floats, and a NaN (as max.NaN gives it) is above them all: it then
      // stands in the scale too
      const float amax =
          __uint_as_float(__reduce_max_sync((threadIdx.x & 16) ? 0xffff0000u : 0x0000ffffu, __float_as_uint(m)));
      float s = __fmul_rn(amax, 1.0f / 448.0f);
      if (s < 1e-12f) s = 1e-12f;
      const float inv = __frcp_rn(s);
      uint2 out;
      out.x = quantize_pair(r[i][0].x, r[i][0].y, inv) | (quantize_pair(r[i][1].x, r[i][1].y, inv) << 16);
      out.y = quantize_pair(r[i][2].x, r[i][2].y, inv) | (quantize_pair(r[i][3].x, r[i][3].y, inv) << 16);
      reinterpret_cast<uint2*>(q)[row + v] = out;
      if ((tid & 15) == 0) scale[static_cast<long long>(v >> 4) * T + t] = s;
    }
  }
}

// A CTA works on `groups` tokens at a time, `row_threads` threads each (narrow rows: several; wide rows: one), grid-stride
// over the tokens.  A thread keeps its columns, so dweight accumulates in registers over the CTA's tokens; the groups' sums
// are added in order at the end and leave as one float32 row of `partial` per CTA.  Fixed order of every sum: two runs give
// the same bits.
//
// The rows of a group's next STAGES - 1 tokens are under way in shared memory (16-byte asynchronous copies) while one is worked
// on: a row's two passes (sums, then output) have a sum over its threads between them, in which nothing would be loaded
// otherwise.  A thread copies exactly the pieces that it reads itself, so its own wait orders them and the pipeline needs no
// barrier.  Two stages (a third, measured with one token per CTA before the rest was faster, cost the second CTA per SM:
// 16384 x 7168 bf16 289 us against 209).  One where two rows do not fit, 2 * columns * (sizeof X + sizeof R * (2 with
// grad_stream, else 1)) > MAX_DYNAMIC_SMEM: float32 rows of more than 14464 columns, of more than 9642 with grad_stream, and
// 16-bit rows with a float32 stream and grad_stream of more than 11571.
//
// EXACT: every thread has VPT vectors (7168 columns: 4 x 224 threads), so that no vector is predicated: with the weight kept in
// registers, 8192 x 7168 bf16 94 -> 79 us.
template <typename X, typename R, typename W, int VPT, int STAGES, bool EXACT>
__global__ void __launch_bounds__(MAX_WARPS * 32)
k_add_rms_norm_backward(const uint8_t* grad_y, long long grad_y_pitch, const uint8_t* grad_stream,
                        long long grad_stream_pitch, const uint8_t* stream, long long stream_pitch, const uint8_t* weight,
                        int T, int n_vec, int row_threads, float eps, uint8_t* grad_x, uint8_t* grad_residual,
                        float* partial) {
  extern __shared__ uint4 s_rows[];   // [groups][STAGES][grad_y | stream | grad_stream (if given)]
  __shared__ float s_sum[2][2][MAX_WARPS];
  constexpr int PX = Vec8<X>::PIECES, PR = Vec8<R>::PIECES;
  const int groups = blockDim.x / row_threads, group = threadIdx.x / row_threads;
  const int tid = threadIdx.x - group * row_threads, lane = threadIdx.x & 31;
  const int stage_pieces = n_vec * (PX + PR + (grad_stream ? PR : 0));
  const uint4* rows = s_rows + group * STAGES * stage_pieces;
  const uint32_t base = smem_u32(rows);
  const int step = gridDim.x * groups;
  pdl_launch_dependents();
  pdl_wait();
  auto fetch = [&](int t, int stage) {
    if (t < T) {
      const uint32_t slot = base + stage * stage_pieces * 16;
      const uint8_t* g_row = grad_y + t * grad_y_pitch;
      const uint8_t* r_row = stream + t * stream_pitch;
      const uint8_t* o_row = grad_stream + t * grad_stream_pitch;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int v = tid + i * row_threads;
        if (!EXACT && v >= n_vec) continue;
        copy_vec8<X>(slot, g_row, v);
        copy_vec8<R>(slot + n_vec * PX * 16, r_row, v);
        if (grad_stream) copy_vec8<R>(slot + n_vec * (PX + PR) * 16, o_row, v);
      }
    }
    cp_async_commit();   // a group per token, empty behind the last
  };
  float2 acc[VPT][4];
  Vec8<W> wv[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = both(0.f);
    const int v = tid + i * row_threads;
    if (EXACT || v < n_vec) wv[i] = load_vec8<W>(weight, v);
  }
  const int first = blockIdx.x * groups + group;
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) fetch(first + i * step, i);
  int parity = 0, stage = 0;
  for (int t = first; t < T; t += step, parity ^= 1) {
    fetch(t + (STAGES - 1) * step, stage == 0 ? STAGES - 1 : stage - 1);
    cp_async_wait_group<STAGES - 1>();
    const uint4* slot = rows + stage * stage_pieces;
    stage = stage + 1 == STAGES ? 0 : stage + 1;
    float2 squares = both(0.f), mixed = both(0.f);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = tid + i * row_threads;
      if (!EXACT && v >= n_vec) continue;
      float2 g[4], r[4], w[4];
      unpack_vec8<X>(shared_vec8<X>(slot, v), g);
      unpack_vec8<R>(shared_vec8<R>(slot + n_vec * PX, v), r);
      unpack_vec8<W>(wv[i], w);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        squares = fma2(r[j], r[j], squares);
        mixed = fma2(mul2(g[j], r[j]), w[j], mixed);
      }
    }
    float half = warp_sum_halves(squares.x + squares.y, mixed.x + mixed.y);
    if (row_threads > 32) {
      const int warp = threadIdx.x >> 5, row_warps = row_threads >> 5;
      if ((lane & 15) == 0) s_sum[parity][lane >> 4][warp] = half;
      row_barrier(group, row_threads);
      half = (lane & 15) < row_warps ? s_sum[parity][lane >> 4][group * row_warps + (lane & 15)] : 0.f;
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) half += __shfl_xor_sync(0xffffffffu, half, d);
    }
    const float n = static_cast<float>(n_vec * 8);
    const float rstd1 = __frsqrt_rn(__shfl_sync(0xffffffffu, half, 0) / n + eps);
    const float mean = __shfl_sync(0xffffffffu, half, 16) / n;
    const float2 rstd = both(rstd1), c = both(-(rstd1 * (rstd1 * mean)));
    const long long row = static_cast<long long>(t) * n_vec;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = tid + i * row_threads;
      if (!EXACT && v >= n_vec) continue;
      float2 g[4], r[4], w[4], d[4];
      unpack_vec8<X>(shared_vec8<X>(slot, v), g);
      unpack_vec8<R>(shared_vec8<R>(slot + n_vec * PX, v), r);
      unpack_vec8<W>(wv[i], w);
#pragma unroll
      for (int j = 0; j < 4; ++j) d[j] = both(0.f);
      if (grad_stream) unpack_vec8<R>(shared_vec8<R>(slot + n_vec * (PX + PR), v), d);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        r[j] = mul2(r[j], rstd);
        acc[i][j] = fma2(g[j], r[j], acc[i][j]);
        d[j] = fma2(mul2(g[j], rstd), w[j], fma2(r[j], c, d[j]));
      }
      if (grad_x) store_vec8<X>(grad_x + row * 8 * sizeof(X), v, pack_vec8<X>(d));
      if (grad_residual) store_vec8<R>(grad_residual + row * 8 * sizeof(R), v, pack_vec8<R>(d));
    }
  }
  cp_async_wait_group<0>();
  if (!partial) return;
  if (groups > 1) {   // the rows' space is free behind the barrier: it holds the sums of groups 1, 2, ... (checked by the host)
    __syncthreads();
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = tid + i * row_threads;
      if (group > 0 && v < n_vec) store_shared_vec8<float>(s_rows, (group - 1) * n_vec + v, pack_vec8<float>(acc[i]));
    }
    __syncthreads();
    if (group > 0) return;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = tid + i * row_threads;
      if (v >= n_vec) continue;
      for (int k = 1; k < groups; ++k) {
        float2 more[4];
        unpack_vec8<float>(shared_vec8<float>(s_rows, (k - 1) * n_vec + v), more);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = add2(acc[i][j], more[j]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = tid + i * row_threads;
    if (v < n_vec)
      store_vec8<float>(reinterpret_cast<uint8_t*>(partial + static_cast<long long>(blockIdx.x) * n_vec * 8), v,
                        pack_vec8<float>(acc[i]));
  }
}

// dweight[c] = sum of the rows of `partial`, rounded once: 32 columns per CTA, 16 bytes per lane (four rows a warp and load),
// all of a thread's loads in flight at once.
constexpr int WEIGHT_GRAD_WARPS = 16;
__global__ void __launch_bounds__(WEIGHT_GRAD_WARPS * 32)
k_norm_weight_grad(const float* partial, int rows, int columns, int type, void* grad_weight) {
  __shared__ float4 s[WEIGHT_GRAD_WARPS][8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + (lane & 7) * 4;   // `columns` is a multiple of 8: four columns are inside it or outside
  constexpr int STEP = WEIGHT_GRAD_WARPS * 4, LOADS = B200MOE_NORM_PARTIAL_ROWS / STEP;
  static_assert(LOADS * STEP == B200MOE_NORM_PARTIAL_ROWS, "whole rounds");
  pdl_launch_dependents();
  pdl_wait();
  float4 v[LOADS], sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int r = warp * 4 + (lane >> 3) + i * STEP;
    v[i] = r < rows && c < columns ? ld_dep(reinterpret_cast<const float4*>(partial + static_cast<long long>(r) * columns + c))
                                   : make_float4(0.f, 0.f, 0.f, 0.f);
  }
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    sum.x += v[i].x;
    sum.y += v[i].y;
    sum.z += v[i].z;
    sum.w += v[i].w;
  }
#pragma unroll
  for (int d = 8; d <= 16; d <<= 1) {
    sum.x += __shfl_xor_sync(0xffffffffu, sum.x, d);
    sum.y += __shfl_xor_sync(0xffffffffu, sum.y, d);
    sum.z += __shfl_xor_sync(0xffffffffu, sum.z, d);
    sum.w += __shfl_xor_sync(0xffffffffu, sum.w, d);
  }
  if (lane < 8) s[warp][lane] = sum;
  __syncthreads();
  const int column = blockIdx.x * 32 + lane;
  if (warp != 0 || column >= columns) return;
  float all = 0.f;
#pragma unroll
  for (int i = 0; i < WEIGHT_GRAD_WARPS; ++i) all += reinterpret_cast<const float*>(s[i])[lane];
  if (type == B200MOE_DTYPE_F32) {
    static_cast<float*>(grad_weight)[column] = all;
  } else if (type == B200MOE_DTYPE_F16) {
    static_cast<__half*>(grad_weight)[column] = __float2half_rn(all);
  } else {
    static_cast<__nv_bfloat16*>(grad_weight)[column] = __float2bfloat16_rn(all);
  }
}

constexpr int MAX_DYNAMIC_SMEM = 227 * 1024 - 1024;   // of a CTA, less the static arrays

// Vectors of eight columns per thread.  Forward: few tokens want many threads each (a CTA's latency is the call's), many tokens
// few and fat ones (the row's sum costs per warp).  us with two / four vectors:
//   bf16, e4m3 out, 7168 columns: 1 token 2.35 / 2.89, 700 tokens 8.8 / 9.5, 8192 tokens 66.3 / 64.7, 16384 130 / 124, 8192 without
//   a residual 46 / 40; 2048 columns: 1 token 1.9 / 2.6, 700 tokens 4.2 / 4.7.
// The rule is one for all widths and types, and above 1024 tokens two would be faster outside of wide 16-bit rows: 1100 x
// 7168 bf16 12.1 / 12.9, 8192 x 2048 bf16 19.5 / 20.8, 8192 x 7168 with a float32 stream 95.5 / 97.3, 1100 x 2048 float32 6.2
// / 7.9. Another number of threads adds a row's squares in another order: see the note on batch sizes at add_rms_norm in
// norm.py.
static int forward_vpt(int T, int n_vec) { return n_vec > 1024 || (n_vec > 64 && T > 1024) ? 4 : n_vec > 32 ? 2 : 1; }
// Backward, us with two / four vectors: 8192 tokens of 7168 columns bf16 75.0 / 75.5, f16 91 / 74, bf16 with a float32 stream
// 142 / 156, float32 151 / 163; 6144 columns f16 65.8 / 64.2; 4096 columns bf16 46.4 / 48.0; 2048 columns 25.8 / 27.6; 700
// tokens of 7168 columns bf16 13.5 / 13.2.
static int backward_vpt(bool wide_stream, int n_vec) {
  return n_vec > 1024 || (n_vec > 512 && !wide_stream) ? 4 : n_vec > 32 ? 2 : 1;
}
// Tokens that a CTA of the backward kernel works on at once.  More of them leave fewer rows of partial sums to add (us with
// about 256 / 512 threads per CTA: 8192 x 2048 29.3 / 27.2, 4096 x 7168 45.1 / 42.2, 1000 x 4096 15.2 / 12.5), as long as the
// SMs are evenly used (333 x 7168 7.9 / 9.5: 84 CTAs with four tokens each) and a small batch has a CTA for each token (us
// with one token / 512 threads per CTA: 64 x 512 3.2 / 5.0, 64 x 2048 4.2 / 4.7, 64 x 7168 6.2 / 6.3).  The limit of 64 suits
// wide rows (200 x 4096 6.7 / 6.3, 333 x 2048 5.5 / 4.9); narrow ones would gain from one token per CTA far above it (65 x
// 512 3.3 / 5.1, 1000 x 512 4.7 / 5.3, 2000 x 512 6.2 / 5.6).
static int backward_groups(int T, int row_threads, int num_sms) {
  const int most = MAX_WARPS * 32 / row_threads, half = MAX_WARPS * 16 / row_threads;
  if (T <= 64) return 1;
  if (T < 4 * num_sms && (T + most - 1) / most > num_sms) return half > 1 ? half : 1;
  return most;
}
struct NormShape {
  int n_vec, vpt, threads;   // threads: of a row
};
static NormShape norm_shape(int columns, int vpt) {
  NormShape s;
  s.n_vec = columns / 8;
  s.vpt = vpt;
  s.threads = ((s.n_vec + vpt - 1) / vpt + 31) / 32 * 32;
  return s;
}

// Calls f with tags of the types and VPT.  The residual stream and the weight have x's type or float32.
template <typename X, typename R, typename W, typename F>
static int with_vpt(int vpt, F&& f) {
  if (vpt == 4) return f(X(), R(), W(), std::integral_constant<int, 4>());
  if (vpt == 2) return f(X(), R(), W(), std::integral_constant<int, 2>());
  return f(X(), R(), W(), std::integral_constant<int, 1>());
}
template <typename X, typename F>
static int with_16_bit(bool wide_stream, bool wide_weight, int vpt, F&& f) {
  if (wide_stream) return wide_weight ? with_vpt<X, float, float>(vpt, f) : with_vpt<X, float, X>(vpt, f);
  return wide_weight ? with_vpt<X, X, float>(vpt, f) : with_vpt<X, X, X>(vpt, f);
}
template <typename F>
static int with_types(int x_type, int stream_type, int weight_type, int vpt, F&& f) {
  const bool wide_stream = stream_type == B200MOE_DTYPE_F32, wide_weight = weight_type == B200MOE_DTYPE_F32;
  if (x_type == B200MOE_DTYPE_F32) return with_vpt<float, float, float>(vpt, f);
  if (x_type == B200MOE_DTYPE_F16) return with_16_bit<__half>(wide_stream, wide_weight, vpt, f);
  return with_16_bit<__nv_bfloat16>(wide_stream, wide_weight, vpt, f);
}

int launch_add_rms_norm(const void* x, long long x_pitch, int x_type, const void* residual, long long residual_pitch,
                        int residual_type, const void* weight, int weight_type, int T, int columns, float eps,
                        void* stream_out, void* y, void* q, float* scale, cudaStream_t st) {
  const NormShape s = norm_shape(columns, forward_vpt(T, columns / 8));
  return with_types(x_type, residual ? residual_type : x_type, weight_type, s.vpt,
                    [&](auto xt, auto rt, auto wt, auto vpt) -> int {
    using X = decltype(xt);
    using R = decltype(rt);
    using W = decltype(wt);
    constexpr int VPT = decltype(vpt)::value;
    constexpr int ROWS = 4;   // of a CTA where a warp has a row to itself
    const bool warp_row = s.threads == 32;
    auto kern = warp_row ? k_add_rms_norm<X, R, W, VPT, true> : k_add_rms_norm<X, R, W, VPT, false>;
    B200MOE_CUDA_TRY(launch_pdl(kern, dim3(warp_row ? (T + ROWS - 1) / ROWS : T), dim3(warp_row ? 32 * ROWS : s.threads), 0,
                                st, static_cast<const uint8_t*>(x), x_pitch, static_cast<const uint8_t*>(residual),
                                residual_pitch, static_cast<const uint8_t*>(weight), T, s.n_vec, eps,
                                static_cast<uint8_t*>(stream_out), static_cast<uint8_t*>(y), static_cast<uint8_t*>(q),
                                scale));
    return B200MOE_OK;
  });
}

int launch_add_rms_norm_backward(const void* grad_y, long long grad_y_pitch, int type, const void* grad_stream,
                                 long long grad_stream_pitch, const void* stream, long long stream_pitch, int stream_type,
                                 const void* weight, int weight_type, int T, int columns, float eps, void* grad_x,
                                 void* grad_residual, void* grad_weight, float* partial, int num_sms, cudaStream_t st) {
  const NormShape s = norm_shape(columns, backward_vpt(stream_type == B200MOE_DTYPE_F32, columns / 8));
  int ctas = 0;
  const int rc = with_types(type, stream_type, weight_type, s.vpt, [&](auto xt, auto rt, auto wt, auto vpt) -> int {
    using X = decltype(xt);
    using R = decltype(rt);
    using W = decltype(wt);
    constexpr int VPT = decltype(vpt)::value;
    const size_t stage = static_cast<size_t>(columns) * (sizeof(X) + sizeof(R) * (grad_stream ? 2 : 1));
    int groups = backward_groups(T, s.threads, num_sms);
    while (groups > 1 && 2 * stage * groups > static_cast<size_t>(MAX_DYNAMIC_SMEM)) --groups;
    auto launch = [&](auto stages, auto is_exact) -> int {
      auto kern = k_add_rms_norm_backward<X, R, W, VPT, decltype(stages)::value, decltype(is_exact)::value>;
      const size_t smem = stage * stages * groups;
      static_assert(sizeof(X) + sizeof(R) >= 4, "two stages of a row hold its columns in float32: the groups' sums fit");
      // this kernel's last answer to this thread is kept (a lambda of its own, and so a variable, for each pair of tags): the
      // two calls take microseconds
      static thread_local struct {
        int device = -1, threads = 0, per_sm = 0;
        size_t smem = 0;
      } known;
      int device = 0;
      B200MOE_CUDA_TRY(cudaGetDevice(&device));
      if (known.device != device || known.threads != s.threads * groups || known.smem != smem) {
        known.device = -1;
        B200MOE_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_DYNAMIC_SMEM));
        B200MOE_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&known.per_sm, kern, s.threads * groups, smem));
        known.device = device;
        known.threads = s.threads * groups;
        known.smem = smem;
      }
      int most = num_sms * (known.per_sm > 0 ? known.per_sm : 1);
      if (most > B200MOE_NORM_PARTIAL_ROWS) most = B200MOE_NORM_PARTIAL_ROWS;
      const int batches = (T + groups - 1) / groups;
      const int rounds = (batches + most - 1) / most;   // of the busiest CTA; no more CTAs than that takes
      ctas = (batches + rounds - 1) / rounds;
      B200MOE_CUDA_TRY(launch_pdl(kern, dim3(ctas), dim3(s.threads * groups), smem, st, static_cast<const uint8_t*>(grad_y),
                                  grad_y_pitch, static_cast<const uint8_t*>(grad_stream), grad_stream_pitch,
                                  static_cast<const uint8_t*>(stream), stream_pitch,
                                  static_cast<const uint8_t*>(weight), T, s.n_vec, s.threads, eps,
                                  static_cast<uint8_t*>(grad_x), static_cast<uint8_t*>(grad_residual),
                                  grad_weight ? partial : nullptr));
      return B200MOE_OK;
    };
    const bool exact = s.n_vec == VPT * s.threads;
    if (2 * stage * groups <= static_cast<size_t>(MAX_DYNAMIC_SMEM))
      return exact ? launch(std::integral_constant<int, 2>(), std::true_type())
                   : launch(std::integral_constant<int, 2>(), std::false_type());
    return launch(std::integral_constant<int, 1>(), std::false_type());
  });
  if (rc || !grad_weight) return rc;
  B200MOE_CUDA_TRY(launch_pdl(k_norm_weight_grad, dim3((columns + 31) / 32), dim3(WEIGHT_GRAD_WARPS * 32), 0, st,
                              static_cast<const float*>(partial), ctas, columns, weight_type, grad_weight));
  return B200MOE_OK;
}

}  // namespace b200moe
