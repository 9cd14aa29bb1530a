// Rows of bf16, f16 or f32 elements in 16-byte pieces: loads below the dependency wait, conversion to float32 and back (round to
// nearest even), stores.  Used by the norm and token-permutation kernels, which take the element type as a template argument.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace b200moe {

template <typename T>
constexpr int PIECE_ELEMS = 16 / static_cast<int>(sizeof(T));   // elements of a 16-byte piece: 8, or 4 of float32

template <typename T>
__device__ __forceinline__ void unpack_piece(const uint4& raw, float (&f)[PIECE_ELEMS<T>]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = __uint_as_float(w[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 2 && __is_same(T, __nv_bfloat16)) {
        f[2 * j] = __uint_as_float(w[j] << 16);
        f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      } else {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        f[2 * j] = v.x;
        f[2 * j + 1] = v.y;
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack_piece(const float (&f)[PIECE_ELEMS<T>]) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (sizeof(T) == 4) {
      w[j] = __float_as_uint(f[j]);
    } else if constexpr (__is_same(T, __nv_bfloat16)) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&b);
    } else {
      const __half2 b = __floats2half2_rn(f[2 * j], f[2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&b);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Eight consecutive elements (one or two pieces), the unit of a thread in the norm kernels: element 8 * v of the row at `row`.
template <typename T>
struct Vec8 {
  uint4 p[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Vec8<T> load_vec8(const uint8_t* row, int v) {
  Vec8<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
    r.p[i] = ld_dep(reinterpret_cast<const uint4*>(row) + v * (sizeof(T) / 2) + i);
  return r;
}
template <typename T>
__device__ __forceinline__ void unpack_vec8(const Vec8<T>& r, float (&f)[8]) {
  constexpr int N = PIECE_ELEMS<T>;
#pragma unroll
  for (int i = 0; i < 8 / N; ++i) {
    float g[N];
    unpack_piece<T>(r.p[i], g);
#pragma unroll
    for (int j = 0; j < N; ++j) f[i * N + j] = g[j];
  }
}
template <typename T>
__device__ __forceinline__ Vec8<T> pack_vec8(const float (&f)[8]) {
  constexpr int N = PIECE_ELEMS<T>;
  Vec8<T> r;
#pragma unroll
  for (int i = 0; i < 8 / N; ++i) {
    float g[N];
#pragma unroll
    for (int j = 0; j < N; ++j) g[j] = f[i * N + j];
    r.p[i] = pack_piece<T>(g);
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void store_vec8(uint8_t* row, int v, const Vec8<T>& r) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) reinterpret_cast<uint4*>(row)[v * (sizeof(T) / 2) + i] = r.p[i];
}
// Eight elements of a type known at run time only (the norm's weight: small, shared by all rows, in L1 or L2).
__device__ __forceinline__ void load_vec8_any(const uint8_t* row, int v, int type, float (&f)[8]) {
  if (type == B200MOE_DTYPE_F32) {
    unpack_vec8<float>(load_vec8<float>(row, v), f);
  } else if (type == B200MOE_DTYPE_F16) {
    unpack_vec8<__half>(load_vec8<__half>(row, v), f);
  } else {
    unpack_vec8<__nv_bfloat16>(load_vec8<__nv_bfloat16>(row, v), f);
  }
}

}  // namespace b200moe
