// Rows of bf16, f16 or f32 elements in 16-byte pieces: loads below the dependency wait, conversion to float32 and back (round
// to nearest even), stores.  Used by the norm and token-permutation kernels, which take the element type as a template
// argument.
//
// Values are held and computed in pairs: sm_100 multiplies, adds and fuses two float32 per instruction, each rounded as by
// itself.  The kernels here stream rows at the memory's rate, where issue slots are what runs out next.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace b200moe {

__device__ __forceinline__ unsigned long long pair_bits(float2 a) { return *reinterpret_cast<unsigned long long*>(&a); }
__device__ __forceinline__ float2 bits_pair(unsigned long long a) { return *reinterpret_cast<float2*>(&a); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(pair_bits(a)), "l"(pair_bits(b)), "l"(pair_bits(c)));
  return bits_pair(d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(pair_bits(a)), "l"(pair_bits(b)));
  return bits_pair(d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(pair_bits(a)), "l"(pair_bits(b)));
  return bits_pair(d);
}
__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }

template <typename T>
constexpr int PIECE_PAIRS = 8 / static_cast<int>(sizeof(T));   // pairs of elements in a 16-byte piece: 4, or 2 of float32

template <typename T>
__device__ __forceinline__ void unpack_piece(const uint4& raw, float2 (&f)[PIECE_PAIRS<T>]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 2; ++j) f[j] = make_float2(__uint_as_float(w[2 * j]), __uint_as_float(w[2 * j + 1]));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (__is_same(T, __nv_bfloat16))
        f[j] = make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
      else
        f[j] = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
    }
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack_piece(const float2 (&f)[PIECE_PAIRS<T>]) {
  uint32_t w[4];
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      w[2 * j] = __float_as_uint(f[j].x);
      w[2 * j + 1] = __float_as_uint(f[j].y);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (__is_same(T, __nv_bfloat16)) {
        const __nv_bfloat162 b = __float22bfloat162_rn(f[j]);
        w[j] = *reinterpret_cast<const uint32_t*>(&b);
      } else {
        const __half2 b = __float22half2_rn(f[j]);
        w[j] = *reinterpret_cast<const uint32_t*>(&b);
      }
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Eight consecutive elements (one or two pieces), the unit of a thread in the norm kernels: element 8 * v of the row at `row`.
template <typename T>
struct Vec8 {
  static constexpr int PIECES = sizeof(T) / 2;
  uint4 p[PIECES];
};
template <typename T>
__device__ __forceinline__ Vec8<T> load_vec8(const uint8_t* row, int v) {
  Vec8<T> r;
#pragma unroll
  for (int i = 0; i < Vec8<T>::PIECES; ++i) r.p[i] = ld_dep(reinterpret_cast<const uint4*>(row) + v * Vec8<T>::PIECES + i);
  return r;
}
template <typename T>
__device__ __forceinline__ void unpack_vec8(const Vec8<T>& r, float2 (&f)[4]) {
  constexpr int N = PIECE_PAIRS<T>;
#pragma unroll
  for (int i = 0; i < Vec8<T>::PIECES; ++i) {
    float2 g[N];
    unpack_piece<T>(r.p[i], g);
#pragma unroll
    for (int j = 0; j < N; ++j) f[i * N + j] = g[j];
  }
}
template <typename T>
__device__ __forceinline__ Vec8<T> pack_vec8(const float2 (&f)[4]) {
  constexpr int N = PIECE_PAIRS<T>;
  Vec8<T> r;
#pragma unroll
  for (int i = 0; i < Vec8<T>::PIECES; ++i) {
    float2 g[N];
#pragma unroll
    for (int j = 0; j < N; ++j) g[j] = f[i * N + j];
    r.p[i] = pack_piece<T>(g);
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void store_vec8(uint8_t* row, int v, const Vec8<T>& r) {
#pragma unroll
  for (int i = 0; i < Vec8<T>::PIECES; ++i) reinterpret_cast<uint4*>(row)[v * Vec8<T>::PIECES + i] = r.p[i];
}
// The same through shared memory: an asynchronous copy into it, a store, a read.
template <typename T>
__device__ __forceinline__ void copy_vec8(uint32_t slot, const uint8_t* row, int v) {
#pragma unroll
  for (int i = 0; i < Vec8<T>::PIECES; ++i) {
    const int at = (v * Vec8<T>::PIECES + i) * 16;
    cp_async16(slot + at, row + at);
  }
}
template <typename T>
__device__ __forceinline__ void store_shared_vec8(uint4* slot, int v, const Vec8<T>& r) {
#pragma unroll
  for (int i = 0; i < Vec8<T>::PIECES; ++i) slot[v * Vec8<T>::PIECES + i] = r.p[i];
}
template <typename T>
__device__ __forceinline__ Vec8<T> shared_vec8(const uint4* slot, int v) {
  Vec8<T> r;
#pragma unroll
  for (int i = 0; i < Vec8<T>::PIECES; ++i) r.p[i] = slot[v * Vec8<T>::PIECES + i];
  return r;
}

}  // namespace b200moe
