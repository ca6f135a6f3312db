// What the kernels of head norms and rotations (norm_rope.cu, rope_axes.cu) share: rows of T in 16-byte units, a lane's pairs.
#pragma once

#include "common.cuh"

namespace tattn {

template <typename T>
constexpr int kVec = 16 / int(sizeof(T));

// 16 bytes of T as floats, and back (rounded to nearest).
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& v, float* x) {
  if constexpr (sizeof(T) == 2) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  } else {
    x[0] = __uint_as_float(v.x);
    x[1] = __uint_as_float(v.y);
    x[2] = __uint_as_float(v.z);
    x[3] = __uint_as_float(v.w);
  }
}
template <typename T>
__device__ __forceinline__ uint4 load_raw(const T* p) {
  return *reinterpret_cast<const uint4*>(p);
}
template <typename T>
__device__ __forceinline__ void load16(const T* p, float* x) {
  unpack16<T>(load_raw(p), x);
}
template <typename T>
__device__ __forceinline__ void store16(T* p, const float* x) {
  if constexpr (sizeof(T) == 2)
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]), pack_half2(x[4], x[5]),
                                              pack_half2(x[6], x[7]));
  else
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
}

// N consecutive floats (N = 2, 4 or 8; aligned to their size, at most 16 bytes).
template <int N>
__device__ __forceinline__ void load_floats(const float* p, float* x) {
  if constexpr (N == 2) {
    const float2 v = *reinterpret_cast<const float2*>(p);
    x[0] = v.x;
    x[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + i);
      x[i] = v.x;
      x[i + 1] = v.y;
      x[i + 2] = v.z;
      x[i + 3] = v.w;
    }
  }
}

// Sum over the L lanes of a group (L a power of two, groups aligned in the warp).
template <int L>
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
  for (int o = L / 2; o > 0; o /= 2) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// The lane's 2 VEC values of a row as VEC pairs: value e of the first 16 bytes pairs with value e of the
// second (half-split), or neighbours pair, those of the second 16 bytes after those of the first
// (interleaved). first(j), second(j): where pair j's two values are.
template <int VEC, bool INTERLEAVED>
struct Pairs {
  static __device__ __forceinline__ constexpr int first(int j) { return INTERLEAVED ? 2 * j : j; }
  static __device__ __forceinline__ constexpr int second(int j) { return INTERLEAVED ? 2 * j + 1 : VEC + j; }
};

}  // namespace tattn
