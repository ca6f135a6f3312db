// The K/V cache held in 4 bits: rows in, rows out.
//
// A group of 64 head dims of a row x: m = min(x), s = fp16((max(x) - m) / 15), code n = round((x - m) / s) in
// [0, 15] (ties to even; 0 where s = 0); it stands for fp16(s n + m). m is one of the inputs, hence exact in
// fp16. Every step but the roundings named is in fp32.
//
// The bound is HBM: 2 D bytes in and D / 2 + D / 16 out a row, or the reverse. 8 lanes take a group, each the 16
// bytes of 8 dims, which are 4 bytes of codes.
#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.h"

namespace tattn {
namespace {

constexpr int kThreads = 256;

// This thread's 8 dims: dims [8 i, 8 i + 8) of row t of head hk of sequence z, and the cache's row for them (or
// -1: none, the position lies outside the cache). kv: 0 keys, 1 values.
struct Place {
  int kv, z, hk, t, i;
  int64_t row;
};
template <int D>
__device__ __forceinline__ bool place(const Int4CacheArgs& a, Place* p) {
  constexpr int L = D / 8;
  const int64_t id = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  int64_t r = id / L;
  p->i = int(id % L);
  p->t = int(r % a.T);
  r /= a.T;
  p->hk = int(r % a.Hk);
  r /= a.Hk;
  p->z = int(r % a.Z);
  p->kv = int(r / a.Z);
  if (p->kv > 1) return false;
  const int64_t pos = int64_t(a.start ? a.start[p->z] : 0) + p->t;
  p->row = pos >= 0 && pos < a.C ? (int64_t(p->z) * a.Hk + p->hk) * a.C + pos : -1;
  return true;
}

template <int D>
__global__ void __launch_bounds__(kThreads) int4_append_kernel(const Int4CacheArgs a) {
  Place p;
  bool any = place<D>(a, &p);
  if (any && a.counts && p.t >= a.counts[p.z]) any = false;
  if (any && p.row < 0) {
    if (p.i == 0) atomicOr(a.status, kStatusIndexRange);
    any = false;
  }
  float x[8];
  if (any) {
    const Strides3 s = p.kv ? a.sv : a.sk;
    const __half* src = static_cast<const __half*>(p.kv ? a.v : a.k) + p.z * s.z + p.hk * s.h + p.t * s.n + 8 * p.i;
    const uint4 u = *reinterpret_cast<const uint4*>(src);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
      x[2 * e] = f.x;
      x[2 * e + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.f;
  }
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) {
    lo = fminf(lo, x[e]);
    hi = fmaxf(hi, x[e]);
  }
#pragma unroll
  for (int o = 1; o < 8; o *= 2) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  if (!any) return;
  const __half scale = __float2half_rn((hi - lo) / 15.f);
  const float s = __half2float(scale);
  uint32_t code = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float n = s > 0.f ? fminf(fmaxf(rintf((x[e] - lo) / s), 0.f), 15.f) : 0.f;
    code |= uint32_t(n) << (4 * e);
  }
  *reinterpret_cast<uint32_t*>((p.kv ? a.v_codes : a.k_codes) + p.row * (D / 2) + 4 * p.i) = code;
  if (p.i % 8 == 0)
    static_cast<__half2*>(p.kv ? a.v_params : a.k_params)[p.row * (D / 64) + p.i / 8] =
        __halves2half2(scale, __float2half_rn(lo));
}

template <int D>
__global__ void __launch_bounds__(kThreads) int4_read_kernel(const Int4CacheArgs a) {
  Place p;
  if (!place<D>(a, &p)) return;
  uint32_t w[4] = {0u, 0u, 0u, 0u};  // a position outside the cache reads as zeros
  if (p.row >= 0) {
    const uint32_t code = *reinterpret_cast<const uint32_t*>((p.kv ? a.v_codes : a.k_codes) + p.row * (D / 2) + 4 * p.i);
    const __half2 sm = static_cast<const __half2*>(p.kv ? a.v_params : a.k_params)[p.row * (D / 64) + p.i / 8];
    const __half2 s = __low2half2(sm), m = __high2half2(sm);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const __half2 n = __floats2half2_rn(float((code >> (8 * e)) & 15u), float((code >> (8 * e + 4)) & 15u));
      const __half2 v = __hfma2(s, n, m);  // one rounding
      w[e] = *reinterpret_cast<const uint32_t*>(&v);
    }
  } else if (p.i == 0) {
    atomicOr(a.status, kStatusIndexRange);
  }
  const int64_t row = (int64_t(p.z) * a.Hk + p.hk) * a.T + p.t;
  *reinterpret_cast<uint4*>(static_cast<__half*>(p.kv ? a.v_out : a.k_out) + row * D + 8 * p.i) =
      make_uint4(w[0], w[1], w[2], w[3]);
}

// One thread for each 8 dims of K and V.
cudaError_t grid_for(int D, const Int4CacheArgs& a, unsigned* grid) {
  const double blocks = 2.0 * a.Z * a.Hk * a.T * (D / 8) / kThreads + 1.0;
  if (blocks > 2147483647.0) return cudaErrorInvalidConfiguration;
  *grid = unsigned((2 * int64_t(a.Z) * a.Hk * a.T * (D / 8) + kThreads - 1) / kThreads);
  return cudaSuccess;
}

}  // namespace

cudaError_t launch_int4_append(int D, const Int4CacheArgs& a, cudaStream_t s) {
  unsigned grid;
  const cudaError_t e = grid_for(D, a, &grid);
  if (e != cudaSuccess || grid == 0) return e;
  if (D == 64)
    int4_append_kernel<64><<<grid, kThreads, 0, s>>>(a);
  else
    int4_append_kernel<128><<<grid, kThreads, 0, s>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_int4_read(int D, const Int4CacheArgs& a, cudaStream_t s) {
  unsigned grid;
  const cudaError_t e = grid_for(D, a, &grid);
  if (e != cudaSuccess || grid == 0) return e;
  if (D == 64)
    int4_read_kernel<64><<<grid, kThreads, 0, s>>>(a);
  else
    int4_read_kernel<128><<<grid, kThreads, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace tattn
