// The K/V cache held in 4 bits: rows in, rows out.
//
// A group of 64 head dims of a row x: m = min(x), s = fp16((max(x) - m) / 15), code n = round((x - m) / s) in
// [0, 15] (ties to even; 0 where s = 0); it stands for fp16(s n + m). m is one of the inputs, hence exact in
// fp16. Where s rounded up would make 15 s + m infinite, s is rounded down. Every step but the roundings named is in
// fp32. A group with a NaN or an infinity has no range: its scale is NaN, and all of it reads as NaN. (The two rules cost
// append 0.5 us of the 17.5 below.)
//
// A row is 2 D bytes in and D / 2 + D / 16 out, or the reverse; what bounds both kernels is the conversions in between
// (append: issue slots 80 % busy; read: the ALU pipe 73 %), then a launch's start and end. 8 lanes take a group, each the 16
// bytes of 8 dims, which are 4 bytes of codes. A CTA works on one head of one sequence of K or V, and a thread
// on the same dims of up to kRows rows, all of whose loads it issues first; so the divisions that find the
// head are done once, for the whole CTA.
//
// Measured (B200): 4 sequences of 4,096 tokens, 4 heads of 128, K and V (33.5 MB in fp16, 9.4 MB in 4 bits), passes over 8
// sets of them: append 17.5 us, 2.5 TB/s; read 11.0 us, 3.9 TB/s. HBM would take 6.7 us for either.
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"
#include "kernels.h"

namespace tattn {
namespace {

constexpr int kThreads = 256, kRows = 4;

// A NaN on either side is the result (fminf gives the other side), as of max_or_nan.
__device__ __forceinline__ float min_or_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// This thread's work: dims [8 i, 8 i + 8) of rows t, t + step, ... (kRows of them, below T) of head hk of
// sequence z. kv: 0 keys, 1 values.
struct Place {
  int kv, z, hk, t, step, i;
  int64_t head, start;  // the cache's head; the position of row 0
};
template <int D>
__device__ __forceinline__ Place place(const Int4CacheArgs& a) {
  constexpr int L = D / 8;
  const int rows = int(blockDim.x) / L, chunks = (a.T + kRows * rows - 1) / (kRows * rows);
  Place p;
  int head = int(blockIdx.x) / chunks;
  p.step = rows;
  p.t = int(blockIdx.x) % chunks * kRows * rows + int(threadIdx.x) / L;
  p.i = int(threadIdx.x) % L;
  p.hk = head % a.Hk;
  head /= a.Hk;
  p.z = head % a.Z;
  p.kv = head / a.Z;
  p.head = int64_t(p.z) * a.Hk + p.hk;
  p.start = a.start ? a.start[p.z] : 0;
  return p;
}
// The cache's row for row t, or -1: its position lies outside the cache.
__device__ __forceinline__ int64_t cache_row(const Int4CacheArgs& a, const Place& p, int t) {
  const int64_t pos = p.start + t;
  return pos >= 0 && pos < a.C ? p.head * a.C + pos : -1;
}

template <int D>
__global__ void __launch_bounds__(kThreads) int4_append_kernel(const Int4CacheArgs a) {
  const Place p = place<D>(a);
  const int T = a.counts ? min(a.T, a.counts[p.z]) : a.T;
  const Strides3 st = p.kv ? a.sv : a.sk;
  const __half* src = static_cast<const __half*>(p.kv ? a.v : a.k) + p.z * st.z + p.hk * st.h + 8 * p.i;
  uint8_t* codes = p.kv ? a.v_codes : a.k_codes;
  __half2* params = static_cast<__half2*>(p.kv ? a.v_params : a.k_params);
  uint4 u[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int t = p.t + r * p.step;
    u[r] = t < T ? *reinterpret_cast<const uint4*>(src + t * st.n) : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int t = p.t + r * p.step;
    const uint32_t w[4] = {u[r].x, u[r].y, u[r].z, u[r].w};
    float x[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
      x[2 * e] = f.x;
      x[2 * e + 1] = f.y;
    }
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) {
      lo = min_or_nan(lo, x[e]);
      hi = max_or_nan(hi, x[e]);
    }
#pragma unroll
    for (int o = 1; o < 8; o *= 2) {
      lo = min_or_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = max_or_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    if (t >= T) continue;
    const int64_t row = cache_row(a, p, t);
    if (row < 0) {
      if (p.i == 0) atomicOr(a.status, kStatusIndexRange);
      continue;
    }
    const float range = hi - lo;  // infinite or NaN where a value is
    const float step = range < INFINITY ? range / 15.f : NAN;
    __half scale = __float2half_rn(step);
    // A step rounded up may take the largest code's value past fp16 (65520 rounds to infinity); rounded down it cannot.
    if (fmaf(15.f, __half2float(scale), lo) >= 65520.f) scale = __float2half_rd(step);
    const float s = __half2float(scale);
    // The quotient (x - lo) / s, correctly rounded, by Markstein's theorem: with inv the correctly rounded 1 /
    // s and q0 = d inv, the remainder d - q0 s is exact in one FMA and q0 + remainder * inv rounds to the quotient.
    // (Eight divisions took two thirds of the kernel's time.) Adding 1.5 2^23 rounds it to the nearest integer,
    // ties to even, in the low bits.
    const float inv = s > 0.f ? __frcp_rn(s) : 0.f;
    uint32_t code = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = x[e] - lo, q0 = d * inv;
      const float q = fminf(fmaf(fmaf(-q0, s, d), inv, q0), 15.f);
      code |= (__float_as_uint(q + 12582912.f) & 15u) << (4 * e);
    }
    *reinterpret_cast<uint32_t*>(codes + row * (D / 2) + 4 * p.i) = code;
    if (p.i % 8 == 0) params[row * (D / 64) + p.i / 8] = __halves2half2(scale, __float2half_rn(lo));
  }
}

template <int D>
__global__ void __launch_bounds__(kThreads) int4_read_kernel(const Int4CacheArgs a) {
  const Place p = place<D>(a);
  const uint8_t* codes = p.kv ? a.v_codes : a.k_codes;
  const __half2* params = static_cast<const __half2*>(p.kv ? a.v_params : a.k_params);
  __half* out = static_cast<__half*>(p.kv ? a.v_out : a.k_out) + p.head * a.T * D + 8 * p.i;
  uint32_t code[kRows];
  __half2 sm[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {  // a position outside the cache reads as zeros
    const int t = p.t + r * p.step;
    const int64_t row = t < a.T ? cache_row(a, p, t) : 0;
    const bool in = t < a.T && row >= 0;
    code[r] = in ? *reinterpret_cast<const uint32_t*>(codes + row * (D / 2) + 4 * p.i) : 0u;
    sm[r] = in ? params[row * (D / 64) + p.i / 8] : __float2half2_rn(0.f);
    if (row < 0 && p.i == 0) atomicOr(a.status, kStatusIndexRange);
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int t = p.t + r * p.step;
    if (t >= a.T) break;
    const __half2 s = __low2half2(sm[r]), m = __high2half2(sm[r]);
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const __half2 n = __floats2half2_rn(float((code[r] >> (8 * e)) & 15u), float((code[r] >> (8 * e + 4)) & 15u));
      const __half2 v = __hfma2(s, n, m);  // one rounding
      w[e] = *reinterpret_cast<const uint32_t*>(&v);
    }
    *reinterpret_cast<uint4*>(out + int64_t(t) * D) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <typename Kernel>
cudaError_t launch(Kernel kernel, int D, const Int4CacheArgs& a, cudaStream_t s) {
  // Fewer threads where all the rows of a head need fewer (whole warps).
  const int64_t need = (int64_t(a.T) * (D / 8) + 31) / 32 * 32;
  const int threads = need < kThreads ? int(need) : kThreads, rows = threads / (D / 8);
  const int64_t chunks = (a.T + int64_t(kRows) * rows - 1) / (kRows * rows);
  if (double(chunks) * 2.0 * a.Z * a.Hk > 2147483647.0) return cudaErrorInvalidConfiguration;
  const int64_t grid = chunks * 2 * a.Z * a.Hk;
  if (grid == 0) return cudaSuccess;
  kernel<<<unsigned(grid), threads, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_int4_append(int D, const Int4CacheArgs& a, cudaStream_t s) {
  return D == 64 ? launch(int4_append_kernel<64>, D, a, s) : launch(int4_append_kernel<128>, D, a, s);
}

cudaError_t launch_int4_read(int D, const Int4CacheArgs& a, cudaStream_t s) {
  return D == 64 ? launch(int4_read_kernel<64>, D, a, s) : launch(int4_read_kernel<128>, D, a, s);
}

}  // namespace tattn
