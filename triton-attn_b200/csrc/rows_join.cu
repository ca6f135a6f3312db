// Joins the parts of query rows whose keys were cut into several (RowsArgs): O = sum of 2^(m_i - m) O_i over sum of
// 2^(m_i - m) l_i, m the largest of the parts' maxima.
//
// A CTA takes one row, its threads 4 dims of every so many-th part. The parts were just written, so they come from L2; what
// bounds it is its launch and the loads' latency, so it is launched while the last parts are made, and a thread's first
// loads do not wait for the maximum. What it adds to a call (B200, 1,024 rows, the calls with and without it): 18 parts of 64
// dims 3.2 us, 39 parts of 128 9.0 us.
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <math.h>

#include "common.cuh"
#include "kernels.h"

namespace tattn {
namespace {

constexpr int kThreads = 128;

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) rows_join_kernel(const JoinArgs a) {
  constexpr int V = D / 4, LANES = kThreads / V;  // threads of a row, parts in flight
  __shared__ float4 so[LANES][V];
  __shared__ float sl[LANES];
  const int64_t index = blockIdx.x;
  const int head = int(index / a.N), row = int(index % a.N), z = head / a.H, h = head % a.H;
  const int outer = row / a.inner, in = row - outer * a.inner;
  const int64_t rows[2] = {index, z * a.other.z + h * a.other.h + outer * a.other.outer + in * a.other.in};
  const int t = threadIdx.x % V, p = threadIdx.x / V, total = a.n[0] + a.n[1];
  // Part s of both lists: its maximum and sum, and this thread's dims.
  auto part_ml = [&](int s) {
    const bool second = s >= a.n[0];
    const int64_t at = second ? rows[1] * a.n[1] + s - a.n[0] : rows[0] * a.n[0] + s;
    return __ldcg(reinterpret_cast<const float2*>(a.part_ml[second]) + at);
  };
  auto part_row = [&](int s) {
    const bool second = s >= a.n[0];
    const int64_t at = second ? rows[1] * a.n[1] + s - a.n[0] : rows[0] * a.n[0] + s;
    return __ldcg(reinterpret_cast<const float4*>(a.part[second]) + at * V + t);
  };
  wait_for_last_kernel();
  // The thread's first parts on their way before the maximum is known. (What stands in the row of a part without keys is
  // read and not used.)
  constexpr int AHEAD = 4;
  float2 c[AHEAD];
  float4 v[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    const int s = p + i * LANES;
    c[i] = make_float2(-INFINITY, 0.f);
    v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (s < total) {
      c[i] = part_ml(s);
      v[i] = part_row(s);
    }
  }
  float m = -INFINITY;
  for (int s = threadIdx.x % 32; s < total; s += 32) m = max_or_nan(m, part_ml(s).x);
#pragma unroll
  for (int o = 1; o < 32; o *= 2) m = max_or_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float use = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](const float2& c, const float4& v) {
    if (c.x == -INFINITY) return;
    const float f = exp2f(c.x - use);
    l = fmaf(f, c.y, l);
    acc = make_float4(fmaf(f, v.x, acc.x), fmaf(f, v.y, acc.y), fmaf(f, v.z, acc.z), fmaf(f, v.w, acc.w));
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) add(c[i], v[i]);
#pragma unroll 4
  for (int s = p + AHEAD * LANES; s < total; s += LANES) add(part_ml(s), part_row(s));
  so[p][t] = acc;
  if (t == 0) sl[p] = l;
  __syncthreads();
  if (p > 0) return;
#pragma unroll
  for (int i = 1; i < LANES; ++i) {
    const float4 v = so[i][t];
    acc = make_float4(acc.x + v.x, acc.y + v.y, acc.z + v.z, acc.w + v.w);
    l += sl[i];
  }
  // No keys: zeros. No result where the largest score is NaN, or infinite of either sign (l = 0).
  const float inv = m == -INFINITY ? 0.f : m - m == 0.f ? 1.f / l : NAN;
  const float x[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
  T* out = row_of(static_cast<T*>(a.o), a.so, a.inner, z, h, row) + 4 * t;
  if constexpr (sizeof(T) == 2) {
    const uint2 r = make_uint2(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]));
    *reinterpret_cast<uint2*>(out) = r;
    if (a.o_rest != nullptr) {
      const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&r.x)), hi = __half22float2(*reinterpret_cast<const __half2*>(&r.y));
      const uint32_t r0 = __nv_cvt_float2_to_fp8x2(make_float2((x[0] - lo.x) * kRestScale, (x[1] - lo.y) * kRestScale), __NV_SATFINITE, __NV_E5M2);
      const uint32_t r1 = __nv_cvt_float2_to_fp8x2(make_float2((x[2] - hi.x) * kRestScale, (x[3] - hi.y) * kRestScale), __NV_SATFINITE, __NV_E5M2);
      *reinterpret_cast<uint32_t*>(a.o_rest + index * D + 4 * t) = r0 | r1 << 16;
    }
  } else {
    *reinterpret_cast<float4*>(out) = make_float4(x[0], x[1], x[2], x[3]);
  }
  if (a.m != nullptr && t == 0) a.m[index] = m + (m == -INFINITY ? 0.f : log2f(l));
}

template <int D>
cudaError_t join_impl(bool is_f16, const JoinArgs& a, cudaStream_t s) {
  const int64_t rows = int64_t(a.Z) * a.H * a.N;
  if (rows == 0) return cudaSuccess;
  if (rows > 0x7fffffff) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t c{};
  c.gridDim = dim3(unsigned(rows));
  c.blockDim = dim3(kThreads);
  c.stream = s;
  cudaLaunchAttribute attr = overlapping_launch();
  c.attrs = &attr;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, is_f16 ? rows_join_kernel<__half, D> : rows_join_kernel<float, D>, a);
}

}  // namespace

cudaError_t launch_rows_join(int D, bool is_f16, const JoinArgs& a, cudaStream_t s) {
  switch (D) {
    case 16: return join_impl<16>(is_f16, a, s);
    case 32: return join_impl<32>(is_f16, a, s);
    case 64: return join_impl<64>(is_f16, a, s);
    case 128: return join_impl<128>(is_f16, a, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace tattn
