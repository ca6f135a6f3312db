// Norms of query and key heads with the position rotation in the same pass, and the gradients; the rotation by
// positions on several axes, with the norms or alone.
//
// A row x (one head of one token, D values) at position p, with the tensor's weight w and the tables
// cos[p], sin[p] (D / 2 values each):
//   r = 1 / sqrt(mean(x^2) + eps),  z = x r w,  y = R z:
//   y_i = z_i cos_j - z_i' sin_j,  y_i' = z_i' cos_j + z_i sin_j
// for pair j = (i, i') = (j, j + D / 2), or (2 j, 2 j + 1) where `interleaved`. Backward, from dy:
//   g = R^T dy,  dw = sum over rows of g x r,  h = g w,  dx = r (h - x r mean(h x r)).
// On several axes (kAxesNorm, kAxes) a token has a position on each, and pair j is rotated by the tables' row at its
// position on axis axes[j]. kAxes has no norm: y = R x and dx = R^T dy, the same kernel turning the other way.
// Everything between the loads and the stores is fp32; results are rounded once.
//
// The bound is HBM: x is read and y written once (backward: x, dy, dx), about 3 (7) FMAs a value. A group of
// L = D / (2 VEC) lanes owns a token's row: lane c holds the 16 bytes at c and the 16 bytes half a row
// further, so a half-split pair lies in one lane, and so does an interleaved one. A work item is one token
// and HB consecutive heads of one tensor, which share the token's cos and sin and the weight in
// registers; HB = kMany where there are enough items to fill the GPU with, else 1 (a decoding step's few rows).
// dw: every CTA works on one tensor, adds its rows' terms in registers and then shared memory and writes one
// partial; a second small kernel sums the partials in a fixed order, so dw is bitwise reproducible.
//
// Measured (B200, B4 N4096, passes over three sets of tensors): fp16, 16 query and 4 key heads of 64: forward 16 us, 5.1
// TB/s, backward 38 us, 3.3 TB/s (dw's second kernel, 3 us, among them; a lane holds 16 values each of x, dy, w, dw and
// the result in fp32, so two CTAs fit an SM, and 16 warps that load, compute and store in turn leave HBM idle between:
// issue slots 50 % busy); fp32, 16 and 16 heads of 64: 42 us, 6.4 TB/s, and 67 us, 6.0 TB/s. One
// token of 8 sequences, 16 and 4 heads of 128 in fp16: 2.5 us, the launch.
#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.h"

namespace tattn {
namespace {

constexpr int kThreads = 256;
// Heads of a work item. fp16 lanes hold twice the values, in 128 registers: fewer CTAs with more loads each. (Backward in
// fp16 with one head and 4 CTAs an SM 46 us for the 38 above, with 8-byte loads 45 to 53; fp32 with 2 CTAs an SM and 4
// and 2 heads 46 and 78 us for 42 and 67.)
template <typename T, bool BACKWARD>
constexpr int kMany = sizeof(T) == 4 ? (BACKWARD ? 1 : 2) : (BACKWARD ? 2 : 4);

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

// One tensor's items: tokens x chunks of HB heads, in memory order (heads first where a token's heads lie
// next to each other).
struct Item {
  int z, n, h0;
};
__device__ __forceinline__ Item rope_item(const RopeArgs& a, const RopeTensor& t, int HB, int item) {
  const int chunks = (t.H + HB - 1) / HB;
  Item it;
  int chunk;
  if (t.x.h < t.x.n) {
    chunk = item % chunks;
    it.n = item / chunks % a.N;
    it.z = item / chunks / a.N;
  } else {
    it.n = item % a.N;
    chunk = item / a.N % chunks;
    it.z = item / a.N / chunks;
  }
  it.h0 = chunk * HB;
  return it;
}

// The cosines (or sines) of the lane's VEC pairs, from a row of their table.
template <int D, int VEC, bool INTERLEAVED>
__device__ __forceinline__ void load_angles(const float* row, int col, float* x) {
  if constexpr (INTERLEAVED) {
    load_floats<VEC / 2>(row + col / 2, x);
    load_floats<VEC / 2>(row + D / 4 + col / 2, x + VEC / 2);
  } else {
    load_floats<VEC>(row + col, x);
  }
}

// Which axis each of the lane's VEC pairs turns by (2 bits a pair from bit 0 on), and the set of those axes (from
// bit 16 on).
template <int D, int VEC, bool INTERLEAVED>
__device__ __forceinline__ uint32_t lane_axes(const RopeArgs& a, int col) {
  uint32_t x = 0;
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    const int pair = !INTERLEAVED ? col + j : j < VEC / 2 ? col / 2 + j : D / 4 + col / 2 + j - VEC / 2;
    const uint32_t axis = (a.axes[pair / 16] >> (2 * (pair % 16))) & 3u;
    x |= axis << (2 * j) | 0x10000u << axis;
  }
  return x;
}

template <typename T, int D, bool INTERLEAVED, int HB, bool BACKWARD, RopeForm FORM>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 4 : 2) norm_rope_kernel(const RopeArgs a) {
  constexpr int VEC = kVec<T>, L = D / (2 * VEC), GROUPS = kThreads / L;
  constexpr bool NORM = FORM != kAxes;
  static_assert(NORM || !BACKWARD, "a rotation alone is turned back by the forward kernel");
  using P = Pairs<VEC, INTERLEAVED>;
  const int which = int(blockIdx.x) < a.t[0].blocks ? 0 : 1;  // the CTA's tensor
  const RopeTensor& t = a.t[which];
  const int block = int(blockIdx.x) - (which ? a.t[0].blocks : 0);
  const int c = threadIdx.x % L;
  const int col = c * VEC;  // and D / 2 + col
  float w[2 * VEC];
  if constexpr (NORM) {
    if (a.w_f32) {
      load_floats<VEC>(static_cast<const float*>(t.w) + col, w);
      load_floats<VEC>(static_cast<const float*>(t.w) + D / 2 + col, w + VEC);
    } else {
      load16(static_cast<const T*>(t.w) + col, w);
      load16(static_cast<const T*>(t.w) + D / 2 + col, w + VEC);
    }
  }
  uint32_t axes = 0;
  if constexpr (FORM != kOnePosition) axes = lane_axes<D, VEC, INTERLEAVED>(a, col);
  float dw[2 * VEC];
#pragma unroll
  for (int e = 0; e < 2 * VEC; ++e) dw[e] = 0.f;

  // Whole warps stay in the loop together (group_sum): the last items of a warp may be none.
  for (int base = block * GROUPS; base < t.items; base += t.blocks * GROUPS) {
    const int item = base + int(threadIdx.x) / L;
    const bool any = item < t.items;
    const Item it = rope_item(a, t, HB, any ? item : 0);
    // All of the item's loads first, as they come: they are what takes time. (On several axes also before the
    // positions, which the tables' loads wait for.)
    uint4 rx[HB][2], rdy[BACKWARD ? HB : 1][2];
    auto load_rows = [&] {
#pragma unroll
      for (int i = 0; i < HB; ++i) {
        const bool row = any && it.h0 + i < t.H;
        const int64_t h = row ? it.h0 + i : 0;
        const T* px = static_cast<const T*>(t.px) + it.z * t.x.z + h * t.x.h + it.n * t.x.n + col;
        rx[i][0] = load_raw(px);
        rx[i][1] = load_raw(px + D / 2);
        if constexpr (BACKWARD) {
          const T* pd = static_cast<const T*>(t.pdy) + it.z * t.dy.z + h * t.dy.h + it.n * t.dy.n + col;
          rdy[i][0] = load_raw(pd);
          rdy[i][1] = load_raw(pd + D / 2);
        }
      }
    };
    if (FORM != kOnePosition) load_rows();
    float cs[VEC], sn[VEC];
    bool in_table = true;
    if constexpr (FORM == kOnePosition) {
      const int pos = a.positions ? a.positions[it.z * a.pos_z + it.n * a.pos_n] : it.n;
      in_table = pos >= 0 && pos < a.P;
      const int64_t at = int64_t(in_table ? pos : 0) * (D / 2);
      load_angles<D, VEC, INTERLEAVED>(a.cos + at, col, cs);
      load_angles<D, VEC, INTERLEAVED>(a.sin + at, col, sn);
    } else {
      int pos[kRopeAxes];
#pragma unroll
      for (int x = 0; x < kRopeAxes; ++x) {  // all of them, whichever axes the lane's pairs use: a row is NaN as a whole
        pos[x] = x < a.A ? a.positions[x * a.pos_a + it.z * a.pos_z + it.n * a.pos_n] : 0;
        in_table = in_table && pos[x] >= 0 && pos[x] < a.P;
      }
      // A row of each axis that some pair of the lane uses, 16 bytes at a time, and of it what those pairs need.
#pragma unroll
      for (int j = 0; j < VEC; ++j) cs[j] = sn[j] = 0.f;
#pragma unroll
      for (int x = 0; x < kRopeAxes; ++x) {
        if ((axes & (0x10000u << x)) == 0u) continue;
        const int64_t at = int64_t(in_table ? pos[x] : 0) * (D / 2);
        float c4[VEC], s4[VEC];
        load_angles<D, VEC, INTERLEAVED>(a.cos + at, col, c4);
        load_angles<D, VEC, INTERLEAVED>(a.sin + at, col, s4);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const bool mine = ((axes >> (2 * j)) & 3u) == uint32_t(x);
          cs[j] = mine ? c4[j] : cs[j];
          sn[j] = mine ? s4[j] : sn[j];
        }
      }
      if (FORM == kAxes && a.back) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) sn[j] = -sn[j];
      }
    }
    if (!in_table && any) {  // no rotation exists: the rows become NaN, and the status word says why
#pragma unroll
      for (int j = 0; j < VEC; ++j) cs[j] = sn[j] = __int_as_float(0x7fffffff);
      if (c == 0) atomicOr(a.status, kStatusIndexRange);
    }
    if (FORM == kOnePosition) load_rows();
#pragma unroll
    for (int i = 0; i < HB; ++i) {
      const bool row = any && it.h0 + i < t.H;
      float x[2 * VEC];
      unpack16<T>(rx[i][0], x);
      unpack16<T>(rx[i][1], x + VEC);
      float r = 1.f;
      if constexpr (NORM) {
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 2 * VEC; ++e) sum = fmaf(x[e], x[e], sum);
        r = rsqrtf(group_sum<L>(sum) * (1.f / D) + a.eps);
      }
      float out[2 * VEC];
      if constexpr (!BACKWARD) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int f = P::first(j), s = P::second(j);
          const float zf = NORM ? x[f] * r * w[f] : x[f], zs = NORM ? x[s] * r * w[s] : x[s];
          out[f] = zf * cs[j] - zs * sn[j];
          out[s] = zs * cs[j] + zf * sn[j];
        }
      } else {
        float dy[2 * VEC], dot = 0.f;
        unpack16<T>(rdy[i][0], dy);
        unpack16<T>(rdy[i][1], dy + VEC);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int f = P::first(j), s = P::second(j);
          const float gf = dy[f] * cs[j] + dy[s] * sn[j], gs = dy[s] * cs[j] - dy[f] * sn[j];
          x[f] *= r;
          x[s] *= r;
          if (row) {
            dw[f] = fmaf(gf, x[f], dw[f]);
            dw[s] = fmaf(gs, x[s], dw[s]);
          }
          out[f] = gf * w[f];
          out[s] = gs * w[s];
          dot = fmaf(out[f], x[f], dot);
          dot = fmaf(out[s], x[s], dot);
        }
        const float mean = group_sum<L>(dot) * (1.f / D);
#pragma unroll
        for (int e = 0; e < 2 * VEC; ++e) out[e] = r * (out[e] - x[e] * mean);
      }
      if (row) {
        T* py = static_cast<T*>(t.py) + it.z * t.y.z + int64_t(it.h0 + i) * t.y.h + it.n * t.y.n + col;
        store16(py, out);
        store16(py + D / 2, out + VEC);
      }
    }
  }
  if constexpr (BACKWARD) {
    // The CTA's sum over its groups of lanes, in a fixed order; value e of lane c is column col + e or
    // D / 2 + col + e - VEC.
    __shared__ float part[GROUPS][D];
#pragma unroll
    for (int e = 0; e < 2 * VEC; ++e) part[threadIdx.x / L][(e < VEC ? col + e : D / 2 + col + e - VEC)] = dw[e];
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += kThreads) {
      float s = 0.f;
      for (int g = 0; g < GROUPS; ++g) s += part[g][d];
      a.part[int64_t(blockIdx.x) * D + d] = s;
    }
  }
}

// dw of both tensors from the CTAs' partials: 8 columns (a 32-byte sector) a block, 32 threads a column.
constexpr int kDwCols = 8;
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_rope_dw_kernel(const RopeArgs a, int D) {
  __shared__ float part[32][kDwCols + 1];
  const int which = blockIdx.y, c = threadIdx.x % kDwCols, col = blockIdx.x * kDwCols + c, lane = threadIdx.x / kDwCols;
  const int b0 = which ? a.t[0].blocks : 0, b1 = b0 + a.t[which].blocks;
  float s = 0.f;
#pragma unroll 8
  for (int b = b0 + lane; b < b1; b += 32) s += a.part[int64_t(b) * D + col];
  part[lane][c] = s;
  __syncthreads();
  if (lane == 0) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += part[i][c];
    if (a.w_f32)
      static_cast<float*>(a.t[which].dw)[col] = s;
    else if constexpr (sizeof(T) == 2)
      static_cast<T*>(a.t[which].dw)[col] = __float2half_rn(s);
    else
      static_cast<T*>(a.t[which].dw)[col] = s;
  }
}

template <typename T, int D, bool INTERLEAVED, bool BACKWARD, RopeForm FORM>
cudaError_t rope_impl(RopeArgs& a, cudaStream_t s) {
  constexpr int GROUPS = kThreads / (D / (2 * kVec<T>));
  const int sms = device_sm_count();
  // Several heads an item (fp32 backward: one at all sizes) once that still gives every SM's 2048 threads something to do.
  constexpr int MANY = kMany<T, BACKWARD>;
  const int64_t rows = int64_t(a.Z) * a.N * (a.t[0].H + a.t[1].H);
  const bool many = rows * (D / (2 * kVec<T>)) >= int64_t(sms) * 2048 * MANY;
  const int HB = many ? MANY : 1;
  for (RopeTensor& t : a.t) t.items = a.Z * a.N * ((t.H + HB - 1) / HB);
  const int most = kRopeBlocksPerSm * sms;
  for (int i = 0; i < 2; ++i) {
    const int64_t all = int64_t(a.t[0].items) + a.t[1].items;
    const int need = (a.t[i].items + GROUPS - 1) / GROUPS;
    // Backward: a bounded number of partials, shared out by work. Forward: every item its own group.
    const int share = int((int64_t(most) * a.t[i].items + all - 1) / (all > 0 ? all : 1));
    a.t[i].blocks = BACKWARD && need > share ? share : need;
  }
  const int grid = a.t[0].blocks + a.t[1].blocks;
  if (grid > 0) {
    if (many)
      norm_rope_kernel<T, D, INTERLEAVED, MANY, BACKWARD, FORM><<<grid, kThreads, 0, s>>>(a);
    else
      norm_rope_kernel<T, D, INTERLEAVED, 1, BACKWARD, FORM><<<grid, kThreads, 0, s>>>(a);
  }
  if (BACKWARD) norm_rope_dw_kernel<T><<<dim3(D / kDwCols, 2), kThreads, 0, s>>>(a, D);
  return cudaGetLastError();
}

template <typename T, bool BACKWARD, RopeForm FORM>
cudaError_t rope_dispatch(int D, bool interleaved, RopeArgs& a, cudaStream_t s) {
#define TATTN_ROPE_CASE(DD) \
  case DD: return interleaved ? rope_impl<T, DD, true, BACKWARD, FORM>(a, s) : rope_impl<T, DD, false, BACKWARD, FORM>(a, s);
  switch (D) {
    TATTN_ROPE_CASE(16)
    TATTN_ROPE_CASE(32)
    TATTN_ROPE_CASE(64)
    TATTN_ROPE_CASE(128)
    default: return cudaErrorInvalidValue;
  }
#undef TATTN_ROPE_CASE
}

template <typename T>
cudaError_t rope_form(int D, RopeForm form, bool interleaved, bool backward, RopeArgs& a, cudaStream_t s) {
  switch (form) {
    case kOnePosition:
      return backward ? rope_dispatch<T, true, kOnePosition>(D, interleaved, a, s)
                      : rope_dispatch<T, false, kOnePosition>(D, interleaved, a, s);
    case kAxesNorm:
      return backward ? rope_dispatch<T, true, kAxesNorm>(D, interleaved, a, s)
                      : rope_dispatch<T, false, kAxesNorm>(D, interleaved, a, s);
    default:
      return rope_dispatch<T, false, kAxes>(D, interleaved, a, s);
  }
}

}  // namespace

cudaError_t launch_norm_rope(int D, bool is_f16, RopeForm form, bool interleaved, bool backward, RopeArgs a, cudaStream_t s) {
  return is_f16 ? rope_form<__half>(D, form, interleaved, backward, a, s)
                : rope_form<float>(D, form, interleaved, backward, a, s);
}

}  // namespace tattn
