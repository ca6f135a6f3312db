// The position rotation of query and key heads by positions on several axes (a video's time, row and column), with the
// heads' norms or alone, and the gradients.
//
// A row x (one head of one token) is R (x r w) or R x, as in norm_rope.cu: r = 1 / sqrt(mean(x^2) + eps), and R turns pair j
// by the angle whose cosine and sine are the tables' at [p, j], here of the token's position p = positions[axes[j]].
// Backward, from dy: g = R^T dy, dw = sum over rows of g x r, h = g w, dx = r (h - x r mean(h x r)); of the rotation alone
// dx = R^T dy, which is the forward kernel turning by the negative angles.
//
// The bound is HBM: x in and y out (backward: x, dy, dx). An item is one token and HB consecutive heads of one tensor,
// which share the angles; a group of L = D / (2 VEC) lanes owns a row, lane c its 16 bytes at c and the 16 bytes half a row
// further, which are VEC pairs. The angles of a lane's pairs come from up to four rows of each table: where they are
// all of one axis as 16-byte loads, else pair by pair (whole rows of every axis with a choice among them took 1.5 times the
// instructions). What is left is instructions: arithmetic on pairs of floats (fma.rn.f32x2), the forward's weight times
// the angle once for an item's heads, divisions by multiplication.
// Measured (B200, B4 N4096, passes over three sets of tensors, axes in turn over the pairs, with norms): fp16, 16 and 4 heads
// of 128: forward 40 us, 4.2 TB/s, backward 62 us, 4.1 TB/s (dw's second kernel, 5 us, among them); issue slots are 50 % busy
// with 16 warps an SM, the rest is loads that they wait for (with 2 heads an item and 3 CTAs an SM 47 us; backward with one
// head and 3 CTAs 69). fp32, 16 and 16 heads of 64: 47 us, 5.7 TB/s, and 74 us, 5.5 TB/s. The rotation alone: 37 us (fp16).
// dw: each CTA adds its rows' terms in registers and writes one partial; norm_rope.cu's second kernel sums them in order.
#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.h"
#include "rope.cuh"

namespace tattn {
namespace {

constexpr int kThreads = 256;
template <typename T, bool BACKWARD>
constexpr int kMany = sizeof(T) == 4 ? (BACKWARD ? 1 : 2) : (BACKWARD ? 2 : 4);  // heads of an item
template <typename T, bool BACKWARD>
constexpr int kCtas = sizeof(T) == 4 ? 4 : 2;  // an SM's

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t both(float x) { return f2(x, x); }
__device__ __forceinline__ uint64_t neg2(uint64_t a) { return a ^ 0x8000000080000000ull; }

// A lane's VEC pairs: their first and second values, two pairs to a register pair.
template <int VEC>
struct Row {
  uint64_t f[VEC / 2], s[VEC / 2];
};
// From the lane's 2 VEC values in the order of its two units.
template <int VEC, bool INTERLEAVED>
__device__ __forceinline__ Row<VEC> pairs_of(const float* x) {
  using P = Pairs<VEC, INTERLEAVED>;
  Row<VEC> r;
#pragma unroll
  for (int k = 0; k < VEC / 2; ++k) {
    r.f[k] = f2(x[P::first(2 * k)], x[P::first(2 * k + 1)]);
    r.s[k] = f2(x[P::second(2 * k)], x[P::second(2 * k + 1)]);
  }
  return r;
}
template <int VEC, bool INTERLEAVED>
__device__ __forceinline__ void values_of(const Row<VEC>& r, float* x) {
  using P = Pairs<VEC, INTERLEAVED>;
#pragma unroll
  for (int k = 0; k < VEC / 2; ++k) {
    const float2 f = f2_unpack(r.f[k]), s = f2_unpack(r.s[k]);
    x[P::first(2 * k)] = f.x;
    x[P::first(2 * k + 1)] = f.y;
    x[P::second(2 * k)] = s.x;
    x[P::second(2 * k + 1)] = s.y;
  }
}
template <typename T, bool INTERLEAVED>
__device__ __forceinline__ Row<kVec<T>> row_from(const uint4* raw) {
  float x[2 * kVec<T>];
  unpack16<T>(raw[0], x);
  unpack16<T>(raw[1], x + kVec<T>);
  return pairs_of<kVec<T>, INTERLEAVED>(x);
}
template <typename T, int D, bool INTERLEAVED>
__device__ __forceinline__ void store_row(T* p, const Row<kVec<T>>& r) {
  float x[2 * kVec<T>];
  values_of<kVec<T>, INTERLEAVED>(r, x);
  store16(p, x);
  store16(p + D / 2, x + kVec<T>);
}

// Pair j of a lane is pair pair_at(col, j) of its row.
template <int D, int VEC, bool INTERLEAVED>
__device__ __forceinline__ int pair_at(int col, int j) {
  return !INTERLEAVED ? col + j : j < VEC / 2 ? col / 2 + j : D / 4 + col / 2 + j - VEC / 2;
}

template <typename T, int D, bool INTERLEAVED, int HB, bool BACKWARD, bool NORM>
__global__ void __launch_bounds__(kThreads, kCtas<T, BACKWARD>) rope_axes_kernel(const RopeAxesArgs a) {
  constexpr int VEC = kVec<T>, L = D / (2 * VEC), GROUPS = kThreads / L;
  static_assert(NORM || !BACKWARD, "a rotation alone is turned back by the forward kernel");
  const int which = int(blockIdx.x) < a.t[0].blocks ? 0 : 1;  // the CTA's tensor
  const RopeTensor& t = a.t[which];
  const int block = int(blockIdx.x) - (which ? a.t[0].blocks : 0);
  const int lane = threadIdx.x % 32, c = lane % L, base_lane = lane - c;
  const int col = c * VEC;  // and D / 2 + col
  const bool heads_first = t.x.h < t.x.n;
  Row<VEC> w;
  if constexpr (NORM) {
    float x[2 * VEC];
    if (a.w_f32) {
      load_floats<VEC>(static_cast<const float*>(t.w) + col, x);
      load_floats<VEC>(static_cast<const float*>(t.w) + D / 2 + col, x + VEC);
    } else {
      load16(static_cast<const T*>(t.w) + col, x);
      load16(static_cast<const T*>(t.w) + D / 2 + col, x + VEC);
    }
    w = pairs_of<VEC, INTERLEAVED>(x);
  }
  uint32_t axes = 0;  // 2 bits a pair
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    const int pair = pair_at<D, VEC, INTERLEAVED>(col, j);
    axes |= ((a.axes[pair / 16] >> (2 * (pair % 16))) & 3u) << (2 * j);
  }
  const bool one_axis = axes == (axes & 3u) * (0x55555555u >> (32 - 2 * VEC));
  Row<VEC> dw{};

  // Whole warps stay in the loop together (shuffles): the last items of a warp may be none.
  for (int base = block * GROUPS; base < t.items; base += t.blocks * GROUPS) {
    const int number = base + int(threadIdx.x) / L;
    const bool any = number < t.items;
    const uint32_t item = any ? number : 0;
    const ByMultiple& inner = heads_first ? a.chunks[which] : a.tokens;
    const ByMultiple& outer = heads_first ? a.tokens : a.chunks[which];
    const uint32_t q0 = inner.quotient(item), i0 = item - q0 * inner.d, z = outer.quotient(q0), i1 = q0 - z * outer.d;
    const int n = heads_first ? i1 : i0, h0 = int(heads_first ? i0 : i1) * HB;

    // The item's rows first, and of them all: they are what takes time.
    uint4 rx[HB][2], rdy[BACKWARD ? HB : 1][2];
#pragma unroll
    for (int i = 0; i < HB; ++i) {
      const int64_t h = any && h0 + i < t.H ? h0 + i : 0;
      const T* px = static_cast<const T*>(t.px) + z * t.x.z + h * t.x.h + n * t.x.n + col;
      rx[i][0] = load_raw(px);
      rx[i][1] = load_raw(px + D / 2);
      if constexpr (BACKWARD) {
        const T* pd = static_cast<const T*>(t.pdy) + z * t.dy.z + h * t.dy.h + n * t.dy.n + col;
        rdy[i][0] = load_raw(pd);
        rdy[i][1] = load_raw(pd + D / 2);
      }
    }
    // Positions: lane x of a group reads axis x's, or every lane all of them. A token with one outside the tables is NaN
    // throughout, whichever axes its pairs use.
    const int* at = a.positions + z * a.pos_z + n * a.pos_n;
    int pos[L >= kRopeAxes ? 1 : kRopeAxes];
    bool in_table;
    if constexpr (L >= kRopeAxes) {
      pos[0] = c < a.A ? at[c * a.pos_a] : 0;
      const uint32_t ok = __ballot_sync(0xffffffffu, pos[0] >= 0 && pos[0] < a.P);
      in_table = ((~ok >> base_lane) & (0xffffffffu >> (32 - L))) == 0u;
    } else {
      in_table = true;
#pragma unroll
      for (int x = 0; x < kRopeAxes; ++x) {
        pos[x] = x < a.A ? at[x * a.pos_a] : 0;
        in_table = in_table && pos[x] >= 0 && pos[x] < a.P;
      }
    }
    auto position = [&](int j) {  // of the lane's pair j
      const int axis = (axes >> (2 * j)) & 3u;
      int p;
      if constexpr (L >= kRopeAxes)
        p = __shfl_sync(0xffffffffu, pos[0], base_lane + axis);
      else
        p = axis < 2 ? (axis == 0 ? pos[0] : pos[1]) : axis == 2 ? pos[2] : pos[3];
      return in_table ? p : 0;
    };
    float cs[VEC], sn[VEC];
    {
      int p[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) p[j] = position(j);
      const float *ct = a.cos + pair_at<D, VEC, INTERLEAVED>(col, 0), *st = a.sin + pair_at<D, VEC, INTERLEAVED>(col, 0);
      constexpr int RUN = INTERLEAVED ? VEC / 2 : VEC;  // pairs that lie one after another in the tables
      if (one_axis) {
        const int64_t row = int64_t(p[0]) * (D / 2);
#pragma unroll
        for (int j = 0; j < VEC; j += RUN) {
          load_floats<RUN>(ct + row + j / RUN * (D / 4), cs + j);
          load_floats<RUN>(st + row + j / RUN * (D / 4), sn + j);
        }
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int64_t row = int64_t(p[j]) * (D / 2);
          const int in_row = j % RUN + j / RUN * (D / 4);
          cs[j] = ct[row + in_row];
          sn[j] = st[row + in_row];
        }
      }
    }
    if (!in_table && any) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) cs[j] = sn[j] = __int_as_float(0x7fffffff);
      if (c == 0) atomicOr(a.status, kStatusIndexRange);
    }
    Row<VEC> angle;  // cosines and sines
#pragma unroll
    for (int k = 0; k < VEC / 2; ++k) {
      angle.f[k] = f2(cs[2 * k], cs[2 * k + 1]);
      angle.s[k] = f2(sn[2 * k], sn[2 * k + 1]);
      if (!NORM && a.back) angle.s[k] = neg2(angle.s[k]);
    }
    // Forward: y = r (x_f wc - x_s ws', x_s wc' + x_f ws): the angles with the weights.
    Row<VEC> wc, ws;
    if constexpr (!BACKWARD) {
#pragma unroll
      for (int k = 0; k < VEC / 2; ++k) {
        wc.f[k] = NORM ? mul2(w.f[k], angle.f[k]) : angle.f[k];
        wc.s[k] = NORM ? mul2(w.s[k], angle.f[k]) : angle.f[k];
        ws.f[k] = NORM ? mul2(w.f[k], angle.s[k]) : angle.s[k];
        ws.s[k] = neg2(NORM ? mul2(w.s[k], angle.s[k]) : angle.s[k]);
      }
    }
#pragma unroll
    for (int i = 0; i < HB; ++i) {
      const bool row = any && h0 + i < t.H;
      Row<VEC> x = row_from<T, INTERLEAVED>(rx[i]), out;
      uint64_t r = 0;
      if constexpr (NORM) {
        uint64_t sum = mul2(x.f[0], x.f[0]);
#pragma unroll
        for (int k = 0; k < VEC / 2; ++k) {
          if (k > 0) sum = ffma2(x.f[k], x.f[k], sum);
          sum = ffma2(x.s[k], x.s[k], sum);
        }
        const float2 two = f2_unpack(sum);
        r = both(rsqrtf(group_sum<L>(two.x + two.y) * (1.f / D) + a.eps));
      }
      if constexpr (!BACKWARD) {
#pragma unroll
        for (int k = 0; k < VEC / 2; ++k) {
          out.f[k] = ffma2(x.f[k], wc.f[k], mul2(x.s[k], ws.s[k]));
          out.s[k] = ffma2(x.s[k], wc.s[k], mul2(x.f[k], ws.f[k]));
          if (NORM) out.f[k] = mul2(out.f[k], r);
          if (NORM) out.s[k] = mul2(out.s[k], r);
        }
      } else {
        const Row<VEC> dy = row_from<T, INTERLEAVED>(rdy[i]);
        uint64_t dot = 0;
#pragma unroll
        for (int k = 0; k < VEC / 2; ++k) {
          const uint64_t gf = ffma2(dy.f[k], angle.f[k], mul2(dy.s[k], angle.s[k]));
          const uint64_t gs = ffma2(dy.s[k], angle.f[k], mul2(dy.f[k], neg2(angle.s[k])));
          x.f[k] = mul2(x.f[k], r);
          x.s[k] = mul2(x.s[k], r);
          if (row) {
            dw.f[k] = ffma2(gf, x.f[k], dw.f[k]);
            dw.s[k] = ffma2(gs, x.s[k], dw.s[k]);
          }
          out.f[k] = mul2(gf, w.f[k]);
          out.s[k] = mul2(gs, w.s[k]);
          dot = k == 0 ? mul2(out.f[k], x.f[k]) : ffma2(out.f[k], x.f[k], dot);
          dot = ffma2(out.s[k], x.s[k], dot);
        }
        const float2 two = f2_unpack(dot);
        const uint64_t mean = both(group_sum<L>(two.x + two.y) * (-1.f / D));
#pragma unroll
        for (int k = 0; k < VEC / 2; ++k) {
          out.f[k] = mul2(r, ffma2(x.f[k], mean, out.f[k]));
          out.s[k] = mul2(r, ffma2(x.s[k], mean, out.s[k]));
        }
      }
      if (row)
        store_row<T, D, INTERLEAVED>(static_cast<T*>(t.py) + z * t.y.z + int64_t(h0 + i) * t.y.h + n * t.y.n + col, out);
    }
  }
  if constexpr (BACKWARD) {
    // The CTA's sum over its groups of lanes, in a fixed order.
    __shared__ float part[GROUPS][D];
    float x[2 * VEC];
    values_of<VEC, INTERLEAVED>(dw, x);
#pragma unroll
    for (int e = 0; e < 2 * VEC; ++e) part[threadIdx.x / L][(e < VEC ? col + e : D / 2 + col + e - VEC)] = x[e];
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += kThreads) {
      float s = 0.f;
      for (int g = 0; g < GROUPS; ++g) s += part[g][d];
      a.part[int64_t(blockIdx.x) * D + d] = s;
    }
  }
}

template <typename T, int D, bool INTERLEAVED, bool BACKWARD, bool NORM>
cudaError_t axes_impl(RopeAxesArgs& a, cudaStream_t s) {
  constexpr int GROUPS = kThreads / (D / (2 * kVec<T>)), MANY = kMany<T, BACKWARD>;
  const int sms = device_sm_count();
  // Several heads an item once that still gives every SM's 2048 threads something to do.
  const int64_t rows = int64_t(a.Z) * a.N * (a.t[0].H + a.t[1].H);
  const bool many = rows * (D / (2 * kVec<T>)) >= int64_t(sms) * 2048 * MANY;
  const int HB = many ? MANY : 1;
  a.tokens = by_multiple(a.N);
  for (int i = 0; i < 2; ++i) {
    const int chunks = (a.t[i].H + HB - 1) / HB;
    a.chunks[i] = by_multiple(chunks);
    a.t[i].items = a.Z * a.N * chunks;
  }
  const int64_t all = int64_t(a.t[0].items) + a.t[1].items, fit = int64_t(kCtas<T, BACKWARD>) * sms;
  for (RopeTensor& t : a.t) {
    // Forward: every item its own group. Backward: no more CTAs than run at a time, each with its share (one more, and the
    // rest wait for it).
    const int need = (t.items + GROUPS - 1) / GROUPS;
    const int64_t share = all > 0 ? fit * t.items / all : 0;
    t.blocks = BACKWARD && need > share ? int(share > 1 ? share : 1) : need;
  }
  const int grid = a.t[0].blocks + a.t[1].blocks;
  if (grid > 0) {
    if (many)
      rope_axes_kernel<T, D, INTERLEAVED, MANY, BACKWARD, NORM><<<grid, kThreads, 0, s>>>(a);
    else
      rope_axes_kernel<T, D, INTERLEAVED, 1, BACKWARD, NORM><<<grid, kThreads, 0, s>>>(a);
  }
  const cudaError_t e = cudaGetLastError();
  return e != cudaSuccess || !BACKWARD ? e : launch_norm_rope_dw(sizeof(T) == 2, D, a, s);
}

template <typename T, bool BACKWARD, bool NORM>
cudaError_t axes_dispatch(int D, bool interleaved, RopeAxesArgs& a, cudaStream_t s) {
#define TATTN_AXES_CASE(DD) \
  case DD: return interleaved ? axes_impl<T, DD, true, BACKWARD, NORM>(a, s) : axes_impl<T, DD, false, BACKWARD, NORM>(a, s);
  switch (D) {
    TATTN_AXES_CASE(16)
    TATTN_AXES_CASE(32)
    TATTN_AXES_CASE(64)
    TATTN_AXES_CASE(128)
    default: return cudaErrorInvalidValue;
  }
#undef TATTN_AXES_CASE
}

template <typename T>
cudaError_t axes_form(int D, bool norm, bool interleaved, bool backward, RopeAxesArgs& a, cudaStream_t s) {
  if (!norm) return axes_dispatch<T, false, false>(D, interleaved, a, s);
  return backward ? axes_dispatch<T, true, true>(D, interleaved, a, s) : axes_dispatch<T, false, true>(D, interleaved, a, s);
}

}  // namespace

cudaError_t launch_rope_axes(int D, bool is_f16, bool norm, bool interleaved, bool backward, RopeAxesArgs a, cudaStream_t s) {
  return is_f16 ? axes_form<__half>(D, norm, interleaved, backward, a, s) : axes_form<float>(D, norm, interleaved, backward, a, s);
}

}  // namespace tattn
