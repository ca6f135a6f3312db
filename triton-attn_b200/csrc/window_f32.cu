// Sliding-window attention with sinks for fp32 on CUDA cores: forward, dK/dV and dQ.
//
// The mathematics is the fp16 kernels' (base-2 online softmax, M = m + log2 l, P rebuilt from M in the
// backward) with every product and sum in fp32: tcgen05 has no fp32 MMA, and fp32 calls are held to fp32
// accuracy. Two kernels for the backward, dK/dV by key tiles and dQ by query tiles, so that nothing is
// summed by atomics and results are bitwise reproducible.
//
// The bound is the FMA pipe (4 D flop forward and 14 D backward a pair) fed from shared memory: tiles of T x 64, and a
// thread computes R x 4 scores (rows R ty + i, columns tx + 16 j) from 16-byte reads along D, then R rows x D / 16
// columns of the products with V, K, Q and dO the same way. A read that 16 threads share costs 1 to 2 cycles of shared
// memory and one of 16 different units 4: with R = 4 they outweigh the FMAs (72 % of the cycles against 53 %, dK/dV at
// B4 H16 N2048 D64, window 512), with R = 8 they do not. The next block's rows are on their way while this one's are
// computed with (cp.async).
//
// T = 64 (R = 8; 4 at D = 128, for the registers): 580 -> 515 us forward and 1822 -> 1635 backward there against R = 4.
// With fewer tiles than 5 an SM, T = 32 (R = 4): more CTAs to spread and fewer masked pairs (B1 H4 N700 D64, causal:
// 72 -> 42 forward, 153 -> 106 backward; B2 H8 N1500 D128, window 300: 195 -> 185 and 660 -> 630; with 14 tiles an SM 527
// and 1850 for the 515 and 1635 above), and for D = 16, whose 64 rows take more threads than they give work (B4 H16 N2048,
// window 512: 248 -> 220 and 704 -> 640). Rates by visible pairs, of the FMA pipes' 74 TFLOP/s: 29 forward and 32 backward
// at the first size (40 with the masked pairs of its tiles), 13 to 14 at B3 H5 N1000 D64, window 200, 4 sinks (56 us
// forward, 172 backward; 19 with the masked ones), where the 480 tiles differ in length and the busiest SM has 1.55
// times the mean.
#include <math.h>

#include "common.cuh"
#include "kernels.h"

namespace tattn {
namespace {

constexpr int TB = kWindowF32Block;  // columns of a tile: the rows that are loaded one block after another
template <int D, int T>              // T: rows of a tile, 64 or 32
constexpr int kRows = T == 64 && (D == 32 || D == 64) ? 8 : 4;  // a thread's
template <int D, int T>
constexpr int kThreads = 16 * T / kRows<D, T>;
constexpr float kLog2e = 1.4426950408889634f;

// Row pitch in floats: 16-byte units a row odd in number, so that 16 rows at one unit are in different banks.
template <int D>
constexpr int kPitch = D + 4;
constexpr int kPitchP = TB + 4;

// Rows [r0, r0 + ROWS) of a [n, D] matrix into shared memory, 16 bytes at a time and asynchronously (cp_async_wait) where
// its rows allow; rows past n are zeros.
template <int D, int ROWS, int THREADS>
__device__ __forceinline__ void load_rows(float* dst, const float* src, const Strides4& s, int r0, int n) {
  if (s.d == 1 && s.n % 4 == 0 && (reinterpret_cast<uintptr_t>(src) & 15u) == 0) {
#pragma unroll
    for (int i = 0; i < ROWS * D / 4 / THREADS; ++i) {
      const int e = i * THREADS + threadIdx.x, r = e / (D / 4), d = e % (D / 4) * 4;
      cp_async16(smem_u32(dst + r * kPitch<D> + d), src + int64_t(min(r0 + r, n - 1)) * s.n + d, r0 + r < n);
    }
    return;
  }
#pragma unroll 4
  for (int e = threadIdx.x; e < ROWS * D; e += THREADS) {
    const int r = e / D, d = e % D;
    dst[r * kPitch<D> + d] = r0 + r < n ? __ldg(src + int64_t(r0 + r) * s.n + d * s.d) : 0.f;
  }
}

// c[i][j] = a[R ty + i] . b[tx + 16 j] over D.
template <int D, int R>
__device__ __forceinline__ void rows_dot(const float* a, const float* b, int ty, int tx, float (*c)[4]) {
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) c[i][j] = 0.f;
#pragma unroll 2
  for (int d = 0; d < D; d += 4) {
    float4 x[R], y[4];
#pragma unroll
    for (int i = 0; i < R; ++i) x[i] = *reinterpret_cast<const float4*>(a + (R * ty + i) * kPitch<D> + d);
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const float4*>(b + (tx + 16 * j) * kPitch<D> + d);
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        c[i][j] = fmaf(x[i].w, y[j].w, fmaf(x[i].z, y[j].z, fmaf(x[i].y, y[j].y, fmaf(x[i].x, y[j].x, c[i][j]))));
  }
}

// acc[i][e] += sum over r of p[R ty + i][r] b[r][D / 16 tx + e], two e in a packed FMA.
template <int D, int R>
__device__ __forceinline__ void rows_times(const float* p, const float* b, int ty, int tx, float (*acc)[D / 16]) {
  constexpr int E = D / 16;
#pragma unroll 2
  for (int r = 0; r < TB; r += 4) {
    float4 x[R];
#pragma unroll
    for (int i = 0; i < R; ++i) x[i] = *reinterpret_cast<const float4*>(p + (R * ty + i) * kPitchP + r);
#pragma unroll
    for (int rr = 0; rr < 4; ++rr) {
      float y[E];
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] = b[(r + rr) * kPitch<D> + E * tx + e];
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float w = rr == 0 ? x[i].x : rr == 1 ? x[i].y : rr == 2 ? x[i].z : x[i].w;
        if constexpr (E == 1) {
          acc[i][0] = fmaf(w, y[0], acc[i][0]);
        } else {
#pragma unroll
          for (int e = 0; e < E; e += 2) {
            const float2 f = f2_unpack(ffma2(f2(w, w), f2(y[e], y[e + 1]), f2(acc[i][e], acc[i][e + 1])));
            acc[i][e] = f.x;
            acc[i][e + 1] = f.y;
          }
        }
      }
    }
  }
}

// The CTA's head among Z * H: the grid's second and third dimension, as one is limited to 65535.
__device__ __forceinline__ int64_t cta_head() { return int64_t(blockIdx.z) * gridDim.y + blockIdx.y; }

// Does query row `row` of N see key `col`?
__device__ __forceinline__ bool sees(int row, int col, int N, const WindowArgs& w) {
  const int p = row + w.off;
  return row < N && col <= p && (col > p - w.window || col < w.sinks);
}

// Blocks of keys of the query rows from r0 on: those with sinks, then those that a window reaches, up to the diagonal.
__device__ __forceinline__ int next_keys(int k0, int r0, const WindowArgs& w) {
  k0 += TB;
  return k0 >= w.sinks ? max(k0, max(0, r0 + w.off - w.window + 1) / TB * TB) : k0;
}

template <int D, int T>
__global__ void __launch_bounds__(kThreads<D, T>) window_fwd_f32_kernel(const float* q, const float* k, const float* v,
                                                                  Strides4 sq, Strides4 sk, Strides4 sv, FwdArgs a) {
  constexpr int R = kRows<D, T>, TH = kThreads<D, T>;
  extern __shared__ __align__(16) float smem[];
  float *Qs = smem, *Ks = Qs + T * kPitch<D>, *Vs = Ks + TB * kPitch<D>, *Ps = Vs + TB * kPitch<D>;
  const int N = a.N, Nk = a.win.Nk, r0 = blockIdx.x * T;
  const int64_t head = cta_head();
  if (head >= int64_t(a.Z) * a.H) return;
  const int zi = int(head / a.H), hi = int(head % a.H), hk = hi / a.win.group;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  k += zi * sk.z + hk * sk.h;
  v += zi * sv.z + hk * sv.h;
  int k0 = next_keys(-TB, r0, a.win);
  load_rows<D, T, TH>(Qs, q + zi * sq.z + hi * sq.h, sq, r0, N);
  load_rows<D, TB, TH>(Ks, k, sk, k0, Nk);
  float m[R], l[R], acc[R][D / 16];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int e = 0; e < D / 16; ++e) acc[i][e] = 0.f;
  }
  const int end = min(r0 + T + a.win.off, Nk);
  for (int next; k0 < end; k0 = next) {
    cp_async_wait_all();
    __syncthreads();  // K is here, and V's last tile has been read
    load_rows<D, TB, TH>(Vs, v, sv, k0, Nk);
    float s[R][4];
    rows_dot<D, R>(Qs, Ks, ty, tx, s);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float mx = m[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = sees(r0 + R * ty + i, k0 + tx + 16 * j, N, a.win) ? s[i][j] * a.qk_scale : -INFINITY;
        mx = fmaxf(mx, s[i][j]);
      }
#pragma unroll
      for (int o = 1; o < 16; o *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float use = mx == -INFINITY ? 0.f : mx, alpha = exp2f(m[i] - use);
      m[i] = mx;
      l[i] *= alpha;
#pragma unroll
      for (int e = 0; e < D / 16; ++e) acc[i][e] *= alpha;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = exp2f(s[i][j] - use);
        l[i] += p;  // this thread's columns
        Ps[(R * ty + i) * kPitchP + tx + 16 * j] = p;
      }
    }
    cp_async_wait_all();
    __syncthreads();  // V is here, and K has been read
    next = next_keys(k0, r0, a.win);
    if (next < end) load_rows<D, TB, TH>(Ks, k, sk, next, Nk);
    rows_times<D, R>(Ps, Vs, ty, tx, acc);
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
#pragma unroll
    for (int o = 1; o < 16; o *= 2) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
    const int row = r0 + R * ty + i;
    if (row >= N) continue;
    float* o = static_cast<float*>(a.o) + zi * a.so.z + hi * a.so.h + int64_t(row) * a.so.n;
    const float inv = 1.f / l[i];
#pragma unroll
    for (int e = 0; e < D / 16; ++e) o[(D / 16 * tx + e) * a.so.d] = acc[i][e] * inv;
    if (tx == 0) a.m[head * N + row] = m[i] + log2f(l[i]);
  }
}

// P and dS of rows R ty + i of A (with C) and rows tx + 16 j of B (with E): A, B are queries and keys, or keys
// and queries (KEYS); C, E their dO and V, or V and dO.
template <int D, int R, bool KEYS>
__device__ __forceinline__ void p_ds(const BwdArgs& a, const float* A, const float* B, const float* C, const float* E,
                                     int ty, int tx, int a0, int b0, const float* Ms, const float* Ds, float (*p)[4],
                                     float (*ds)[4]) {
  float s[R][4], dp[R][4];
  rows_dot<D, R>(A, B, ty, tx, s);
  rows_dot<D, R>(C, E, ty, tx, dp);
  const float qks = a.sm_scale * kLog2e;
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int ra = R * ty + i, rb = tx + 16 * j, row = KEYS ? rb : ra;  // the tile's query row
      const bool see = KEYS ? sees(b0 + rb, a0 + ra, a.N, a.win) : sees(a0 + ra, b0 + rb, a.N, a.win);
      p[i][j] = see ? exp2f(s[i][j] * qks - Ms[row]) : 0.f;
      ds[i][j] = p[i][j] * (dp[i][j] - Ds[row]);
    }
}

template <int D, int T>
__global__ void __launch_bounds__(kThreads<D, T>) window_dq_f32_kernel(BwdArgs a) {
  constexpr int R = kRows<D, T>, TH = kThreads<D, T>;
  extern __shared__ __align__(16) float smem[];
  float *Qs = smem, *Os = Qs + T * kPitch<D>, *Vs = Os + T * kPitch<D>;
  float *Ks = Vs + TB * kPitch<D>, *Kn = Ks + TB * kPitch<D>;  // K's tile and the next one
  float *DSs = Kn + TB * kPitch<D>, *Ms = DSs + T * kPitchP, *Ds = Ms + T;
  const int N = a.N, Nk = a.win.Nk, r0 = blockIdx.x * T;
  const int64_t head = cta_head();
  if (head >= int64_t(a.Z) * a.H) return;
  const int zi = int(head / a.H), hi = int(head % a.H), hk = hi / a.win.group;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const float* k = static_cast<const float*>(a.k) + zi * a.sk.z + hk * a.sk.h;
  const float* v = static_cast<const float*>(a.v) + zi * a.sv.z + hk * a.sv.h;
  load_rows<D, T, TH>(Qs, static_cast<const float*>(a.q) + zi * a.sq.z + hi * a.sq.h, a.sq, r0, N);
  load_rows<D, T, TH>(Os, static_cast<const float*>(a.dout) + zi * a.sdo.z + hi * a.sdo.h, a.sdo, r0, N);
  int k0 = next_keys(-TB, r0, a.win);
  load_rows<D, TB, TH>(Ks, k, a.sk, k0, Nk);
  load_rows<D, TB, TH>(Vs, v, a.sv, k0, Nk);
  if (threadIdx.x < T) {
    const int row = r0 + threadIdx.x;
    Ms[threadIdx.x] = row < N ? a.m[head * N + row] : 0.f;
    Ds[threadIdx.x] = row < N ? a.delta[head * N + row] : 0.f;
  }
  float acc[R][D / 16] = {};
  const int end = min(r0 + T + a.win.off, Nk);
  for (int next; k0 < end; k0 = next) {
    cp_async_wait_all();
    __syncthreads();  // K and V are here, and K's last tile has been read
    next = next_keys(k0, r0, a.win);
    if (next < end) load_rows<D, TB, TH>(Kn, k, a.sk, next, Nk);
    float p[R][4], ds[R][4];
    p_ds<D, R, false>(a, Qs, Ks, Os, Vs, ty, tx, r0, k0, Ms, Ds, p, ds);
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) DSs[(R * ty + i) * kPitchP + tx + 16 * j] = ds[i][j];
    __syncthreads();  // V has been read
    if (next < end) load_rows<D, TB, TH>(Vs, v, a.sv, next, Nk);
    rows_times<D, R>(DSs, Ks, ty, tx, acc);
    float* t = Ks;
    Ks = Kn;
    Kn = t;
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = r0 + R * ty + i;
    if (row >= N) continue;
    float* dq = static_cast<float*>(a.dq) + (head * N + row) * D + D / 16 * tx;
#pragma unroll
    for (int e = 0; e < D / 16; ++e) dq[e] = acc[i][e] * a.sm_scale;
  }
}

// One unit (window_unit): a key tile of a key/value head, summed over the query heads that share it, or a part of
// that sum.
template <int D, int T>
__global__ void __launch_bounds__(kThreads<D, T>) window_dkdv_f32_kernel(BwdArgs a) {
  constexpr int R = kRows<D, T>, TH = kThreads<D, T>;
  extern __shared__ __align__(16) float smem[];
  float *Ks = smem, *Vs = Ks + T * kPitch<D>, *Os = Vs + T * kPitch<D>;
  float *Qs = Os + TB * kPitch<D>, *Qn = Qs + TB * kPitch<D>;  // Q's tile and the next one
  float *Ps = Qn + TB * kPitch<D>, *Ms = Ps + T * kPitchP, *Mn = Ms + 2 * TB;  // M and delta of them
  const int N = a.N, Nk = a.win.Nk;
  if (cta_head() >= int64_t(a.Z) * a.win.Hk) return;
  const WindowUnit u = window_unit<T, TB>(a.split, a.win, a.Z, N, unsigned(cta_head() * gridDim.x + blockIdx.x));
  const int k0 = T * u.kt;
  const int64_t head = u.head;
  const int zi = int(head / a.win.Hk), hk = int(head % a.win.Hk);
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  load_rows<D, T, TH>(Ks, static_cast<const float*>(a.k) + zi * a.sk.z + hk * a.sk.h, a.sk, k0, Nk);
  load_rows<D, T, TH>(Vs, static_cast<const float*>(a.v) + zi * a.sv.z + hk * a.sv.h, a.sv, k0, Nk);
  float dk[R][D / 16] = {}, dv[R][D / 16] = {};
  auto rows_of = [&](const void* x, const Strides4& st, int i, float* to) {  // the tile of pair i
    const int hi = hk * a.win.group + i / u.nb, r0 = (u.lo + i % u.nb) * TB;
    load_rows<D, TB, TH>(to, static_cast<const float*>(x) + zi * st.z + hi * st.h, st, r0, N);
  };
  auto load_q = [&](int i, float* to, float* md) {
    rows_of(a.q, a.sq, i, to);
    if (threadIdx.x < TB) {
      const int hi = hk * a.win.group + i / u.nb, row = (u.lo + i % u.nb) * TB + threadIdx.x;
      const int64_t at = (int64_t(zi) * a.H + hi) * N + row;
      md[threadIdx.x] = row < N ? a.m[at] : 0.f;
      md[TB + threadIdx.x] = row < N ? a.delta[at] : 0.f;
    }
  };
  const int end = u.start + u.n;
  if (u.n > 0) {
    load_q(u.start, Qs, Ms);
    rows_of(a.dout, a.sdo, u.start, Os);
  }
  for (int i = u.start; i < end; ++i) {
    const int r0 = (u.lo + i % u.nb) * TB;
    cp_async_wait_all();
    __syncthreads();  // Q and dO are here, and Q's last tile has been read
    if (i + 1 < end) load_q(i + 1, Qn, Mn);
    float p[R][4], ds[R][4];
    p_ds<D, R, true>(a, Ks, Qs, Vs, Os, ty, tx, k0, r0, Ms, Ms + TB, p, ds);
    auto put = [&](const float(*x)[4]) {  // a row is written and read by the 16 threads of one half warp
      __syncwarp();
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) Ps[(R * ty + i) * kPitchP + tx + 16 * j] = x[i][j];
      __syncwarp();
    };
    put(p);
    rows_times<D, R>(Ps, Os, ty, tx, dv);
    __syncthreads();  // dO has been read
    if (i + 1 < end) rows_of(a.dout, a.sdo, i + 1, Os);
    put(ds);
    rows_times<D, R>(Ps, Qs, ty, tx, dk);
    float *q = Qs, *md = Ms;
    Qs = Qn;
    Qn = q;
    Ms = Mn;
    Mn = md;
  }
  cp_async_wait_all();  // K and V, where no query sees the tile
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int key = k0 + R * ty + i;
    if (key >= Nk) continue;
    if (u.slot >= 0) {
      const int64_t slot = head * a.split.slots((Nk + T - 1) / T) + u.slot;
      float* part = a.part + (slot * 2 * T + R * ty + i) * D + D / 16 * tx;
#pragma unroll
      for (int e = 0; e < D / 16; ++e) {
        part[e] = dv[i][e];
        part[T * D + e] = dk[i][e];
      }
      continue;
    }
    const int64_t at = (head * Nk + key) * D + D / 16 * tx;
#pragma unroll
    for (int e = 0; e < D / 16; ++e) {
      static_cast<float*>(a.dk)[at + e] = dk[i][e] * a.sm_scale;
      static_cast<float*>(a.dv)[at + e] = dv[i][e];
    }
  }
}

constexpr int kJoinThreads = 256;

// dV and dK of the tiles of several units: the sums of the units' partials, in their order.
__global__ void __launch_bounds__(kJoinThreads) window_join_f32_kernel(BwdArgs a, int T, int D) {
  const int key_tiles = (a.win.Nk + T - 1) / T, tiles = a.split.units > 1 ? key_tiles : a.split.tiles;
  const int64_t i = int64_t(blockIdx.x) * kJoinThreads + threadIdx.x, tile = T * D;
  const int which = int(i / tile % 2);  // 0: dV, 1: dK
  const int64_t t = i / (2 * tile), head = t / tiles;
  const int kt = int(t % tiles), key = kt * T + int(i % tile / D);
  const bool sink = kt < a.split.tiles;
  const int count = sink ? a.split.sink_units : a.split.units;
  if (head >= int64_t(a.Z) * a.win.Hk || count == 1 || key >= a.win.Nk) return;
  const int first = sink ? kt * count : a.split.tiles * a.split.sink_units + (kt - a.split.tiles) * count;
  const float* p = a.part + ((head * a.split.slots(key_tiles) + first) * 2 + which) * tile + i % tile;
  float sum = 0.f;
  for (int c = 0; c < count; ++c) sum += p[c * 2 * tile];
  float* out = static_cast<float*>(which ? a.dk : a.dv);
  out[(head * a.win.Nk + key) * D + i % D] = which ? sum * a.sm_scale : sum;
}

template <typename Kernel, typename... Args>
cudaError_t launch(Kernel kernel, int tiles, long long heads, int threads, int floats, cudaStream_t s, const Args&... args) {
  const long long y = heads < 65535 ? heads : 65535, z = (heads + y - 1) / y;
  if (z > 65535) return cudaErrorInvalidConfiguration;
  const int smem = floats * 4;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  kernel<<<dim3(tiles, unsigned(y), unsigned(z)), threads, smem, s>>>(args...);
  return cudaGetLastError();
}

template <int D, int T>
cudaError_t fwd_impl(const float* q, const float* k, const float* v, const Strides4& sq, const Strides4& sk,
                     const Strides4& sv, const FwdArgs& a, cudaStream_t s) {
  return launch(window_fwd_f32_kernel<D, T>, (a.N + T - 1) / T, (long long)a.Z * a.H, kThreads<D, T>,
                (T + 2 * TB) * kPitch<D> + T * kPitchP, s, q, k, v, sq, sk, sv, a);
}

template <int D, int T>
cudaError_t dkdv_impl(const BwdArgs& a, cudaStream_t s) {
  const int key_tiles = (a.win.Nk + T - 1) / T;
  const cudaError_t e = launch(window_dkdv_f32_kernel<D, T>, a.split.per_head(key_tiles), (long long)a.Z * a.win.Hk, kThreads<D, T>,
                               (2 * T + 3 * TB) * kPitch<D> + T * kPitchP + 4 * TB, s, a);
  if (e != cudaSuccess || a.split.slots(key_tiles) == 0) return e;
  const int64_t values = int64_t(a.Z) * a.win.Hk * (a.split.units > 1 ? key_tiles : a.split.tiles) * 2 * T * D;
  window_join_f32_kernel<<<unsigned((values + kJoinThreads - 1) / kJoinThreads), kJoinThreads, 0, s>>>(a, T, D);
  return cudaGetLastError();
}
template <int D, int T>
cudaError_t dq_impl(const BwdArgs& a, cudaStream_t s) {
  return launch(window_dq_f32_kernel<D, T>, (a.N + T - 1) / T, (long long)a.Z * a.H, kThreads<D, T>,
                (2 * T + 3 * TB) * kPitch<D> + T * kPitchP + 2 * T, s, a);
}

template <int D>
cudaError_t fwd_tiles(const float* q, const float* k, const float* v, const Strides4& sq, const Strides4& sk,
                      const Strides4& sv, const FwdArgs& a, cudaStream_t s) {
  if constexpr (D > 16)
    if (window_f32_tile(D, (long long)a.Z * a.H, a.N) == 64) return fwd_impl<D, 64>(q, k, v, sq, sk, sv, a, s);
  return fwd_impl<D, 32>(q, k, v, sq, sk, sv, a, s);
}
template <int D>
cudaError_t bwd_tiles(const BwdArgs& a, cudaStream_t s) {
  auto of_keys = dkdv_impl<D, 32>;
  auto of_queries = dq_impl<D, 32>;
  if constexpr (D > 16) {
    if (window_f32_tile(D, (long long)a.Z * a.win.Hk, a.win.Nk) == 64) of_keys = dkdv_impl<D, 64>;
    if (window_f32_tile(D, (long long)a.Z * a.H, a.N) == 64) of_queries = dq_impl<D, 64>;
  }
  const cudaError_t e = of_keys(a, s);
  return e != cudaSuccess ? e : of_queries(a, s);
}

}  // namespace

int window_f32_tile(int D, long long heads, int rows) {
  return D == 16 || heads * ((rows + 63) / 64) < 5LL * device_sm_count() ? 32 : 64;
}

cudaError_t launch_window_fwd_f32(int D, const void* q, const void* k, const void* v, Strides4 sq, Strides4 sk,
                                  Strides4 sv, const FwdArgs& a, cudaStream_t s) {
  const float *qf = static_cast<const float*>(q), *kf = static_cast<const float*>(k), *vf = static_cast<const float*>(v);
  switch (D) {
    case 16: return fwd_tiles<16>(qf, kf, vf, sq, sk, sv, a, s);
    case 32: return fwd_tiles<32>(qf, kf, vf, sq, sk, sv, a, s);
    case 64: return fwd_tiles<64>(qf, kf, vf, sq, sk, sv, a, s);
    case 128: return fwd_tiles<128>(qf, kf, vf, sq, sk, sv, a, s);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_window_bwd_f32(int D, const BwdArgs& a, cudaStream_t s) {
  switch (D) {
    case 16: return bwd_tiles<16>(a, s);
    case 32: return bwd_tiles<32>(a, s);
    case 64: return bwd_tiles<64>(a, s);
    case 128: return bwd_tiles<128>(a, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace tattn
