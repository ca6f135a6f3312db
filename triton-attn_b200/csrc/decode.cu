// Attention of one new token of each sequence over a cache of keys and values: fp16, 4-bit and fp32 caches.
//
// Sequence z holds len = lengths[z] tokens, the newest (the query's own) at len - 1. The query sees the last
// `window` of them and the first `sinks`: t = 0 .. nvis - 1 counts those tokens in order, token(t) is where
// one lies. O = softmax(q K^T scale) V over them, in base 2; nothing seen (len = 0) gives zeros.
//
// The bound is HBM: every visible row of K and V is read once, for all the query heads that share it. A CTA
// takes one key/value head, up to 8 NT of its query heads and one of nsplit equal parts of the visible
// tokens; its warps take 16- or 32-key tiles in turn through rings of their own (cp.async, no barrier
// between warps) and keep their own running maximum and sum, which are joined at the end: within the CTA
// through shared memory, over the parts, where they are at most kClusterParts, by the cluster that they form,
// through each other's shared memory, else by a second small kernel. With few heads a matrix instruction of 8
// columns is enough: S^T = K Q^T and O^T += V^T P^T as mma.m16n8k16 with keys (then dims) as the 16 rows
// and query heads as the 8 columns, so nothing is computed for rows that do not exist, and the S^T
// accumulators become the P^T operand by one 8 x 8 transposition in registers. (tcgen05 has 64 rows at
// least and takes its operands from shared memory in its own layout; unpacked 4-bit codes would have to be
// written there first.)
//
// Measured (B200): fp16, 64 sequences of 4,096 visible tokens, 4 key/value heads of 128 for 16 query heads: 538 MB in 82
// us, 6.5 TB/s, a copy's rate. 4 bits, 16 sequences of 35,536 to 65,536 tokens, the same heads: 471 MB in 112 us, 4.2
// TB/s: there it is the making of fp16 values from codes, most of about 340 instructions for a warp's 16 keys (the fp16
// pipes are busy 49 % of the time and the integer ones 45 %). Issue slots are at 65 %: the rest is the latency of each
// subtile's shared-memory reads and conversions, which an SM's 16 warps do not cover. One sequence of 512 or 1,000
// tokens: 4.5 and 5 us, of which the launch, the loads' latency and the join are each 1 to 2. fp32: beside its kernel.
#include <cuda_fp16.h>
#include <float.h>
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace tattn {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kGroupDims = 64;  // head dims that share a scale and a minimum in the 4-bit cache

// The tokens a sequence's query sees.
struct Visible {
  int sinks, jump, n;  // t < sinks: token t; else token t + jump
  __device__ __forceinline__ int token(int t) const { return t < sinks ? t : t + jump; }
};
__device__ __forceinline__ Visible visible_tokens(const DecodeArgs& a, int z, bool report) {
  int len = a.lengths ? a.lengths[z] : a.C;
  if (len < 0 || len > a.C) {
    if (report) atomicOr(a.status, kStatusIndexRange);
    len = len < 0 ? 0 : a.C;
  }
  const int lo = max(0, len - a.window);
  Visible v;
  v.sinks = min(a.sinks, lo);
  v.jump = lo - v.sinks;
  v.n = v.sinks + len - lo;
  return v;
}

// A CTA's work: key/value head hk of sequence z, query heads [h0, h0 + heads), tokens [t0, t1) of the
// visible ones (a multiple of `tile` each, so that parts begin with whole tiles).
struct Part {
  int z, hk, h0, heads, split, t0, t1;
};
__device__ __forceinline__ Part decode_part(const DecodeArgs& a, int heads_per_cta, int tile, Visible* vis) {
  const int group = a.H / a.Hk, chunks = (group + heads_per_cta - 1) / heads_per_cta;
  int i = blockIdx.x;
  Part p;
  p.split = i % a.nsplit;
  i /= a.nsplit;
  const int first = i % chunks * heads_per_cta;
  i /= chunks;
  p.hk = i % a.Hk;
  p.z = i / a.Hk;
  p.h0 = p.hk * group + first;
  p.heads = min(heads_per_cta, group - first);
  *vis = visible_tokens(a, p.z, threadIdx.x == 0);
  const int per = ((vis->n + a.nsplit - 1) / a.nsplit + tile - 1) / tile * tile;
  p.t0 = int(min(int64_t(vis->n), int64_t(per) * p.split));
  p.t1 = min(vis->n, p.t0 + per);
  return p;
}

template <int BYTES>
__device__ __forceinline__ void cp_async_small(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(valid ? BYTES : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// Transposes an 8 x 8 matrix of 16-bit values held two to a lane (row lane / 4, columns 2 (lane % 4), + 1).
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// c[16 x 8] += a[16 x 16] b[16 x 8], fp16 with fp32 sums. Lane (g, t) = (lane / 4, lane % 4) holds of a: rows
// g, g + 8 at columns 2t, 2t + 1, then the same rows at columns 2t + 8, 2t + 9; of b: rows 2t, 2t + 1, then
// 2t + 8, 2t + 9 of column g; of c: row g, then g + 8 at columns 2t, 2t + 1.
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The same with c = a b.
__device__ __forceinline__ void mma16816_first(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// A warp's running softmax over its tiles. Lane (g, t) holds columns (query heads) 2t, 2t + 1 of each of the
// NT 8-head tiles: off = -m for a maximum m of the base-2 scores (the same in all g; the largest float before the
// first score above -infinity, infinity if the warp has no tile) and its own rows' share of the sum l. M tiles of
// 16 output dims: o[mt][nt] as mma16816's c.
template <int D, int NT>
struct WarpState {
  float off[NT][2], l[NT][2], o[D / 16][NT][4];
  __device__ __forceinline__ void reset(bool has_tile) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) off[nt][0] = off[nt][1] = has_tile ? FLT_MAX : INFINITY, l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
    for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[mt][nt][e] = 0.f;
  }
};

__device__ __forceinline__ float positive_scale(float qk_scale) {
  // Below 2^-60 scores vanish against 1: a scale of 0 gives the weights that it should and still leaves the
  // -infinity of a key that does not exist what it is. The sign goes into Q.
  return fabsf(qk_scale) < 0x1p-60f ? 0x1p-60f : fabsf(qk_scale);  // (NaN stays)
}
template <int D, int NT>
__device__ __forceinline__ void rescale(WarpState<D, NT>& st, const float (*alpha)[2]) {
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      st.l[nt][e] *= alpha[nt][e];
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt) {
        st.o[mt][nt][e] *= alpha[nt][e];
        st.o[mt][nt][2 + e] *= alpha[nt][e];
      }
    }
}

// Raw scores x[s][nt] (16-key subtile s; as mma16816's c) become p = 2^(scale (x - m)). The lane's keys are
// 16 s + row and 16 s + row + 8; those from `left` on do not exist. m, a column's maximum over the keys so far,
// is only raised (and what was summed before rescaled) where some x lies more than 2^kRaise above it in
// weight: until then p <= 2^kRaise does fp16 no harm, and a tile takes a vote in place of the maximum's
// shuffles. scale > 0 (positive_scale).
constexpr float kRaise = 8.f;
template <int D, int NT, int NS>
__device__ __forceinline__ void softmax_tile(WarpState<D, NT>& st, float (*x)[NT][4], int left, int row, float scale) {
  if (left < 16 * NS) {
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (16 * s + row + e / 2 * 8 >= left) x[s][nt][e] = -INFINITY;
  }
  float mx[NT][2];
  bool raise = false;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      mx[nt][e] = fmaxf(x[0][nt][e], x[0][nt][2 + e]);
#pragma unroll
      for (int s = 1; s < NS; ++s) mx[nt][e] = fmax3(mx[nt][e], x[s][nt][e], x[s][nt][2 + e]);
      raise |= fmaf(mx[nt][e], scale, st.off[nt][e]) > kRaise;
    }
  if (__any_sync(0xffffffffu, raise)) {
    float alpha[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int o = 4; o < 32; o *= 2) mx[nt][e] = fmaxf(mx[nt][e], __shfl_xor_sync(0xffffffffu, mx[nt][e], o));
        const float off = fminf(-scale * mx[nt][e], st.off[nt][e]);
        alpha[nt][e] = ex2_approx(off - st.off[nt][e]);  // (nothing summed yet: of zeros)
        st.off[nt][e] = off;
      }
    rescale(st, alpha);
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        x[s][nt][e] = ex2_approx(fmaf(x[s][nt][e], scale, st.off[nt][e]));
        x[s][nt][2 + e] = ex2_approx(fmaf(x[s][nt][2 + e], scale, st.off[nt][e]));
        st.l[nt][e] += x[s][nt][e] + x[s][nt][2 + e];
      }
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// The address in the cluster's CTA `rank` of what lies at `addr` in this one's shared memory, and loads from it.
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 load_cluster4(uint32_t addr) {
  float4 x;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(addr) : "memory");
  return x;
}
__device__ __forceinline__ float2 load_cluster2(uint32_t addr) {
  float2 x;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(x.x), "=f"(x.y) : "r"(addr) : "memory");
  return x;
}

// o is divided by l, the sum beside the maximum m. m = -infinity: no token is seen, and the row is zeros. l = 0
// otherwise: every score is -infinity, and the row 0 / 0.
template <int D>
__device__ __forceinline__ void write_row4(const DecodeArgs& a, int z, int h, int d, const float4& o, float m, float l) {
  const float inv = m == -INFINITY ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(static_cast<__half*>(a.o) + z * a.so.z + h * a.so.h + d) =
      make_uint2(pack_half2(o.x * inv, o.y * inv), pack_half2(o.z * inv, o.w * inv));
}

// Floats of shared memory that finish() needs: every warp's rows with their maxima and sums, and their join.
template <int D>
constexpr int finish_floats(int NT) {
  return (kWarps + 1) * 8 * NT * (D + 2);
}

// Joins the warps' results through shared memory, then the parts': writes finished rows if there is only one
// part or the parts are a cluster, else the part's unnormalised rows with their maxima and sums.
// dim(mt, half): the head dim of this lane's row g + 8 half of M tile mt.
template <int D, int NT, bool OVERLAP, typename Dim>
__device__ __forceinline__ void finish(const DecodeArgs& a, const Part& p, WarpState<D, NT>& st, float* smem, Dim dim) {
  constexpr int HEADS = 8 * NT;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  float* ml = smem + kWarps * HEADS * D;            // [warp][head][2]
  float* mine = smem + kWarps * HEADS * (D + 2);    // the CTA's [head][D], then [head][2]
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float l = st.l[nt][e];
#pragma unroll
      for (int o = 4; o < 32; o *= 2) l += __shfl_xor_sync(0xffffffffu, l, o);
      const int head = 8 * nt + 2 * t + e;
      if (g == 0) {
        ml[(warp * HEADS + head) * 2] = -st.off[nt][e];
        ml[(warp * HEADS + head) * 2 + 1] = l;
      }
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt) {
        smem[(warp * HEADS + head) * D + dim(mt, 0)] = st.o[mt][nt][e];
        smem[(warp * HEADS + head) * D + dim(mt, 1)] = st.o[mt][nt][2 + e];
      }
    }
  __syncthreads();
  if (OVERLAP) wait_for_last_kernel();
  for (int i = threadIdx.x; i < p.heads * (D / 4); i += kThreads) {
    const int head = i / (D / 4), d = i % (D / 4) * 4;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, ml[(w * HEADS + head) * 2]);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = m == -INFINITY ? 0.f : ex2_approx(ml[(w * HEADS + head) * 2] - m);
      const float4 x = *reinterpret_cast<const float4*>(smem + (w * HEADS + head) * D + d);
      l = fmaf(f, ml[(w * HEADS + head) * 2 + 1], l);
      o = make_float4(fmaf(f, x.x, o.x), fmaf(f, x.y, o.y), fmaf(f, x.z, o.z), fmaf(f, x.w, o.w));
    }
    const int h = p.h0 + head;
    if (a.nsplit == 1 && !a.parts_only) {
      write_row4<D>(a, p.z, h, d, o, m, l);
    } else if (a.nsplit <= kClusterParts && !a.parts_only) {
      *reinterpret_cast<float4*>(mine + head * D + d) = o;
      if (d == 0) *reinterpret_cast<float2*>(mine + HEADS * D + head * 2) = make_float2(m, l);
    } else {
      const int64_t row = (int64_t(p.z) * a.H + h) * a.nsplit + p.split;
      *reinterpret_cast<float4*>(a.part + row * D + d) = o;
      if (d == 0) *reinterpret_cast<float2*>(a.part_ml + row * 2) = make_float2(m, l);
    }
  }
  if (a.nsplit == 1 || a.nsplit > kClusterParts || a.parts_only) return;
  // The cluster's CTAs are the parts in order; each finishes a share of the rows.
  cluster_sync();
  const uint32_t rows = smem_u32(mine);
  for (int i = p.split * kThreads + threadIdx.x; i < p.heads * (D / 4); i += a.nsplit * kThreads) {
    const int head = i / (D / 4), d = i % (D / 4) * 4;
    float2 ml_of[kClusterParts];
    float4 x[kClusterParts];
    float m = -INFINITY;
#pragma unroll
    for (int c = 0; c < kClusterParts; ++c) {
      if (c >= a.nsplit) break;
      ml_of[c] = load_cluster2(in_cta(rows + (HEADS * D + head * 2) * 4, c));
      x[c] = load_cluster4(in_cta(rows + (head * D + d) * 4, c));
      m = fmaxf(m, ml_of[c].x);
    }
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll
    for (int c = 0; c < kClusterParts; ++c) {
      if (c >= a.nsplit) break;
      const float f = m == -INFINITY ? 0.f : ex2_approx(ml_of[c].x - m);
      l = fmaf(f, ml_of[c].y, l);
      o = make_float4(fmaf(f, x[c].x, o.x), fmaf(f, x[c].y, o.y), fmaf(f, x[c].z, o.z), fmaf(f, x[c].w, o.w));
    }
    write_row4<D>(a, p.z, p.h0 + head, d, o, m, l);
  }
  cluster_sync();  // no CTA leaves while another reads its rows
}

// ------------------------------------------------------------------------------------- fp16 cache
// Rows in shared memory keep their 16-byte units in an order that gives the 8 rows an ldmatrix reads 8
// different bank groups.
template <int D>
__device__ __forceinline__ uint32_t row_unit(int row, int unit) {
  constexpr int U = D / 8;  // units of a row
  const int x = U >= 8 ? row : U == 4 ? row >> 1 : row >> 2;
  return uint32_t(row * U + (unit ^ (x & (U >= 8 ? 7 : U - 1)))) * 16;
}

template <int D>
struct F16Cfg {
  static constexpr int KT = D == 128 ? 16 : 32, NS = KT / 16;  // keys per tile
  static constexpr int STAGES = 3;
  static constexpr int TILE = KT * D * 2;  // bytes of a K or V tile
  static constexpr int RING = kWarps * STAGES * 2 * TILE;
  static constexpr int smem(int NT) {
    const int join = finish_floats<D>(NT) * 4;
    return RING > join ? RING : join;
  }
};

// OVERLAP: the kernel runs beside the stream's last one, of which it reads nothing, and ends after it.
template <int D, int NT, bool OVERLAP>
__global__ void __launch_bounds__(kThreads) decode_f16_kernel(const DecodeArgs a) {
  using C = F16Cfg<D>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  Visible vis;
  const Part p = decode_part(a, 8 * NT, C::KT, &vis);
  const uint32_t ring = smem_u32(smem) + warp * C::STAGES * 2 * C::TILE;
  const __half* kb = static_cast<const __half*>(a.k) + p.z * a.sk.z + p.hk * a.sk.h;
  const __half* vb = static_cast<const __half*>(a.v) + p.z * a.sv.z + p.hk * a.sv.h;

  // A tile of this warp: tokens from `base` on, into ring slot `to`.
  auto load = [&](int base, uint32_t to) {
    constexpr int ROWS = 32 / (D / 8) > 0 ? 32 / (D / 8) : 1;  // rows a step of the warp copies
    const int row = lane / (D / 8), unit = lane % (D / 8);
    if (base >= vis.sinks && base + C::KT <= p.t1) {  // rows one after another
      const __half* k = kb + int64_t(base + vis.jump + row) * a.sk.n + unit * 8;
      const __half* v = vb + int64_t(base + vis.jump + row) * a.sv.n + unit * 8;
#pragma unroll
      for (int j = 0; j < C::KT / ROWS; ++j) {
        cp_async16(to + row_unit<D>(j * ROWS + row, unit), k, true);
        cp_async16(to + C::TILE + row_unit<D>(j * ROWS + row, unit), v, true);
        k += ROWS * a.sk.n;
        v += ROWS * a.sv.n;
      }
      return;
    }
#pragma unroll
    for (int j = 0; j < C::KT / ROWS; ++j) {
      const int t = base + j * ROWS + row;
      const bool in = t < p.t1;
      const int64_t tok = in ? vis.token(t) : 0;  // rows past the end are zeros
      cp_async16(to + row_unit<D>(j * ROWS + row, unit), kb + tok * a.sk.n + unit * 8, in);
      cp_async16(to + C::TILE + row_unit<D>(j * ROWS + row, unit), vb + tok * a.sv.n + unit * 8, in);
    }
  };
  // The warp's tiles begin at every kWarps * KT-th token from `base` on; the next load is STAGES - 1 ahead.
  constexpr int STEP = kWarps * C::KT;
  int base = p.t0 + warp * C::KT, slot = 0, next = C::STAGES - 1;
#pragma unroll
  for (int i = 0; i < C::STAGES - 1; ++i) {
    if (base + i * STEP < p.t1) load(base + i * STEP, ring + i * 2 * C::TILE);
    cp_async_commit();
  }

  const float scale = positive_scale(a.qk_scale);
  const uint32_t sign = a.qk_scale < 0.f ? 0x80008000u : 0u;
  // Q^T as the B operand: column g is head g, rows are dims.
  uint32_t q[D / 16][NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int head = 8 * nt + g;
    const __half* qr = static_cast<const __half*>(a.q) + p.z * a.sq.z + (p.h0 + head) * a.sq.h;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        q[kk][nt][e] =
            head < p.heads ? *reinterpret_cast<const uint32_t*>(qr + kk * 16 + 2 * t + 8 * e) ^ sign : 0u;
  }

  WarpState<D, NT> st;
  st.reset(base < p.t1);
  for (; base < p.t1; base += STEP) {
    cp_async_wait<C::STAGES - 2>();
    __syncwarp();
    const uint32_t kt = ring + slot * 2 * C::TILE, vt = kt + C::TILE;
    float x[C::NS][NT][4];
#pragma unroll
    for (int s = 0; s < C::NS; ++s) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        uint32_t f[4];  // keys 0-7, 8-15 at 8 dims, then at the next 8
        ldmatrix_x4(f, kt + row_unit<D>(16 * s + lane % 16, 2 * kk + lane / 16));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (kk == 0)
            mma16816_first(x[s][nt], f, q[kk][nt][0], q[kk][nt][1]);
          else
            mma16816(x[s][nt], f, q[kk][nt][0], q[kk][nt][1]);
        }
      }
    }
    softmax_tile<D, NT, C::NS>(st, x, p.t1 - base, g, scale);
#pragma unroll
    for (int s = 0; s < C::NS; ++s) {
      // P is rounded to fp16 for the matrix instruction (2^-12 relative on average per weight, the same as
      // the output's own rounding, and 2^-25 of the largest weight for those below 2^-14 of it); its sum l is not.
      uint32_t pt[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        pt[nt][0] = transpose8x8(pack_half2(x[s][nt][0], x[s][nt][1]));
        pt[nt][1] = transpose8x8(pack_half2(x[s][nt][2], x[s][nt][3]));
      }
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt) {
        uint32_t f[4];  // V^T: dims 0-7, 8-15 at keys 0-7, then at keys 8-15
        ldmatrix_x4_trans(f, vt + row_unit<D>(16 * s + (lane & 7) + (lane & 16) / 2, 2 * mt + (lane & 8) / 8));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma16816(st.o[mt][nt], f, pt[nt][0], pt[nt][1]);
      }
    }
    __syncwarp();  // every lane has read the slot that the next load overwrites
    if (base + (C::STAGES - 1) * STEP < p.t1) load(base + (C::STAGES - 1) * STEP, ring + next * 2 * C::TILE);
    cp_async_commit();
    slot = slot + 1 == C::STAGES ? 0 : slot + 1;
    next = next + 1 == C::STAGES ? 0 : next + 1;
  }
  cp_async_wait<0>();
  __syncthreads();  // the rings become the join's memory
  finish<D, NT, OVERLAP>(a, p, st, reinterpret_cast<float*>(smem), [&](int mt, int half) { return 16 * mt + 8 * half + g; });
}

// ------------------------------------------------------------------------------------ 4-bit cache
// A group of 64 head dims of a row is 32 bytes of codes n (0 .. 15) with a scale s and a minimum m; it stands
// for the fp16 values s n + m, which are what the matrix instructions take. Four bits become fp16 without a
// conversion: in the low (high) half of a byte's 8 bits, under the exponent of 1024, where an fp16's last place is 1,
// they are 1024 + n (1024 + 16 n; a published technique: Kim, Henry, Fahim, Awadalla 2022), from which one subtraction (one fused multiply-add by 1/16) leaves n exactly and another
// fused multiply-add s n + m, rounded once. Two codes an instruction, and 5 (K) to 6 (V) integer instructions for 8
// codes.
template <int D>
struct Int4Cfg {
  static constexpr int KT = 32, NS = KT / 16, GR = D / kGroupDims;
  static constexpr int STAGES = 3;
  static constexpr int CODES = KT * D / 2, PARAMS = KT * GR * 4;  // bytes of a tile
  static constexpr int TILE = 2 * (CODES + PARAMS);               // K codes, V codes, K params, V params
  static constexpr int RING = kWarps * STAGES * TILE;
  static constexpr int smem(int NT) {
    const int join = finish_floats<D>(NT) * 4;
    return RING > join ? RING : join;
  }
  // Where a group's 32 bytes lie in a tile: so that the four rows a quarter of the lanes reads at a time, 0, 4,
  // 1, 5 or 2, 6, 3, 7 (K) and 0 .. 3 or 4 .. 7 (V) of every 8, are in different banks.
  static __device__ __forceinline__ uint32_t at(int row, int group) {
    if (GR == 2) return uint32_t(row * 64 + (group ^ (((row >> 1) ^ (row >> 2)) & 1)) * 32);
    return uint32_t((row ^ ((row >> 1) & 2)) * 32);
  }
};

__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t x;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x) : "r"(addr) : "memory");
  return x;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 x;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(x.x), "=r"(x.y) : "r"(addr) : "memory");
  return x;
}
__device__ __forceinline__ __half2 as_half2(uint32_t x) { return *reinterpret_cast<const __half2*>(&x); }
__device__ __forceinline__ uint32_t as_bits(__half2 x) { return *reinterpret_cast<const uint32_t*>(&x); }
// The values of the codes in the low (HIGH: high) 4 bits of bytes 0 and 2 of `word`. k1024: 1024 twice, in a
// register (an instruction has room for one constant, the mask; with two the compiler makes two of it).
template <bool HIGH>
__device__ __forceinline__ uint32_t code_values(uint32_t word, __half2 s, __half2 m, uint32_t k1024) {
  uint32_t bits;  // (word & mask) | k1024
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(bits) : "r"(word), "n"(HIGH ? 0x00f000f0u : 0x000f000fu), "r"(k1024));
  const __half2 x = as_half2(bits);
  const __half2 n = HIGH ? __hfma2(x, __float2half2_rn(0.0625f), __float2half2_rn(-64.f))
                         : __hadd2(x, __float2half2_rn(-1024.f));
  return as_bits(__hfma2(s, n, m));
}

template <int D, int NT>
__global__ void __launch_bounds__(kThreads) decode_int4_kernel(const DecodeArgs a) {
  using C = Int4Cfg<D>;
  constexpr int GR = C::GR;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  Visible vis;
  const Part p = decode_part(a, 8 * NT, C::KT, &vis);
  const uint32_t ring = smem_u32(smem) + warp * C::STAGES * C::TILE;
  const int64_t row0 = (int64_t(p.z) * a.Hk + p.hk) * a.C;
  const uint8_t* codes[2] = {static_cast<const uint8_t*>(a.k) + row0 * (D / 2), static_cast<const uint8_t*>(a.v) + row0 * (D / 2)};
  const uint8_t* params[2] = {static_cast<const uint8_t*>(a.k_params) + row0 * (GR * 4),
                              static_cast<const uint8_t*>(a.v_params) + row0 * (GR * 4)};

  // A tile of this warp: tokens from `base` on, into ring slot `to`. Rows one after another are one run of
  // bytes; the lane's place in the slot is the same for every 32 units of 16 bytes (8 or 16 rows).
  const uint32_t place = C::at(lane / (D / 32), lane % (D / 32) / 2) + lane % 2 * 16;
  auto load = [&](int base, uint32_t to) {
    if (base >= vis.sinks && base + C::KT <= p.t1) {
      const int64_t tok = base + vis.jump;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint8_t* src = codes[x] + tok * (D / 2) + lane * 16;
#pragma unroll
        for (int j = 0; j < C::CODES / 512; ++j) cp_async16(to + x * C::CODES + place + j * 512, src + j * 512, true);
        cp_async_small<GR * 4>(to + 2 * C::CODES + x * C::PARAMS + lane * GR * 4, params[x] + (tok + lane) * (GR * 4), true);
      }
      return;
    }
#pragma unroll
    for (int j = 0; j < C::CODES / 512; ++j) {
      const int e = j * 32 + lane, t = base + e / (D / 32), unit = e % (D / 32);
      const bool in = t < p.t1;
      const int64_t tok = in ? vis.token(t) : 0;  // rows past the end are zeros
#pragma unroll
      for (int x = 0; x < 2; ++x)
        cp_async16(to + x * C::CODES + place + j * 512, codes[x] + tok * (D / 2) + unit * 16, in);
    }
    const bool in = base + lane < p.t1;
    const int64_t tok = in ? vis.token(base + lane) : 0;
#pragma unroll
    for (int x = 0; x < 2; ++x)
      cp_async_small<GR * 4>(to + 2 * C::CODES + x * C::PARAMS + lane * GR * 4, params[x] + tok * (GR * 4), in);
  };
  constexpr int STEP = kWarps * C::KT;
  int base = p.t0 + warp * C::KT, slot = 0, next = C::STAGES - 1;
#pragma unroll
  for (int i = 0; i < C::STAGES - 1; ++i) {
    if (base + i * STEP < p.t1) load(base + i * STEP, ring + i * C::TILE);
    cp_async_commit();
  }
  const float scale = positive_scale(a.qk_scale);
  const uint32_t sign = a.qk_scale < 0.f ? 0x80008000u : 0u;

  // Q^T as the B operand (column g is head g), its rows in the order in which the codes of K come out of
  // their words: lane t holds 16 dims of each group, step j of 4 takes codes 2 (j % 2), + 4, + 1, + 5 of
  // word j / 2.
  uint32_t q[GR][4][NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int head = 8 * nt + g;
    const bool has = head < p.heads;
    const __half* qr = static_cast<const __half*>(a.q) + p.z * a.sq.z + (p.h0 + (has ? head : 0)) * a.sq.h + 16 * t;
#pragma unroll
    for (int gr = 0; gr < GR; ++gr)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const uint4 x = has ? *reinterpret_cast<const uint4*>(qr + gr * kGroupDims + 8 * w) : make_uint4(0u, 0u, 0u, 0u);
        const uint32_t u[4] = {x.x ^ sign, x.y ^ sign, x.z ^ sign, x.w ^ sign};  // dims 0,1 | 2,3 | 4,5 | 6,7
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          q[gr][2 * w + j][nt][0] = __byte_perm(u[j], u[j + 2], 0x5410);  // dims 2j, 2j + 4
          q[gr][2 * w + j][nt][1] = __byte_perm(u[j], u[j + 2], 0x7632);  // dims 2j + 1, 2j + 5
        }
      }
  }

  WarpState<D, NT> st;
  st.reset(base < p.t1);
  // Keys in the order of mma16816's rows lie in the tile's rows (k >> 1) + 4 (k & 1) of each 8.
  const int row = (g >> 1) | ((g & 1) << 2);
  // The lane's places in a slot: of rows `row` (K) and t, t + 4 (V), the same in every 8 rows but for 8 ROW.
  constexpr uint32_t ROW = D / 2;
  uint32_t at_k[GR], at_v[GR][2];
#pragma unroll
  for (int gr = 0; gr < GR; ++gr) {
    at_k[gr] = C::at(row, gr) + 8 * t;
    at_v[gr][0] = C::CODES + C::at(t, gr) + 4 * g;
    at_v[gr][1] = C::CODES + C::at(t + 4, gr) + 4 * g;
  }
  uint32_t k1024;
  asm volatile("mov.b32 %0, 0x64006400;" : "=r"(k1024));
  const uint32_t at_kp = 2 * C::CODES + row * GR * 4, at_vp = 2 * C::CODES + C::PARAMS + t * GR * 4;
  for (; base < p.t1; base += STEP) {
    cp_async_wait<C::STAGES - 2>();
    __syncwarp();
    const uint32_t tile = ring + slot * C::TILE;
    float x[C::NS][NT][4];
#pragma unroll
    for (int s = 0; s < C::NS; ++s) {
#pragma unroll
      for (int gr = 0; gr < GR; ++gr) {
        const uint2 lo = lds64(tile + at_k[gr] + 16 * s * ROW), hi = lds64(tile + at_k[gr] + (16 * s + 8) * ROW);
        const __half2 pl = as_half2(lds32(tile + at_kp + (16 * s * GR + gr) * 4));
        const __half2 ph = as_half2(lds32(tile + at_kp + ((16 * s + 8) * GR + gr) * 4));
        const __half2 sl = __low2half2(pl), ml = __high2half2(pl), sh = __low2half2(ph), mh = __high2half2(ph);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t wl = (j < 2 ? lo.x : lo.y) >> (j % 2 * 8), wh = (j < 2 ? hi.x : hi.y) >> (j % 2 * 8);
          const uint32_t f[4] = {code_values<false>(wl, sl, ml, k1024), code_values<false>(wh, sh, mh, k1024),
                                 code_values<true>(wl, sl, ml, k1024), code_values<true>(wh, sh, mh, k1024)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if (gr == 0 && j == 0)
              mma16816_first(x[s][nt], f, q[gr][j][nt][0], q[gr][j][nt][1]);
            else
              mma16816(x[s][nt], f, q[gr][j][nt][0], q[gr][j][nt][1]);
          }
        }
      }
    }
    softmax_tile<D, NT, C::NS>(st, x, p.t1 - base, row, scale);
#pragma unroll
    for (int s = 0; s < C::NS; ++s) {
      uint32_t pt[NT][2];  // P, rounded as in the fp16 path
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        pt[nt][0] = transpose8x8(pack_half2(x[s][nt][0], x[s][nt][1]));
        pt[nt][1] = transpose8x8(pack_half2(x[s][nt][2], x[s][nt][3]));
      }
#pragma unroll
      for (int gr = 0; gr < GR; ++gr) {
        // Key rows t, t + 4 (then + 8, + 12) are columns 2t, 2t + 1 (then 2t + 8, 2t + 9) of V^T; lane g holds
        // 8 dims of the group, two of them for each M tile: byte mt of the rows' words.
        uint32_t w[4], par[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          w[r] = lds32(tile + at_v[gr][r % 2] + (16 * s + r / 2 * 8) * ROW);
          par[r] = lds32(tile + at_vp + ((16 * s + 4 * r) * GR + gr) * 4);
        }
        __half2 sv[2], mv[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          sv[r] = as_half2(__byte_perm(par[2 * r], par[2 * r + 1], 0x5410));
          mv[r] = as_half2(__byte_perm(par[2 * r], par[2 * r + 1], 0x7632));
        }
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
          const uint32_t first = __byte_perm(w[0], w[1], mt | (4 + mt) << 8), second = __byte_perm(w[2], w[3], mt | (4 + mt) << 8);
          const uint32_t f[4] = {code_values<false>(first, sv[0], mv[0], k1024), code_values<true>(first, sv[0], mv[0], k1024),
                                 code_values<false>(second, sv[1], mv[1], k1024), code_values<true>(second, sv[1], mv[1], k1024)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816(st.o[4 * gr + mt][nt], f, pt[nt][0], pt[nt][1]);
        }
      }
    }
    __syncwarp();  // every lane has read the slot that the next load overwrites
    if (base + (C::STAGES - 1) * STEP < p.t1) load(base + (C::STAGES - 1) * STEP, ring + next * C::TILE);
    cp_async_commit();
    slot = slot + 1 == C::STAGES ? 0 : slot + 1;
    next = next + 1 == C::STAGES ? 0 : next + 1;
  }
  cp_async_wait<0>();
  __syncthreads();  // the rings become the join's memory
  finish<D, NT, false>(a, p, st, reinterpret_cast<float*>(smem),
                [&](int mt, int half) { return mt / 4 * kGroupDims + 8 * g + 2 * (mt % 4) + half; });
}

// ------------------------------------------------------------------------------------- fp32 cache
// fp32 throughout, on CUDA cores: a CTA takes one query head, a warp every kWarps-th group of U tokens, its lanes the
// head dims. K and V of a head that query heads share are read once for each of them, from L2 where they fit it.
// Measured (B200, 16 sequences of 8,192 tokens, D 128): 16 key/value heads for 16 query heads, 2.1 GB in 358 us, 6.0
// TB/s; 4 for 16, 0.54 GB in 324 us, 1.7 TB/s of those bytes and 6.6 of those asked for: the fourfold reading bounds it.
// One sequence of 1,000 tokens, 16 heads of 64: 7.3 us.
template <int D, bool OVERLAP>
__global__ void __launch_bounds__(kThreads) decode_f32_kernel(const DecodeArgs a) {
  constexpr int E = D >= 32 ? D / 32 : 1, U = 4;  // dims a lane, tokens at a time
  __shared__ float so[kWarps][D], sml[kWarps][2];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  Visible vis;
  const Part p = decode_part(a, 1, U, &vis);
  const bool has = lane * E < D;
  const int d = has ? lane * E : 0;
  const float* q = static_cast<const float*>(a.q) + p.z * a.sq.z + p.h0 * a.sq.h + d;
  const float* kb = static_cast<const float*>(a.k) + p.z * a.sk.z + p.hk * a.sk.h + d;
  const float* vb = static_cast<const float*>(a.v) + p.z * a.sv.z + p.hk * a.sv.h + d;
  float qv[E], o[E], m = p.t0 + warp * U < p.t1 ? -FLT_MAX : -INFINITY, l = 0.f;  // as WarpState's -off
#pragma unroll
  for (int e = 0; e < E; ++e) {
    qv[e] = has ? q[e] * a.qk_scale : 0.f;
    o[e] = 0.f;
  }
  for (int t = p.t0 + warp * U; t < p.t1; t += kWarps * U) {
    float x[U], v[U][E];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = t + u < p.t1;
      const int64_t tok = in ? vis.token(t + u) : 0;
      x[u] = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        x[u] = fmaf(in ? kb[tok * a.sk.n + e] : 0.f, qv[e], x[u]);
        v[u][e] = in ? vb[tok * a.sv.n + e] : 0.f;
      }
    }
    float mx = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int s = 1; s < 32; s *= 2) x[u] += __shfl_xor_sync(0xffffffffu, x[u], s);
      if (t + u >= p.t1) x[u] = -INFINITY;
      mx = fmaxf(mx, x[u]);
    }
    const float alpha = exp2f(m - mx);
    m = mx;
    l *= alpha;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= alpha;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float w = exp2f(x[u] - m);
      l += w;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(w, v[u][e], o[e]);
    }
  }
  if (has)
#pragma unroll
    for (int e = 0; e < E; ++e) so[warp][d + e] = o[e];
  if (lane == 0) {
    sml[warp][0] = m;
    sml[warp][1] = l;
  }
  __syncthreads();
  if (OVERLAP) wait_for_last_kernel();
  for (int c = threadIdx.x; c < D; c += kThreads) {
    m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, sml[w][0]);
    float acc = 0.f;
    l = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = m == -INFINITY ? 0.f : exp2f(sml[w][0] - m);
      l = fmaf(f, sml[w][1], l);
      acc = fmaf(f, so[w][c], acc);
    }
    if (a.nsplit == 1 && !a.parts_only) {
      static_cast<float*>(a.o)[p.z * a.so.z + p.h0 * a.so.h + c] = m == -INFINITY ? 0.f : acc / l;
    } else {
      const int64_t row = (int64_t(p.z) * a.H + p.h0) * a.nsplit + p.split;
      a.part[row * D + c] = acc;
      if (c == 0) *reinterpret_cast<float2*>(a.part_ml + row * 2) = make_float2(m, l);
    }
  }
}

// Joins the parts of each query head: one CTA a head, whose threads take 4 dims of every so many-th part.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) decode_join_kernel(const DecodeArgs a) {
  constexpr int V = D / 4, LANES = kThreads / V;  // threads of a row, rows in flight
  __shared__ float4 so[LANES][V];
  __shared__ float sl[LANES];
  const int row = blockIdx.x, t = threadIdx.x % V, p = threadIdx.x / V;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + int64_t(row) * a.nsplit;
  float m = -INFINITY;
  for (int s = threadIdx.x % 32; s < a.nsplit; s += 32) m = fmaxf(m, ml[s].x);
#pragma unroll
  for (int o = 1; o < 32; o *= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float use = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  const float4* o = reinterpret_cast<const float4*>(a.part) + int64_t(row) * a.nsplit * V + t;
#pragma unroll 4
  for (int s = p; s < a.nsplit; s += LANES) {
    const float2 x = ml[s];
    const float4 v = o[int64_t(s) * V];
    const float f = exp2f(x.x - use);
    l = fmaf(f, x.y, l);
    acc = make_float4(fmaf(f, v.x, acc.x), fmaf(f, v.y, acc.y), fmaf(f, v.z, acc.z), fmaf(f, v.w, acc.w));
  }
  so[p][t] = acc;
  if (t == 0) sl[p] = l;
  __syncthreads();
  if (p > 0) return;
#pragma unroll
  for (int q = 1; q < LANES; ++q) {
    const float4 v = so[q][t];
    acc = make_float4(acc.x + v.x, acc.y + v.y, acc.z + v.z, acc.w + v.w);
    l += sl[q];
  }
  const int z = row / a.H, h = row % a.H;
  if constexpr (sizeof(T) == 2) {
    write_row4<D>(a, z, h, 4 * t, acc, m, l);
  } else {
    float* out = static_cast<float*>(a.o) + z * a.so.z + h * a.so.h + 4 * t;
    const float den = m == -INFINITY ? 1.f : l;  // (acc is 0 then)
    *reinterpret_cast<float4*>(out) = make_float4(acc.x / den, acc.y / den, acc.z / den, acc.w / den);
  }
}

// `cluster`: the parts of a unit, which are neighbours in the grid, as one cluster.
template <typename K>
cudaError_t launch(K kernel, int smem, long long units, bool cluster, const DecodeArgs& a, cudaStream_t s, bool overlap = false) {
  if (units * a.nsplit > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t c{};
  c.gridDim = dim3(unsigned(units * a.nsplit));
  c.blockDim = dim3(kThreads);
  c.dynamicSmemBytes = size_t(smem);
  c.stream = s;
  cudaLaunchAttribute attr[2] = {};
  if (cluster) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(a.nsplit);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  }
  if (overlap) attr[cluster ? 1 : 0] = overlapping_launch();
  c.attrs = attr;
  c.numAttrs = unsigned(cluster) + unsigned(overlap);
  return cudaLaunchKernelEx(&c, kernel, a);
}

// CTAs before splitting: sequences, key/value heads and chunks of their query heads.
long long decode_units(const DecodeArgs& a, int heads_per_cta) {
  const int group = a.H / a.Hk;
  return (long long)a.Z * a.Hk * ((group + heads_per_cta - 1) / heads_per_cta);
}

template <int D>
cudaError_t decode_impl(DecodeCache cache, const DecodeArgs& a, cudaStream_t s) {
  const bool join = decode_joins(a.nsplit, cache) && !a.parts_only, wide = a.H / a.Hk > 8;
  const bool cluster = a.nsplit > 1 && !decode_joins(a.nsplit, cache) && !a.parts_only;
  cudaError_t e;
  if (cache == kCacheF32) {
    e = a.overlap ? launch(decode_f32_kernel<D, true>, 0, decode_units(a, 1), false, a, s, true)
                    : launch(decode_f32_kernel<D, false>, 0, decode_units(a, 1), false, a, s);
  } else if (cache == kCacheF16 && a.overlap) {
    e = wide ? launch(decode_f16_kernel<D, 2, true>, F16Cfg<D>::smem(2), decode_units(a, 16), cluster, a, s, true)
             : launch(decode_f16_kernel<D, 1, true>, F16Cfg<D>::smem(1), decode_units(a, 8), cluster, a, s, true);
  } else if (cache == kCacheF16) {
    e = wide ? launch(decode_f16_kernel<D, 2, false>, F16Cfg<D>::smem(2), decode_units(a, 16), cluster, a, s)
             : launch(decode_f16_kernel<D, 1, false>, F16Cfg<D>::smem(1), decode_units(a, 8), cluster, a, s);
  } else if constexpr (D % kGroupDims == 0) {
    e = wide ? launch(decode_int4_kernel<D, 2>, Int4Cfg<D>::smem(2), decode_units(a, 16), cluster, a, s)
             : launch(decode_int4_kernel<D, 1>, Int4Cfg<D>::smem(1), decode_units(a, 8), cluster, a, s);
  } else {
    e = cudaErrorNotSupported;
  }
  if (e != cudaSuccess || !join) return e;
  if (cache == kCacheF32)
    decode_join_kernel<float, D><<<unsigned(a.Z * a.H), kThreads, 0, s>>>(a);
  else
    decode_join_kernel<__half, D><<<unsigned(a.Z * a.H), kThreads, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

int decode_splits(const DecodeArgs& a, int D, DecodeCache cache) {
  const int heads = cache == kCacheF32 ? 1 : a.H / a.Hk <= 8 ? 8 : 16;
  const long long units = decode_units(a, heads);
  if (units == 0) return 1;
  const long long most = a.window < a.C ? std::min<long long>(a.C, (long long)a.window + a.sinks) : a.C;
  // Enough CTAs to fill the GPU several times over, none with less than a tile for each warp.
  const int tile = kWarps * (cache == kCacheF32 ? 4 : cache == kCacheF16 && D == 128 ? 16 : 32);
  const long long want = (decode_ctas(cache) * (long long)device_sm_count() + units - 1) / units;
  const long long n = std::max<long long>(1, std::min<long long>(want, (most + tile - 1) / tile));
  // A few parts more than a cluster has are not worth a second kernel where parts are short.
  return int(decode_joins(int(n), cache) && n <= 2 * kClusterParts && most <= kClusterParts * 2048 && cache != kCacheF32 ? kClusterParts : n);
}

cudaError_t launch_decode(int D, DecodeCache cache, const DecodeArgs& a, cudaStream_t s) {
  if (a.Z * a.H == 0) return cudaSuccess;
  switch (D) {
    case 16: return decode_impl<16>(cache, a, s);
    case 32: return decode_impl<32>(cache, a, s);
    case 64: return decode_impl<64>(cache, a, s);
    case 128: return decode_impl<128>(cache, a, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace tattn
