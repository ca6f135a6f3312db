// C-ABI boundary (include/tattn.h) of the operators around the attention kernels: head norms with rotation,
// the 4-bit cache, and the attention of single tokens over a cache.
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/tattn.h"
#include "kernels.h"

using namespace tattn;

namespace {

bool head_dim_ok(int D) { return D == 16 || D == 32 || D == 64 || D == 128; }

// [Z, H, N, D] rows read and written 16 bytes at a time. Strides of extent-1 dimensions never move an
// address and are ignored.
bool rows16(const void* p, const int64_t* s, int Z, int H, int N, int esz) {
  if (s[3] != 1 || (reinterpret_cast<uintptr_t>(p) & 15u) != 0) return false;
  const int extent[3] = {Z, H, N};
  for (int i = 0; i < 3; ++i)
    if (extent[i] > 1 && (s[i] * esz) % 16 != 0) return false;
  return true;
}

Strides3 strides3(const int64_t* s) { return Strides3{s[0], s[1], s[2]}; }

// The arguments of both rotations but for the positions' strides. strides: of q, k, q_out, k_out (backward: of q, k,
// q_grad, k_grad, dq, dk).
int rope_args(RopeArgs& a, bool backward, const int64_t* strides, int Z, int H, int Hk, int N, int P, int dtype, int w_dtype) {
  const int esz = dtype == TATTN_F16 ? 2 : 4, heads[2] = {H, Hk};
  for (int i = 0; i < 2; ++i) {
    RopeTensor& t = a.t[i];
    const int64_t *sx = strides + 4 * i, *sdy = strides + 8 + 4 * i, *sy = strides + (backward ? 16 : 8) + 4 * i;
    if (!rows16(t.px, sx, Z, heads[i], N, esz) || (backward && !rows16(t.pdy, sdy, Z, heads[i], N, esz)) ||
        !rows16(t.py, sy, Z, heads[i], N, esz) || (reinterpret_cast<uintptr_t>(t.w) & 15u) != 0)
      return TATTN_ERR_LAYOUT;
    t.x = strides3(sx);
    t.dy = strides3(sdy);
    t.y = strides3(sy);
    t.H = heads[i];
  }
  if (((reinterpret_cast<uintptr_t>(a.cos) | reinterpret_cast<uintptr_t>(a.sin)) & 15u) != 0) return TATTN_ERR_LAYOUT;
  a.Z = Z;
  a.N = N;
  a.P = P;
  a.w_f32 = w_dtype == TATTN_F32;
  return device_ready(&a.status);
}

int norm_rope(RopeArgs& a, bool backward, const int64_t* strides, int Z, int H, int Hk, int N, int D, int P, int dtype,
              int w_dtype, int interleaved, void* stream) {
  const int rc = rope_args(a, backward, strides, Z, H, Hk, N, P, dtype, w_dtype);
  if (rc != TATTN_OK) return rc;
  const int64_t* pos = strides + (backward ? 24 : 16);
  a.pos_z = pos[0];
  a.pos_n = pos[1];
  return cuda_rc(launch_norm_rope(D, dtype == TATTN_F16, interleaved != 0, backward, a, static_cast<cudaStream_t>(stream)));
}

int rope_axes(RopeAxesArgs& a, bool norm, bool backward, const int64_t* strides, const int64_t* pos, int Z, int H, int Hk, int N,
              int D, int P, int dtype, int w_dtype, int interleaved, void* stream) {
  const int rc = rope_args(a, backward, strides, Z, H, Hk, N, P, dtype, w_dtype);
  if (rc != TATTN_OK) return rc;
  a.pos_a = pos[0];
  a.pos_z = pos[1];
  a.pos_n = pos[2];
  return cuda_rc(launch_rope_axes(D, dtype == TATTN_F16, norm, interleaved != 0, backward, a, static_cast<cudaStream_t>(stream)));
}

int norm_rope_dims(int Z, int H, int Hk, int N, int D, int P, int dtype, int w_dtype) {
  if (Z < 0 || N < 0 || H < 1 || Hk < 1 || !head_dim_ok(D) || P < 0 || (dtype != TATTN_F16 && dtype != TATTN_F32) ||
      (w_dtype != dtype && w_dtype != TATTN_F32))
    return TATTN_ERR_INVALID_ARGUMENT;
  // int item counts in the kernel, with room for a last stride past them
  if (int64_t(Z) * N >= (1 << 30) / (H > Hk ? H : Hk)) return TATTN_ERR_TOO_LARGE;
  if (P == 0 && int64_t(Z) * N > 0) return TATTN_ERR_INVALID_ARGUMENT;
  return TATTN_OK;
}

}  // namespace

extern "C" int tattn_qk_norm_rope(const void* q, const void* k, const void* wq, const void* wk, void* q_out, void* k_out,
                                  const float* cos, const float* sin, const int32_t* positions, const int64_t* strides,
                                  int Z, int H, int Hk, int N, int D, int P, int dtype, int w_dtype, float eps,
                                  int interleaved, void* stream) {
  if (!strides) return TATTN_ERR_INVALID_ARGUMENT;
  const int rc = norm_rope_dims(Z, H, Hk, N, D, P, dtype, w_dtype);
  if (rc != TATTN_OK) return rc;
  if (int64_t(Z) * N == 0) return TATTN_OK;
  if (!q || !k || !wq || !wk || !q_out || !k_out || !cos || !sin) return TATTN_ERR_INVALID_ARGUMENT;
  RopeArgs a{};
  a.t[0].px = q;
  a.t[1].px = k;
  a.t[0].py = q_out;
  a.t[1].py = k_out;
  a.t[0].w = wq;
  a.t[1].w = wk;
  a.cos = cos;
  a.sin = sin;
  a.positions = positions;
  a.eps = eps;
  return norm_rope(a, false, strides, Z, H, Hk, N, D, P, dtype, w_dtype, interleaved, stream);
}

extern "C" int tattn_qk_norm_rope_bwd(const void* q, const void* k, const void* wq, const void* wk, const void* q_grad,
                                      const void* k_grad, void* dq, void* dk, void* dwq, void* dwk, const float* cos,
                                      const float* sin, const int32_t* positions, void* workspace,
                                      const int64_t* strides, int Z, int H, int Hk, int N, int D, int P, int dtype,
                                      int w_dtype, float eps, int interleaved, void* stream) {
  if (!strides) return TATTN_ERR_INVALID_ARGUMENT;
  const int rc = norm_rope_dims(Z, H, Hk, N, D, P, dtype, w_dtype);
  if (rc != TATTN_OK) return rc;
  if (!dwq || !dwk || !workspace) return TATTN_ERR_INVALID_ARGUMENT;
  if (int64_t(Z) * N > 0 && (!q || !k || !wq || !wk || !q_grad || !k_grad || !dq || !dk || !cos || !sin))
    return TATTN_ERR_INVALID_ARGUMENT;
  RopeArgs a{};
  a.t[0].px = q;
  a.t[1].px = k;
  a.t[0].pdy = q_grad;
  a.t[1].pdy = k_grad;
  a.t[0].py = dq;
  a.t[1].py = dk;
  a.t[0].w = wq;
  a.t[1].w = wk;
  a.t[0].dw = dwq;
  a.t[1].dw = dwk;
  a.cos = cos;
  a.sin = sin;
  a.positions = positions;
  a.eps = eps;
  a.part = static_cast<float*>(workspace);
  return norm_rope(a, true, strides, Z, H, Hk, N, D, P, dtype, w_dtype, interleaved, stream);
}

extern "C" int64_t tattn_qk_norm_rope_bwd_workspace_bytes(int D) {
  if (!head_dim_ok(D)) return -1;
  return (int64_t(kRopeBlocksPerSm) * device_sm_count() + 2) * D * 4;
}

namespace {

// The axis of each pair into a.axes; false where one is outside [0, A).
bool pair_axes(RopeAxesArgs& a, const int32_t* axes, int A, int D) {
  if (!axes || A < 1 || A > kRopeAxes) return false;
  a.A = A;
  for (int j = 0; j < D / 2; ++j) {
    if (axes[j] < 0 || axes[j] >= A) return false;
    a.axes[j / 16] |= uint32_t(axes[j]) << (2 * (j % 16));
  }
  return true;
}

}  // namespace

extern "C" int tattn_qk_rope_axes(const void* q, const void* k, const void* wq, const void* wk, void* q_out, void* k_out,
                                  const float* cos, const float* sin, const int32_t* positions, const int32_t* axes,
                                  const int64_t* strides, int Z, int H, int Hk, int N, int D, int P, int A, int dtype,
                                  int w_dtype, float eps, int interleaved, void* stream) {
  if (!strides) return TATTN_ERR_INVALID_ARGUMENT;
  const int rc = norm_rope_dims(Z, H, Hk, N, D, P, dtype, w_dtype);
  if (rc != TATTN_OK) return rc;
  RopeAxesArgs a{};
  if (!pair_axes(a, axes, A, D) || (wq == nullptr) != (wk == nullptr)) return TATTN_ERR_INVALID_ARGUMENT;
  if (int64_t(Z) * N == 0) return TATTN_OK;
  if (!q || !k || !q_out || !k_out || !cos || !sin || !positions) return TATTN_ERR_INVALID_ARGUMENT;
  a.t[0].px = q;
  a.t[1].px = k;
  a.t[0].py = q_out;
  a.t[1].py = k_out;
  a.t[0].w = wq;
  a.t[1].w = wk;
  a.cos = cos;
  a.sin = sin;
  a.positions = positions;
  a.eps = eps;
  return rope_axes(a, wq != nullptr, false, strides, strides + 16, Z, H, Hk, N, D, P, dtype, w_dtype, interleaved, stream);
}

extern "C" int tattn_qk_rope_axes_bwd(const void* q, const void* k, const void* wq, const void* wk, const void* q_grad,
                                      const void* k_grad, void* dq, void* dk, void* dwq, void* dwk, const float* cos,
                                      const float* sin, const int32_t* positions, const int32_t* axes, void* workspace,
                                      const int64_t* strides, int Z, int H, int Hk, int N, int D, int P, int A, int dtype,
                                      int w_dtype, float eps, int interleaved, void* stream) {
  if (!strides) return TATTN_ERR_INVALID_ARGUMENT;
  const int rc = norm_rope_dims(Z, H, Hk, N, D, P, dtype, w_dtype);
  if (rc != TATTN_OK) return rc;
  RopeAxesArgs a{};
  const bool norm = wq != nullptr, any = int64_t(Z) * N > 0;
  if (!pair_axes(a, axes, A, D) || norm != (wk != nullptr) || (norm && (!dwq || !dwk || !workspace)))
    return TATTN_ERR_INVALID_ARGUMENT;
  if (any && (!q_grad || !k_grad || !dq || !dk || !cos || !sin || !positions || (norm && (!q || !k))))
    return TATTN_ERR_INVALID_ARGUMENT;
  a.cos = cos;
  a.sin = sin;
  a.positions = positions;
  a.t[0].py = dq;
  a.t[1].py = dk;
  if (!norm) {  // the gradients turned back
    if (!any) return TATTN_OK;
    a.t[0].px = q_grad;
    a.t[1].px = k_grad;
    a.back = 1;
    return rope_axes(a, false, false, strides + 8, strides + 24, Z, H, Hk, N, D, P, dtype, w_dtype, interleaved, stream);
  }
  a.t[0].px = q;
  a.t[1].px = k;
  a.t[0].pdy = q_grad;
  a.t[1].pdy = k_grad;
  a.t[0].w = wq;
  a.t[1].w = wk;
  a.t[0].dw = dwq;
  a.t[1].dw = dwk;
  a.eps = eps;
  a.part = static_cast<float*>(workspace);
  return rope_axes(a, true, true, strides, strides + 24, Z, H, Hk, N, D, P, dtype, w_dtype, interleaved, stream);
}

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// The sizes that every single-token call shares; `a` gets them. window <= 0: everything.
bool decode_dims(DecodeArgs& a, int Z, int H, int Hk, int C, int D, int window, int sinks) {
  if (Z < 0 || H < 1 || Hk < 1 || H % Hk != 0 || C < 0 || C > (1 << 30) || !head_dim_ok(D) || sinks < 0 || int64_t(Z) * H > 0x3fffffff)
    return false;
  a.Z = Z;
  a.H = H;
  a.Hk = Hk;
  a.C = C;
  a.window = window > 0 && window < C ? window : C;
  a.sinks = sinks < C ? sinks : C;
  return true;
}

int64_t decode_workspace(const DecodeArgs& a, int D, DecodeCache cache) {
  const int nsplit = decode_splits(a, D, cache);
  return decode_joins(nsplit, cache) ? int64_t(a.Z) * a.H * nsplit * (D + 2) * 4 : 0;
}

int decode(DecodeArgs& a, int D, DecodeCache cache, void* workspace, float sm_scale, void* stream) {
  int rc = device_ready(&a.status);
  if (rc != TATTN_OK) return rc;
  a.nsplit = decode_splits(a, D, cache);
  if (decode_joins(a.nsplit, cache)) {
    if (!workspace) return TATTN_ERR_INVALID_ARGUMENT;
    if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return TATTN_ERR_LAYOUT;
    a.part = static_cast<float*>(workspace);
    a.part_ml = a.part + int64_t(a.Z) * a.H * a.nsplit * D;
  }
  a.qk_scale = sm_scale * kLog2e;
  return cuda_rc(launch_decode(D, cache, a, static_cast<cudaStream_t>(stream)));
}

}  // namespace

extern "C" int tattn_decode(const void* q, const void* k, const void* v, const int32_t* lengths, void* o,
                            void* workspace, const int64_t* strides, int Z, int H, int Hk, int C, int D, int dtype,
                            int window, int sinks, float sm_scale, void* stream) {
  DecodeArgs a{};
  if (!strides || !decode_dims(a, Z, H, Hk, C, D, window, sinks) || (dtype != TATTN_F16 && dtype != TATTN_F32))
    return TATTN_ERR_INVALID_ARGUMENT;
  if (Z == 0) return TATTN_OK;
  if (!q || !lengths || !o || (C > 0 && (!k || !v))) return TATTN_ERR_INVALID_ARGUMENT;
  const int64_t *sq = strides, *sk = strides + 4, *sv = strides + 8, *so = strides + 12;
  const int esz = dtype == TATTN_F16 ? 2 : 4;
  if (!rows16(q, sq, Z, H, 1, esz) || !rows16(o, so, Z, H, 1, esz) || !rows16(k, sk, Z, Hk, C, esz) ||
      !rows16(v, sv, Z, Hk, C, esz))
    return TATTN_ERR_LAYOUT;
  a.q = q;
  a.k = k;
  a.v = v;
  a.o = o;
  a.lengths = lengths;
  a.sq = strides3(sq);
  a.sk = strides3(sk);
  a.sv = strides3(sv);
  a.so = strides3(so);
  return decode(a, D, dtype == TATTN_F16 ? kCacheF16 : kCacheF32, workspace, sm_scale, stream);
}

extern "C" int64_t tattn_decode_workspace_bytes(int Z, int H, int Hk, int C, int D, int dtype, int window, int sinks) {
  DecodeArgs a{};
  if (!decode_dims(a, Z, H, Hk, C, D, window, sinks) || (dtype != TATTN_F16 && dtype != TATTN_F32)) return -1;
  return decode_workspace(a, D, dtype == TATTN_F16 ? kCacheF16 : kCacheF32);
}

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

bool int4_dims(int Z, int Hk, int T, int C, int D) {
  return Z >= 0 && Hk >= 1 && T >= 0 && C >= 0 && (D == 64 || D == 128);
}

}  // namespace

extern "C" int tattn_int4_append(const void* k, const void* v, void* k_codes, void* k_params, void* v_codes,
                                 void* v_params, const int32_t* start, const int32_t* counts, const int64_t* strides,
                                 int Z, int Hk, int T, int C, int D, void* stream) {
  if (!strides || !int4_dims(Z, Hk, T, C, D)) return TATTN_ERR_INVALID_ARGUMENT;
  if (int64_t(Z) * T == 0) return TATTN_OK;
  if (!k || !v || !k_codes || !k_params || !v_codes || !v_params) return TATTN_ERR_INVALID_ARGUMENT;
  if (!rows16(k, strides, Z, Hk, T, 2) || !rows16(v, strides + 4, Z, Hk, T, 2) || !aligned16(k_codes) ||
      !aligned16(k_params) || !aligned16(v_codes) || !aligned16(v_params))
    return TATTN_ERR_LAYOUT;
  Int4CacheArgs a{};
  const int rc = device_ready(&a.status);
  if (rc != TATTN_OK) return rc;
  a.k = k;
  a.v = v;
  a.sk = strides3(strides);
  a.sv = strides3(strides + 4);
  a.k_codes = static_cast<uint8_t*>(k_codes);
  a.v_codes = static_cast<uint8_t*>(v_codes);
  a.k_params = k_params;
  a.v_params = v_params;
  a.start = start;
  a.counts = counts;
  a.Z = Z;
  a.Hk = Hk;
  a.T = T;
  a.C = C;
  return cuda_rc(launch_int4_append(D, a, static_cast<cudaStream_t>(stream)));
}

extern "C" int tattn_int4_read(const void* k_codes, const void* k_params, const void* v_codes, const void* v_params,
                               const int32_t* start, void* k, void* v, int Z, int Hk, int T, int C, int D,
                               void* stream) {
  if (!int4_dims(Z, Hk, T, C, D)) return TATTN_ERR_INVALID_ARGUMENT;
  if (int64_t(Z) * T == 0) return TATTN_OK;
  if (!k || !v || (C > 0 && (!k_codes || !k_params || !v_codes || !v_params))) return TATTN_ERR_INVALID_ARGUMENT;
  if (!aligned16(k) || !aligned16(v) || !aligned16(k_codes) || !aligned16(k_params) || !aligned16(v_codes) ||
      !aligned16(v_params))
    return TATTN_ERR_LAYOUT;
  Int4CacheArgs a{};
  const int rc = device_ready(&a.status);
  if (rc != TATTN_OK) return rc;
  a.k_out = k;
  a.v_out = v;
  a.k_codes = static_cast<uint8_t*>(const_cast<void*>(k_codes));
  a.v_codes = static_cast<uint8_t*>(const_cast<void*>(v_codes));
  a.k_params = const_cast<void*>(k_params);
  a.v_params = const_cast<void*>(v_params);
  a.start = start;
  a.Z = Z;
  a.Hk = Hk;
  a.T = T;
  a.C = C;
  return cuda_rc(launch_int4_read(D, a, static_cast<cudaStream_t>(stream)));
}

extern "C" int tattn_int4_decode(const void* q, const void* k_codes, const void* k_params, const void* v_codes,
                                 const void* v_params, const int32_t* lengths, void* o, void* workspace,
                                 const int64_t* strides, int Z, int H, int Hk, int C, int D, int window, int sinks,
                                 float sm_scale, void* stream) {
  DecodeArgs a{};
  if (!strides || !decode_dims(a, Z, H, Hk, C, D, window, sinks) || !int4_dims(Z, Hk, 0, C, D))
    return TATTN_ERR_INVALID_ARGUMENT;
  if (Z == 0) return TATTN_OK;
  if (!q || !lengths || !o || (C > 0 && (!k_codes || !k_params || !v_codes || !v_params)))
    return TATTN_ERR_INVALID_ARGUMENT;
  if (!rows16(q, strides, Z, H, 1, 2) || !rows16(o, strides + 4, Z, H, 1, 2) || !aligned16(k_codes) ||
      !aligned16(k_params) || !aligned16(v_codes) || !aligned16(v_params))
    return TATTN_ERR_LAYOUT;
  a.q = q;
  a.o = o;
  a.k = k_codes;
  a.v = v_codes;
  a.k_params = k_params;
  a.v_params = v_params;
  a.lengths = lengths;
  a.sq = strides3(strides);
  a.so = strides3(strides + 4);
  return decode(a, D, kCacheInt4, workspace, sm_scale, stream);
}

extern "C" int64_t tattn_int4_decode_workspace_bytes(int Z, int H, int Hk, int C, int D, int window, int sinks) {
  DecodeArgs a{};
  if (!decode_dims(a, Z, H, Hk, C, D, window, sinks) || !int4_dims(Z, Hk, 0, C, D)) return -1;
  return decode_workspace(a, D, kCacheInt4);
}
