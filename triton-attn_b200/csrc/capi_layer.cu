// C-ABI boundary (include/tattn.h) of the operators around the attention kernels: head norms with rotation.
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

int norm_rope(RopeArgs& a, bool backward, const int64_t* strides, int Z, int H, int Hk, int N, int D, int P, int dtype,
              int w_dtype, int interleaved, void* stream) {
  const int esz = dtype == TATTN_F16 ? 2 : 4, heads[2] = {H, Hk};
  for (int i = 0; i < 2; ++i) {
    RopeTensor& t = a.t[i];
    // forward: q, k, q_out, k_out; backward: q, k, q_grad, k_grad, dq, dk
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
  const int64_t* pos = strides + (backward ? 24 : 16);
  a.pos_z = pos[0];
  a.pos_n = pos[1];
  a.Z = Z;
  a.N = N;
  a.P = P;
  a.w_f32 = w_dtype == TATTN_F32;
  const int rc = device_ready(&a.status);
  if (rc != TATTN_OK) return rc;
  return cuda_rc(launch_norm_rope(D, dtype == TATTN_F16, interleaved != 0, backward, a, static_cast<cudaStream_t>(stream)));
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
