// C-ABI boundary (include/tattn.h) of attention to keys of another length than the queries' (kMaskRows) and of single
// tokens over a prefix that several sequences share.
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/tattn.h"
#include "kernels.h"

using namespace tattn;

namespace {

constexpr float kLog2e = 1.4426950408889634f;

bool head_dim_ok(int D) { return D == 16 || D == 32 || D == 64 || D == 128; }
bool dtype_ok(int dtype) { return dtype == TATTN_F16 || dtype == TATTN_F32; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Can rows of D values be read 16 bytes at a time?
bool rows16(const void* p, const int64_t* s, int Z, int H, int N, int esz) {
  if (s[3] != 1 || !aligned16(p)) return false;
  const int extent[3] = {Z, H, N};
  for (int i = 0; i < 3; ++i)
    if (extent[i] > 1 && (s[i] * esz) % 16 != 0) return false;
  return true;
}

bool cross_dims(int Z, int H, int Hk, int Nq, int Nk, int D, int dtype) {
  return Z >= 0 && H >= 0 && Hk >= 1 && H % Hk == 0 && Nq >= 0 && Nk >= 0 && Nk <= (1 << 29) && head_dim_ok(D) && dtype_ok(dtype) &&
         int64_t(H / Hk) * Nq <= (1 << 29);
}
// Sizes whose counts of CTAs, rows and units the kernels hold in 32 bits.
bool cross_fits(int Z, int H, int Hk, int Nq, int Nk) {
  return double(Z) * H * Nq < 1e9 && double(Z) * Hk * (Nk / 128 + 1) < 1e7;
}

float positive(float sm_scale) {
  // Positive, so that a hidden score stays -infinity; below 2^-60 scores vanish against 1 anyway.
  return std::max((sm_scale < 0.f ? -sm_scale : sm_scale) * kLog2e, 0x1p-60f);
}

// Parts for `rows` rows of each of `heads` key/value heads against Nk keys. A CTA begins and ends at the cost of some
// blocks of its own, and the join of the parts is another launch.
int row_parts(int D, int dtype, int64_t heads, int rows, int Nk) {
  const int sms = device_sm_count();
  if (dtype == TATTN_F32) {
    const int tile = window_f32_tile(D, heads, rows);
    return rows_splits(heads * ((rows + tile - 1) / tile), (int64_t(Nk) + kWindowF32Block - 1) / kWindowF32Block, 4 * sms, 1, 2);
  }
  const int tiles = rows_f16_tiles(D, rows), block = rows_f16_block(D, rows);
  return rows_splits(heads * ((rows + 128 * tiles - 1) / (128 * tiles)), (int64_t(Nk) + block - 1) / block,
                     int64_t(sms) * (tiles == 1 ? 2 : 1), 4, 4);
}
int64_t part_bytes(int D, int64_t rows, int nsplit) { return (rows * nsplit * (D + 2) * 4 + 15) / 16 * 16; }

// The rows against K and V [Z, Hk, Nk, D]; a.rows but for the scale and the device's state is the caller's.
int run_rows(int D, int dtype, const void* k, const void* v, const int64_t* sk, const int64_t* sv, RowsFwdArgs& a, float sm_scale,
             cudaStream_t s) {
  int rc = device_ready(&a.status);
  if (rc != TATTN_OK) return rc;
  a.wait_limit_ns = wait_limit_ns();
  const int Nk = a.rows.Nk;
  const Strides4 tk = load_strides(sk), tv = load_strides(sv);
  if (dtype == TATTN_F32) {
    a.qk_scale = sm_scale * kLog2e;
    return cuda_rc(launch_rows_f32(D, k, v, tk, tv, a, s));
  }
  a.qk_scale = positive(sm_scale);
  a.negate_s = sm_scale < 0.f ? 1 : 0;
  if (!layout_ok(k, tk, a.Z, a.H, Nk, D) || !layout_ok(v, tv, a.Z, a.H, Nk, D)) return TATTN_ERR_LAYOUT;
  const int block = rows_f16_block(D, a.N);
  CUtensorMap mk, mv;
  if ((rc = encode_f16(&mk, k, tk, a.Z, a.H, Nk, D, block)) != TATTN_OK) return rc;
  if ((rc = encode_f16(&mv, v, tv, a.Z, a.H, Nk, D, block)) != TATTN_OK) return rc;
  return cuda_rc(launch_rows_f16(D, mk, mv, a, s));
}

// Single tokens (and in fp16 a few, where a head's group and they are one run of rows) go through the single-token
// kernels: 16 rows at most, which is what those take at a time.
bool few_rows(int H, int Hk, int Nq, int dtype) { return Nq == 1 || (dtype == TATTN_F16 && int64_t(H / Hk) * Nq <= 16); }
bool one_run(const int64_t* s, int H, int Nq) { return Nq == 1 || H == 1 || s[1] == Nq * s[2]; }

DecodeArgs token_args(int Z, int H, int Hk, int Nq, int Nk) {
  DecodeArgs a{};
  a.Z = Z;
  a.H = H * Nq;
  a.Hk = Hk;
  a.C = Nk;
  a.window = a.sinks = Nk;
  return a;
}
DecodeCache cache_of(int dtype) { return dtype == TATTN_F16 ? kCacheF16 : kCacheF32; }
// Parts of a sequence's keys: as for a cache, but no more than run at a time. (8 sequences of up to 1500 keys, 16 heads of
// 64: 14.3 us with the cache's 3 parts, 2 of which an SM holds, 10.6 with 2.)
int token_parts(const DecodeArgs& a, int D, int dtype) {
  const int n = decode_splits(a, D, cache_of(dtype)), heads = dtype == TATTN_F32 ? 1 : a.H / a.Hk <= 8 ? 8 : 16;
  const int64_t units = int64_t(a.Z) * a.Hk * ((a.H / a.Hk + heads - 1) / heads);
  const int64_t most = int64_t(decode_ctas(cache_of(dtype))) * device_sm_count() / std::max<int64_t>(units, 1);
  return int(std::max<int64_t>(1, std::min<int64_t>(n, most)));
}

}  // namespace

extern "C" int64_t tattn_cross_fwd_workspace_bytes(int Z, int H, int Hk, int Nq, int Nk, int D, int dtype) {
  if (!cross_dims(Z, H, Hk, Nq, Nk, D, dtype) || !cross_fits(Z, H, Hk, Nq, Nk)) return -1;
  if (int64_t(Z) * H * Nq == 0) return 0;
  const int64_t rows = int64_t(Z) * H * Nq;
  const int parts = row_parts(D, dtype, int64_t(Z) * Hk, H / Hk * Nq, Nk);
  int64_t bytes = parts > 1 ? part_bytes(D, rows, parts) : 0;
  if (few_rows(H, Hk, Nq, dtype)) {
    const int n = token_parts(token_args(Z, H, Hk, Nq, Nk), D, dtype);
    if (decode_joins(n, cache_of(dtype))) bytes = std::max(bytes, part_bytes(D, rows, n));
  }
  return bytes;
}

extern "C" int tattn_cross_fwd(const void* q, const void* k, const void* v, const int32_t* lengths, void* o, float* m,
                               void* o_rest, void* workspace, const int64_t* strides, int Z, int H, int Hk, int Nq, int Nk,
                               int D, int dtype, float sm_scale, void* stream) {
  if (!strides || !cross_dims(Z, H, Hk, Nq, Nk, D, dtype)) return TATTN_ERR_INVALID_ARGUMENT;
  if (!cross_fits(Z, H, Hk, Nq, Nk)) return TATTN_ERR_TOO_LARGE;
  if (int64_t(Z) * H * Nq == 0) return TATTN_OK;
  if (!q || !o || (Nk > 0 && (!k || !v))) return TATTN_ERR_INVALID_ARGUMENT;
  const int64_t *sq = strides, *sk = strides + 4, *sv = strides + 8, *so = strides + 12;
  const int esz = dtype == TATTN_F16 ? 2 : 4, group = H / Hk;
  if (!rows16(q, sq, Z, H, Nq, esz) || !rows16(o, so, Z, H, Nq, esz) || !rows16(k, sk, Z, Hk, Nk, esz) ||
      !rows16(v, sv, Z, Hk, Nk, esz) || !aligned16(o_rest) || !aligned16(workspace))
    return TATTN_ERR_LAYOUT;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t rows = int64_t(Z) * H * Nq;
  if (!m && !o_rest && few_rows(H, Hk, Nq, dtype) && one_run(sq, H, Nq) && one_run(so, H, Nq)) {
    DecodeArgs a = token_args(Z, H, Hk, Nq, Nk);
    const int rc = device_ready(&a.status);
    if (rc != TATTN_OK) return rc;
    a.nsplit = token_parts(a, D, dtype);
    if (decode_joins(a.nsplit, cache_of(dtype))) {
      if (!workspace) return TATTN_ERR_INVALID_ARGUMENT;
      a.part = static_cast<float*>(workspace);
      a.part_ml = a.part + rows * a.nsplit * D;
    }
    a.q = q;
    a.k = k;
    a.v = v;
    a.o = o;
    a.lengths = lengths;
    a.sq = Strides3{sq[0], Nq == 1 ? sq[1] : sq[2], 0};
    a.so = Strides3{so[0], Nq == 1 ? so[1] : so[2], 0};
    a.sk = Strides3{sk[0], sk[1], sk[2]};
    a.sv = Strides3{sv[0], sv[1], sv[2]};
    a.qk_scale = sm_scale * kLog2e;
    return cuda_rc(launch_decode(D, cache_of(dtype), a, s));
  }
  RowsFwdArgs a{};
  a.o = o;
  a.m = m;
  a.o_rest = dtype == TATTN_F16 ? static_cast<uint8_t*>(o_rest) : nullptr;
  a.Z = Z;
  a.H = Hk;
  a.N = group * Nq;
  a.rows.q = q;
  a.rows.sq = RowMap{sq[0], group * sq[1], sq[1], sq[2]};
  a.rows.so = RowMap{so[0], group * so[1], so[1], so[2]};
  a.rows.inner = Nq;
  a.rows.Nk = Nk;
  a.rows.lengths = lengths;
  a.rows.nsplit = row_parts(D, dtype, int64_t(Z) * Hk, a.N, Nk);
  if (a.rows.nsplit > 1) {
    if (!workspace) return TATTN_ERR_INVALID_ARGUMENT;
    a.rows.part = static_cast<float*>(workspace);
    a.rows.part_ml = a.rows.part + rows * a.rows.nsplit * D;
  }
  JoinArgs j{};
  if (Nk > 0) {  // (else the join of no parts: zeros)
    const int rc = run_rows(D, dtype, k, v, sk, sv, a, sm_scale, s);
    if (rc != TATTN_OK || a.rows.nsplit == 1) return rc;
    j.part[0] = a.rows.part;
    j.part_ml[0] = a.rows.part_ml;
    j.n[0] = a.rows.nsplit;
  }
  j.o = o;
  j.so = a.rows.so;
  j.inner = Nq;
  j.Z = Z;
  j.H = Hk;
  j.N = a.N;
  j.m = m;
  j.o_rest = a.o_rest;
  return cuda_rc(launch_rows_join(D, dtype == TATTN_F16, j, s));
}

namespace {

// The backward takes the heads of a group as one where their rows are one run: no block of queries is then cut short by
// a head's end.
bool folds(int H, int Hk, int Nq) { return H > Hk && Nq % 128 != 0; }
void fold(int& H, int Hk, int& Nq) {
  Nq *= H / Hk;
  H = Hk;
}

WindowSplit cross_split(int Z, int H, int Hk, int Nq, int Nk, int D, int dtype) {
  const WindowArgs w = whole_window(H, Hk, Nq, Nk);
  // (fp32: as the window's)
  return dtype == TATTN_F32 ? window_split(window_f32_tile(D, (long long)Z * Hk, Nk), kWindowF32Block, Z, w, Nq, D, 4 * device_sm_count())
                            : window_split(128, bwd_fused_query_rows(D), Z, w, Nq, D, device_sm_count());
}
int64_t cross_part_bytes(int Z, int H, int Hk, int Nq, int Nk, int D, int dtype) {
  return window_part_bytes(dtype == TATTN_F32 ? window_f32_tile(D, (long long)Z * Hk, Nk) : 128, Z, whole_window(H, Hk, Nq, Nk), D,
                           cross_split(Z, H, Hk, Nq, Nk, D, dtype));
}

// fp32: parts of the keys for dq, and where their sums stand behind the tiles' partials. As many CTAs as shared memory lets
// run at a time; a part's beginning counts for nothing, as lengths may differ and smaller parts even them out (B3 H5, 200
// queries of up to 777 keys: the backward 88 -> 79 us at D64, 70 -> 64 at D32, nothing lost with equal lengths; one block
// for it: 88. Twice the CTAs at D64: 79, but 40 queries of 5,000 keys 71 -> 82).
int dq_parts(int Z, int H, int Nq, int Nk, int D) {
  const int tile = window_f32_tile(D, (long long)Z * H, Nq);
  return rows_splits(int64_t(Z) * H * ((Nq + tile - 1) / tile), (int64_t(Nk) + kWindowF32Block - 1) / kWindowF32Block,
                     (D <= 32 ? 4 : 2) * device_sm_count(), 0, 1);
}
int64_t dq_part_bytes(int Z, int H, int Nq, int Nk, int D) {
  const int parts = dq_parts(Z, H, Nq, Nk, D);
  return parts > 1 ? int64_t(parts) * Z * H * Nq * D * 4 : 0;
}

}  // namespace

extern "C" int64_t tattn_cross_bwd_workspace_bytes(int Z, int H, int Hk, int Nq, int Nk, int D, int dtype) {
  if (!cross_dims(Z, H, Hk, Nq, Nk, D, dtype) || !cross_fits(Z, H, Hk, Nq, Nk)) return -1;
  if (int64_t(Z) * H * Nq == 0) return 0;
  const int64_t dq = dtype == TATTN_F16 ? bwd_fused_workspace_bytes(Z, H, Nq, D) : 0;
  if (Nk == 0) return dq;
  auto parts = [&] {
    return cross_part_bytes(Z, H, Hk, Nq, Nk, D, dtype) + (dtype == TATTN_F32 ? dq_part_bytes(Z, H, Nq, Nk, D) : 0);
  };
  int64_t part = parts();
  if (folds(H, Hk, Nq)) {
    fold(H, Hk, Nq);
    part = std::max(part, parts());
  }
  return dq + part;
}

extern "C" int tattn_cross_bwd(const void* q, const void* k, const void* v, const int32_t* lengths, const void* o,
                               const void* dout, void* dq, void* dk, void* dv, const float* m, const void* o_rest, float* delta,
                               void* workspace, const int64_t* strides, int Z, int H, int Hk, int Nq, int Nk, int D, int dtype,
                               float sm_scale, void* stream) {
  if (!strides || !cross_dims(Z, H, Hk, Nq, Nk, D, dtype)) return TATTN_ERR_INVALID_ARGUMENT;
  if (!cross_fits(Z, H, Hk, Nq, Nk)) return TATTN_ERR_TOO_LARGE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool half = dtype == TATTN_F16;
  const int64_t rows = int64_t(Z) * H * Nq, keys = int64_t(Z) * Hk * Nk;
  if ((rows > 0 && !dq) || (keys > 0 && (!dk || !dv))) return TATTN_ERR_INVALID_ARGUMENT;
  if (rows == 0 || keys == 0) {  // queries without keys, or keys that no query sees
    const size_t row = size_t(D) * (half ? 2 : 4);
    if (rows > 0 && cudaMemsetAsync(dq, 0, rows * row, s) != cudaSuccess) return TATTN_ERR_CUDA;
    for (void* p : {dk, dv})
      if (keys > 0 && cudaMemsetAsync(p, 0, keys * row, s) != cudaSuccess) return TATTN_ERR_CUDA;
    return TATTN_OK;
  }
  if (!q || !k || !v || !o || !dout || !m || !delta || (half && !workspace)) return TATTN_ERR_INVALID_ARGUMENT;
  int64_t st[20];
  std::copy(strides, strides + 20, st);
  int64_t *sq = st, *sk = st + 4, *sv = st + 8, *so = st + 12, *sdo = st + 16;
  if (folds(H, Hk, Nq) && one_run(sq, H, Nq) && one_run(so, H, Nq) && one_run(sdo, H, Nq)) {
    const int group = H / Hk;
    for (int64_t* x : {sq, so, sdo}) {
      if (Nq == 1) x[2] = x[1];  // (the stride along one token says nothing)
      x[1] *= group;
    }
    fold(H, Hk, Nq);
  }
  const int esz = half ? 2 : 4;
  if (!rows16(q, sq, Z, H, Nq, esz) || !rows16(o, so, Z, H, Nq, esz) || !rows16(dout, sdo, Z, H, Nq, esz) ||
      !rows16(k, sk, Z, Hk, Nk, esz) || !rows16(v, sv, Z, Hk, Nk, esz))
    return TATTN_ERR_LAYOUT;
  for (const void* p : {static_cast<const void*>(dq), static_cast<const void*>(dk), static_cast<const void*>(dv),
                        static_cast<const void*>(workspace), o_rest})
    if (!aligned16(p)) return TATTN_ERR_LAYOUT;
  RowsBwdArgs a{};
  int rc = device_ready(&a.status);
  if (rc != TATTN_OK) return rc;
  a.q = q;
  a.k = k;
  a.v = v;
  a.o = o;
  a.dout = dout;
  a.sq = load_strides(sq);
  a.sk = load_strides(sk);
  a.sv = load_strides(sv);
  a.so = load_strides(so);
  a.sdo = load_strides(sdo);
  a.m = m;
  a.delta = delta;
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  a.Z = Z;
  a.H = H;
  a.N = Nq;
  a.sm_scale = sm_scale;
  a.qk_scale = (sm_scale < 0.f ? -sm_scale : sm_scale) * kLog2e;
  a.negate_s = sm_scale < 0.f ? 1 : 0;
  a.wait_limit_ns = wait_limit_ns();
  a.win = whole_window(H, Hk, Nq, Nk);
  a.split = cross_split(Z, H, Hk, Nq, Nk, D, dtype);
  a.lengths = lengths;
  const int64_t parts = cross_part_bytes(Z, H, Hk, Nq, Nk, D, dtype);
  if (!half) {
    a.dq_split = dq_parts(Z, H, Nq, Nk, D);
    if (parts > 0 || a.dq_split > 1) {
      if (!workspace) return TATTN_ERR_INVALID_ARGUMENT;
      a.part = static_cast<float*>(workspace);  // (a multiple of 16 bytes, then dq's)
      a.dq_part = a.part + parts / 4;
    }
    rc = cuda_rc(launch_bwd_preprocess(D, false, a, s));
    return rc != TATTN_OK ? rc : cuda_rc(launch_rows_bwd_f32(D, a, s));
  }
  if (!layout_ok(q, a.sq, Z, H, Nq, D) || !layout_ok(k, a.sk, Z, Hk, Nk, D) || !layout_ok(v, a.sv, Z, Hk, Nk, D) ||
      !layout_ok(o, a.so, Z, H, Nq, D) || !layout_ok(dout, a.sdo, Z, H, Nq, D))
    return TATTN_ERR_LAYOUT;
  a.o_rest = static_cast<const uint8_t*>(o_rest);
  a.dq_acc = static_cast<float*>(workspace);
  char* after = static_cast<char*>(workspace) + int64_t(Z) * H * Nq * D * 4;
  a.grid_sync = reinterpret_cast<unsigned*>(after);
  a.part = parts > 0 ? reinterpret_cast<float*>(after + 16) : nullptr;
  CUtensorMap tq, tk, tv, tdo, tdk, tdv, tdqacc;
  const int q_rows = bwd_fused_query_rows(D), acc_cols = D == 128 ? 32 : D / 2;  // as tattn_bwd_fused
  if ((rc = encode_f16(&tq, q, a.sq, Z, H, Nq, D, q_rows)) != TATTN_OK) return rc;
  if ((rc = encode_f16(&tk, k, a.sk, Z, Hk, Nk, D, 128)) != TATTN_OK) return rc;
  if ((rc = encode_f16(&tv, v, a.sv, Z, Hk, Nk, D, 128)) != TATTN_OK) return rc;
  if ((rc = encode_f16(&tdo, dout, a.sdo, Z, H, Nq, D, q_rows)) != TATTN_OK) return rc;
  const Strides4 dense{int64_t(Hk) * Nk * D, int64_t(Nk) * D, D, 1};
  if ((rc = encode_f16(&tdk, dk, dense, Z, Hk, Nk, D, kBwdStoreRows, D / 2)) != TATTN_OK) return rc;
  if ((rc = encode_f16(&tdv, dv, dense, Z, Hk, Nk, D, kBwdStoreRows, D / 2)) != TATTN_OK) return rc;
  if ((rc = encode_f32_dense(&tdqacc, a.dq_acc, Z, H, Nq, D, kBwdStoreRows, acc_cols)) != TATTN_OK) return rc;
  a.so = normalize(a.so, Z, H, Nq, D);
  a.sdo = normalize(a.sdo, Z, H, Nq, D);
  if ((rc = cuda_rc(launch_bwd_preprocess(D, true, a, s))) != TATTN_OK) return rc;  // delta, zeroed workspace
  return cuda_rc(launch_bwd_rows_f16(D, tq, tk, tv, tdo, tdk, tdv, tdqacc, a, s));
}

namespace {

bool prefix_dims(int prompts, int samples, int H, int Hk, int P, int C, int D, int dtype) {
  return prompts >= 0 && samples >= 1 && H >= 1 && Hk >= 1 && H % Hk == 0 && P >= 0 && P <= (1 << 29) && C >= 0 &&
         C <= (1 << 30) && head_dim_ok(D) && dtype_ok(dtype);
}
bool prefix_fits(int prompts, int samples, int H, int Hk, int P) {
  return double(prompts) * samples * H < 5e8 && double(prompts) * Hk * (P / 128 + 1) < 1e7;
}
DecodeArgs own_args(int prompts, int samples, int H, int Hk, int C) { return token_args(prompts * samples, H, Hk, 1, C); }
// Parts of the sequences' own tokens: as for a cache, but in fp16 of 256 tokens at least, as the prefix's parts are joined
// anyhow (16 samples of up to 256 tokens: 11.4 us with 2 parts, 10.6 with one).
int own_parts(const DecodeArgs& a, int D, int dtype) {
  const int n = decode_splits(a, D, cache_of(dtype));
  return dtype == TATTN_F32 ? n : std::min(n, std::max(1, a.C / 256));
}

}  // namespace

extern "C" int64_t tattn_prefix_decode_workspace_bytes(int prompts, int samples, int H, int Hk, int P, int C, int D, int dtype) {
  if (!prefix_dims(prompts, samples, H, Hk, P, C, D, dtype) || !prefix_fits(prompts, samples, H, Hk, P)) return -1;
  const int64_t rows = int64_t(prompts) * samples * H;
  if (rows == 0) return 0;
  return part_bytes(D, rows, row_parts(D, dtype, int64_t(prompts) * Hk, samples * (H / Hk), P)) +
         part_bytes(D, rows, own_parts(own_args(prompts, samples, H, Hk, C), D, dtype));
}

extern "C" int tattn_prefix_decode(const void* q, const void* prefix_k, const void* prefix_v, const int32_t* prefix_lengths,
                                   const void* k, const void* v, const int32_t* lengths, void* o, void* workspace,
                                   const int64_t* strides, int prompts, int samples, int H, int Hk, int P, int C, int D,
                                   int dtype, float sm_scale, void* stream) {
  if (!strides || !prefix_dims(prompts, samples, H, Hk, P, C, D, dtype)) return TATTN_ERR_INVALID_ARGUMENT;
  if (!prefix_fits(prompts, samples, H, Hk, P)) return TATTN_ERR_TOO_LARGE;
  const int B = prompts * samples, group = H / Hk;
  const int64_t rows = int64_t(B) * H;
  if (rows == 0) return TATTN_OK;
  if (!q || !o || !lengths || !workspace || (P > 0 && (!prefix_k || !prefix_v)) || (C > 0 && (!k || !v)))
    return TATTN_ERR_INVALID_ARGUMENT;
  const int64_t *sq = strides, *spk = strides + 4, *spv = strides + 8, *sk = strides + 12, *sv = strides + 16, *so = strides + 20;
  const int esz = dtype == TATTN_F16 ? 2 : 4;
  if (!rows16(q, sq, B, H, 1, esz) || !rows16(o, so, B, H, 1, esz) || !rows16(prefix_k, spk, prompts, Hk, P, esz) ||
      !rows16(prefix_v, spv, prompts, Hk, P, esz) || !rows16(k, sk, B, Hk, C, esz) || !rows16(v, sv, B, Hk, C, esz) ||
      !aligned16(workspace))
    return TATTN_ERR_LAYOUT;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  RowsFwdArgs a{};
  a.Z = prompts;
  a.H = Hk;
  a.N = samples * group;
  a.rows.q = q;
  a.rows.sq = RowMap{samples * sq[0], group * sq[1], sq[0], sq[1]};
  a.rows.inner = group;
  a.rows.Nk = P;
  a.rows.lengths = prefix_lengths;
  a.rows.nsplit = row_parts(D, dtype, int64_t(prompts) * Hk, a.N, P);
  a.rows.part = static_cast<float*>(workspace);
  a.rows.part_ml = a.rows.part + rows * a.rows.nsplit * D;
  DecodeArgs d = own_args(prompts, samples, H, Hk, C);
  int rc = device_ready(&d.status);
  if (rc != TATTN_OK) return rc;
  d.nsplit = own_parts(d, D, dtype);
  d.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + part_bytes(D, rows, a.rows.nsplit));
  d.part_ml = d.part + rows * d.nsplit * D;
  d.parts_only = true;
  d.q = q;
  d.k = k;
  d.v = v;
  d.lengths = lengths;
  d.sq = Strides3{sq[0], sq[1], 0};
  d.sk = Strides3{sk[0], sk[1], sk[2]};
  d.sv = Strides3{sv[0], sv[1], sv[2]};
  d.qk_scale = sm_scale * kLog2e;
  if (P > 0) {
    if ((rc = run_rows(D, dtype, prefix_k, prefix_v, spk, spv, a, sm_scale, s)) != TATTN_OK) return rc;
    d.overlap = true;
  }
  if ((rc = cuda_rc(launch_decode(D, cache_of(dtype), d, s))) != TATTN_OK) return rc;
  JoinArgs j{};
  j.part[0] = a.rows.part;
  j.part_ml[0] = a.rows.part_ml;
  j.n[0] = P > 0 ? a.rows.nsplit : 0;
  j.part[1] = d.part;
  j.part_ml[1] = d.part_ml;
  j.n[1] = d.nsplit;
  j.other = RowMap{int64_t(samples) * H, group, H, 1};
  j.o = o;
  j.so = RowMap{samples * so[0], group * so[1], so[0], so[1]};
  j.inner = group;
  j.Z = prompts;
  j.H = Hk;
  j.N = a.N;
  return cuda_rc(launch_rows_join(D, dtype == TATTN_F16, j, s));
}
