// Host-side launcher interface between the C-ABI layer (capi.cu) and the kernel translation units.
// Nothing here is exported from the shared library; include/tattn.h is the public boundary.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace tattn {

// Element strides of one [Z, H, N, D] tensor (the D stride is always 1 for the fp16 kernels).
struct Strides4 {
  int64_t z, h, n, d;
};

// Which keys a query sees (template parameter of the attention kernels).
enum Mask : int {
  kMaskNone = 0,    // all
  kMaskCausal = 1,  // key <= query
  kMaskWindow = 2,  // a sliding window and the first tokens (WindowArgs)
  kMaskRows = 3,    // the first lengths[z] of them (RowsArgs)
};

// kMaskWindow: query row i stands at position i + off of its sequence and sees the keys j <= i + off with
// j > i + off - window or j < sinks. K and V have H / group heads of Nk tokens, shared by `group`
// consecutive query heads each.
struct WindowArgs {
  int Hk, group;  // key/value heads, query heads per key/value head
  int Nk, off;    // tokens of K and V; off = Nk - N >= 0
  int window;     // 1 <= window <= Nk
  int sinks;      // 0 <= sinks <= Nk
};

// What rounding the window forward's O to fp16 took off, times kRestScale, as 8-bit floats of 5 exponent bits (the
// upper byte of an fp16): a rest is half a unit in O's last place at most, so the scale keeps the rests of all
// finite O, the subnormal ones included, in range, and 2 mantissa bits leave an eighth of it.
constexpr float kRestScale = 2048.f;

// kMaskRows: `N` query rows against each of Z * H key/value heads, all of which see the head's first lengths[z] keys.
// Row r lies at element r / inner * outer + r % inner * in behind the head's first: rows of several query heads, tokens
// or sequences that share the keys are one matrix.
struct RowMap {
  int64_t z, h;      // of sequence z's and key/value head h's first row
  int64_t outer, in;
};
constexpr int kMaxRowSplits = 128;
template <typename T>
__device__ __forceinline__ T* row_of(T* p, const RowMap& s, int inner, int z, int h, int row) {
  const int o = row / inner;
  return p + z * s.z + h * s.h + o * s.outer + (row - o * inner) * s.in;
}
struct RowsArgs {
  const void* q;
  RowMap sq, so;
  int inner;
  int Nk;               // rows of K and V
  const int* lengths;   // [Z], or null: all Nk
  // The blocks of keys are cut into nsplit equal parts, a CTA each. part not null: their unnormalised rows [Z * H, N,
  // nsplit, D] and their maxima and sums [Z * H, N, nsplit, 2] (decode.cu's convention) are written, to be joined; else
  // nsplit is 1.
  int nsplit;
  float* part;
  float* part_ml;
};
// Parts that the `blocks` key blocks of `tiles` row tiles are cut into, of which `slots` run at a time: the number with
// the shortest time, in blocks, when a CTA takes `start` to begin and to end and the parts' join `join`.
// (Of the numbers that take equally many rounds, the largest.)
inline int rows_splits(long long tiles, long long blocks, long long slots, int start, int join) {
  long long best = 1, least = (tiles + slots - 1) / slots * (blocks + start);
  for (long long rounds = 1; rounds <= 4; ++rounds) {
    long long n = rounds * slots / tiles;
    n = n < blocks ? n : blocks;
    n = n < kMaxRowSplits ? n : kMaxRowSplits;
    if (n <= 1) continue;
    const long long cost = (tiles * n + slots - 1) / slots * ((blocks + n - 1) / n + start) + join;
    if (cost < least) {
      least = cost;
      best = n;
    }
  }
  return int(best);
}

struct FwdArgs {
  void* o;           // [Z, H, N, D], strides `so`
  float* m;          // [Z, H, N] dense fp32: rowmax + log2(rowsum), base-2 units
  Strides4 so;
  int Z, H, N;
  float qk_scale;    // |sm_scale| * log2(e); the sign goes into the S MMA (negate A) for fp16
  int negate_s;      // 1 when sm_scale < 0 (fp16 path)
  int* status;       // device status word
  unsigned long long wait_limit_ns;  // bound of every mbarrier wait (tattn_set_wait_limit_ns)
  WindowArgs win;    // kMaskWindow only
  uint8_t* o_rest;   // kMaskWindow, kMaskRows in fp16: what rounding O took off (kRestScale), dense [Z, H, N, D], or null
};
// kMaskRows (apart from the others' arguments, whose kernels' registers a longer list costs); `so` is rows.so, and m
// may be null.
struct RowsFwdArgs : FwdArgs {
  RowsArgs rows;
};

// Keys of sequence z that its queries see; a length outside [0, Nk] counts as the nearer end.
__device__ __forceinline__ int held_keys(const int* lengths, int z, int Nk, bool* outside) {
  const int len = lengths ? lengths[z] : Nk;
  *outside = len < 0 || len > Nk;
  return len < 0 ? 0 : len > Nk ? Nk : len;
}

// Window backward: its units of work. A key tile of a key/value head meets the query blocks that see it, once
// for each query head of the group: a run of (head, block) pairs, head by head, which is cut into equal units.
// The `tiles` first key tiles hold sinks, which all later queries see: sink_units units each; the others are seen
// by one window of queries: `units` each. A tile of several units is the sum of fp32 partials, added up in the
// units' order.
//
// The units' order: `heads` heads at a time, first each head's tiles that meet a whole window of queries (those
// of the sinks first), then the tiles whose window the first query (`before` of them) or the last one cuts short
// (from tile `last` on), for all heads at once from the longest to the shortest.
struct WindowSplit {
  int tiles, sink_units, units;
  int before, last, heads;
  __host__ __device__ int per_head(int key_tiles) const { return tiles * sink_units + (key_tiles - tiles) * units; }
  // Partials of a head: of every unit, of those of the sink tiles, or none.
  __host__ __device__ int slots(int key_tiles) const {
    return units > 1 ? per_head(key_tiles) : sink_units > 1 ? tiles * sink_units : 0;
  }
};

// Unit p of all heads: part `piece` of key tile kt (of TILE rows) of key/value head `head`, which is pairs
// [start, start + n) of the tile's run over the query blocks (of BQ) [lo, lo + nb) of each query head.
struct WindowUnit {
  int head;
  int kt, lo, nb;
  int start, n;  // n may be 0: the queries begin after the tile's window
  int slot;      // its partial in the head, or -1: it is the whole tile
};
template <int TILE, int BQ>
__host__ __device__ inline WindowUnit window_unit(const WindowSplit& s, const WindowArgs& w, int Z, int N, unsigned p) {
  using u32 = unsigned;  // unsigned 32-bit divisions: they stand between one unit and the next
  const u32 key_tiles = u32(w.Nk + TILE - 1) / TILE, sink_part = s.tiles * s.sink_units;
  const u32 set = p / (s.per_head(key_tiles) * s.heads), rest = p - set * s.per_head(key_tiles) * s.heads;
  const u32 first = set * s.heads, left = u32(Z) * w.Hk - first, heads = left < u32(s.heads) ? left : s.heads;
  const u32 whole = sink_part + (s.last - s.before - s.tiles) * s.units;
  u32 head, kt, piece;
  if (rest < heads * whole) {
    head = rest / whole;
    const u32 i = rest - head * whole;
    const bool sink = i < sink_part;
    const u32 j = sink ? i : i - sink_part, count = sink ? s.sink_units : s.units;
    kt = j / count;
    piece = j - kt * count;
    if (!sink) kt += s.tiles + s.before;
  } else {
    const u32 tail = rest - heads * whole, rank = tail / (heads * s.units), i = tail - rank * heads * s.units;
    head = i / s.units;
    piece = i - head * s.units;
    const u32 after = key_tiles - s.last, both = 2 * (after < u32(s.before) ? after : s.before);
    const bool late = rank < both ? rank % 2 == 0 : after > u32(s.before);  // the two ends' tiles in turn
    const u32 j = rank < both ? rank / 2 : rank - both / 2;
    kt = late ? s.last + j : s.tiles + s.before - 1 - j;
  }
  WindowUnit u;
  u.head = first + head;
  u.kt = kt;
  const bool sink = u.kt < s.tiles;
  const int k0 = TILE * u.kt, blocks = int(u32(N + BQ - 1) / BQ), count = sink ? s.sink_units : s.units;
  const int last = k0 + TILE - 2 + w.window - w.off;  // the last query that sees the tile's last key
  const int end = sink ? blocks : last < 0 ? 0 : (last / BQ + 1 < blocks ? last / BQ + 1 : blocks);
  u.lo = (k0 > w.off ? k0 - w.off : 0) / BQ;
  u.nb = end > u.lo ? end - u.lo : 0;
  const u32 pairs = u32(u.nb) * w.group, each = pairs / count, more = pairs - each * count;
  u.start = each * piece + (piece < more ? piece : more);
  u.n = each + (piece < more ? 1 : 0);
  u.slot = count > 1 ? (sink ? 0 : s.tiles * (s.sink_units - s.units)) + u.kt * count + int(piece) : -1;
  return u;
}

// Parts of rows that are to be joined: of every row up to two lists of unnormalised parts with their maxima and sums.
// The join is launched to overlap with the kernel that writes them (overlapping_launch).
struct JoinArgs {
  const float *part[2], *part_ml[2];  // [rows, n, D] and [rows, n, 2]
  int n[2];
  RowMap other;        // where a row (as RowsArgs counts them) lies in the second list, in rows
  void* o;
  RowMap so;
  int inner;
  int Z, H, N;
  float* m;            // as FwdArgs; null: not wanted
  uint8_t* o_rest;     // as FwdArgs, or null
};

struct BwdArgs {
  // inputs
  const void* q; const void* k; const void* v; const void* o; const void* dout;
  Strides4 sq, sk, sv, so, sdo;
  const float* m;    // [Z, H, N]
  float* delta;      // [Z, H, N]: rowsum(dO * O)
  // outputs (dense [Z, H, N, D])
  void* dq; void* dk; void* dv;
  float* dq_acc;     // fused backward: dense fp32 [Z, H, N, D] dQ workspace (zeroed by the preprocess), or null
  unsigned* grid_sync;  // fused backward: its grid-barrier counter (zeroed by the preprocess), or null
  int Z, H, N;
  float sm_scale;    // signed
  float qk_scale;    // |sm_scale| * log2(e)
  int negate_s;
  int* status;
  unsigned long long wait_limit_ns;  // bound of every mbarrier wait (tattn_set_wait_limit_ns)
  const uint8_t* o_rest;  // kMaskWindow in fp16: the forward's, or null
  WindowArgs win;    // kMaskWindow only: dk and dv are then dense [Z, win.Hk, win.Nk, D]
  WindowSplit split; // kMaskWindow
  float* part;       // kMaskWindow: partial dV and dK of the tiles of several units, or null
};
// kMaskRows: a window (`win`, `split`) that shows every query every key, of which sequence z has the first lengths[z].
struct RowsBwdArgs : BwdArgs {
  const int* lengths;  // [Z], or null: all
  // fp32: the keys that dq sums over are cut into dq_split parts; more than one: their sums [dq_split, Z, H, N, D], to be
  // added up.
  int dq_split;
  float* dq_part;
};
// The window that hides nothing.
inline WindowArgs whole_window(int H, int Hk, int Nq, int Nk) { return WindowArgs{Hk, H / Hk, Nk, Nk, Nk + Nq, 0}; }

// Host helpers of the C-ABI layer (capi.cu). device_ready: the current device is an sm_100 one whose primary
// context is current on this thread, and *status its status word (a TATTN_* code). device_sm_count: its
// streaming multiprocessors (cached per device). cuda_rc: a launch's result as a TATTN_* code.
int device_ready(int** status);
unsigned long long wait_limit_ns();
// fp16 tensors for TMA (capi.cu): normalize replaces the strides of extent-1 dimensions, layout_ok says whether TMA can
// address a tensor, encode_* make the maps (TATTN_* codes).
Strides4 load_strides(const int64_t* s);
Strides4 normalize(Strides4 s, int Z, int H, int N, int D);
bool layout_ok(const void* p, Strides4 s, int Z, int H, int N, int D);
int encode_f16(CUtensorMap* tm, const void* p, Strides4 s, int Z, int H, int N, int D, int box_rows, int box_cols = 0);
int encode_f32_dense(CUtensorMap* tm, void* p, int Z, int H, int N, int D, int box_rows, int box_cols);
int device_sm_count();
int cuda_rc(cudaError_t e);
// A launch that may start before the stream's last kernel has ended, which it then waits for itself (common.cuh).
inline cudaLaunchAttribute overlapping_launch() {
  cudaLaunchAttribute a{};
  a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a.val.programmaticStreamSerializationAllowed = 1;
  return a;
}

// `variant` below is a 0-based tile variant of tiles.h (kFwdTiles / kBwdTiles); launchers return
// cudaErrorNotSupported for a variant that does not fit head dim D.
// Rows per K/V block of the fp16 forward variant for head dim D: the TMA box height of its K and V
// tensor maps (the Q map always uses 128-row boxes); 0 if the variant does not fit D.
int fwd_f16_kv_rows(int D, int variant);
// kMaskRows: K and V in boxes of rows_f16_block keys.
cudaError_t launch_rows_f16(int D, const CUtensorMap& tk, const CUtensorMap& tv, const RowsFwdArgs& a, cudaStream_t s);
// kMaskRows: query tiles of a CTA, and keys of a block, by the number of rows. One tile (two CTAs an SM) at D <= 64 (B2 H16 N4096
// D64: 265 us with two, 220 with one), and at D = 128 where it holds all rows.
constexpr int rows_f16_tiles(int D, int rows) { return rows <= 128 || D <= 64 ? 1 : 2; }
constexpr int rows_f16_block(int D, int rows) { return rows <= 64 || (D == 128 && rows <= 128) ? 64 : 128; }
// TMA box heights of the fp16 split-backward kernels' Q/dO and K/V tensor maps for head dim D, dQ pass
// or dK/dV pass, and tile variant.
void bwd_f16_box_rows(int D, bool dq_pass, int variant, int* q_rows, int* kv_rows);

// fp16 tcgen05 kernels (tensor maps describe [Z, H, N, D] tensors as 4-D {D, N, H, Z}).
cudaError_t launch_fwd_f16(int D, Mask mask, int variant, const CUtensorMap& tq, const CUtensorMap& tk,
                           const CUtensorMap& tv, const FwdArgs& a, cudaStream_t s);
// tdq: store map of the dense dQ output, kBwdStoreRows-row boxes of D/2 columns (D <= 64).
cudaError_t launch_bwd_dq_f16(int D, bool causal, int variant, const CUtensorMap& tq, const CUtensorMap& tk,
                              const CUtensorMap& tv, const CUtensorMap& tdo, const CUtensorMap& tdq, const BwdArgs& a,
                              cudaStream_t s);
// tdk / tdv: store maps of the dense dK / dV outputs, kBwdStoreRows-row boxes of D/2 columns (D <= 64).
cudaError_t launch_bwd_dkdv_f16(int D, bool causal, int variant, const CUtensorMap& tq, const CUtensorMap& tk,
                                const CUtensorMap& tv, const CUtensorMap& tdo, const CUtensorMap& tdk,
                                const CUtensorMap& tdv, const BwdArgs& a, cudaStream_t s);
// Fused backward kernel (any supported D, causal or not; one cooperative launch): dK, dV and the dQ
// sums into the fp32 workspace a.dq_acc [Z, H, N, D], then a grid barrier and a.dq = sm_scale * dq_acc
// as fp16. a.dq_acc, a.delta and the barrier counter a.grid_sync come from launch_bwd_preprocess.
// tq/tdo with boxes of bwd_fused_query_rows(D) rows, tk/tv 128-row boxes, tdk/tdv store maps of
// kBwdStoreRows-row boxes of D/2 columns, tdqacc a reduce map over a.dq_acc (kBwdStoreRows-row boxes
// of D/2 columns; 32 columns at D = 128).
cudaError_t launch_bwd_fused_f16(int D, Mask mask, const CUtensorMap& tq, const CUtensorMap& tk,
                                 const CUtensorMap& tv, const CUtensorMap& tdo, const CUtensorMap& tdk,
                                 const CUtensorMap& tdv, const CUtensorMap& tdqacc, const BwdArgs& a, cudaStream_t s);
cudaError_t launch_bwd_rows_f16(int D, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                                const CUtensorMap& tdo, const CUtensorMap& tdk, const CUtensorMap& tdv,
                                const CUtensorMap& tdqacc, const RowsBwdArgs& a, cudaStream_t s);
// Box height of the backward's output store maps (one warp's 32 TMEM lanes).
constexpr int kBwdStoreRows = 32;
// Query rows per block of the fused backward (its Q / dO box height): 128, or 64 at D = 128.
__host__ __device__ constexpr int bwd_fused_query_rows(int D) { return D == 128 ? 64 : 128; }
// Workspace of tattn_bwd_fused: the fp32 dQ rows [Z, H, N, D], then 16 bytes for the grid-barrier counter.
inline int64_t bwd_fused_workspace_bytes(int Z, int H, int N, int D) { return int64_t(Z) * H * N * D * 4 + 16; }
// Units of about one size for `workers` CTAs that take them in turn: what a tile without sinks costs (one
// window's blocks for the group) or, where that is less, a CTA's share; 8 blocks at least and at most 64 units a
// tile. (A unit starts and ends at the cost of about 2 blocks, and partials are written and read again. Share, half
// and third of it: B2 H16 Hk4 N2500 D128, window 777, 130 sinks: 214, 205, 222 us; B1 H16 Hk4, 4096 queries of
// 16384 tokens, D64, window 4096: 236, 255, 250; B1 H32 Hk8 N1000 D128, causal: 71, 79, 98.)
inline WindowSplit window_split(int tile, int bq, int Z, const WindowArgs& w, int N, int D, int workers) {
  const int64_t blocks = (N + bq - 1) / bq, key_tiles = (w.Nk + tile - 1) / tile, tiles = (w.sinks + tile - 1) / tile;
  const int64_t span = (int64_t(w.window) + tile - 1 + bq - 1) / bq + 1, one = span < blocks ? span : blocks;
  const int64_t unseen = (w.off > w.window ? w.off - w.window : 0) / tile;  // tiles before every query's window
  const int64_t seen = key_tiles - (unseen > tiles ? unseen : tiles);
  const int64_t all = int64_t(Z) * w.Hk * w.group * (tiles * blocks + seen * one);
  const int64_t share = all / workers + 1;
  int64_t len = w.group * one < share ? w.group * one : share;
  const int64_t least = (w.group * blocks + 63) / 64;
  len = len < 8 ? 8 : len;
  len = len < least ? least : len;
  const int64_t cut = (w.group * one + len - 1) / len;  // equal parts of a tile without sinks
  if (cut > 0) len = (w.group * one + cut - 1) / cut > least ? (w.group * one + cut - 1) / cut : least;
  auto units = [&](int64_t pairs) { return int((pairs + len - 1) / len > 0 ? (pairs + len - 1) / len : 1); };
  // Tiles [tiles, tiles + before) begin before the first query; the window of those from `last` on ends behind
  // the last one.
  const int64_t cut_low = w.off > 0 ? (w.off + tile - 1) / tile - tiles : 0, before = cut_low > 0 ? cut_low : 0;
  const int64_t room = int64_t(w.Nk) - w.window - tile + 2, high = room > 0 ? (room + tile - 1) / tile : 0;
  const int64_t last = high < tiles + before ? tiles + before : high < key_tiles ? high : key_tiles;
  // Heads whose short tiles run together share L2 with their Q and dO rows and (fp16) their dQ sums: 64 MB of
  // them at most.
  const int64_t rows = N < w.window ? N : w.window, bytes = rows * w.group * D * 8, fit = (int64_t(64) << 20) / (bytes > 0 ? bytes : 1);
  const int64_t zh = int64_t(Z) * w.Hk < 65536 ? int64_t(Z) * w.Hk : 65536, heads = fit < 1 ? 1 : fit < zh ? fit : zh;
  return WindowSplit{int(tiles), units(w.group * blocks), units(w.group * one), int(before), int(last), int(heads > 0 ? heads : 1)};
}
constexpr int kWindowF32Block = 64;  // rows that the fp32 window kernels load at a time
// Rows of their tiles: queries or keys of `heads` heads.
int window_f32_tile(int D, long long heads, int rows);
// The partials: fp32 [Z * Hk, slots, 2 (dV, dK), tile, D].
inline int64_t window_part_bytes(int tile, int Z, const WindowArgs& w, int D, const WindowSplit& s) {
  return int64_t(Z) * w.Hk * s.slots((w.Nk + tile - 1) / tile) * 2 * tile * D * 4;
}

// SIMT kernels (fp32 inputs; any strides).
cudaError_t launch_fwd_f32(int D, bool causal, const void* q, const void* k, const void* v, Strides4 sq,
                           Strides4 sk, Strides4 sv, const FwdArgs& a, float sm_scale, cudaStream_t s);
cudaError_t launch_bwd_dq_f32(int D, bool causal, const BwdArgs& a, cudaStream_t s);
cudaError_t launch_bwd_dkdv_f32(int D, bool causal, const BwdArgs& a, cudaStream_t s);

// Sliding window with sinks in fp32 (window_f32.cu; any strides). The backward writes dk, dv and dq from
// a.delta in the units of a.split; a.qk_scale and a.sm_scale are signed.
cudaError_t launch_window_fwd_f32(int D, const void* q, const void* k, const void* v, Strides4 sq, Strides4 sk,
                                  Strides4 sv, const FwdArgs& a, cudaStream_t s);
cudaError_t launch_window_bwd_f32(int D, const BwdArgs& a, cudaStream_t s);
// The same of rows against a sequence's first keys (kMaskRows; any strides but a unit one along D).
cudaError_t launch_rows_f32(int D, const void* k, const void* v, Strides4 sk, Strides4 sv, const RowsFwdArgs& a, cudaStream_t s);
cudaError_t launch_rows_bwd_f32(int D, const RowsBwdArgs& a, cudaStream_t s);
cudaError_t launch_rows_join(int D, bool is_f16, const JoinArgs& a, cudaStream_t s);

// delta = rowsum(dO * O) in fp32 (fp16 or fp32 inputs); also zeroes the rows of a.dq_acc and the
// counter a.grid_sync when they are set (the fused backward's workspace).
cudaError_t launch_bwd_preprocess(int D, bool is_f16, const BwdArgs& a, cudaStream_t s);

// Norms and rotation of query and key heads (norm_rope.cu). Strides in elements; the D stride is 1 and rows
// are 16-byte aligned.
struct Strides3 {
  int64_t z, h, n;
};
struct RopeTensor {
  const void* px;   // [Z, H, N, D]
  const void* pdy;  // backward: the gradient of the result
  void* py;         // the result or, backward, dx
  const void* w;    // [D]
  void* dw;         // backward: [D]
  Strides3 x, dy, y;
  int H;
  int items, blocks;  // work items and CTAs (set by the launcher)
};
struct RopeArgs {
  RopeTensor t[2];            // queries, keys
  const float *cos, *sin;     // [P, D / 2] dense
  const int* positions;       // [Z, N], or null: a row's own index n
  int64_t pos_z, pos_n;
  float* part;                // backward: a [D] partial of dw for each CTA (kRopeBlocksPerSm * SMs + 2 at most)
  int Z, N, P;
  int w_f32;                  // weights (and dw) are fp32, else the tensors' type
  float eps;
  int* status;
};
constexpr int kRopeBlocksPerSm = 4;
cudaError_t launch_norm_rope(int D, bool is_f16, bool interleaved, bool backward, RopeArgs a, cudaStream_t s);
// The weights' gradients from the CTAs' partials (a.part, of a.t[0].blocks CTAs, then a.t[1].blocks).
cudaError_t launch_norm_rope_dw(bool is_f16, int D, const RopeArgs& a, cudaStream_t s);

// A division by d of numbers below 2^31: of the high half of a product (Granlund and Montgomery, 1994). With l =
// ceil(log2 d) and m = ceil(2^(31 + l) / d) < 2^32 it is exact, as m d - 2^(31 + l) < d <= 2^l.
struct ByMultiple {
  uint32_t d, m;
  int shift;  // l - 1; -1: d is 1
  __device__ __forceinline__ uint32_t quotient(uint32_t x) const { return shift < 0 ? x : __umulhi(x, m) >> shift; }
};
inline ByMultiple by_multiple(int d) {
  int l = 0;
  while ((int64_t(1) << l) < d) ++l;
  return d <= 1 ? ByMultiple{1, 0, -1} : ByMultiple{uint32_t(d), uint32_t(((uint64_t(1) << (31 + l)) + d - 1) / d), l - 1};
}

// Rotation by positions on several axes (rope_axes.cu): positions is [A, Z, N].
constexpr int kRopeAxes = 4;
struct RopeAxesArgs : RopeArgs {
  int64_t pos_a;       // the axes' stride
  int A;               // 1 to kRopeAxes
  int back;            // without norms: turn by the negative angles
  uint32_t axes[4];    // the axis of each of the D / 2 pairs, 2 bits a pair
  ByMultiple chunks[2], tokens;  // divisions by a tensor's chunks of heads and by N (set by the launcher)
};
// Without the norms only forward (`back` for the gradients).
cudaError_t launch_rope_axes(int D, bool is_f16, bool norm, bool interleaved, bool backward, RopeAxesArgs a, cudaStream_t s);

// Attention of single tokens over a cache (decode.cu).
enum DecodeCache : int { kCacheF16, kCacheInt4, kCacheF32 };
struct DecodeArgs {
  const void* q;        // [Z, H, D]
  void* o;              // [Z, H, D]
  const void *k, *v;    // [Z, Hk, C, D], or the 4-bit cache's codes (Int4CacheArgs)
  const void *k_params, *v_params;  // 4-bit cache: its scales and minima
  Strides3 sq, so, sk, sv;
  const int* lengths;   // [Z]: tokens held, the query's own among them; null: all C
  float* part;          // [Z, H, nsplit, D] unnormalised partial rows (nsplit > 1)
  float* part_ml;       // [Z, H, nsplit, 2] their maxima and sums
  int Z, H, Hk, C;
  int window, sinks;    // window >= C: everything
  int nsplit;
  float qk_scale;       // sm_scale * log2(e)
  int* status;
  bool parts_only;      // write the parts, also one alone, and do not join them
  bool overlap;         // run beside the stream's last kernel (fp16, fp32)
};
// CTAs per SM that decode_splits aims at: as many as an SM holds. (fp16, 64 sequences of 4096 visible tokens, 4
// heads of 128: 2 parts each 82 us, 3 parts 86, 4 parts 90. 4 bits, 16 sequences of up to 65536 tokens: 10
// parts 112 us, 14 to 37 parts 110 to 106, but 2 such sequences: 27 us with 4 CTAs an SM, 32 with 8.)
constexpr int decode_ctas(DecodeCache cache) { return cache == kCacheF16 ? 2 : 4; }
// Up to so many parts are one cluster (the most that any GPU takes) and join through its shared memory; more, and
// the fp32 kernel's, are joined by a second kernel through the workspace.
constexpr int kClusterParts = 8;
inline bool decode_joins(int nsplit, DecodeCache cache) {
  return nsplit > (cache == kCacheF32 ? 1 : kClusterParts);
}
// Parts that the visible tokens are cut into: by the sizes alone, never by the lengths on the device.
int decode_splits(const DecodeArgs& a, int D, DecodeCache cache);
// The 4-bit cache (int4_cache.cu), for k and v each: codes [Z, Hk, C, D / 2] bytes, head dim 2 i in the low half
// of byte i; params [Z, Hk, C, D / 64, 2] fp16, the scale and minimum of each 64 head dims. All dense.
struct Int4CacheArgs {
  const void *k, *v;                // append: [Z, Hk, T, D] fp16 rows
  Strides3 sk, sv;
  void *k_out, *v_out;              // read: dense [Z, Hk, T, D] fp16
  uint8_t *k_codes, *v_codes;
  void *k_params, *v_params;
  const int* start;                 // [Z], or null (0): the position of row t = 0
  const int* counts;                // append, [Z], or null (T): rows t >= counts[z] are not kept
  int Z, Hk, T, C;
  int* status;
};
cudaError_t launch_int4_append(int D, const Int4CacheArgs& a, cudaStream_t s);
cudaError_t launch_int4_read(int D, const Int4CacheArgs& a, cudaStream_t s);

cudaError_t launch_decode(int D, DecodeCache cache, const DecodeArgs& a, cudaStream_t s);

}  // namespace tattn
