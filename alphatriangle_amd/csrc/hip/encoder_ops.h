// What the encoder operators' kernels (encoder_attn_*.hip, residual_norm_kernels.hip) and their host side
// (csrc/torch/encoder_ops.cpp) share: argument blocks, entry points and the rules that pick a tiling.  No HIP in here.
#pragma once

struct ihipStream_t;

namespace atrihip {

constexpr int kTile = 64;  // keys (queries in the key-owned pass) staged per step of the attention kernels

struct EncAttnArgs {
  const void* q;       // [B, Lq, H M, D] by strides
  const void* k;       // [B, Lk, KV M, D]
  const void* v;       // [B, Lk, KV, DV]
  const void* dout;    // [B, Lq, H, DV]
  void* out;           // [B, Lq, H, DV]
  void* dq;
  void* dk;
  void* dv;
  const float* table;  // [buckets, H M]; nullptr: no position bias
  const int* lut;      // [2 R + 1] bucket of every clamped position difference
  const int* order;    // [2 R + 1] differences by bucket: those of bucket b at start[b] .. start[b + 1] - 1
  const int* start;
  const float* lam;    // [H] (M = 2)
  const unsigned char* mask;  // [B, Lk] bytes by strides (nonzero: the key takes part); nullptr: all keys
  unsigned long long* words;  // [B, ceil(Lk / 64)] validity bit of every key, made from mask by the forward pass; nullptr: all keys
  const int* qoff;     // [B] position of the first query, nullptr: q0 for all samples
  float* stat;         // [M, B H Lq, 2] row maximum of x / scale (+inf: no key) and 1 / sum (0: no key); nullptr: not wanted
  float* o32;          // [M] x [B, Lq, H, DV] per-map outputs in 32 bits by strides (backward: their product with dO is delta)
  float* delta;        // [M, B H Lq]
  float* part_o;       // [splits, M, B H Lq, DV] unnormalised partial outputs (splits > 1)
  float* part_ml;      // [splits, M, B H Lq, 2] their maxima and sums
  float* hist;         // [workgroups of the query-owned pass, M, 2 R + 1] sums of dS by position difference; nullptr: not wanted
  float* mid;          // [shares, H M, 2 R + 1] the same, added up over shares of the samples and query tiles
  float* dq_part;      // [q_splits, B, H, Lq, M D] partial dQ in 32 bits (q_splits > 1)
  float* kv_part;      // [k_splits, B, KV, Lk, M D + DV] partial dK and dV (k_splits > 1)
  float* dtable;       // [buckets, H M]
  float* dlam_part;    // [workgroups of the query-owned pass, 4] sums of delta_2 by wave
  float* dlam;         // [H]; nullptr: not wanted
  long long qs[3], ks[3], vs[3], os[3], gs[3], dqs[3], dks[3], dvs[3];  // element strides: sample, token, head
  long long o32s[4];   // o32: sample, token, head, map
  long long ms[2];     // mask: sample, key
  int B, Lq, Lk, H, KV, D, DV, M;
  int R, W, q0;        // clamp of the position difference; board width (0: sequence); position of the first query
  int buckets, bf16, shares, hist_rows;
  int splits, chunk;      // forward: key ranges per query tile, samples a workgroup walks one after the other
  int q_splits, q_chunk;  // query-owned pass: the same
  int k_splits, k_chunk;  // key-owned pass: query ranges per key tile, samples
  long long q_groups;     // workgroups of the query-owned pass that hist and dlam_part have room for: refused unless they are the launch's
  float scale;
};

// Boards of 2 to 4 key tiles keep their bias (and the sums of dS by pair) in registers over all samples a workgroup walks: every
// sample has the same positions.  The tiles are then unrolled: NT of them, with as many 16-row columns per wave as
// keep 64 registers for each.  0: the general form (sequences, smaller and larger boards).
inline int enc_board_tiles(int W, int Lk, int D, int M) {
  const int tiles = (Lk + kTile - 1) / kTile;
  if (W <= 0 || D > 32 || tiles < 2) return 0;
  return tiles == 2 ? 2 : tiles <= 4 && M == 1 ? 4 : 0;
}
enum EncPass { kEncForward = 0, kEncQueries = 1, kEncKeys = 2 };  // forward, query-owned and key-owned backward pass
// 16-row columns per wave: queries in the forward and the query-owned pass, keys in the key-owned one.
constexpr int enc_columns_of(int D, int M, int nt, bool bf16, int pass) {
  if (M == 2 || D > 64 || nt == 4) return 1;
  // fp32 operands take three times the registers: one where two spill (two 2048-token sequences of eight 64-wide heads, backward:
  // 574 us with two, 408 us with one; 32-wide heads: 258 and 316 us)
  if (!bf16 && D > 32 && pass != kEncForward) return 1;
  // two: every staged fragment feeds two products (256 boards of 120 cells, fp32, forward: 33 us with one, 29 us with two); one
  // where bias and sums of dS share the registers (query-owned pass, with the fp32 instruction: 68 us with two, 51 us with one)
  return nt == 2 && pass == kEncQueries ? 1 : 2;
}
inline int enc_columns(int W, int L, int Lk, int D, int M, bool bf16, int pass) {
  const int nt = enc_board_tiles(W, Lk, D, M);
  return nt == 0 && pass == kEncForward && L <= 64 ? 1 : enc_columns_of(D, M, nt, bf16, pass);
}
// Waves per SIMD the register allocation of a kernel leaves room for.  These kernels wait on LDS and on the matrix and
// exponential pipes, so a second wave is worth some spilled registers (two 4095-token sequences in bf16, both backward
// passes: 857 us with one, 466 us with two); a third is not, except where the kernel nearly fits anyway.  One where a
// workgroup's tiles take more than half of the LDS (three parts of 128 values, or of two maps of 64) or it keeps the sums of two maps.
constexpr int enc_waves(int D, int M, int nt, int columns, bool bf16, int pass) {
  if (!bf16 && D * M == 128) return 1;
  if (pass == kEncForward) return bf16 && (nt == 4 || (nt == 0 && M == 1 && D == 64 && columns == 2)) ? 3 : 2;
  return pass == kEncQueries && nt == 2 && M == 2 ? 1 : 2;
}

// LDS of a workgroup.  Form of the staged rows: bf16, three bf16 parts of fp32, fp32.
enum EncForm { kRowsBf16 = 0, kRowsParts = 1, kRowsFp32 = 2 };
constexpr int kMaxLds = 160 * 1024;  // of a compute unit
constexpr int kDsPitch = kTile + 4;  // row pitch of a wave's 16 x 64 tile of dS on its way to the sums by position
constexpr int enc_row_bytes(int form, int width, bool transposed) {  // the paddings of Ops<T>::row_pitch and tr_pitch
  return form == kRowsFp32 ? 4 * (width + 4) : (form == kRowsParts ? 6 : 2) * (width + (transposed ? 16 : 8));
}
constexpr int enc_tile_bytes(int form, int D, int M, int pass) { return kTile * (M * enc_row_bytes(form, D, false) + enc_row_bytes(form, D * M, pass == kEncForward)); }
// slots: positions of the table (0: no bias); hist_rows: rows of sums by position (query-owned pass).
constexpr int enc_lds_bytes(int form, int D, int M, int nt, int pass, int slots, int hist_rows) {
  const int fixed = enc_tile_bytes(form, D, M, pass) + (nt ? nt : 1) * kTile * 4;
  if (pass == kEncForward) return fixed + 4 * M * slots;
  if (pass == kEncKeys) return fixed + 4 * (3 * M * kTile + 4 + M * slots);
  return fixed + (slots ? 4 * ((M * slots + 3) / 4 * 4 + 4 * 16 * kDsPitch + hist_rows * M * slots) : 0);
}
// The query-owned pass of two 64-wide maps takes fp32 rows as they are where three parts leave no room for the table (more than 2416 positions).
constexpr int enc_query_form(bool bf16, int D, int M, int slots) {
  return bf16 ? kRowsBf16 : D == 64 && M == 2 && enc_lds_bytes(kRowsParts, D, M, 0, kEncQueries, slots, 1) > kMaxLds ? kRowsFp32 : kRowsParts;
}
constexpr int enc_per_cu(int waves, int lds) { return lds > kMaxLds ? 0 : kMaxLds / lds < waves ? kMaxLds / lds : waves; }
// Rows of sums by position: one per wave; one for all, which the waves add to in turns, where four do not fit or would cost a
// workgroup per compute unit.
constexpr int enc_hist_rows(int form, int D, int M, int nt, int slots, int waves) {
  const int four = enc_per_cu(waves, enc_lds_bytes(form, D, M, nt, kEncQueries, slots, 4));
  return four > 0 && four >= enc_per_cu(waves, enc_lds_bytes(form, D, M, nt, kEncQueries, slots, 1)) ? 4 : 1;
}
// Workgroups of a pass that a compute unit holds: as many as its registers and its LDS leave room for.  R: clamp of the position
// difference (-1: no bias); own_heads: no shared key / value heads; sums: sums by position are wanted.
inline int enc_workgroups(bool bf16, int D, int M, int R, int W, int Lq, int Lk, bool own_heads, int pass, bool sums) {
  const int board = pass == kEncKeys && !own_heads ? 0 : W;  // shared heads take the general form of the key-owned pass
  const int nt = enc_board_tiles(board, Lk, D, M), width = D <= 32 ? 32 : D <= 64 ? 64 : 128, slots = 2 * R + 1 > 0 ? 2 * R + 1 : 0;
  const int waves = enc_waves(width, M, nt, enc_columns(board, Lq, Lk, D, M, bf16, pass), bf16, pass);
  const int form = pass == kEncQueries ? enc_query_form(bf16, width, M, slots) : bf16 ? kRowsBf16 : kRowsParts;
  const int n = enc_per_cu(waves, enc_lds_bytes(form, width, M, nt, pass, slots, sums && slots ? enc_hist_rows(form, width, M, nt, slots, waves) : 0));
  return n > 0 ? n : 1;
}

// The residual joint: threads that own a row (8 values each) and threads of a workgroup.
inline int lanes_of(int D) {
  int lanes = 16;
  while (lanes * 8 < D) lanes *= 2;
  return lanes;
}
constexpr int threads_of(int lanes) { return lanes < 256 ? 256 : lanes; }

struct ResNormArgs {
  const void* x;        // [N, D] residual stream
  const void* z;        // [N, D] block output
  const void* gate;     // gate logits in z's type: [N, D] (mode 2), [N] (mode 1), nullptr (mode 0)
  const float* scale;   // [D]
  const float* post_w;
  const float* post_b;
  const float* pre_w;
  const float* pre_b;
  void* y;              // [N, D] in x's type
  void* h;              // [N, D] in z's type
  float* stats;         // [N, 4]: mean and 1 / deviation of z, of y; nullptr in the forward pass: not wanted
  const void* dy;       // gradients of y and h; nullptr: zero
  const void* dh;
  void* dx;
  void* dz;
  void* dgate;
  float* part;          // [workgroups, 5, D] partial sums of dscale, dpost_w, dpost_b, dpre_w, dpre_b
  float* dparams;       // [5, D]
  long long N;
  int D, gate_mode, groups, x_bf16, z_bf16;
  float eps;
};

}  // namespace atrihip

extern "C" {
// 0, a HIP error code, or a negative code for arguments rejected before any launch.
int atri_enc_attn_fwd(const atrihip::EncAttnArgs* args, ihipStream_t* stream);
int atri_enc_attn_bwd(const atrihip::EncAttnArgs* args, ihipStream_t* stream);
int atri_resnorm_fwd(const atrihip::ResNormArgs* args, ihipStream_t* stream);
int atri_resnorm_bwd(const atrihip::ResNormArgs* args, ihipStream_t* stream);
}
