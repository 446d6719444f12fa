// Backward pass of the encoder attention operators (encoder_attn.hpp has the operand layout).  Two passes over the score
// matrix, each recomputing it from Q, K and the forward's row maximum and sum (kept apart:
// their joint logarithm would lose the sum beside a large maximum), so that every gradient is summed by one owner in a
// fixed order (a single pass would add dQ with floating-point atomics):
//   query-owned:  dS = P (dP - delta), dP = dO V^T;  dQ = scale dS K;  delta = dO . o per map;  sums of dS by position
//                 difference (the bias table's gradient before it is folded into buckets)
//   key-owned:    dV = (P_1 - lam P_2)^T dO;  dK_m = scale dS_m^T Q_m
// With two maps dP_1 = dO V^T and dP_2 = -lam dP_1, so one product serves both; d lam = -sum delta_2.
#include <type_traits>

#include "encoder_attn.hpp"

using namespace atrihip;

namespace {

__device__ const float kZeroRow[8] __attribute__((aligned(16))) = {};  // read in place of rows and columns that are not there
// Fragments per probability and score gradient: two in bf16, 16 bits, so that a gradient's own rounding is the only one that counts
// (with one: 2.4e-3 off where rounding alone leaves 1.66e-3; two 4095-token sequences, query- and key-owned pass: 210 and 230 us with one,
// 241 and 289 us with two).
template <typename T>
constexpr int grad_parts() { return Ops<T>::kBf16 ? 2 : 1; }

__device__ __forceinline__ void wave_lds_fence() {  // orders a wave's own LDS writes before its other lanes' reads
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Adds a wave's 16 x 64 tile of dS (LDS, row = query) to its sums by position difference, without atomics (LDS additions of
// floats took 2.8 cycles a lane here) and in a fixed order.
// Sequences: lane l adds up the wrapped diagonal key = (l - 15 + row) mod 64, each element of the tile once, in registers;
// different diagonals have different (unclamped) differences, so every slot has one writer.  Clamped ones go to lo / hi.
// Boards: row by row; a row's 64 keys lie at 64 different positions, so again no two lanes meet in a slot.
__device__ __forceinline__ void add_tile(const EncAttnArgs& a, float* sums, const float* ds, int pos_k, int pos_q, int k0, int q0, int lane, float& lo,
                                         float& hi) {
  const int R2 = 2 * a.R;
  if (a.W == 0) {
    float before = 0.f, after = 0.f;  // rows past the wrap (diagonal lane - 15), rows before it (diagonal lane + 49)
#pragma unroll
    for (int row = 0; row < 16; ++row) {
      const float v = ds[row * kDsPitch + ((lane - 15 + row) & 63)];
      if (row >= 15 - lane) before += v; else after += v;
    }
    const int slot = k0 - q0 + a.R + lane - 15, slot2 = slot + 64;
    if (slot <= 0) lo += before; else if (slot >= R2) hi += before; else sums[slot] += before;
    if (lane < 15) {
      if (slot2 <= 0) lo += after; else if (slot2 >= R2) hi += after; else sums[slot2] += after;
    }
    return;
  }
#pragma unroll
  for (int row = 0; row < 16; ++row) {
    const int slot = pos_k - __builtin_amdgcn_readlane(pos_q, row) + a.R;
    const float v = ds[row * kDsPitch + lane];
    if (v != 0.f && slot >= 0 && slot <= R2) sums[slot] += v;  // rows and keys beyond the board hold zeros
    wave_lds_fence();
  }
}

// One 4-wave workgroup per (head, 64 QS queries, key range) and q_chunk samples, one after the other.
// Measured (sizes as in the forward pass): boards of 120 cells, fp32 44 us; 252 cells, bf16 67 us; 4095 tokens, bf16 241 us; 2000
// tokens, two maps, fp32 252 us; bound like the forward pass, with five LDS reads and 36 vector instructions per pair and lane in
// the fp32 form.  K is read transposed from a tile at row_pitch, where two of eight rows share banks: two conflict cycles per LDS
// instruction.
template <typename T, int D, int M, int QS, bool BIAS, int NT>
__global__ __launch_bounds__(256, enc_waves(D, M, NT, QS, Ops<T>::kBf16, kEncQueries)) void enc_attn_bwd_q_kernel(EncAttnArgs a) {
  using O = Ops<T>;
  using Frag = typename O::Frag;
  constexpr int DV = D * M, DC = D / O::kDims, VC = DV / O::kDims, ND = D / 16, NKB = 4 / O::kSub, PL = grad_parts<T>();
  constexpr bool TILE_SUMS = NT == 0 && std::is_same<T, Split>::value;  // as in the forward pass
  constexpr int PK = O::row_pitch(D), PV = O::row_pitch(DV), TK = O::kParts * kTile * PK;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  typename O::Lds* k_lds = reinterpret_cast<typename O::Lds*>(smem);
  typename O::Lds* v_lds = k_lds + M * TK;
  int* pos_lds = reinterpret_cast<int*>(v_lds + O::kParts * kTile * PV);
  float* bias_lds = reinterpret_cast<float*>(pos_lds + (NT ? NT : 1) * kTile);
  const int slots = BIAS ? 2 * a.R + 1 : 0, R2 = 2 * a.R;
  float* ds_lds = bias_lds + ((M * slots + 3) & ~3);
  float* sum_lds = ds_lds + 4 * 16 * kDsPitch;

  const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, q4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // what follows from it (owned rows, clamped sides) stays in scalar registers
  const int nqt = (a.Lq + 64 * QS - 1) / (64 * QS);
  const int group_id = xcd_order(blockIdx.x, gridDim.x);
  int id = group_id;
  const int qt = id % nqt;
  id /= nqt;
  const int split = id % a.q_splits;
  id /= a.q_splits;
  const int h = id % a.H, kvh = h / (a.H / a.KV);
  const int b_first = id / a.H * a.q_chunk, b_last = b_first + a.q_chunk < a.B ? b_first + a.q_chunk : a.B;
  const int tiles = (a.Lk + kTile - 1) / kTile;
  const int per = (tiles + a.q_splits - 1) / a.q_splits;
  const int t_first = split * per, t_last = t_first + per < tiles ? t_first + per : tiles;
  const bool want_sums = BIAS && a.hist != nullptr;
  float* my_sums = sum_lds + (a.hist_rows == 4 ? wave * M * slots : 0);
  const long long rows = (long long)a.B * a.H * a.Lq;
  const int q_first = (qt * 4 + wave) * 16 * QS;
  const bool busy = q_first < a.Lq;
  const float lam = M == 2 ? a.lam[h] : 0.f;
  const float sl2 = a.scale * kLog2E;

  Stage<T, D> sk[M];
  Stage<T, DV> sv;
  auto fetch = [&](const TileWalk& w) {
    const typename O::Mem* kb = reinterpret_cast<const typename O::Mem*>(a.k) + w.sample * a.ks[0] + (long long)kvh * M * a.ks[2];
#pragma unroll
    for (int m = 0; m < M; ++m) sk[m].load(kb + m * a.ks[2], a.ks[1], w.tile * kTile, w.word, a.D, tid);
    sv.load(reinterpret_cast<const typename O::Mem*>(a.v) + w.sample * a.vs[0] + kvh * a.vs[2], a.vs[1], w.tile * kTile, w.word, a.DV, tid);
  };
  TileWalk walk;
  if constexpr (NT == 0) {
    walk.start(a, b_first, b_last, t_first, t_last);
  } else {
    walk.sample = b_first;
    walk.tile = 0;
    walk.word = board_word(a, b_first, 0);
  }
  if (walk.sample < b_last) fetch(walk);
  if constexpr (BIAS) fill_bias(a, bias_lds, h, M, tid);
  if (want_sums)
    for (int i = tid; i < a.hist_rows * M * slots; i += 256) sum_lds[i] = 0.f;
  float lo[M], hi[M];
#pragma unroll
  for (int m = 0; m < M; ++m) lo[m] = hi[m] = 0.f;
  float delta2_sum = 0.f;  // of this lane's queries over the samples
  int token_q[QS];
#pragma unroll
  for (int s = 0; s < QS; ++s) token_q[s] = BIAS ? token_pos(q_first + s * 16 + l15, a.W) : 0;
  // Boards: the bias of this wave's pairs, and the sums of their dS over the samples.
  float4v bias_reg[M][QS][NT ? NT * 4 : 1], sum_reg[M][QS][NT ? NT * 4 : 1];
  if constexpr (NT > 0) {
    if (tid < NT * kTile) pos_lds[tid] = token_pos(tid, a.W);
    __syncthreads();
#pragma unroll
    for (int kt = 0; kt < NT * 4; ++kt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = kt * 16 + q4 * 4 + j, pos = pos_lds[key];
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
          for (int s = 0; s < QS; ++s) {
            bias_reg[m][s][kt][j] = key < a.Lk ? bias_lds[m * slots + clamp_slot(pos - token_q[s] + a.R, R2)] : -INFINITY;
            sum_reg[m][s][kt][j] = 0.f;
          }
      }
  }

  for (int b = b_first; b < b_last; ++b) {
    const int origin = BIAS ? query_origin(a, b) : 0;
    const long long row0 = ((long long)b * a.H + h) * a.Lq;
    Frag qf[M][QS][DC], dof[QS][VC];
    float top[M][QS], inv[M][QS], delta[M][QS];
#pragma unroll
    for (int s = 0; s < QS; ++s) {
      const int query = q_first + s * 16 + l15;
      const bool valid = query < a.Lq;
      load_rows<T, VC>(dof[s], reinterpret_cast<const typename O::Mem*>(a.dout) + b * a.gs[0] + (long long)query * a.gs[1] + h * a.gs[2], valid, a.DV, q4);
      // The matrix instructions round sums down by a little (0.01 to 0.03 units in the last place on average), which adds up over
      // the pairs that share a table entry: every second row takes the other sign, from dO and delta to the 1 / sum that its
      // results meet (one sequence of 3000 tokens, error of the far buckets: 1e-5 without).
      const bool other = ((query + b + h) & 1) != 0;
#pragma unroll
      for (int c = 0; c < VC; ++c) O::negate(dof[s][c], other);
#pragma unroll
      for (int m = 0; m < M; ++m) {
        load_rows<T, DC>(qf[m][s], reinterpret_cast<const typename O::Mem*>(a.q) + b * a.qs[0] + (long long)query * a.qs[1] + (long long)(h * M + m) * a.qs[2], valid,
                         a.D, q4);
        float2 st = make_float2(INFINITY, 0.f);
        if (valid) st = *reinterpret_cast<const float2*>(a.stat + 2 * (m * rows + row0 + query));
        top[m][s] = st.x;
        inv[m][s] = other ? -st.y : st.y;
        const float* o = a.o32 + b * a.o32s[0] + (long long)query * a.o32s[1] + h * a.o32s[2] + m * a.o32s[3];
        // delta = dO . o by the instructions that make dP (o rows as the other operand, the diagonal of the product): where a row
        // has a single key, o is v and dP - delta is what the rounding of its probability leaves.
        float4v prod = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < VC; ++c) {
          const int col = c * O::kDims + q4 * O::kLane;
          prod = O::mma_rows32(valid && col < a.DV ? o + col : kZeroRow, dof[s][c], prod);
        }
        const float mine = l15 & 2 ? (l15 & 1 ? prod[3] : prod[2]) : (l15 & 1 ? prod[1] : prod[0]);
        delta[m][s] = quad_row_sum(q4 == l15 >> 2 ? mine : 0.f);
        if (valid && q4 == 0 && split == 0) {
          const float signless = other ? -delta[m][s] : delta[m][s];
          a.delta[m * rows + row0 + query] = signless;
          if (M == 2 && m == 1) delta2_sum += signless;
        }
      }
    }
    float4v dq[M][QS][ND];
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int s = 0; s < QS; ++s)
#pragma unroll
        for (int n = 0; n < ND; ++n) dq[m][s][n] = float4v{0.f, 0.f, 0.f, 0.f};

    float base[M][QS];
    bool far_any = false;
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int s = 0; s < QS; ++s) {
        base[m][s] = Exponent::base_of(top[m][s], sl2);
        far_any |= Exponent::far(base[m][s]);
      }
    const bool far = __any(far_any);
    // One staged tile; kt0 is its first 16-key block where bias and sums are in registers.
    auto tile = [&](auto kt0_) {
      constexpr int kt0 = decltype(kt0_)::value;
      const unsigned long long word = NT > 0 && !a.words ? ~0ULL : walk.word;
      const int t0 = walk.tile * kTile;
      __syncthreads();
#pragma unroll
      for (int m = 0; m < M; ++m) sk[m].store(k_lds + m * TK, PK, tid);
      sv.store(v_lds, PV, tid);
      if (BIAS && NT == 0 && tid < kTile) pos_lds[tid] = token_pos(t0 + tid, a.W);
      __syncthreads();
      if constexpr (NT == 0) {
        walk.next();
      } else {
        constexpr bool last = kt0 / 4 + 1 == NT;
        walk.tile = last ? 0 : kt0 / 4 + 1;
        walk.sample = b + (last ? 1 : 0);
        if (walk.sample < b_last) walk.word = board_word(a, walk.sample, walk.tile);
      }
      if (walk.sample < b_last) fetch(walk);
      float4v ds[M][QS][4];  // without the row's 1 / sum, which joins at the end of the row
      float4v dq_tile[M][QS][ND];  // TILE_SUMS
      int side[QS];
      if (busy) {
#pragma unroll
        for (int s = 0; s < QS; ++s) {
          const int qa = q_first + s * 16 + origin;
          side[s] = BIAS && NT == 0 ? clamped_side(a, t0, t0 + kTile - 1, qa, qa + 15) : 0;
        }
        // PLAIN: no far row and no masked key, one basic block
        auto scores = [&](auto plain_) {
          constexpr bool PLAIN = decltype(plain_)::value;
#pragma unroll
          for (int kb = 0; kb < NKB; ++kb) {
            // where the scores start
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
              for (int s = 0; s < QS; ++s) {
                float4v* x = &ds[m][s][kb * O::kSub];
                if constexpr (NT > 0) {
#pragma unroll
                  for (int u = 0; u < O::kSub; ++u) x[u] = bias_reg[m][s][kt0 + kb * O::kSub + u];
                } else if constexpr (BIAS) {
                  const float* bias = bias_lds + m * slots;
                  if (side[s] != 0) {
                    const float c = bias[side[s] > 0 ? R2 : 0];
#pragma unroll
                    for (int u = 0; u < O::kSub; ++u) x[u] = float4v{c, c, c, c};
                  } else {
                    const int off = a.R - token_q[s] - origin;
#pragma unroll
                    for (int u = 0; u < O::kSub; ++u) {
                      const int4 p4 = *reinterpret_cast<const int4*>(pos_lds + (kb * O::kSub + u) * 16 + q4 * 4);
                      const int pj[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
                      for (int j = 0; j < 4; ++j) x[u][j] = bias[clamp_slot(pj[j] + off, R2)];
                    }
                  }
                } else {
#pragma unroll
                  for (int u = 0; u < O::kSub; ++u) x[u] = float4v{0.f, 0.f, 0.f, 0.f};
                }
              }
#pragma unroll
            for (int u = 0; u < O::kSub; ++u) {
              const int kt = kb * O::kSub + u;
              float4v dp[QS];
#pragma unroll
              for (int s = 0; s < QS; ++s) dp[s] = float4v{0.f, 0.f, 0.f, 0.f};  // not -delta: every partial sum would be rounded at its size
#pragma unroll
              for (int c = 0; c < VC; ++c) {
                const Frag vf = O::row_frag(v_lds, PV, kt * 16 + l15, c, q4);
#pragma unroll
                for (int s = 0; s < QS; ++s) dp[s] = O::mma(vf, dof[s][c], dp[s]);
              }
#pragma unroll
              for (int m = 0; m < M; ++m) {
#pragma unroll
                for (int c = 0; c < DC; ++c) {
                  const Frag kf = O::row_frag(k_lds + m * TK, PK, kt * 16 + l15, c, q4);
#pragma unroll
                  for (int s = 0; s < QS; ++s) ds[m][s][kt] = O::mma(kf, qf[m][s][c], ds[m][s][kt]);
                }
#pragma unroll
                for (int s = 0; s < QS; ++s) {
                  float4v x = ds[m][s][kt];
                  if (!PLAIN && far) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[j] = Exponent::far_(x[j], top[m][s], sl2);
                  } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[j] = Exponent::near_(x[j], base[m][s], sl2);
                  }
#pragma unroll
                  for (int j = 0; j < 4; ++j) x[j] *= dp[s][j] - delta[m][s];
                  if (!PLAIN && word != ~0ULL) {
                    const unsigned bits = (unsigned)(word >> (kt * 16 + q4 * 4));
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[j] = (bits >> j) & 1 ? x[j] : 0.f;
                  }
                  ds[m][s][kt] = x;
                }
              }
            }
#pragma unroll
            for (int m = 0; m < M; ++m) {
              Frag sf[QS][PL];
#pragma unroll
              for (int s = 0; s < QS; ++s) acc_parts<T>(sf[s], &ds[m][s][kb * O::kSub]);
#pragma unroll
              for (int n = 0; n < ND; ++n) {
                const Frag kf = O::tr_frag(k_lds + m * TK, PK, kb, n, l15, q4);
#pragma unroll
                for (int s = 0; s < QS; ++s) {
                  if constexpr (TILE_SUMS) dq_tile[m][s][n] = mma_parts<T>(kf, sf[s], kb == 0 ? float4v{0.f, 0.f, 0.f, 0.f} : dq_tile[m][s][n]);
                  else dq[m][s][n] = mma_parts<T>(kf, sf[s], dq[m][s][n]);
                }
              }
            }
          }
        };
        if (far || word != ~0ULL) scores(std::false_type{});
        else scores(std::true_type{});
        if constexpr (TILE_SUMS) {
#pragma unroll
          for (int m = 0; m < M; ++m)
#pragma unroll
            for (int s = 0; s < QS; ++s)
#pragma unroll
              for (int n = 0; n < ND; ++n) dq[m][s][n] += dq_tile[m][s][n];
        }
        if constexpr (NT > 0) {
#pragma unroll
          for (int m = 0; m < M; ++m)
#pragma unroll
            for (int s = 0; s < QS; ++s) {
              const float c = m == 0 ? inv[m][s] : -lam * inv[m][s];
#pragma unroll
              for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                for (int j = 0; j < 4; ++j) sum_reg[m][s][kt0 + kt][j] = fmaf(ds[m][s][kt][j], c, sum_reg[m][s][kt0 + kt][j]);
            }
        }
      }
      if constexpr (BIAS && NT == 0) {
        if (want_sums) {
          const int pos_k = pos_lds[lane];
          for (int turn = 0; turn < (a.hist_rows == 4 ? 1 : 4); ++turn) {  // one row of sums for all waves: they take turns
            if (busy && (a.hist_rows == 4 || turn == wave)) {
              float* buf = ds_lds + wave * 16 * kDsPitch;
#pragma unroll
              for (int m = 0; m < M; ++m)
#pragma unroll
                for (int s = 0; s < QS; ++s) {
                  const float c = m == 0 ? inv[m][s] : -lam * inv[m][s];
                  if (side[s] != 0) {
                    float all = 0.f;
#pragma unroll
                    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                      for (int j = 0; j < 4; ++j) all += ds[m][s][kt][j];
                    if (side[s] > 0) hi[m] = fmaf(all, c, hi[m]); else lo[m] = fmaf(all, c, lo[m]);
                  } else {
#pragma unroll
                    for (int kt = 0; kt < 4; ++kt)
                      *reinterpret_cast<float4v*>(buf + l15 * kDsPitch + kt * 16 + q4 * 4) = ds[m][s][kt] * c;
                    wave_lds_fence();
                    add_tile(a, my_sums + m * slots, buf, pos_k, token_q[s] + origin, t0, q_first + s * 16 + origin, lane, lo[m], hi[m]);
                    wave_lds_fence();
                  }
                }
            }
            if (a.hist_rows != 4) __syncthreads();
          }
        }
      }
    };
    if constexpr (NT == 0) {
      while (walk.sample == b) tile(std::integral_constant<int, 0>{});
    } else {
      tile(std::integral_constant<int, 0>{});
      tile(std::integral_constant<int, 4>{});
      if constexpr (NT == 4) {
        tile(std::integral_constant<int, 8>{});
        tile(std::integral_constant<int, 12>{});
      }
    }

    if (!busy) continue;
#pragma unroll
    for (int s = 0; s < QS; ++s) {
      const int query = q_first + s * 16 + l15;
      if (query >= a.Lq) continue;
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const float c = a.scale * (m == 0 ? inv[m][s] : -lam * inv[m][s]);
        typename O::Mem* row = reinterpret_cast<typename O::Mem*>(a.dq) + b * a.dqs[0] + (long long)query * a.dqs[1] + (long long)(h * M + m) * a.dqs[2];
        float* part = a.dq_part + ((split * rows + row0 + query) * M + m) * a.D;
#pragma unroll
        for (int n = 0; n < ND; ++n) {
          const int dim = n * 16 + q4 * 4;
          const float4v g = dq[m][s][n] * c;
          if (dim >= a.D) continue;
          if (a.q_splits > 1) Ops<float>::store4(part + dim, g[0], g[1], g[2], g[3]);
          else O::store4(row + dim, g[0], g[1], g[2], g[3]);
        }
      }
    }
  }
  if (M == 2 && a.dlam) {
    const float all = wave_sum(delta2_sum);
    if (lane == 0) a.dlam_part[(size_t)group_id * 4 + wave] = all;
  }
  if (!want_sums) return;
  if constexpr (NT > 0) {  // the board's pairs, once for all samples
    float* buf = ds_lds + wave * 16 * kDsPitch;
    for (int turn = 0; turn < (a.hist_rows == 4 ? 1 : 4); ++turn) {
      if (busy && (a.hist_rows == 4 || turn == wave)) {
#pragma unroll
        for (int tt = 0; tt < NT; ++tt)
#pragma unroll
          for (int m = 0; m < M; ++m)
#pragma unroll
            for (int s = 0; s < QS; ++s) {
#pragma unroll
              for (int kt = 0; kt < 4; ++kt)
                *reinterpret_cast<float4v*>(buf + l15 * kDsPitch + kt * 16 + q4 * 4) = sum_reg[m][s][tt * 4 + kt];
              wave_lds_fence();
              add_tile(a, my_sums + m * slots, buf, pos_lds[tt * kTile + lane], token_q[s], 0, 0, lane, lo[m], hi[m]);
              wave_lds_fence();
            }
      }
      if (a.hist_rows != 4) __syncthreads();
    }
  }
  // The clamped ends, wave by wave, then the four rows of sums in order.
#pragma unroll
  for (int m = 0; m < M; ++m) {
    const float l = wave_sum(lo[m]), u = wave_sum(hi[m]);
    for (int turn = 0; turn < 4; ++turn) {
      __syncthreads();
      if (turn == wave && lane == 0) {
        my_sums[m * slots] += l;
        my_sums[m * slots + R2] += u;
      }
    }
  }
  __syncthreads();
  float* part = a.hist + (size_t)group_id * M * slots;
  for (int i = tid; i < M * slots; i += 256) {
    float s = sum_lds[i];
    if (a.hist_rows == 4) s = (s + sum_lds[M * slots + i]) + (sum_lds[2 * M * slots + i] + sum_lds[3 * M * slots + i]);
    part[i] = s;
  }
}

// One 4-wave workgroup per (key / value head, 64 KS keys, query range) and k_chunk samples; a wave owns 16 KS keys and walks the
// query tiles of every query head that shares them.
// Measured (same sizes): 53 us, 82 us, 289 us and 333 us; Q and dO are read transposed at row_pitch as K above.  One pass over the
// pairs for all gradients would save two of seven products, but needs dQ summed across workgroups (or a board's dS through LDS, as
// many reads as the products it saves).
template <typename T, int D, int M, int KS, bool BIAS, int NT>
__global__ __launch_bounds__(256, enc_waves(D, M, NT, KS, Ops<T>::kBf16, kEncKeys)) void enc_attn_bwd_k_kernel(EncAttnArgs a) {
  using O = Ops<T>;
  using Frag = typename O::Frag;
  constexpr int DV = D * M, DC = D / O::kDims, VC = DV / O::kDims, ND = D / 16, NV = DV / 16, NKB = 4 / O::kSub, PL = grad_parts<T>();
  constexpr bool TILE_SUMS = NT == 0 && std::is_same<T, Split>::value;  // as in the forward pass
  constexpr int PQ = O::row_pitch(D), PG = O::row_pitch(DV), TQ = O::kParts * kTile * PQ;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  typename O::Lds* q_lds = reinterpret_cast<typename O::Lds*>(smem);
  typename O::Lds* g_lds = q_lds + M * TQ;
  int* pos_lds = reinterpret_cast<int*>(g_lds + O::kParts * kTile * PG);
  float* top_lds = reinterpret_cast<float*>(pos_lds + (NT ? NT : 1) * kTile);
  float* inv_lds = top_lds + M * kTile;
  float* delta_lds = inv_lds + M * kTile;
  int* far_lds = reinterpret_cast<int*>(delta_lds + M * kTile);  // one flag per map (and padding)
  float* bias_lds = reinterpret_cast<float*>(far_lds + 4);

  const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, q4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // what follows from it (owned rows, clamped sides) stays in scalar registers
  const int nkt = (a.Lk + 64 * KS - 1) / (64 * KS);
  int id = xcd_order(blockIdx.x, gridDim.x);
  const int kt_ = id % nkt;
  id /= nkt;
  const int split = id % a.k_splits;
  id /= a.k_splits;
  const int kvh = id % a.KV, group = a.H / a.KV;
  const int b_first = id / a.KV * a.k_chunk, b_last = b_first + a.k_chunk < a.B ? b_first + a.k_chunk : a.B;
  const int tiles = (a.Lk + kTile - 1) / kTile, qtiles = (a.Lq + kTile - 1) / kTile;
  const int all = group * qtiles, per = (all + a.k_splits - 1) / a.k_splits;
  const int s_first = split * per, s_last = s_first + per < all ? s_first + per : all;
  const int k_first = (kt_ * 4 + wave) * 16 * KS;
  const int R2 = 2 * a.R, slots = BIAS ? R2 + 1 : 0;
  const float sl2 = a.scale * kLog2E;
  const long long rows = (long long)a.B * a.H * a.Lq;
  int pos_k[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) pos_k[s] = BIAS ? token_pos(k_first + s * 16 + l15, a.W) : 0;

  Stage<T, D> sq[M];
  Stage<T, DV> sg;
  float2 stat = make_float2(0.f, 0.f);  // waves 0 .. M - 1: maximum and 1 / sum of a query, waves M .. 2 M - 1: its delta
  auto fetch = [&](int b, int step) {
    const int h = kvh * group + step / qtiles, t0 = (step % qtiles) * kTile;
    const unsigned long long word = range_word(t0, a.Lq);
#pragma unroll
    for (int m = 0; m < M; ++m)
      sq[m].load(reinterpret_cast<const typename O::Mem*>(a.q) + b * a.qs[0] + (long long)(h * M + m) * a.qs[2], a.qs[1], t0, word, a.D, tid);
    sg.load(reinterpret_cast<const typename O::Mem*>(a.dout) + b * a.gs[0] + h * a.gs[2], a.gs[1], t0, word, a.DV, tid);
    const int which = tid >> 6, i = t0 + (tid & 63);
    const long long row = ((long long)b * a.H + h) * a.Lq + i;
    if (which < M) {
      stat = make_float2(INFINITY, 0.f);
      if (i < a.Lq) stat = *reinterpret_cast<const float2*>(a.stat + 2 * (which * rows + row));
    } else if (which < 2 * M) {
      stat.x = i < a.Lq ? a.delta[(which - M) * rows + row] : 0.f;
    }
  };
  if (s_first < s_last) fetch(b_first, s_first);
  int bias_head = -1;
  float4v bias_reg[M][KS][NT ? NT * 4 : 1];  // boards (no key range, no shared heads): the bias of this wave's pairs
  if constexpr (NT > 0) {
    fill_bias(a, bias_lds, kvh, M, tid);
    bias_head = kvh;
    if (tid < NT * kTile) pos_lds[tid] = token_pos(tid, a.W);
    __syncthreads();
#pragma unroll
    for (int qt = 0; qt < NT * 4; ++qt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int pos = pos_lds[qt * 16 + q4 * 4 + j];
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
          for (int s = 0; s < KS; ++s) bias_reg[m][s][qt][j] = bias_lds[m * slots + clamp_slot(pos_k[s] - pos + a.R, R2)];
      }
  }

  for (int b = b_first; b < b_last; ++b) {
    const int origin = BIAS ? query_origin(a, b) : 0;
    Frag kf[M][KS][DC], vf[KS][VC];
    bool live[KS];
    bool any = false;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int key = k_first + s * 16 + l15;
      live[s] = key < a.Lk && (!a.words || ((a.words[(size_t)b * tiles + (key >> 6)] >> (key & 63)) & 1));
      any |= live[s];
#pragma unroll
      for (int m = 0; m < M; ++m)
        load_rows<T, DC>(kf[m][s], reinterpret_cast<const typename O::Mem*>(a.k) + b * a.ks[0] + (long long)key * a.ks[1] + (long long)(kvh * M + m) * a.ks[2],
                         live[s], a.D, q4);
      load_rows<T, VC>(vf[s], reinterpret_cast<const typename O::Mem*>(a.v) + b * a.vs[0] + (long long)key * a.vs[1] + kvh * a.vs[2], live[s], a.DV, q4);
    }
    float4v dk[M][KS][ND], dv[KS][NV];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
#pragma unroll
      for (int n = 0; n < NV; ++n) dv[s][n] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int n = 0; n < ND; ++n) dk[m][s][n] = float4v{0.f, 0.f, 0.f, 0.f};
    }
    const bool busy = __ballot(any) != 0;                         // this wave has a key that takes part
    const int last = __syncthreads_or(any) ? s_last : s_first;    // the workgroup has one
    // One staged query tile; qt0 is its first 16-query block where the bias is in registers.
    auto tile = [&](int step, auto qt0_) {
      constexpr int qt0 = decltype(qt0_)::value;
      const int h = kvh * group + step / qtiles, t0 = (step % qtiles) * kTile;
      const float lam = M == 2 ? a.lam[h] : 0.f;
      __syncthreads();
#pragma unroll
      for (int m = 0; m < M; ++m) sq[m].store(q_lds + m * TQ, PQ, tid);
      sg.store(g_lds, PG, tid);
      if (tid < M * kTile) {
        top_lds[tid] = stat.x;
        inv_lds[tid] = stat.y;
        const bool far = __any(Exponent::far(Exponent::base_of(stat.x, sl2)));
        if (lane == 0) far_lds[wave] = far;
      } else if (tid < 2 * M * kTile) {
        delta_lds[tid - M * kTile] = stat.x;
      }
      if (BIAS && NT == 0 && tid < kTile) pos_lds[tid] = token_pos(t0 + tid, a.W) + origin;
      if (BIAS && h != bias_head) {
        fill_bias(a, bias_lds, h, M, tid);
        bias_head = h;
      }
      __syncthreads();
      if (step + 1 < last) fetch(b, step + 1);
      else if (b + 1 < b_last) fetch(b + 1, s_first);
      if (!busy) return;
      const bool far = far_lds[0] | (M == 2 ? far_lds[1] : 0);
      int side[KS];
#pragma unroll
      for (int s = 0; s < KS; ++s)
        side[s] = BIAS && NT == 0 ? clamped_side(a, k_first + s * 16, k_first + s * 16 + 15, t0 + origin, t0 + kTile - 1 + origin) : 0;
      auto block = [&](auto kb_, int kb) {
        constexpr int kbc = decltype(kb_)::value;  // the block where it has to be a constant (registers), 0 otherwise
        float4v pmix[KS][O::kSub], ds[M][KS][O::kSub];
#pragma unroll
        for (int u = 0; u < O::kSub; ++u) {
          const int qt = kb * O::kSub + u;
          float4v dp[KS];
#pragma unroll
          for (int s = 0; s < KS; ++s) dp[s] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < VC; ++c) {
            const Frag gf = O::row_frag(g_lds, PG, qt * 16 + l15, c, q4);
#pragma unroll
            for (int s = 0; s < KS; ++s) dp[s] = O::mma_mirrored(gf, vf[s][c], dp[s]);
          }
          int4 p4 = make_int4(0, 0, 0, 0);
          if constexpr (BIAS && NT == 0) p4 = *reinterpret_cast<const int4*>(pos_lds + qt * 16 + q4 * 4);
          const int pj[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
          for (int m = 0; m < M; ++m) {
            float4v x[KS];
#pragma unroll
            for (int s = 0; s < KS; ++s) {
              if constexpr (NT > 0) {
                x[s] = bias_reg[m][s][qt0 + kbc * O::kSub + u];
              } else if constexpr (BIAS) {
                const float* bias = bias_lds + m * slots;
                if (side[s] != 0) {
                  const float c = bias[side[s] > 0 ? R2 : 0];
                  x[s] = float4v{c, c, c, c};
                } else {
                  const int off = a.R + pos_k[s];
#pragma unroll
                  for (int j = 0; j < 4; ++j) x[s][j] = bias[clamp_slot(off - pj[j], R2)];
                }
              } else {
                x[s] = float4v{0.f, 0.f, 0.f, 0.f};
              }
            }
#pragma unroll
            for (int c = 0; c < DC; ++c) {
              const Frag qf = O::row_frag(q_lds + m * TQ, PQ, qt * 16 + l15, c, q4);
#pragma unroll
              for (int s = 0; s < KS; ++s) x[s] = O::mma(qf, kf[m][s][c], x[s]);
            }
            const float4v top4 = *reinterpret_cast<const float4v*>(top_lds + m * kTile + qt * 16 + q4 * 4);
            const float4v inv4 = *reinterpret_cast<const float4v*>(inv_lds + m * kTile + qt * 16 + q4 * 4);
            const float4v del4 = *reinterpret_cast<const float4v*>(delta_lds + m * kTile + qt * 16 + q4 * 4);
            const float4v base4 = {Exponent::base_of(top4[0], sl2), Exponent::base_of(top4[1], sl2), Exponent::base_of(top4[2], sl2), Exponent::base_of(top4[3], sl2)};
#pragma unroll
            for (int s = 0; s < KS; ++s) {
              // a masked key's column is garbage of its own (its rows were read as zeros) and is zeroed when written
              if (far) {
#pragma unroll
                for (int j = 0; j < 4; ++j) x[s][j] = Exponent::far_(x[s][j], top4[j], sl2);
              } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) x[s][j] = Exponent::near_(x[s][j], base4[j], sl2);
              }
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float p = x[s][j] * inv4[j];
                if (m == 0) {
                  pmix[s][u][j] = p;
                  ds[m][s][u][j] = p * (dp[s][j] - del4[j]);
                } else {
                  const float w = -lam * p;
                  pmix[s][u][j] += w;
                  ds[m][s][u][j] = w * (dp[s][j] - del4[j]);
                }
              }
            }
          }
        }
        Frag pf[KS][PL];
#pragma unroll
        for (int s = 0; s < KS; ++s) acc_parts<T>(pf[s], pmix[s]);
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          const Frag gf = O::tr_frag(g_lds, PG, kb, n, l15, q4);
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            if constexpr (TILE_SUMS) dv[s][n] += mma_parts<T>(gf, pf[s], float4v{0.f, 0.f, 0.f, 0.f});
            else dv[s][n] = mma_parts<T>(gf, pf[s], dv[s][n]);
          }
        }
#pragma unroll
        for (int m = 0; m < M; ++m) {
          Frag sf[KS][PL];
#pragma unroll
          for (int s = 0; s < KS; ++s) acc_parts<T>(sf[s], ds[m][s]);
#pragma unroll
          for (int n = 0; n < ND; ++n) {
            const Frag qf = O::tr_frag(q_lds + m * TQ, PQ, kb, n, l15, q4);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
              if constexpr (TILE_SUMS) dk[m][s][n] += mma_parts<T>(qf, sf[s], float4v{0.f, 0.f, 0.f, 0.f});
              else dk[m][s][n] = mma_parts<T>(qf, sf[s], dk[m][s][n]);
            }
          }
        }
      };
      if constexpr (NT > 0) {
        block(std::integral_constant<int, 0>{}, 0);
        block(std::integral_constant<int, 1>{}, 1);
        if constexpr (NKB == 4) {
          block(std::integral_constant<int, 2>{}, 2);
          block(std::integral_constant<int, 3>{}, 3);
        }
      } else {
#pragma unroll 1
        for (int kb = 0; kb < NKB; ++kb) block(std::integral_constant<int, 0>{}, kb);
      }
    };
    if constexpr (NT == 0) {
      for (int step = s_first; step < last; ++step) tile(step, std::integral_constant<int, 0>{});
    } else if (last > s_first) {
      tile(0, std::integral_constant<int, 0>{});
      tile(1, std::integral_constant<int, 4>{});
      if constexpr (NT == 4) {
        tile(2, std::integral_constant<int, 8>{});
        if (last > 3) tile(3, std::integral_constant<int, 12>{});
      }
    }
    if (last == s_first && b + 1 < b_last && s_first < s_last) fetch(b + 1, s_first);  // nothing took part: the tile under way was this sample's
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int key = k_first + s * 16 + l15;
      if (key >= a.Lk) continue;
      const long long krow = ((long long)b * a.KV + kvh) * a.Lk + key;
      float* part = a.kv_part + (split * ((long long)a.B * a.KV * a.Lk) + krow) * (M * a.D + a.DV);
      typename O::Mem* dv_row = reinterpret_cast<typename O::Mem*>(a.dv) + b * a.dvs[0] + (long long)key * a.dvs[1] + kvh * a.dvs[2];
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const int dim = n * 16 + q4 * 4;
        if (dim >= a.DV) continue;
        const float4v g = live[s] ? dv[s][n] : float4v{0.f, 0.f, 0.f, 0.f};
        if (a.k_splits > 1) Ops<float>::store4(part + M * a.D + dim, g[0], g[1], g[2], g[3]);
        else O::store4(dv_row + dim, g[0], g[1], g[2], g[3]);
      }
#pragma unroll
      for (int m = 0; m < M; ++m) {
        typename O::Mem* dk_row = reinterpret_cast<typename O::Mem*>(a.dk) + b * a.dks[0] + (long long)key * a.dks[1] + (long long)(kvh * M + m) * a.dks[2];
#pragma unroll
        for (int n = 0; n < ND; ++n) {
          const int dim = n * 16 + q4 * 4;
          if (dim >= a.D) continue;
          const float4v g = live[s] ? dk[m][s][n] * a.scale : float4v{0.f, 0.f, 0.f, 0.f};
          if (a.k_splits > 1) Ops<float>::store4(part + m * a.D + dim, g[0], g[1], g[2], g[3]);
          else O::store4(dk_row + dim, g[0], g[1], g[2], g[3]);
        }
      }
    }
  }
}

// dest (heads of `width` values) = sum over the splits of rows [S][B, G, L][pitch] from column `from`, in order: four values per thread.
template <typename T>
__global__ __launch_bounds__(256) void enc_grad_join_kernel(const float* part, int splits, int B, int G, int L, int pitch, int from, int maps, int width,
                                                            T* dest, long long sb, long long st, long long sh) {
  const int quads = maps * width / 4;
  const long long rows = (long long)B * G * L, i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * quads) return;
  const long long row = i / quads;
  const int col = (int)(i - row * quads) * 4, m = col / width;
  float4v s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int p = 0; p < splits; ++p) s += *reinterpret_cast<const float4v*>(part + (p * rows + row) * pitch + from + col);
  const int token = (int)(row % L);
  const long long bg = row / L;
  const int b = (int)(bg / G), g = (int)(bg - (long long)b * G);
  Ops<T>::store4(dest + b * sb + token * st + ((long long)g * maps + m) * sh + (col - m * width), s[0], s[1], s[2], s[3]);
}

// The small gradients, in a fixed order and (beyond one workgroup's share) 64 bits: the terms of these sums cancel.
struct SmallGrads {
  const float* sums;   // [outer, H, per_head, M, slots] sums of dS by position difference
  const int* order;    // differences by bucket
  const int* start;
  float* dtable;       // [buckets, H M]
  const float* delta2; // [outer, H, per_head, 4] sums of delta_2 by wave
  float* dlam;         // [H]
  int outer, H, per_head, M, slots, buckets, table_groups;
};

// mid[z][h][m][slot] = sum over a share of head h's rows: the first of two steps where there are many sums (SmallGrads then has
// outer = shares and per_head = 1).
__global__ __launch_bounds__(256) void enc_hist_sum_kernel(const float* hist, float* mid, int outer, int H, int per_head, int M, int slots, int shares) {
  __shared__ float part[4][64];
  const int slot = blockIdx.x * 64 + (threadIdx.x & 63), wave = threadIdx.x >> 6;
  const int hm = blockIdx.y, h = hm / M, m = hm - h * M, z = blockIdx.z;
  const int total = outer * per_head, per = (total + shares - 1) / shares;
  const int first = z * per, last = first + per < total ? first + per : total;
  float s = 0.f;
  if (slot < slots) {
#pragma unroll 4
    for (int r = first + wave; r < last; r += 4) {
      const int o = r / per_head, i = r - o * per_head;
      s += hist[(((size_t)o * H + h) * per_head + i) * M * slots + (size_t)m * slots + slot];
    }
  }
  part[wave][threadIdx.x & 63] = s;
  __syncthreads();
  if (wave == 0 && slot < slots) {
    const int l = threadIdx.x;
    mid[((size_t)z * H * M + hm) * slots + slot] = (part[0][l] + part[1][l]) + (part[2][l] + part[3][l]);
  }
}

__device__ __forceinline__ double wave_sum_d(double s) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) s += __shfl_xor(s, off, 64);
  return s;
}

// One wave per (bucket, head and map) adds the bucket's differences over all rows; the workgroups behind them, one per head, lam's
// gradient -sum delta_2.
__global__ __launch_bounds__(256) void enc_small_grads_kernel(SmallGrads a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if ((int)blockIdx.x < a.table_groups) {
    const int hm = a.H * a.M, w = blockIdx.x * 4 + wave;
    if (w >= a.buckets * hm) return;
    const int bucket = w / hm, col = w - bucket * hm, h = col / a.M, m = col - h * a.M;
    const int first = a.start[bucket], n = a.start[bucket + 1] - first, rows = a.outer * a.per_head;
    double s = 0.0;
#pragma unroll 4
    for (int i = lane; i < n * rows; i += 64) {
      const int r = i / n, e = i - r * n, o = r / a.per_head;
      s += (double)a.sums[((((size_t)o * a.H + h) * a.per_head + (r - o * a.per_head)) * a.M + m) * a.slots + a.order[first + e]];
    }
    s = wave_sum_d(s);
    if (lane == 0) a.dtable[(size_t)bucket * hm + col] = (float)s;
    return;
  }
  __shared__ double part[4];
  const int h = blockIdx.x - a.table_groups, n = a.per_head * 4;
  double s = 0.0;
#pragma unroll 4
  for (int i = threadIdx.x; i < a.outer * n; i += 256) {
    const int o = i / n;
    s += (double)a.delta2[((size_t)o * a.H + h) * n + (i - o * n)];
  }
  s = wave_sum_d(s);
  if (lane == 0) part[wave] = s;
  __syncthreads();
  if (threadIdx.x == 0) a.dlam[h] = (float)-((part[0] + part[1]) + (part[2] + part[3]));
}

template <typename T, int D, int M, bool BIAS, int NT>
int launch_bwd_k(const EncAttnArgs& a, hipStream_t stream) {
  constexpr int KS = enc_columns_of(D, M, NT, Ops<T>::kBf16, kEncKeys);
  static_assert(enc_tiles_agree<T, D, M, kEncKeys>());
  const int lds = enc_lds_bytes(enc_form<T>(), D, M, NT, kEncKeys, BIAS ? 2 * a.R + 1 : 0, 0);
  const int rc = enc_lds(enc_attn_bwd_k_kernel<T, D, M, KS, BIAS, NT>, lds);
  if (rc) return rc;
  const int nkt = (a.Lk + 64 * KS - 1) / (64 * KS);
  hipLaunchKernelGGL((enc_attn_bwd_k_kernel<T, D, M, KS, BIAS, NT>), dim3((unsigned)((a.B + a.k_chunk - 1) / a.k_chunk * a.KV * nkt * a.k_splits)), dim3(256),
                     lds, stream, a);
  return hip_err(hipGetLastError());
}

// TQ: rows of the query-owned pass
template <typename TQ, typename T, int D, int M, bool BIAS, int NT = 0>
int launch_bwd(EncAttnArgs a, hipStream_t stream) {
  constexpr int QS = enc_columns_of(D, M, NT, Ops<TQ>::kBf16, kEncQueries);
  static_assert(enc_tiles_agree<TQ, D, M, kEncQueries>());
  const int slots = BIAS ? 2 * a.R + 1 : 0;
  a.hist_rows = enc_hist_rows(enc_form<TQ>(), D, M, NT, slots, enc_waves(D, M, NT, QS, Ops<TQ>::kBf16, kEncQueries));
  const int lds = enc_lds_bytes(enc_form<TQ>(), D, M, NT, kEncQueries, slots, BIAS && a.hist ? a.hist_rows : 0);
  int rc = enc_lds(enc_attn_bwd_q_kernel<TQ, D, M, QS, BIAS, NT>, lds);
  if (rc) return rc;
  const int nqt = (a.Lq + 64 * QS - 1) / (64 * QS);
  const long long groups = (long long)((a.B + a.q_chunk - 1) / a.q_chunk) * a.H * nqt * a.q_splits;
  if (groups != a.q_groups) return -21;  // a host side built with other rules
  hipLaunchKernelGGL((enc_attn_bwd_q_kernel<TQ, D, M, QS, BIAS, NT>), dim3((unsigned)groups), dim3(256), lds, stream, a);
  rc = hip_err(hipGetLastError());
  if (rc) return rc;
  if (!a.dk) return 0;
  // the key-owned pass of a board unrolls where no heads are shared
  return NT > 0 && a.KV == a.H ? launch_bwd_k<T, D, M, BIAS, NT>(a, stream) : launch_bwd_k<T, D, M, BIAS, 0>(a, stream);
}

template <typename T>
int join_grad(const EncAttnArgs& a, const float* part, int splits, int G, int L, int pitch, int from, int maps, int width, void* dest, const long long* st,
              hipStream_t stream) {
  const long long n = (long long)a.B * G * L * (maps * width / 4);
  if ((n + 255) / 256 >= (1LL << 31)) return -15;
  hipLaunchKernelGGL((enc_grad_join_kernel<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, part, splits, a.B, G, L, pitch, from, maps, width,
                     reinterpret_cast<T*>(dest), st[0], st[1], st[2]);
  return hip_err(hipGetLastError());
}

template <typename T>
int join_grads(const EncAttnArgs& a, hipStream_t stream) {
  if (a.q_splits > 1) {
    const int rc = join_grad<T>(a, a.dq_part, a.q_splits, a.H, a.Lq, a.M * a.D, 0, a.M, a.D, a.dq, a.dqs, stream);
    if (rc) return rc;
  }
  if (a.dk && a.k_splits > 1) {
    const int pitch = a.M * a.D + a.DV;
    const int rc = join_grad<T>(a, a.kv_part, a.k_splits, a.KV, a.Lk, pitch, 0, a.M, a.D, a.dk, a.dks, stream);
    if (rc) return rc;
    return join_grad<T>(a, a.kv_part, a.k_splits, a.KV, a.Lk, pitch, a.M * a.D, 1, a.DV, a.dv, a.dvs, stream);
  }
  return 0;
}

// T: bf16 rows, or Split; W: fp32 rows with the fp32 matrix instruction where three parts of the query-owned pass's tiles leave no
// room for the table.  Parts otherwise: two 2000-token sequences of four two-map 64-wide heads, forward and backward,
// 812 us and 3.1e-7 off, 1396 us and 7e-7 with the instruction; 16 boards of 400 cells 323 and 487 us; 256 boards of
// 120 cells, two 32-wide maps, 178 and 182 us, dq 2.4e-7 and 3.8e-7 off.
template <typename T, typename W>
int dispatch_bwd(const EncAttnArgs& a, hipStream_t stream) {
  const int w = enc_width(a.D), nt = enc_board_tiles(a.table ? a.W : 0, a.Lk, a.D, a.M);
  if (nt > 0 && (a.q_splits > 1 || (a.KV == a.H && a.k_splits > 1))) return -18;
  if (a.M == 1) {
    if (nt == 2) return launch_bwd<T, T, 32, 1, true, 2>(a, stream);
    if (nt == 4) return launch_bwd<T, T, 32, 1, true, 4>(a, stream);
    if (w == 32) return launch_bwd<T, T, 32, 1, true>(a, stream);
    if (w == 64) return launch_bwd<T, T, 64, 1, true>(a, stream);
    return launch_bwd<T, T, 128, 1, true>(a, stream);
  }
  if (nt == 2) return launch_bwd<T, T, 32, 2, true, 2>(a, stream);
  if (w == 32) return a.table ? launch_bwd<T, T, 32, 2, true>(a, stream) : launch_bwd<T, T, 32, 2, false>(a, stream);
  if (!a.table) return launch_bwd<T, T, 64, 2, false>(a, stream);
  // whether sums are wanted or not: the same results
  return enc_query_form(a.bf16 != 0, 64, 2, 2 * a.R + 1) == kRowsFp32 ? launch_bwd<W, T, 64, 2, true>(a, stream) : launch_bwd<T, T, 64, 2, true>(a, stream);
}

}  // namespace

extern "C" {

// dq, dk and dv (every element written; both null: not wanted), delta and, where hist / dlam are set, the gradients of the table and of lam.
int atri_enc_attn_bwd(const EncAttnArgs* args, hipStream_t stream) {
  if (!args) return -1;
  const EncAttnArgs& a = *args;
  int rc = enc_check(a);
  if (rc) return rc;
  if (!a.q || !a.k || !a.v || !a.dout || !a.dq || !a.dk != !a.dv || !a.stat || !a.o32 || !a.delta) return -17;
  const int slots = 2 * a.R + 1, hm = a.H * a.M;
  if (a.hist) {
    if (!a.table || !a.mid || !a.order || !a.start || !a.dtable) return -17;
    if (a.buckets < 1 || a.shares < 1 || a.shares > 65535 || hm > 65535 || (long long)a.buckets * hm >= (1LL << 31) ||
        (long long)slots * a.shares >= (1LL << 31))
      return -15;
  }
  if (a.dlam && (a.M != 2 || !a.dlam_part)) return -14;
  if ((a.q_splits > 1 && !a.dq_part) || (a.dk && a.k_splits > 1 && !a.kv_part)) return -17;
  rc = a.bf16 ? dispatch_bwd<unsigned short, unsigned short>(a, stream) : dispatch_bwd<Split, float>(a, stream);
  if (rc) return rc;
  rc = a.bf16 ? join_grads<unsigned short>(a, stream) : join_grads<float>(a, stream);
  if (rc) return rc;
  if (!a.hist && !a.dlam) return 0;
  const int per = 64 * enc_columns(a.table ? a.W : 0, a.Lq, a.Lk, a.D, a.M, a.bf16 != 0, kEncQueries), nqt = (a.Lq + per - 1) / per;
  SmallGrads g{a.hist, a.order, a.start, a.dtable, a.dlam_part, a.dlam, (a.B + a.q_chunk - 1) / a.q_chunk, a.H, nqt * a.q_splits, a.M, slots, a.buckets, 0};
  if (a.hist) {
    g.table_groups = (a.buckets * hm + 3) / 4;
    // in one step while the sums are few enough to be read slot by slot from L2; each step is a launch of 4.5 us
    if ((long long)g.outer * g.per_head * hm * slots > (1 << 20)) {
      hipLaunchKernelGGL(enc_hist_sum_kernel, dim3((slots + 63) / 64, hm, a.shares), dim3(256), 0, stream, a.hist, a.mid, g.outer, a.H, g.per_head, a.M, slots,
                         a.shares);
      rc = hip_err(hipGetLastError());
      if (rc) return rc;
      SmallGrads t = g;
      t.sums = a.mid;
      t.outer = a.shares;
      t.per_head = 1;
      hipLaunchKernelGGL(enc_small_grads_kernel, dim3(g.table_groups), dim3(256), 0, stream, t);
      rc = hip_err(hipGetLastError());
      if (rc || !a.dlam) return rc;
      g.table_groups = 0;
    }
  }
  const int groups = g.table_groups + (a.dlam ? a.H : 0);
  hipLaunchKernelGGL(enc_small_grads_kernel, dim3(groups), dim3(256), 0, stream, g);
  return hip_err(hipGetLastError());
}

}  // extern "C"
