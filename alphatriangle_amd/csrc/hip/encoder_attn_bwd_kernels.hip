// Backward pass of the encoder attention operators (encoder_attn.hpp has the operand layout).  Two passes over the score
// matrix, each recomputing it from Q, K and the forward's row maximum and sum (kept apart:
// their joint logarithm would lose the sum beside a large maximum), so that every gradient is summed by one owner in a
// fixed order (a single pass would add dQ with floating-point atomics):
//   query-owned:  dS = P (dP - delta), dP = dO V^T;  dQ = scale dS K;  delta = dO . o per map;  sums of dS by position
//                 difference (the bias table's gradient before it is folded into buckets)
//   key-owned:    dV = (P_1 - lam P_2)^T dO;  dK_m = scale dS_m^T Q_m
// With two maps dP_1 = dO V^T and dP_2 = -lam dP_1, so one product serves both; d lam = -sum delta_2.
#include "encoder_attn.hpp"

using namespace atrihip;

namespace {

constexpr int kDsPitch = kTile + 4;  // row pitch of a wave's 16 x 64 tile of dS on its way to the diagonal sums

__device__ __forceinline__ void wave_lds_fence() {  // orders a wave's own LDS writes before its other lanes' reads
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Adds a wave's 16 x 64 tile of dS (LDS, row = query) to the sums by position difference.  Lane l reads the element of every
// row on its wrapped diagonal: key (l - 15 + row) mod 64, conflict free and each element once.  Pairs on different
// diagonals never have the same (unclamped) difference, on a board either, so every slot of `sums` has one writer per
// step and the order of the additions is fixed.  Clamped differences go to the lane's own lo / hi.
__device__ __forceinline__ void add_diagonals(const EncAttnArgs& a, float* sums, const float* ds, const int* pos_k, int k0, int q0, int origin,
                                              int lane, float& lo, float& hi) {
  const int R2 = 2 * a.R;
  if (a.W == 0) {
    float low_part = 0.f, high_part = 0.f;  // rows below the wrap (diagonal lane - 15), rows above it (diagonal lane + 49)
#pragma unroll
    for (int row = 0; row < 16; ++row) {
      const float v = ds[row * kDsPitch + ((lane - 15 + row) & 63)];
      if (row >= 15 - lane) low_part += v; else high_part += v;
    }
    const int slot = k0 - q0 - origin + a.R + lane - 15;
    if (slot <= 0) lo += low_part; else if (slot >= R2) hi += low_part; else sums[slot] += low_part;
    if (lane < 15) {
      const int s2 = slot + 64;
      if (s2 <= 0) lo += high_part; else if (s2 >= R2) hi += high_part; else sums[s2] += high_part;
    }
    wave_lds_fence();
    return;
  }
  float run = 0.f;
  int slot = -1;
#pragma unroll
  for (int row = 0; row < 16; ++row) {
    const int key = (lane - 15 + row) & 63;
    const float v = ds[row * kDsPitch + key];
    const bool valid = k0 + key < a.Lk && q0 + row < a.Lq;
    const int s = valid ? clamp_slot(pos_k[key] - token_pos(q0 + row, a.W) + a.R, R2) : slot;
    if (s != slot && slot >= 0) {
      sums[slot] += run;
      run = 0.f;
    }
    slot = s;
    run += valid ? v : 0.f;
  }
  if (slot >= 0) sums[slot] += run;
  wave_lds_fence();
}

// One 4-wave workgroup per (sample, head, 64 QS queries).
template <typename T, int D, int M, int QS, bool BIAS>
__global__ __launch_bounds__(256) void enc_attn_bwd_q_kernel(EncAttnArgs a) {
  using O = Ops<T>;
  using Frag = typename O::Frag;
  constexpr int DV = D * M, DC = D / O::kDims, VC = DV / O::kDims, ND = D / 16, NKB = 4 / O::kSub;
  constexpr int PK = O::row_pitch(D), PV = O::row_pitch(DV);
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  T* k_lds = reinterpret_cast<T*>(smem);
  T* v_lds = k_lds + M * kTile * PK;
  int* pos_lds = reinterpret_cast<int*>(v_lds + kTile * PV);
  float* bias_lds = reinterpret_cast<float*>(pos_lds + kTile);
  const int slots = BIAS ? 2 * a.R + 1 : 0, R2 = 2 * a.R;
  float* ds_lds = bias_lds + ((M * slots + 3) & ~3);
  float* sum_lds = ds_lds + 4 * 16 * kDsPitch;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l15 = lane & 15, q4 = lane >> 4;
  const int nqt = (a.Lq + 64 * QS - 1) / (64 * QS);
  const int id = xcd_order(blockIdx.x, gridDim.x);
  const int qt = id % nqt, bh = id / nqt;
  const int b = bh / a.H, h = bh - b * a.H, kvh = h / (a.H / a.KV);
  const int tiles = (a.Lk + kTile - 1) / kTile;
  const T* kb_ = reinterpret_cast<const T*>(a.k) + b * a.ks[0] + (long long)kvh * M * a.ks[2];
  const T* vb_ = reinterpret_cast<const T*>(a.v) + b * a.vs[0] + kvh * a.vs[2];
  const bool want_sums = BIAS && a.hist != nullptr;
  if constexpr (BIAS) fill_bias(a, bias_lds, h, M, tid);
  if (want_sums)
    for (int i = tid; i < a.hist_rows * M * slots; i += 256) sum_lds[i] = 0.f;
  float* my_sums = sum_lds + (a.hist_rows == 4 ? wave * M * slots : 0);

  const long long rows = (long long)a.B * a.H * a.Lq;
  const int q_first = (qt * 4 + wave) * 16 * QS;
  const bool busy = q_first < a.Lq;
  const int origin = BIAS ? query_origin(a, b) : 0;
  const float lam = M == 2 ? a.lam[h] : 0.f;
  Frag qf[M][QS][DC], dof[QS][VC];
  float top[M][QS], inv[M][QS], delta[M][QS];
  int pos_q[QS];
#pragma unroll
  for (int s = 0; s < QS; ++s) {
    const int query = q_first + s * 16 + l15;
    const bool valid = query < a.Lq;
    pos_q[s] = BIAS ? token_pos(query, a.W) + origin : 0;
    load_rows<T, VC>(dof[s], reinterpret_cast<const T*>(a.dout) + b * a.gs[0] + (long long)query * a.gs[1] + h * a.gs[2], valid, a.DV, q4);
#pragma unroll
    for (int m = 0; m < M; ++m) {
      load_rows<T, DC>(qf[m][s], reinterpret_cast<const T*>(a.q) + b * a.qs[0] + (long long)query * a.qs[1] + (long long)(h * M + m) * a.qs[2], valid,
                       a.D, q4);
      float2 st = make_float2(INFINITY, 0.f);
      if (valid) st = *reinterpret_cast<const float2*>(a.stat + 2 * (m * rows + (long long)bh * a.Lq + query));
      top[m][s] = st.x;
      inv[m][s] = st.y;
      const float* o = a.o32 + b * a.o32s[0] + (long long)query * a.o32s[1] + h * a.o32s[2] + m * a.o32s[3];
      float dot = 0.f;
#pragma unroll
      for (int c = 0; c < VC; ++c) {
        const int col = c * O::kDims + q4 * O::kVec;
        if (!valid || col >= a.DV) continue;
        float v[O::kVec];
#pragma unroll
        for (int e = 0; e < O::kVec; e += 4) {
          const float4 u = *reinterpret_cast<const float4*>(o + col + e);
          v[e] = u.x; v[e + 1] = u.y; v[e + 2] = u.z; v[e + 3] = u.w;
        }
        dot += O::dot(dof[s][c], v);
      }
      delta[m][s] = quad_row_sum(dot);
      if (valid && q4 == 0) a.delta[m * rows + (long long)bh * a.Lq + query] = delta[m][s];
    }
  }
  float4v dq[M][QS][ND];
  float lo[M], hi[M];
#pragma unroll
  for (int m = 0; m < M; ++m) {
    lo[m] = hi[m] = 0.f;
#pragma unroll
    for (int s = 0; s < QS; ++s)
#pragma unroll
      for (int n = 0; n < ND; ++n) dq[m][s][n] = float4v{0.f, 0.f, 0.f, 0.f};
  }
  const float sl2 = a.scale * kLog2E;

  Stage<T, D> sk[M];
  Stage<T, DV> sv;
  TileWalk walk;
  walk.start(a.words ? a.words + (size_t)b * tiles : nullptr, a.Lk, 0, tiles);
  int t = walk.next();
  if (t < tiles) {
#pragma unroll
    for (int m = 0; m < M; ++m) sk[m].load(kb_ + m * a.ks[2], a.ks[1], t * kTile, walk.word, a.D, tid);
    sv.load(vb_, a.vs[1], t * kTile, walk.word, a.DV, tid);
  }
  while (t < tiles) {
    const unsigned long long word = walk.word;
    const int t0 = t * kTile;
    __syncthreads();
#pragma unroll
    for (int m = 0; m < M; ++m) sk[m].store(k_lds + m * kTile * PK, PK, tid);
    sv.store(v_lds, PV, tid);
    if (BIAS && tid < kTile) pos_lds[tid] = token_pos(t0 + tid, a.W);
    __syncthreads();
    t = walk.next();
    if (t < tiles) {
#pragma unroll
      for (int m = 0; m < M; ++m) sk[m].load(kb_ + m * a.ks[2], a.ks[1], t * kTile, walk.word, a.D, tid);
      sv.load(vb_, a.vs[1], t * kTile, walk.word, a.DV, tid);
    }
    float4v ds[M][QS][4];
    int side[QS];
    if (busy) {
#pragma unroll
      for (int s = 0; s < QS; ++s) {
        const int qa = q_first + s * 16 + origin;
        side[s] = BIAS ? clamped_side(a, t0, t0 + kTile - 1, qa, qa + 15) : 0;
      }
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) {
        float4v dp[QS][O::kSub];
#pragma unroll
        for (int u = 0; u < O::kSub; ++u) {
          const int kt = kb * O::kSub + u;
#pragma unroll
          for (int s = 0; s < QS; ++s) dp[s][u] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < VC; ++c) {
            const Frag vf = O::row_frag(v_lds, PV, kt * 16 + l15, c, q4);
#pragma unroll
            for (int s = 0; s < QS; ++s) dp[s][u] = O::mma(vf, dof[s][c], dp[s][u]);
          }
#pragma unroll
          for (int m = 0; m < M; ++m) {
            float4v x[QS];
#pragma unroll
            for (int s = 0; s < QS; ++s) x[s] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < DC; ++c) {
              const Frag kf = O::row_frag(k_lds + m * kTile * PK, PK, kt * 16 + l15, c, q4);
#pragma unroll
              for (int s = 0; s < QS; ++s) x[s] = O::mma(kf, qf[m][s][c], x[s]);
            }
            const unsigned bits = (unsigned)(word >> (kt * 16 + q4 * 4));
            int4 p4 = make_int4(0, 0, 0, 0);
            if constexpr (BIAS) p4 = *reinterpret_cast<const int4*>(pos_lds + kt * 16 + q4 * 4);
            const int pj[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
            for (int s = 0; s < QS; ++s) {
              float add[4] = {0.f, 0.f, 0.f, 0.f};
              if constexpr (BIAS) {
                const float* bias = bias_lds + m * slots;
                if (side[s] != 0) {
                  const float c = bias[side[s] > 0 ? R2 : 0];
#pragma unroll
                  for (int j = 0; j < 4; ++j) add[j] = c;
                } else {
                  const int off = a.R - pos_q[s];
#pragma unroll
                  for (int j = 0; j < 4; ++j) add[j] = bias[clamp_slot(pj[j] + off, R2)];
                }
              }
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                float p = __builtin_amdgcn_exp2f(fmaf(x[s][j], sl2, add[j]) - top[m][s]) * inv[m][s];
                p = (bits >> j) & 1 ? p : 0.f;
                const float g = p * (dp[s][u][j] - delta[m][s]);
                ds[m][s][kt][j] = m == 0 ? g : -lam * g;
              }
            }
          }
        }
#pragma unroll
        for (int m = 0; m < M; ++m) {
          Frag sf[QS];
#pragma unroll
          for (int s = 0; s < QS; ++s) sf[s] = O::acc_frag(&ds[m][s][kb * O::kSub]);
#pragma unroll
          for (int n = 0; n < ND; ++n) {
            const Frag kf = O::tr_frag(k_lds + m * kTile * PK, PK, kb, n, l15, q4);
#pragma unroll
            for (int s = 0; s < QS; ++s) dq[m][s][n] = O::mma(kf, sf[s], dq[m][s][n]);
          }
        }
      }
    }
    if constexpr (BIAS) {
      if (want_sums) {
        for (int turn = 0; turn < (a.hist_rows == 4 ? 1 : 4); ++turn) {  // one row of sums for all waves: they take turns
          if (busy && (a.hist_rows == 4 || turn == wave)) {
            float* tile = ds_lds + wave * 16 * kDsPitch;
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
              for (int s = 0; s < QS; ++s) {
                if (side[s] != 0) {
                  float all = 0.f;
#pragma unroll
                  for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                    for (int j = 0; j < 4; ++j) all += ds[m][s][kt][j];
                  if (side[s] > 0) hi[m] += all; else lo[m] += all;
                } else {
#pragma unroll
                  for (int kt = 0; kt < 4; ++kt)
                    *reinterpret_cast<float4v*>(tile + l15 * kDsPitch + kt * 16 + q4 * 4) = ds[m][s][kt];
                  wave_lds_fence();
                  add_diagonals(a, my_sums + m * slots, tile, pos_lds, t0, q_first + s * 16, origin, lane, lo[m], hi[m]);
                }
              }
          }
          if (a.hist_rows != 4) __syncthreads();
        }
      }
    }
  }

  if (busy) {
#pragma unroll
    for (int s = 0; s < QS; ++s) {
      const int query = q_first + s * 16 + l15;
      if (query >= a.Lq) continue;
#pragma unroll
      for (int m = 0; m < M; ++m) {
        T* row = reinterpret_cast<T*>(a.dq) + b * a.dqs[0] + (long long)query * a.dqs[1] + (long long)(h * M + m) * a.dqs[2];
#pragma unroll
        for (int n = 0; n < ND; ++n) {
          const int dim = n * 16 + q4 * 4;
          if (dim < a.D) O::store4(row + dim, dq[m][s][n][0] * a.scale, dq[m][s][n][1] * a.scale, dq[m][s][n][2] * a.scale, dq[m][s][n][3] * a.scale);
        }
      }
    }
  }
  if (!want_sums) return;
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
  float* part = a.hist + (size_t)(bh * (long long)nqt + qt) * M * slots;
  for (int i = tid; i < M * slots; i += 256) {
    float s = sum_lds[i];
    if (a.hist_rows == 4) s = (s + sum_lds[M * slots + i]) + (sum_lds[2 * M * slots + i] + sum_lds[3 * M * slots + i]);
    part[i] = s;
  }
}

// One 4-wave workgroup per (sample, key / value head, 64 KS keys); a wave owns 16 KS keys and walks the query tiles of every
// query head that shares them.
template <typename T, int D, int M, int KS, bool BIAS>
__global__ __launch_bounds__(256) void enc_attn_bwd_k_kernel(EncAttnArgs a) {
  using O = Ops<T>;
  using Frag = typename O::Frag;
  constexpr int DV = D * M, DC = D / O::kDims, VC = DV / O::kDims, ND = D / 16, NV = DV / 16, NKB = 4 / O::kSub;
  constexpr int PQ = O::row_pitch(D), PG = O::row_pitch(DV);
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  T* q_lds = reinterpret_cast<T*>(smem);
  T* g_lds = q_lds + M * kTile * PQ;
  int* pos_lds = reinterpret_cast<int*>(g_lds + kTile * PG);
  float* top_lds = reinterpret_cast<float*>(pos_lds + kTile);
  float* inv_lds = top_lds + M * kTile;
  float* delta_lds = inv_lds + M * kTile;
  float* bias_lds = delta_lds + M * kTile;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l15 = lane & 15, q4 = lane >> 4;
  const int nkt = (a.Lk + 64 * KS - 1) / (64 * KS);
  const int id = xcd_order(blockIdx.x, gridDim.x);
  const int kt_ = id % nkt, bkv = id / nkt;
  const int b = bkv / a.KV, kvh = bkv - b * a.KV, group = a.H / a.KV;
  const int tiles = (a.Lk + kTile - 1) / kTile, qtiles = (a.Lq + kTile - 1) / kTile;
  const int k_first = (kt_ * 4 + wave) * 16 * KS;
  const int R2 = 2 * a.R, slots = BIAS ? R2 + 1 : 0;

  Frag kf[M][KS][DC], vf[KS][VC];
  bool live[KS];
  int pos_k[KS];
  bool any = false;
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int key = k_first + s * 16 + l15;
    live[s] = key < a.Lk && (!a.words || ((a.words[(size_t)b * tiles + (key >> 6)] >> (key & 63)) & 1));
    any |= live[s];
    pos_k[s] = BIAS ? token_pos(key, a.W) : 0;
#pragma unroll
    for (int m = 0; m < M; ++m)
      load_rows<T, DC>(kf[m][s], reinterpret_cast<const T*>(a.k) + b * a.ks[0] + (long long)key * a.ks[1] + (long long)(kvh * M + m) * a.ks[2], live[s],
                       a.D, q4);
    load_rows<T, VC>(vf[s], reinterpret_cast<const T*>(a.v) + b * a.vs[0] + (long long)key * a.vs[1] + kvh * a.vs[2], live[s], a.DV, q4);
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
  const float sl2 = a.scale * kLog2E;
  const long long rows = (long long)a.B * a.H * a.Lq;
  const bool busy = __ballot(any) != 0;                 // this wave has a key that takes part
  const int steps = __syncthreads_or(any) ? group * qtiles : 0;  // the workgroup has one
  const int origin = BIAS ? query_origin(a, b) : 0;

  Stage<T, D> sq[M];
  Stage<T, DV> sg;
  float2 stat = make_float2(0.f, 0.f);  // waves 0 .. M - 1: maximum and 1 / sum of a query, waves M .. 2 M - 1: its delta
  auto fetch = [&](int step) {
    const int h = kvh * group + step / qtiles, t0 = (step % qtiles) * kTile;
    const unsigned long long word = range_word(t0, a.Lq);
#pragma unroll
    for (int m = 0; m < M; ++m)
      sq[m].load(reinterpret_cast<const T*>(a.q) + b * a.qs[0] + (long long)(h * M + m) * a.qs[2], a.qs[1], t0, word, a.D, tid);
    sg.load(reinterpret_cast<const T*>(a.dout) + b * a.gs[0] + h * a.gs[2], a.gs[1], t0, word, a.DV, tid);
    const int which = tid >> 6, i = t0 + (tid & 63);
    const long long row = ((long long)b * a.H + h) * a.Lq + i;
    if (which < M) {
      stat = make_float2(INFINITY, 0.f);
      if (i < a.Lq) stat = *reinterpret_cast<const float2*>(a.stat + 2 * (which * rows + row));
    } else if (which < 2 * M) {
      stat.x = i < a.Lq ? a.delta[(which - M) * rows + row] : 0.f;
    }
  };
  if (steps) fetch(0);
  for (int step = 0; step < steps; ++step) {
    const int h = kvh * group + step / qtiles, t0 = (step % qtiles) * kTile;
    const float lam = M == 2 ? a.lam[h] : 0.f;
    __syncthreads();
#pragma unroll
    for (int m = 0; m < M; ++m) sq[m].store(q_lds + m * kTile * PQ, PQ, tid);
    sg.store(g_lds, PG, tid);
    if (tid < M * kTile) {
      top_lds[tid] = stat.x;
      inv_lds[tid] = stat.y;
    } else if (tid < 2 * M * kTile) {
      delta_lds[tid - M * kTile] = stat.x;
    }
    if (BIAS && tid < kTile) pos_lds[tid] = token_pos(t0 + tid, a.W) + origin;
    if (BIAS && step % qtiles == 0) fill_bias(a, bias_lds, h, M, tid);
    __syncthreads();
    if (step + 1 < steps) fetch(step + 1);
    if (!busy) continue;
    int side[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) side[s] = BIAS ? clamped_side(a, k_first + s * 16, k_first + s * 16 + 15, t0 + origin, t0 + kTile - 1 + origin) : 0;
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb) {
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
          for (int s = 0; s < KS; ++s) dp[s] = O::mma(gf, vf[s][c], dp[s]);
        }
        int4 p4 = make_int4(0, 0, 0, 0);
        if constexpr (BIAS) p4 = *reinterpret_cast<const int4*>(pos_lds + qt * 16 + q4 * 4);
        const int pj[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
        for (int m = 0; m < M; ++m) {
          float4v x[KS];
#pragma unroll
          for (int s = 0; s < KS; ++s) x[s] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < DC; ++c) {
            const Frag qf = O::row_frag(q_lds + m * kTile * PQ, PQ, qt * 16 + l15, c, q4);
#pragma unroll
            for (int s = 0; s < KS; ++s) x[s] = O::mma(qf, kf[m][s][c], x[s]);
          }
          const float4v top4 = *reinterpret_cast<const float4v*>(top_lds + m * kTile + qt * 16 + q4 * 4);
          const float4v inv4 = *reinterpret_cast<const float4v*>(inv_lds + m * kTile + qt * 16 + q4 * 4);
          const float4v del4 = *reinterpret_cast<const float4v*>(delta_lds + m * kTile + qt * 16 + q4 * 4);
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            float add[4] = {0.f, 0.f, 0.f, 0.f};
            if constexpr (BIAS) {
              const float* bias = bias_lds + m * slots;
              if (side[s] != 0) {
                const float c = bias[side[s] > 0 ? R2 : 0];
#pragma unroll
                for (int j = 0; j < 4; ++j) add[j] = c;
              } else {
                const int off = a.R + pos_k[s];
#pragma unroll
                for (int j = 0; j < 4; ++j) add[j] = bias[clamp_slot(off - pj[j], R2)];
              }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float p = __builtin_amdgcn_exp2f(fmaf(x[s][j], sl2, add[j]) - top4[j]) * inv4[j];
              p = live[s] ? p : 0.f;
              const float g = p * (dp[s][j] - del4[j]);
              if (m == 0) {
                pmix[s][u][j] = p;
                ds[m][s][u][j] = g;
              } else {
                pmix[s][u][j] = fmaf(-lam, p, pmix[s][u][j]);
                ds[m][s][u][j] = -lam * g;
              }
            }
          }
        }
      }
      Frag pf[KS];
#pragma unroll
      for (int s = 0; s < KS; ++s) pf[s] = O::acc_frag(pmix[s]);
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const Frag gf = O::tr_frag(g_lds, PG, kb, n, l15, q4);
#pragma unroll
        for (int s = 0; s < KS; ++s) dv[s][n] = O::mma(gf, pf[s], dv[s][n]);
      }
#pragma unroll
      for (int m = 0; m < M; ++m) {
        Frag sf[KS];
#pragma unroll
        for (int s = 0; s < KS; ++s) sf[s] = O::acc_frag(ds[m][s]);
#pragma unroll
        for (int n = 0; n < ND; ++n) {
          const Frag qf = O::tr_frag(q_lds + m * kTile * PQ, PQ, kb, n, l15, q4);
#pragma unroll
          for (int s = 0; s < KS; ++s) dk[m][s][n] = O::mma(qf, sf[s], dk[m][s][n]);
        }
      }
    }
  }
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int key = k_first + s * 16 + l15;
    if (key >= a.Lk) continue;
    T* dv_row = reinterpret_cast<T*>(a.dv) + b * a.dvs[0] + (long long)key * a.dvs[1] + kvh * a.dvs[2];
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int dim = n * 16 + q4 * 4;
      if (dim < a.DV) O::store4(dv_row + dim, dv[s][n][0], dv[s][n][1], dv[s][n][2], dv[s][n][3]);
    }
#pragma unroll
    for (int m = 0; m < M; ++m) {
      T* dk_row = reinterpret_cast<T*>(a.dk) + b * a.dks[0] + (long long)key * a.dks[1] + (long long)(kvh * M + m) * a.dks[2];
#pragma unroll
      for (int n = 0; n < ND; ++n) {
        const int dim = n * 16 + q4 * 4;
        if (dim < a.D) O::store4(dk_row + dim, dk[m][s][n][0] * a.scale, dk[m][s][n][1] * a.scale, dk[m][s][n][2] * a.scale, dk[m][s][n][3] * a.scale);
      }
    }
  }
}

// mid[z][h M + m][slot] = sum of hist over a share of the (sample, query tile) workgroups of head h: one wave per share row, in order.
__global__ __launch_bounds__(256) void enc_hist_sum_kernel(const float* hist, float* mid, int B, int H, int nqt, int M, int slots, int shares) {
  __shared__ float part[4][64];
  const int slot = blockIdx.x * 64 + (threadIdx.x & 63), wave = threadIdx.x >> 6;
  const int hm = blockIdx.y, h = hm / M, m = hm - h * M, z = blockIdx.z;
  const int total = B * nqt, per = (total + shares - 1) / shares;
  const int first = z * per, last = first + per < total ? first + per : total;
  float s = 0.f;
  if (slot < slots) {
#pragma unroll 4
    for (int r = first + wave; r < last; r += 4) {
      const int b = r / nqt, qt = r - b * nqt;
      s += hist[(((size_t)b * H + h) * nqt + qt) * M * slots + (size_t)m * slots + slot];
    }
  }
  part[wave][threadIdx.x & 63] = s;
  __syncthreads();
  if (wave == 0 && slot < slots) {
    const int l = threadIdx.x;
    mid[((size_t)z * H * M + hm) * slots + slot] = (part[0][l] + part[1][l]) + (part[2][l] + part[3][l]);
  }
}

// dtable[bucket][h M + m]: one wave per (bucket, column) adds the slots of the bucket (order[start[b]] .. order[start[b + 1] - 1]) over
// all shares, in 64 bits (the terms of these sums cancel).
__global__ __launch_bounds__(256) void enc_bucket_sum_kernel(const float* mid, const int* order, const int* start, float* dtable, int buckets, int hm,
                                                             int slots, int shares) {
  const int w = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (w >= buckets * hm) return;
  const int bucket = w / hm, col = w - bucket * hm;
  const int first = start[bucket], n = start[bucket + 1] - first;
  double s = 0.0;
  for (int i = lane; i < n * shares; i += 64) {
    const int z = i / n, e = i - z * n;
    s += (double)mid[((size_t)z * hm + col) * slots + order[first + e]];
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) s += __shfl_xor(s, off, 64);
  if (lane == 0) dtable[(size_t)bucket * hm + col] = (float)s;
}

// dlam[h] = -sum of delta_2 over samples and queries: one workgroup per head, fixed order, 64-bit sums.
__global__ __launch_bounds__(1024) void enc_dlam_kernel(const float* delta2, float* dlam, int B, int H, int Lq) {
  __shared__ double part[16];
  const int h = blockIdx.x, tid = threadIdx.x;
  const long long n = (long long)B * Lq;
  double s = 0.0;
#pragma unroll 4
  for (long long i = tid; i < n; i += 1024) {
    const long long b = i / Lq;
    s += (double)delta2[(b * H + h) * Lq + (i - b * Lq)];
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) s += __shfl_xor(s, off, 64);
  if ((tid & 63) == 0) part[tid >> 6] = s;
  __syncthreads();
  if (tid == 0) {
    double all = 0.0;
    for (int i = 0; i < 16; ++i) all += part[i];
    dlam[h] = (float)-all;
  }
}

template <typename T, int D, int M, int S, bool BIAS>
int launch_bwd(EncAttnArgs a, hipStream_t stream) {
  using O = Ops<T>;
  const size_t slots = BIAS ? 2 * a.R + 1 : 0;
  const size_t tiles = sizeof(T) * (size_t)kTile * (M * O::row_pitch(D) + O::row_pitch(D * M)) + kTile * sizeof(int);
  size_t lds_q = tiles;
  if (BIAS) lds_q += sizeof(float) * ((M * slots + 3) / 4 * 4 + 4 * 16 * kDsPitch);
  a.hist_rows = 4;
  if (BIAS && a.hist) {
    // a row of sums per wave; one for all where four rows would leave a single workgroup per CU
    if (lds_q + sizeof(float) * 4 * M * slots > kMaxLds / 2) a.hist_rows = 1;
    lds_q += sizeof(float) * a.hist_rows * M * slots;
  }
  int rc = enc_lds(enc_attn_bwd_q_kernel<T, D, M, S, BIAS>, lds_q);
  if (rc) return rc;
  const size_t lds_k = tiles + sizeof(float) * (3 * M * kTile + M * slots);
  rc = enc_lds(enc_attn_bwd_k_kernel<T, D, M, S, BIAS>, lds_k);
  if (rc) return rc;
  const int nqt = (a.Lq + 64 * S - 1) / (64 * S), nkt = (a.Lk + 64 * S - 1) / (64 * S);
  hipLaunchKernelGGL((enc_attn_bwd_q_kernel<T, D, M, S, BIAS>), dim3((unsigned)(a.B * a.H * nqt)), dim3(256), lds_q, stream, a);
  rc = hip_err(hipGetLastError());
  if (rc) return rc;
  if (!a.dk) return 0;
  hipLaunchKernelGGL((enc_attn_bwd_k_kernel<T, D, M, S, BIAS>), dim3((unsigned)(a.B * a.KV * nkt)), dim3(256), lds_k, stream, a);
  return hip_err(hipGetLastError());
}

template <typename T>
int dispatch_bwd(const EncAttnArgs& a, hipStream_t stream) {
  const int w = enc_width(a.D);
  if (a.M == 1) {
    if (w == 32) return launch_bwd<T, 32, 1, 2, true>(a, stream);
    if (w == 64) return launch_bwd<T, 64, 1, 2, true>(a, stream);
    return launch_bwd<T, 128, 1, 1, true>(a, stream);
  }
  if (w == 32) return a.table ? launch_bwd<T, 32, 2, 1, true>(a, stream) : launch_bwd<T, 32, 2, 1, false>(a, stream);
  return a.table ? launch_bwd<T, 64, 2, 1, true>(a, stream) : launch_bwd<T, 64, 2, 1, false>(a, stream);
}

}  // namespace

extern "C" {

// Queries per workgroup of the query-owned pass (rows of EncAttnArgs::hist per (sample, head): ceil(Lq / this)).
int atri_enc_attn_bwd_queries(int D, int M) { return M == 1 && D <= 64 ? 128 : 64; }

// dq, dk, dv (every element written), delta and, where hist is set, the sums of dS by position difference.
int atri_enc_attn_bwd(const EncAttnArgs* args, hipStream_t stream) {
  if (!args) return -1;
  const EncAttnArgs& a = *args;
  const int rc = enc_check(a);
  if (rc) return rc;
  if (!a.q || !a.k || !a.v || !a.dout || !a.dq || !a.dk || !a.dv || !a.stat || !a.o32 || !a.delta) return -17;
  return a.bf16 ? dispatch_bwd<unsigned short>(a, stream) : dispatch_bwd<float>(a, stream);
}

// dtable [buckets, H M] from hist [B H nqt, M, slots]; mid is [shares, H M, slots] scratch; order / start list the slots of every bucket.
int atri_enc_table_grad(const float* hist, float* mid, const int* order, const int* start, float* dtable, int B, int H, int M, int nqt, int slots,
                        int buckets, int shares, hipStream_t stream) {
  if (!hist || !mid || !order || !start || !dtable) return -17;
  if (B < 1 || H < 1 || M < 1 || nqt < 1 || slots < 1 || buckets < 1 || shares < 1 || shares > 65535 || (long long)H * M > 65535) return -10;
  if ((long long)B * nqt >= (1LL << 31) || (long long)buckets * H * M >= (1LL << 31) || (long long)slots * shares >= (1LL << 31)) return -15;
  hipLaunchKernelGGL(enc_hist_sum_kernel, dim3((slots + 63) / 64, H * M, shares), dim3(256), 0, stream, hist, mid, B, H, nqt, M, slots, shares);
  const int rc = hip_err(hipGetLastError());
  if (rc) return rc;
  hipLaunchKernelGGL(enc_bucket_sum_kernel, dim3((unsigned)((buckets * H * M + 3) / 4)), dim3(256), 0, stream, mid, order, start, dtable, buckets, H * M,
                     slots, shares);
  return hip_err(hipGetLastError());
}

int atri_enc_dlam(const float* delta2, float* dlam, int B, int H, int Lq, hipStream_t stream) {
  if (!delta2 || !dlam || B < 1 || H < 1 || Lq < 1) return -10;
  hipLaunchKernelGGL(enc_dlam_kernel, dim3(H), dim3(1024), 0, stream, delta2, dlam, B, H, Lq);
  return hip_err(hipGetLastError());
}

}  // extern "C"
