// Forward pass of the encoder attention operators (see encoder_attn.hpp for the mathematics and the operand layout), the
// join of key splits, and the key-validity words.
#include <type_traits>

#include "encoder_attn.hpp"

using namespace atrihip;

namespace {

// One 4-wave workgroup per (head, 64 QS queries, key split) and `chunk` samples, one after the other: the bias is laid out once
// and the next sample's first tile loads while this one's last is multiplied.  A wave owns 16 QS queries and walks the key tiles with the
// running maximum and sum of the softmax; per lane the sum is partial (its own keys) until the end.
// PL bf16 fragments per probability: two, 16 bits, for inference, so that the result's own rounding is the only one that counts (one
// fragment: 2.1e-3 off where rounding alone leaves 1.66e-3); three, all 24 bits, when a backward pass follows, for
// delta = dO . o has to match dP = dO V^T to 32 bits: the gradients of the table and of lam are sums of p (dP - delta) in which
// everything but the error of delta cancels (with one fragment they were 1e-3 off).
// Measured: 256 boards of 120 cells, four heads, fp32 29 us; 4096 of them in bf16 without gradients 149 us (3.4 TB/s; 133 us with one
// fragment); 256 boards of 252 cells, bf16, training 57 us; two sequences of 4095 tokens, eight 64-wide heads, bf16, training
// 192 us; two of 2000 tokens, four two-map 64-wide heads, fp32 225 us; one token of four sequences of up to 8190, 17 us
// (2.0 TB/s).  At two waves per SIMD the long ones wait: half of the wave cycles for LDS reads and barriers, a third issue vector
// instructions, a fifth matrix instructions.  A second LDS buffer (one barrier per tile instead of two) changed nothing.
template <typename T, int D, int M, int QS, bool BIAS, int PL, int NT>
__global__ __launch_bounds__(256, enc_waves(D, M, NT, QS, Ops<T>::kBf16, kEncForward)) void enc_attn_fwd_kernel(EncAttnArgs a) {
  using O = Ops<T>;
  using Frag = typename O::Frag;
  constexpr int DV = D * M, DC = D / O::kDims, NV = DV / 16, NKB = 4 / O::kSub;
  constexpr int PK = O::row_pitch(D), PV = O::tr_pitch(DV), TK = O::kParts * kTile * PK;
  // Where 32 bits of the output count, a sum per tile, joined to the long one together with the change of maximum: one rounding per 64
  // keys where the products would take twelve (fp32, 2000 tokens: output 5e-7 off without, 2e-7 with; bf16 training, 4095 tokens: the
  // table's gradient 7 to 12e-7 off without, 5 to 8e-7 with, 190 -> 200 us).
  constexpr bool TILE_SUMS = NT == 0 && (PL == 3 || !O::kBf16);
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  typename O::Lds* k_lds = reinterpret_cast<typename O::Lds*>(smem);
  typename O::Lds* v_lds = k_lds + M * TK;
  int* pos_lds = reinterpret_cast<int*>(v_lds + O::kParts * kTile * PV);
  float* bias_lds = reinterpret_cast<float*>(pos_lds + (NT ? NT : 1) * kTile);

  const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, q4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // what follows from it (owned rows, clamped sides) stays in scalar registers
  const int nqt = (a.Lq + 64 * QS - 1) / (64 * QS);
  int id = xcd_order(blockIdx.x, gridDim.x);
  const int qt = id % nqt;
  id /= nqt;
  const int split = id % a.splits;
  id /= a.splits;
  const int h = id % a.H, kvh = h / (a.H / a.KV);
  const int b_first = id / a.H * a.chunk, b_last = b_first + a.chunk < a.B ? b_first + a.chunk : a.B;
  const int tiles = (a.Lk + kTile - 1) / kTile;
  const int per = (tiles + a.splits - 1) / a.splits;
  const int t_first = split * per, t_last = t_first + per < tiles ? t_first + per : tiles;
  const int R2 = 2 * a.R;
  const int q_first = (qt * 4 + wave) * 16 * QS;
  const bool busy = q_first < a.Lq;  // wave-uniform
  const float sl2 = a.scale * kLog2E;
  const float lam = M == 2 ? a.lam[h] : 0.f;

  Stage<T, D> sk[M];
  Stage<T, DV> sv;
  auto fetch = [&](const TileWalk& w) {
    const typename O::Mem* kb = reinterpret_cast<const typename O::Mem*>(a.k) + w.sample * a.ks[0] + (long long)kvh * M * a.ks[2];
#pragma unroll
    for (int m = 0; m < M; ++m) sk[m].load(kb + m * a.ks[2], a.ks[1], w.tile * kTile, w.word, a.D, tid);
    sv.load(reinterpret_cast<const typename O::Mem*>(a.v) + w.sample * a.vs[0] + kvh * a.vs[2], a.vs[1], w.tile * kTile, w.word, a.DV, tid);
  };
  Frag qf[M][QS][DC];
  auto fetch_queries = [&](int b) {
#pragma unroll
    for (int s = 0; s < QS; ++s) {
      const int query = q_first + s * 16 + l15;
#pragma unroll
      for (int m = 0; m < M; ++m)
        load_rows<T, DC>(qf[m][s], reinterpret_cast<const typename O::Mem*>(a.q) + b * a.qs[0] + (long long)query * a.qs[1] + (long long)(h * M + m) * a.qs[2],
                         query < a.Lq, a.D, q4);
    }
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
  fetch_queries(b_first);
  if constexpr (BIAS) fill_bias(a, bias_lds, h, M, tid);
  int token_q[QS];
#pragma unroll
  for (int s = 0; s < QS; ++s) token_q[s] = BIAS ? token_pos(q_first + s * 16 + l15, a.W) : 0;
  float4v bias_reg[M][QS][NT ? NT * 4 : 1];
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
          for (int s = 0; s < QS; ++s) bias_reg[m][s][kt][j] = key < a.Lk ? bias_lds[m * (R2 + 1) + clamp_slot(pos - token_q[s] + a.R, R2)] : -INFINITY;
      }
  }

  for (int b = b_first; b < b_last; ++b) {
    const int origin = BIAS ? query_origin(a, b) : 0;
    float4v o[M][QS][NV];
    float run_max[M][QS], run_sum[M][QS];
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int s = 0; s < QS; ++s) {
        run_max[m][s] = -INFINITY;
        run_sum[m][s] = 0.f;
#pragma unroll
        for (int n = 0; n < NV; ++n) o[m][s][n] = float4v{0.f, 0.f, 0.f, 0.f};
      }
    // One staged tile; kt0 is its first 16-key block where the bias is in registers.
    auto tile = [&](auto kt0_) {
      constexpr int kt0 = decltype(kt0_)::value;
      // tail keys of a board are -inf in its bias already
      const unsigned long long word = NT > 0 && !a.words ? ~0ULL : walk.word;
      const int t0 = walk.tile * kTile;
      __syncthreads();  // every wave is past its reads of the previous tile
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
      if (walk.sample < b_last) fetch(walk);  // the next tile's loads (this sample's or the next one's) run under this tile's products
      if (!busy) return;

      // Few and wide basic blocks per map: the start of the scores, all products, one branch each for masked keys, far rows and
      // new maxima.
      float4v st[M][QS][4];
      float fade[M][QS];
#pragma unroll
      for (int m = 0; m < M; ++m) {
#pragma unroll
        for (int s = 0; s < QS; ++s) {
          float4v* x = st[m][s];
          if constexpr (NT > 0) {
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) x[kt] = bias_reg[m][s][kt0 + kt];
          } else if constexpr (BIAS) {
            const float* bias = bias_lds + m * (R2 + 1);
            const int qa = q_first + s * 16 + origin;
            const int side = clamped_side(a, t0, t0 + kTile - 1, qa, qa + 15);
            if (side != 0) {
              const float c = bias[side > 0 ? R2 : 0];
#pragma unroll
              for (int kt = 0; kt < 4; ++kt) x[kt] = float4v{c, c, c, c};
            } else {
              const int off = a.R - token_q[s] - origin;
#pragma unroll
              for (int kt = 0; kt < 4; ++kt) {
                const int4 p = *reinterpret_cast<const int4*>(pos_lds + kt * 16 + q4 * 4);
                const int pj[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) x[kt][j] = bias[clamp_slot(pj[j] + off, R2)];
              }
            }
          } else {
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) x[kt] = float4v{0.f, 0.f, 0.f, 0.f};
          }
        }
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int c = 0; c < DC; ++c) {
            const Frag kf = O::row_frag(k_lds + m * TK, PK, kt * 16 + l15, c, q4);
#pragma unroll
            for (int s = 0; s < QS; ++s) st[m][s][kt] = O::mma(kf, qf[m][s][c], st[m][s][kt]);
          }
        if (word != ~0ULL) {
#pragma unroll
          for (int kt = 0; kt < 4; ++kt) {
            const unsigned bits = (unsigned)(word >> (kt * 16 + q4 * 4));
#pragma unroll
            for (int s = 0; s < QS; ++s)
#pragma unroll
              for (int j = 0; j < 4; ++j) st[m][s][kt][j] = (bits >> j) & 1 ? st[m][s][kt][j] : -INFINITY;
          }
        }
        float from[QS];
        bool far = false;
#pragma unroll
        for (int s = 0; s < QS; ++s) {
          float top = run_max[m][s];
#pragma unroll
          for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int j = 0; j < 4; ++j) top = fmaxf(top, st[m][s][kt][j]);
          top = quad_row_max(top);
          from[s] = top == -INFINITY ? 0.f : top;  // nothing seen yet: exp2(-inf - 0) = 0, never inf - inf
          fade[m][s] = run_max[m][s];
          run_max[m][s] = top;
          far |= Exponent::far(Exponent::base_of(from[s], sl2));
        }
        if (__any(far)) {
#pragma unroll
          for (int s = 0; s < QS; ++s) {
            fade[m][s] = Exponent::far_(fade[m][s], from[s], sl2);
#pragma unroll
            for (int kt = 0; kt < 4; ++kt)
#pragma unroll
              for (int j = 0; j < 4; ++j) st[m][s][kt][j] = Exponent::far_(st[m][s][kt][j], from[s], sl2);
          }
        } else {
#pragma unroll
          for (int s = 0; s < QS; ++s) {
            const float base = Exponent::base_of(from[s], sl2);
            fade[m][s] = __builtin_amdgcn_exp2f(Exponent::base_of(fade[m][s], sl2) - base);
#pragma unroll
            for (int kt = 0; kt < 4; ++kt)
#pragma unroll
              for (int j = 0; j < 4; ++j) st[m][s][kt][j] = Exponent::near_(st[m][s][kt][j], base, sl2);
          }
        }
        bool faded = false;
#pragma unroll
        for (int s = 0; s < QS; ++s) {
          float sum = 0.f;
#pragma unroll
          for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int j = 0; j < 4; ++j) sum += st[m][s][kt][j];
          run_sum[m][s] = fmaf(run_sum[m][s], fade[m][s], sum);
          faded |= fade[m][s] != 1.0f;
        }
        if (!TILE_SUMS && __any(faded)) {
#pragma unroll
          for (int s = 0; s < QS; ++s)
#pragma unroll
            for (int n = 0; n < NV; ++n)
#pragma unroll
              for (int j = 0; j < 4; ++j) o[m][s][n][j] *= fade[m][s];
        }
      }
      if constexpr (TILE_SUMS) {
        Frag pf[NKB][M][QS][PL];
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
          for (int m = 0; m < M; ++m)
#pragma unroll
            for (int s = 0; s < QS; ++s)
#pragma unroll
              for (int p = 0; p < PL; ++p) {
                pf[kb][m][s][p] = O::acc_frag(&st[m][s][kb * O::kSub]);
                if (p + 1 < PL) O::take(&st[m][s][kb * O::kSub], pf[kb][m][s][p]);
              }
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          float4v sum[M][QS];
#pragma unroll
          for (int kb = 0; kb < NKB; ++kb) {
            const Frag vf = O::tr_frag(v_lds, PV, kb, n, l15, q4);
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
              for (int s = 0; s < QS; ++s)
#pragma unroll
                for (int p = PL - 1; p >= 0; --p)
                  sum[m][s] = O::mma(vf, pf[kb][m][s][p], kb == 0 && p == PL - 1 ? float4v{0.f, 0.f, 0.f, 0.f} : sum[m][s]);
          }
#pragma unroll
          for (int m = 0; m < M; ++m)
#pragma unroll
            for (int s = 0; s < QS; ++s)
#pragma unroll
              for (int j = 0; j < 4; ++j) o[m][s][n][j] = fmaf(o[m][s][n][j], fade[m][s], sum[m][s][j]);
        }
      } else {
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb) {
          Frag pf[M][QS][PL];
#pragma unroll
          for (int m = 0; m < M; ++m)
#pragma unroll
            for (int s = 0; s < QS; ++s)
#pragma unroll
              for (int p = 0; p < PL; ++p) {
                pf[m][s][p] = O::acc_frag(&st[m][s][kb * O::kSub]);
                if (p + 1 < PL) O::take(&st[m][s][kb * O::kSub], pf[m][s][p]);
              }
#pragma unroll
          for (int n = 0; n < NV; ++n) {
            const Frag vf = O::tr_frag(v_lds, PV, kb, n, l15, q4);
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
              for (int s = 0; s < QS; ++s)
#pragma unroll
                for (int p = PL - 1; p >= 0; --p) o[m][s][n] = O::mma(vf, pf[m][s][p], o[m][s][n]);
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
    if (b + 1 < b_last) fetch_queries(b + 1);
    if (!busy) continue;
    const long long rows = (long long)a.B * a.H * a.Lq;
#pragma unroll
    for (int s = 0; s < QS; ++s) {
      const int query = q_first + s * 16 + l15;
      float inv[M];
      const long long row = ((long long)b * a.H + h) * a.Lq + query;
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const float sum = quad_row_sum(run_sum[m][s]);
        inv[m] = sum == 0.f ? 0.f : 1.0f / sum;
        if (query < a.Lq && q4 == 0) {
          if (a.splits > 1) {
            float* ml = a.part_ml + 2 * (((long long)split * M + m) * rows + row);
            ml[0] = run_max[m][s];
            ml[1] = sum;
          } else if (a.stat) {
            *reinterpret_cast<float2*>(a.stat + 2 * (m * rows + row)) = make_float2(sum == 0.f ? INFINITY : run_max[m][s], inv[m]);
          }
        }
      }
      if (query >= a.Lq) continue;
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const int dim = n * 16 + q4 * 4;
        if (dim >= a.DV) continue;
        float4v r[M];
#pragma unroll
        for (int m = 0; m < M; ++m) {
          r[m] = o[m][s][n];
          if (a.splits > 1) {
            Ops<float>::store4(a.part_o + (((long long)split * M + m) * rows + row) * a.DV + dim, r[m][0], r[m][1], r[m][2], r[m][3]);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) r[m][j] *= inv[m];
            if (a.o32) Ops<float>::store4(a.o32 + b * a.o32s[0] + (long long)query * a.o32s[1] + h * a.o32s[2] + m * a.o32s[3] + dim, r[m][0], r[m][1], r[m][2], r[m][3]);
          }
        }
        if (a.splits > 1) continue;
        if constexpr (M == 2) {
#pragma unroll
          for (int j = 0; j < 4; ++j) r[0][j] = fmaf(-lam, r[1][j], r[0][j]);
        }
        O::store4(reinterpret_cast<typename O::Mem*>(a.out) + b * a.os[0] + (long long)query * a.os[1] + h * a.os[2] + dim, r[0][0], r[0][1], r[0][2], r[0][3]);
      }
    }
  }
}

// Joins the partial softmaxes of `splits` key ranges, four output values of a row at a time.  SHARES = 4: by four threads, each with a
// quarter of the ranges, whose loads are under way together - with few rows the kernel is a chain of latencies (one token
// of four sequences: 7 -> 4.5 us); one thread reads whole lines (two maps of 12004 rows: 19 us with four, 11 us with one).
template <typename T, int M, int SHARES>
__global__ __launch_bounds__(256) void enc_attn_join_kernel(EncAttnArgs a) {
  const long long rows = (long long)a.B * a.H * a.Lq;
  const int quads = a.DV / 4, share = SHARES == 4 ? (threadIdx.x >> 4) & 3 : 0;
  const long long i = SHARES == 4 ? ((long long)blockIdx.x * 4 + (threadIdx.x >> 6)) * 16 + (threadIdx.x & 15) : (long long)blockIdx.x * 256 + threadIdx.x;
  const bool on = i < rows * quads;
  const long long row = on ? i / quads : 0;
  const int dim = on ? (int)(i - row * quads) * 4 : 0;
  const int query = (int)(row % a.Lq);
  const long long bh = row / a.Lq;
  const int b = (int)(bh / a.H), h = (int)(bh - (long long)b * a.H);
  const float sl2 = a.scale * kLog2E;
  const long long step = (long long)M * rows;
  float4v r[M];
#pragma unroll
  for (int m = 0; m < M; ++m) {
    const float* ml = a.part_ml + 2 * (m * rows + row);
    const float* po = a.part_o + (m * rows + row) * a.DV + dim;
    float top = -INFINITY;
#pragma unroll 4
    for (int s = share; s < a.splits; s += SHARES) top = fmaxf(top, ml[2 * s * step]);
    if constexpr (SHARES == 4) top = quad_row_max(top);
    const float from = top == -INFINITY ? 0.f : top, base = Exponent::base_of(from, sl2);
    float sum = 0.f;
    float4v acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = share; s < a.splits; s += SHARES) {
      const float t = ml[2 * s * step];
      const float w = Exponent::far(base) ? Exponent::far_(t, from, sl2) : __builtin_amdgcn_exp2f(Exponent::base_of(t, sl2) - base);
      const float4v p = *reinterpret_cast<const float4v*>(po + s * step * a.DV);
      sum = fmaf(ml[2 * s * step + 1], w, sum);
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] = fmaf(p[j], w, acc[j]);
    }
    if constexpr (SHARES == 4) sum = quad_row_sum(sum);
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
    for (int j = 0; j < 4; ++j) r[m][j] = (SHARES == 4 ? quad_row_sum(acc[j]) : acc[j]) * inv;
    if (!on || share != 0) continue;
    if (a.stat && dim == 0) *reinterpret_cast<float2*>(a.stat + 2 * (m * rows + row)) = make_float2(sum == 0.f ? INFINITY : top, inv);
    if (a.o32) Ops<float>::store4(a.o32 + b * a.o32s[0] + (long long)query * a.o32s[1] + h * a.o32s[2] + m * a.o32s[3] + dim, r[m][0], r[m][1], r[m][2], r[m][3]);
  }
  if (!on || share != 0) return;
  if constexpr (M == 2) {
    const float lam = a.lam[h];
#pragma unroll
    for (int j = 0; j < 4; ++j) r[0][j] = fmaf(-lam, r[1][j], r[0][j]);
  }
  Ops<T>::store4(reinterpret_cast<T*>(a.out) + b * a.os[0] + (long long)query * a.os[1] + h * a.os[2] + dim, r[0][0], r[0][1], r[0][2], r[0][3]);
}

// One 64-bit word per 64 keys of a byte mask [B, Lk] (strides in bytes); one wave per word.
__global__ __launch_bounds__(256) void key_words_kernel(const unsigned char* mask, long long sb, long long sk, unsigned long long* words, int B, int Lk) {
  const int tiles = (Lk + 63) / 64;
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (w >= (long long)B * tiles) return;
  const int b = (int)(w / tiles), key = (int)(w - (long long)b * tiles) * 64 + (threadIdx.x & 63);
  const bool on = key < Lk && mask[b * sb + key * sk] != 0;
  const unsigned long long bits = __ballot(on);
  if ((threadIdx.x & 63) == 0) words[w] = bits;
}

template <typename T, int D, int M, int QS, bool BIAS, int PL, int NT>
int launch_fwd_planes(const EncAttnArgs& a, hipStream_t stream) {
  static_assert(enc_tiles_agree<T, D, M, kEncForward>());
  const int lds = enc_lds_bytes(enc_form<T>(), D, M, NT, kEncForward, BIAS ? 2 * a.R + 1 : 0, 0);
  const int rc = enc_lds(enc_attn_fwd_kernel<T, D, M, QS, BIAS, PL, NT>, lds);
  if (rc) return rc;
  const int nqt = (a.Lq + 64 * QS - 1) / (64 * QS);
  hipLaunchKernelGGL((enc_attn_fwd_kernel<T, D, M, QS, BIAS, PL, NT>), dim3((unsigned)((a.B + a.chunk - 1) / a.chunk * a.H * nqt * a.splits)), dim3(256), lds,
                     stream, a);
  return hip_err(hipGetLastError());
}

template <typename T, int D, int M, int QS, bool BIAS, int NT = 0>
int launch_fwd(const EncAttnArgs& a, hipStream_t stream) {
  if constexpr (Ops<T>::kBf16) {
    return a.o32 ? launch_fwd_planes<T, D, M, QS, BIAS, 3, NT>(a, stream) : launch_fwd_planes<T, D, M, QS, BIAS, 2, NT>(a, stream);
  } else {
    return launch_fwd_planes<T, D, M, QS, BIAS, 1, NT>(a, stream);
  }
}

// T: bf16 rows, or Split
template <typename T>
int dispatch_fwd(const EncAttnArgs& a, hipStream_t stream) {
  const int w = enc_width(a.D), nt = enc_board_tiles(a.table ? a.W : 0, a.Lk, a.D, a.M);
  if (nt > 0 && a.splits > 1) return -18;
  const bool two = enc_columns(a.table ? a.W : 0, a.Lq, a.Lk, a.D, a.M, a.bf16 != 0, kEncForward) == 2;
  if (a.M == 1) {
    if (nt == 2) return launch_fwd<T, 32, 1, enc_columns_of(32, 1, 2, Ops<T>::kBf16, kEncForward), true, 2>(a, stream);
    if (nt == 4) return launch_fwd<T, 32, 1, 1, true, 4>(a, stream);
    if (w == 32) return two ? launch_fwd<T, 32, 1, 2, true>(a, stream) : launch_fwd<T, 32, 1, 1, true>(a, stream);
    if (w == 64) return two ? launch_fwd<T, 64, 1, 2, true>(a, stream) : launch_fwd<T, 64, 1, 1, true>(a, stream);
    return launch_fwd<T, 128, 1, 1, true>(a, stream);
  }
  if (nt == 2) return launch_fwd<T, 32, 2, 1, true, 2>(a, stream);
  if (w == 32) return a.table ? launch_fwd<T, 32, 2, 1, true>(a, stream) : launch_fwd<T, 32, 2, 1, false>(a, stream);
  return a.table ? launch_fwd<T, 64, 2, 1, true>(a, stream) : launch_fwd<T, 64, 2, 1, false>(a, stream);
}

template <typename T, int M>
int launch_join(const EncAttnArgs& a, hipStream_t stream) {
  const long long n = (long long)a.B * a.H * a.Lq * (a.DV / 4);
  if ((n + 255) / 256 >= (1LL << 31)) return -15;
  if (n <= 65536) hipLaunchKernelGGL((enc_attn_join_kernel<T, M, 4>), dim3((unsigned)((n + 63) / 64)), dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((enc_attn_join_kernel<T, M, 1>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, a);
  return hip_err(hipGetLastError());
}
template <typename T>
int join(const EncAttnArgs& a, hipStream_t stream) {
  return a.M == 1 ? launch_join<T, 1>(a, stream) : launch_join<T, 2>(a, stream);
}

}  // namespace

extern "C" {

// out (and, where the pointers are set, stat and o32) of one attention call.
int atri_enc_attn_fwd(const EncAttnArgs* args, hipStream_t stream) {
  if (!args) return -1;
  const EncAttnArgs& a = *args;
  const int rc = enc_check(a);
  if (rc) return rc;
  if (!a.q || !a.k || !a.v || !a.out || (a.splits > 1 && (!a.part_o || !a.part_ml))) return -17;
  if (a.mask) {
    if (!a.words) return -17;
    const long long n = ((long long)a.B * ((a.Lk + 63) / 64) + 3) / 4;
    if (n >= (1LL << 31)) return -15;
    hipLaunchKernelGGL(key_words_kernel, dim3((unsigned)n), dim3(256), 0, stream, a.mask, a.ms[0], a.ms[1], a.words, a.B, a.Lk);
    const int rc1 = hip_err(hipGetLastError());
    if (rc1) return rc1;
  }
  const int rc2 = a.bf16 ? dispatch_fwd<unsigned short>(a, stream) : dispatch_fwd<Split>(a, stream);
  if (rc2 || a.splits == 1) return rc2;
  return a.bf16 ? join<unsigned short>(a, stream) : join<float>(a, stream);
}

}  // extern "C"
