// Shared parts of the encoder attention kernels (encoder_attn_*_kernels.hip): arguments, operand fragments, tile staging,
// key validity, relative positions.
//
// One family of kernels serves both operators.  With M maps per head (M = 1: softmax attention with a relative position
// bias, M = 2: two-map "differential" attention), head h of sample b computes
//     x_m[i][j] = scale q_m[i] . k_m[j] + T[bucket(pos(j) - pos(i))][h M + m],   P_m = softmax_j(x_m),
//     o[i] = sum_j P_1[i][j] v[j]                     (M = 1, values D wide)
//     o[i] = sum_j (P_1 - lam_h P_2)[i][j] v[j]       (M = 2, values 2 D wide)
// and its gradients.  The bias, divided by the scale, is where the matrix product's accumulator starts, so the scores cost
// no vector instruction until the exponential, exp2(fma(x, scale log2 e, -base)): see Exponent.
//
// Matrix operands.  bf16 rows use v_mfma_f32_16x16x32_bf16 as they are.  fp32 rows are cut into three bf16 values that
// carry all 24 bits (Split), and a product is the six of the nine partial products that reach above 2^-25 of it: 96 cycles for
// a depth of 32, where eight v_mfma_f32_16x16x4_f32 take 256 (two 2048-token sequences of eight 32-wide heads: forward 107 ->
// 82 us, backward 349 -> 258 us).  Two parts and three products would carry 16 bits, 30 times the rounding of an fp32 product.
// Where three parts do not fit, the fp32 instruction stays (see the dispatch).
// A fragment covers kDims values of the contraction: lane (l15 = lane & 15, q4 = lane >> 4) holds, for row / column l15,
//   bf16, Split: values 8 q4 .. 8 q4 + 7 of 32;   fp32: values 4 q4 .. 4 q4 + 3 of 16 (four 4-deep instructions, one value each);
// an accumulator gives the lane C[4 q4 + j][l15], j = 0..3.  With the owned rows (queries in the forward and the dQ pass,
// keys in the dK / dV pass) as COLUMNS of every product, softmax sums stay inside a lane plus one exchange over q4, and
// an accumulator (two of them for bf16) is the B fragment of the product that follows, without any exchange: the
// contraction order it implies is 4 q4 + e (+ 16 for the second half), which tr_frag reads from LDS.
#pragma once
#include "common.hpp"
#include "encoder_ops.h"

namespace atrihip {

typedef __attribute__((ext_vector_type(4))) short short4v;

constexpr float kLog2E = 1.4426950408889634f;

template <typename T>
struct Ops;

struct Split {};  // tag: fp32 rows as three bf16 parts

template <>
struct Ops<unsigned short> {
  using Frag = short8;
  using Mem = unsigned short;        // element in memory
  using Lds = unsigned short;        // element of a staged tile
  static constexpr bool kBf16 = true;
  static constexpr int kDims = 32;   // contraction values per fragment
  static constexpr int kLane = 8;    // of them in a lane
  static constexpr int kVec = 8;     // elements in memory per 16 bytes
  static constexpr int kSub = 2;     // 16-row accumulators per B fragment
  static constexpr int kParts = 1;   // tiles of [kTile][pitch] that make a staged one
  static constexpr int row_pitch(int d) { return d + 8; }   // 16-lane b128 row reads: all 64 banks once
  static constexpr int tr_pitch(int d) { return d + 16; }   // transposing reads: eight 32-byte rows on distinct banks
  static __device__ __forceinline__ Frag from_memory(const unsigned short* p) { return *reinterpret_cast<const short8*>(p); }
  static __device__ __forceinline__ void stage(unsigned short* t, int pitch, int row, int col, const uint4& v) {
    *reinterpret_cast<uint4*>(t + row * pitch + col) = v;
  }
  static __device__ __forceinline__ Frag row_frag(const unsigned short* t, int pitch, int row, int c, int q4) {
    return *reinterpret_cast<const short8*>(t + row * pitch + c * 32 + q4 * 8);
  }
  // A fragment of the transpose: column n 16 + l15 of rows 32 kb + 4 q4 + e and 32 kb + 16 + 4 q4 + e, e = 0..3.  A 16-lane
  // group of the transposing read takes four rows of 16 values; the lane supplies the address of a quarter row.
  static __device__ __forceinline__ Frag tr_frag(const unsigned short* t, int pitch, int kb, int n, int l15, int q4) {
    typedef __attribute__((address_space(3))) short4v* lds4;
    unsigned short* p = const_cast<unsigned short*>(t) + (kb * 32 + 4 * q4 + (l15 >> 2)) * pitch + n * 16 + (l15 & 3) * 4;
    const short4v a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p);
    const short4v b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + 16 * pitch));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  static __device__ __forceinline__ Frag acc_frag(const float4v* s) {
    return pack_bf16x8(s[0][0], s[0][1], s[0][2], s[0][3], s[1][0], s[1][1], s[1][2], s[1][3]);
  }
  static __device__ __forceinline__ float4v mma(const Frag& a, const Frag& b, float4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float4v mma_mirrored(const Frag& a, const Frag& b, float4v c) { return mma(a, b, c); }
  // rows of 32-bit values against bf16 ones: three parts carry all of them, and a row of bf16 values gives the bits of mma
  static __device__ __forceinline__ float4v mma_rows32(const float* row, const Frag& b, float4v c) {
    float4v s[2] = {*reinterpret_cast<const float4v*>(row), *reinterpret_cast<const float4v*>(row + 4)};
    Frag part[3];
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      part[p] = acc_frag(s);
      if (p < 2) take(s, part[p]);
    }
#pragma unroll
    for (int p = 2; p >= 0; --p) c = mma(part[p], b, c);
    return c;
  }
  // s -= value(f): what the next of several fragments of the same values has to carry.
  static __device__ __forceinline__ void take(float4v* s, const Frag& f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e >> 2][e & 3] -= bf16_to_float((unsigned short)f[e]);
  }
  static __device__ __forceinline__ void negate(Frag& f, bool on) {
    uint4v u = __builtin_bit_cast(uint4v, f);
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] ^= on ? 0x80008000u : 0u;
    f = __builtin_bit_cast(Frag, u);
  }
  static __device__ __forceinline__ void store4(unsigned short* p, float a, float b, float c, float d) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(a, b), pack_bf16x2(c, d));
  }
};

template <>
struct Ops<float> {
  using Frag = float4v;
  using Mem = float;
  using Lds = float;
  static constexpr bool kBf16 = false;
  static constexpr int kDims = 16;
  static constexpr int kLane = 4;
  static constexpr int kVec = 4;
  static constexpr int kSub = 1;
  static constexpr int kParts = 1;
  static constexpr int row_pitch(int d) { return d + 4; }
  static constexpr int tr_pitch(int d) { return d + 4; }
  static __device__ __forceinline__ Frag from_memory(const float* p) { return *reinterpret_cast<const float4v*>(p); }
  static __device__ __forceinline__ void stage(float* t, int pitch, int row, int col, const uint4& v) {
    *reinterpret_cast<uint4*>(t + row * pitch + col) = v;
  }
  static __device__ __forceinline__ Frag row_frag(const float* t, int pitch, int row, int c, int q4) {
    return *reinterpret_cast<const float4v*>(t + row * pitch + c * 16 + q4 * 4);
  }
  static __device__ __forceinline__ Frag tr_frag(const float* t, int pitch, int kb, int n, int l15, int q4) {
    const float* p = t + (kb * 16 + 4 * q4) * pitch + n * 16 + l15;
    return Frag{p[0], p[pitch], p[2 * pitch], p[3 * pitch]};
  }
  static __device__ __forceinline__ Frag acc_frag(const float4v* s) { return s[0]; }
  static __device__ __forceinline__ void take(float4v*, const Frag&) {}
  static __device__ __forceinline__ float4v mma(const Frag& a, const Frag& b, float4v c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ float4v mma_mirrored(const Frag& a, const Frag& b, float4v c) { return mma(a, b, c); }
  static __device__ __forceinline__ float4v mma_rows32(const float* row, const Frag& b, float4v c) { return mma(from_memory(row), b, c); }
  static __device__ __forceinline__ void negate(Frag& f, bool on) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = on ? -f[i] : f[i];
  }
  static __device__ __forceinline__ void store4(float* p, float a, float b, float c, float d) {
    *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
  }
};

template <>
struct Ops<Split> {
  using One = Ops<unsigned short>;
  struct Frag {
    short8 part[3];
  };
  using Mem = float;
  using Lds = unsigned short;
  static constexpr bool kBf16 = false;
  static constexpr int kDims = 32;
  static constexpr int kLane = 8;
  static constexpr int kVec = 4;
  static constexpr int kSub = 2;
  static constexpr int kParts = 3;
  static constexpr int row_pitch(int d) { return One::row_pitch(d); }
  static constexpr int tr_pitch(int d) { return One::tr_pitch(d); }
  // Eight values, each the sum of its three parts: bf16(x), bf16 of the rest, and what then remains, at most 8 bits.
  static __device__ __forceinline__ Frag cut(float4v a, float4v b) {
    Frag f;
    float4v s[2] = {a, b};
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      f.part[p] = One::acc_frag(s);
      if (p < 2) One::take(s, f.part[p]);
    }
    return f;
  }
  static __device__ __forceinline__ Frag from_memory(const float* p) {
    return cut(*reinterpret_cast<const float4v*>(p), *reinterpret_cast<const float4v*>(p + 4));
  }
  static __device__ __forceinline__ void stage(unsigned short* t, int pitch, int row, int col, const uint4& v) {
    float4v s = __builtin_bit_cast(float4v, v);
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      const uint2 w = make_uint2(pack_bf16x2(s[0], s[1]), pack_bf16x2(s[2], s[3]));
      *reinterpret_cast<uint2*>(t + (p * kTile + row) * pitch + col) = w;
      s[0] -= __uint_as_float(w.x << 16);
      s[1] -= __uint_as_float(w.x & 0xffff0000u);
      s[2] -= __uint_as_float(w.y << 16);
      s[3] -= __uint_as_float(w.y & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ Frag row_frag(const unsigned short* t, int pitch, int row, int c, int q4) {
    Frag f;
#pragma unroll
    for (int p = 0; p < 3; ++p) f.part[p] = One::row_frag(t + p * kTile * pitch, pitch, row, c, q4);
    return f;
  }
  static __device__ __forceinline__ Frag tr_frag(const unsigned short* t, int pitch, int kb, int n, int l15, int q4) {
    Frag f;
#pragma unroll
    for (int p = 0; p < 3; ++p) f.part[p] = One::tr_frag(t + p * kTile * pitch, pitch, kb, n, l15, q4);
    return f;
  }
  static __device__ __forceinline__ Frag acc_frag(const float4v* s) { return cut(s[0], s[1]); }
  static __device__ __forceinline__ void take(float4v*, const Frag&) {}
  static __device__ __forceinline__ float4v mma(const Frag& a, const Frag& b, float4v c) {  // smallest terms first
    c = One::mma(a.part[2], b.part[0], c);
    c = One::mma(a.part[0], b.part[2], c);
    c = One::mma(a.part[1], b.part[1], c);
    c = One::mma(a.part[1], b.part[0], c);
    c = One::mma(a.part[0], b.part[1], c);
    return One::mma(a.part[0], b.part[0], c);
  }
  static __device__ __forceinline__ float4v mma_mirrored(const Frag& a, const Frag& b, float4v c) {  // the bits of mma(b, a)
    c = One::mma(a.part[0], b.part[2], c);
    c = One::mma(a.part[2], b.part[0], c);
    c = One::mma(a.part[1], b.part[1], c);
    c = One::mma(a.part[0], b.part[1], c);
    c = One::mma(a.part[1], b.part[0], c);
    return One::mma(a.part[0], b.part[0], c);
  }
  static __device__ __forceinline__ float4v mma_rows32(const float* row, const Frag& b, float4v c) { return mma(from_memory(row), b, c); }
  static __device__ __forceinline__ void negate(Frag& f, bool on) {
#pragma unroll
    for (int p = 0; p < 3; ++p) One::negate(f.part[p], on);
  }
  static __device__ __forceinline__ void store4(float* p, float a, float b, float c, float d) { Ops<float>::store4(p, a, b, c, d); }
};

// An accumulator as the B fragments of the product that follows, PL of them where one holds fewer bits (bf16), and that product,
// smallest terms first.
template <typename T, int PL>
__device__ __forceinline__ void acc_parts(typename Ops<T>::Frag (&f)[PL], const float4v* s) {
  float4v rest[Ops<T>::kSub];
#pragma unroll
  for (int u = 0; u < Ops<T>::kSub; ++u) rest[u] = s[u];
#pragma unroll
  for (int p = 0; p < PL; ++p) {
    f[p] = Ops<T>::acc_frag(rest);
    if (p + 1 < PL) Ops<T>::take(rest, f[p]);
  }
}
template <typename T, int PL>
__device__ __forceinline__ float4v mma_parts(const typename Ops<T>::Frag& a, const typename Ops<T>::Frag (&b)[PL], float4v c) {
#pragma unroll
  for (int p = PL - 1; p >= 0; --p) c = Ops<T>::mma(a, b[p], c);
  return c;
}

// Consecutive logical workgroups on the same XCD (the hardware deals blockIdx out round robin over eight), so that the query
// tiles of one (sample, head), and the heads that share keys, meet in one L2.
__device__ __forceinline__ int xcd_order(int id, int n) {
  const int per = n >> 3, extra = n & 7, xcd = id & 7, slot = id >> 3;
  return xcd * per + (xcd < extra ? xcd : extra) + slot;
}

// Position of token t: its index, or on a W-wide board r (2 W - 1) + c, whose differences name (dr, dc) uniquely.
__device__ __forceinline__ int token_pos(int t, int W) { return W > 0 ? t + (t / W) * (W - 1) : t; }
__device__ __forceinline__ int query_origin(const EncAttnArgs& a, int b) {
  const int o = a.qoff ? a.qoff[b] : a.q0;
  return o < -(1 << 29) ? -(1 << 29) : o > (1 << 29) ? (1 << 29) : o;  // differences stay within 32 bits
}
__device__ __forceinline__ int clamp_slot(int d, int R2) { return max(0, min(d, R2)); }

// exp2 of (x - top) sl2, x and top in units of 1 / scale, sl2 = scale log2 e.  One fused multiply-add: base = top sl2 is rounded
// once, and every value of a row carries the same base, so its rounding cancels against the sum.  Far rows (|base| of a
// million: a table used as a mask) take the difference first, which is exact where they are equal; +inf (a row
// without keys, a query behind the last) gives zeros either way.
struct Exponent {
  // The rounded product itself, never fused into what follows: a row's values, the factors between its maxima (exp2 of the
  // difference of two bases) and the backward pass agree on it.  With the unrounded one in the factors, every new maximum moved
  // the row by 1e-7 against its sum.
  static __device__ __forceinline__ float base_of(float top, float sl2) {
#pragma clang fp contract(off)
    return top * sl2;
  }
  static __device__ __forceinline__ bool far(float base) { return fabsf(base) >= 1e6f && base != INFINITY; }
  static __device__ __forceinline__ float near_(float x, float base, float sl2) { return __builtin_amdgcn_exp2f(fmaf(x, sl2, -base)); }
  static __device__ __forceinline__ float far_(float x, float top, float sl2) { return __builtin_amdgcn_exp2f((x - top) * sl2); }
};

// The bias in units of 1 / scale; a finite bias stays finite (a table may hold the type's lowest value as a mask).
__device__ __forceinline__ float bias_units(float t, float scale) {
  const float x = t / scale;
  if (__builtin_isinf(x) && !__builtin_isinf(t)) return copysignf(3.4028234663852886e38f, t);
  return x;
}
__device__ __forceinline__ void fill_bias(const EncAttnArgs& a, float* bias, int head, int M, int tid) {
  const int n = 2 * a.R + 1, hm = a.H * M;
  for (int i = tid; i < n; i += 256) {
    const float* row = a.table + (size_t)a.lut[i] * hm + head * M;
    for (int m = 0; m < M; ++m) bias[m * n + i] = bias_units(row[m], a.scale);
  }
}

// Rows [t0, t0 + 64) of a [tokens, D] matrix on their way from memory to LDS: 16 bytes per thread and step, zeros where the row's
// bit in `word` is clear (whatever the masked row holds) and beyond the matrix's width.
template <typename T, int D>
struct Stage {
  using O = Ops<T>;
  static constexpr int kVecsPerRow = D / O::kVec;
  static constexpr int kN = kTile * kVecsPerRow / 256;
  uint4 r[kN];
  __device__ __forceinline__ void load(const typename O::Mem* base, long long pitch, int t0, unsigned long long word, int width, int tid) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int vi = tid + i * 256, row = vi / kVecsPerRow, col = (vi % kVecsPerRow) * O::kVec;
      r[i] = make_uint4(0, 0, 0, 0);
      if (((word >> row) & 1) && col < width) r[i] = *reinterpret_cast<const uint4*>(base + (long long)(t0 + row) * pitch + col);
    }
  }
  __device__ __forceinline__ void store(typename O::Lds* lds, int pitch, int tid) const {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int vi = tid + i * 256;
      O::stage(lds, pitch, vi / kVecsPerRow, (vi % kVecsPerRow) * O::kVec, r[i]);
    }
  }
};

// Row fragments of up to 16 owned tokens straight from memory (each value is read by one lane).
template <typename T, int C>
__device__ __forceinline__ void load_rows(typename Ops<T>::Frag (&f)[C], const typename Ops<T>::Mem* row, bool valid, int width, int q4) {
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int col = c * Ops<T>::kDims + q4 * Ops<T>::kLane;
    f[c] = typename Ops<T>::Frag{};
    if (valid && col < width) f[c] = Ops<T>::from_memory(row + col);
  }
}

__device__ __forceinline__ unsigned long long range_word(int t0, int L) {  // bits of rows t0 .. t0 + 63 that are below L
  const int n = L - t0;
  return n >= 64 ? ~0ULL : n <= 0 ? 0ULL : ((1ULL << n) - 1);
}

__device__ __forceinline__ unsigned long long board_word(const EncAttnArgs& a, int b, int tile) {
  if (tile * kTile >= a.Lk) return 0;
  return a.words ? a.words[(size_t)b * ((a.Lk + kTile - 1) / kTile) + tile] : range_word(tile * kTile, a.Lk);
}

// The key tiles [first, last) of samples [sample, samples) that hold a valid key, in order: (sample, tile, word) names the tile
// whose loads are under way, sample == samples the end.  64 validity words are held across the wave at a time; every wave
// of a workgroup walks the same list.
struct TileWalk {
  const unsigned long long* words;
  int Lk, tiles, first, last, samples, base;
  unsigned long long mine, live;
  int sample, tile;
  unsigned long long word;
  __device__ __forceinline__ void open() {
    base = first - (words ? 64 : 1);
    live = 0;
  }
  __device__ __forceinline__ void start(const EncAttnArgs& a, int b0, int b1, int t0, int t1) {
    words = a.words;
    Lk = a.Lk;
    tiles = (a.Lk + kTile - 1) / kTile;
    first = t0;
    last = t1;
    samples = b1;
    sample = b0;
    mine = 0;
    open();
    next();
  }
  __device__ __forceinline__ void next() {
    for (; sample < samples; ++sample, open()) {
      if (!words) {
        if (++base < last) {
          tile = base;
          word = range_word(base * kTile, Lk);
          return;
        }
        continue;
      }
      while (!live && base + 64 < last) {
        base += 64;
        const int lane = threadIdx.x & 63;
        mine = base + lane < last ? words[(size_t)sample * tiles + base + lane] : 0;
        live = __ballot(mine != 0);
      }
      if (live) {
        const int i = __ffsll(live) - 1;
        live &= live - 1;
        const unsigned lo = __builtin_amdgcn_readlane((unsigned)mine, i), hi = __builtin_amdgcn_readlane((unsigned)(mine >> 32), i);
        word = ((unsigned long long)hi << 32) | lo;
        tile = base + i;
        return;
      }
    }
  }
};

// Bias of a 16-query column against a 64-key tile when every difference is clamped the same way (long sequences).
// -1: all below, +1: all above, 0: mixed.
__device__ __forceinline__ int clamped_side(const EncAttnArgs& a, int kmin, int kmax, int qmin, int qmax) {
  if (a.W > 0) return 0;
  return kmin - qmax >= a.R ? 1 : kmax - qmin <= -a.R ? -1 : 0;
}

inline int enc_check(const EncAttnArgs& a) {
  if (a.B < 1 || a.Lq < 1 || a.Lk < 1 || a.H < 1 || a.KV < 1 || a.H % a.KV != 0) return -10;
  if (a.M < 1 || a.M > 2 || a.D < 8 || a.D % 8 != 0 || a.D > (a.M == 1 ? 128 : 64) || a.DV != a.D * a.M) return -11;
  if (a.table && (a.R < 0 || a.R > 2047 || a.lut == nullptr)) return -12;
  if (!(a.scale > 0.f) || !(a.scale < 3e38f)) return -19;
  if (a.M == 1 && !a.table) return -13;
  if (a.M == 2 && !a.lam) return -14;
  if (a.splits < 1 || a.q_splits < 1 || a.k_splits < 1 || a.chunk < 1 || a.q_chunk < 1 || a.k_chunk < 1) return -18;
  const long long most = a.splits > a.q_splits ? a.splits : a.q_splits;
  if ((long long)a.B * a.H * ((a.Lq + 63) / 64) * most >= (1LL << 31)) return -15;
  if ((long long)a.B * a.KV * ((a.Lk + 63) / 64) * a.k_splits >= (1LL << 31)) return -15;
  if (a.Lq > (1 << 29) || a.Lk > (1 << 29)) return -16;
  return 0;
}
// The padded head width a kernel is built for.
inline int enc_width(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }

template <typename T>
constexpr int enc_form() { return Ops<T>::kBf16 ? kRowsBf16 : Ops<T>::kParts == 3 ? kRowsParts : kRowsFp32; }
// What a kernel lays out is what the shared rule counts.
template <typename T, int D, int M, int PASS>
constexpr bool enc_tiles_agree() {
  using O = Ops<T>;
  const int pitches = M * O::row_pitch(D) + (PASS == kEncForward ? O::tr_pitch(D * M) : O::row_pitch(D * M));
  return enc_tile_bytes(enc_form<T>(), D, M, PASS) == (int)sizeof(typename O::Lds) * O::kParts * kTile * pitches;
}

// Raises a kernel's dynamic LDS limit (attribute of the function on the current device) and reports what does not fit.
template <typename F>
inline int enc_lds(F* fn, int bytes) {
  if (bytes > kMaxLds) return -20;
  return hip_err(hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
}

}  // namespace atrihip
