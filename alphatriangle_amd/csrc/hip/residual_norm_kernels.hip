// The joint between two blocks of a residual stream, in one pass over the rows:
//     y = x + s * sigmoid(g) * LN_post(z),    h = LN_pre(y)
// (LN_post: the norm after the block that produced z, with its residual scale s and an optional gate g per value or per
// token; LN_pre: the norm in front of the block that reads h) and its gradients.  Every value is read once and written
// once, so memory bounds it; everything between is in 32 bits, and y is never read back rounded: the backward pass
// recomputes it from x, z and g.
//
// LANES threads own a row (16 up to 128 values, 512 up to 4096) and hold 8 values of it each: with 16 the backward pass, which
// keeps five operands and five running sums per value, spilled.  Statistics are two-pass (mean, then centred squares) in
// registers.  With VEC a thread's 8 values are neighbours (16-byte accesses; widths in eights), otherwise they are LANES
// apart (any width).  Parameter gradients: a workgroup walks many rows,
// sums in registers, joins its row groups in a fixed order and writes one partial row; a second launch adds those.
#include "common.hpp"
#include "encoder_ops.h"

using namespace atrihip;

namespace {

__device__ __forceinline__ float read1(const float* p) { return *p; }
__device__ __forceinline__ float read1(const unsigned short* p) { return bf16_to_float(*p); }
__device__ __forceinline__ void write1(float* p, float v) { *p = v; }
__device__ __forceinline__ void write1(unsigned short* p, float v) { *p = float_to_bf16(v); }
__device__ __forceinline__ void read8(const float* p, float* v) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void read8(const unsigned short* p, float* v) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void write8(float* p, const float* v) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void write8(unsigned short* p, const float* v) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

// A thread's share of a row: the column of its value e, and whole-share transfers (zeros beyond the row).
template <int LANES, bool VEC>
struct Share {
  static __device__ __forceinline__ int col(int lane, int e) { return VEC ? lane * 8 + e : e * LANES + lane; }
  template <typename T>
  static __device__ __forceinline__ void read(const T* row, int D, int lane, float (&v)[8]) {
    if constexpr (VEC) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.f;
      if (lane * 8 < D) read8(row + lane * 8, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = col(lane, e) < D ? read1(row + col(lane, e)) : 0.f;
    }
  }
  template <typename T>
  static __device__ __forceinline__ void write(T* row, int D, int lane, const float (&v)[8]) {
    if constexpr (VEC) {
      if (lane * 8 < D) write8(row + lane * 8, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (col(lane, e) < D) write1(row + col(lane, e), v[e]);
    }
  }
};

constexpr int kScratch = 8;  // floats per use: one per wave

// Sum over the LANES threads of a row, the same value in all of them.  Rows of several waves meet in `scratch`, a slot of its own
// for every sum of a step and two sets of slots in turn, so that one barrier per sum is enough.
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* scratch) {
#pragma unroll
  for (int off = (LANES < 64 ? LANES : 64) / 2; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  if constexpr (LANES > 64) {
    constexpr int kWaves = LANES / 64;
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    const float* mine = scratch + threadIdx.x / LANES * kWaves;
    v = mine[0];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) v += mine[i];
  }
  return v;
}

template <int LANES, bool VEC>
__device__ __forceinline__ void moments(const float (&v)[8], int D, float inv_d, float eps, int lane, float* scratch, float& mean, float& rstd) {
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) s += v[e];
  mean = row_sum<LANES>(s, scratch) * inv_d;
  float q = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float d = Share<LANES, VEC>::col(lane, e) < D ? v[e] - mean : 0.f;
    q = fmaf(d, d, q);
  }
  rstd = rsqrtf(row_sum<LANES>(q, scratch + kScratch) * inv_d + eps);
}

__device__ __forceinline__ float sigmoid(float g) { return 1.0f / (1.0f + __expf(-g)); }

template <typename TX, typename TZ, int LANES, bool VEC>
__global__ __launch_bounds__(threads_of(LANES)) void resnorm_fwd_kernel(ResNormArgs a) {
  using S = Share<LANES, VEC>;
  constexpr int kRows = threads_of(LANES) / LANES;
  __shared__ float scratch[2][4 * kScratch];
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES, D = a.D;
  const float inv_d = 1.0f / (float)D;
  float sc[8], pw[8], pb[8], qw[8], qb[8];
  S::read(a.scale, D, lane, sc);
  S::read(a.post_w, D, lane, pw);
  S::read(a.post_b, D, lane, pb);
  S::read(a.pre_w, D, lane, qw);
  S::read(a.pre_b, D, lane, qb);
  int turn = 0;
  for (long long r0 = (long long)blockIdx.x * kRows; r0 < a.N; r0 += (long long)gridDim.x * kRows, turn ^= 1) {
    const long long row = r0 + group;
    const bool on = row < a.N;  // a row group behind the last row computes that one again and writes nothing
    const long long at = (on ? row : a.N - 1) * D;
    float x[8], z[8], g[8];
    S::read(reinterpret_cast<const TZ*>(a.z) + at, D, lane, z);
    S::read(reinterpret_cast<const TX*>(a.x) + at, D, lane, x);
    if (a.gate_mode == 2) S::read(reinterpret_cast<const TZ*>(a.gate) + at, D, lane, g);
    const float open_row = a.gate_mode == 1 ? sigmoid(read1(reinterpret_cast<const TZ*>(a.gate) + (on ? row : a.N - 1))) : 1.0f;
    float mean, rstd, mean_y, rstd_y;
    moments<LANES, VEC>(z, D, inv_d, a.eps, lane, scratch[turn], mean, rstd);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float n = fmaf((z[e] - mean) * rstd, pw[e], pb[e]);
      const float open = a.gate_mode == 2 ? sigmoid(g[e]) : open_row;
      x[e] = fmaf(sc[e] * open, n, x[e]);  // beyond the row: parameters and x are zero
    }
    moments<LANES, VEC>(x, D, inv_d, a.eps, lane, scratch[turn] + 2 * kScratch, mean_y, rstd_y);
    if (on) {
      S::write(reinterpret_cast<TX*>(a.y) + at, D, lane, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = fmaf((x[e] - mean_y) * rstd_y, qw[e], qb[e]);
      S::write(reinterpret_cast<TZ*>(a.h) + at, D, lane, x);
      if (a.stats && lane == 0) *reinterpret_cast<float4*>(a.stats + 4 * row) = make_float4(mean, rstd, mean_y, rstd_y);
    }
  }
}

template <typename TX, typename TZ, int LANES, bool VEC>
__global__ __launch_bounds__(threads_of(LANES)) void resnorm_bwd_kernel(ResNormArgs a) {
  using S = Share<LANES, VEC>;
  constexpr int kRows = threads_of(LANES) / LANES;
  __shared__ float scratch[2][5 * kScratch];
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES, D = a.D;
  const float inv_d = 1.0f / (float)D;
  float sc[8], pw[8], pb[8], qw[8];
  S::read(a.scale, D, lane, sc);
  S::read(a.post_w, D, lane, pw);
  S::read(a.post_b, D, lane, pb);
  S::read(a.pre_w, D, lane, qw);
  float sum[5][8];
#pragma unroll
  for (int i = 0; i < 5; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[i][e] = 0.f;
  int turn = 0;
  for (long long r0 = (long long)blockIdx.x * kRows; r0 < a.N; r0 += (long long)gridDim.x * kRows, turn ^= 1) {
    const long long row = r0 + group;
    const bool on = row < a.N;
    const long long at = (on ? row : a.N - 1) * D;
    float x[8], z[8], g[8], dy[8], dh[8];
    S::read(reinterpret_cast<const TZ*>(a.z) + at, D, lane, z);
    S::read(reinterpret_cast<const TX*>(a.x) + at, D, lane, x);
    if (a.gate_mode == 2) S::read(reinterpret_cast<const TZ*>(a.gate) + at, D, lane, g);
#pragma unroll
    for (int e = 0; e < 8; ++e) dy[e] = dh[e] = 0.f;
    if (a.dy && on) S::read(reinterpret_cast<const TX*>(a.dy) + at, D, lane, dy);
    if (a.dh && on) S::read(reinterpret_cast<const TZ*>(a.dh) + at, D, lane, dh);
    const float4 st = *reinterpret_cast<const float4*>(a.stats + 4 * (on ? row : a.N - 1));
    const float open_row = a.gate_mode == 1 ? sigmoid(read1(reinterpret_cast<const TZ*>(a.gate) + (on ? row : a.N - 1))) : 1.0f;
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool in = S::col(lane, e) < D;
      z[e] = in ? (z[e] - st.x) * st.y : 0.f;  // normalised z
      if (a.gate_mode == 2) g[e] = sigmoid(g[e]); else g[e] = open_row;
      const float y = fmaf(sc[e] * g[e], fmaf(z[e], pw[e], pb[e]), x[e]);
      x[e] = in ? (y - st.z) * st.w : 0.f;        // normalised y
      sum[4][e] += dh[e];
      sum[3][e] = fmaf(dh[e], x[e], sum[3][e]);
      dh[e] *= qw[e];
      s1 += dh[e];
      s2 = fmaf(dh[e], x[e], s2);
    }
    s1 = row_sum<LANES>(s1, scratch[turn]) * inv_d;
    s2 = row_sum<LANES>(s2, scratch[turn] + kScratch) * inv_d;
    float t1 = 0.f, t2 = 0.f, tg = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = on ? fmaf(st.w, dh[e] - s1 - x[e] * s2, dy[e]) : 0.f;  // whole gradient of y
      dy[e] = S::col(lane, e) < D ? d : 0.f;
      const float n = fmaf(z[e], pw[e], pb[e]);
      const float opened = dy[e] * g[e];
      sum[0][e] = fmaf(opened, n, sum[0][e]);
      const float dn = opened * sc[e];
      sum[2][e] += dn;
      sum[1][e] = fmaf(dn, z[e], sum[1][e]);
      g[e] = dn * n * (1.0f - g[e]);           // gradient of the gate's logit
      tg += g[e];
      x[e] = dn * pw[e];
      t1 += x[e];
      t2 = fmaf(x[e], z[e], t2);
    }
    t1 = row_sum<LANES>(t1, scratch[turn] + 2 * kScratch) * inv_d;
    t2 = row_sum<LANES>(t2, scratch[turn] + 3 * kScratch) * inv_d;
    if (a.gate_mode == 1) tg = row_sum<LANES>(tg, scratch[turn] + 4 * kScratch);
    if (!on) continue;
    S::write(reinterpret_cast<TX*>(a.dx) + at, D, lane, dy);
    if (a.gate_mode == 2) S::write(reinterpret_cast<TZ*>(a.dgate) + at, D, lane, g);
    if (a.gate_mode == 1 && lane == 0) write1(reinterpret_cast<TZ*>(a.dgate) + row, tg);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = st.y * (x[e] - t1 - z[e] * t2);
    S::write(reinterpret_cast<TZ*>(a.dz) + at, D, lane, x);
  }
  // Row groups of a wave, then the four waves, in order.
  if constexpr (LANES < 64) {
#pragma unroll
    for (int i = 0; i < 5; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int off = LANES; off < 64; off <<= 1) sum[i][e] += __shfl_xor(sum[i][e], off, 64);
  }
  float* part = a.part + (size_t)blockIdx.x * 5 * D;
  if constexpr (LANES >= 256) {
#pragma unroll
    for (int i = 0; i < 5; ++i) S::write(part + (size_t)i * D, D, lane, sum[i]);
  } else {
    constexpr int kParts = LANES < 64 ? 4 : 256 / LANES;  // waves, or row groups of several waves
    __shared__ float wave_part[4][LANES * 8];
    const int which = LANES < 64 ? threadIdx.x >> 6 : group, wl = LANES < 64 ? threadIdx.x & 63 : lane;
#pragma unroll
    for (int i = 0; i < 5; ++i) {
      __syncthreads();
      if (wl < LANES) {
#pragma unroll
        for (int e = 0; e < 8; ++e) wave_part[which][S::col(wl, e)] = sum[i][e];
      }
      __syncthreads();
      for (int k = threadIdx.x; k < D; k += 256) {
        float v = wave_part[0][k];
#pragma unroll
        for (int w = 1; w < kParts; ++w) v += wave_part[w][k];
        part[(size_t)i * D + k] = v;
      }
    }
  }
}

// dparams[k] = sum over the workgroups' partial rows: 32 columns and 32 row shares per workgroup, fixed order.
__global__ __launch_bounds__(1024) void resnorm_params_kernel(const float* part, float* out, int groups, int n) {
  __shared__ float s[32][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), share = threadIdx.x >> 5;
  float v = 0.f;
  if (col < n) {
#pragma unroll 8
    for (int r = share; r < groups; r += 32) v += part[(size_t)r * n + col];
  }
  s[share][threadIdx.x & 31] = v;
  __syncthreads();
  if (share == 0 && col < n) {
    float all = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) all += s[i][threadIdx.x];
    out[col] = all;
  }
}

template <typename TX, typename TZ, int LANES, bool VEC>
void launch(const ResNormArgs& a, bool backward, hipStream_t stream) {
  if (backward) hipLaunchKernelGGL((resnorm_bwd_kernel<TX, TZ, LANES, VEC>), dim3(a.groups), dim3(threads_of(LANES)), 0, stream, a);
  else hipLaunchKernelGGL((resnorm_fwd_kernel<TX, TZ, LANES, VEC>), dim3(a.groups), dim3(threads_of(LANES)), 0, stream, a);
}

template <typename TX, typename TZ, bool VEC>
void by_width(const ResNormArgs& a, bool backward, hipStream_t stream) {
  switch (lanes_of(a.D)) {
    case 16: return launch<TX, TZ, 16, VEC>(a, backward, stream);
    case 32: return launch<TX, TZ, 32, VEC>(a, backward, stream);
    case 64: return launch<TX, TZ, 64, VEC>(a, backward, stream);
    case 128: return launch<TX, TZ, 128, VEC>(a, backward, stream);
    case 256: return launch<TX, TZ, 256, VEC>(a, backward, stream);
    default: return launch<TX, TZ, 512, VEC>(a, backward, stream);
  }
}

int run(const ResNormArgs& a, bool backward, hipStream_t stream) {
  const bool x_bf16 = a.x_bf16 != 0, z_bf16 = a.z_bf16 != 0;
  // 16-byte accesses: widths in eights (rows then start on 16 bytes; the caller's buffers do)
  const bool vec = a.D % 8 == 0;
  if (x_bf16 && z_bf16) vec ? by_width<unsigned short, unsigned short, true>(a, backward, stream) : by_width<unsigned short, unsigned short, false>(a, backward, stream);
  else if (!x_bf16 && z_bf16) vec ? by_width<float, unsigned short, true>(a, backward, stream) : by_width<float, unsigned short, false>(a, backward, stream);
  else if (!x_bf16 && !z_bf16) vec ? by_width<float, float, true>(a, backward, stream) : by_width<float, float, false>(a, backward, stream);
  else return -12;
  return hip_err(hipGetLastError());
}

int check(const ResNormArgs& a) {
  if (a.N < 1 || a.D < 1 || a.D > 4096 || a.groups < 1) return -10;
  if (a.gate_mode < 0 || a.gate_mode > 2 || (a.gate_mode != 0) != (a.gate != nullptr)) return -11;
  if (!a.x || !a.z || !a.scale || !a.post_w || !a.post_b || !a.pre_w) return -17;
  return 0;
}

}  // namespace

extern "C" {

int atri_resnorm_fwd(const ResNormArgs* args, hipStream_t stream) {
  if (!args) return -1;
  const int rc = check(*args);
  if (rc) return rc;
  if (!args->y || !args->h || !args->pre_b) return -17;
  return run(*args, false, stream);
}

// dx, dz, dgate (every element) and dparams [5, D]: dscale, dpost_w, dpost_b, dpre_w, dpre_b.
int atri_resnorm_bwd(const ResNormArgs* args, hipStream_t stream) {
  if (!args) return -1;
  const ResNormArgs& a = *args;
  int rc = check(a);
  if (rc) return rc;
  if (!a.stats || !a.dx || !a.dz || !a.part || !a.dparams || (a.gate_mode && !a.dgate)) return -17;
  rc = run(a, true, stream);
  if (rc) return rc;
  const int n = 5 * a.D;
  hipLaunchKernelGGL(resnorm_params_kernel, dim3((n + 31) / 32), dim3(1024), 0, stream, a.part, a.dparams, a.groups, n);
  return hip_err(hipGetLastError());
}

}  // extern "C"
