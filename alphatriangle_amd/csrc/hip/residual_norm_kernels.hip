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
//
// Measured: 30720 rows of 128 in fp32 with a gate per value, forward 15.5 us (5.1 TB/s), backward 30 us (4.2 TB/s) and 4 us for
// the partial rows; 491520 rows of 128, bf16 branch, forward 146 us (5.2 TB/s); 16381 rows of 2000 in bf16 with a gate per
// row, forward 58 us (4.5 TB/s), backward 123 us (3.5 TB/s with the partial rows: eight waves per CU hold its operands and
// sums in registers and meet twice per row).
// A large copy reaches 4.8 TB/s.
#include "common.hpp"
#include "encoder_ops.h"

using namespace atrihip;

namespace {

__device__ __forceinline__ float read1(const float* p) { return *p; }
__device__ __forceinline__ float read1(const unsigned short* p) { return bf16_to_float(*p); }
__device__ __forceinline__ void write1(float* p, float v) { *p = v; }
__device__ __forceinline__ void write1(unsigned short* p, float v) { *p = float_to_bf16(v); }
__device__ __forceinline__ void write8(float* p, const float* v) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void write8(unsigned short* p, const float* v) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

// A thread's share of a row as it lies in memory: 16-byte pieces (VEC) or single values, zeros beyond the row.  Rows are read into
// these one step ahead of their use, so that a workgroup always has loads under way.
template <typename T, int LANES, bool VEC>
struct Raw {
  static constexpr int kPieces = sizeof(T) / 2;  // of 16 bytes
  uint4 v[VEC ? kPieces : 1];
  T one[VEC ? 1 : 8];
  static __device__ __forceinline__ int col(int lane, int e) { return VEC ? lane * 8 + e : e * LANES + lane; }
  __device__ __forceinline__ void read(const T* row, int D, int lane) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        v[i] = make_uint4(0, 0, 0, 0);
        if (lane * 8 < D) v[i] = reinterpret_cast<const uint4*>(row + lane * 8)[i];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) one[e] = col(lane, e) < D ? row[col(lane, e)] : T(0);
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (VEC ? kPieces : 1); ++i) v[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int e = 0; e < (VEC ? 1 : 8); ++e) one[e] = T(0);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    if constexpr (VEC && sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f[4 * i] = __uint_as_float(v[i].x); f[4 * i + 1] = __uint_as_float(v[i].y);
        f[4 * i + 2] = __uint_as_float(v[i].z); f[4 * i + 3] = __uint_as_float(v[i].w);
      }
    } else if constexpr (VEC) {
      const unsigned w[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = read1(&one[e]);
    }
  }
};

template <int LANES, bool VEC>
struct Share {
  static __device__ __forceinline__ int col(int lane, int e) { return VEC ? lane * 8 + e : e * LANES + lane; }
  template <typename T>
  static __device__ __forceinline__ void read(const T* row, int D, int lane, float (&v)[8]) {
    Raw<T, LANES, VEC> r;
    r.read(row, D, lane);
    r.get(v);
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

// Sums over the LANES threads of a row, the same values in all of them.  Rows of several waves meet in `scratch` (N floats per wave):
// slots of their own for every set of sums of a step and two sets of slots in turn, so that one barrier per set is enough.
constexpr int kScratch = 8 * 3;
template <int LANES, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float* scratch) {
#pragma unroll
  for (int off = (LANES < 64 ? LANES : 64) / 2; off >= 1; off >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], off, 64);
  if constexpr (LANES > 64) {
    constexpr int kWaves = LANES / 64;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) scratch[(threadIdx.x >> 6) * N + i] = v[i];
    }
    __syncthreads();
    const float* mine = scratch + threadIdx.x / LANES * kWaves * N;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = mine[i];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) v[i] += mine[w * N + i];
    }
  }
}
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* scratch) {
  float a[1] = {v};
  row_sums<LANES>(a, scratch);
  return a[0];
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
  Raw<TX, LANES, VEC> raw_x;
  Raw<TZ, LANES, VEC> raw_z, raw_g;
  float open_next = 1.0f;
  const long long step = (long long)gridDim.x * kRows;
  // a row group behind the last row computes that one again and writes nothing
  auto fetch = [&](long long r) {
    r = r < a.N ? r : a.N - 1;
    raw_z.read(reinterpret_cast<const TZ*>(a.z) + r * D, D, lane);
    raw_x.read(reinterpret_cast<const TX*>(a.x) + r * D, D, lane);
    if (a.gate_mode == 2) raw_g.read(reinterpret_cast<const TZ*>(a.gate) + r * D, D, lane);
    if (a.gate_mode == 1) open_next = read1(reinterpret_cast<const TZ*>(a.gate) + r);
  };
  fetch((long long)blockIdx.x * kRows + group);
  int turn = 0;
  for (long long r0 = (long long)blockIdx.x * kRows; r0 < a.N; r0 += step, turn ^= 1) {
    const long long row = r0 + group;
    const bool on = row < a.N;
    const long long at = row * D;
    float x[8], z[8], g[8];
    raw_z.get(z);
    raw_x.get(x);
    if (a.gate_mode == 2) raw_g.get(g);
    const float open_row = a.gate_mode == 1 ? sigmoid(open_next) : 1.0f;
    if (r0 + step < a.N) fetch(row + step);
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
  __shared__ float scratch[2][2 * kScratch];
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
  Raw<TX, LANES, VEC> raw_x, raw_dy;
  Raw<TZ, LANES, VEC> raw_z, raw_g, raw_dh;
  float4 st_next;
  float open_next = 0.f;
  const long long step = (long long)gridDim.x * kRows;
  auto fetch = [&](long long r) {
    const bool on = r < a.N;
    r = on ? r : a.N - 1;
    raw_z.read(reinterpret_cast<const TZ*>(a.z) + r * D, D, lane);
    raw_x.read(reinterpret_cast<const TX*>(a.x) + r * D, D, lane);
    if (a.gate_mode == 2) raw_g.read(reinterpret_cast<const TZ*>(a.gate) + r * D, D, lane);
    if (a.gate_mode == 1) open_next = read1(reinterpret_cast<const TZ*>(a.gate) + r);
    raw_dy.zero();
    raw_dh.zero();
    if (a.dy && on) raw_dy.read(reinterpret_cast<const TX*>(a.dy) + r * D, D, lane);
    if (a.dh && on) raw_dh.read(reinterpret_cast<const TZ*>(a.dh) + r * D, D, lane);
    st_next = *reinterpret_cast<const float4*>(a.stats + 4 * r);
  };
  fetch((long long)blockIdx.x * kRows + group);
  int turn = 0;
  for (long long r0 = (long long)blockIdx.x * kRows; r0 < a.N; r0 += step, turn ^= 1) {
    const long long row = r0 + group;
    const bool on = row < a.N;
    const long long at = row * D;
    float x[8], z[8], g[8], dy[8], dh[8];
    raw_z.get(z);
    raw_x.get(x);
    if (a.gate_mode == 2) raw_g.get(g);
    raw_dy.get(dy);
    raw_dh.get(dh);
    const float4 st = st_next;
    const float open_row = a.gate_mode == 1 ? sigmoid(open_next) : 1.0f;
    if (r0 + step < a.N) fetch(row + step);
    float s12[2] = {0.f, 0.f};
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
      s12[0] += dh[e];
      s12[1] = fmaf(dh[e], x[e], s12[1]);
    }
    row_sums<LANES>(s12, scratch[turn]);
    const float s1 = s12[0] * inv_d, s2 = s12[1] * inv_d;
    float t12[3] = {0.f, 0.f, 0.f};
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
      t12[2] += g[e];
      x[e] = dn * pw[e];
      t12[0] += x[e];
      t12[1] = fmaf(x[e], z[e], t12[1]);
    }
    row_sums<LANES>(t12, scratch[turn] + kScratch);
    const float t1 = t12[0] * inv_d, t2 = t12[1] * inv_d;
    if (!on) continue;
    S::write(reinterpret_cast<TX*>(a.dx) + at, D, lane, dy);
    if (a.gate_mode == 2) S::write(reinterpret_cast<TZ*>(a.dgate) + at, D, lane, g);
    if (a.gate_mode == 1 && lane == 0) write1(reinterpret_cast<TZ*>(a.dgate) + row, t12[2]);
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
