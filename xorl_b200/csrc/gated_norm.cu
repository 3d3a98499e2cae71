// RMS norm over column groups, fused with the SiLU gate that stands before it (Mamba2) or behind it (GatedDeltaNet):
//
//   norm first:  y = x r w silu(z),   r = rsqrt(mean x^2 + eps) over the group
//   gate first:  h = x silu(z),  y = h r w,  r = rsqrt(mean h^2 + eps)
//
// Backward, with n = x r (or h r), s = silu(z), s' its slope:
//   norm first:  dn = dy w s,  dx = r (dn - n mean(dn n)),  dz = dy n w s',  dw = sum dy n s
//   gate first:  dn = dy w,    dh = r (dn - n mean(dn n)),  dx = dh s,  dz = dh x s',  dw = sum dy n
//
// Memory-bound: forward reads x and z and writes y, backward reads x, z and dy and writes dx and dz, each once.  A
// team of lanes owns one group of one row in registers, 16 bytes per lane and load (up to 64 bytes of each input in
// flight per lane), so the statistics cost shuffles only up to 1024 columns; wider groups add up through shared
// memory.  A lane keeps its columns from row to row, so the weight's gradient is summed in registers and written once
// per block; a second kernel adds the blocks' parts in a fixed order.
#include "common.cuh"

namespace {

using bf16 = __nv_bfloat16;

struct Args {
  const bf16 *x, *z, *dy;
  long long ldx, ldz, lddy;
  const void* w;
  float* rstd;                // [T, groups]
  bf16 *y, *dx, *dz;          // contiguous [T, groups * d]
  float* part;                // [gridDim.x, groups * d]
  int T, groups, d, w_f32, w_shared;
  float eps;
};

__device__ __forceinline__ void unpack8(const uint4 u, float (&v)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = unpack_bf16x2(w[j]);
    v[2 * j] = f.x, v[2 * j + 1] = f.y;
  }
}
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ float sigm(float x) { return 1.f / (1.f + __expf(-x)); }

// sum over the LG lanes of a team, or over all NW warps of a block (WIDE)
template <int LG, bool WIDE>
__device__ __forceinline__ float team_sum(float v, float* red, int& phase) {
#pragma unroll
  for (int o = LG / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (WIDE) {
    const int w = threadIdx.x >> 5, nw = blockDim.x >> 5;
    float* r = red + (phase & 1) * 32;       // two buffers: one barrier per sum
    ++phase;
    if ((threadIdx.x & 31) == 0) r[w] = v;
    __syncthreads();
    v = 0.f;
    for (int i = 0; i < nw; ++i) v += r[i];
  }
  return v;
}

template <int U>
__device__ __forceinline__ void load_weight(const Args& a, int g, const int (&c)[U], const bool (&ok)[U], float (&w)[U][8]) {
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long at = (a.w_shared ? 0 : (long long)g * a.d) + c[u];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      w[u][i] = !ok[u] ? 0.f : a.w_f32 ? ((const float*)a.w)[at + i] : __bfloat162float(((const bf16*)a.w)[at + i]);
  }
}

// LG lanes per group (WIDE: the whole block), U 16-byte units per lane
template <int LG, int U, bool WIDE, bool FIRST>
__global__ void __launch_bounds__(256) gated_norm_fwd(const Args a) {
  __shared__ float red[64];
  int phase = 0;
  const int lanes = WIDE ? blockDim.x : LG, team = WIDE ? 0 : threadIdx.x / LG, teams = WIDE ? 1 : blockDim.x / LG;
  const int l = threadIdx.x % lanes, g = blockIdx.y, W = a.groups * a.d;
  int c[U];
  bool ok[U];
#pragma unroll
  for (int u = 0; u < U; ++u) c[u] = (u * lanes + l) * 8, ok[u] = c[u] < a.d;
  float w[U][8];
  load_weight<U>(a, g, c, ok, w);
  const float inv = 1.f / (float)a.d;
  for (long long t0 = (long long)blockIdx.x * teams; t0 < a.T; t0 += (long long)gridDim.x * teams) {
    const long long t = t0 + team;
    const bool row = t < a.T;                        // all lanes take part in the sums
    uint4 rx[U], rz[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      rx[u] = rz[u] = make_uint4(0, 0, 0, 0);
      if (row && ok[u]) {
        rx[u] = *reinterpret_cast<const uint4*>(a.x + t * a.ldx + g * a.d + c[u]);
        rz[u] = *reinterpret_cast<const uint4*>(a.z + t * a.ldz + g * a.d + c[u]);
      }
    }
    float h[U][8], ss = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      unpack8(rx[u], h[u]);
      if (!FIRST) {
        float z[8];
        unpack8(rz[u], z);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[u][i] *= z[i] * sigm(z[i]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += h[u][i] * h[u][i];
    }
    const float r = rsqrtf(team_sum<LG, WIDE>(ss, red, phase) * inv + a.eps);
    if (!row) continue;
    if (l == 0 && a.rstd != nullptr) a.rstd[t * a.groups + g] = r;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float y[8], z[8];
      if (FIRST) unpack8(rz[u], z);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = h[u][i] * r * w[u][i] * (FIRST ? z[i] * sigm(z[i]) : 1.f);
      if (ok[u]) *reinterpret_cast<uint4*>(a.y + t * W + g * a.d + c[u]) = pack8(y);
    }
  }
}

template <int LG, int U, bool WIDE, bool FIRST>
__global__ void __launch_bounds__(256) gated_norm_bwd(const Args a) {
  extern __shared__ float sums[];                    // teams x d, for the weight's gradient
  __shared__ float red[64];
  int phase = 0;
  const int lanes = WIDE ? blockDim.x : LG, team = WIDE ? 0 : threadIdx.x / LG, teams = WIDE ? 1 : blockDim.x / LG;
  const int l = threadIdx.x % lanes, g = blockIdx.y, W = a.groups * a.d;
  int c[U];
  bool ok[U];
#pragma unroll
  for (int u = 0; u < U; ++u) c[u] = (u * lanes + l) * 8, ok[u] = c[u] < a.d;
  float w[U][8], dw[U][8] = {};
  load_weight<U>(a, g, c, ok, w);
  const float inv = 1.f / (float)a.d;
  for (long long t0 = (long long)blockIdx.x * teams; t0 < a.T; t0 += (long long)gridDim.x * teams) {
    const long long t = t0 + team;
    const bool row = t < a.T;
    uint4 rx[U], rz[U], ry[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      rx[u] = rz[u] = ry[u] = make_uint4(0, 0, 0, 0);
      if (row && ok[u]) {
        rx[u] = *reinterpret_cast<const uint4*>(a.x + t * a.ldx + g * a.d + c[u]);
        rz[u] = *reinterpret_cast<const uint4*>(a.z + t * a.ldz + g * a.d + c[u]);
        ry[u] = *reinterpret_cast<const uint4*>(a.dy + t * a.lddy + g * a.d + c[u]);
      }
    }
    const float r = row ? a.rstd[t * a.groups + g] : 0.f;
    float n[U][8], dn[U][8], dot = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[8], z[8], y[8];
      unpack8(rx[u], x), unpack8(rz[u], z), unpack8(ry[u], y);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float s = z[i] * sigm(z[i]);
        n[u][i] = x[i] * r * (FIRST ? 1.f : s);
        dn[u][i] = y[i] * w[u][i] * (FIRST ? s : 1.f);
        dw[u][i] += y[i] * n[u][i] * (FIRST ? s : 1.f);
        dot += dn[u][i] * n[u][i];
      }
    }
    const float m = team_sum<LG, WIDE>(dot, red, phase) * inv;
    if (!row) continue;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[8], z[8], y[8], dx[8], dz[8];
      unpack8(rx[u], x), unpack8(rz[u], z), unpack8(ry[u], y);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float sg = sigm(z[i]), s = z[i] * sg, slope = sg * (1.f + z[i] * (1.f - sg));
        const float dh = r * (dn[u][i] - n[u][i] * m);
        dx[i] = FIRST ? dh : dh * s;
        dz[i] = (FIRST ? y[i] * n[u][i] * w[u][i] : dh * x[i]) * slope;
      }
      if (ok[u]) {
        *reinterpret_cast<uint4*>(a.dx + t * W + g * a.d + c[u]) = pack8(dx);
        *reinterpret_cast<uint4*>(a.dz + t * W + g * a.d + c[u]) = pack8(dz);
      }
    }
  }
  if (a.part == nullptr) return;
  float* out = a.part + (long long)blockIdx.x * W + g * a.d;
  if (teams == 1) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (ok[u])
#pragma unroll
        for (int i = 0; i < 8; ++i) out[c[u] + i] = dw[u][i];
    return;
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (ok[u])
#pragma unroll
      for (int i = 0; i < 8; ++i) sums[team * a.d + c[u] + i] = dw[u][i];
  __syncthreads();
  for (int i = threadIdx.x; i < a.d; i += blockDim.x) {
    float s = 0.f;
    for (int j = 0; j < teams; ++j) s += sums[j * a.d + i];
    out[i] = s;
  }
}

// dw[c] = sum of `rows` rows of part [rows, n]: 32 columns per block, 8 threads of each share the rows
__global__ void __launch_bounds__(256) gated_norm_dw(const float* __restrict__ part, float* __restrict__ dw, int rows, int n) {
  __shared__ float red[8][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), k = threadIdx.x >> 5;
  float s = 0.f;
  if (col < n)
    for (int r = k; r < rows; r += 8) s += part[(long long)r * n + col];
  red[k][threadIdx.x & 31] = s;
  __syncthreads();
  if (k == 0 && col < n) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += red[i][threadIdx.x];
    dw[col] = s;
  }
}

// Rows that a block walks: enough blocks for `per_sm` of 256 threads on every SM, no more than there are rows.
dim3 grid_of(int T, int groups, int teams, int per_sm) {
  const int want = (xb_sm_count() * per_sm + groups - 1) / groups, most = (T + teams - 1) / teams;
  return dim3((unsigned)max(1, min(want, most)), (unsigned)groups);
}

struct Shape { int lanes, units, threads; bool wide; };
// Narrow groups: the fewest lanes that hold a group in one 16-byte unit each; from 512 columns a warp with 2, then 4
// units; wider ones a block of warps with 4 units per lane.
Shape shape_of(int d) {
  const int units = d / 8;
  if (units <= 8) return {8, 1, 256, false};
  if (units <= 16) return {16, 1, 256, false};
  if (units <= 32) return {32, 1, 256, false};
  if (units <= 64) return {32, 2, 256, false};
  if (units <= 128) return {32, 4, 256, false};
  return {32, 4, (units + 127) / 128 * 32, true};
}

template <bool BWD, bool FIRST>
int run(const Args& a, cudaStream_t st) {
  const Shape s = shape_of(a.d);
  const int teams = s.wide ? 1 : s.threads / s.lanes;
  const dim3 grid = grid_of(a.T, a.groups, teams, BWD ? 4 : 8);
  const size_t smem = BWD && a.part != nullptr && teams > 1 ? (size_t)teams * a.d * 4 : 0;
#define XB_RUN(L, U, WD)                                                        \
  do {                                                                          \
    if (BWD) gated_norm_bwd<L, U, WD, FIRST><<<grid, s.threads, smem, st>>>(a); \
    else gated_norm_fwd<L, U, WD, FIRST><<<grid, s.threads, 0, st>>>(a);        \
  } while (0)
  if (s.wide) XB_RUN(32, 4, true);
  else if (s.units == 4) XB_RUN(32, 4, false);
  else if (s.units == 2) XB_RUN(32, 2, false);
  else if (s.lanes == 32) XB_RUN(32, 1, false);
  else if (s.lanes == 16) XB_RUN(16, 1, false);
  else XB_RUN(8, 1, false);
#undef XB_RUN
  return cudaGetLastError() == cudaSuccess ? 0 : -11;
}

bool bad(const Args& a) {
  return a.T < 0 || a.groups <= 0 || a.groups > 65535 || a.d <= 0 || a.d % 8 || a.d > 8192 || a.ldx % 8 || a.ldz % 8 || a.lddy % 8;
}

}  // namespace

// Rows of the buffer that the backward pass needs for the weight's gradient.
XB_API int xb_gated_norm_partial_rows(int T, int groups, int d) {
  if (T <= 0 || groups <= 0 || d <= 0 || d % 8) return 0;
  const Shape s = shape_of(d);
  return (int)grid_of(T, groups, s.wide ? 1 : s.threads / s.lanes, 4).x;
}

XB_API int xb_gated_norm_fwd(const void* x, long long ldx, const void* z, long long ldz, const void* w, int w_f32,
                             int w_shared, void* y, float* rstd, int T, int groups, int d, float eps, int norm_first,
                             void* stream) {
  Args a{};
  a.x = (const bf16*)x, a.z = (const bf16*)z, a.ldx = ldx, a.ldz = ldz, a.w = w, a.w_f32 = w_f32, a.w_shared = w_shared;
  a.y = (bf16*)y, a.rstd = rstd, a.T = T, a.groups = groups, a.d = d, a.eps = eps;
  if (bad(a)) return -1;
  if (T == 0) return 0;
  return norm_first ? run<false, true>(a, (cudaStream_t)stream) : run<false, false>(a, (cudaStream_t)stream);
}

// dw: fp32 [d] (shared weight) or [groups * d]; with part null it is not computed.
XB_API int xb_gated_norm_bwd(const void* dy, long long lddy, const void* x, long long ldx, const void* z, long long ldz,
                             const void* w, int w_f32, int w_shared, const float* rstd, void* dx, void* dz, float* part,
                             float* dw, int T, int groups, int d, int norm_first, void* stream) {
  Args a{};
  a.dy = (const bf16*)dy, a.lddy = lddy;
  a.x = (const bf16*)x, a.z = (const bf16*)z, a.ldx = ldx, a.ldz = ldz, a.w = w, a.w_f32 = w_f32, a.w_shared = w_shared;
  a.rstd = const_cast<float*>(rstd), a.dx = (bf16*)dx, a.dz = (bf16*)dz, a.part = part, a.T = T, a.groups = groups, a.d = d;
  if (bad(a) || (part != nullptr && dw == nullptr)) return -1;
  cudaStream_t st = (cudaStream_t)stream;
  if (T > 0) {
    const int rc = norm_first ? run<true, true>(a, st) : run<true, false>(a, st);
    if (rc) return rc;
  }
  if (part == nullptr) return 0;
  const int rows = xb_gated_norm_partial_rows(T, groups, d) * (w_shared ? groups : 1), n = w_shared ? d : groups * d;
  gated_norm_dw<<<(n + 31) / 32, 256, 0, st>>>(part, dw, rows, n);
  return cudaGetLastError() == cudaSuccess ? 0 : -11;
}
