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
// team of lanes owns one group of one row, 16 bytes per lane and load; the rows behind it are already on their way to
// shared memory.  Statistics cost shuffles up to 256 columns and one barrier of the team beyond.  A lane keeps its
// columns from row to row, so the weight's gradient is summed in registers and written once per block; a second kernel
// adds the blocks' parts in a fixed order.
//
// 16384 rows of 8192 in groups of 1024: forward 143 us, 5.6 TB/s (rows ahead in registers: 148 us; 3 or 5 blocks per SM
// instead of 4: 146 and 168 us).  4095 rows: backward 64 us, 5.2 TB/s (in registers: 69 us).  4096 rows of 4096 in groups
// of 128: forward 21 us, backward 32 us.
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
// 1 / (1 + e^-x) with the fast divide: a denominator above 2^126 gives 0, where the value is below 2^-126
__device__ __forceinline__ float sigm(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }

// Where a thread works: teams of L lanes own a group each; the teams of a block cover `gpw` neighbouring groups (a
// window of at most 256 U units) of `rows` rows, so that a block reads contiguous row segments.
template <int L, int U>
struct Place {
  int l, row, rows, g, phase = 0;
  bool on;                       // false: a team without a group
  int c[U];                      // first column of each unit inside the group
  bool ok[U];
  __device__ Place(const Args& a) {
    constexpr int TEAMS = 256 / L;
    const int team = threadIdx.x / L, gpw = min(a.groups, TEAMS);
    l = threadIdx.x % L, rows = TEAMS / gpw, row = team / gpw, g = blockIdx.y * gpw + team % gpw;
    on = row < rows && g < a.groups;
#pragma unroll
    for (int u = 0; u < U; ++u) c[u] = (u * L + l) * 8, ok[u] = on && c[u] < a.d;
  }
  // sum over the team; wide teams meet at a barrier of their own, two buffers take turns
  __device__ float sum(float v, float* red) {
#pragma unroll
    for (int o = (L < 32 ? L : 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (L > 32) {
      constexpr int NW = L > 32 ? L / 32 : 1;
      const int team = threadIdx.x / L;
      float* r = red + (phase & 1) * 8 + team * NW;
      ++phase;
      if ((threadIdx.x & 31) == 0) r[(threadIdx.x / 32) % NW] = v;
      asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(L) : "memory");
      v = r[0];
#pragma unroll
      for (int i = 1; i < NW; ++i) v += r[i];
    }
    return v;
  }
};

template <int L, int U>
__device__ __forceinline__ void load_weight(const Args& a, const Place<L, U>& p, float (&w)[U][8]) {
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long at = (a.w_shared ? 0 : (long long)p.g * a.d) + p.c[u];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      w[u][i] = !p.ok[u] ? 0.f : a.w_f32 ? ((const float*)a.w)[at + i] : __bfloat162float(((const bf16*)a.w)[at + i]);
  }
}
// Rows on their way: every thread copies its own 16-byte units of N tensors asynchronously into its own places in shared
// memory, DEPTH - 1 rows ahead of the one it works on, and reads them back itself: no barrier, and no registers held.
template <int N, int U>
constexpr int depth() { return U == 1 ? 4 : U == 2 ? 3 : 2; }
template <int N, int U>
constexpr int ring_bytes() { return depth<N, U>() * N * U * 256 * 16; }
template <int N, int L, int U>
struct Ring {
  static constexpr int D = depth<N, U>(), SLOT = N * U * 256 * 16;
  uint32_t base;
  int next = 0;                  // slot of the row that is read next
  __device__ explicit Ring(const uint8_t* smem) : base(xb_smem_u32(smem) + threadIdx.x * 16) {}
  __device__ void load(const Place<L, U>& p, const bf16* const (&src)[N], const long long (&ld)[N], long long t, int T, int d, int slot) {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool on = t < T && p.ok[u];
        const bf16* at = on ? src[n] + t * ld[n] + p.g * d + p.c[u] : src[n];
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(base + slot * SLOT + (n * U + u) * 4096), "l"(at), "r"(on ? 16 : 0) : "memory");
      }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // the next row's units; the row D - 1 further on sets out
  __device__ void step(const Place<L, U>& p, const bf16* const (&src)[N], const long long (&ld)[N], long long t, int T, int d, uint4 (&r)[N][U]) {
    load(p, src, ld, t, T, d, next == 0 ? D - 1 : next - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(D - 1) : "memory");
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int u = 0; u < U; ++u)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[n][u].x), "=r"(r[n][u].y), "=r"(r[n][u].z), "=r"(r[n][u].w)
                     : "r"(base + next * SLOT + (n * U + u) * 4096) : "memory");
    next = next + 1 == D ? 0 : next + 1;
  }
};

template <int L, int U, bool FIRST>
__global__ void __launch_bounds__(256, U == 1 ? 4 : 2) gated_norm_fwd(const Args a) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float red[16];
  Place<L, U> p(a);
  const long long W = (long long)a.groups * a.d, step = (long long)gridDim.x * p.rows;
  float w[U][8];
  load_weight(a, p, w);
  const float inv = 1.f / (float)a.d;
  long long t = (long long)blockIdx.x * p.rows + p.row;
  Ring<2, L, U> ring(smem);
  const bf16* const src[2] = {a.x, a.z};
  const long long ld[2] = {a.ldx, a.ldz};
#pragma unroll
  for (int i = 0; i + 1 < ring.D; ++i) ring.load(p, src, ld, t + i * step, a.T, a.d, i);
  for (long long t0 = (long long)blockIdx.x * p.rows; t0 < a.T; t0 += step, t += step) {
    uint4 r2[2][U];
    ring.step(p, src, ld, t + (ring.D - 1) * step, a.T, a.d, r2);
    const uint4(&rx)[U] = r2[0], (&rz)[U] = r2[1];
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
    const float r = rsqrtf(p.sum(ss, red) * inv + a.eps);
    if (t < a.T) {
      if (p.on && p.l == 0 && a.rstd != nullptr) a.rstd[t * a.groups + p.g] = r;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float y[8], z[8];
        if (FIRST) unpack8(rz[u], z);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = h[u][i] * r * w[u][i] * (FIRST ? z[i] * sigm(z[i]) : 1.f);
        if (p.ok[u]) *reinterpret_cast<uint4*>(a.y + t * W + p.g * a.d + p.c[u]) = pack8(y);
      }
    }
  }
}

template <int L, int U, bool FIRST>
__global__ void __launch_bounds__(256, U == 1 ? 2 : 1) gated_norm_bwd(const Args a) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float sums[U == 1 ? 2048 : 1];          // weight gradients of the block's rows
  __shared__ float red[16];
  Place<L, U> p(a);
  const long long W = (long long)a.groups * a.d, step = (long long)gridDim.x * p.rows;
  float w[U][8], dw[U][8] = {};
  load_weight(a, p, w);
  const float inv = 1.f / (float)a.d;
  long long t = (long long)blockIdx.x * p.rows + p.row;
  float nr = p.on && t < a.T ? a.rstd[t * a.groups + p.g] : 0.f;
  Ring<3, L, U> ring(smem);
  const bf16* const src[3] = {a.x, a.z, a.dy};
  const long long ld[3] = {a.ldx, a.ldz, a.lddy};
#pragma unroll
  for (int i = 0; i + 1 < ring.D; ++i) ring.load(p, src, ld, t + i * step, a.T, a.d, i);
  for (long long t0 = (long long)blockIdx.x * p.rows; t0 < a.T; t0 += step, t += step) {
    uint4 r3[3][U];
    const float r = nr;
    nr = p.on && t + step < a.T ? a.rstd[(t + step) * a.groups + p.g] : 0.f;
    ring.step(p, src, ld, t + (ring.D - 1) * step, a.T, a.d, r3);
    const uint4(&rx)[U] = r3[0], (&rz)[U] = r3[1], (&ry)[U] = r3[2];
    float sg[U][8], dot = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[8], z[8], y[8];
      unpack8(rx[u], x), unpack8(rz[u], z), unpack8(ry[u], y);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sg[u][i] = sigm(z[i]);
        const float s = z[i] * sg[u][i], f = x[i] * r * s * y[i];      // n dy s or n dy: the same product either way
        dw[u][i] += f;
        dot += f * w[u][i];
      }
    }
    const float m = p.sum(dot, red) * inv;
    if (t < a.T) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float x[8], z[8], y[8], dx[8], dz[8];
        unpack8(rx[u], x), unpack8(rz[u], z), unpack8(ry[u], y);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float s = z[i] * sg[u][i], slope = sg[u][i] * (1.f + z[i] * (1.f - sg[u][i]));
          const float n = x[i] * r * (FIRST ? 1.f : s), dn = y[i] * w[u][i] * (FIRST ? s : 1.f);
          const float dh = r * (dn - n * m);
          dx[i] = FIRST ? dh : dh * s;
          dz[i] = (FIRST ? y[i] * n * w[u][i] : dh * x[i]) * slope;
        }
        if (p.ok[u]) {
          *reinterpret_cast<uint4*>(a.dx + t * W + p.g * a.d + p.c[u]) = pack8(dx);
          *reinterpret_cast<uint4*>(a.dz + t * W + p.g * a.d + p.c[u]) = pack8(dz);
        }
      }
    }
  }
  if (a.part == nullptr) return;
  // one row of `part` per block: [gridDim.x, groups * d], or [blocks, d] where the groups share the weight
  float* out = a.w_shared ? a.part + ((long long)blockIdx.x * gridDim.y + blockIdx.y) * a.d
                          : a.part + (long long)blockIdx.x * W + (long long)p.g * a.d;
  if (U == 1) {                                      // teams meet in shared memory: those of other rows, or all
    const int gpw = min(a.groups, 256 / L), team = threadIdx.x / L;
    const int mine = a.w_shared ? 0 : team % gpw, n = a.w_shared ? 256 / L : p.rows, stride = a.w_shared ? 1 : gpw;
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[threadIdx.x * 8 + i] = dw[0][i];          // 0 in teams without a group
    __syncthreads();
    if (team != mine || p.c[0] >= a.d || (!a.w_shared && !p.on)) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float s = 0.f;
      for (int j = 0; j < n; ++j) s += sums[((mine + j * stride) * L + p.l) * 8 + i];
      out[p.c[0] + i] = s;
    }
    return;
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (p.ok[u])
#pragma unroll
      for (int i = 0; i < 8; ++i) out[p.c[u] + i] = dw[u][i];
}

// dw[c] = sum of `rows` rows of part [rows, n]: 32 columns per block, 8 threads of each share the rows
__global__ void __launch_bounds__(256) gated_norm_dw(const float* __restrict__ part, void* __restrict__ dw, int f32, int rows, int n) {
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
    if (f32) ((float*)dw)[col] = s;
    else ((bf16*)dw)[col] = __float2bfloat16(s);
  }
}

// Lanes per group: the fewest that hold it in one 16-byte unit each, up to 256; wider groups take 2 or 4 units per lane.
int lanes_of(int d) {
  int l = 8;
  while (l < 256 && l * 8 < d) l *= 2;
  return l;
}
// Blocks side by side over the groups, and enough along the rows to fill the SMs once.
dim3 grid_of(int T, int groups, int d, bool bwd) {
  const int teams = 256 / lanes_of(d), gpw = min(groups, teams), rows = teams / gpw, wy = (groups + gpw - 1) / gpw;
  const int per_sm = d <= 2048 ? (bwd ? 2 : 4) : (bwd ? 1 : 2);
  const int want = xb_sm_count() * per_sm / wy, most = (T + rows - 1) / rows;
  return dim3((unsigned)max(1, min(want, most)), (unsigned)wy);
}

template <auto KERNEL, int SMEM>
int launch(dim3 grid, const Args& a, cudaStream_t st) {
  static bool done[64] = {false};                    // dynamic shared memory above 48 KB, once per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (!done[dev & 63]) {
    if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess) {
      cudaGetLastError();
      return -5;
    }
    done[dev & 63] = true;
  }
  KERNEL<<<grid, 256, SMEM, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? 0 : -11;
}

template <bool BWD, bool FIRST>
int run(const Args& a, cudaStream_t st) {
  const dim3 grid = grid_of(a.T, a.groups, a.d, BWD);
  int rc = 0;
#define XB_RUN(L, U)                                                                                \
  do {                                                                                              \
    if (BWD) rc = launch<gated_norm_bwd<L, U, FIRST>, ring_bytes<3, U>()>(grid, a, st);             \
    else rc = launch<gated_norm_fwd<L, U, FIRST>, ring_bytes<2, U>()>(grid, a, st);                 \
  } while (0)
  switch (lanes_of(a.d)) {
    case 8: XB_RUN(8, 1); break;
    case 16: XB_RUN(16, 1); break;
    case 32: XB_RUN(32, 1); break;
    case 64: XB_RUN(64, 1); break;
    case 128: XB_RUN(128, 1); break;
    default:
      if (a.d <= 2048) XB_RUN(256, 1);
      else if (a.d <= 4096) XB_RUN(256, 2);
      else XB_RUN(256, 4);
  }
#undef XB_RUN
  return rc;
}

bool bad(const Args& a) {
  uintptr_t at = 0;
  for (const void* p : {a.x, a.z, a.dy, (const bf16*)a.y, (const bf16*)a.dx, (const bf16*)a.dz}) at |= (uintptr_t)p;
  return at % 16 || a.T < 0 || a.groups <= 0 || a.groups > 65535 || a.d <= 0 || a.d % 8 || a.d > 8192 || a.ldx % 8 || a.ldz % 8 || a.lddy % 8;
}

}  // namespace

// fp32 values of the buffer that the backward pass needs on the current device for the weight's gradient.
XB_API int xb_gated_norm_partial(int T, int groups, int d, int w_shared) {
  if (T <= 0 || groups <= 0 || d <= 0 || d % 8) return 0;
  const dim3 g = grid_of(T, groups, d, true);
  return (int)(w_shared ? g.x * g.y * d : g.x * groups * d);
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

// dw: [d] (shared weight) or [groups * d], fp32 or bf16; with part null it is not computed.  part_n: values that part holds.
XB_API int xb_gated_norm_bwd(const void* dy, long long lddy, const void* x, long long ldx, const void* z, long long ldz,
                             const void* w, int w_f32, int w_shared, const float* rstd, void* dx, void* dz, float* part,
                             long long part_n, void* dw, int dw_f32, int T, int groups, int d, int norm_first, void* stream) {
  Args a{};
  a.dy = (const bf16*)dy, a.lddy = lddy;
  a.x = (const bf16*)x, a.z = (const bf16*)z, a.ldx = ldx, a.ldz = ldz, a.w = w, a.w_f32 = w_f32, a.w_shared = w_shared;
  a.rstd = const_cast<float*>(rstd), a.dx = (bf16*)dx, a.dz = (bf16*)dz, a.part = part, a.T = T, a.groups = groups, a.d = d;
  if (bad(a) || (part != nullptr && (dw == nullptr || part_n < xb_gated_norm_partial(T, groups, d, w_shared)))) return -1;
  cudaStream_t st = (cudaStream_t)stream;
  if (T > 0) {
    const int rc = norm_first ? run<true, true>(a, st) : run<true, false>(a, st);
    if (rc) return rc;
  }
  if (part == nullptr) return 0;
  const int n = w_shared ? d : groups * d, rows = xb_gated_norm_partial(T, groups, d, w_shared) / n;
  gated_norm_dw<<<(n + 31) / 32, 256, 0, st>>>(part, dw, dw_f32, rows, n);
  return cudaGetLastError() == cudaSuccess ? 0 : -11;
}
