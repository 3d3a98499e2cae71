// Gated linear recurrences, documents of a few tokens (single ones when a model answers): token by token, the state in
// registers (the formulas stand in recurrence.cu).
//
// What counts is the state: 64 KB read and written per head of 128 x 128, next to nothing to compute.  A CTA holds 16 KB
// of one head's state, each row segment 128 bytes; all its loads are issued before the first token, whose inputs travel
// beside them.  Products with k and q are fp32 sums over the state's rows.  With the old state S and k.q,
//
//   delta:  u = b (v - a S^T k),  o = a S^T q + (k.q) u,      scan:  o = a S^T q + (k.q) b v + D v
//
// so that one round of sums per token serves both products.
#include "recurrence_core.cuh"

namespace {

constexpr int THREADS = 128;

template <int N>
struct Row {                                   // N bf16 values, 4 or 8
  uint2 w[N / 4];
  __device__ void load(const bf16* p, bool on) {
    if (!on) {
#pragma unroll
      for (int i = 0; i < N / 4; ++i) w[i] = make_uint2(0, 0);
    } else if (N == 8) {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      w[0] = make_uint2(u.x, u.y), w[N / 4 - 1] = make_uint2(u.z, u.w);
    } else {
      w[0] = *reinterpret_cast<const uint2*>(p);
    }
  }
  __device__ void floats(float (&x)[N]) const {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const float2 a = unpack_bf16x2(w[i].x), b = unpack_bf16x2(w[i].y);
      x[4 * i] = a.x, x[4 * i + 1] = a.y, x[4 * i + 2] = b.x, x[4 * i + 3] = b.y;
    }
  }
};
__device__ __forceinline__ float4 state_load(const float* p, bool on) {
  return on ? __ldcs(reinterpret_cast<const float4*>(p)) : make_float4(0.f, 0.f, 0.f, 0.f);
}

// The delta rule: 32 columns of a head.  A thread has R neighbouring rows (16 R in all) and 4 columns; sums over the rows
// go through the warp and one exchange of the four warps.
template <int R>
__global__ void __launch_bounds__(THREADS) delta_step(const __grid_constant__ XbRecArgs p) {
  __shared__ float4 red[2][3][4][8];
  const int slices = (p.dv + NV - 1) / NV, sl = blockIdx.x % slices, h = (blockIdx.x / slices) % p.Hv, doc = blockIdx.x / (slices * p.Hv);
  const int kh = h / (p.Hv / p.Hk), cg = threadIdx.x & 7, rg = threadIdx.x >> 3, warp = threadIdx.x >> 5;
  const int col = sl * NV + cg * 4, row = rg * R;
  const int2 r = doc_range(p.cu, p.n_docs, p.T, doc);
  const int len = r.y - r.x;
  if (len > p.step) return;
  const bool vok = col < p.dv, kok = row < p.dk, first = rg == 0 && vok;
  bf16* o = (bf16*)p.o + ((long long)r.x * p.Hv + h) * p.dv + col;
  const long long o_t = (long long)p.Hv * p.dv;
  if (doc >= p.n_docs) {                       // rows outside the documents
    for (int t = 0; first && t < len; ++t) *reinterpret_cast<uint2*>(o + t * o_t) = make_uint2(0, 0);
    return;
  }
  const long long at = (((long long)doc * p.Hv + h) * p.dk + row) * p.dv + col;
  float4 s[R];
#pragma unroll
  for (int i = 0; i < R; ++i) s[i] = state_load(p.s_in + at + i * p.dv, p.s_in != nullptr && kok && vok);
  Row<R> kn, qn;
  Row<4> vn;
  float gn = 0.f, bn = 0.f;
  auto fetch = [&](int t) {
    const long long tok = r.x + t;
    kn.load((const bf16*)p.k + tok * p.k_t + kh * p.k_h + row, kok);
    qn.load((const bf16*)p.q + tok * p.q_t + kh * p.q_h + row, kok);
    vn.load((const bf16*)p.v + tok * p.v_t + h * p.v_h + col, vok);
    gn = p.g[tok * p.g_t + h * p.g_h], bn = p.b[tok * p.b_t + h * p.b_h];
  };
  if (len > 0) fetch(0);
  for (int t = 0; t < len; ++t) {
    float k[R], q[R], v[4];
    kn.floats(k), qn.floats(q), vn.floats(v);
    const float a = expf(gn), b = bn;
    if (t + 1 < len) fetch(t + 1);
    float x[12] = {};                          // k S, q S of four columns; k.k, q.q, k.q
#pragma unroll
    for (int i = 0; i < R; ++i) {
      x[0] += k[i] * s[i].x, x[1] += k[i] * s[i].y, x[2] += k[i] * s[i].z, x[3] += k[i] * s[i].w;
      x[4] += q[i] * s[i].x, x[5] += q[i] * s[i].y, x[6] += q[i] * s[i].z, x[7] += q[i] * s[i].w;
      x[8] += k[i] * k[i], x[9] += q[i] * q[i], x[10] += k[i] * q[i];
    }
#pragma unroll
    for (int i = 0; i < 11; ++i) {
      x[i] += __shfl_xor_sync(0xffffffffu, x[i], 8);
      x[i] += __shfl_xor_sync(0xffffffffu, x[i], 16);
    }
    float4(&m)[3][4][8] = red[t & 1];
    if ((threadIdx.x & 31) < 8) {
#pragma unroll
      for (int i = 0; i < 3; ++i) m[i][warp][cg] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
    }
    __syncthreads();                           // the buffer of the token before is free behind the next one
    float4 y[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const float4 c = m[i][0][cg], d = m[i][1][cg], e = m[i][2][cg], f = m[i][3][cg];
      y[i] = make_float4((c.x + d.x) + (e.x + f.x), (c.y + d.y) + (e.y + f.y), (c.z + d.z) + (e.z + f.z), (c.w + d.w) + (e.w + f.w));
    }
    const float rk = p.l2norm ? 1.f / fmaxf(sqrtf(y[2].x), 1e-12f) : 1.f, rq = p.scale * (p.l2norm ? 1.f / fmaxf(sqrtf(y[2].y), 1e-12f) : 1.f);
    const float f = a * rk, w = a * rq, kq = rk * rq * y[2].z;
    const float4 u = make_float4(b * (v[0] - f * y[0].x), b * (v[1] - f * y[0].y), b * (v[2] - f * y[0].z), b * (v[3] - f * y[0].w));
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float z = rk * k[i];
      s[i].x = a * s[i].x + z * u.x, s[i].y = a * s[i].y + z * u.y, s[i].z = a * s[i].z + z * u.z, s[i].w = a * s[i].w + z * u.w;
    }
    if (first)
      *reinterpret_cast<uint2*>(o + t * o_t) =
          make_uint2(pack_bf16x2(w * y[1].x + kq * u.x, w * y[1].y + kq * u.y), pack_bf16x2(w * y[1].z + kq * u.z, w * y[1].w + kq * u.w));
  }
  if (p.s_out != nullptr && kok && vok)
#pragma unroll
    for (int i = 0; i < R; ++i) __stcs(reinterpret_cast<float4*>(p.s_out + at + i * p.dv), s[i]);
}

// The scan: a state's rows are its columns v, contiguous in memory along k.  Eight lanes hold a row, J pieces of 32 values;
// a thread has 8 / J rows, 16 apart, and the eight lanes of a row add up its products.
template <int J>
__global__ void __launch_bounds__(THREADS) scan_step(const __grid_constant__ XbRecArgs p) {
  constexpr int R = 8 / J, ROWS = 16 * R;
  const int blocks = (p.dv + ROWS - 1) / ROWS, cb = blockIdx.x % blocks, h = (blockIdx.x / blocks) % p.Hv, doc = blockIdx.x / (blocks * p.Hv);
  const int kh = h / (p.Hv / p.Hk), cg = threadIdx.x & 7, row = cb * ROWS + (threadIdx.x >> 3);
  const int2 r = doc_range(p.cu, p.n_docs, p.T, doc);
  const int len = r.y - r.x;
  if (len > p.step) return;
  const bool state = doc < p.n_docs;
  const long long at = (((long long)doc * p.Hv + h) * p.dv + row) * p.dk + cg * 4;
  float4 s[R][J];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < J; ++j)
      s[i][j] = state_load(p.s_in + at + (long long)16 * i * p.dk + 32 * j, p.s_in != nullptr && state && row + 16 * i < p.dv && 32 * j + cg * 4 < p.dk);
  const float A = p.A[h], skip = p.D[h];
  Row<4> kn[J], qn[J];
  float vn[R], bn = 0.f;
  auto fetch = [&](int t) {
    const long long tok = r.x + t;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const bool on = 32 * j + cg * 4 < p.dk;
      kn[j].load((const bf16*)p.k + tok * p.k_t + kh * p.k_h + 32 * j + cg * 4, on);
      qn[j].load((const bf16*)p.q + tok * p.q_t + kh * p.q_h + 32 * j + cg * 4, on);
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
      vn[i] = row + 16 * i < p.dv ? __bfloat162float(((const bf16*)p.v)[tok * p.v_t + h * p.v_h + row + 16 * i]) : 0.f;
    bn = p.b[tok * p.b_t + h * p.b_h];
  };
  if (len > 0) fetch(0);
  for (int t = 0; t < len; ++t) {
    float k[J][4], q[J][4], v[R];
#pragma unroll
    for (int j = 0; j < J; ++j) kn[j].floats(k[j]), qn[j].floats(q[j]);
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = vn[i];
    const float b = bn, z = b * A, a = z < MIN_LOG ? 0.f : expf(z) * (1.f + fmaf(b, A, -z));        // the product's rounding error included
    if (t + 1 < len) fetch(t + 1);
    float x[R] = {}, kq = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
#pragma unroll
      for (int i = 0; i < R; ++i) x[i] += (q[j][0] * s[i][j].x + q[j][1] * s[i][j].y) + (q[j][2] * s[i][j].z + q[j][3] * s[i][j].w);
      kq += (k[j][0] * q[j][0] + k[j][1] * q[j][1]) + (k[j][2] * q[j][2] + k[j][3] * q[j][3]);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
#pragma unroll
      for (int i = 0; i < R; ++i) x[i] += __shfl_xor_sync(0xffffffffu, x[i], o);
      kq += __shfl_xor_sync(0xffffffffu, kq, o);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float u = b * v[i];
#pragma unroll
      for (int j = 0; j < J; ++j)
        s[i][j] = make_float4(a * s[i][j].x + u * k[j][0], a * s[i][j].y + u * k[j][1], a * s[i][j].z + u * k[j][2], a * s[i][j].w + u * k[j][3]);
      if (cg == 0 && row + 16 * i < p.dv)
        ((bf16*)p.o)[((long long)(r.x + t) * p.Hv + h) * p.dv + row + 16 * i] = __float2bfloat16(a * x[i] + kq * u + skip * v[i]);
    }
  }
  if (p.s_out != nullptr && state)
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (row + 16 * i < p.dv && 32 * j + cg * 4 < p.dk) __stcs(reinterpret_cast<float4*>(p.s_out + at + (long long)16 * i * p.dk + 32 * j), s[i][j]);
}

template <int J>
int scan(const XbRecArgs& a, cudaStream_t st) {
  constexpr int ROWS = 128 / J;
  return rec_launch(scan_step<J>, (long long)(a.n_docs + 2) * a.Hv * ((a.dv + ROWS - 1) / ROWS), THREADS, 0, a, st);
}

}  // namespace

int xb_recurrence_step(const XbRecArgs& a, int delta, cudaStream_t st) {
  if (!delta) return a.dk <= 32 ? scan<1>(a, st) : a.dk <= 64 ? scan<2>(a, st) : scan<4>(a, st);
  const long long blocks = (long long)(a.n_docs + 2) * a.Hv * ((a.dv + NV - 1) / NV);
  return a.dk <= 64 ? rec_launch(delta_step<4>, blocks, THREADS, 0, a, st) : rec_launch(delta_step<8>, blocks, THREADS, 0, a, st);
}
