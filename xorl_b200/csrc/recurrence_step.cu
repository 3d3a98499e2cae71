// Gated linear recurrences, documents of a few tokens, down to single ones whose states come from the call before: token by
// token, the state in registers (the formulas stand in recurrence.cu).  Forward only: a backward pass works on chunks.
//
// What counts is the state: 64 KB read and written per head of 128 x 128, next to nothing to compute.  A CTA holds 16 KB
// of one head's state, each row segment 128 bytes; all its loads, and those of the document's inputs, are issued before the
// first token.  Products with k and q are fp32 sums over the state's rows.  With the old state S and k.q,
//
//   delta:  u = b (v - a S^T k),  o = a S^T q + (k.q) u,      scan:  o = a S^T q + (k.q) b v + D v
//
// so that one round of sums per token serves both products.
//
// 48 documents of one token, 32 heads of 128 x 128 (201 MB): 35 us, 5.7 TB/s; 200 documents: 131 us, 6.4 TB/s.  Scan, 48
// documents, 128 heads of 64 x 128 (403 MB): 64 us, 6.3 TB/s (L2 full of other data to be written back: 38, 140 and 70 us).
// Further tokens cost about 8 and 14 us each; their inputs come from shared memory, since one at a time from global memory
// each cost another 7 and 12 us.  At 16 tokens the chunked kernels take about as long: 48 documents of 16, delta rule 150 us
// (chunks: 222), scan 279 us (chunks: 339), with 45 and 59 us for chunked kernels that find nothing to do.
#include "recurrence_core.cuh"

namespace {

constexpr int THREADS = 128;

constexpr int MAX_STEP = 16;                    // tokens whose inputs fit the shared memory

// The inputs of a document's tokens, 16 bytes per copy: rows of at most 128 bf16 values of k, q and of the CTA's columns of v
struct Inputs {
  uint4 k[MAX_STEP][16], q[MAX_STEP][16], v[MAX_STEP][16];
  float g[MAX_STEP], b[MAX_STEP];
};
__device__ __forceinline__ void fetch(const XbRecArgs& p, Inputs& in, int t0, int len, int h, int kh, int v0, int cols) {
  const int ku = p.dk / 8, vu = min(cols, p.dv - v0) / 8;
  for (int i = threadIdx.x; i < len * ku; i += THREADS) {
    const long long tok = t0 + i / ku;
    const int u = i % ku;
    cp16(xb_smem_u32(&in.k[i / ku][u]), (const bf16*)p.k + tok * p.k_t + kh * p.k_h + u * 8, true);
    cp16(xb_smem_u32(&in.q[i / ku][u]), (const bf16*)p.q + tok * p.q_t + kh * p.q_h + u * 8, true);
  }
  for (int i = threadIdx.x; i < len * vu; i += THREADS)
    cp16(xb_smem_u32(&in.v[i / vu][i % vu]), (const bf16*)p.v + (t0 + i / vu) * p.v_t + h * p.v_h + v0 + (i % vu) * 8, true);
  cp_commit();
  if (threadIdx.x < len) {
    const long long tok = t0 + threadIdx.x;
    if (p.g != nullptr) in.g[threadIdx.x] = p.g[tok * p.g_t + h * p.g_h];
    in.b[threadIdx.x] = p.b[tok * p.b_t + h * p.b_h];
  }
}
template <int N>                               // N bf16 values, 4 or 8
__device__ __forceinline__ void unpack(const uint4* row, int at, bool on, float (&x)[N]) {
  const uint32_t* src = reinterpret_cast<const uint32_t*>(row) + at / 2;
  uint32_t w[N / 2] = {};
  if (on) {
    if (N == 8) {
      const uint4 u = *reinterpret_cast<const uint4*>(src);
      w[0] = u.x, w[1] = u.y, w[N / 2 - 2] = u.z, w[N / 2 - 1] = u.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(src);
      w[0] = u.x, w[1] = u.y;
    }
  }
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const float2 f = unpack_bf16x2(w[i]);
    x[2 * i] = f.x, x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ float4 state_load(const float* p, bool on) {
  return on ? __ldcs(reinterpret_cast<const float4*>(p)) : make_float4(0.f, 0.f, 0.f, 0.f);
}

// The delta rule: 32 columns of a head.  A thread has R neighbouring rows (16 R in all) and 4 columns; sums over the rows
// go through the warp and one exchange of the four warps.
template <int R>
__global__ void __launch_bounds__(THREADS, 7) delta_step(const __grid_constant__ XbRecArgs p) {
  __shared__ Inputs in;
  __shared__ float4 red[2][2][4][8];
  __shared__ float norm[MAX_STEP][3];          // factors of k and q, and the product of the scaled rows
  const int slices = (p.dv + NV - 1) / NV, sl = blockIdx.x % slices, h = (blockIdx.x / slices) % p.Hv, doc = blockIdx.x / (slices * p.Hv);
  const int kh = h / (p.Hv / p.Hk), cg = threadIdx.x & 7, rg = threadIdx.x >> 3, warp = threadIdx.x >> 5;
  const int col = sl * NV + cg * 4, row = rg * R;
  const int2 r = doc_range(p.cu, p.n_docs, p.T, doc);
  const int len = r.y - r.x;
  if (sl == 0 && h == 0 && threadIdx.x == 0 && bad_bounds(p.cu, p.n_docs, p.T, doc)) xb_report(p.status, XB_ERR_BAD_ARG, XB_K_RECURRENCE, doc);
  if (len > p.step) return;
  const bool vok = col < p.dv, kok = row < p.dk, first = rg == 0 && vok;
  bf16* o = (bf16*)p.o + ((long long)r.x * p.Hv + h) * p.dv + col;
  const long long o_t = (long long)p.Hv * p.dv;
  if (doc >= p.n_docs) {                       // rows outside the documents
    for (int t = 0; first && t < len; ++t) *reinterpret_cast<uint2*>(o + t * o_t) = make_uint2(0, 0);
    return;
  }
  fetch(p, in, r.x, len, h, kh, sl * NV, NV);
  const long long at = (((long long)doc * p.Hv + h) * p.dk + row) * p.dv + col;
  float4 s[R];
#pragma unroll
  for (int i = 0; i < R; ++i) s[i] = state_load(p.s_in + at + i * p.dv, p.s_in != nullptr && kok && vok);
  cp_wait<0>();
  __syncthreads();
  for (int t = warp; t < len; t += THREADS / 32) {
    float k[4], q[4], kk = 0.f, qq = 0.f, kq = 0.f;
    const int lane = threadIdx.x & 31;
    unpack<4>(in.k[t], lane * 4, lane * 4 < p.dk, k), unpack<4>(in.q[t], lane * 4, lane * 4 < p.dk, q);
#pragma unroll
    for (int i = 0; i < 4; ++i) kk += k[i] * k[i], qq += q[i] * q[i], kq += k[i] * q[i];
    kk = warp_sum(kk), qq = warp_sum(qq), kq = warp_sum(kq);
    const float rk = p.l2norm ? 1.f / fmaxf(sqrtf(kk), 1e-12f) : 1.f, rq = p.scale * (p.l2norm ? 1.f / fmaxf(sqrtf(qq), 1e-12f) : 1.f);
    if (lane == 0) norm[t][0] = rk, norm[t][1] = rq, norm[t][2] = rk * rq * kq;
  }
  __syncthreads();
  const int b3 = (threadIdx.x >> 3) & 1, b4 = (threadIdx.x >> 4) & 1;
  for (int t = 0; t < len; ++t) {
    float k[R], q[R], v[4];
    unpack<R>(in.k[t], row, kok, k), unpack<R>(in.q[t], row, kok, q), unpack<4>(in.v[t], cg * 4, vok, v);
    const float a = expf(in.g[t]), b = in.b[t];
    float x[8] = {};                           // k S, q S of four columns
#pragma unroll
    for (int i = 0; i < R; ++i) {
      x[0] += k[i] * s[i].x, x[1] += k[i] * s[i].y, x[2] += k[i] * s[i].z, x[3] += k[i] * s[i].w;
      x[4] += q[i] * s[i].x, x[5] += q[i] * s[i].y, x[6] += q[i] * s[i].z, x[7] += q[i] * s[i].w;
    }
    // over the warp's four row groups: each keeps two of the eight sums
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float mine = b3 ? x[4 + i] : x[i], other = b3 ? x[i] : x[4 + i];
      x[i] = mine + __shfl_xor_sync(0xffffffffu, other, 8);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float mine = b4 ? x[2 + i] : x[i], other = b4 ? x[i] : x[2 + i];
      x[i] = mine + __shfl_xor_sync(0xffffffffu, other, 16);
    }
    float4(&m)[2][4][8] = red[t & 1];
    reinterpret_cast<float2*>(&m[b3][warp][cg])[b4] = make_float2(x[0], x[1]);
    __syncthreads();                           // the buffer of the token before is free behind the next one
    float4 y[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 c = m[i][0][cg], d = m[i][1][cg], e = m[i][2][cg], f = m[i][3][cg];
      y[i] = make_float4((c.x + d.x) + (e.x + f.x), (c.y + d.y) + (e.y + f.y), (c.z + d.z) + (e.z + f.z), (c.w + d.w) + (e.w + f.w));
    }
    const float rk = norm[t][0], f = a * rk, w = a * norm[t][1], kq = norm[t][2];
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
__global__ void __launch_bounds__(THREADS, 5) scan_step(const __grid_constant__ XbRecArgs p) {
  constexpr int R = 8 / J, ROWS = 16 * R;
  const int blocks = (p.dv + ROWS - 1) / ROWS, cb = blockIdx.x % blocks, h = (blockIdx.x / blocks) % p.Hv, doc = blockIdx.x / (blocks * p.Hv);
  const int kh = h / (p.Hv / p.Hk), cg = threadIdx.x & 7, row = cb * ROWS + (threadIdx.x >> 3);
  const int2 r = doc_range(p.cu, p.n_docs, p.T, doc);
  const int len = r.y - r.x;
  if (cb == 0 && h == 0 && threadIdx.x == 0 && bad_bounds(p.cu, p.n_docs, p.T, doc)) xb_report(p.status, XB_ERR_BAD_ARG, XB_K_RECURRENCE, doc);
  if (len > p.step) return;
  const bool state = doc < p.n_docs;
  __shared__ Inputs in;
  fetch(p, in, r.x, len, h, kh, cb * ROWS, ROWS);
  const long long at = (((long long)doc * p.Hv + h) * p.dv + row) * p.dk + cg * 4;
  float4 s[R][J];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < J; ++j)
      s[i][j] = state_load(p.s_in + at + (long long)16 * i * p.dk + 32 * j, p.s_in != nullptr && state && row + 16 * i < p.dv && 32 * j + cg * 4 < p.dk);
  const float A = p.A[h], skip = p.D[h];
  cp_wait<0>();
  __syncthreads();
  for (int t = 0; t < len; ++t) {
    float k[J][4], q[J][4], v[R];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const bool on = 32 * j + cg * 4 < p.dk;
      unpack<4>(in.k[t], 32 * j + cg * 4, on, k[j]), unpack<4>(in.q[t], 32 * j + cg * 4, on, q[j]);
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
      v[i] = row + 16 * i < p.dv ? __bfloat162float(reinterpret_cast<const bf16*>(in.v[t])[(threadIdx.x >> 3) + 16 * i]) : 0.f;
    const float b = in.b[t], z = b * A, a = z < MIN_LOG ? 0.f : expf(z) * (1.f + fmaf(b, A, -z));        // the product's rounding error included
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
  if (a.step > MAX_STEP) return -1;
  if (!delta) return a.dk <= 32 ? scan<1>(a, st) : a.dk <= 64 ? scan<2>(a, st) : scan<4>(a, st);
  const long long blocks = (long long)(a.n_docs + 2) * a.Hv * ((a.dv + NV - 1) / NV);
  return a.dk <= 64 ? rec_launch(delta_step<4>, blocks, THREADS, 0, a, st) : rec_launch(delta_step<8>, blocks, THREADS, 0, a, st);
}
