// Gated linear recurrences over packed documents, forward and backward: the gated delta rule (GatedDeltaNet)
// and the state-space scan with a scalar decay per head (Mamba2).
//
//   delta:  S_t = a_t S_{t-1} + k_t (x) u_t,  u_t = b_t (v_t - (a_t S_{t-1})^T k_t),  o_t = S_t^T q_t
//   scan:   S_t = a_t S_{t-1} + k_t (x) u_t,  u_t = b_t v_t,                          o_t = S_t^T q_t + D v_t
//
// (scan: q = C, k = B, v = x, b = dt, log a = dt A.)  S is [dk, dv] per head; q / k heads are shared by groups of v heads.
// A document is cut into chunks of 64 tokens.  With G the running sum of log a inside a chunk, gamma = e^G,
// D_ij = e^{G_i - G_j} for j <= i, d_j = e^{G_last - G_j}, and S the state that enters the chunk:
//
//   L = diag(b) tril(D o K K^T, -1),  T = (I + L)^-1,  R = diag(b) (V - diag(gamma) K S),  U = T R     (scan: U = diag(b) V)
//   O = diag(gamma) Q S + tril(D o Q K^T) U,     S' = gamma_last S + K^T diag(d) U
//
// and backwards, from dS' and dO, with P = tril(D o Q K^T):
//
//   dU = P^T dO + diag(d) K dS',  dR = T^T dU,  dV = diag(b) dR,
//   dS = gamma_last dS' + Q^T diag(gamma) dO - K^T diag(b gamma) dR
//   dP = dO U^T,  dL = -dR U^T (strictly below the diagonal),  Z = D o dP,  W = diag(b) (D o dL)
//   dQ = diag(gamma) dO S^T + Z K,   dK = -diag(b gamma) dR S^T + W K + W^T K + Z^T Q + diag(d) U dS'^T
//
// The gradient of G_i is the sum of q.dq and k.dk over the places where row i carries e^{G_i}, minus those where it
// carries e^{-G_i}; the gradient of log a_t is its suffix sum inside the chunk.
//
// Precision: q, k, v and dO are bf16 and enter the products as they are.  Whatever is computed (states, T, U, P and
// their gradients) is kept in 32 bits and enters a product as the sum of two bf16 values, which keeps 17 bits of its
// significand: one bf16 value (9 bits) would cost the fp32 gradients of the decay three decimal digits.  Products of
// two such sums leave out low x low.  Decays are sums in fp64 of log2 units, kept as two floats, so that differences
// of large sums stay exact.  L2 norms of q and k are row factors and are applied behind the products.
#include "recurrence_core.cuh"

namespace {

// ---- plan: chunks of the documents -----------------------------------------------------------------------------
// Documents 0 .. n-1 lie between the boundaries; n is the tail behind the last boundary, n + 1 the rows before the first.
__device__ __forceinline__ int2 doc_range(const int* cu, int n, int T, int d) {
  auto cut = [&](int i) { return min(max(cu[i], 0), T); };
  if (d == n) return make_int2(cut(n), T);
  if (d == n + 1) return make_int2(0, cut(0));
  const int s = cut(d);
  return make_int2(s, max(s, cut(d + 1)));
}

__global__ void __launch_bounds__(1024) rec_plan(const int* __restrict__ cu, int n, int T, int nc_max, int4* chunks,
                                                 int* doc_off, int* status) {
  __shared__ int warp_tot[32];
  __shared__ int carry;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, nd = n + 2;
  if (tid == 0) carry = 0, doc_off[0] = 0;
  __syncthreads();
  for (int base = 0; base < nd; base += 1024) {
    const int d = base + tid;
    int v = 0;
    if (d < nd) {
      const int2 r = doc_range(cu, n, T, d);
      v = (r.y - r.x + C - 1) / C;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    if (lane == 31) warp_tot[w] = v;
    __syncthreads();
    if (w == 0) {
      int t = warp_tot[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, t, o);
        if (lane >= o) t += u;
      }
      warp_tot[lane] = t;
    }
    __syncthreads();
    const int incl = carry + v + (w ? warp_tot[w - 1] : 0);
    // boundaries that overlap would need more chunks than the rows have: what does not fit is left out and reported
    if (d < nd) {
      doc_off[d + 1] = min(incl, nc_max);
      if (incl > nc_max) xb_report(status, XB_ERR_BAD_ARG, XB_K_RECURRENCE, d);
    }
    __syncthreads();
    if (tid == 0) carry += warp_tot[31];
    __syncthreads();
  }
  const int total = doc_off[nd];
  for (int c = tid; c < total; c += 1024) {
    int lo = 0, hi = nd;                                     // doc_off[lo] <= c < doc_off[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (doc_off[mid] <= c) lo = mid; else hi = mid;
    }
    const int2 r = doc_range(cu, n, T, lo);
    const int s = r.x + (c - doc_off[lo]) * C;
    chunks[c] = make_int4(s, min(C, r.y - s), lo, 0);
  }
}

// ---- prepare: what depends on one chunk alone --------------------------------------------------------------------
template <int DKP, bool DELTA>
struct PrepSmem {
  uint8_t q[C * DKP * 2], k[C * DKP * 2];
  float kk[DELTA ? C * C : 4];
  float l[DELTA ? 2 : 1][DELTA ? C * C : 4];
  float ghi[2][C], glo[2][C], b[2][C], rq[C], rk[C];
};

template <int DKP, bool DELTA>
__global__ void __launch_bounds__(128) rec_prep(const XbRecArgs p) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  PrepSmem<DKP, DELTA>& sm = *reinterpret_cast<PrepSmem<DKP, DELTA>*>(smem_raw);
  constexpr int U = DKP / 8;
  const int kh = blockIdx.x % p.Hk, c = blockIdx.x / p.Hk;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, t = lane & 3;
  if (c >= p.doc_off[p.n_docs + 2]) return;
  const int4 ch = reinterpret_cast<const int4*>(p.chunks)[c];
  if (DELTA && ch.z >= p.n_docs) return;
  const int len = ch.y, rep = p.Hv / p.Hk;
  const uint32_t sq = xb_smem_u32(sm.q), sk = xb_smem_u32(sm.k);
  load_tile<U, C, 128>(sq, (const bf16*)p.q + ch.x * p.q_t + kh * p.q_h, p.q_t, len, p.dk);
  load_tile<U, C, 128>(sk, (const bf16*)p.k + ch.x * p.k_t + kh * p.k_h, p.k_t, len, p.dk);
  cp_commit();
  cp_wait<0>();
  __syncthreads();
  {  // row factors: thread pair per row, one for q and one for k
    const int row = tid & 63;
    const uint32_t base = tid < C ? sq : sk;
    float ss = 0.f;
    if (p.l2norm) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint4 v = lds128(base + swz<U>(row, u));
        const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = unpack_bf16x2(x[i]);
          ss += f.x * f.x + f.y * f.y;
        }
      }
    }
    float r = p.l2norm ? 1.f / fmaxf(sqrtf(ss), 1e-12f) : 1.f;
    if (tid < C) r *= p.scale;
    if (row >= len) r = 0.f;
    (tid < C ? sm.rq : sm.rk)[row] = r;
    p.rqk[((long long)c * p.Hk + kh) * RQK + (tid < C ? 0 : C) + row] = r;
  }
  __syncthreads();
  float* qk = p.qk + ((long long)c * p.Hk + kh) * (C * C);
  float* kkg = DELTA ? p.kk + ((long long)c * p.Hk + kh) * (C * C) : nullptr;
  const int r0 = w * 16 + g;
#pragma unroll
  for (int nt = 0; nt < 8; nt += 2) {
    if (nt * 8 > w * 16 + 15) break;              // columns above the diagonal block are never read
    float a1[2][4] = {}, a2[2][4] = {};
#pragma unroll
    for (int ks = 0; ks < DKP / 16; ++ks) {
      uint32_t fq[4], fk[4], fb[4];
      ldsm4(fb, sk + addr_b<U>(nt * 8, ks * 16));
      ldsm4(fq, sq + addr_a<U>(w * 16, ks * 16));
      mma(a1[0], fq, fb[0], fb[1]);
      mma(a1[1], fq, fb[2], fb[3]);
      if (DELTA) {
        ldsm4(fk, sk + addr_a<U>(w * 16, ks * 16));
        mma(a2[0], fk, fb[0], fb[1]);
        mma(a2[1], fk, fb[2], fb[3]);
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int row = r0 + hh * 8, col = (nt + j) * 8 + 2 * t;
        const float c0 = sm.rk[col], c1 = sm.rk[col + 1];
        *reinterpret_cast<float2*>(qk + row * C + col) =
            make_float2(sm.rq[row] * c0 * a1[j][2 * hh], sm.rq[row] * c1 * a1[j][2 * hh + 1]);
        if (DELTA) {
          const float2 v = make_float2(sm.rk[row] * c0 * a2[j][2 * hh], sm.rk[row] * c1 * a2[j][2 * hh + 1]);
          *reinterpret_cast<float2*>(kkg + row * C + col) = v;
          *reinterpret_cast<float2*>(sm.kk + row * C + col) = v;
        }
      }
  }
  // per v head: running log decays; the inverse of I + L, two heads at a time
  for (int h0 = 0; h0 < rep; h0 += DELTA ? 2 : 4) {
    if (!DELTA || w < 2) {
      const int hh = h0 + w, h = kh * rep + hh;
      if (hh < rep) {
        double x[2];
        float bb[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = 2 * lane + i;
          x[i] = 0.0, bb[i] = 0.f;
          if (row < len) {
            const long long tok = ch.x + row;
            bb[i] = p.b[tok * p.b_t + h * p.b_h];
            float gv;
            if (DELTA) {
              gv = p.g[tok * p.g_t + h * p.g_h];
              x[i] = (double)(gv < MIN_LOG ? MIN_LOG : gv) * 1.4426950408889634;
            } else {
              const double z = (double)bb[i] * (double)p.A[h];
              x[i] = (z < (double)MIN_LOG ? (double)MIN_LOG : z) * 1.4426950408889634;
            }
          }
        }
        double s = x[0] + x[1];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double u = __shfl_up_sync(0xffffffffu, s, o);
          if (lane >= o) s += u;
        }
        float* out = p.hd + ((long long)c * p.Hv + h) * HD;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = 2 * lane + i;
          const double G = i ? s : s - x[1];
          const float hi = (float)G, lo = (float)(G - (double)hi);
          out[row] = hi, out[C + row] = lo, out[2 * C + row] = bb[i];
          if (DELTA) sm.ghi[w][row] = hi, sm.glo[w][row] = lo, sm.b[w][row] = bb[i];
        }
      }
    }
    if (DELTA) {
      __syncthreads();                        // also: kk is complete, the previous pair's L has been read
      const int m = tid >> 6, j = tid & 63, hh = h0 + m;
      if (hh < rep) {
        // L, one column per thread: rows below the diagonal
        for (int i = 0; i < C; ++i) {
          float v = 0.f;
          if (i > j) v = sm.b[m][i] * xb_ex2((sm.ghi[m][i] - sm.ghi[m][j]) + (sm.glo[m][i] - sm.glo[m][j])) * sm.kk[i * C + j];
          sm.l[m][i * C + j] = v;
        }
      }
      __syncthreads();
      if (hh < rep) {
        // column j of (I + L)^-1 by forward substitution; all threads of a head read the same row of L
        float x[C];
        const float4* L4 = reinterpret_cast<const float4*>(sm.l[m]);
        float* out = ((float*)p.pt) + ((long long)c * p.Hv + kh * rep + hh) * (C * C) + j;
#pragma unroll
        for (int i = 0; i < C; ++i) {
          float a0 = i == j ? 1.f : 0.f, a1 = 0.f, a2 = 0.f, a3 = 0.f;
#pragma unroll
          for (int k4 = 0; k4 < (i + 3) / 4; ++k4) {
            const float4 l = L4[i * (C / 4) + k4];
            a0 -= l.x * x[4 * k4];
            if (4 * k4 + 1 < i) a1 -= l.y * x[4 * k4 + 1];
            if (4 * k4 + 2 < i) a2 -= l.z * x[4 * k4 + 2];
            if (4 * k4 + 3 < i) a3 -= l.w * x[4 * k4 + 3];
          }
          x[i] = (a0 + a1) + (a2 + a3);
          out[i * C] = x[i];
        }
      }
      __syncthreads();
    }
  }
}

// ---- forward: one CTA carries NV columns of one head's state through one document ----------------------------------
template <int DKP>
struct SeqStage {
  uint8_t q[C * DKP * 2], k[C * DKP * 2], v[C * NV * 2];
  float hd[HD], rqk[RQK];
};
template <int DKP, bool DELTA>
struct FwdSmem {
  SeqStage<DKP> st[2];
  uint8_t shi[DKP * NV * 2], slo[DKP * NV * 2];
  uint8_t xhi[DELTA ? C * NV * 2 : 16], xlo[DELTA ? C * NV * 2 : 16];   // R
  uint8_t uhi[DELTA ? C * NV * 2 : 16], ulo[DELTA ? C * NV * 2 : 16];   // U
  uint8_t dhi[C * NV * 2], dlo[C * NV * 2];                             // K's row factor x d x U
};

template <int DKP, bool DELTA, bool SAVE>
__global__ void __launch_bounds__(128) rec_fwd(const XbRecArgs p) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  FwdSmem<DKP, DELTA>& sm = *reinterpret_cast<FwdSmem<DKP, DELTA>*>(smem_raw);
  constexpr int U = DKP / 8;
  const int slices = p.dvp / NV, rep = p.Hv / p.Hk;
  const int sl = blockIdx.x % slices, h = (blockIdx.x / slices) % p.Hv, doc = blockIdx.x / (slices * p.Hv);
  const int kh = h / rep, v0 = sl * NV, vcols = min(NV, p.dv - v0);
  const int lane = xb_lane(), w = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int c0 = p.doc_off[doc], c1 = p.doc_off[doc + 1];
  const int4* chunks = reinterpret_cast<const int4*>(p.chunks);
  bf16* o = (bf16*)p.o + (long long)h * p.dv + v0;
  const long long o_t = (long long)p.Hv * p.dv;
  if (DELTA && doc >= p.n_docs) {                                    // rows outside the documents
    if (!SAVE)
      for (int c = c0; c < c1; ++c)
        for (int i = threadIdx.x; i < chunks[c].y * NV; i += 128)
          if (i % NV < vcols) o[(chunks[c].x + i / NV) * o_t + i % NV] = __float2bfloat16(0.f);
    return;
  }
  float s[DKP / 64][4][4] = {};
  const long long soff = ((long long)doc * p.Hv + h) * p.dk * p.dv + v0 * p.s_v;
  if (p.s_in != nullptr && doc < p.n_docs) state_global<DKP, false>(s, const_cast<float*>(p.s_in) + soff, p.s_k, p.s_v, p.dk, vcols);
  const uint32_t shi = xb_smem_u32(sm.shi), slo = xb_smem_u32(sm.slo);
  auto fetch = [&](int c, int b) {
    const int4 ch = chunks[c];
    SeqStage<DKP>& st = sm.st[b];
    load_tile<U, C, 128>(xb_smem_u32(st.k), (const bf16*)p.k + ch.x * p.k_t + kh * p.k_h, p.k_t, ch.y, p.dk);
    if (!SAVE) load_tile<U, C, 128>(xb_smem_u32(st.q), (const bf16*)p.q + ch.x * p.q_t + kh * p.q_h, p.q_t, ch.y, p.dk);
    load_tile<4, C, 128>(xb_smem_u32(st.v), (const bf16*)p.v + ch.x * p.v_t + h * p.v_h + v0, p.v_t, ch.y, vcols);
    load_floats<128>(xb_smem_u32(st.hd), p.hd + ((long long)c * p.Hv + h) * HD, HD);
    load_floats<128>(xb_smem_u32(st.rqk), p.rqk + ((long long)c * p.Hk + kh) * RQK, RQK);
  };
  if (c0 < c1) fetch(c0, 0);
  cp_commit();
  state_to_smem<DKP>(s, shi, slo);
  for (int c = c0; c < c1; ++c) {
    SeqStage<DKP>& st = sm.st[(c - c0) & 1];
    const int4 ch = chunks[c];
    const uint32_t sk = xb_smem_u32(st.k), sq = xb_smem_u32(st.q), sv = xb_smem_u32(st.v);
    cp_wait<0>();
    __syncthreads();                       // this chunk's tiles and the state's planes are complete
    if (c + 1 < c1) fetch(c + 1, (c - c0 + 1) & 1);
    cp_commit();
    const long long ch_h = (long long)c * p.Hv + h;
    if (SAVE) state_save<DKP>(shi, slo, (uint8_t*)p.s_tiles + (ch_h * slices + sl) * HALF);
    const int ra = w * 16 + g;             // this thread's rows: ra and ra + 8
    float acc_k[4][4] = {}, acc_q[4][4] = {};
    if (DELTA || !SAVE) {
#pragma unroll
      for (int ks = 0; ks < DKP / 16; ++ks) {
        uint32_t fk[4], fq[4], bh[2][4], bl[2][4];
        if (DELTA) ldsm4(fk, sk + addr_a<U>(w * 16, ks * 16));
        if (!SAVE) ldsm4(fq, sq + addr_a<U>(w * 16, ks * 16));
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          ldsm4t(bh[n], shi + addr_bt<4>(ks * 16, n * 16));
          ldsm4t(bl[n], slo + addr_bt<4>(ks * 16, n * 16));
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int a = n >> 1, b = (n & 1) * 2;
          if (DELTA) {
            mma(acc_k[n], fk, bl[a][b], bl[a][b + 1]);
            mma(acc_k[n], fk, bh[a][b], bh[a][b + 1]);
          }
          if (!SAVE) {
            mma(acc_q[n], fq, bl[a][b], bl[a][b + 1]);
            mma(acc_q[n], fq, bh[a][b], bh[a][b + 1]);
          }
        }
      }
    }
    if (DELTA) {
      // R = b (V - gamma rk K S)
      const uint32_t xhi = xb_smem_u32(sm.xhi), xlo = xb_smem_u32(sm.xlo);
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int row = ra + hh * 8;
        const float b = st.hd[2 * C + row], f = ex2_sum(st.hd, row) * st.rqk[C + row];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const uint32_t off = at2<4>(row, n * 8 + 2 * t);
          const float2 v = unpack_bf16x2(lds32(sv + off));
          uint32_t hi, lo;
          split2(b * (v.x - f * acc_k[n][2 * hh]), b * (v.y - f * acc_k[n][2 * hh + 1]), hi, lo);
          sts32(xhi + off, hi);
          sts32(xlo + off, lo);
        }
      }
      __syncthreads();
      // U = T R, T lower triangular
      float u[4][4] = {};
      const float* tm = ((float*)p.pt) + ch_h * (C * C);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        if (ks <= w) {
          uint32_t ah[4], al[4], bh[2][4], bl[2][4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 x = *reinterpret_cast<const float2*>(tm + (ra + (e & 1) * 8) * C + ks * 16 + (e >> 1) * 8 + 2 * t);
            split2(x.x, x.y, ah[e], al[e]);
          }
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            ldsm4t(bh[n], xhi + addr_bt<4>(ks * 16, n * 16));
            ldsm4t(bl[n], xlo + addr_bt<4>(ks * 16, n * 16));
          }
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const int a = n >> 1, b = (n & 1) * 2;
            mma(u[n], al, bh[a][b], bh[a][b + 1]);
            mma(u[n], ah, bl[a][b], bl[a][b + 1]);
            mma(u[n], ah, bh[a][b], bh[a][b + 1]);
          }
        }
      }
      const uint32_t uhi = xb_smem_u32(sm.uhi), ulo = xb_smem_u32(sm.ulo);
      const uint32_t dhi = xb_smem_u32(sm.dhi), dlo = xb_smem_u32(sm.dlo);
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int row = ra + hh * 8;
        const float f = ex2_diff(st.hd, C - 1, row) * st.rqk[C + row];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const uint32_t off = at2<4>(row, n * 8 + 2 * t);
          uint32_t hi, lo;
          split2(u[n][2 * hh], u[n][2 * hh + 1], hi, lo);
          if (SAVE) {
          } else {
            sts32(uhi + off, hi);
            sts32(ulo + off, lo);
          }
          split2(f * u[n][2 * hh], f * u[n][2 * hh + 1], hi, lo);
          sts32(dhi + off, hi);
          sts32(dlo + off, lo);
        }
      }
    } else {
      // b d V, two neighbouring values per thread
      const uint32_t dhi = xb_smem_u32(sm.dhi), dlo = xb_smem_u32(sm.dlo);
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int row = ra + hh * 8;
        const float f = ex2_diff(st.hd, C - 1, row) * st.hd[2 * C + row];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const uint32_t off = at2<4>(row, n * 8 + 2 * t);
          const float2 v = unpack_bf16x2(lds32(sv + off));
          uint32_t hi, lo;
          split2(f * v.x, f * v.y, hi, lo);
          sts32(dhi + off, hi);
          sts32(dlo + off, lo);
        }
      }
    }
    __syncthreads();
    if (!SAVE) {
      // O = gamma rq Q S + P U
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const float f = ex2_sum(st.hd, ra + hh * 8) * st.rqk[ra + hh * 8];
#pragma unroll
        for (int n = 0; n < 4; ++n) acc_q[n][2 * hh] *= f, acc_q[n][2 * hh + 1] *= f;
      }
      const float* qk = p.qk + ((long long)c * p.Hk + kh) * (C * C);
      const uint32_t uhi = DELTA ? xb_smem_u32(sm.uhi) : sv, ulo = xb_smem_u32(sm.ulo);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        if (ks <= w) {
          uint32_t ah[4], al[4], bh[2][4], bl[2][4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int row = ra + (e & 1) * 8, col = ks * 16 + (e >> 1) * 8 + 2 * t;
            const float2 x = *reinterpret_cast<const float2*>(qk + row * C + col);
            float y0 = col <= row ? x.x * ex2_diff(st.hd, row, col) : 0.f;
            float y1 = col + 1 <= row ? x.y * ex2_diff(st.hd, row, col + 1) : 0.f;
            if (!DELTA) y0 *= st.hd[2 * C + col], y1 *= st.hd[2 * C + col + 1];
            split2(y0, y1, ah[e], al[e]);
          }
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            ldsm4t(bh[n], uhi + addr_bt<4>(ks * 16, n * 16));
            if (DELTA) ldsm4t(bl[n], ulo + addr_bt<4>(ks * 16, n * 16));
          }
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const int a = n >> 1, b = (n & 1) * 2;
            mma(acc_q[n], al, bh[a][b], bh[a][b + 1]);
            if (DELTA) mma(acc_q[n], ah, bl[a][b], bl[a][b + 1]);
            mma(acc_q[n], ah, bh[a][b], bh[a][b + 1]);
          }
        }
      }
      const float skip = DELTA ? 0.f : p.D[h];
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int row = ra + hh * 8;
        if (row < ch.y) {
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const int col = n * 8 + 2 * t;
            if (col < vcols) {
              float y0 = acc_q[n][2 * hh], y1 = acc_q[n][2 * hh + 1];
              if (!DELTA) {
                const float2 v = unpack_bf16x2(lds32(sv + at2<4>(row, col)));
                y0 += skip * v.x, y1 += skip * v.y;
              }
              *reinterpret_cast<uint32_t*>(o + (ch.x + row) * o_t + col) = pack_bf16x2(y0, y1);
            }
          }
        }
      }
    }
    {  // S = gamma_last S + K^T (d U)
      const uint32_t dhi = xb_smem_u32(sm.dhi), dlo = xb_smem_u32(sm.dlo);
      const float f = ex2_sum(st.hd, C - 1);
#pragma unroll
      for (int m = 0; m < DKP / 64; ++m)
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[m][n][e] *= f;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        uint32_t bh[2][4], bl[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          ldsm4t(bh[n], dhi + addr_bt<4>(ks * 16, n * 16));
          ldsm4t(bl[n], dlo + addr_bt<4>(ks * 16, n * 16));
        }
#pragma unroll
        for (int m = 0; m < DKP / 64; ++m) {
          uint32_t fa[4];
          ldsm4t(fa, sk + addr_at<U>(w * (DKP / 4) + m * 16, ks * 16));
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const int a = n >> 1, b = (n & 1) * 2;
            mma(s[m][n], fa, bl[a][b], bl[a][b + 1]);
            mma(s[m][n], fa, bh[a][b], bh[a][b + 1]);
          }
        }
      }
      state_to_smem<DKP>(s, shi, slo);     // the old planes were last read before the barrier above
    }
  }
  cp_wait<0>();
  if (p.s_out != nullptr && doc < p.n_docs) state_global<DKP, true>(s, p.s_out + soff, p.s_k, p.s_v, p.dk, vcols);
}

// ---- backward, sequential part: the state's gradient through one document, last chunk first -----------------------
template <int DKP>
struct BwdStage {
  uint8_t q[C * DKP * 2], k[C * DKP * 2], dy[C * NV * 2];
  float hd[HD], rqk[RQK];
};
template <int DKP, bool DELTA>
struct BwdSmem {
  BwdStage<DKP> st[2];
  uint8_t shi[DKP * NV * 2], slo[DKP * NV * 2];                         // dS'
  uint8_t uhi[DELTA ? C * NV * 2 : 16], ulo[DELTA ? C * NV * 2 : 16];   // dU
  uint8_t xhi[DELTA ? C * NV * 2 : 16], xlo[DELTA ? C * NV * 2 : 16];   // -b gamma rk dR
  uint8_t yhi[C * NV * 2], ylo[C * NV * 2];                             // gamma rq dO
};

template <int DKP, bool DELTA>
__global__ void __launch_bounds__(128) rec_bwd(const XbRecArgs p) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  BwdSmem<DKP, DELTA>& sm = *reinterpret_cast<BwdSmem<DKP, DELTA>*>(smem_raw);
  constexpr int U = DKP / 8;
  const int slices = p.dvp / NV, rep = p.Hv / p.Hk;
  const int sl = blockIdx.x % slices, h = (blockIdx.x / slices) % p.Hv, doc = blockIdx.x / (slices * p.Hv);
  const int kh = h / rep, v0 = sl * NV, vcols = min(NV, p.dv - v0);
  const int lane = xb_lane(), w = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int c0 = p.doc_off[doc], c1 = p.doc_off[doc + 1];
  const int4* chunks = reinterpret_cast<const int4*>(p.chunks);
  bf16* dv = (bf16*)p.dv_out + (long long)h * p.dv + v0;
  const long long dv_t = (long long)p.Hv * p.dv;
  if (DELTA && doc >= p.n_docs) {
    for (int c = c0; c < c1; ++c)
      for (int i = threadIdx.x; i < chunks[c].y * NV; i += 128)
        if (i % NV < vcols) dv[(chunks[c].x + i / NV) * dv_t + i % NV] = __float2bfloat16(0.f);
    return;
  }
  float s[DKP / 64][4][4] = {};
  const long long soff = ((long long)doc * p.Hv + h) * p.dk * p.dv + v0 * p.s_v;
  if (p.ds_out != nullptr && doc < p.n_docs) state_global<DKP, false>(s, const_cast<float*>(p.ds_out) + soff, p.s_k, p.s_v, p.dk, vcols);
  const uint32_t shi = xb_smem_u32(sm.shi), slo = xb_smem_u32(sm.slo);
  auto fetch = [&](int c, int b) {
    const int4 ch = chunks[c];
    BwdStage<DKP>& st = sm.st[b];
    load_tile<U, C, 128>(xb_smem_u32(st.k), (const bf16*)p.k + ch.x * p.k_t + kh * p.k_h, p.k_t, ch.y, p.dk);
    load_tile<U, C, 128>(xb_smem_u32(st.q), (const bf16*)p.q + ch.x * p.q_t + kh * p.q_h, p.q_t, ch.y, p.dk);
    load_tile<4, C, 128>(xb_smem_u32(st.dy), (const bf16*)p.dy + ch.x * p.dy_t + h * p.dy_h + v0, p.dy_t, ch.y, vcols);
    load_floats<128>(xb_smem_u32(st.hd), p.hd + ((long long)c * p.Hv + h) * HD, HD);
    load_floats<128>(xb_smem_u32(st.rqk), p.rqk + ((long long)c * p.Hk + kh) * RQK, RQK);
  };
  if (c0 < c1) fetch(c1 - 1, 0);
  cp_commit();
  state_to_smem<DKP>(s, shi, slo);
  for (int c = c1 - 1; c >= c0; --c) {
    BwdStage<DKP>& st = sm.st[(c1 - 1 - c) & 1];
    const int4 ch = chunks[c];
    const uint32_t sk = xb_smem_u32(st.k), sq = xb_smem_u32(st.q), sy = xb_smem_u32(st.dy);
    const uint32_t yhi = xb_smem_u32(sm.yhi), ylo = xb_smem_u32(sm.ylo);
    cp_wait<0>();
    __syncthreads();
    if (c > c0) fetch(c - 1, (c1 - c) & 1);
    cp_commit();
    const long long ch_h = (long long)c * p.Hv + h;
    state_save<DKP>(shi, slo, (uint8_t*)p.ds_tiles + (ch_h * slices + sl) * HALF);
    const int ra = w * 16 + g;
    // K dS'
    float du[4][4] = {};
#pragma unroll
    for (int ks = 0; ks < DKP / 16; ++ks) {
      uint32_t fk[4], bh[2][4], bl[2][4];
      ldsm4(fk, sk + addr_a<U>(w * 16, ks * 16));
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        ldsm4t(bh[n], shi + addr_bt<4>(ks * 16, n * 16));
        ldsm4t(bl[n], slo + addr_bt<4>(ks * 16, n * 16));
      }
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int a = n >> 1, b = (n & 1) * 2;
        mma(du[n], fk, bl[a][b], bl[a][b + 1]);
        mma(du[n], fk, bh[a][b], bh[a][b + 1]);
      }
    }
    // dU = d rk K dS' + P^T dO; beside it gamma rq dO for the state
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const int row = ra + hh * 8;
      const float f = ex2_diff(st.hd, C - 1, row) * st.rqk[C + row], y = ex2_sum(st.hd, row) * st.rqk[row];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        du[n][2 * hh] *= f, du[n][2 * hh + 1] *= f;
        const uint32_t off = at2<4>(row, n * 8 + 2 * t);
        const float2 v = unpack_bf16x2(lds32(sy + off));
        uint32_t hi, lo;
        split2(y * v.x, y * v.y, hi, lo);
        sts32(yhi + off, hi);
        sts32(ylo + off, lo);
      }
    }
    const float* qk = p.qk + ((long long)c * p.Hk + kh) * (C * C);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      if (ks >= w) {
        uint32_t ah[4], al[4], bh[2][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = ra + (e & 1) * 8, i = ks * 16 + (e >> 1) * 8 + 2 * t;     // element (j, i) of P^T
          const float y0 = i >= j ? qk[i * C + j] * ex2_diff(st.hd, i, j) : 0.f;
          const float y1 = i + 1 >= j ? qk[(i + 1) * C + j] * ex2_diff(st.hd, i + 1, j) : 0.f;
          split2(y0, y1, ah[e], al[e]);
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) ldsm4t(bh[n], sy + addr_bt<4>(ks * 16, n * 16));
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int a = n >> 1, b = (n & 1) * 2;
          mma(du[n], al, bh[a][b], bh[a][b + 1]);
          mma(du[n], ah, bh[a][b], bh[a][b + 1]);
        }
      }
    }
    if (DELTA) {
      const uint32_t uhi = xb_smem_u32(sm.uhi), ulo = xb_smem_u32(sm.ulo), xhi = xb_smem_u32(sm.xhi), xlo = xb_smem_u32(sm.xlo);
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const uint32_t off = at2<4>(ra + hh * 8, n * 8 + 2 * t);
          uint32_t hi, lo;
          split2(du[n][2 * hh], du[n][2 * hh + 1], hi, lo);
          sts32(uhi + off, hi);
          sts32(ulo + off, lo);
        }
      __syncthreads();
      // dR = T^T dU
      float dr[4][4] = {};
      const float* tm = ((float*)p.pt) + ch_h * (C * C);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        if (ks >= w) {
          uint32_t ah[4], al[4], bh[2][4], bl[2][4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = ra + (e & 1) * 8, i = ks * 16 + (e >> 1) * 8 + 2 * t;
            split2(tm[i * C + j], tm[(i + 1) * C + j], ah[e], al[e]);
          }
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            ldsm4t(bh[n], uhi + addr_bt<4>(ks * 16, n * 16));
            ldsm4t(bl[n], ulo + addr_bt<4>(ks * 16, n * 16));
          }
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const int a = n >> 1, b = (n & 1) * 2;
            mma(dr[n], al, bh[a][b], bh[a][b + 1]);
            mma(dr[n], ah, bl[a][b], bl[a][b + 1]);
            mma(dr[n], ah, bh[a][b], bh[a][b + 1]);
          }
        }
      }
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int row = ra + hh * 8;
        const float b = st.hd[2 * C + row], f = -b * ex2_sum(st.hd, row) * st.rqk[C + row];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int col = n * 8 + 2 * t;
          const uint32_t off = at2<4>(row, col);
          const float y0 = dr[n][2 * hh], y1 = dr[n][2 * hh + 1];
          uint32_t hi, lo;
          split2(y0, y1, hi, lo);
          split2(f * y0, f * y1, hi, lo);
          sts32(xhi + off, hi);
          sts32(xlo + off, lo);
          if (row < ch.y && col < vcols)
            *reinterpret_cast<uint32_t*>(dv + (ch.x + row) * dv_t + col) = pack_bf16x2(b * y0, b * y1);
        }
      }
    } else {
      const float skip = p.D[h];
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int row = ra + hh * 8;
        const float b = st.hd[2 * C + row];
        if (row < ch.y) {
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const int col = n * 8 + 2 * t;
            if (col < vcols) {
              const float2 y = unpack_bf16x2(lds32(sy + at2<4>(row, col)));
              *reinterpret_cast<uint32_t*>(dv + (ch.x + row) * dv_t + col) =
                  pack_bf16x2(b * du[n][2 * hh] + skip * y.x, b * du[n][2 * hh + 1] + skip * y.y);
            }
          }
        }
      }
    }
    __syncthreads();
    {  // dS = gamma_last dS' + Q^T (gamma rq dO) + K^T (-b gamma rk dR)
      const float f = ex2_sum(st.hd, C - 1);
#pragma unroll
      for (int m = 0; m < DKP / 64; ++m)
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[m][n][e] *= f;
#pragma unroll
      for (int part = 0; part < (DELTA ? 2 : 1); ++part) {
        const uint32_t base = part ? sk : sq, bhi = part ? xb_smem_u32(sm.xhi) : yhi, blo = part ? xb_smem_u32(sm.xlo) : ylo;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          uint32_t bh[2][4], bl[2][4];
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            ldsm4t(bh[n], bhi + addr_bt<4>(ks * 16, n * 16));
            ldsm4t(bl[n], blo + addr_bt<4>(ks * 16, n * 16));
          }
#pragma unroll
          for (int m = 0; m < DKP / 64; ++m) {
            uint32_t fa[4];
            ldsm4t(fa, base + addr_at<U>(w * (DKP / 4) + m * 16, ks * 16));
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              const int a = n >> 1, b = (n & 1) * 2;
              mma(s[m][n], fa, bl[a][b], bl[a][b + 1]);
              mma(s[m][n], fa, bh[a][b], bh[a][b + 1]);
            }
          }
        }
      }
      state_to_smem<DKP>(s, shi, slo);
    }
  }
  cp_wait<0>();
  if (p.ds_in != nullptr && doc < p.n_docs) state_global<DKP, true>(s, p.ds_in + soff, p.s_k, p.s_v, p.dk, vcols);
}

// dA and dD: sums of the chunks' parts, in a fixed order
__global__ void __launch_bounds__(128) rec_reduce(const XbRecArgs p) {
  __shared__ double red[2][4];
  const int h = blockIdx.x, n = p.doc_off[p.n_docs + 2], lane = threadIdx.x & 31;
  double a = 0.0, b = 0.0;
  for (int c = threadIdx.x; c < n; c += 128) {
    const float2 v = *reinterpret_cast<const float2*>(p.part + ((long long)c * p.Hv + h) * 2);
    a += v.x, b += v.y;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if (lane == 0) red[0][threadIdx.x >> 5] = a, red[1][threadIdx.x >> 5] = b;
  __syncthreads();
  if (threadIdx.x == 0) {
    p.dA[h] = (float)((red[0][0] + red[0][1]) + (red[0][2] + red[0][3]));
    p.dD[h] = (float)((red[1][0] + red[1][1]) + (red[1][2] + red[1][3]));
  }
}

bool bad_args(const XbRecArgs& a) {
  return a.T < 0 || a.n_docs < 0 || a.Hk <= 0 || a.Hv <= 0 || a.Hv % a.Hk || a.dk <= 0 || a.dk > 128 || a.dk % 8 || a.dv <= 0 ||
         a.dv % 8 || a.dvp != (a.dv + 63) / 64 * 64 || a.dkp != (a.dk <= 64 ? 64 : 128) || a.nc_max < a.T / C + a.n_docs + 2;
}

int plan(const XbRecArgs& a, cudaStream_t st) {
  rec_plan<<<1, 1024, 0, st>>>(a.cu, a.n_docs, a.T, a.nc_max, (int4*)a.chunks, a.doc_off, a.status);
  return cudaGetLastError() == cudaSuccess ? 0 : -11;
}

template <int DKP>
int scan_fwd(const XbRecArgs& a, cudaStream_t st) {
  const long long seq = (long long)(a.n_docs + 2) * a.Hv * (a.dvp / NV);
  if (int rc = rec_launch(rec_prep<DKP, false>, (long long)a.nc_max * a.Hk, 128, sizeof(PrepSmem<DKP, false>), a, st)) return rc;
  return rec_launch(rec_fwd<DKP, false, false>, seq, 128, sizeof(FwdSmem<DKP, false>), a, st);
}

template <int DKP>
int scan_bwd(const XbRecArgs& a, cudaStream_t st) {
  const long long seq = (long long)(a.n_docs + 2) * a.Hv * (a.dvp / NV);
  XbRecArgs again = a;
  again.s_out = nullptr;
  if (int rc = rec_launch(rec_fwd<DKP, false, true>, seq, 128, sizeof(FwdSmem<DKP, false>), again, st)) return rc;
  return rec_launch(rec_bwd<DKP, false>, seq, 128, sizeof(BwdSmem<DKP, false>), a, st);
}

}  // namespace

XB_API int xb_recurrence_chunk() { return C; }

XB_API int xb_recurrence_fwd(const XbRecArgs* args, int delta, void* stream) {
  if (args == nullptr || bad_args(*args)) return -1;
  XbRecArgs mine = *args, *a = &mine;
  mine.status = xb_status_ptr();
  cudaStream_t st = (cudaStream_t)stream;
  if (int rc = plan(*a, st)) return rc;
  if (delta) return xb_delta_fwd(*a, st);
  return a->dk <= 64 ? scan_fwd<64>(*a, st) : scan_fwd<128>(*a, st);
}

XB_API int xb_recurrence_bwd(const XbRecArgs* args, int delta, void* stream) {
  if (args == nullptr || bad_args(*args)) return -1;
  XbRecArgs mine = *args, *a = &mine;
  mine.status = xb_status_ptr();
  cudaStream_t st = (cudaStream_t)stream;
  if (delta) {
    if (int rc = xb_delta_bwd(*a, st)) return rc;
    return xb_recurrence_grad(*a, 1, st);
  }
  if (int rc = a->dk <= 64 ? scan_bwd<64>(*a, st) : scan_bwd<128>(*a, st)) return rc;
  if (int rc = xb_recurrence_grad(*a, 0, st)) return rc;
  return rec_launch(rec_reduce, a->Hv, 128, 0, *a, st);
}
