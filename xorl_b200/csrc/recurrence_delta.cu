// The gated delta rule's own kernels: prepare, forward, and the sequential part of the backward pass (the formulas
// stand in recurrence.cu).
//
// A chunk's chain  K S -> R -> U = T R -> S' = gamma S + K^T d U  is sequential, and with one long document there are
// only heads x column slices of them (32 x 4 for 32 heads of 128), less than one per SM: the time of a step is what
// counts.  So a CTA of eight warps carries 32 state columns; four warps run the chain, the other four what hangs on it
// (forward: Q S and P U; backward: the state's own update).  Everything that depends on the chunk alone is made once,
// by the prepare kernel, in the form that the products read: P = tril(D o Q K^T) and T = (I + L)^-1 as two bf16 parts
// in blocks of 16 x 16, lower triangle only, so the chain has no exponentials, no splits of T and no loads that it
// waits for.  mma.sync and not tcgen05: operands change hands between registers three times per step on 64 x 32 tiles,
// and a round trip through tensor memory (commit, wait, load) costs more than the 100 to 500 cycles that such a
// product takes on the register path.
#include "recurrence_core.cuh"

namespace {

constexpr int BLK = 512;                    // bytes of a 16 x 16 bf16 block: four 8 x 8 matrices in fragment order
constexpr int TRI = 10 * 2 * BLK;           // lower triangle of a 64 x 64 matrix, two planes
__device__ __forceinline__ int blk_of(int rb, int cb) { return (rb * (rb + 1) / 2 + cb) * 2 * BLK; }
// A fragment of a block, and of its transpose
__device__ __forceinline__ uint32_t addr_blk(int l) { return (uint32_t)l * 16u; }
__device__ __forceinline__ uint32_t addr_blk_t(int l) { return (uint32_t)((l & 7) + ((l >> 3) & 1) * 16 + (l >> 4) * 8) * 16u; }

__device__ __forceinline__ void bar(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
__device__ __forceinline__ void bar_arrive(int id, int n) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(n) : "memory"); }

// ---- prepare -----------------------------------------------------------------------------------------------------
constexpr int LS = 72;                      // row stride of L: rows of a fragment fall into different banks
template <int DKP>
struct DPrepSmem {
  union {
    struct { uint8_t q[C * DKP * 2], k[C * DKP * 2]; };
    float l[2][C * LS];
  };
  float2 qk[8 * 2 * 128], kk[8 * 2 * 128];  // Q K^T and K K^T, each thread's own fragments
  float hd[2][3][C];
  float rq[C], rk[C];
};

// x = column j of (I + L)^-1, whose first FROM rows are zero
template <int FROM>
__device__ __forceinline__ void solve(float (&x)[C], const float* L, int j) {
  const float4* L4 = reinterpret_cast<const float4*>(L);
#pragma unroll
  for (int i = 0; i < FROM; ++i) x[i] = 0.f;
#pragma unroll
  for (int i = FROM; i < C; ++i) {
    float a0 = i == j ? 1.f : 0.f, a1 = 0.f, a2 = 0.f, a3 = 0.f;
#pragma unroll
    for (int k4 = FROM / 4; k4 < (i + 3) / 4; ++k4) {
      const float4 l = L4[i * (LS / 4) + k4];
      a0 -= l.x * x[4 * k4];
      if (4 * k4 + 1 < i) a1 -= l.y * x[4 * k4 + 1];
      if (4 * k4 + 2 < i) a2 -= l.z * x[4 * k4 + 2];
      if (4 * k4 + 3 < i) a3 -= l.w * x[4 * k4 + 3];
    }
    x[i] = (a0 + a1) + (a2 + a3);
  }
}

template <int DKP>
__global__ void __launch_bounds__(128, 3) delta_prep(const XbRecArgs p) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  DPrepSmem<DKP>& sm = *reinterpret_cast<DPrepSmem<DKP>*>(smem_raw);
  constexpr int U = DKP / 8;
  const int kh = blockIdx.x % p.Hk, c = blockIdx.x / p.Hk;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, t = lane & 3;
  if (c >= p.doc_off[p.n_docs + 2]) return;
  const int4 ch = reinterpret_cast<const int4*>(p.chunks)[c];
  if (ch.z >= p.n_docs) return;
  const int len = ch.y, rep = p.Hv / p.Hk;
  const uint32_t sq = xb_smem_u32(sm.q), sk = xb_smem_u32(sm.k);
  load_tile<U, C, 128>(sq, (const bf16*)p.q + ch.x * p.q_t + kh * p.q_h, p.q_t, len, p.dk);
  load_tile<U, C, 128>(sk, (const bf16*)p.k + ch.x * p.k_t + kh * p.k_h, p.k_t, len, p.dk);
  cp_commit();
  // warps 0 and 1 own the running decay of one head of a pair each: two rows per lane
  float gv[2] = {}, bv[2] = {};
  auto read_head = [&](int hh) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = 2 * lane + i;
      gv[i] = bv[i] = 0.f;
      if (w < 2 && hh < rep && row < len) {
        const long long tok = ch.x + row;
        gv[i] = p.g[tok * p.g_t + (kh * rep + hh) * p.g_h];
        bv[i] = p.b[tok * p.b_t + (kh * rep + hh) * p.b_h];
      }
    }
  };
  read_head(w);
  cp_wait<0>();
  __syncthreads();
  {  // row factors: one thread per row of q and of k
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
  const int r0 = w * 16 + g;
  float* qkg = p.qk == nullptr ? nullptr : p.qk + ((long long)c * p.Hk + kh) * (C * C);
  float* kkg = p.kk == nullptr ? nullptr : p.kk + ((long long)c * p.Hk + kh) * (C * C);
#pragma unroll
  for (int nt = 0; nt < 8; nt += 2) {
    if (nt * 8 > w * 16 + 15) break;              // columns above the diagonal block are never read
    float a1[2][4] = {}, a2[2][4] = {};
#pragma unroll
    for (int ks = 0; ks < DKP / 16; ++ks) {
      uint32_t fq[4], fk[4], fb[4];
      ldsm4(fb, sk + addr_b<U>(nt * 8, ks * 16));
      ldsm4(fq, sq + addr_a<U>(w * 16, ks * 16));
      ldsm4(fk, sk + addr_a<U>(w * 16, ks * 16));
      mma(a1[0], fq, fb[0], fb[1]);
      mma(a1[1], fq, fb[2], fb[3]);
      mma(a2[0], fk, fb[0], fb[1]);
      mma(a2[1], fk, fb[2], fb[3]);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int row = r0 + hh * 8, col = (nt + j) * 8 + 2 * t;
        const float c0 = sm.rk[col], c1 = sm.rk[col + 1], fq = sm.rq[row], fk = sm.rk[row];
        const float2 x = make_float2(fq * c0 * a1[j][2 * hh], fq * c1 * a1[j][2 * hh + 1]);
        const float2 y = make_float2(fk * c0 * a2[j][2 * hh], fk * c1 * a2[j][2 * hh + 1]);
        sm.qk[((nt + j) * 2 + hh) * 128 + tid] = x;
        sm.kk[((nt + j) * 2 + hh) * 128 + tid] = y;
        if (qkg != nullptr) {
          *reinterpret_cast<float2*>(qkg + row * C + col) = x;
          *reinterpret_cast<float2*>(kkg + row * C + col) = y;
        }
      }
  }
  for (int h0 = 0; h0 < rep; h0 += 2) {
    if (w < 2 && h0 + w < rep) {
      double x[2], s = 0.0;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        x[i] = 2 * lane + i < len ? (double)(gv[i] < MIN_LOG ? MIN_LOG : gv[i]) * 1.4426950408889634 : 0.0;
        s += x[i];
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double u = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += u;
      }
      float* out = p.hd + ((long long)c * p.Hv + kh * rep + h0 + w) * HD;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = 2 * lane + i;
        const double G = i ? s : s - x[1];
        const float hi = (float)G, lo = (float)(G - (double)hi);
        out[row] = hi, out[C + row] = lo, out[2 * C + row] = bv[i];
        sm.hd[w][0][row] = hi, sm.hd[w][1][row] = lo, sm.hd[w][2][row] = bv[i];
      }
    }
    read_head(h0 + 2 + w);
    __syncthreads();                              // also: the tiles, or the pair before, have been read
#pragma unroll 1
    for (int m = 0; m < 2; ++m) {
      if (h0 + m >= rep) break;
      const float* hd = sm.hd[m][0];
      uint8_t* pl = (uint8_t*)p.pt + ((long long)c * p.Hv + kh * rep + h0 + m) * (2 * TRI);
#pragma unroll
      for (int nt = 0; nt < 8; ++nt) {
        if (nt > 2 * w + 1) break;
        const int col = nt * 8 + 2 * t;
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const int row = r0 + hh * 8;
          const float2 x = sm.qk[(nt * 2 + hh) * 128 + tid], y = sm.kk[(nt * 2 + hh) * 128 + tid];
          const float d0 = ex2_diff(hd, row, col), d1 = ex2_diff(hd, row, col + 1), b = hd[2 * C + row];
          uint32_t hi, lo;
          split2(col <= row ? d0 * x.x : 0.f, col + 1 <= row ? d1 * x.y : 0.f, hi, lo);
          uint32_t* dst = reinterpret_cast<uint32_t*>(pl + blk_of(w, nt >> 1) + (hh + 2 * (nt & 1)) * 128 + g * 16 + t * 4);
          dst[0] = hi;
          dst[BLK / 4] = lo;
          *reinterpret_cast<float2*>(&sm.l[m][row * LS + col]) =
              make_float2(col < row ? b * d0 * y.x : 0.f, col + 1 < row ? b * d1 * y.y : 0.f);
        }
      }
    }
    __syncthreads();
    // column j of (I + L)^-1 by forward substitution: all threads of a head read the same row of L, and a warp of
    // columns 32 .. 63 starts at row 32
    const int m = tid >> 6, j = tid & 63;
    float x[C];
    if (h0 + m < rep) {
      if (w & 1) solve<32>(x, sm.l[m], j);
      else solve<0>(x, sm.l[m], j);
    }
    __syncthreads();
    if (h0 + m < rep) {
#pragma unroll
      for (int i = 0; i < C; ++i) sm.l[m][i * LS + j] = x[i];
    }
    __syncthreads();
    for (int it = tid; it < 2 * 320; it += 128) {
      const int mm = it / 320, e = it % 320, blk = e >> 5, mat = (e >> 3) & 3, r = e & 7;
      if (h0 + mm >= rep) break;
      const int rb = blk < 1 ? 0 : blk < 3 ? 1 : blk < 6 ? 2 : 3, cb = blk - rb * (rb + 1) / 2;
      const float4* src = reinterpret_cast<const float4*>(&sm.l[mm][(rb * 16 + (mat & 1) * 8 + r) * LS + cb * 16 + (mat >> 1) * 8]);
      const float4 a = src[0], b = src[1];
      uint4 hi, lo;
      split2(a.x, a.y, hi.x, lo.x), split2(a.z, a.w, hi.y, lo.y), split2(b.x, b.y, hi.z, lo.z), split2(b.z, b.w, hi.w, lo.w);
      uint8_t* dst = (uint8_t*)p.pt + ((long long)c * p.Hv + kh * rep + h0 + mm) * (2 * TRI) + TRI + blk * 2 * BLK + mat * 128 + r * 16;
      *reinterpret_cast<uint4*>(dst) = hi;
      *reinterpret_cast<uint4*>(dst + BLK) = lo;
    }
  }
}

// ---- what a step reads ---------------------------------------------------------------------------------------------
template <int DKP>
struct DStage {
  uint8_t q[C * DKP * 2], k[C * DKP * 2], x[C * NV * 2];      // x: v, or dO
  uint8_t pt[2 * TRI];                                        // P, T
  float hd[HD], rqk[RQK];
};
template <int THREADS>
__device__ __forceinline__ void load_bytes(uint32_t dst, const uint8_t* src, int n) {
  for (int i = threadIdx.x; i < n / 16; i += THREADS) cp16(dst + i * 16, src + i * 16, true);
}
template <int DKP, int THREADS, bool Q, bool P>
__device__ __forceinline__ void fetch_stage(const XbRecArgs& p, DStage<DKP>& st, const int4 ch, int c, int h, int kh, const bf16* x,
                                            long long x_t, int vcols) {
  constexpr int U = DKP / 8;
  load_tile<U, C, THREADS>(xb_smem_u32(st.k), (const bf16*)p.k + ch.x * p.k_t + kh * p.k_h, p.k_t, ch.y, p.dk);
  if (Q) load_tile<U, C, THREADS>(xb_smem_u32(st.q), (const bf16*)p.q + ch.x * p.q_t + kh * p.q_h, p.q_t, ch.y, p.dk);
  load_tile<4, C, THREADS>(xb_smem_u32(st.x), x, x_t, ch.y, vcols);
  const uint8_t* pt = (const uint8_t*)p.pt + ((long long)c * p.Hv + h) * (2 * TRI);
  load_bytes<THREADS>(xb_smem_u32(st.pt) + (P ? 0 : TRI), pt + (P ? 0 : TRI), P ? 2 * TRI : TRI);
  load_floats<THREADS>(xb_smem_u32(st.hd), p.hd + ((long long)c * p.Hv + h) * HD, HD);
  load_floats<THREADS>(xb_smem_u32(st.rqk), p.rqk + ((long long)c * p.Hk + kh) * RQK, RQK);
}

// B fragments of two planes of a [rows][NV] tile: 16 rows, all four column tiles
struct BFrag { uint32_t h[2][4], l[2][4]; };
__device__ __forceinline__ void load_b(BFrag& b, uint32_t hi, uint32_t lo, int k0) {
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    ldsm4t(b.h[n], hi + addr_bt<4>(k0, n * 16));
    ldsm4t(b.l[n], lo + addr_bt<4>(k0, n * 16));
  }
}
__device__ __forceinline__ void mma2(float (&d)[4][4], const uint32_t (&a)[4], const BFrag& b) {          // a exact
#pragma unroll
  for (int n = 0; n < 4; ++n) mma(d[n], a, b.l[n >> 1][(n & 1) * 2], b.l[n >> 1][(n & 1) * 2 + 1]);
#pragma unroll
  for (int n = 0; n < 4; ++n) mma(d[n], a, b.h[n >> 1][(n & 1) * 2], b.h[n >> 1][(n & 1) * 2 + 1]);
}
__device__ __forceinline__ void mma3(float (&d)[4][4], const uint32_t (&ah)[4], const uint32_t (&al)[4], const BFrag& b) {
#pragma unroll
  for (int n = 0; n < 4; ++n) mma(d[n], al, b.h[n >> 1][(n & 1) * 2], b.h[n >> 1][(n & 1) * 2 + 1]);
  mma2(d, ah, b);
}
// 64 x 32 accumulators, scaled by row, to two planes
__device__ __forceinline__ void put_planes(const float (&d)[4][4], float f0, float f1, uint32_t hi, uint32_t lo, int row0, int t) {
#pragma unroll
  for (int hh = 0; hh < 2; ++hh)
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const uint32_t off = at2<4>(row0 + hh * 8, n * 8 + 2 * t);
      const float f = hh ? f1 : f0;
      uint32_t a, b;
      split2(f * d[n][2 * hh], f * d[n][2 * hh + 1], a, b);
      sts32(hi + off, a);
      sts32(lo + off, b);
    }
}

// ---- forward -------------------------------------------------------------------------------------------------------
template <int DKP>
struct DFwdSmem {
  DStage<DKP> st[2];
  uint8_t s[2][2][DKP * NV * 2];            // the state's planes, this chunk's and the next one's
  uint8_t r[2][C * NV * 2], u[2][C * NV * 2], d[2][C * NV * 2];
};

template <int DKP, bool SAVE>
__global__ void __launch_bounds__(SAVE ? 128 : 256, 1) delta_fwd(const XbRecArgs p) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  DFwdSmem<DKP>& sm = *reinterpret_cast<DFwdSmem<DKP>*>(smem_raw);
  constexpr int U = DKP / 8, THREADS = SAVE ? 128 : 256;
  const int slices = p.dvp / NV, rep = p.Hv / p.Hk;
  const int sl = blockIdx.x % slices, h = (blockIdx.x / slices) % p.Hv, doc = blockIdx.x / (slices * p.Hv);
  const int kh = h / rep, v0 = sl * NV, vcols = min(NV, p.dv - v0);
  const int lane = xb_lane(), warp = threadIdx.x >> 5, w = warp & 3, g = lane >> 2, t = lane & 3, ra = w * 16 + g;
  const int c0 = p.doc_off[doc], c1 = p.doc_off[doc + 1];
  const int4* chunks = reinterpret_cast<const int4*>(p.chunks);
  bf16* o = (bf16*)p.o + (long long)h * p.dv + v0;
  const long long o_t = (long long)p.Hv * p.dv;
  if (doc >= p.n_docs) {                                             // rows outside the documents
    if (!SAVE)
      for (int c = c0; c < c1; ++c)
        for (int i = threadIdx.x; i < chunks[c].y * NV; i += THREADS)
          if (i % NV < vcols) o[(chunks[c].x + i / NV) * o_t + i % NV] = __float2bfloat16(0.f);
    return;
  }
  float s[DKP / 64][4][4] = {};
  const long long soff = ((long long)doc * p.Hv + h) * p.dk * p.dv + v0 * p.s_v;
  auto fetch = [&](int c, int b) {
    const int4 ch = chunks[c];
    fetch_stage<DKP, THREADS, !SAVE, !SAVE>(p, sm.st[b], ch, c, h, kh, (const bf16*)p.v + ch.x * p.v_t + h * p.v_h + v0, p.v_t, vcols);
  };
  if (c0 < c1) fetch(c0, 0);
  cp_commit();
  if (warp < 4) {
    if (p.s_in != nullptr) state_global<DKP, false>(s, const_cast<float*>(p.s_in) + soff, p.s_k, p.s_v, p.dk, vcols);
    state_to_smem<DKP>(s, xb_smem_u32(sm.s[0][0]), xb_smem_u32(sm.s[0][1]));
  }
  for (int c = c0; c < c1; ++c) {
    const int par = (c - c0) & 1;
    DStage<DKP>& st = sm.st[par];
    const uint32_t sk = xb_smem_u32(st.k), sq = xb_smem_u32(st.q), sv = xb_smem_u32(st.x), spt = xb_smem_u32(st.pt);
    const uint32_t shi = xb_smem_u32(sm.s[par][0]), slo = xb_smem_u32(sm.s[par][1]);
    const uint32_t uhi = xb_smem_u32(sm.u[0]), ulo = xb_smem_u32(sm.u[1]);
    cp_wait<0>();
    __syncthreads();                       // this chunk's tiles and the state's planes are complete
    if (c + 1 < c1) fetch(c + 1, par ^ 1);
    cp_commit();
    const long long ch_h = (long long)c * p.Hv + h;
    if (warp < 4) {
      if (SAVE) state_save<DKP>(shi, slo, (bf16*)p.s_planes + ch_h * 2 * DKP * p.dvp, p.dvp, v0);
      float acc[4][4] = {};
#pragma unroll
      for (int ks = 0; ks < DKP / 16; ++ks) {
        uint32_t fk[4];
        BFrag b;
        ldsm4(fk, sk + addr_a<U>(w * 16, ks * 16));
        load_b(b, shi, slo, ks * 16);
        mma2(acc, fk, b);
      }
      // R = b (V - gamma rk K S)
      const uint32_t rhi = xb_smem_u32(sm.r[0]), rlo = xb_smem_u32(sm.r[1]);
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int row = ra + hh * 8;
        const float b = st.hd[2 * C + row], f = ex2_sum(st.hd, row) * st.rqk[C + row];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const uint32_t off = at2<4>(row, n * 8 + 2 * t);
          const float2 v = unpack_bf16x2(lds32(sv + off));
          uint32_t hi, lo;
          split2(b * (v.x - f * acc[n][2 * hh]), b * (v.y - f * acc[n][2 * hh + 1]), hi, lo);
          sts32(rhi + off, hi);
          sts32(rlo + off, lo);
        }
      }
      bar(1, 128);
      // U = T R
      float u[4][4] = {};
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        if (ks <= w) {
          uint32_t ah[4], al[4];
          BFrag b;
          ldsm4(ah, spt + TRI + blk_of(w, ks) + addr_blk(lane));
          ldsm4(al, spt + TRI + blk_of(w, ks) + BLK + addr_blk(lane));
          load_b(b, rhi, rlo, ks * 16);
          mma3(u, ah, al, b);
        }
      }
      const uint32_t dhi = xb_smem_u32(sm.d[0]), dlo = xb_smem_u32(sm.d[1]);
      if (SAVE) {
#pragma unroll
        for (int hh = 0; hh < 2; ++hh)
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            uint32_t* pl = reinterpret_cast<uint32_t*>((bf16*)p.u_planes + (ch_h * 2 * C + ra + hh * 8) * p.dvp + v0 + n * 8 + 2 * t);
            split2(u[n][2 * hh], u[n][2 * hh + 1], pl[0], pl[C * p.dvp / 2]);
          }
      } else {
        put_planes(u, 1.f, 1.f, uhi, ulo, ra, t);
        bar_arrive(3, 256);                // the output warps may read U
      }
      put_planes(u, ex2_diff(st.hd, C - 1, ra) * st.rqk[C + ra], ex2_diff(st.hd, C - 1, ra + 8) * st.rqk[C + ra + 8], dhi, dlo, ra, t);
      const float f = ex2_sum(st.hd, C - 1);
#pragma unroll
      for (int m = 0; m < DKP / 64; ++m)
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[m][n][e] *= f;
      bar(2, 128);
      // S = gamma_last S + K^T (rk d U)
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        BFrag b;
        load_b(b, dhi, dlo, ks * 16);
#pragma unroll
        for (int m = 0; m < DKP / 64; ++m) {
          uint32_t fa[4];
          ldsm4t(fa, sk + addr_at<U>(w * (DKP / 4) + m * 16, ks * 16));
          mma2(s[m], fa, b);
        }
      }
      state_to_smem<DKP>(s, xb_smem_u32(sm.s[par ^ 1][0]), xb_smem_u32(sm.s[par ^ 1][1]));
    } else {
      // O = gamma rq Q S + P U
      const int4 ch = chunks[c];
      float acc[4][4] = {};
#pragma unroll
      for (int ks = 0; ks < DKP / 16; ++ks) {
        uint32_t fq[4];
        BFrag b;
        ldsm4(fq, sq + addr_a<U>(w * 16, ks * 16));
        load_b(b, shi, slo, ks * 16);
        mma2(acc, fq, b);
      }
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const float f = ex2_sum(st.hd, ra + hh * 8) * st.rqk[ra + hh * 8];
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[n][2 * hh] *= f, acc[n][2 * hh + 1] *= f;
      }
      bar(3, 256);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        if (ks <= w) {
          uint32_t ah[4], al[4];
          BFrag b;
          ldsm4(ah, spt + blk_of(w, ks) + addr_blk(lane));
          ldsm4(al, spt + blk_of(w, ks) + BLK + addr_blk(lane));
          load_b(b, uhi, ulo, ks * 16);
          mma3(acc, ah, al, b);
        }
      }
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
        if (ra + hh * 8 < ch.y)
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const int col = n * 8 + 2 * t;
            if (col < vcols)
              *reinterpret_cast<uint32_t*>(o + (ch.x + ra + hh * 8) * o_t + col) = pack_bf16x2(acc[n][2 * hh], acc[n][2 * hh + 1]);
          }
    }
  }
  cp_wait<0>();
  if (warp < 4 && p.s_out != nullptr) state_global<DKP, true>(s, p.s_out + soff, p.s_k, p.s_v, p.dk, vcols);
}

// ---- backward, sequential part: dS through one document, last chunk first -----------------------------------------
template <int DKP>
struct DBwdSmem {
  DStage<DKP> st[2];
  uint8_t s[2][DKP * NV * 2];               // dS'
  uint8_t u[2][C * NV * 2];                 // dU
  uint8_t x[2][C * NV * 2], y[2][C * NV * 2];   // -b gamma rk dR, gamma rq dO
};

template <int DKP>
__global__ void __launch_bounds__(256, 1) delta_bwd(const XbRecArgs p) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  DBwdSmem<DKP>& sm = *reinterpret_cast<DBwdSmem<DKP>*>(smem_raw);
  constexpr int U = DKP / 8;
  const int slices = p.dvp / NV, rep = p.Hv / p.Hk;
  const int sl = blockIdx.x % slices, h = (blockIdx.x / slices) % p.Hv, doc = blockIdx.x / (slices * p.Hv);
  const int kh = h / rep, v0 = sl * NV, vcols = min(NV, p.dv - v0);
  const int lane = xb_lane(), warp = threadIdx.x >> 5, w = warp & 3, g = lane >> 2, t = lane & 3, ra = w * 16 + g;
  const int c0 = p.doc_off[doc], c1 = p.doc_off[doc + 1];
  const int4* chunks = reinterpret_cast<const int4*>(p.chunks);
  bf16* dv = (bf16*)p.dv_out + (long long)h * p.dv + v0;
  const long long dv_t = (long long)p.Hv * p.dv;
  if (doc >= p.n_docs) {
    for (int c = c0; c < c1; ++c)
      for (int i = threadIdx.x; i < chunks[c].y * NV; i += 256)
        if (i % NV < vcols) dv[(chunks[c].x + i / NV) * dv_t + i % NV] = __float2bfloat16(0.f);
    return;
  }
  float s[DKP / 64][4][4] = {};             // warps 4 .. 7: the state's gradient
  const long long soff = ((long long)doc * p.Hv + h) * p.dk * p.dv + v0 * p.s_v;
  auto fetch = [&](int c, int b) {
    const int4 ch = chunks[c];
    fetch_stage<DKP, 256, true, true>(p, sm.st[b], ch, c, h, kh, (const bf16*)p.dy + ch.x * p.dy_t + h * p.dy_h + v0, p.dy_t, vcols);
  };
  if (c0 < c1) fetch(c1 - 1, 0);
  cp_commit();
  const uint32_t shi = xb_smem_u32(sm.s[0]), slo = xb_smem_u32(sm.s[1]), xhi = xb_smem_u32(sm.x[0]), xlo = xb_smem_u32(sm.x[1]);
  if (warp >= 4) {
    if (p.ds_out != nullptr) state_global<DKP, false>(s, const_cast<float*>(p.ds_out) + soff, p.s_k, p.s_v, p.dk, vcols);
    state_to_smem<DKP>(s, shi, slo);
  }
  for (int c = c1 - 1; c >= c0; --c) {
    DStage<DKP>& st = sm.st[(c1 - 1 - c) & 1];
    const int4 ch = chunks[c];
    const uint32_t sk = xb_smem_u32(st.k), sq = xb_smem_u32(st.q), sy = xb_smem_u32(st.x), spt = xb_smem_u32(st.pt);
    cp_wait<0>();
    __syncthreads();
    if (c > c0) fetch(c - 1, (c1 - c) & 1);
    cp_commit();
    const long long ch_h = (long long)c * p.Hv + h;
    if (warp < 4) {
      // dU = d rk K dS' + P^T dO
      float du[4][4] = {};
#pragma unroll
      for (int ks = 0; ks < DKP / 16; ++ks) {
        uint32_t fk[4];
        BFrag b;
        ldsm4(fk, sk + addr_a<U>(w * 16, ks * 16));
        load_b(b, shi, slo, ks * 16);
        mma2(du, fk, b);
      }
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const float f = ex2_diff(st.hd, C - 1, ra + hh * 8) * st.rqk[C + ra + hh * 8];
#pragma unroll
        for (int n = 0; n < 4; ++n) du[n][2 * hh] *= f, du[n][2 * hh + 1] *= f;
      }
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        if (ks >= w) {
          uint32_t ah[4], al[4], by[2][4];
          ldsm4t(ah, spt + blk_of(ks, w) + addr_blk_t(lane));
          ldsm4t(al, spt + blk_of(ks, w) + BLK + addr_blk_t(lane));
#pragma unroll
          for (int n = 0; n < 2; ++n) ldsm4t(by[n], sy + addr_bt<4>(ks * 16, n * 16));
#pragma unroll
          for (int n = 0; n < 4; ++n) mma(du[n], al, by[n >> 1][(n & 1) * 2], by[n >> 1][(n & 1) * 2 + 1]);
#pragma unroll
          for (int n = 0; n < 4; ++n) mma(du[n], ah, by[n >> 1][(n & 1) * 2], by[n >> 1][(n & 1) * 2 + 1]);
        }
      }
      const uint32_t uhi = xb_smem_u32(sm.u[0]), ulo = xb_smem_u32(sm.u[1]);
      put_planes(du, 1.f, 1.f, uhi, ulo, ra, t);
      bar(1, 128);
      // dR = T^T dU
      float dr[4][4] = {};
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        if (ks >= w) {
          uint32_t ah[4], al[4];
          BFrag b;
          ldsm4t(ah, spt + TRI + blk_of(ks, w) + addr_blk_t(lane));
          ldsm4t(al, spt + TRI + blk_of(ks, w) + BLK + addr_blk_t(lane));
          load_b(b, uhi, ulo, ks * 16);
          mma3(dr, ah, al, b);
        }
      }
      const float b0 = st.hd[2 * C + ra], b1 = st.hd[2 * C + ra + 8];
      put_planes(dr, -b0 * ex2_sum(st.hd, ra) * st.rqk[C + ra], -b1 * ex2_sum(st.hd, ra + 8) * st.rqk[C + ra + 8], xhi, xlo, ra, t);
      bar_arrive(2, 256);
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int row = ra + hh * 8;
        const float b = hh ? b1 : b0;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int col = n * 8 + 2 * t;
          const float y0 = dr[n][2 * hh], y1 = dr[n][2 * hh + 1];
          uint32_t* pl = reinterpret_cast<uint32_t*>((bf16*)p.dr_planes + (ch_h * 2 * C + row) * p.dvp + v0 + col);
          split2(y0, y1, pl[0], pl[C * p.dvp / 2]);
          if (row < ch.y && col < vcols) *reinterpret_cast<uint32_t*>(dv + (ch.x + row) * dv_t + col) = pack_bf16x2(b * y0, b * y1);
        }
      }
    } else {
      // dS = gamma_last dS' + Q^T (gamma rq dO) + K^T (-b gamma rk dR)
      const uint32_t yhi = xb_smem_u32(sm.y[0]), ylo = xb_smem_u32(sm.y[1]);
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int row = ra + hh * 8;
        const float y = ex2_sum(st.hd, row) * st.rqk[row];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const uint32_t off = at2<4>(row, n * 8 + 2 * t);
          const float2 v = unpack_bf16x2(lds32(sy + off));
          uint32_t hi, lo;
          split2(y * v.x, y * v.y, hi, lo);
          sts32(yhi + off, hi);
          sts32(ylo + off, lo);
        }
      }
      bar(3, 128);
      const float f = ex2_sum(st.hd, C - 1);
#pragma unroll
      for (int m = 0; m < DKP / 64; ++m)
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[m][n][e] *= f;
      state_save<DKP>(shi, slo, (bf16*)p.ds_planes + ch_h * 2 * DKP * p.dvp, p.dvp, v0);
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        const uint32_t a = part ? sk : sq;
        if (part) bar(2, 256);               // dR is there, and dS' has been read
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          BFrag b;
          load_b(b, part ? xhi : yhi, part ? xlo : ylo, ks * 16);
#pragma unroll
          for (int m = 0; m < DKP / 64; ++m) {
            uint32_t fa[4];
            ldsm4t(fa, a + addr_at<U>(w * (DKP / 4) + m * 16, ks * 16));
            mma2(s[m], fa, b);
          }
        }
      }
      state_to_smem<DKP>(s, shi, slo);
    }
  }
  cp_wait<0>();
  if (warp >= 4 && p.ds_in != nullptr) state_global<DKP, true>(s, p.ds_in + soff, p.s_k, p.s_v, p.dk, vcols);
}

template <int DKP>
int forward(const XbRecArgs& a, long long seq, cudaStream_t st) {
  if (int rc = rec_launch(delta_prep<DKP>, (long long)a.nc_max * a.Hk, 128, sizeof(DPrepSmem<DKP>), a, st)) return rc;
  return rec_launch(delta_fwd<DKP, false>, seq, 256, sizeof(DFwdSmem<DKP>), a, st);
}
template <int DKP>
int backward(const XbRecArgs& a, long long seq, cudaStream_t st) {
  XbRecArgs again = a;
  again.s_out = nullptr;
  if (int rc = rec_launch(delta_fwd<DKP, true>, seq, 128, sizeof(DFwdSmem<DKP>), again, st)) return rc;
  return rec_launch(delta_bwd<DKP>, seq, 256, sizeof(DBwdSmem<DKP>), a, st);
}

}  // namespace

int xb_delta_fwd(const XbRecArgs& a, cudaStream_t st) {
  const long long seq = (long long)(a.n_docs + 2) * a.Hv * (a.dvp / NV);
  return a.dk <= 64 ? forward<64>(a, seq, st) : forward<128>(a, seq, st);
}
int xb_delta_bwd(const XbRecArgs& a, cudaStream_t st) {
  const long long seq = (long long)(a.n_docs + 2) * a.Hv * (a.dvp / NV);
  return a.dk <= 64 ? backward<64>(a, seq, st) : backward<128>(a, seq, st);
}
