// The gated delta rule's own kernels: prepare, forward, and the sequential part of the backward pass (the formulas
// stand in recurrence.cu).
//
// A chunk's chain  K S -> R -> U = T R -> S' = gamma S + K^T d U  is sequential, and with one long document there are
// only heads x column slices of them (32 x 4 for 32 heads of 128), less than one per SM: the time of a step is what
// counts.  A CTA carries 32 state columns through three products per step that wait for one another:
//
//   forward   K S           -> R
//             (T - I) R     -> U = R + (T - I) R
//             K^T (d U)     -> added to the state, whose 128 rows live in the registers of 128 x 2 threads
//             Q S, P U      -> O, beside the chain
//   backward  P^T dO        -> beside the step before
//             K dS'         -> Y = d K dS' + P^T dO
//             (T - I)^T Y   -> dR = Y + (T - I)^T Y
//             [K; Q]^T [-b gamma dR; gamma dO] -> added to dS  (the dO part is issued early)
//
// A computed operand enters as two bf16 parts side by side, [hi | lo], 64 columns of one product; the parts of T and
// P are two products into the same accumulator.  The third parts of T - I, R and Y take part too, as products of 32 columns
// with the first parts of the other operand; of a call without gradients as well, so that its outputs are those of the
// call that a backward pass follows, to the bit.  P = tril(D o Q K^T) and T = (I + L)^-1 depend on the chunk alone and
// come from the prepare kernel as operand tiles, T without its diagonal of ones: what they pass on stays in 32 bits, which
// takes a fifth off the error of the decay's gradient.  Products with 64 rows lie in half of each warp's lanes and are read as
// fragments, which gives every lane values.  Eight warps work on the accumulators, one issues the products, one moves
// tiles in and out.
//
// A forward step takes 3000 cycles (with two parts 2800): three times about 450 to 500 of products and their latency, the rest
// on the way from accumulator to operand (four or sixteen warps on it: 2 % and 13 % more; mma.sync instead of tcgen05: 5800
// cycles).  32 heads of 128 x 128: forward 397 us for a document of 16384 tokens (370) and 136 us for 4096 tokens in five
// documents with their tiles kept (0.26 GB written; 125), backward 136 us (118); prepare 151 and 50 us (0.34 and 0.11 GB
// written: latencies of small steps, three CTAs per SM).
#include "recurrence_core.cuh"

namespace {

// named barriers want whole warps
__device__ __forceinline__ void bar(int id, int n) {
  __syncwarp();
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory");
}
__device__ __forceinline__ void bar_arrive(int id, int n) {
  __syncwarp();
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(n) : "memory");
}

// ---- prepare -----------------------------------------------------------------------------------------------------
// One CTA per chunk and key head, two v heads at a time with four warps each.
constexpr int PT = 256;                     // threads
constexpr int LS = 72;                      // row stride of L: rows of a fragment fall into different banks
template <int DKP>
struct DPrepSmem {
  union {
    struct { uint8_t q[C * DKP * 2], k[C * DKP * 2]; };
    float l[2][C * LS];
  };
  float2 qk[8 * 2 * 128], kk[8 * 2 * 128];  // Q K^T and K K^T as fragments, by lane of four warps
  float hd[2][3][C];
  float rq[C], rk[C], part[2][2 * C];
};

// T - I, 64 x 64 values per head, to the upper half of its operand tile: two planes of [128 rows][128 bytes] whose 16-byte
// units are swizzled as the tensor core reads them
constexpr int TP_PLANE = 128 * 128, T3 = 64 * 128, TP = 2 * TP_PLANE + T3;     // the third plane has T alone
__device__ __forceinline__ void put_tile(const XbRecArgs& p, const float (&l)[2][C * LS], int c, int h, int heads) {
  for (int it = threadIdx.x; it < 2 * C * 8; it += PT) {
    const int mm = it / (C * 8), r = (it >> 3) % C, u = it & 7;
    if (mm >= heads) break;
    const float4* src = reinterpret_cast<const float4*>(&l[mm][r * LS + u * 8]);
    const bool above = (u >> 1) > (r >> 4);            // blocks above the diagonal are not written by anybody
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    float4 a = above ? zero : src[0], b = above ? zero : src[1];
    if (u == r >> 3) {                                 // the ones of the diagonal
      const int e = r & 7;
      a.x = e == 0 ? 0.f : a.x, a.y = e == 1 ? 0.f : a.y, a.z = e == 2 ? 0.f : a.z, a.w = e == 3 ? 0.f : a.w;
      b.x = e == 4 ? 0.f : b.x, b.y = e == 5 ? 0.f : b.y, b.z = e == 6 ? 0.f : b.z, b.w = e == 7 ? 0.f : b.w;
    }
    uint4 hi, lo, third;
    split3(pair(a.x, a.y), hi.x, lo.x, third.x), split3(pair(a.z, a.w), hi.y, lo.y, third.y);
    split3(pair(b.x, b.y), hi.z, lo.z, third.z), split3(pair(b.z, b.w), hi.w, lo.w, third.w);
    uint8_t* dst = (uint8_t*)p.pt + ((long long)c * p.Hv + h + mm) * TP + r * 128 + ((u ^ (r & 7)) << 4);
    *reinterpret_cast<uint4*>(dst) = hi;
    *reinterpret_cast<uint4*>(dst + TP_PLANE) = lo;
    *reinterpret_cast<uint4*>(dst + 2 * TP_PLANE) = third;
  }
}

// d (16 x 16, two column tiles) += A B of blocks in shared memory (row stride LS).  Three bf16 parts of each operand keep
// the 24 bits of its significand, so the inverse is as exact as fp32 makes it.
__device__ __forceinline__ void split3(float x, float y, uint32_t (&p)[3]) {
  p[0] = pack_bf16x2(x, y);
  const float2 h = unpack_bf16x2(p[0]);
  x -= h.x, y -= h.y;
  p[1] = pack_bf16x2(x, y);
  const float2 m = unpack_bf16x2(p[1]);
  p[2] = pack_bf16x2(x - m.x, y - m.y);
}
__device__ __forceinline__ void block_mma(float (&d)[2][4], const float* A, const float* B) {
  const int lane = xb_lane(), g = lane >> 2, t = lane & 3;
  uint32_t a[3][4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 x = *reinterpret_cast<const float2*>(A + (g + (e & 1) * 8) * LS + (e >> 1) * 8 + 2 * t);
    uint32_t q[3];
    split3(x.x, x.y, q);
    a[0][e] = q[0], a[1][e] = q[1], a[2][e] = q[2];
  }
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const float* b = B + 2 * t * LS + n * 8 + g;
    uint32_t b0[3], b1[3];
    split3(b[0], b[LS], b0);
    split3(b[8 * LS], b[9 * LS], b1);
    mma(d[n], a[2], b0[0], b1[0]);
    mma(d[n], a[0], b0[2], b1[2]);
    mma(d[n], a[1], b0[1], b1[1]);
    mma(d[n], a[1], b0[0], b1[0]);
    mma(d[n], a[0], b0[1], b1[1]);
    mma(d[n], a[0], b0[0], b1[0]);
  }
}
__device__ __forceinline__ void block_put(float* dst, const float (&d)[2][4], float sign) {
  const int lane = xb_lane(), g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int hh = 0; hh < 2; ++hh)
      *reinterpret_cast<float2*>(dst + (g + hh * 8) * LS + n * 8 + 2 * t) = make_float2(sign * d[n][2 * hh], sign * d[n][2 * hh + 1]);
}
// L (strictly lower, two heads) becomes (I + L)^-1 in place: the four diagonal blocks by substitution, one column per
// thread, then T21 = -T22 L21 T11 for blocks of 16 and of 32.  (Substitution down all 64 rows is 2000 multiply-adds of
// straight-line code for a thread, which ran at the speed of the instruction cache: 28,000 cycles.)
__device__ __forceinline__ void invert(float (&l)[2][C * LS]) {
  const int tid = threadIdx.x, w = (tid >> 5) & 3, m = tid >> 7;
  float* L = l[m];
  const int blk = (tid & 63) >> 4, j = tid & 15;
  float* D = L + blk * 16 * (LS + 1);
  float x[16];
  if (w < 2) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s0 = i == j ? 1.f : 0.f, s1 = 0.f;
#pragma unroll
      for (int k = 0; k < i; ++k) {
        if (k & 1) s1 -= D[i * LS + k] * x[k];
        else s0 -= D[i * LS + k] * x[k];
      }
      x[i] = s0 + s1;
    }
  }
  __syncthreads();
  if (w < 2) {
#pragma unroll
    for (int i = 0; i < 16; ++i) D[i * LS + j] = x[i];
  }
  __syncthreads();
  if (w < 2) {  // blocks of 16: one pair per warp
    float* T11 = L + w * 32 * (LS + 1);
    float* L21 = T11 + 16 * LS;
    float* T22 = L21 + 16;
    float d[2][4] = {}, e[2][4] = {};
    block_mma(d, L21, T11);
    __syncwarp();
    block_put(L21, d, 1.f);
    __syncwarp();
    block_mma(e, T22, L21);
    __syncwarp();
    block_put(L21, e, -1.f);
  }
  __syncthreads();
  {  // blocks of 32: a warp has 16 of the 32 rows and 16 of the 32 columns
    const int i = w & 1, c = w >> 1;
    float* row = L + (32 + 16 * i) * LS;
    const float* M = L + 32 * LS + 16 * c;
    float d[2][4] = {}, e[2][4] = {};
    if (c == 0) block_mma(d, row, L);
    block_mma(d, row + 16, L + 16 * LS + 16 * c);
    __syncthreads();
    block_put(row + 16 * c, d, 1.f);
    __syncthreads();
    block_mma(e, row + 32, M);
    if (i) block_mma(e, row + 48, M + 16 * LS);
    __syncthreads();
    block_put(row + 16 * c, e, -1.f);
  }
  __syncthreads();
}

template <int DKP>
__global__ void __launch_bounds__(PT, 3) delta_prep(const XbRecArgs p) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  DPrepSmem<DKP>& sm = *reinterpret_cast<DPrepSmem<DKP>*>(smem_raw);
  constexpr int U = DKP / 8;
  const int kh = blockIdx.x % p.Hk, c = blockIdx.x / p.Hk;
  const int tid = threadIdx.x, lane = tid & 31, w = (tid >> 5) & 3, m = tid >> 7, g = lane >> 2, t = lane & 3;
  if (c >= p.doc_off[p.n_docs + 2]) return;
  const int4 ch = reinterpret_cast<const int4*>(p.chunks)[c];
  if (ch.z >= p.n_docs) return;
  const int len = ch.y, rep = p.Hv / p.Hk;
  const uint32_t sq = xb_smem_u32(sm.q), sk = xb_smem_u32(sm.k);
  load_tile<U, C, PT>(sq, (const bf16*)p.q + ch.x * p.q_t + kh * p.q_h, p.q_t, len, p.dk);
  load_tile<U, C, PT>(sk, (const bf16*)p.k + ch.x * p.k_t + kh * p.k_h, p.k_t, len, p.dk);
  cp_commit();
  // the first warp of each head's four owns its running decay: two rows per lane
  float gv[2] = {}, bv[2] = {};
  auto read_head = [&](int hh) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = 2 * lane + i;
      gv[i] = bv[i] = 0.f;
      if (w == 0 && hh < rep && row < len) {
        const long long tok = ch.x + row;
        gv[i] = p.g[tok * p.g_t + (kh * rep + hh) * p.g_h];
        bv[i] = p.b[tok * p.b_t + (kh * rep + hh) * p.b_h];
      }
    }
  };
  read_head(m);
  cp_wait<0>();
  __syncthreads();
  if (p.l2norm) {  // sums of squares: two threads per row of q and of k
    const int row = tid & 63, half = m;
    const uint32_t base = tid & 64 ? sk : sq;
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int u = 0; u < U / 2; ++u) {
      const uint4 v = lds128(base + swz<U>(row, half * (U / 2) + u));
      const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack_bf16x2(x[i]);
        s0 += f.x * f.x, s1 += f.y * f.y;
      }
    }
    sm.part[half][tid & 127] = s0 + s1;
    __syncthreads();
  }
  if (tid < 2 * C) {
    const int row = tid & 63;
    float r = p.l2norm ? 1.f / fmaxf(sqrtf(sm.part[0][tid] + sm.part[1][tid]), 1e-12f) : 1.f;
    if (tid < C) r *= p.scale;
    if (row >= len) r = 0.f;
    (tid < C ? sm.rq : sm.rk)[row] = r;
    p.rqk[((long long)c * p.Hk + kh) * RQK + tid] = r;
  }
  __syncthreads();
  const int r0 = w * 16 + g;
  {  // Q K^T by the first four warps, K K^T by the others
    float* out = m ? p.kk : p.qk;
    if (out != nullptr) out += ((long long)c * p.Hk + kh) * (C * C);
    const uint32_t sa = m ? sk : sq;
    const float* ra = m ? sm.rk : sm.rq;
    float2* keep = m ? sm.kk : sm.qk;
#pragma unroll
    for (int nt = 0; nt < 8; nt += 2) {
      if (nt * 8 > w * 16 + 15) break;              // columns above the diagonal block are never read
      float a1[2][4] = {};
#pragma unroll
      for (int ks = 0; ks < DKP / 16; ++ks) {
        uint32_t fa[4], fb[4];
        ldsm4(fb, sk + addr_b<U>(nt * 8, ks * 16));
        ldsm4(fa, sa + addr_a<U>(w * 16, ks * 16));
        mma(a1[0], fa, fb[0], fb[1]);
        mma(a1[1], fa, fb[2], fb[3]);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const int row = r0 + hh * 8, col = (nt + j) * 8 + 2 * t;
          const float2 rc = *reinterpret_cast<const float2*>(&sm.rk[col]);
          const float2 x = make_float2(ra[row] * rc.x * a1[j][2 * hh], ra[row] * rc.y * a1[j][2 * hh + 1]);
          keep[((nt + j) * 2 + hh) * 128 + w * 32 + lane] = x;
          if (out != nullptr) *reinterpret_cast<float2*>(out + row * C + col) = x;
        }
    }
  }
  for (int h0 = 0; h0 < rep; h0 += 2) {
    const bool on = h0 + m < rep;
    if (w == 0 && on) {
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
      float* out = p.hd + ((long long)c * p.Hv + kh * rep + h0 + m) * HD;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = 2 * lane + i;
        const double G = i ? s : s - x[1];
        const float hi = (float)G, lo = (float)(G - (double)hi);
        out[row] = hi, out[C + row] = lo, out[2 * C + row] = bv[i];
        sm.hd[m][0][row] = hi, sm.hd[m][1][row] = lo, sm.hd[m][2][row] = bv[i];
      }
    }
    read_head(h0 + 2 + m);
    __syncthreads();                              // also: the tiles, or the pair before, have been read
    if (on) {
      const float* hd = sm.hd[m][0];
      // P as the lower half of the operand tile, L for the inverse
      uint8_t* tile = (uint8_t*)p.pt + ((long long)c * p.Hv + kh * rep + h0 + m) * TP + C * 128;
      float gh[2], gl[2], bb[2];
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) gh[hh] = hd[r0 + hh * 8], gl[hh] = hd[C + r0 + hh * 8], bb[hh] = hd[2 * C + r0 + hh * 8];
#pragma unroll
      for (int nt = 0; nt < 8; ++nt) {
        const int col = nt * 8 + 2 * t;
        const bool above = nt > 2 * w + 1;            // blocks above the diagonal
        const float2 ch = *reinterpret_cast<const float2*>(hd + col), cl = *reinterpret_cast<const float2*>(hd + C + col);
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const int row = r0 + hh * 8;
          uint32_t hi = 0, lo = 0;
          if (!above) {
            const float2 x = sm.qk[(nt * 2 + hh) * 128 + w * 32 + lane], y = sm.kk[(nt * 2 + hh) * 128 + w * 32 + lane];
            const float d0 = xb_ex2((gh[hh] - ch.x) + (gl[hh] - cl.x)), d1 = xb_ex2((gh[hh] - ch.y) + (gl[hh] - cl.y)), b = bb[hh];
            split2(col <= row ? d0 * x.x : 0.f, col + 1 <= row ? d1 * x.y : 0.f, hi, lo);
            *reinterpret_cast<float2*>(&sm.l[m][row * LS + col]) =
                make_float2(col < row ? b * d0 * y.x : 0.f, col + 1 < row ? b * d1 * y.y : 0.f);
          }
          uint8_t* dst = tile + row * 128 + ((nt ^ (row & 7)) << 4) + t * 4;
          *reinterpret_cast<uint32_t*>(dst) = hi;
          *reinterpret_cast<uint32_t*>(dst + TP_PLANE) = lo;
        }
      }
    }
    __syncthreads();
    invert(sm.l);                                 // of a missing second head: values that nobody reads
    put_tile(p, sm.l, c, kh * rep + h0, rep - h0);
  }
}

// ---- the step of both directions ------------------------------------------------------------------------------------
// HALF: [128 rows][64 bf16], K rows 0 .. 63, Q rows 64 .. 127
constexpr int ST_KQ = 0, ST_TP = 2 * HALF, ST_X = ST_TP + 2 * TP_PLANE, ST_HD = ST_X + C * NV * 2, ST_RQK = ST_HD + HD * 4;
constexpr int ST_T3 = (ST_RQK + RQK * 4 + 1023) / 1024 * 1024, ST_V = ST_T3 + T3;      // T's third plane; v beside dO, backward
constexpr int STAGE_BYTES = ST_RQK + RQK * 4;      // what the loads bring, boxes outside a tensor included; T3 and v besides
// Shared memory.  Backward: two stages, operand tiles of 128 rows.  Forward: tiles of 64 rows; two stages, or one and two
// CTAs per SM, where U takes the place of R, which T R has read by then (P U is complete before the next R).
template <bool BWD, int STAGES>
struct Lay {
  static constexpr int ROWS = BWD ? HALF : HALF / 2, STAGE = BWD ? ST_V + C * NV * 2 : ST_V;
  static constexpr int SM_S = STAGES * STAGE, SM_B2 = SM_S + HALF, SM_B3 = SM_B2 + ROWS, SM_U = STAGES == 2 ? SM_B3 + ROWS : SM_B2,
                       SM_BAR = STAGES == 2 ? SM_U + HALF / 2 : SM_B3 + ROWS;
  static constexpr int SMEM = SM_BAR + 128 + 1024;
};
constexpr int NB = 2;                        // units of 8 columns per worker
constexpr int WORKERS = 128 * (NV / 8 / NB), ISSUER = WORKERS / 32, LOADER = ISSUER + 1, THREADS = WORKERS + 64;
constexpr int MEET = WORKERS + 32;           // workers and the issuing warp
// Accumulators, 64 columns each: those of the three products of the chain and Q S, or P^T dO.  Forward with one CTA per SM,
// Q S of the next step and P U have their own, and O is written behind R; else P U takes the place of T R, which has been
// read by then, and O is written before R.
constexpr int D1 = 0, D2 = 64, D3 = 128, D4 = 192, D5 = 256, D6 = 320;

struct __align__(8) Bars {
  uint64_t full[2], done[4], free[2], kept;
  uint32_t tmem;
  int abort_flag;
};
static_assert(sizeof(Bars) <= 128, "barriers");

// What every thread of a step knows.
struct Cta {
  uint8_t* smem;
  Bars* bars;
  uint32_t tmem, sm;                         // tensor memory, shared memory
  int h, kh, doc, v0, vcols, c0, c1;
  int sm_s, sm_u;
  int* status;
  __device__ void wait1(uint64_t* b, uint32_t parity, int detail) {         // one thread
    rec_wait(b, parity, &bars->abort_flag, status, detail);
  }
  __device__ void wait(uint64_t* b, uint32_t parity, int detail) {          // a whole warp: what follows is collective
    wait1(b, parity, detail);
    __syncwarp();
  }
};

// The loads of one chunk, by one thread.
__device__ __forceinline__ void load_stage(const XbRecArgs& p, const Cta& a, const CUtensorMap* mk, const CUtensorMap* mq,
                                           const CUtensorMap* mx, const CUtensorMap* mv, int c, uint8_t* st, uint64_t* full) {
  const int t0 = reinterpret_cast<const int4*>(p.chunks)[c].x;
  const uint8_t* tp = (const uint8_t*)p.pt + ((long long)c * p.Hv + a.h) * TP;
  mbar_expect_tx(full, STAGE_BYTES + T3 + (mv ? C * NV * 2 : 0));
  if (mv) tma_load_3d(st + ST_V, mv, full, a.v0, a.h, t0);
  bulk_load(st + ST_T3, tp + 2 * TP_PLANE, T3, full);
  for (int i = 0; i < 2; ++i) {
    tma_load_3d(st + ST_KQ + i * HALF, mk, full, i * 64, a.kh, t0);
    tma_load_3d(st + ST_KQ + i * HALF + HALF / 2, mq, full, i * 64, a.kh, t0);
  }
  tma_load_3d(st + ST_X, mx, full, a.v0, a.h, t0);
  bulk_load(st + ST_TP, tp, 2 * TP_PLANE, full);
  bulk_load(st + ST_HD, p.hd + ((long long)c * p.Hv + a.h) * HD, HD * 4, full);
  bulk_load(st + ST_RQK, p.rqk + ((long long)c * p.Hk + a.kh) * RQK, RQK * 4, full);
}

// The state tile of chunk `cs` and the 64-row tile of chunk `cu` to global memory, as they are (-1: none).
__device__ __forceinline__ void keep_tiles(const XbRecArgs& p, const Cta& a, void* states, void* rows, int cs, int cu) {
  const int slices = p.dvp / NV, sl = a.v0 / NV;
  if (cs >= 0) bulk_store((uint8_t*)states + (((long long)cs * p.Hv + a.h) * slices + sl) * HALF, a.smem + a.sm_s, HALF);
  if (cu >= 0) bulk_store((uint8_t*)rows + (((long long)cu * p.Hv + a.h) * slices + sl) * (HALF / 2), a.smem + a.sm_u, HALF / 2);
  tma_store_commit();
  tma_store_wait_read<0>();
  mbar_arrive(&a.bars->kept);
}

// Rows of K and Q behind the document's end: they hold the next document's, and 0 x Inf is NaN.
__device__ __forceinline__ void clear_rows(uint32_t st, int len) {
  const int n = (C - len) * 8;
  for (int i = threadIdx.x; i < 4 * n; i += WORKERS) {
    const int part = i / n, r = len + (i % n) / 8;
    sts128(st + ST_KQ + part * (HALF / 2) + r * 128 + (i & 7) * 16, 0, 0, 0, 0);
  }
}

// Workers: of the state a row and 8 NB columns per thread (warp w: rows 32 (w % 4) .., columns 8 NB (w / 4) ..), of what has
// 64 rows 16 rows and 8 NB columns per warp, as fragments: of every 8 columns rows g and g + 8, columns 2 t and 2 t + 1,
// element 4 n + 2 h + column.  An operand tile's row is 128 bytes, [hi 32 | lo 32]; u0 is the warp's first unit of it.
__device__ __forceinline__ void put_row(uint32_t tile, int row, int u0, const Pair (&x)[4 * NB]) {
  const uint32_t r = tile + row * 128;
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) split2(x[4 * n + i], hi[i], lo[i]);
    sts128(r + (((u0 + n) ^ (row & 7)) << 4), hi[0], hi[1], hi[2], hi[3]);
    sts128(r + (((u0 + n + 4) ^ (row & 7)) << 4), lo[0], lo[1], lo[2], lo[3]);
  }
}
// this lane's address of a warp's 16 rows and first 8 columns, hi and lo; a unit further is the address ^ 16 (u0 is even)
__device__ __forceinline__ uint32_t frag_addr(uint32_t tile, int r0, int u0) {
  const int l = xb_lane(), row = r0 + (l & 15), u = u0 + (l >> 4) * 4;
  return tile + row * 128 + ((u ^ (row & 7)) << 4);
}
__device__ __forceinline__ void put_frag(uint32_t addr, const Pair (&x)[2 * NB]) {
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    uint32_t hi[2], lo[2];
    split2(x[2 * n], hi[0], lo[0]), split2(x[2 * n + 1], hi[1], lo[1]);
    stsm4(addr ^ (n << 4), hi[0], hi[1], lo[0], lo[1]);
  }
}
// Three parts: the first two as above, the third as an operand tile of its own (units 0 .. 3) or to global memory.
__device__ __forceinline__ void put_frag3(uint32_t addr, const Pair (&x)[2 * NB], uint32_t (&third)[2 * NB]) {
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    uint32_t hi[2], lo[2];
    split3(x[2 * n], hi[0], lo[0], third[2 * n]), split3(x[2 * n + 1], hi[1], lo[1], third[2 * n + 1]);
    stsm4(addr ^ (n << 4), hi[0], hi[1], lo[0], lo[1]);
  }
}
__device__ __forceinline__ uint32_t third_addr(uint32_t tile, int r0, int u0) {
  const int l = xb_lane(), row = r0 + (l & 15);
  return tile + row * 128 + (((u0 + (l >> 4)) ^ (row & 7)) << 4);
}
// 8 KB tiles of 64 columns; lanes t and t ^ 1 trade as in store_frag.  `row`: r0 + frag_row(), u: the warp's first unit.
__device__ __forceinline__ void keep_third(uint8_t* tile, int row, int u, const uint32_t (&third)[2 * NB]) {
  const bool odd = xb_lane() & 1;
#pragma unroll
  for (int m = 0; m < NB; ++m) {
    const uint32_t other = __shfl_xor_sync(0xffffffffu, odd ? third[2 * m] : third[2 * m + 1], 1);
    *reinterpret_cast<uint2*>(tile + row * 128 + (((u + m) ^ (row & 7)) << 4) + 8 * ((xb_lane() >> 1) & 1)) =
        odd ? make_uint2(other, third[2 * m + 1]) : make_uint2(third[2 * m], other);
  }
}
static_assert(NB == 2, "one stmatrix for a warp's third parts");
// the sum of an accumulator's two halves
template <int N>
__device__ __forceinline__ void add_halves(const uint32_t (&a)[2 * N], const uint32_t (&b)[2 * N], Pair (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = pair(a[2 * i], a[2 * i + 1]) + pair(b[2 * i], b[2 * i + 1]);
}
__device__ __forceinline__ void read_rows(uint32_t addr, Pair (&x)[4 * NB]) {
  uint32_t a[8 * NB], b[8 * NB];
  tmem_ld_32x16(addr, a);
  tmem_ld_32x16(addr + 32, b);
  tc_wait_ld();
  add_halves(a, b, x);
}
__device__ __forceinline__ void read_frag(uint32_t addr, Pair (&x)[2 * NB]) {
  uint32_t a[4 * NB], b[4 * NB];
  tmem_ld_frag(addr, a);
  tmem_ld_frag(addr + 32, b);
  tc_wait_ld();
  add_halves(a, b, x);
}
__device__ __forceinline__ Pair twice(float x) { return pair(x, x); }
__device__ __forceinline__ Pair bf16_pair(uint32_t v) { return pair(v << 16, v & 0xffff0000u); }
// A warp's 16 rows to global memory as bf16: lanes t and t ^ 1 trade, for four columns of one row each.  `dst` is row
// frag_row() at the warp's first column; `cols` are left from there.
__device__ __forceinline__ int frag_row() { return (xb_lane() >> 2) + 8 * (xb_lane() & 1); }
__device__ __forceinline__ void store_frag(bf16* dst, bool on, int cols, const Pair (&x)[2 * NB]) {
  const bool odd = xb_lane() & 1;
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const float2 r0 = both(x[2 * n]), r1 = both(x[2 * n + 1]);
    const uint32_t w0 = pack_bf16x2(r0.x, r0.y), w1 = pack_bf16x2(r1.x, r1.y);
    const uint32_t other = __shfl_xor_sync(0xffffffffu, odd ? w0 : w1, 1);
    if (on && 8 * n < cols) *reinterpret_cast<uint2*>(dst + 8 * n + 4 * ((xb_lane() >> 1) & 1)) = odd ? make_uint2(other, w1) : make_uint2(w0, other);
  }
}
// a thread's part of a state row in global memory
__device__ __forceinline__ void state_row(float* base, long long sk, long long sv, int row, int dk, int col, int cols, bool store, Pair (&s)[4 * NB]) {
  if (row >= dk) return;
#pragma unroll
  for (int i = 0; i < 2 * NB; ++i) {
    if (col + 4 * i >= cols) return;                                 // columns come in multiples of 8
    float* at = base + row * sk + (col + 4 * i) * sv;
    if (store) {
      const float2 a = both(s[2 * i]), b = both(s[2 * i + 1]);
      if (sv == 1) *reinterpret_cast<float4*>(at) = make_float4(a.x, a.y, b.x, b.y);
      else at[0] = a.x, at[sv] = a.y, at[2 * sv] = b.x, at[3 * sv] = b.y;
    } else {
      const float4 v = sv == 1 ? *reinterpret_cast<const float4*>(at) : make_float4(at[0], at[sv], at[2 * sv], at[3 * sv]);
      s[2 * i] = pair(v.x, v.y), s[2 * i + 1] = pair(v.z, v.w);
    }
  }
}

constexpr uint64_t KMAJ = xb_smem_desc_base_sw128(16, 1024), MNMAJ = xb_smem_desc_base_sw128(HALF, 1024);

__device__ __forceinline__ bool cta_setup(const XbRecArgs& p, Cta& a, uint8_t* raw, int sm_s, int sm_u, int sm_bar) {
  const int slices = p.dvp / NV, rep = p.Hv / p.Hk;
  a.smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  a.bars = reinterpret_cast<Bars*>(a.smem + sm_bar);
  a.sm = xb_smem_u32(a.smem), a.sm_s = sm_s, a.sm_u = sm_u;
  const int sl = blockIdx.x % slices;
  a.h = (blockIdx.x / slices) % p.Hv, a.doc = rec_doc(p, blockIdx.x / (slices * p.Hv)), a.kh = a.h / rep;
  a.v0 = sl * NV, a.vcols = min(NV, p.dv - a.v0);
  a.c0 = a.c1 = 0;
  if (a.doc >= 0) a.c0 = p.doc_off[a.doc], a.c1 = p.doc_off[a.doc + 1];
  a.status = p.status;
  return a.doc >= 0 && a.doc < p.n_docs;
}
template <int COLS>
__device__ __forceinline__ void cta_begin(Cta& a) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) mbar_init(&a.bars->full[i], 1), mbar_init(&a.bars->free[i], 1);
    for (int i = 0; i < 4; ++i) mbar_init(&a.bars->done[i], 1);
    mbar_init(&a.bars->kept, 1);
    a.bars->abort_flag = 0;
    mbar_fence_init();
  }
  if (threadIdx.x / 32 == ISSUER) {
    tmem_alloc(&a.bars->tmem, COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  a.tmem = a.bars->tmem;
}
template <int COLS>
__device__ __forceinline__ void cta_end(Cta& a) {
  // after a wait that ran out, loads and products may still be on their way: give them 0.2 s
  if (*(volatile int*)&a.bars->abort_flag && threadIdx.x == 0)
    for (const uint64_t t0 = xb_globaltimer(); xb_globaltimer() - t0 < 200000000ull;) {}
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x / 32 == ISSUER) {
    tc_fence_after();
    tmem_dealloc(a.tmem, COLS);
  }
}
// A descriptor `bytes` further on.
__device__ __forceinline__ uint64_t ahead(uint64_t desc, int bytes) { return desc + (uint64_t)(bytes >> 4); }
// rows outside the documents: zeros
__device__ __forceinline__ void zero_rows(const XbRecArgs& p, const Cta& a, bf16* out, long long ld) {
  const int4* chunks = reinterpret_cast<const int4*>(p.chunks);
  for (int c = a.c0; c < a.c1; ++c)
    for (int i = threadIdx.x; i < chunks[c].y * NV; i += THREADS)
      if (i % NV < a.vcols) out[(chunks[c].x + i / NV) * ld + i % NV] = __float2bfloat16(0.f);
}

// Workers tell the issuing warp through barriers 1 (state tile and this chunk's loads), 2 and 3 (operands of the second
// and third product) and 4 (of the one beside the chain) that operands are written, and learn through done[0 .. 3] that a
// product is complete.  A wait that runs out raises a flag; everybody then walks through the remaining steps without
// waiting, so that no barrier is left with a thread missing.

// OUT: outputs are wanted.  SAVE: the tiles of the states and of U go to global memory.
template <bool OUT, bool SAVE, int STAGES>
__global__ void __launch_bounds__(THREADS, 3 - STAGES)
delta_fwd(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mv,
          const __grid_constant__ CUtensorMap, const __grid_constant__ XbRecArgs p) {
  using L = Lay<false, STAGES>;
  extern __shared__ uint8_t smem_raw[];
  Cta a;
  const bool inside = cta_setup(p, a, smem_raw, L::SM_S, L::SM_U, L::SM_BAR);
  bf16* o = (bf16*)p.o + (long long)a.h * p.dv + a.v0;
  const long long o_t = (long long)p.Hv * p.dv;
  if (!inside) {
    if (OUT) zero_rows(p, a, o, o_t);
    return;
  }
  static_assert(STAGES == 2 || (OUT && !SAVE), "one stage: U lies over R, and the wait for P U frees both");
  constexpr bool LATE = STAGES == 2;         // where O is written
  constexpr int COLS = LATE ? 512 : 256, DPU = LATE ? D5 : D2;
  cta_begin<COLS>(a);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int4* chunks = reinterpret_cast<const int4*>(p.chunks);
  constexpr int FIRST = MEET + (SAVE ? 32 : 0);    // whom barrier 1 brings together
  if (warp == LOADER) {
    const bool one = xb_elect_one();
    const int steps = a.c1 - a.c0;
    for (int n = 0; n < STAGES; ++n)
      if (one && n < steps) load_stage(p, a, &mk, &mq, &mv, nullptr, a.c0 + n, a.smem + n * L::STAGE, &a.bars->full[n]);
    for (int n = 0; n < steps; ++n) {
      if (SAVE) {
        bar(1, FIRST);
        if (one) keep_tiles(p, a, p.s_tiles, p.u_tiles, a.c0 + n, n > 0 ? a.c0 + n - 1 : -1);
      }
      // The stage is free when the chunk's last product has read it.  A barrier per stage: without tiles to keep nothing else
      // holds this warp to the walk's pace, and of one barrier for all chunks it could miss a phase.
      if (one && n + STAGES < steps) {
        a.wait1(&a.bars->free[n % STAGES], (n / STAGES) & 1, 2);
        load_stage(p, a, &mk, &mq, &mv, nullptr, a.c0 + n + STAGES, a.smem + (n % STAGES) * L::STAGE, &a.bars->full[n % STAGES]);
      }
      __syncwarp();
    }
    if (SAVE && steps > 0) {
      bar(1, FIRST);
      if (one) keep_tiles(p, a, p.s_tiles, p.u_tiles, -1, a.c1 - 1);
    }
  } else if (warp == ISSUER) {
    const bool one = xb_elect_one();
    constexpr uint32_t id = xb_idesc(1, 1, 64, 64, 0, 1), idh = xb_idesc(1, 1, 64, 32, 0, 1);
    const uint64_t b1 = xb_smem_desc(MNMAJ, a.sm + L::SM_S), b2 = xb_smem_desc(MNMAJ, a.sm + L::SM_B2), b3 = xb_smem_desc(MNMAJ, a.sm + L::SM_B3),
                   u = xb_smem_desc(MNMAJ, a.sm + L::SM_U);
    const int ksteps = (p.dk + 15) / 16;           // columns of K and Q behind dk are zeros
    for (int n = 0; n < a.c1 - a.c0; ++n) {
      const uint32_t st = a.sm + (n % STAGES) * L::STAGE;
      const uint64_t kq = xb_smem_desc(KMAJ, st + ST_KQ), kt = xb_smem_desc(MNMAJ, st + ST_KQ), tp = xb_smem_desc(KMAJ, st + ST_TP);
      if (one) a.wait1(&a.bars->full[n % STAGES], (n / STAGES) & 1, 1);
      bar(1, FIRST);
      if (one) {
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < ksteps) tc_mma_f16_ss(a.tmem + D1, ahead(kq, (k >> 2) * HALF + (k & 3) * 32), ahead(b1, k * 2048), id, k > 0);
        tc_commit(&a.bars->done[0]);
      }
      bar(2, MEET);
      if (one) {
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < 8; ++k)
          tc_mma_f16_ss(a.tmem + D2, ahead(tp, (k >> 2) * TP_PLANE + (k & 3) * 32), ahead(b2, (k & 3) * 2048), id, k > 0);
        // the third parts, with the first ones of the other operand
        const uint64_t t3 = xb_smem_desc(KMAJ, st + ST_T3);
#pragma unroll
        for (int k = 0; k < 4; ++k) tc_mma_f16_ss(a.tmem + D2, ahead(t3, k * 32), ahead(b2, k * 2048), idh, 1);
#pragma unroll
        for (int k = 0; k < 4; ++k) tc_mma_f16_ss(a.tmem + D2, ahead(tp, k * 32), ahead(b3, k * 2048), idh, 1);
        tc_commit(&a.bars->done[1]);
        if (OUT) {
#pragma unroll
          for (int k = 0; k < 8; ++k)        // Q S: nobody waits for it
            if (k < ksteps)
              tc_mma_f16_ss(a.tmem + (LATE && (n & 1) ? D6 : D4), ahead(kq, HALF / 2 + (k >> 2) * HALF + (k & 3) * 32), ahead(b1, k * 2048), id, k > 0);
        }
      }
      bar(3, MEET);
      if (one) {
        tc_fence_after();
        constexpr uint32_t id3 = xb_idesc(1, 1, 128, 64, 1, 1);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          tc_mma_f16_ss(a.tmem + D3, ahead(kt, k * 2048), ahead(b3, k * 2048), id3, k > 0);
        tc_commit(&a.bars->done[2]);
        if (!OUT && n + STAGES < a.c1 - a.c0) tc_commit(&a.bars->free[n % STAGES]);
      }
      if (OUT) {
        bar(4, MEET);
        if (one) {
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < 8; ++k)
            tc_mma_f16_ss(a.tmem + DPU, ahead(tp, HALF / 2 + (k >> 2) * TP_PLANE + (k & 3) * 32), ahead(u, (k & 3) * 2048), id, k > 0);
          tc_commit(&a.bars->done[3]);
          if (n + STAGES < a.c1 - a.c0) tc_commit(&a.bars->free[n % STAGES]);
        }
      }
      __syncwarp();
    }
    if (SAVE && a.c0 < a.c1) bar(1, FIRST);
  } else {
    const int q4 = warp & 3, part = warp >> 2, r = q4 * 32 + lane, r0 = q4 * 16, g = lane >> 2;
    const int row[2] = {r0 + g, r0 + g + 8}, u0 = part * NB, fcol = u0 * 8, orow = r0 + frag_row();
    const uint32_t quad = a.tmem + ((uint32_t)(q4 * 32) << 16) + fcol;
    const uint32_t f2 = frag_addr(a.sm + L::SM_B2, r0, u0), f3 = frag_addr(a.sm + L::SM_B3, r0, u0), fu = frag_addr(a.sm + L::SM_U, r0, u0),
                   t3 = third_addr(a.sm + L::SM_B3, r0, u0);
    const long long soff = ((long long)a.doc * p.Hv + a.h) * p.dk * p.dv + a.v0 * p.s_v;
    Pair s[4 * NB];
#pragma unroll
    for (int e = 0; e < 4 * NB; ++e) s[e] = twice(0.f);
    if (p.s_in != nullptr) state_row(const_cast<float*>(p.s_in) + soff, p.s_k, p.s_v, r, p.dk, fcol, a.vcols, false, s);
    // O = gamma rq Q S + P U of a chunk
    auto finish = [&](int n, int4 ch, const float (&f)[2]) {
      a.wait(&a.bars->done[3], n & 1, 7);
      tc_fence_after();
      uint32_t v[4][4 * NB];
      Pair y[2 * NB], x[2 * NB];
      const uint32_t qs = quad + (LATE && (n & 1) ? D6 : D4);
      tmem_ld_frag(qs, v[0]), tmem_ld_frag(qs + 32, v[1]);
      tmem_ld_frag(quad + DPU, v[2]), tmem_ld_frag(quad + DPU + 32, v[3]);
      tc_wait_ld();
      add_halves(v[0], v[1], y), add_halves(v[2], v[3], x);
#pragma unroll
      for (int e = 0; e < 2 * NB; ++e) x[e] = fma2(twice(f[e & 1]), y[e], x[e]);
      store_frag(o + (long long)(ch.x + orow) * o_t + fcol, orow < ch.y, a.vcols - fcol, x);
      tc_fence_before();
      __syncwarp();
    };
    const int steps = a.c1 - a.c0;
    int4 ch = steps > 0 ? chunks[a.c0] : make_int4(0, 0, 0, 0), old = ch;
    float fo[2] = {};                        // gamma rq of the chunk before
    for (int n = 0; n < steps; ++n) {
      const uint32_t st = a.sm + (n % STAGES) * L::STAGE, hd = st + ST_HD, rqk = st + ST_RQK;
      put_row(a.sm + L::SM_S, r, u0, s);
      if (ch.y < C) {
        a.wait(&a.bars->full[n % STAGES], (n / STAGES) & 1, 3);
        clear_rows(st, ch.y);
      }
      fence_proxy_async_smem();
      tc_fence_before();
      bar_arrive(1, FIRST);
      a.wait(&a.bars->full[n % STAGES], (n / STAGES) & 1, 3);
      if (OUT && !LATE && n > 0) finish(n - 1, old, fo);
      // row factors, and v, while the first product runs
      const float last = ex2_sum(hd, C - 1);
      float f[2], b[2], dec[2], fn[2];
      uint32_t v[NB][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int i = row[h];
        const float gam = ex2_sum(hd, i), rk = ldsf(rqk + (C + i) * 4);
        f[h] = gam * rk, b[h] = ldsf(hd + (2 * C + i) * 4), dec[h] = ex2_diff(hd, C - 1, i) * rk;
        fn[h] = gam * ldsf(rqk + i * 4);
#pragma unroll
        for (int m = 0; m < NB; ++m) v[m][h] = i < ch.y ? lds32(st + ST_X + swz<4>(i, u0 + m) + (lane & 3) * 4) : 0u;
      }
      const int4 now = ch;
      if (n + 1 < steps) ch = chunks[a.c0 + n + 1];
      Pair x[2 * NB], z[2 * NB];
      a.wait(&a.bars->done[0], n & 1, 4);
      tc_fence_after();
      read_frag(quad + D1, x);
#pragma unroll
      for (int e = 0; e < 2 * NB; ++e)       // R = b (V - gamma rk K S)
        x[e] = twice(b[e & 1]) * fma2(twice(-f[e & 1]), x[e], bf16_pair(v[e >> 1][e & 1]));
      uint32_t third[2 * NB];
      put_frag3(f2, x, third);               // R's third part where d U comes afterwards
      stsm4(t3, third[0], third[1], third[2], third[3]);
      fence_proxy_async_smem();
      tc_fence_before();
      bar_arrive(2, MEET);
      if (OUT && LATE && n > 0) finish(n - 1, old, fo);
      old = now, fo[0] = fn[0], fo[1] = fn[1];
      a.wait(&a.bars->done[1], n & 1, 5);
      tc_fence_after();
      read_frag(quad + D2, z);               // d rk U, then U itself
#pragma unroll
      for (int e = 0; e < 2 * NB; ++e) x[e] = x[e] + z[e];
#pragma unroll
      for (int e = 0; e < 2 * NB; ++e) z[e] = twice(dec[e & 1]) * x[e];
      put_frag(f3, z);
      fence_proxy_async_smem();
      tc_fence_before();
      bar_arrive(3, MEET);
      if (SAVE) a.wait(&a.bars->kept, n & 1, 8);          // the tiles on their way out have been read
      if (SAVE) {
        put_frag3(fu, x, third);
        keep_third((uint8_t*)p.r_tiles + (((long long)(a.c0 + n) * p.Hv + a.h) * (p.dvp / 64) + (a.v0 >> 6)) * HALF, orow,
                   ((a.v0 >> 3) & 7) + u0, third);
      } else {
        put_frag(fu, x);
      }
      fence_proxy_async_smem();
      if (OUT) bar_arrive(4, MEET);
      a.wait(&a.bars->done[2], n & 1, 6);
      tc_fence_after();
      Pair d[4 * NB];
      read_rows(quad + D3, d);
#pragma unroll
      for (int e = 0; e < 4 * NB; ++e) s[e] = fma2(twice(last), s[e], d[e]);
    }
    if (OUT && steps > 0) finish(steps - 1, old, fo);
    if (SAVE && steps > 0) bar_arrive(1, FIRST);
    if (p.s_out != nullptr) state_row(p.s_out + soff, p.s_k, p.s_v, r, p.dk, fcol, a.vcols, true, s);
  }
  cta_end<COLS>(a);
}

// dS through one document, last chunk first.
__global__ void __launch_bounds__(THREADS, 1)
delta_bwd(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap my,
          const __grid_constant__ CUtensorMap mv, const __grid_constant__ XbRecArgs p) {
  using L = Lay<true, 2>;
  extern __shared__ uint8_t smem_raw[];
  Cta a;
  const bool inside = cta_setup(p, a, smem_raw, L::SM_S, L::SM_U, L::SM_BAR);
  bf16* dv = (bf16*)p.dv_out + (long long)a.h * p.dv + a.v0;
  const long long dv_t = (long long)p.Hv * p.dv;
  if (!inside) {
    zero_rows(p, a, dv, dv_t);
    return;
  }
  cta_begin<256>(a);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, steps = a.c1 - a.c0;
  const int4* chunks = reinterpret_cast<const int4*>(p.chunks);
  constexpr int FIRST = MEET + 32;
  if (warp == LOADER) {
    const bool one = xb_elect_one();
    for (int n = 0; n < 2; ++n)
      if (one && n < steps) load_stage(p, a, &mk, &mq, &my, &mv, a.c1 - 1 - n, a.smem + n * L::STAGE, &a.bars->full[n]);
    for (int n = 0; n < steps; ++n) {
      bar(1, FIRST);
      if (one) keep_tiles(p, a, p.ds_tiles, p.dr_tiles, a.c1 - 1 - n, n > 0 ? a.c1 - n : -1);
      if (one && n + 2 < steps) {
        a.wait1(&a.bars->done[2], n & 1, 2);
        load_stage(p, a, &mk, &mq, &my, &mv, a.c1 - 1 - (n + 2), a.smem + (n & 1) * L::STAGE, &a.bars->full[n & 1]);
      }
      __syncwarp();
    }
    if (steps > 0) {
      bar(1, FIRST);
      if (one) keep_tiles(p, a, p.ds_tiles, p.dr_tiles, -1, a.c0);
    }
  } else if (warp == ISSUER) {
    const bool one = xb_elect_one();
    const uint64_t b1 = xb_smem_desc(MNMAJ, a.sm + L::SM_S), b2 = xb_smem_desc(MNMAJ, a.sm + L::SM_B2), b3 = xb_smem_desc(MNMAJ, a.sm + L::SM_B3);
    const int ksteps = (p.dk + 15) / 16;
    for (int n = 0; n < steps; ++n) {
      const uint32_t st = a.sm + (n & 1) * L::STAGE;
      const uint64_t kq = xb_smem_desc(KMAJ, st + ST_KQ), kt = xb_smem_desc(MNMAJ, st + ST_KQ), tp = xb_smem_desc(MNMAJ, st + ST_TP);
      constexpr uint32_t id3 = xb_idesc(1, 1, 128, 64, 1, 1);
      constexpr uint32_t id1 = xb_idesc(1, 1, 64, 64, 0, 1), id2 = xb_idesc(1, 1, 64, 64, 1, 1), id4 = xb_idesc(1, 1, 64, 32, 1, 1);
      if (one) a.wait1(&a.bars->full[n & 1], (n >> 1) & 1, 1);
      bar(4, MEET);
      if (one) {
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < 8; ++k)          // P^T dO
          tc_mma_f16_ss(a.tmem + D4, ahead(tp, (k >> 2) * TP_PLANE + HALF / 2 + (k & 3) * 2048), ahead(b2, HALF / 2 + (k & 3) * 2048), id4, k > 0);
      }
      bar(1, FIRST);
      if (one) {
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < ksteps) tc_mma_f16_ss(a.tmem + D1, ahead(kq, (k >> 2) * HALF + (k & 3) * 32), ahead(b1, k * 2048), id1, k > 0);
        tc_commit(&a.bars->done[0]);
#pragma unroll
        for (int k = 4; k < 8; ++k)          // rows of Q
          tc_mma_f16_ss(a.tmem + D3, ahead(kt, k * 2048), ahead(b3, k * 2048), id3, k > 4);
      }
      bar(2, MEET);
      if (one) {
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < 8; ++k)
          tc_mma_f16_ss(a.tmem + D2, ahead(tp, (k >> 2) * TP_PLANE + (k & 3) * 2048), ahead(b2, (k & 3) * 2048), id2, k > 0);
        const uint64_t t3 = xb_smem_desc(MNMAJ, st + ST_T3);
#pragma unroll
        for (int k = 0; k < 4; ++k) tc_mma_f16_ss(a.tmem + D2, ahead(t3, k * 2048), ahead(b2, k * 2048), id4, 1);
#pragma unroll
        for (int k = 0; k < 4; ++k) tc_mma_f16_ss(a.tmem + D2, ahead(tp, k * 2048), ahead(b3, k * 2048), id4, 1);
        tc_commit(&a.bars->done[1]);
      }
      bar(3, MEET);
      if (one) {
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < 4; ++k)          // rows of K
          tc_mma_f16_ss(a.tmem + D3, ahead(kt, k * 2048), ahead(b3, k * 2048), id3, 1);
        tc_commit(&a.bars->done[2]);
      }
      __syncwarp();
    }
    if (steps > 0) bar(1, FIRST);
  } else {
    const int q4 = warp & 3, part = warp >> 2, r = q4 * 32 + lane, i = r & 63, r0 = q4 * 16, g = lane >> 2;
    const int row[2] = {r0 + g, r0 + g + 8}, u0 = part * NB, fcol = u0 * 8, orow = r0 + frag_row();
    const bool krow = r < C;
    const uint32_t quad = a.tmem + ((uint32_t)(q4 * 32) << 16) + fcol;
    const uint32_t f2 = frag_addr(a.sm + L::SM_B2, r0, u0), f3 = frag_addr(a.sm + L::SM_B3, r0, u0), fu = frag_addr(a.sm + L::SM_U, r0, u0),
                   t3 = third_addr(a.sm + L::SM_B3, r0, u0);
    const long long soff = ((long long)a.doc * p.Hv + a.h) * p.dk * p.dv + a.v0 * p.s_v;
    Pair s[4 * NB];
#pragma unroll
    for (int e = 0; e < 4 * NB; ++e) s[e] = twice(0.f);
    if (p.ds_out != nullptr) state_row(const_cast<float*>(p.ds_out) + soff, p.s_k, p.s_v, r, p.dk, fcol, a.vcols, false, s);
    // operands that need dO alone: dO beside Y's tile, gamma rq dO of the third product (threads of Q's rows)
    auto put_dy = [&](int n) {
      const int len = chunks[a.c1 - 1 - n].y;
      const uint32_t st = a.sm + (n & 1) * L::STAGE;
      a.wait(&a.bars->full[n & 1], (n >> 1) & 1, 3);
      if (len < C) clear_rows(st, len);
      if (krow) return;
      const float f = ex2_sum(st + ST_HD, i) * ldsf(st + ST_RQK + i * 4);
      Pair x[4 * NB];
#pragma unroll
      for (int m = 0; m < NB; ++m) {
        const uint4 v = i < len ? lds128(st + ST_X + swz<4>(i, u0 + m)) : make_uint4(0, 0, 0, 0);
        sts128(a.sm + L::SM_B2 + r * 128 + (((u0 + m) ^ (r & 7)) << 4), v.x, v.y, v.z, v.w);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * m + e] = twice(f) * bf16_pair(w[e]);
      }
      put_row(a.sm + L::SM_B3, r, u0, x);
    };
    if (steps > 0) {
      put_dy(0);
      fence_proxy_async_smem();
      bar_arrive(4, MEET);
    }
    int4 ch = steps > 0 ? chunks[a.c1 - 1] : make_int4(0, 0, 0, 0);
    for (int n = 0; n < steps; ++n) {
      const int len = ch.y;
      const long long t0 = ch.x;
      const uint32_t st = a.sm + (n & 1) * L::STAGE, hd = st + ST_HD, rqk = st + ST_RQK;
      put_row(a.sm + L::SM_S, r, u0, s);
      fence_proxy_async_smem();
      tc_fence_before();
      bar_arrive(1, FIRST);
      const float last = ex2_sum(hd, C - 1);
      float w1[2], w2[2], b[2];
      uint32_t v[NB][2];                     // the loads that take this stage next wait for the third product only
      Pair x[2 * NB], y[2 * NB];
      uint32_t third[2 * NB];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float rk = ldsf(rqk + (C + row[h]) * 4);
#pragma unroll
        for (int m = 0; m < NB; ++m) v[m][h] = row[h] < len ? lds32(st + ST_V + swz<4>(row[h], u0 + m) + (lane & 3) * 4) : 0u;
        b[h] = ldsf(hd + (2 * C + row[h]) * 4), w1[h] = ex2_diff(hd, C - 1, row[h]) * rk, w2[h] = -b[h] * ex2_sum(hd, row[h]) * rk;
      }
      a.wait(&a.bars->done[0], n & 1, 4);
      tc_fence_after();
      {                                      // Y = d rk K dS' + P^T dO
        uint32_t d[4 * NB];
        tmem_ld_frag(quad + D4, d);
        read_frag(quad + D1, x);
#pragma unroll
        for (int e = 0; e < 2 * NB; ++e) x[e] = fma2(twice(w1[e & 1]), x[e], pair(d[2 * e], d[2 * e + 1]));
        put_frag3(f2, x, third);             // Y's third part where -b gamma dR comes afterwards
        stsm4(t3, third[0], third[1], third[2], third[3]);
      }
      fence_proxy_async_smem();
      tc_fence_before();
      bar_arrive(2, MEET);
      a.wait(&a.bars->done[1], n & 1, 5);
      tc_fence_after();
      read_frag(quad + D2, y);               // -b gamma rk dR
#pragma unroll
      for (int e = 0; e < 2 * NB; ++e) x[e] = x[e] + y[e];
#pragma unroll
      for (int e = 0; e < 2 * NB; ++e) y[e] = twice(w2[e & 1]) * x[e];
      put_frag(f3, y);
      fence_proxy_async_smem();
      tc_fence_before();
      bar_arrive(3, MEET);
      a.wait(&a.bars->kept, n & 1, 8);       // the tiles on their way out have been read
      put_frag3(fu, x, third);
      keep_third((uint8_t*)p.r_tiles + (((long long)(a.c1 - 1 - n) * p.Hv + a.h) * (p.dvp / 64) + (a.v0 >> 6)) * HALF + HALF / 2, orow,
                 ((a.v0 >> 3) & 7) + u0, third);
      {                                      // dR.v for the gradient of b
        float d[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          Pair w = twice(0.f);
#pragma unroll
          for (int m = 0; m < NB; ++m) {
            w = fma2(x[2 * m + h], bf16_pair(v[m][h]), w);
          }
          const float2 e = both(w);
          d[h] = e.x + e.y;
          d[h] += __shfl_xor_sync(0xffffffffu, d[h], 1);
          d[h] += __shfl_xor_sync(0xffffffffu, d[h], 2);
        }
        if ((lane & 3) < 2)
          p.part[(((long long)(a.c1 - 1 - n) * p.Hv + a.h) * (p.dvp / 16) + (a.v0 >> 4) + part) * C + ((lane & 1) ? row[1] : row[0])] = (lane & 1) ? d[1] : d[0];
      }
#pragma unroll
      for (int e = 0; e < 2 * NB; ++e) x[e] = twice(b[e & 1]) * x[e];
      store_frag(dv + (t0 + orow) * dv_t + fcol, orow < len, a.vcols - fcol, x);
      if (n + 1 < steps) {                   // beside the third product: the first two have read these rows
        ch = chunks[a.c1 - 2 - n];
        put_dy(n + 1);
        fence_proxy_async_smem();
        bar_arrive(4, MEET);
      }
      a.wait(&a.bars->done[2], n & 1, 6);
      tc_fence_after();
      Pair d[4 * NB];
      read_rows(quad + D3, d);
#pragma unroll
      for (int e = 0; e < 4 * NB; ++e) s[e] = fma2(twice(last), s[e], d[e]);
    }
    fence_proxy_async_smem();
    if (steps > 0) bar_arrive(1, FIRST);
    if (p.ds_in != nullptr) state_row(p.ds_in + soff, p.s_k, p.s_v, r, p.dk, fcol, a.vcols, true, s);
  }
  cta_end<256>(a);
}

template <auto KERNEL, int SMEM>
int run(const XbRecArgs& a, const void* x, long long x_t, long long x_h, cudaStream_t st) {
  const long long blocks = (long long)rec_docs(a) * a.Hv * (a.dvp / NV);
  if (blocks > 0x7fffffffLL) return -4;
  if (blocks == 0) return 0;
  CUtensorMap mk{}, mq{}, mx{}, mv{};
  if (a.T > 0 && (rec_tile_map(&mk, a.k, a.T, a.Hk, a.dk, a.k_t, a.k_h, 64, CU_TENSOR_MAP_SWIZZLE_128B) ||
                  rec_tile_map(&mq, a.q, a.T, a.Hk, a.dk, a.q_t, a.q_h, 64, CU_TENSOR_MAP_SWIZZLE_128B) ||
                  rec_tile_map(&mx, x, a.T, a.Hv, a.dv, x_t, x_h, NV, CU_TENSOR_MAP_SWIZZLE_64B) ||
                  rec_tile_map(&mv, a.v, a.T, a.Hv, a.dv, a.v_t, a.v_h, NV, CU_TENSOR_MAP_SWIZZLE_64B)))
    return -2;
  if (!rec_configure<KERNEL>(SMEM)) return -5;
  KERNEL<<<(unsigned)blocks, THREADS, SMEM, st>>>(mk, mq, mx, mv, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -11;
}

template <int DKP>
int prep(const XbRecArgs& a, cudaStream_t st) {
  if (!rec_configure<delta_prep<DKP>>(sizeof(DPrepSmem<DKP>))) return -5;
  return rec_launch(delta_prep<DKP>, (long long)a.nc_max * a.Hk, PT, sizeof(DPrepSmem<DKP>), a, st);
}

}  // namespace

int xb_delta_prep(const XbRecArgs& a, cudaStream_t st) { return a.dk <= 64 ? prep<64>(a, st) : prep<128>(a, st); }
int xb_delta_fwd(const XbRecArgs& a, cudaStream_t st) {
  if (a.s_tiles != nullptr) return run<delta_fwd<true, true, 2>, Lay<false, 2>::SMEM>(a, a.v, a.v_t, a.v_h, st);
  // Two CTAs per SM, one stage each, hide one another's way in and out, but a chunk's loads wait for the chunk before.  They pay
  // where there are more CTAs than SMs and a document has eight chunks or fewer on average.  One stage and two stages, heads of
  // 128 x 128 without gradients, us: 32 heads, 40 documents of 64 tokens 131 and 192, of 128 212 and 272, of 256 371 and 422, of
  // 400 611 and 655; 16 documents of 1000 537 and 542, three of 1000 150 and 129, two of 4000 310 and 287.  At most one CTA per
  // SM, 4 heads: one document of 128 tokens 25 and 23, of 256 29 and 26, of 1000 60 and 43; eight of 400 38 and 31.
  if ((long long)a.n_docs * a.Hv * (a.dvp / NV) > xb_sm_count() && 8ll * C * a.n_docs >= a.T)
    return run<delta_fwd<true, false, 1>, Lay<false, 1>::SMEM>(a, a.v, a.v_t, a.v_h, st);
  return run<delta_fwd<true, false, 2>, Lay<false, 2>::SMEM>(a, a.v, a.v_t, a.v_h, st);
}
int xb_delta_bwd(const XbRecArgs& a, int tiles, cudaStream_t st) {
  if (!tiles) {
    XbRecArgs again = a;
    again.s_out = nullptr;
    if (int rc = run<delta_fwd<false, true, 2>, Lay<false, 2>::SMEM>(again, a.v, a.v_t, a.v_h, st)) return rc;
  }
  return run<delta_bwd, Lay<true, 2>::SMEM>(a, a.dy, a.dy_t, a.dy_h, st);
}
