// The state-space scan's own kernels: prepare, and one kernel for the sequential part of both directions (the formulas
// stand in recurrence.cu).  With P_ij = D_ij (Q K^T)_ij b_j for j <= i:
//
//   forward   O = gamma Q S + P V + D V,             S' = gamma_last S + K^T (d b V)
//   backward  dV = d b K dS' + P^T dO + D dO,        dS = gamma_last dS' + Q^T (gamma dO)
//
// The two are one computation with Q and K, and the row factors gamma and d b, exchanged, P transposed and the chunks
// walked the other way.  The state does not feed back into what is added to it, so the products of a step need not wait
// for one another: a CTA carries 64 state columns of one head through one document, ten warps make the operands that
// depend on the chunk alone (P, and d b V or gamma dO) ahead of the products, sixteen add up the state and write the
// outputs, one loads and one issues.  Computed operands are [hi 32 | lo 32] tiles (P: two planes, the other operand three;
// kept states go with their third parts, straight from the registers).  Per step and CTA 24
// products, about 1300 cycles of the tensor pipe of 3700: issue slots (66 % taken) and latencies of the warps that add and
// split bound it.  128 heads of 64 x 128: forward 500 us for a document of 16384 tokens (with two parts 470) and 181 us for 4095
// tokens in five documents with their states kept (0.43 GB written; with two parts and 0.29 GB 146), backward 183 us; prepare 37 and 11 us.  Eight adding warps instead
// of sixteen: 1.7 times the time.
#include "recurrence_core.cuh"

namespace {

// ---- prepare: Q K^T of a chunk and group, running decays of the group's heads -----------------------------------------
template <int DKP>
__global__ void __launch_bounds__(128) scan_prep(const XbRecArgs p) {
  __shared__ __align__(128) uint8_t q[C * DKP * 2];
  __shared__ __align__(128) uint8_t k[C * DKP * 2];
  constexpr int U = DKP / 8;
  const int kh = blockIdx.x % p.Hk, c = blockIdx.x / p.Hk;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, t = lane & 3;
  if (c >= p.doc_off[p.n_docs + 2]) return;
  const int4 ch = reinterpret_cast<const int4*>(p.chunks)[c];
  const int len = ch.y, rep = p.Hv / p.Hk;
  const uint32_t sq = xb_smem_u32(q), sk = xb_smem_u32(k);
  load_tile<U, C, 128>(sq, (const bf16*)p.q + ch.x * p.q_t + kh * p.q_h, p.q_t, len, p.dk);
  load_tile<U, C, 128>(sk, (const bf16*)p.k + ch.x * p.k_t + kh * p.k_h, p.k_t, len, p.dk);
  cp_commit();
  p.rqk[((long long)c * p.Hk + kh) * RQK + tid] = (tid & 63) < len ? 1.f : 0.f;
  for (int hh = w; hh < rep; hh += 4) {
    const int h = kh * rep + hh;
    double x[2];
    float bb[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = 2 * lane + i;
      x[i] = 0.0, bb[i] = 0.f;
      if (row < len) {
        bb[i] = p.b[(ch.x + row) * p.b_t + h * p.b_h];
        const double z = (double)bb[i] * (double)p.A[h];
        x[i] = (z < (double)MIN_LOG ? (double)MIN_LOG : z) * 1.4426950408889634;
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
      const float hi = (float)G;
      out[row] = hi, out[C + row] = (float)(G - (double)hi), out[2 * C + row] = bb[i];
    }
  }
  cp_wait<0>();
  __syncthreads();
  float* qk = p.qk + ((long long)c * p.Hk + kh) * (C * C);
#pragma unroll
  for (int nt = 0; nt < 8; nt += 2) {
    if (nt * 8 > w * 16 + 15) break;              // columns above the diagonal block are never used
    float a[2][4] = {};
#pragma unroll
    for (int ks = 0; ks < DKP / 16; ++ks) {
      uint32_t fq[4], fb[4];
      ldsm4(fb, sk + addr_b<U>(nt * 8, ks * 16));
      ldsm4(fq, sq + addr_a<U>(w * 16, ks * 16));
      mma(a[0], fq, fb[0], fb[1]);
      mma(a[1], fq, fb[2], fb[3]);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
        *reinterpret_cast<float2*>(qk + (w * 16 + g + hh * 8) * C + (nt + j) * 8 + 2 * t) = make_float2(a[j][2 * hh], a[j][2 * hh + 1]);
  }
}

// ---- the sequential part -------------------------------------------------------------------------------------------
constexpr int T64 = HALF / 2;
// warps: 16 add up the state and write outputs, 6 make P (a block of 32 rows and 16 columns each), 4 the other operand
constexpr int ADDERS = 512, PMAKERS = 192, XMAKERS = 128, MAKERS = PMAKERS + XMAKERS, THREADS = ADDERS + MAKERS + 64;
// K and Q: [64 rows][128 bytes] twice each; v or dO: [64][64 columns]; Q K^T: [64][32 fp32] and, of the
// right half, the lower 32 rows; decays and b; the row factors of the outputs
constexpr int ST_K = 0, ST_Q = 2 * T64, ST_X = 4 * T64, ST_QK = 5 * T64, ST_HD = ST_QK + T64 + T64 / 2, ST_ROW = ST_HD + HD * 4, STAGE = ST_ROW + C * 4;
constexpr int SM_S = 2 * STAGE, SM_P = SM_S + 2 * HALF, SM_D = SM_P + 2 * HALF, SM_BAR = SM_D + 6 * T64;
constexpr int SMEM = SM_BAR + 256 + 1024;
constexpr int D1 = 0, D2 = 128, DSTEP = 192, D3 = 384;      // D1, D2 of even and odd steps; D3

struct __align__(8) Bars {
  uint64_t full[2], empty[2], pd_full[2], pd_empty[2], s_full, s_empty, out_full[2], out_empty[2], d3_full, d3_empty;
  uint32_t tmem;
  int abort_flag;
};
static_assert(sizeof(Bars) <= 256, "barriers");

// BWD: the direction.  OUT: outputs are wanted.  KEEP: the state tiles of every chunk go to global memory.
template <bool BWD, bool OUT, bool KEEP>
__global__ void __launch_bounds__(THREADS, 1)
scan_seq(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mx,
         const __grid_constant__ CUtensorMap mqk, const __grid_constant__ XbRecArgs p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  Bars* bars = reinterpret_cast<Bars*>(smem + SM_BAR);
  const int blocks = p.dvp / 64, rep = p.Hv / p.Hk;
  const int cb = blockIdx.x % blocks, h = (blockIdx.x / blocks) % p.Hv, doc = rec_doc(p, blockIdx.x / (blocks * p.Hv));
  if (doc < 0) return;
  const int kh = h / rep, v0 = cb * 64, c0 = p.doc_off[doc], steps = p.doc_off[doc + 1] - c0;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int4* chunks = reinterpret_cast<const int4*>(p.chunks);
  auto chunk_of = [&](int n) { return BWD ? c0 + steps - 1 - n : c0 + n; };
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->full[i], 1), mbar_init(&bars->empty[i], 1 + ((OUT ? MAKERS : XMAKERS) + ADDERS) / 32);
      mbar_init(&bars->pd_full[i], (OUT ? MAKERS : XMAKERS) / 32), mbar_init(&bars->pd_empty[i], 1);
      mbar_init(&bars->out_full[i], 1), mbar_init(&bars->out_empty[i], ADDERS / 32);
    }
    mbar_init(&bars->s_full, ADDERS / 32), mbar_init(&bars->s_empty, (OUT ? 1 : 0) + (KEEP ? 1 : 0));
    mbar_init(&bars->d3_full, 1), mbar_init(&bars->d3_empty, ADDERS / 32);
    bars->abort_flag = 0;
    mbar_fence_init();
  }
  constexpr int LOADER = (MAKERS + ADDERS) / 32, ISSUER = LOADER + 1;
  if (warp == LOADER) {
    tmem_alloc(&bars->tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem, sm = xb_smem_u32(smem);
  // a wait that runs out raises a flag; from then on waits return at once and every role walks to its end
  auto wait = [&](uint64_t* b, uint32_t parity, int detail) { rec_wait(b, parity, &bars->abort_flag, p.status, detail); };
  auto wwait = [&](uint64_t* b, uint32_t parity, int detail) {
    wait(b, parity, detail);
    __syncwarp();
  };
  auto arrive = [&](uint64_t* b) {
    __syncwarp();
    if (lane == 0) mbar_arrive(b);
  };

  if (warp == LOADER) {
    if (xb_elect_one()) {
      for (int n = 0; n < steps; ++n) {
        const int s = n & 1, c = chunk_of(n), t0 = chunks[c].x;
        uint8_t* st = smem + s * STAGE;
        uint64_t* full = &bars->full[s];
        wait(&bars->empty[s], ((n >> 1) & 1) ^ 1, 1);
        mbar_expect_tx(full, (OUT ? ST_HD : 3 * T64) + HD * 4);
        for (int i = 0; i < 2; ++i) {
          if (OUT || !BWD) tma_load_3d(st + ST_K + i * T64, &mk, full, i * 64, kh, t0);
          if (OUT || BWD) tma_load_3d(st + ST_Q + i * T64, &mq, full, i * 64, kh, t0);
        }
        for (int i = 0; OUT && i < 3; ++i)   // blocks of 32 x 32 on and below the diagonal
          tma_load_2d(st + ST_QK + i * (T64 / 2), &mqk, full, i == 2 ? 32 : 0, (c * p.Hk + kh) * C + (i ? 32 : 0));
        tma_load_3d(st + ST_X, &mx, full, v0, h, t0);
        bulk_load(st + ST_HD, p.hd + ((long long)c * p.Hv + h) * HD, HD * 4, full);
      }
    }
    __syncwarp();
  } else if (warp == ISSUER) {
    if (xb_elect_one()) {
      constexpr uint64_t kmaj = xb_smem_desc_base_sw128(16, 1024), mn64 = xb_smem_desc_base_sw128(T64, 1024),
                         mn128 = xb_smem_desc_base_sw128(HALF, 1024);
      constexpr uint32_t id1 = xb_idesc(1, 1, 64, 128, 0, 1), id2 = xb_idesc(1, 1, 64, 64, BWD ? 1 : 0, 1), id3 = xb_idesc(1, 1, 128, 128, 1, 1), id4 = xb_idesc(1, 1, 128, 64, 1, 1);
      const uint32_t bs = xb_smem_u32(smem + SM_S);
      for (int n = 0; n < steps; ++n) {
        const int s = n & 1;
        const uint32_t ph = (n >> 1) & 1, st = xb_smem_u32(smem + s * STAGE);
        const uint32_t pt = xb_smem_u32(smem + SM_P + s * HALF), dt = xb_smem_u32(smem + SM_D + s * 3 * T64);
        const uint32_t row = st + (BWD ? ST_K : ST_Q), col = st + (BWD ? ST_Q : ST_K);
        wait(&bars->full[s], ph, 10);
        wait(&bars->pd_full[s], ph, 11);
        wait(&bars->d3_empty, (n & 1) ^ 1, 12);
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < 4; ++k)          // K^T (d b V), Q^T (gamma dO)
          tc_mma_f16_ss(tmem + D3, xb_smem_desc(mn64, col + k * 2048), xb_smem_desc(mn64, dt + k * 2048), id3, k > 0);
#pragma unroll
        for (int k = 0; k < 4; ++k)          // the third parts, added to the second's
          tc_mma_f16_ss(tmem + D3 + 64, xb_smem_desc(mn64, col + k * 2048), xb_smem_desc(mn64, dt + 2 * T64 + k * 2048), id4, 1);
        tc_commit(&bars->d3_full);
        if (OUT) {
          wait(&bars->out_empty[s], ph ^ 1, 13);
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < 8; ++k) {      // P V, P^T dO: planes hi, lo
            const uint32_t a = pt + (k >> 2) * T64;
            tc_mma_f16_ss(tmem + D2 + s * DSTEP, BWD ? xb_smem_desc(mn64, a + (k & 3) * 2048) : xb_smem_desc(kmaj, a + (k & 3) * 32),
                          xb_smem_desc(mn64, st + ST_X + (k & 3) * 2048), id2, k > 0);
          }
        }
        tc_commit(&bars->pd_empty[s]);
        wait(&bars->s_full, n & 1, 14);
        tc_fence_after();
        if (KEEP) {
          const int slices = p.dvp / NV;
          uint8_t* dst = (uint8_t*)(BWD ? p.ds_tiles : p.s_tiles) + (((long long)chunk_of(n) * p.Hv + h) * slices + 2 * cb) * HALF;
          bulk_store(dst, smem + SM_S, 2 * HALF);
          tma_store_commit();
        }
        if (OUT) {
#pragma unroll
          for (int k = 0; k < 8; ++k)        // Q S, K dS'
            tc_mma_f16_ss(tmem + D1 + s * DSTEP, xb_smem_desc(kmaj, row + (k >> 2) * T64 + (k & 3) * 32), xb_smem_desc(mn128, bs + k * 2048), id1, k > 0);
          tc_commit(&bars->s_empty);
          tc_commit(&bars->out_full[s]);
        }
        tc_commit(&bars->empty[s]);
        if (KEEP) {
          tma_store_wait_read<0>();
          mbar_arrive(&bars->s_empty);
        }
      }
    }
    __syncwarp();
  } else if (warp >= (ADDERS + PMAKERS) / 32) {
    // ------------------------------------ gamma dO, or d b V: 32 columns of a row ------------------------------------
    const int t = tid - ADDERS - PMAKERS, row = t & 63, half = t >> 6;
    for (int n = 0; n < steps; ++n) {
      const int s = n & 1, len = chunks[chunk_of(n)].y;
      const uint32_t st = sm + s * STAGE, hd = st + ST_HD;
      wwait(&bars->full[s], (n >> 1) & 1, 20);
      // rows behind the document's end hold the next one's: they must not meet a product's zeros (0 x Inf is NaN)
      if (len < C) {
        for (int i = t; i < 5 * (C - len) * 8; i += XMAKERS) {
          const int part = i / ((C - len) * 8), r = len + (i % ((C - len) * 8)) / 8;
          sts128(st + ST_K + part * T64 + r * 128 + (i & 7) * 16, 0, 0, 0, 0);
        }
        __syncwarp();                        // named barriers want whole warps
        asm volatile("bar.sync 1, %0;" ::"n"(XMAKERS) : "memory");
      }
      const float gam = ex2_sum(hd, row), db = ex2_diff(hd, C - 1, row) * ldsf(hd + (2 * C + row) * 4), f = BWD ? gam : db;
      if (OUT && half == 0) stsf(st + ST_ROW + row * 4, BWD ? db : gam);
      uint4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = lds128(st + ST_X + row * 128 + (((half * 4 + u) ^ (row & 7)) << 4));
      wwait(&bars->pd_empty[s], ((n >> 1) & 1) ^ 1, 21);
      const uint32_t dst = sm + SM_D + s * 3 * T64 + row * 128;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t x[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
        uint32_t hi[4], mid[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) split3(pair(f, f) * pair(x[e] << 16, x[e] & 0xffff0000u), hi[e], mid[e], lo[e]);
        const uint32_t at = dst + (((half * 4 + u) ^ (row & 7)) << 4);
        sts128(at, hi[0], hi[1], hi[2], hi[3]);
        sts128(at + T64, mid[0], mid[1], mid[2], mid[3]);
        sts128(at + 2 * T64, lo[0], lo[1], lo[2], lo[3]);
      }
      fence_proxy_async_smem();
      arrive(&bars->pd_full[s]);
      arrive(&bars->empty[s]);
    }
  } else if (warp >= ADDERS / 32) {
    // ------------------------------------ P: 16 columns of a row -----------------------------------------------------
    // blocks of 32 rows and 16 columns on and below the diagonal: two of the upper rows, four of the lower ones
    const int m = warp - ADDERS / 32, row = (m < 2 ? 0 : 32) + lane, j0 = (m < 2 ? m : m - 2) * 16;
    if (OUT && m < 2)                                                 // the two above it stay zero
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u)
          sts128(sm + SM_P + i * HALF + (u >> 1) * T64 + row * 128 + (((4 + m * 2 + (u & 1)) ^ (row & 7)) << 4), 0, 0, 0, 0);
    for (int n = 0; OUT && n < steps; ++n) {
      const int s = n & 1;
      const uint32_t st = sm + s * STAGE, hd = st + ST_HD;
      wwait(&bars->full[s], (n >> 1) & 1, 22);
      const float gi = ldsf(hd + row * 4), gl = ldsf(hd + (C + row) * 4);
      const uint32_t src = st + ST_QK + (j0 >> 5) * (T64 / 2) + row * 128;
      float y[16];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int j = j0 + q * 4;
        const float4 x = ldsf4(src + ((((j & 31) >> 2) ^ (row & 7)) << 4));
        const float4 a = ldsf4(hd + j * 4), b = ldsf4(hd + (C + j) * 4);
        const float4 w = ldsf4(hd + (2 * C + j) * 4);
        y[4 * q] = j <= row ? x.x * w.x * xb_ex2((gi - a.x) + (gl - b.x)) : 0.f;
        y[4 * q + 1] = j + 1 <= row ? x.y * w.y * xb_ex2((gi - a.y) + (gl - b.y)) : 0.f;
        y[4 * q + 2] = j + 2 <= row ? x.z * w.z * xb_ex2((gi - a.z) + (gl - b.z)) : 0.f;
        y[4 * q + 3] = j + 3 <= row ? x.w * w.w * xb_ex2((gi - a.w) + (gl - b.w)) : 0.f;
      }
      arrive(&bars->empty[s]);
      uint32_t hi[8], lo[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) split2(y[2 * e], y[2 * e + 1], hi[e], lo[e]);
      wwait(&bars->pd_empty[s], ((n >> 1) & 1) ^ 1, 23);
      const uint32_t dst = sm + SM_P + s * HALF + row * 128;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int off = (((j0 >> 3) + u) ^ (row & 7)) << 4;
        sts128(dst + off, hi[4 * u], hi[4 * u + 1], hi[4 * u + 2], hi[4 * u + 3]);
        sts128(dst + T64 + off, lo[4 * u], lo[4 * u + 1], lo[4 * u + 2], lo[4 * u + 3]);
      }
      fence_proxy_async_smem();
      arrive(&bars->pd_full[s]);
    }
  } else {
    // ------------------------------------ the state, and the outputs -------------------------------------------------
    // a row of the state and 16 of its columns; of the 64-row accumulators 16 rows and 16 columns per warp, as fragments
    const int q4 = warp & 3, sl = warp >> 3, part = (warp >> 2) & 1, r = q4 * 32 + lane, r0 = q4 * 16, g = lane >> 2, t = lane & 3;
    const uint32_t base = tmem + ((uint32_t)(q4 * 32) << 16);
    const int col = v0 + sl * NV + part * 16, cols = p.dv - col;
    const long long soff = ((long long)doc * p.Hv + h) * p.dk * p.dv + col * p.s_v + r * p.s_k;
    const float* from = BWD ? p.ds_out : p.s_in;
    float* to = BWD ? p.ds_in : p.s_out;
    Pair x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      auto at = [&](int i) { return from != nullptr && doc < p.n_docs && r < p.dk && i < cols ? from[soff + i * p.s_v] : 0.f; };
      x[e] = pair(at(2 * e), at(2 * e + 1));
    }
    uint32_t hi[8], lo[8];
    // the state of chunk `c`; the third parts of a kept one go to global memory from here
    auto split_row = [&](int c) {
      if constexpr (KEEP) {
        uint32_t third[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) split3(x[e], hi[e], lo[e], third[e]);
        // units 2 part and 2 part + 1 trade places in odd rows and stay 32 bytes side by side
        uint8_t* dst = (uint8_t*)p.r_tiles + (((long long)c * p.Hv + h) * (p.dvp / NV) + 2 * cb + sl) * HALF + r * 128 +
                       (((part * 2 + (BWD ? 4 : 0)) ^ (r & 6)) << 4);
        const bool odd = r & 1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t a = third[e], b = third[4 + e];
          third[e] = odd ? b : a, third[4 + e] = odd ? a : b;
        }
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(third[0]), "r"(third[1]), "r"(third[2]),
                     "r"(third[3]), "r"(third[4]), "r"(third[5]), "r"(third[6]), "r"(third[7]) : "memory");
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) split2(x[e], hi[e], lo[e]);
      }
    };
    auto put = [&]() {                       // the state's row as [hi | lo]
      const uint32_t dst = sm + SM_S + sl * HALF + r * 128;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int u = part * 2 + i;
        sts128(dst + ((u ^ (r & 7)) << 4), hi[4 * i], hi[4 * i + 1], hi[4 * i + 2], hi[4 * i + 3]);
        sts128(dst + (((u + 4) ^ (r & 7)) << 4), lo[4 * i], lo[4 * i + 1], lo[4 * i + 2], lo[4 * i + 3]);
      }
      fence_proxy_async_smem();
      tc_fence_before();
      arrive(&bars->s_full);
    };
    if (steps > 0) {
      split_row(chunk_of(0));
      put();
    }
    const float skip = p.D[h];
    const int xrow = r0 + (lane & 15), xunit = sl * 4 + part * 2 + (lane >> 4), ocol = col + 8 * (t & 1) + 4 * (t >> 1);
    bf16* out = (bf16*)(BWD ? p.dv_out : p.o) + (long long)h * p.dv + ocol;
    for (int n = 0; n < steps; ++n) {
      const int s = n & 1;
      const int4 ch = chunks[chunk_of(n)];
      const uint32_t st = sm + s * STAGE, hd = st + ST_HD;
      wwait(&bars->full[s], (n >> 1) & 1, 30);
      const float last = ex2_sum(hd, C - 1);
      float f[2] = {};
      uint32_t xv[4];
      if (OUT) {
        wwait(&bars->pd_full[s], (n >> 1) & 1, 34);                    // the row factors
        f[0] = ldsf(st + ST_ROW + (r0 + g) * 4), f[1] = ldsf(st + ST_ROW + (r0 + g + 8) * 4);
        ldsm4(xv, st + ST_X + xrow * 128 + ((xunit ^ (xrow & 7)) << 4));
      }
      arrive(&bars->empty[s]);
      wwait(&bars->d3_full, n & 1, 31);
      tc_fence_after();
      {
        uint32_t a[16], b[16];
        tmem_ld_32x16(base + D3 + sl * NV + part * 16, a);
        tmem_ld_32x16(base + D3 + 64 + sl * NV + part * 16, b);
        tc_wait_ld();
        tc_fence_before();
        arrive(&bars->d3_empty);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          x[e] = fma2(pair(last, last), x[e], pair(a[2 * e], a[2 * e + 1]) + pair(b[2 * e], b[2 * e + 1]));
      }
      if (n + 1 < steps) {
        split_row(chunk_of(n + 1));
        wwait(&bars->s_empty, n & 1, 32);    // the tile's readers are done
        put();
      }
      if (OUT) {
        if (n + 1 == steps) wwait(&bars->out_full[s], (n >> 1) & 1, 33);   // else: the wait above was for the same products
        tc_fence_after();
        uint32_t a[8], b[8], d[8], w[4];
        tmem_ld_frag(base + D1 + s * DSTEP + sl * 64 + part * 16, a);
        tmem_ld_frag(base + D1 + s * DSTEP + sl * 64 + 32 + part * 16, b);
        tmem_ld_frag(base + D2 + s * DSTEP + sl * 32 + part * 16, d);
        tc_wait_ld();
        tc_fence_before();
        arrive(&bars->out_empty[s]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {        // e = 2 n + h: row g + 8 h, columns 8 n + 2 t, 8 n + 2 t + 1
          const Pair z = fma2(pair(f[e & 1], f[e & 1]), pair(a[2 * e], a[2 * e + 1]) + pair(b[2 * e], b[2 * e + 1]), pair(d[2 * e], d[2 * e + 1]));
          const float2 y = both(fma2(pair(skip, skip), pair(xv[e] << 16, xv[e] & 0xffff0000u), z));
          w[e] = pack_bf16x2(y.x, y.y);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {        // lanes t and t ^ 1 trade, for four neighbouring columns each
          const uint32_t other = __shfl_xor_sync(0xffffffffu, t & 1 ? w[h] : w[2 + h], 1);
          const int row = r0 + g + 8 * h;
          if (row < ch.y && ocol < p.dv)
            *reinterpret_cast<uint2*>(out + (long long)(ch.x + row) * p.Hv * p.dv) = t & 1 ? make_uint2(other, w[2 + h]) : make_uint2(w[h], other);
        }
      }
    }
    if (to != nullptr && doc < p.n_docs && r < p.dk)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float2 f = both(x[e]);
        if (2 * e < cols) to[soff + 2 * e * p.s_v] = f.x, to[soff + (2 * e + 1) * p.s_v] = f.y;
      }
  }
  // after a wait that ran out, loads and products may still be on their way: give them 0.2 s
  if (*(volatile int*)&bars->abort_flag && tid == 0)
    for (const uint64_t t0 = xb_globaltimer(); xb_globaltimer() - t0 < 200000000ull;) {}
  tc_fence_before();
  __syncthreads();
  if (warp == LOADER) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <bool BWD, bool OUT, bool KEEP>
int run(const XbRecArgs& a, const void* x, long long x_t, long long x_h, cudaStream_t st) {
  const long long blocks = (long long)rec_docs(a) * a.Hv * (a.dvp / 64);
  if (blocks > 0x7fffffffLL) return -4;
  if (blocks == 0) return 0;
  CUtensorMap mk{}, mq{}, mx{}, mqk{};
  if (a.T > 0 && (rec_tile_map(&mk, a.k, a.T, a.Hk, a.dk, a.k_t, a.k_h, 64, CU_TENSOR_MAP_SWIZZLE_128B) ||
                  rec_tile_map(&mq, a.q, a.T, a.Hk, a.dk, a.q_t, a.q_h, 64, CU_TENSOR_MAP_SWIZZLE_128B) ||
                  rec_tile_map(&mx, x, a.T, a.Hv, a.dv, x_t, x_h, 64, CU_TENSOR_MAP_SWIZZLE_128B) ||
                  xb_make_tmap_2d(&mqk, a.qk, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, (uint64_t)a.nc_max * a.Hk * C, C, C, 32, 32, CU_TENSOR_MAP_SWIZZLE_128B)))
    return -2;
  if (!rec_configure<scan_seq<BWD, OUT, KEEP>>(SMEM)) return -5;
  scan_seq<BWD, OUT, KEEP><<<(unsigned)blocks, THREADS, SMEM, st>>>(mk, mq, mx, mqk, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -11;
}

}  // namespace

int xb_scan_prep(const XbRecArgs& a, cudaStream_t st) {
  const long long blocks = (long long)a.nc_max * a.Hk;
  return a.dk <= 64 ? rec_launch(scan_prep<64>, blocks, 128, 0, a, st) : rec_launch(scan_prep<128>, blocks, 128, 0, a, st);
}
int xb_scan_fwd(const XbRecArgs& a, cudaStream_t st) {
  return a.s_tiles != nullptr ? run<false, true, true>(a, a.v, a.v_t, a.v_h, st) : run<false, true, false>(a, a.v, a.v_t, a.v_h, st);
}
int xb_scan_bwd(const XbRecArgs& a, int tiles, cudaStream_t st) {
  if (!tiles) {
    XbRecArgs again = a;
    again.s_out = nullptr;
    if (int rc = run<false, false, true>(again, a.v, a.v_t, a.v_h, st)) return rc;
  }
  return run<true, true, true>(a, a.dy, a.dy_t, a.dy_h, st);
}
