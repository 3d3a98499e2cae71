// Gated linear recurrences, the parallel part of the backward pass: gradients of q, k, the log decay and b of one chunk
// from the states that enter it, the gradients of the states that leave it, U and dR (formulas in recurrence.cu).
//
// One CTA per chunk and q / k head.  It walks over the v heads that share the q / k head and over their state columns,
// 32 at a time, and forms five products in tensor memory, all with 64 rows of tokens:
//   dP = dO U^T,  dL = dR U^T  [64 x 64];   t1 = dO S^T,  t2 = dR S^T,  t3 = U dS'^T  [64 x 128]
// (scan: U = V, no dL and t2.)  A computed operand is a tile of [hi 32 | lo 32] columns; the parts of a product are the
// pairs of 16-column steps; third parts are tiles of their own.  Behind each head the rows of t1 .. t3 are scaled and added up in
// registers, their dot products with q and k give the gradient of the decay and of b, and D o dP, D o dL are added up;
// the products with K and Q are the same for all heads of the group and are made once, from the sums.
// Sixteen worker warps, a loading and an issuing warp, and one that turns the heads' sums into gradients of the decay.
//
// It reads the tiles that the two sequential passes keep (56 KB per head and 32 columns; scan 48 KB).  4096 tokens of 32
// heads of 128 x 128: 217 us, 0.52 GB of tiles at 2.4 TB/s; 4095 tokens of 128 heads of 64 x 128: 276 us, 0.87 GB at 3.2
// TB/s (without third parts 208 and 244 us).  All of tensor memory holds one head's five products (scan: two heads' dP and t1), so that loads overlap the
// workers' turn and products do not; with two heads per CTA a third of the time is its way in and out.
#include "recurrence_core.cuh"

namespace {

constexpr int WORKERS = 512, THREADS = WORKERS + 96;
constexpr int PARTS = WORKERS / 128;                // column parts of the products, 32 and 16 columns per warp
static_assert(WORKERS == 512, "one 16 x 16 block of a state tile per warp");
constexpr int WIDE = 8 / PARTS;                     // pieces of 16 columns of a warp's part of the wide products
constexpr int T64 = HALF / 2;                       // 8 KB: [64 rows][128 bytes]
template <bool DELTA>
struct Lay {
  static constexpr int RING = DELTA ? 2 : 3;
  static constexpr int ST_S = 0, ST_DS = HALF, ST_U = 2 * HALF, ST_R = 2 * HALF + T64, ST_3 = 2 * HALF;
  static constexpr int STAGE = 3 * HALF;
  // dO and V (delta rule: third parts of U and of dR) of a pass: 128 columns each in one buffer, which the next head's loads wait for; scan: 64 columns in two.
  // The decays of two heads.
  static constexpr int SL = DELTA ? 4 : 2, NB = DELTA ? 1 : 2, DOV = DELTA ? 6 * T64 : SL * T64;
  static constexpr int SM_Q = 0, SM_K = 2 * T64, SM_RING = 4 * T64, SM_DOV = SM_RING + RING * STAGE, SM_HD = SM_DOV + NB * DOV,
                       SM_RED = SM_HD + 2 * 1024;
};
struct Red {                                        // what meets across warps, one set per head in turn
  float rd[3][PARTS][C];                            // q.t1, k.t2, k.t3 by column part (scan: the second holds the diagonal of dP o P)
  // Row sums of dP o P and dL o A by column part (scan: dP o P), column sums by row block.  Without the diagonal: it carries no
  // decay and would cancel in the decay's gradient, but as two roundings of what strong decays leave as the largest term.
  float er[PARTS][C], fr[PARTS][C];
  float ec[4][C], fc[4][C];
  float rv[2][C], sdot[WORKERS / 32];                // scan: dO.v by column half of every slice; <S, dS'> by warp
};
struct __align__(8) Bars {
  uint64_t full[4], empty[4], dov_full[2], dov_empty[2], hd_full[2], hd_empty[2], red_full[2], red_empty[2];
  uint64_t qk_full, acc_full, t3_empty, set_empty[2], z_full, last;
  uint32_t tmem;
  int abort_flag;
};
template <bool DELTA>
constexpr int smem_bytes() { return Lay<DELTA>::SM_RED + 2 * (int)sizeof(Red) + RQK * 4 + 256 + 1024; }
// Tensor memory: dP, dL, t1, t2, t3 (scan: dP and t1 of even and odd heads, t3; the next head's products start when t3 has
// been read).  At the end dq and dk in the places of t1 and t2.
constexpr int COL_P = 0, COL_L = 64, COL_T1 = 128, COL_T2 = 256, COL_T3 = 384;

__device__ __forceinline__ float parts(const float (&a)[PARTS][C], int t) {
  float s = a[0][t] + a[1][t];
#pragma unroll
  for (int i = 2; i < PARTS; i += 2) s += a[i][t] + a[i + 1][t];
  return s;
}
__device__ __forceinline__ float2 lds2(uint32_t a) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void wbar() {
  __syncwarp();
  asm volatile("bar.sync 1, %0;" ::"n"(WORKERS) : "memory");
}

// D (64 x N) += A (64 x 16 of a row of 16-column steps) B^T: one step each
__device__ __forceinline__ void step(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool first) {
  constexpr uint64_t kmaj = xb_smem_desc_base_sw128(16, 1024);
  tc_mma_f16_ss(d, xb_smem_desc(kmaj, a), xb_smem_desc(kmaj, b), idesc, first ? 0u : 1u);
}
// all four products of the parts of two [hi | lo] tiles; EXACT: a is 32 plain columns
template <bool EXACT>
__device__ __forceinline__ void product(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool first) {
  step(d, a, b, idesc, first);
  step(d, a + 32, b + 32, idesc, false);
  step(d, a, b + 64, idesc, false);
  step(d, a + 32, b + 96, idesc, false);
  if (!EXACT) {
    step(d, a + 64, b, idesc, false);
    step(d, a + 96, b + 32, idesc, false);
    step(d, a + 64, b + 64, idesc, false);
    step(d, a + 96, b + 96, idesc, false);
  }
}
// Fragments: a thread has rows g and g + 8 of its warp's 16 and, of every 8 columns, 2 t and 2 t + 1.
// The two rows' sums over the four lanes that share them; lane t keeps the one of row t % 2.
__device__ __forceinline__ float row_sum(float a, float b) {
  const bool odd = threadIdx.x & 1;
  const float v = (odd ? b : a) + __shfl_xor_sync(0xffffffffu, odd ? a : b, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
// The same of two sums at once: lanes t < 2 keep the first's, the others the second's.
__device__ __forceinline__ float row_sum2(const float (&a)[2], const float (&b)[2]) {
  const bool odd = threadIdx.x & 1, up = threadIdx.x & 2;
  const float x = (odd ? a[1] : a[0]) + __shfl_xor_sync(0xffffffffu, odd ? a[0] : a[1], 1);
  const float y = (odd ? b[1] : b[0]) + __shfl_xor_sync(0xffffffffu, odd ? b[0] : b[1], 1);
  return (up ? y : x) + __shfl_xor_sync(0xffffffffu, up ? x : y, 2);
}
// Sums over the eight lanes that share columns; lane g keeps column 8 (g & 1) + 2 t + (g >> 1 & 1) of the 16.
__device__ __forceinline__ float col_sum(const float (&v)[2][2]) {
  const bool n = threadIdx.x & 4, e = threadIdx.x & 8;
  const float x = (n ? v[1][0] : v[0][0]) + __shfl_xor_sync(0xffffffffu, n ? v[0][0] : v[1][0], 4);
  const float y = (n ? v[1][1] : v[0][1]) + __shfl_xor_sync(0xffffffffu, n ? v[0][1] : v[1][1], 4);
  const float z = (e ? y : x) + __shfl_xor_sync(0xffffffffu, e ? x : y, 8);
  return z + __shfl_xor_sync(0xffffffffu, z, 16);
}
// 32 bf16 values of row `row` of a [64][256 bytes] tile in two halves of 64 columns
__device__ __forceinline__ uint4 tile_unit(uint32_t tile, int row, int unit) {
  return lds128(tile + (unit >> 3) * T64 + row * 128 + (((unit & 7) ^ (row & 7)) << 4));
}
__device__ __forceinline__ void floats8(const uint4 u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = unpack_bf16x2(w[j]);
    x[2 * j] = f.x, x[2 * j + 1] = f.y;
  }
}
// address of a 16 x 16 block of a [64][256 bytes] tile in two halves of 64 columns, for ldsm4 and stsm4
__device__ __forceinline__ uint32_t block_addr(uint32_t tile, int r0, int col) {
  const int l = xb_lane(), unit = (col >> 3) + (l >> 4), row = r0 + (l & 15);
  return tile + (unit >> 3) * T64 + row * 128 + (((unit & 7) ^ (row & 7)) << 4);
}
__device__ __forceinline__ Pair bf16_pair(uint32_t v) { return pair(v << 16, v & 0xffff0000u); }
// acc += f * t over this thread's rows and columns col .. col + 32; returns t . (the same columns of `tile`)
__device__ __forceinline__ float add_rows(uint32_t addr, uint32_t tile, int r0, int col, const float (&f)[2], Pair (&acc)[WIDE][2][2]) {
  uint32_t t[2][8];
  Pair dot[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
  tmem_ld_frag(addr, t[0]);
#pragma unroll
  for (int i = 0; i < WIDE; ++i) {
    uint32_t x[4];
    ldsm4(x, block_addr(tile, r0, col + 16 * i));
    tc_wait_ld();
    if (i + 1 < WIDE) tmem_ld_frag(addr + 16 * (i + 1), t[(i + 1) & 1]);
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const Pair y = pair(t[i & 1][4 * n + 2 * h], t[i & 1][4 * n + 2 * h + 1]);
        dot[h] = fma2(bf16_pair(x[2 * n + h]), y, dot[h]);
        acc[i][n][h] = fma2(pair(f[h], f[h]), y, acc[i][n][h]);
      }
  }
  const float2 a = both(dot[0]), b = both(dot[1]);
  return row_sum(a.x + a.y, b.x + b.y);
}

template <bool DELTA>
__global__ void __launch_bounds__(THREADS, 1)
rec_grad(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
         const __grid_constant__ CUtensorMap my, const __grid_constant__ XbRecArgs p) {
  using L = Lay<DELTA>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  Red* red = reinterpret_cast<Red*>(smem + L::SM_RED);
  float* rqk = reinterpret_cast<float*>(red + 2);
  Bars* bars = reinterpret_cast<Bars*>(rqk + RQK);
  const int kh = blockIdx.x % p.Hk, c = blockIdx.x / p.Hk, rep = p.Hv / p.Hk;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (c >= p.doc_off[p.n_docs + 2]) return;
  const int4 ch = reinterpret_cast<const int4*>(p.chunks)[c];
  const int len = ch.y;
  bf16* dq = (bf16*)p.dq + (ch.x * (long long)p.Hk + kh) * p.dk;
  bf16* dk = (bf16*)p.dk_out + (ch.x * (long long)p.Hk + kh) * p.dk;
  const long long d_t = (long long)p.Hk * p.dk;
  if (DELTA && ch.z >= p.n_docs) {                  // rows outside the documents
    for (int i = tid; i < len * p.dk; i += THREADS) {
      dq[(i / p.dk) * d_t + i % p.dk] = __float2bfloat16(0.f);
      dk[(i / p.dk) * d_t + i % p.dk] = __float2bfloat16(0.f);
    }
    for (int i = tid; i < len * rep; i += THREADS) {
      const long long at = (long long)(ch.x + i / rep) * p.Hv + kh * rep + i % rep;
      p.dg[at] = 0.f, p.db[at] = 0.f;
    }
    return;
  }
  const int slices = p.dvp / NV, passes = (slices + L::SL - 1) / L::SL;
  if (tid == 0) {
    constexpr int NW = WORKERS / 32;
    for (int i = 0; i < 4; ++i) mbar_init(&bars->full[i], 1), mbar_init(&bars->empty[i], 1 + NW);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->dov_full[i], 1), mbar_init(&bars->dov_empty[i], 1 + NW);
      mbar_init(&bars->hd_full[i], 1), mbar_init(&bars->hd_empty[i], NW + 1);
      mbar_init(&bars->red_full[i], NW), mbar_init(&bars->red_empty[i], 1), mbar_init(&bars->set_empty[i], NW);
    }
    mbar_init(&bars->qk_full, 1), mbar_init(&bars->acc_full, 1), mbar_init(&bars->t3_empty, NW), mbar_init(&bars->z_full, NW);
    mbar_init(&bars->last, 1);
    bars->abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == WORKERS / 32) {
    tmem_alloc(&bars->tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem, sm = xb_smem_u32(smem), srqk = xb_smem_u32(rqk);
  // a wait that runs out raises a flag; from then on waits return at once and every role walks to its end
  auto wait = [&](uint64_t* b, uint32_t parity, int detail) { rec_wait(b, parity, &bars->abort_flag, p.status, detail); };

  if (warp == WORKERS / 32) {
    // ------------------------------------------------ loads ------------------------------------------------
    if (xb_elect_one()) {
      mbar_expect_tx(&bars->qk_full, 4 * T64 + RQK * 4);
      for (int i = 0; i < 2; ++i) {
        tma_load_3d(smem + L::SM_Q + i * T64, &mq, &bars->qk_full, i * 64, kh, ch.x);
        tma_load_3d(smem + L::SM_K + i * T64, &mk, &bars->qk_full, i * 64, kh, ch.x);
      }
      bulk_load(rqk, p.rqk + ((long long)c * p.Hk + kh) * RQK, RQK * 4, &bars->qk_full);
      int n = 0, m = 0;
      for (int hh = 0; hh < rep; ++hh) {
        const int h = kh * rep + hh;
        const long long ch_h = (long long)c * p.Hv + h;
        wait(&bars->hd_empty[hh & 1], ((hh >> 1) & 1) ^ 1, 19);
        mbar_expect_tx(&bars->hd_full[hh & 1], HD * 4);
        bulk_load(smem + L::SM_HD + (hh & 1) * 1024, p.hd + ch_h * HD, HD * 4, &bars->hd_full[hh & 1]);
        for (int pass = 0; pass < passes; ++pass, ++m) {
          const int d = m % L::NB;
          uint8_t* dov = smem + L::SM_DOV + d * L::DOV;
          wait(&bars->dov_empty[d], ((m / L::NB) & 1) ^ 1, 20);
          mbar_expect_tx(&bars->dov_full[d], DELTA ? T64 * (2 + 2 * min(2, slices / 2 - pass * 2)) : L::DOV);
          for (int i = 0; i < L::SL / 2; ++i) {
            tma_load_3d(dov + i * T64, &my, &bars->dov_full[d], pass * L::SL * NV + i * 64, h, ch.x);
            if (!DELTA) {
              tma_load_3d(dov + (L::SL / 2 + i) * T64, &mv, &bars->dov_full[d], pass * L::SL * NV + i * 64, h, ch.x);
            } else if (pass * 2 + i < slices / 2) {
              const uint8_t* third = (const uint8_t*)p.r_tiles + (ch_h * (slices / 2) + pass * 2 + i) * HALF;
              bulk_load(dov + (2 + i) * T64, third, T64, &bars->dov_full[d]);
              bulk_load(dov + (4 + i) * T64, third + T64, T64, &bars->dov_full[d]);
            }
          }
          for (int sl = pass * L::SL; sl < min(slices, pass * L::SL + L::SL); ++sl, ++n) {
            const int s = n % L::RING;
            uint8_t* st = smem + L::SM_RING + s * L::STAGE;
            wait(&bars->empty[s], ((n / L::RING) & 1) ^ 1, 21);
            mbar_expect_tx(&bars->full[s], L::STAGE);
            const long long at = ch_h * slices + sl;
            bulk_load(st + L::ST_S, (const uint8_t*)p.s_tiles + at * HALF, HALF, &bars->full[s]);
            if (DELTA) {
              bulk_load(st + L::ST_U, (const uint8_t*)p.u_tiles + at * T64, T64, &bars->full[s]);
              bulk_load(st + L::ST_R, (const uint8_t*)p.dr_tiles + at * T64, T64, &bars->full[s]);
            } else {
              bulk_load(st + L::ST_3, (const uint8_t*)p.r_tiles + at * HALF, HALF, &bars->full[s]);
            }
            bulk_load(st + L::ST_DS, (const uint8_t*)p.ds_tiles + at * HALF, HALF, &bars->full[s]);
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == WORKERS / 32 + 1) {
    // ------------------------------------------------ products ----------------------------------------------
    if (xb_elect_one()) {
      constexpr uint32_t id64 = xb_idesc(1, 1, 64, 64, 0, 0), id128 = xb_idesc(1, 1, 64, 128, 0, 0);
      int n = 0, m = 0;
      for (int hh = 0; hh < rep; ++hh) {
        wait(&bars->t3_empty, (hh & 1) ^ 1, 30);
        if (!DELTA) wait(&bars->set_empty[hh & 1], ((hh >> 1) & 1) ^ 1, 34);
        const uint32_t set = DELTA ? 0 : hh & 1;
        for (int pass = 0; pass < passes; ++pass, ++m) {
          const uint32_t y0 = sm + L::SM_DOV + (m % L::NB) * L::DOV, x0 = y0 + 2 * T64 / L::NB;
          wait(&bars->dov_full[m % L::NB], (m / L::NB) & 1, 31);
          for (int sl = pass * L::SL; sl < min(slices, pass * L::SL + L::SL); ++sl, ++n) {
            const int s = n % L::RING, q = sl % L::SL;
            const uint32_t st = xb_smem_u32(smem + L::SM_RING + s * L::STAGE);
            const uint32_t y = y0 + (q >> 1) * T64 + (q & 1) * 64, x = x0 + (q >> 1) * T64 + (q & 1) * 64;
            const bool first = sl == 0;
            wait(&bars->full[s], (n / L::RING) & 1, 32);
            tc_fence_after();
            if (DELTA) {
              product<true>(tmem + COL_P, y, st + L::ST_U, id64, first);
              step(tmem + COL_P, y, x, id64, false);             // U's third part
              step(tmem + COL_P, y + 32, x + 32, id64, false);
              product<false>(tmem + COL_L, st + L::ST_R, st + L::ST_U, id64, first);
              step(tmem + COL_L, st + L::ST_R, x, id64, false);
              step(tmem + COL_L, st + L::ST_R + 32, x + 32, id64, false);
              step(tmem + COL_L, x + 2 * T64, st + L::ST_U, id64, false);
              step(tmem + COL_L, x + 2 * T64 + 32, st + L::ST_U + 32, id64, false);
              product<true>(tmem + COL_T1, y, st + L::ST_S, id128, first);
              product<false>(tmem + COL_T2, st + L::ST_R, st + L::ST_S, id128, first);
              product<false>(tmem + COL_T3, st + L::ST_U, st + L::ST_DS, id128, first);
            } else {
              step(tmem + COL_P + set * 64, y, x, id64, first);
              step(tmem + COL_P + set * 64, y + 32, x + 32, id64, false);
              product<true>(tmem + COL_T1 + set * 128, y, st + L::ST_S, id128, first);
              step(tmem + COL_T1 + set * 128, y, st + L::ST_3, id128, false);
              step(tmem + COL_T1 + set * 128, y + 32, st + L::ST_3 + 32, id128, false);
              product<true>(tmem + COL_T3, x, st + L::ST_DS, id128, first);
              step(tmem + COL_T3, x, st + L::ST_3 + 64, id128, false);
              step(tmem + COL_T3, x + 32, st + L::ST_3 + 96, id128, false);
            }
            tc_commit(&bars->empty[s]);
          }
          tc_commit(&bars->dov_empty[m % L::NB]);
        }
        tc_commit(&bars->acc_full);
      }
      // dq = Z K, dk = W K + W^T K + Z^T Q, from the sums over the heads
      wait(&bars->z_full, 0, 33);
      tc_fence_after();
      constexpr uint64_t kmaj = xb_smem_desc_base_sw128(16, 1024), mn = xb_smem_desc_base_sw128(T64, 1024);
      constexpr uint32_t idr = xb_idesc(1, 1, 64, 128, 0, 1), idc = xb_idesc(1, 1, 64, 128, 1, 1);
      const uint32_t z = xb_smem_u32(smem + L::SM_RING), sk = xb_smem_u32(smem + L::SM_K), sq = xb_smem_u32(smem + L::SM_Q);
#pragma unroll
      for (int i = 0; i < 8; ++i) {                  // planes hi, lo; four steps of 16 tokens
        const uint32_t t = z + (i >> 2) * T64, w = t + 2 * T64, k = (uint32_t)(i & 3);
        tc_mma_f16_ss(tmem + COL_T1, xb_smem_desc(kmaj, t + k * 32), xb_smem_desc(mn, sk + k * 2048), idr, i > 0);
        tc_mma_f16_ss(tmem + COL_T2, xb_smem_desc(mn, t + k * 2048), xb_smem_desc(mn, sq + k * 2048), idc, i > 0);
        if (DELTA) {
          tc_mma_f16_ss(tmem + COL_T2, xb_smem_desc(kmaj, w + k * 32), xb_smem_desc(mn, sk + k * 2048), idr, 1);
          tc_mma_f16_ss(tmem + COL_T2, xb_smem_desc(mn, w + k * 2048), xb_smem_desc(mn, sk + k * 2048), idc, 1);
        }
      }
      tc_commit(&bars->last);
    }
    __syncwarp();
  } else if (warp == WORKERS / 32 + 2) {
    // ------------------------------------------------ the heads' sums ---------------------------------------
    wait(&bars->qk_full, 0, 50);
    __syncwarp();
    for (int hh = 0; hh < rep; ++hh) {
      const int h = kh * rep + hh;
      const long long ch_h = (long long)c * p.Hv + h;
      const Red& r = red[hh & 1];
      const float* hd = reinterpret_cast<const float*>(smem + L::SM_HD + (hh & 1) * 1024);
      wait(&bars->hd_full[hh & 1], (hh >> 1) & 1, 52);
      wait(&bars->red_full[hh & 1], (hh >> 1) & 1, 51);
      __syncwarp();
      // gradients of the log decay (suffix sums of dG) and of b: two rows per lane
      double x[2], tail = 0.0, dsum = 0.0;
      float db[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int t = 2 * lane + i;
        const float bt = hd[2 * C + t], ga = ex2_sum(hd, t), de = ex2_diff(hd, C - 1, t);
        const bool on = t < len;
        auto four = [&](const float (&a)[4][C]) { return (a[0][t] + a[1][t]) + (a[2][t] + a[3][t]); };
        auto two = [&](const float (&a)[PARTS][C]) { return parts(a, t); };
        const float q1 = on ? ga * rqk[t] * two(r.rd[0]) : 0.f, k2 = on && DELTA ? ga * rqk[C + t] * two(r.rd[1]) : 0.f;
        const float k3 = on ? de * rqk[C + t] * two(r.rd[2]) : 0.f;
        const float e1 = two(r.er), e2 = four(r.ec), g1 = DELTA ? two(r.fr) : 0.f, g2 = DELTA ? four(r.fc) : 0.f;
        if (DELTA) {
          x[i] = (double)q1 + (double)e1 - (double)e2 + (double)(bt * g1) - (double)g2 - (double)(bt * k2) - (double)k3;
          tail += k3;
          float dot = 0.f;                             // dR.v, from the walk
          for (int e = 0; e < p.dvp / 16; ++e) dot += p.part[(ch_h * (p.dvp / 16) + e) * C + t];
          db[i] = dot - k2 + g1;
        } else {
          x[i] = (double)q1 + (double)e1 - (double)(bt * e2) - (double)(bt * k3);
          tail += (double)(bt * k3);
          db[i] = e2 + r.rd[1][0][t] + k3;
          if (on) dsum += r.rv[0][t] + r.rv[1][t];
        }
      }
      float sd = lane < WORKERS / 32 ? r.sdot[lane] : 0.f;
      sd = warp_sum(sd);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        tail += __shfl_xor_sync(0xffffffffu, tail, o);
        dsum += __shfl_xor_sync(0xffffffffu, dsum, o);
      }
      tail += (double)(ex2_sum(hd, C - 1) * sd);
      double s = x[0] + x[1];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_down_sync(0xffffffffu, s, o);
        if (lane + o < 32) s += y;
      }
      double da = 0.0;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int t = 2 * lane + i;
        const float dg = (float)((i ? s - x[0] : s) + tail);
        if (t < len) {
          const long long at = (long long)(ch.x + t) * p.Hv + h;
          if (DELTA) {
            p.dg[at] = dg, p.db[at] = db[i];
          } else {
            p.db[at] = db[i] + dg * p.A[h];
            da += (double)(dg * hd[2 * C + t]);
          }
        }
      }
      if (!DELTA) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) da += __shfl_xor_sync(0xffffffffu, da, o);
        if (lane == 0) p.part[ch_h * 2] = (float)da, p.part[ch_h * 2 + 1] = (float)dsum;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->red_empty[hh & 1]), mbar_arrive(&bars->hd_empty[hh & 1]);
    }
  } else {
    // ------------------------------------------------ workers -----------------------------------------------
    // 16 rows per warp, of the wide products 32 columns and of the square ones 16, as fragments
    const int q4 = warp & 3, hf = warp >> 2, g = lane >> 2, t = lane & 3, r0 = q4 * 16, j0 = hf * 16, w0 = hf * 16 * WIDE;
    const int row[2] = {r0 + g, r0 + g + 8}, sum_row = r0 + g + 8 * (t & 1);        // whose sums this lane keeps
    const uint32_t base = tmem + ((uint32_t)(q4 * 32) << 16);
    Pair aq[WIDE][2][2], ak[WIDE][2][2], az[2][2], aw[2][2];
    {
      const Pair zero = pair(0.f, 0.f);
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          az[n][h] = aw[n][h] = zero;
#pragma unroll
          for (int i = 0; i < WIDE; ++i) aq[i][n][h] = ak[i][n][h] = zero;
        }
    }
    // first use is behind the first head's products
    const float* qk = p.qk + ((long long)c * p.Hk + kh) * (C * C) + j0 + 2 * t;
    const float* kk = DELTA ? p.kk + ((long long)c * p.Hk + kh) * (C * C) + j0 + 2 * t : nullptr;
    asm volatile("prefetch.global.L2 [%0];" ::"l"(qk + (r0 + (lane & 15)) * C));
    if (DELTA) asm volatile("prefetch.global.L2 [%0];" ::"l"(kk + (r0 + (lane & 15)) * C));
    auto wwait = [&](uint64_t* b, uint32_t parity, int detail) {
      wait(b, parity, detail);
      __syncwarp();
    };
    auto arrive = [&](uint64_t* b) {
      __syncwarp();
      if (lane == 0) mbar_arrive(b);
    };
    // this warp's 16 x 16 block of the state tiles: row block warp & 7, columns 16 (warp >> 3) ..
    const int sa_r = (warp & 7) * 16 + (lane & 15), sb_r = (warp & 7) * 16 + (lane & 7) + (lane >> 4) * 8, su = (warp >> 3) * 2;
    const uint32_t a_off = sa_r * 128, b_off = sb_r * 128;
    const uint32_t a_hi = ((su + (lane >> 4)) ^ (sa_r & 7)) << 4, a_lo = ((su + (lane >> 4) + 4) ^ (sa_r & 7)) << 4;
    const uint32_t b_hi = ((su + ((lane >> 3) & 1)) ^ (sb_r & 7)) << 4, b_lo = ((su + ((lane >> 3) & 1) + 4) ^ (sb_r & 7)) << 4;
    wwait(&bars->qk_full, 0, 40);
    const float rq[2] = {rqk[row[0]], rqk[row[1]]}, rk[2] = {rqk[C + row[0]], rqk[C + row[1]]};
    int n = 0, m = 0;
    for (int hh = 0; hh < rep; ++hh) {
      Red& r = red[hh & 1];
      float sd[2][4] = {}, rv[2][4] = {};
      const uint32_t hd = sm + L::SM_HD + (hh & 1) * 1024, set = DELTA ? 0 : hh & 1;
      for (int pass = 0; pass < passes; ++pass, ++m) {
        const uint32_t dov = sm + L::SM_DOV + (m % L::NB) * L::DOV;
        wwait(&bars->dov_full[m % L::NB], (m / L::NB) & 1, 41);
        for (int sl = pass * L::SL; sl < min(slices, pass * L::SL + L::SL); ++sl, ++n) {
          const int s = n % L::RING;
          const uint32_t st = sm + L::SM_RING + s * L::STAGE;
          wwait(&bars->full[s], (n / L::RING) & 1, 42);
          if (DELTA) {
            {  // <S, dS'>: a unit of eight columns of a row per thread
              const int sr = tid >> 2, u = tid & 3;
              const uint32_t hi = (uint32_t)(sr * 128 + ((u ^ (sr & 7)) << 4)), lo = (uint32_t)(sr * 128 + (((u + 4) ^ (sr & 7)) << 4));
              float a[8], al[8], b[8], bl[8];
              floats8(lds128(st + L::ST_S + hi), a), floats8(lds128(st + L::ST_S + lo), al);
              floats8(lds128(st + L::ST_DS + hi), b), floats8(lds128(st + L::ST_DS + lo), bl);
#pragma unroll
              for (int e = 0; e < 8; ++e) sd[0][0] += (a[e] + al[e]) * (b[e] + bl[e]);
            }
          } else {
            // <S, dS'> and the rows' dO.v are diagonals of products of 16 x 16 blocks: a block per warp.  (Here the state
            // tiles are most of what a head reads and the workers' time counts; the delta rule's products take longer
            // and its tensor pipe has no room: 209 us this way, 221 us with diagonals.)
            {
              const uint32_t sa = st + L::ST_S + a_off, da = st + L::ST_DS + b_off;
              uint32_t ah[4], al[4], bh[4], bl[4];
              ldsm4(ah, sa + a_hi), ldsm4(al, sa + a_lo), ldsm4(bh, da + b_hi), ldsm4(bl, da + b_lo);
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                mma(sd[e], al, bl[2 * e], bl[2 * e + 1]);
                mma(sd[e], al, bh[2 * e], bh[2 * e + 1]);
                mma(sd[e], ah, bl[2 * e], bl[2 * e + 1]);
                mma(sd[e], ah, bh[2 * e], bh[2 * e + 1]);
              }
            }
            if (warp < 8) {
              const int rb = warp & 3, ks = warp >> 2, unit = (sl % L::SL) * 4 + ks * 2;
              const int ra = rb * 16 + (lane & 15), rn = rb * 16 + (lane & 7) + (lane >> 4) * 8;
              const int ub = unit + ((lane >> 3) & 1), ua = unit + (lane >> 4);
              uint32_t a4[4], b4[4];
              ldsm4(b4, dov + L::DOV / 2 + (ub >> 3) * T64 + rn * 128 + (((ub & 7) ^ (rn & 7)) << 4));
              ldsm4(a4, dov + (ua >> 3) * T64 + ra * 128 + (((ua & 7) ^ (ra & 7)) << 4));
#pragma unroll
              for (int e = 0; e < 2; ++e) mma(rv[e], a4, b4[2 * e], b4[2 * e + 1]);
            }
          }
          arrive(&bars->empty[s]);
        }
        arrive(&bars->dov_empty[m % L::NB]);
      }
      wwait(&bars->red_empty[hh & 1], ((hh >> 1) & 1) ^ 1, 45);
      wwait(&bars->hd_full[hh & 1], (hh >> 1) & 1, 47);
      if (DELTA) {
        const float sum = warp_sum(sd[0][0]);
        if (lane == 0) r.sdot[warp] = sum;
      } else {
        // rows 0 .. 7 of a block from the first column tile, 8 .. 15 from the second
        const int g = lane >> 2, t = lane & 3;
        const bool d0 = g == 2 * t, d1 = g == 2 * t + 1;
        const float sum = warp_sum(d0 ? sd[0][0] + sd[1][2] : d1 ? sd[0][1] + sd[1][3] : 0.f);
        if (lane == 0) r.sdot[warp] = sum;
        if (warp < 8 && (d0 || d1)) {
          float* dst = r.rv[warp >> 2] + (warp & 3) * 16 + g;
          dst[0] = d0 ? rv[0][0] : rv[0][1];
          dst[8] = d0 ? rv[1][2] : rv[1][3];
        }
      }
      float f1[2], f2[2], f3[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool on = row[h] < len;                                 // rows behind the end hold other documents' products
        const float b = ldsf(hd + (2 * C + row[h]) * 4), gam = ex2_sum(hd, row[h]), dec = ex2_diff(hd, C - 1, row[h]);
        f1[h] = on ? gam * rq[h] : 0.f, f2[h] = on ? -b * gam * rk[h] : 0.f, f3[h] = on ? dec * rk[h] * (DELTA ? 1.f : b) : 0.f;
      }
      wwait(&bars->acc_full, hh & 1, 43);
      tc_fence_after();
      const float d3 = add_rows(base + COL_T3 + w0, sm + L::SM_K, r0, w0, f3, ak);
      if (!DELTA) {
        tc_fence_before();
        arrive(&bars->t3_empty);
      }
      const float d1 = add_rows(base + COL_T1 + set * 128 + w0, sm + L::SM_Q, r0, w0, f1, aq);
      const float d2 = DELTA ? add_rows(base + COL_T2 + w0, sm + L::SM_K, r0, w0, f2, ak) : 0.f;
      if (t < 2) {
        r.rd[0][hf][sum_row] = d1, r.rd[2][hf][sum_row] = d3;
        if (DELTA) r.rd[1][hf][sum_row] = d2;
      }
      {
        uint32_t x[8], xl[8];
        float2 qr[2][2], kr[2][2];
        tmem_ld_frag(base + COL_P + set * 64 + j0, x);
        if (DELTA) tmem_ld_frag(base + COL_L + j0, xl);
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            qr[n][h] = *reinterpret_cast<const float2*>(qk + row[h] * C + 8 * n);
            if (DELTA) kr[n][h] = *reinterpret_cast<const float2*>(kk + row[h] * C + 8 * n);
          }
        float er[2] = {}, fr[2] = {}, ec[2][2] = {}, fc[2][2] = {}, b[2], gi[2], gl[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
          b[h] = DELTA ? ldsf(hd + (2 * C + row[h]) * 4) : 0.f, gi[h] = ldsf(hd + row[h] * 4), gl[h] = ldsf(hd + (C + row[h]) * 4);
        tc_wait_ld();
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int j = j0 + 8 * n + 2 * t;
          const float2 hi = lds2(hd + j * 4), lo = lds2(hd + (C + j) * 4), kj = lds2(srqk + (C + j) * 4);
          const float2 bj = DELTA ? make_float2(1.f, 1.f) : lds2(hd + (2 * C + j) * 4);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int last = row[h] < len ? row[h] : -1;              // the row's last column; none behind the end
            const float e0 = xb_ex2((gi[h] - hi.x) + (gl[h] - lo.x)), e1 = xb_ex2((gi[h] - hi.y) + (gl[h] - lo.y));
            {
              const float y0 = j <= last ? e0 * __uint_as_float(x[4 * n + 2 * h]) : 0.f, w0 = j <= last ? y0 * qr[n][h].x : 0.f;
              const float y1 = j < last ? e1 * __uint_as_float(x[4 * n + 2 * h + 1]) : 0.f, w1 = j < last ? y1 * qr[n][h].y : 0.f;
              const float s0 = j < row[h] ? w0 : 0.f, s1 = j + 1 < row[h] ? w1 : 0.f;
              if (!DELTA && (j == row[h] || j + 1 == row[h])) r.rd[1][0][row[h]] = j == row[h] ? w0 : w1;
              er[h] += DELTA ? s0 + s1 : bj.x * s0 + bj.y * s1;
              ec[n][0] += s0, ec[n][1] += s1;
              const Pair f = pair(rq[h] * kj.x, rq[h] * kj.y) * pair(y0, y1);
              az[n][h] = DELTA ? az[n][h] + f : fma2(f, pair(bj.x, bj.y), az[n][h]);
            }
            if (DELTA) {
              const float y0 = j < last ? -e0 * __uint_as_float(xl[4 * n + 2 * h]) : 0.f, w0 = j < last ? y0 * kr[n][h].x : 0.f;
              const float y1 = j + 1 < last ? -e1 * __uint_as_float(xl[4 * n + 2 * h + 1]) : 0.f, w1 = j + 1 < last ? y1 * kr[n][h].y : 0.f;
              fr[h] += w0 + w1;
              fc[n][0] += b[h] * w0, fc[n][1] += b[h] * w1;
              const float f = b[h] * rk[h];
              aw[n][h] = fma2(pair(f * kj.x, f * kj.y), pair(y0, y1), aw[n][h]);
            }
          }
        }
        const int col = j0 + 8 * (g & 1) + 2 * t + ((g >> 1) & 1);
        const float es = col_sum(ec), fs = DELTA ? col_sum(fc) : 0.f;
        if (g < 4) r.ec[q4][col] = es, r.fc[q4][col] = fs;
        const float rs = row_sum2(er, fr);
        (t < 2 ? r.er : r.fr)[hf][sum_row] = rs;
      }
      tc_fence_before();
      arrive(DELTA ? &bars->t3_empty : &bars->set_empty[set]);
      arrive(&bars->red_full[hh & 1]);
      arrive(&bars->hd_empty[hh & 1]);
    }
    // Z and W as operand tiles over the ring: the products have read its last tiles (acc_full), the other warps' own reads of S
    // and dS' end at this barrier; K and Q without rows behind the end
    wbar();
#pragma unroll
    for (int part = 0; part < (DELTA ? 2 : 1); ++part) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) split2(part ? aw[n][h] : az[n][h], hi[2 * n + h], lo[2 * n + h]);
      const uint32_t at = block_addr(sm + L::SM_RING + part * 2 * T64, r0, j0);
      stsm4(at, hi[0], hi[1], hi[2], hi[3]);
      stsm4(at + T64, lo[0], lo[1], lo[2], lo[3]);
    }
    for (int i = tid; i < 4 * (C - len) * 8; i += WORKERS) {
      const int part = i / ((C - len) * 8), rr = len + (i % ((C - len) * 8)) / 8;
      sts128(sm + L::SM_Q + part * T64 + rr * 128 + (i & 7) * 16, 0, 0, 0, 0);
    }
    fence_proxy_async_smem();
    tc_fence_before();
    arrive(&bars->z_full);
    wwait(&bars->last, 0, 44);
    tc_fence_after();
    const float one[2] = {1.f, 1.f};
    add_rows(base + COL_T1 + w0, sm + L::SM_Q, r0, w0, one, aq);
    add_rows(base + COL_T2 + w0, sm + L::SM_K, r0, w0, one, ak);
    // gradient through the L2 norms: dq - q^ (q^ . dq), rows of norm below 1e-12 excepted
    float fq[2] = {}, fk[2] = {};
    if (p.l2norm) {
      Pair sq[2], sk[2];
      sq[0] = sq[1] = sk[0] = sk[1] = pair(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < WIDE; ++i) {
        uint32_t x[4], y[4];
        ldsm4(x, block_addr(sm + L::SM_Q, r0, w0 + 16 * i)), ldsm4(y, block_addr(sm + L::SM_K, r0, w0 + 16 * i));
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            sq[h] = fma2(bf16_pair(x[2 * n + h]), aq[i][n][h], sq[h]), sk[h] = fma2(bf16_pair(y[2 * n + h]), ak[i][n][h], sk[h]);
      }
      const float2 q0 = both(sq[0]), q1 = both(sq[1]), k0 = both(sk[0]), k1 = both(sk[1]);
      const float a[2] = {q0.x + q0.y, q1.x + q1.y}, b[2] = {k0.x + k0.y, k1.x + k1.y};
      Red& r = red[rep & 1];
      wwait(&bars->red_empty[rep & 1], ((rep >> 1) & 1) ^ 1, 46);
      const float s = row_sum2(a, b);
      (t < 2 ? r.rd[0] : r.rd[1])[hf][sum_row] = s;
      wbar();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float nq = rq[h] / p.scale;
        if (nq < 0.99e12f) fq[h] = nq * nq * parts(r.rd[0], row[h]);
        if (rk[h] < 0.99e12f) fk[h] = rk[h] * rk[h] * parts(r.rd[1], row[h]);
      }
    }
    // in the places of this warp's blocks of Q and K, and from there in 16-byte pieces
#pragma unroll
    for (int i = 0; i < WIDE; ++i)
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        const uint32_t at = block_addr(sm + (part ? L::SM_K : L::SM_Q), r0, w0 + 16 * i);
        uint32_t x[4];
        ldsm4(x, at);
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float f = part ? -fk[h] : -fq[h];
            const float2 y = both(fma2(pair(f, f), bf16_pair(x[2 * n + h]), part ? ak[i][n][h] : aq[i][n][h]));
            x[2 * n + h] = pack_bf16x2(y.x, y.y);
          }
        stsm4(at, x[0], x[1], x[2], x[3]);
      }
    __syncwarp();
    const int out = r0 + (lane & 15);
    if (out < len)
#pragma unroll
      for (int i = 0; i < WIDE; ++i) {
        const int unit = hf * 2 * WIDE + 2 * i + (lane >> 4), col = unit * 8;
        if (col < p.dk) {
          *reinterpret_cast<uint4*>(dq + out * d_t + col) = tile_unit(sm + L::SM_Q, out, unit);
          *reinterpret_cast<uint4*>(dk + out * d_t + col) = tile_unit(sm + L::SM_K, out, unit);
        }
      }
  }
  // after a wait that ran out, loads and products may still be on their way: give them 0.2 s
  if (*(volatile int*)&bars->abort_flag && tid == 0)
    for (const uint64_t t0 = xb_globaltimer(); xb_globaltimer() - t0 < 200000000ull;) {}
  tc_fence_before();
  __syncthreads();
  if (warp == WORKERS / 32) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <bool DELTA>
int run(const XbRecArgs& a, cudaStream_t st) {
  const long long blocks = (long long)a.nc_max * a.Hk;
  if (blocks > 0x7fffffffLL) return -4;
  CUtensorMap mq{}, mk{}, mv{}, my{};
  if (a.T > 0 && (rec_tile_map(&mq, a.q, a.T, a.Hk, a.dk, a.q_t, a.q_h, 64, CU_TENSOR_MAP_SWIZZLE_128B) ||
                  rec_tile_map(&mk, a.k, a.T, a.Hk, a.dk, a.k_t, a.k_h, 64, CU_TENSOR_MAP_SWIZZLE_128B) ||
                  rec_tile_map(&mv, a.v, a.T, a.Hv, a.dv, a.v_t, a.v_h, 64, CU_TENSOR_MAP_SWIZZLE_128B) ||
                  rec_tile_map(&my, a.dy, a.T, a.Hv, a.dv, a.dy_t, a.dy_h, 64, CU_TENSOR_MAP_SWIZZLE_128B)))
    return -2;
  if (!rec_configure<rec_grad<DELTA>>(smem_bytes<DELTA>())) return -5;
  rec_grad<DELTA><<<(unsigned)blocks, THREADS, smem_bytes<DELTA>(), st>>>(mq, mk, mv, my, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -11;
}

}  // namespace

int xb_recurrence_grad(const XbRecArgs& a, int delta, cudaStream_t st) { return delta ? run<true>(a, st) : run<false>(a, st); }
