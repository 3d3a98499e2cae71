// What the kernels of the gated linear recurrences share: constants, operand fragments, tiles in shared memory.
#pragma once
#include "common.cuh"
#include "recurrence.h"

namespace {

constexpr int C = 64;         // tokens of a chunk
constexpr int HALF = 128 * 128;   // bytes of an operand tile of 128 rows of 128 bytes
constexpr int NV = 32;        // state columns of a CTA of the sequential kernels
constexpr int HD = 3 * C;     // per chunk and v head: G (two floats each, log2 units), b
constexpr int RQK = 2 * C;    // per chunk and q / k head: row factors of q and k
constexpr float MIN_LOG = -120.f;  // e^-120 is 0 in fp32: a stronger decay changes nothing and would cost G its digits

using bf16 = __nv_bfloat16;

// ---- fragments ---------------------------------------------------------------------------------------------
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Pairs of fp32 values: one instruction for two on sm_100.
struct Pair { uint64_t v; };
__device__ __forceinline__ Pair pair(float x, float y) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(x), "f"(y));
  return p;
}
__device__ __forceinline__ Pair pair(uint32_t x, uint32_t y) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "r"(x), "r"(y));
  return p;
}
__device__ __forceinline__ float2 both(Pair p) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p.v));
  return f;
}
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
  asm("add.rn.f32x2 %0, %0, %1;" : "+l"(a.v) : "l"(b.v));
  return a;
}
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
  asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(a.v) : "l"(b.v));
  return a;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c.v) : "l"(a.v), "l"(b.v));
  return c;
}
// two fp32 values as the sums of two bf16 values each
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = pack_bf16x2(x, y);
  const float2 r = both(fma2(pair(hi << 16, hi & 0xffff0000u), pair(-1.f, -1.f), pair(x, y)));     // exact
  lo = pack_bf16x2(r.x, r.y);
}
__device__ __forceinline__ void split2(Pair x, uint32_t& hi, uint32_t& lo) {
  const float2 f = both(x);
  hi = pack_bf16x2(f.x, f.y);
  const float2 r = both(fma2(pair(hi << 16, hi & 0xffff0000u), pair(-1.f, -1.f), x));
  lo = pack_bf16x2(r.x, r.y);
}
// two fp32 values as the sums of three bf16 values each: all 24 bits
__device__ __forceinline__ void split3(Pair x, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  const Pair minus = pair(-1.f, -1.f);
  const float2 f = both(x);
  hi = pack_bf16x2(f.x, f.y);
  const Pair r = fma2(pair(hi << 16, hi & 0xffff0000u), minus, x);
  const float2 g = both(r);
  mid = pack_bf16x2(g.x, g.y);
  const float2 h = both(fma2(pair(mid << 16, mid & 0xffff0000u), minus, r));
  lo = pack_bf16x2(h.x, h.y);
}

// A tile is rows of U 16-byte units; unit u of a row lies at u ^ f(row), so that the eight rows that ldmatrix reads
// at one unit fall into eight different banks.
template <int U>
__device__ __forceinline__ uint32_t swz(int row, int u) {
  return (uint32_t)(row * U + (U == 4 ? (u ^ ((row >> 1) & 3)) : (u ^ (row & 7)))) * 16u;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ float ldsf(uint32_t a) { return __uint_as_float(lds32(a)); }
__device__ __forceinline__ void stsf(uint32_t a, float v) {
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory");
}
__device__ __forceinline__ float4 ldsf4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}

// 16 x 16 bf16 values from fragments (as ldsm4 reads them)
__device__ __forceinline__ void stsm4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// 16 rows and 16 columns of an accumulator as fragments: r[4 n + 2 h + e] is row g + 8 h, column 8 n + 2 t + e (g = lane / 4,
// t = lane % 4).  Of a 64-row accumulator, which lies in 16 lanes of each warp, every thread gets values.
__device__ __forceinline__ void tmem_ld_frag(uint32_t addr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(addr) : "memory");
}

// fragment addresses of this lane; m0, n0, k0 are multiples of 8 (16 for the wide ones)
template <int U>  // A[m][k], k contiguous
__device__ __forceinline__ uint32_t addr_a(int m0, int k0) {
  const int l = xb_lane();
  return swz<U>(m0 + (l & 15), (k0 >> 3) + (l >> 4));
}
template <int U>  // B of two 8-wide column tiles, X[n][k], k contiguous
__device__ __forceinline__ uint32_t addr_b(int n0, int k0) {
  const int l = xb_lane();
  return swz<U>(n0 + (l & 7) + (l >> 4) * 8, (k0 >> 3) + ((l >> 3) & 1));
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// ROWS rows of U units from `src` (row stride ld elements); units behind `cols` and rows behind `rows` become zero
template <int U, int ROWS, int THREADS>
__device__ __forceinline__ void load_tile(uint32_t dst, const bf16* src, long long ld, int rows, int cols) {
#pragma unroll
  for (int i = 0; i < ROWS * U / THREADS; ++i) {
    const int idx = i * THREADS + threadIdx.x, r = idx / U, u = idx % U;
    const bool ok = r < rows && u * 8 < cols;
    cp16(dst + swz<U>(r, u), ok ? src + r * ld + u * 8 : src, ok);
  }
}
__device__ __forceinline__ float ex2_diff(const float* hd, int i, int j) {
  return xb_ex2((hd[i] - hd[j]) + (hd[C + i] - hd[C + j]));
}
__device__ __forceinline__ float ex2_sum(const float* hd, int i) { return xb_ex2(hd[i]) * (1.f + 0.6931472f * hd[C + i]); }

// the same from a shared-memory address (pointers into aligned dynamic shared memory become generic ones)
__device__ __forceinline__ float ex2_diff(uint32_t hd, int i, int j) {
  return xb_ex2((ldsf(hd + i * 4) - ldsf(hd + j * 4)) + (ldsf(hd + (C + i) * 4) - ldsf(hd + (C + j) * 4)));
}
__device__ __forceinline__ float ex2_sum(uint32_t hd, int i) { return xb_ex2(ldsf(hd + i * 4)) * (1.f + 0.6931472f * ldsf(hd + (C + i) * 4)); }

// A bounded wait whose slow path stays out of line: a wait that runs out raises a flag and reports; from then on waits
// return at once and every role walks to its end.  Warps that wait sleep up to 20 us at a time, so that they leave the
// issue slots to those that work.
__device__ __noinline__ void rec_wait_slow(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int detail) {
  const uint64_t t0 = xb_globaltimer();
  for (;;) {
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\nselp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok) : "r"(xb_smem_u32(bar)), "r"(parity), "r"(20000u) : "memory");
    if (ok || *abort_flag) return;
    if (xb_globaltimer() - t0 > XB_WAIT_LIMIT_NS) {
      *abort_flag = 1;
      xb_report(status, XB_ERR_MBAR_TIMEOUT, XB_K_RECURRENCE, detail);
      return;
    }
  }
}
__device__ __forceinline__ void rec_wait(uint64_t* bar, uint32_t parity, int* abort_flag, int* status, int detail) {
  if (!mbar_try_wait(bar, parity)) rec_wait_slow(bar, parity, abort_flag, status, detail);
}

// [T, heads, cols] bf16, boxes of 64 rows of one head
inline int rec_tile_map(CUtensorMap* m, const void* base, int T, int heads, int cols, long long ld_t, long long ld_h, int box, CUtensorMapSwizzle swz) {
  return xb_make_tmap_3d(m, base, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, T, heads, cols, T > 1 ? ld_t : 8, heads > 1 ? ld_h : 8, C, 1, box, swz);
}

// Documents 0 .. n-1 lie between the boundaries; n is the tail behind the last boundary, n + 1 the rows before the first.
__device__ __forceinline__ int2 doc_range(const int* cu, int n, int T, int d) {
  auto cut = [&](int i) { return min(max(cu[i], 0), T); };
  if (d == n) return make_int2(cut(n), T);
  if (d == n + 1) return make_int2(0, cut(0));
  const int s = cut(d);
  return make_int2(s, max(s, cut(d + 1)));
}
// Boundaries ascend from 0 or more to T or less.  What does not is clamped, so that nothing outside the rows is touched, and
// reported: by the plan for all documents, by the token-by-token kernels for each of theirs.
__device__ __forceinline__ bool bad_bounds(const int* cu, int n, int T, int d) {
  return d < n ? cu[d] < 0 || cu[d + 1] < cu[d] || cu[d + 1] > T : d == n && (cu[n] < 0 || cu[n] > T);
}
// Documents that the grids of the chunked kernels cover: all, or at most those that are too long to go token by token.
__host__ __device__ inline int rec_docs(const XbRecArgs& a) { return a.step > 0 ? a.T / (a.step + 1) : a.n_docs + 2; }
// The document of a grid's `i`-th; -1: none.
__device__ __forceinline__ int rec_doc(const XbRecArgs& a, int i) {
  return a.step == 0 ? i : i < a.doc_list[0] ? a.doc_list[1 + i] : -1;
}

// Dynamic shared memory above 48 KB, once per kernel and device.
template <auto KERNEL>
bool rec_configure(int smem) {
  static bool done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (done[dev & 63]) return true;
  if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  return done[dev & 63] = true;
}
template <typename K>
int rec_launch(K kernel, long long blocks, int threads, size_t smem, const XbRecArgs& a, cudaStream_t st) {
  if (blocks <= 0) return 0;
  if (blocks > 0x7fffffffLL) return -4;
  kernel<<<(unsigned)blocks, threads, smem, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? 0 : -11;
}

}  // namespace

// recurrence_delta.cu: prepare; forward (keeping tiles where it is given room for them); forward again for the tiles
// unless they are there, and the state's gradient
int xb_delta_prep(const XbRecArgs& a, cudaStream_t st);
int xb_delta_fwd(const XbRecArgs& a, cudaStream_t st);
int xb_delta_bwd(const XbRecArgs& a, int tiles, cudaStream_t st);
// recurrence_step.cu: documents of at most `step` tokens, forward only
int xb_recurrence_step(const XbRecArgs& a, int delta, cudaStream_t st);
// recurrence_scan.cu: the same for the scan
int xb_scan_prep(const XbRecArgs& a, cudaStream_t st);
int xb_scan_fwd(const XbRecArgs& a, cudaStream_t st);
int xb_scan_bwd(const XbRecArgs& a, int tiles, cudaStream_t st);
// recurrence_grad.cu: gradients of q, k, the decay and b from the kept tiles
int xb_recurrence_grad(const XbRecArgs& a, int delta, cudaStream_t st);
