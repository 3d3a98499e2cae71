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
// Kernels: recurrence_delta.cu and recurrence_scan.cu prepare the chunks and walk through them, forwards and backwards;
// recurrence_grad.cu forms the gradients of q, k, the decay and b of all chunks side by side, from tiles that the two
// walks leave; recurrence_step.cu takes documents of a few tokens.  Here: the plan, the sums over chunks, the entry points.
//
// Precision: q, k, v and dO are bf16 and enter the products as they are.  Whatever is computed (states, T, U, P and
// their gradients) is kept in 32 bits and enters a product as the sum of two bf16 values, which keeps 17 bits of its
// significand: one bf16 value (9 bits) would cost the fp32 gradients of the decay three decimal digits.  Where these
// gradients are differences of large sums a third bf16 value keeps all 24: what is added to the scan's states, the
// scan's kept states and their gradients, and the delta rule's T - I, R, Y, U and dR in T R, T^T Y, dO U^T and
// dR U^T.  A call without gradients does the same arithmetic as one with them: their outputs have the same bits.  Measured against 64 bits over 11,000 calls of up to 1500 tokens, of the norm, median
// and most: gradients of A 5e-7 and 5e-6, of dt 2e-7 and 4e-7, states of the scan 7e-8 and 2e-7; gradients of the delta rule's decay 2e-6
// and 7e-6, of beta 3e-6 and 7e-6, its states 3e-6 (fp32 tensor ops: 1e-7 to 4e-7).  With two parts everywhere it was A 1.2e-5,
// states of the scan 3e-6 and the delta rule's decay 1.6e-5; three everywhere would take the walk's shared memory for two
// stages.  bf16 outputs are off by their rounding.  Decays are sums in
// fp64 of log2 units, kept as two floats, so that differences of large sums stay exact.  L2 norms of q and k are row
// factors and are applied behind the products.
#include <type_traits>

#include "recurrence_core.cuh"

namespace {

// ---- plan: chunks of the documents -----------------------------------------------------------------------------
// Documents of at most `step` tokens have no chunks.  The scan counts chunks in the lower 40 bits, documents above.
__global__ void __launch_bounds__(1024) rec_plan(const int* __restrict__ cu, int n, int T, int nc_max, int step, int4* chunks,
                                                 int* doc_off, int* doc_list, int* status) {
  __shared__ long long warp_tot[32];
  __shared__ long long carry;
  constexpr long long DOC = 1ll << 40;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, nd = n + 2;
  if (tid == 0) carry = 0, doc_off[0] = 0;
  __syncthreads();
  for (int base = 0; base < nd; base += 1024) {
    const int d = base + tid;
    long long v = 0;
    if (d < nd) {
      const int2 r = doc_range(cu, n, T, d);
      v = r.y - r.x > step ? (r.y - r.x + C - 1) / C + DOC : 0;
      if (bad_bounds(cu, n, T, d)) xb_report(status, XB_ERR_BAD_ARG, XB_K_RECURRENCE, d);
    }
    const bool some = v != 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    if (lane == 31) warp_tot[w] = v;
    __syncthreads();
    if (w == 0) {
      long long t = warp_tot[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, t, o);
        if (lane >= o) t += u;
      }
      warp_tot[lane] = t;
    }
    __syncthreads();
    const long long all = carry + v + (w ? warp_tot[w - 1] : 0), incl = all & (DOC - 1);
    // boundaries that overlap may need more chunks than there is room for: what does not fit is left out
    if (d < nd) {
      doc_off[d + 1] = (int)min(incl, (long long)nc_max);
      if (some) doc_list[all / DOC] = d;
      if (d == nd - 1) doc_list[0] = (int)(all / DOC);
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

// 16-byte loads: rows of q, k, v and dO, and the states of the delta rule
bool bad_args(const XbRecArgs& a) {
  const long long strides = a.q_t | a.q_h | a.k_t | a.k_h | a.v_t | a.v_h | a.dy_t | a.dy_h;
  uintptr_t at = 0;
  for (const void* p : {a.q, a.k, a.v, a.dy, (const void*)a.s_in, (const void*)a.s_out, (const void*)a.ds_out, (const void*)a.ds_in}) at |= (uintptr_t)p;
  return strides % 8 || at % 16 || a.T < 0 || a.n_docs < 0 || a.Hk <= 0 || a.Hv <= 0 || a.Hv % a.Hk || a.dk <= 0 || a.dk > 128 || a.dk % 8 || a.dv <= 0 ||
         a.dv % 8 || a.step < 0 || a.step >= C || a.nc_max < a.T / C + rec_docs(a);
}

// plan, and the operands of the chunks
int prepare(const XbRecArgs& a, int delta, cudaStream_t st) {
  rec_plan<<<1, 1024, 0, st>>>(a.cu, a.n_docs, a.T, a.nc_max, a.step, (int4*)a.chunks, a.doc_off, a.doc_list, a.status);
  if (cudaGetLastError() != cudaSuccess) return -11;
  return delta ? xb_delta_prep(a, st) : xb_scan_prep(a, st);
}

}  // namespace

// The arguments as 64-bit words, in the order of XbRecArgs up to `part`, (without doc_list), then T, n_docs, Hk, Hv, dk, dv, nc_max, l2norm, step.
static XbRecArgs unpack(const long long* w, float scale) {
  XbRecArgs a{};
  auto ptr = [&](auto& f) { f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(*w++); };
  auto num = [&](auto& f) { f = static_cast<std::remove_reference_t<decltype(f)>>(*w++); };
  ptr(a.q), ptr(a.k), ptr(a.v), ptr(a.dy);
  num(a.q_t), num(a.q_h), num(a.k_t), num(a.k_h), num(a.v_t), num(a.v_h), num(a.dy_t), num(a.dy_h);
  ptr(a.g), ptr(a.b), num(a.g_t), num(a.g_h), num(a.b_t), num(a.b_h);
  ptr(a.A), ptr(a.D), ptr(a.cu), ptr(a.s_in), ptr(a.s_out), ptr(a.ds_out), ptr(a.ds_in), num(a.s_k), num(a.s_v);
  ptr(a.o), ptr(a.dq), ptr(a.dk_out), ptr(a.dv_out), ptr(a.dg), ptr(a.db), ptr(a.dA), ptr(a.dD);
  ptr(a.chunks), ptr(a.doc_off), ptr(a.hd), ptr(a.rqk), ptr(a.qk), ptr(a.kk), ptr(a.pt);
  ptr(a.s_tiles), ptr(a.u_tiles), ptr(a.r_tiles), ptr(a.ds_tiles), ptr(a.dr_tiles), ptr(a.part);
  num(a.T), num(a.n_docs), num(a.Hk), num(a.Hv), num(a.dk), num(a.dv), num(a.nc_max), num(a.l2norm), num(a.step);
  a.doc_list = a.doc_off + a.n_docs + 3;
  a.dvp = (a.dv + 63) / 64 * 64;
  a.scale = scale;
  a.status = xb_status_ptr();
  return a;
}

XB_API int xb_recurrence_fwd(const long long* words, float scale, int delta, void* stream) {
  if (words == nullptr) return -1;
  const XbRecArgs a = unpack(words, scale);
  XbRecArgs chunked = a;
  if (a.s_tiles != nullptr) chunked.step = 0;                 // tiles are kept of all documents
  if (bad_args(chunked) || a.step < 0 || a.step >= C) return -1;
  cudaStream_t st = (cudaStream_t)stream;
  if (chunked.step == 0 || a.T > a.step) {                    // else no document has chunks
    if (int rc = prepare(chunked, delta, st)) return rc;
    if (int rc = delta ? xb_delta_fwd(chunked, st) : xb_scan_fwd(chunked, st)) return rc;
  }
  // behind the walk: with tiles it has written outputs and states of these documents too
  return a.step > 0 ? xb_recurrence_step(a, delta, st) : 0;
}

// kept: what the forward pass has left, 2: the operands of the chunks and the state tiles, 1: the operands, 0: nothing.
// The rest is made again.
XB_API int xb_recurrence_bwd(const long long* words, float scale, int delta, int kept, void* stream) {
  if (words == nullptr) return -1;
  const XbRecArgs a = unpack(words, scale);
  if (bad_args(a) || a.step > 0) return -1;
  cudaStream_t st = (cudaStream_t)stream;
  if (kept == 0)
    if (int rc = prepare(a, delta, st)) return rc;
  if (int rc = delta ? xb_delta_bwd(a, kept == 2, st) : xb_scan_bwd(a, kept == 2, st)) return rc;
  if (int rc = xb_recurrence_grad(a, delta, st)) return rc;
  return delta ? 0 : rec_launch(rec_reduce, a.Hv, 128, 0, a, st);
}
