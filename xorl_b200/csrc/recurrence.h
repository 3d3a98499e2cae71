// Arguments of the gated linear recurrences, as the kernels get them (recurrence.cu unpacks them).
#pragma once

struct XbRecArgs {
  // inputs: bf16 [T, heads, dim] with element strides of token and head (dim contiguous)
  const void *q, *k, *v, *dy;
  long long q_t, q_h, k_t, k_h, v_t, v_h, dy_t, dy_h;
  const float *g, *b;            // [T, Hv]: log decay (delta rule only), beta or dt
  long long g_t, g_h, b_t, b_h;
  const float *A, *D;            // [Hv], scan only
  const int* cu;                 // n_docs + 1 boundaries
  // states: fp32, [n_docs, Hv, dk * dv] with element strides s_k, s_v inside a head
  const float* s_in;
  float* s_out;
  const float* ds_out;           // gradient of the final states
  float* ds_in;
  long long s_k, s_v;
  // outputs
  void *o;                       // bf16 [T, Hv, dv]
  void *dq, *dk_out, *dv_out;    // bf16, contiguous
  float *dg, *db;                // [T, Hv]
  float *dA, *dD;                // [Hv]
  // workspaces
  void* chunks;                  // int4 [nc_max]: first token, tokens, document
  int* doc_off;                  // [n_docs + 3]: first chunk of every document
  int* doc_list;                 // [n_docs + 3], behind doc_off: how many documents have chunks, and which
  float* hd;                     // [nc_max, Hv, 192]
  float* rqk;                    // [nc_max, Hk, 128]
  float *qk, *kk;                // [nc_max, Hk, 64, 64] (delta rule: for the backward pass, null in calls without gradients)
  void* pt;                      // [nc_max, Hv]: operand tile [T; P], two planes, and a third of T: 40960 bytes (delta rule only)
  // operand tiles of [rows][hi 32 | lo 32] bf16, [nc_max, Hv, dvp / 32]: states entering and gradients of those leaving
  // the chunks (16 KB), U and dR (8 KB, delta rule only)
  void *s_tiles, *u_tiles, *ds_tiles, *dr_tiles;
  // third bf16 parts: scan, of the states (columns 0 .. 31 of a row) and of the gradients (32 ..), 16 KB per 32 columns;
  // delta rule, of U and of dR, 8 KB each per 64 columns
  void* r_tiles;
  float* part;                   // scan: [nc_max, Hv, 2]; delta rule: dR.v by 16 columns, [nc_max, Hv, dvp / 16, 64]
  int* status;                   // filled in by the entry points
  int T, n_docs, Hk, Hv, dk, dv, dvp, nc_max, l2norm, step;   // step: documents of so many tokens at most go token by token (0 in the chunked kernels where they take all); dvp: dv rounded up to 64
  float scale;
};
