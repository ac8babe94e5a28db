// Host entry points of the trajectory form's kernels (attention_scan.cuh, one
// translation unit per element type) and the launch's description.
#pragma once
#include "b200policy.h"
#include <cuda_runtime.h>

namespace b200policy {

// One causal scan over a row's tokens, in token order or backward:
//   out_i = out_scale * (sum_{j <= i} w_ij pair_scale (q_i . k_j) v_j + into_i q_i S)
// with S [kd, vd] the state before the row, and w and into the products of the
// decays between the tokens.  The forward pass is one scan; the gradients are
// three (dq: do, v, k; dk: v, do, q backward; dv: k, q, do backward).
struct Scan {
  const void *q, *k, *v;
  int64_t q_batch, q_time, q_head, k_batch, k_time, k_head, v_batch, v_time, v_head;
  int q_shared, k_shared, v_shared;  // read at the key / value head
  const float *init;                 // before the row; element (i, j) at i * init_row + j * init_col; NULL: zero
  int64_t init_row, init_col;
  void *out;     // dense [batch, time, heads, vd]
  int out_float; // out is float whatever the elements' type
  float *final;  // dense [batch, heads, kd, vd] after the row; NULL: not wanted
  int kd, vd;
  int reverse;
  int parts; // terms of the weighted keys in bf16: 3 where `final` is wanted
  float pair_scale, out_scale;
  int vec_q, vec_k, vec_v, vec_out, vec_final;  // 16-byte accesses are aligned
  // A second output with the same state, read the other way round (S transposed):
  //   twin_out_i = sum_{j <= i} w_ij pair_scale (x_i . v_j) k_j + into_i x_i S^T
  // dk beside dv: one state is kept instead of two.  Heads of up to 64, 16-bit.
  const void *x;
  int64_t x_batch, x_time, x_head;
  int x_shared, vec_x;
  void *twin_out;  // dense [batch, time, heads, kd]; NULL: none
  int vec_twin;
  int slices;                        // of vd
};

struct ScanParams {
  Scan scan[3];
  int scans;
  int units;  // (scan, slice) pairs
  const float *log_decay;
  const uint8_t *first;
  int64_t first_batch, first_time;
  const int32_t *lengths;
  int batch, time, heads, group;
  // long rows are split into pieces: first each piece's own state (state_only),
  // then their sums, then every piece from its sum
  int pieces, piece, state_only;
  float *states;   // [scan][batch * heads][pieces][kd * vd]
  float *factors;  // [scan][batch * heads][pieces]: what is left of the state before the piece
  int64_t states_at[3];
};

constexpr int kTile = 64;         // tokens of a chunk
constexpr int kScanThreads = 128;

template <class T> int scan_resident(int kt, int vt);
template <class T> int scan_launch(const ScanParams &p, int kt, int vt, cudaStream_t s);

// bf16 heads wider than 64 on tcgen05 (attention_tc.cu): chunks of 128 tokens,
// aligned tensors, slices of 64, one CTA an SM.
constexpr int kTcTile = 128;
// call: a number for the status word, not zero, of all launches of one call.
int scan_tc_launch(const ScanParams &p, int *status, int call, cudaStream_t s);

}  // namespace b200policy
