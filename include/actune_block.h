/*
 * actune_block.h - C ABI of libactune_block.so: the operators between a
 * decoder block's packed projections on MI355X (gfx950).
 *
 *   actune_block_norm        residual update with gate and residual scale,
 *                            the norms behind a block and before the next
 *   actune_adapter_add       low-rank adapters of many requests added to a
 *                            shared projection's output
 *   actune_prefix_attention  attention of a batch over a prefix it shares
 *                            and over keys of its own
 *
 * Plain pointers, sizes and a hipStream_t passed as void*. No allocation, no
 * host synchronisation, no exceptions: every entry point is legal inside
 * hipStreamBeginCapture and returns a status; on failure
 * actune_block_last_error() holds a message for the calling thread. Invalid
 * arguments are reported before anything is launched. Strides are in
 * elements; the last dimension of every tensor is dense. Outputs must not
 * overlap inputs unless an entry point says so.
 */
#ifndef ACTUNE_BLOCK_H
#define ACTUNE_BLOCK_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes and dtype codes are those of actune_hip.h:
 * 0 ok, 1 invalid argument, 2 HIP error; 0 bf16, 1 f16, 2 f32. */

/* Message of the last failed call on this thread ("" if none). */
const char* actune_block_last_error(void);

/*
 * hidden = residual_scale * residual + gate * branch'
 * normed = rms(hidden) * (weight_offset + weight) * (1 + scale) + shift
 * with rms(x) = x / sqrt(mean(x^2) + eps) over a row of D, and branch' =
 * branch, or rms(branch) * (weight_offset + branch_weight) where
 * branch_weight is given. One dtype for all tensors; every step in f32, each
 * output rounded once (normed from the unrounded hidden).
 *
 * residual, branch: [M, D] with row strides; hidden, normed: [M, D], dense.
 * NULL: branch (hidden = residual_scale * residual), gate (1), weight (the
 * factor 1, without the offset), scale (0), shift (0), hidden (not written).
 * gate, scale, shift: rows of D elements; row m of the call reads row
 * m / X_rows, or row 0 where X_rows is 0.
 */
typedef struct actune_block_norm_args {
  const void* residual;
  const void* branch;
  const void* branch_weight; /* [D] */
  const void* weight;        /* [D] */
  const void* gate;
  const void* scale;
  const void* shift;
  void* hidden;
  void* normed;
  int64_t residual_stride, branch_stride;
  int64_t gate_stride, scale_stride, shift_stride;
  int64_t gate_rows, scale_rows, shift_rows;
  int64_t M, D;
  float residual_scale, weight_offset, eps;
  int32_t dtype;
} actune_block_norm_args;

int actune_block_norm(const actune_block_norm_args* args, void* stream);

/*
 * out[m] = y[m] + scaling[id] * B[id] (A[id] x[m]) with id =
 * ids[m / ids_rows]; a row whose id is not in [0, L) gets
 * out[m] = y[m]. Products of the 16-bit inputs are exact and summed in f32;
 * A x is held as two 16-bit parts (about 16 bits of mantissa in bf16, 21 in
 * f16) under one power of two for each row in the second product; out is
 * rounded once. Infinities and NaN give what the formula gives. An adapter's
 * values reach only the rows that name it, whatever they are.
 *
 * x: [M, K] and y, out: [M, N] with row strides (out may be y itself, with
 * y's row stride); a: [L, R, K], b: [L, N, R], both dense; scaling: f32 [L];
 * ids: int32, one for each ids_rows rows. x, y, a, b and out have one dtype,
 * bf16 or f16. 1 <= R <= 128.
 * workspace: actune_adapter_workspace_bytes(M, N, K, R) bytes, 16-byte
 * aligned, no other call's at the same time.
 */
typedef struct actune_adapter_args {
  const void* x;
  const void* y;
  const void* a;
  const void* b;
  const float* scaling;
  const int32_t* ids;
  void* out;
  void* workspace;
  int64_t workspace_bytes;
  int64_t x_stride, y_stride, out_stride;
  int64_t ids_rows;
  int64_t M, N, K, R, L;
  int32_t dtype;
} actune_adapter_args;

/* Workspace of a call in bytes; -1 for sizes that no call takes. */
int64_t actune_adapter_workspace_bytes(int64_t M, int64_t N, int64_t K, int64_t R);
int actune_adapter_add(const actune_adapter_args* args, void* stream);

/*
 * Attention of B sequences in G equal groups, T queries each: sequence b sees
 * the P keys of prefix b / (B / G), which the group shares, and S keys of its
 * own.
 *   score_j = scale * q . k_j      out = sum_j softmax(score)_j v_j
 *   lse = log(sum_j exp(score_j))
 * over prefix keys j < prefix_lengths[g] with prefix_mask[g, j] != 0 and own
 * keys j < lengths[b]; causal: query t sees own keys j <= lengths[b] - T + t.
 * Lengths are clamped to [0, P] and [0, S]. A query that sees no key: out 0,
 * lse -inf. Keys and values that a query does not see may hold anything, NaN
 * included. Scores, statistics and sums are f32; the probabilities are rounded
 * to the call's type for their product with the values.
 *
 * q: [B, T, Hq, D]; prefix_k, prefix_v: [G, P, Hkv, D]; k, v: [B, S, Hkv, D];
 * out: [B, T, Hq, D], dense; lse: f32 [B, T, Hq], dense, or NULL. bf16 or
 * f16, one dtype. D a multiple of 8, at most 256; Hq a multiple of Hkv; query
 * head h reads key head h / (Hq / Hkv). Strides {batch or group, token, head}
 * are multiples of 8 elements and data 16-byte aligned; a token stride of
 * keys or values is below 2^23 elements. prefix_lengths: int32 [G] or NULL
 * (P); prefix_mask: bytes, rows of P at stride mask_stride, or NULL; lengths:
 * int32 [B] or NULL (S). P or S may be 0 (their pointers are not read then).
 * workspace: actune_prefix_attention_workspace_bytes(args) bytes (no pointer
 * of args is read), 16-byte aligned, no other call's at the same time.
 */
typedef struct actune_prefix_attention_args {
  const void* q;
  const void* prefix_k;
  const void* prefix_v;
  const void* k;
  const void* v;
  const int32_t* prefix_lengths;
  const uint8_t* prefix_mask;
  const int32_t* lengths;
  void* out;
  float* lse;
  void* workspace;
  int64_t workspace_bytes;
  int64_t q_stride[3], prefix_k_stride[3], prefix_v_stride[3], k_stride[3], v_stride[3];
  int64_t mask_stride;
  int64_t B, G, T, Hq, Hkv, D, P, S;
  float scale;
  int32_t causal;
  int32_t dtype;
} actune_prefix_attention_args;

/* Workspace of a call in bytes; -1 for sizes that no call takes. */
int64_t actune_prefix_attention_workspace_bytes(const actune_prefix_attention_args* args);
int actune_prefix_attention(const actune_prefix_attention_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* ACTUNE_BLOCK_H */
