/*
 * actune_b200 serving operators: what a batch of requests runs beside the packed
 * projections of a decoder layer.  No reference counterpart.  Conventions of
 * actune_b200.h: device pointers on the current device, caller-owned buffers,
 * asynchronous on `stream`, actune_status return codes, no allocation, capturable
 * into a CUDA graph after one call of the same kernel.
 *
 * Operands are passed in a struct; fields left zero take their documented default.
 * `struct_bytes` is sizeof the struct the caller was compiled with (any other size
 * is refused).  Strides are in elements.
 */
#ifndef ACTUNE_B200_SERVING_H
#define ACTUNE_B200_SERVING_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* The glue between two blocks of a decoder layer, in one pass over a row:
 *     u = N(x; post_weight)                    (u = x without post_weight)
 *     s = residual_scale * residual + gate * u (gate = 1 without gate)
 *     h = N(s; pre_weight) + shift             (no shift: 0)
 *     N(a; w) = a * rsqrt(mean(a^2) + eps) * w         (gemma != 0: 1 + w)
 * s is kept in fp32 for h and rounded once to residual_out; h is rounded once to out.
 * x, residual: [T, D] of `dtype` with row strides x_stride / residual_stride; out and
 * residual_out: [T, D] contiguous, overlapping no input.  Each modulation (post_weight,
 * pre_weight, gate, shift; all of `dtype`) is rows of D, row r of the batch reading row
 * r / <name>_rows of it; <name>_rows = 0: one row for the whole batch.
 * quant_bits in {2, 4, 8}: also the group-64 activations of out (D % 64 == 0), as
 * actune_quantize_group64 (codes8 = 0) or actune_quantize_group64_codes (codes8 = 1)
 * would give for it, bit for bit; packed 8-byte aligned, scales float [T, D/64]. */
typedef struct actune_gated_norm_args {
  size_t struct_bytes;
  const void* x;
  const void* residual;
  const void* post_weight; /* or NULL */
  const void* pre_weight;
  const void* gate;  /* or NULL */
  const void* shift; /* or NULL */
  void* out;
  void* residual_out;
  uint8_t* packed; /* with quant_bits */
  float* scales;
  int64_t T, D;
  int64_t x_stride, residual_stride;
  int64_t post_rows, pre_rows, gate_rows, shift_rows;
  float residual_scale, eps;
  int32_t dtype, gemma, quant_bits, codes8;
} actune_gated_norm_args;

int actune_gated_norm(const actune_gated_norm_args* args, void* stream);

/* Low-rank adapters of many requests at once, beside a projection they share:
 *     out[m] = y[m] + scale[s] * up[s] (down[s] x[m]),   s = slots[m],
 * for y the shared projection's output; rows whose slot is outside 0 .. S-1 keep y[m].
 *
 * actune_adapter_plan sorts the rows of a batch by slot (stable) into tiles of `tile`
 * rows (4, 16 or 128) that share one adapter; every projection and layer the batch
 * passes through reads the same plan.  slots: int32 [M] on the device, so a captured
 * graph can follow a batch whose routing changes.  plan: int32 buffer of
 * actune_adapter_plan_size(M, S, tile) bytes, 16-byte aligned.  S <= 8191.
 *
 * actune_adapter_add: x [M, K], y and out [M, N], down [S, R, K], up [S, N, R], all of
 * `dtype` (F16 or BF16), 1 <= R <= 128; scale float [S]; x, y and out have row strides;
 * out may be y itself (same pointer and stride), and overlaps nothing else.  down x
 * is summed in fp32 and goes through the workspace (16-byte aligned, at least
 * actune_adapter_workspace_size bytes).  Where the second product is one of matrix
 * instructions (all but tiles of 4 in the vector form with R <= 64 a multiple of 8) it enters
 * it as two parts of `dtype`: 16 bits of significand in bf16, 22 in fp16.  up (down x) is
 * summed in fp32, and the result is rounded once.  Any K, N, R and
 * alignment; 16-byte aligned operands with K, N and the strides multiples of 8 and R a
 * multiple of 4 run the vector form. */
size_t actune_adapter_plan_size(int64_t M, int64_t S, int tile);
int actune_adapter_plan(const int32_t* slots, int64_t M, int64_t S, int tile, int32_t* plan, void* stream);

typedef struct actune_adapter_args {
  size_t struct_bytes;
  const void* x;
  const void* y;
  const void* down;
  const void* up;
  const float* scale;
  const int32_t* plan;
  void* out;
  void* workspace;
  size_t workspace_bytes;
  int64_t M, N, K, S, R;
  int64_t x_stride, y_stride, out_stride;
  int32_t tile, dtype;
} actune_adapter_args;

size_t actune_adapter_workspace_size(int64_t M, int64_t K, int64_t S, int64_t R, int tile);
int actune_adapter_add(const actune_adapter_args* args, void* stream);

/* Attention of a batch whose sequences share long prefixes.  Sequence b has T query
 * tokens, S rows of keys and values of its own, of which the first lens[b] count, and
 * the prefix g it belongs to (starts[g] <= b < starts[g + 1]), of P rows, of which the
 * first prefix_lens[g] count.  Query head h reads key/value head h / (H / KV).
 *     out[b, t, h] = sum_j p_j v_j,  p = softmax over the keys seen of scale * q . k_j
 * over the prefix and the sequence's own keys; with causal != 0, query t sees own key j
 * only for j <= lens[b] - T + t.  A query that sees no key gets zeros, and rows of the
 * caches that nothing sees are not used whatever they hold.
 * starts: int32 [G + 1], non-decreasing from 0 to B (NULL: sequence b has prefix
 * b * G / B); prefix_lens, lens: int32 [G], [B] (NULL: all of P, S; values outside are
 * clamped).  All three are read on the device.
 * q [B, T, H, D], prefix_k and prefix_v [G, P, KV, D], k and v [B, S, KV, D], D <= 256,
 * of `dtype` (F16 or BF16), with D contiguous and the given strides; out [B, T, H, D]
 * contiguous, overlapping no input.  Scores, softmax and sums are fp32; p is rounded to
 * `dtype` for the product with V, as the tensor core takes it.  A value of v that is not
 * finite may reach queries of its own sequence that causal keeps from it, and reaches no
 * other sequence.
 * workspace: at least actune_prefix_attention_workspace_size bytes, 16-byte aligned.
 * Operands with D a multiple of 8, 16-byte aligned, and strides that are positive
 * multiples of 8 run on the tensor cores; others on a scalar kernel. */
typedef struct actune_prefix_attention_args {
  size_t struct_bytes;
  const void* q;
  const void* prefix_k;
  const void* prefix_v;
  const void* k;
  const void* v;
  const int32_t* starts;
  const int32_t* prefix_lens;
  const int32_t* lens;
  void* out;
  void* workspace;
  size_t workspace_bytes;
  int64_t B, T, H, KV, D, G, P, S;
  int64_t q_b, q_t, q_h;    /* strides of q by sequence, token and head */
  int64_t pk_g, pk_p, pk_h; /* of prefix_k by prefix, row and head */
  int64_t pv_g, pv_p, pv_h;
  int64_t k_b, k_s, k_h;
  int64_t v_b, v_s, v_h;
  float scale;
  int32_t dtype, causal;
} actune_prefix_attention_args;

/* ragged: whether starts will be given. */
size_t actune_prefix_attention_workspace_size(int64_t B, int64_t T, int64_t H, int64_t KV, int64_t D, int64_t G,
                                              int64_t P, int64_t S, int ragged);
int actune_prefix_attention(const actune_prefix_attention_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* ACTUNE_B200_SERVING_H */
