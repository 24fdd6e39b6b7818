/*
 * include/xs_block.h - the operators around and beside the MoE layer: the norm before a block, the join after one (its
 * gate, its scales, the next block's norm), and products of int8 rows with a scale a token and a scale an output (dense
 * layers and experts kept in int8).  None has a counterpart in the reference's MoE path: its norm is the engine's
 * native_qsa_rms_norm_weighted (called at src/core/plain_model.cpp:953 and src/prefill/plain_prompt.cpp:560), its
 * residual add add_inplace (src/core/plain_model.cpp:987), its int8 products iq_mmq's (a scale a 32-value block).
 *
 * Conventions are include/xs_moe.h's: device memory of the caller, nothing allocated, no state between calls (calls on
 * different streams share nothing), return codes and xs_last_error(); a NULL stream is HIP's default stream and the call
 * then synchronises.  Zero or fewer tokens: nothing is done; norms, joins and quantizations take up to 2^21.  Rows are n
 * values long and ld values apart (ld >= n); what lies between is neither read as data nor written.  Every pointer is aligned to its values' size; outputs overlap no
 * input and no other output, except where an entry says so; columns of one buffer (rows of one stride between each
 * other's) are apart.
 *
 * Types of float rows are ggml's ids: F32 0, F16 1, BF16 30.  Results are computed in fp32, each product and sum
 * rounded on its own, and rounded once more (to nearest even) where they are stored in 16 bits.
 *
 * int8 rows: codes q and a float scale s a row; the row's values are q s.  A row of values v is quantized as
 *   s = max(max |v| fl(1 / 127), 2^-126) (one product, as xs_quantize_q8_1_rows takes its scale: within 0.57 steps of
 *       max |v| / 127),
 *   q = the integer nearest the exact v / s (halves to even);
 * a row that holds a NaN or an infinity gets s = NaN and q = 0, so everything computed from it is NaN.
 */
#ifndef XS_BLOCK_H
#define XS_BLOCK_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define XS_F32 0
#define XS_F16 1
#define XS_BF16 30

/* The norm before a block: y[t, c] = (x[t, c] r) w[c], r = 1 / sqrt(mean of x[t, .]^2 + eps) (the mean and the root in 64
 * bits, r rounded once; rows that 16-byte accesses take give the same bits in a call of any number of rows, other rows may
 * differ in r's last bit).  w NULL: no weights.  y (y_type, ldy) and the int8 rows of the fp32 y (q, ldq bytes apart, and
 * q_scale [n_tok]) are written where given; one of them has to be.  y may be x itself (the same type and ld).
 * n_embd 1 .. 16384; eps finite, not negative. */
int xs_block_norm(const void* x, int x_type, int64_t ldx, const float* w, float eps, void* y, int y_type, int64_t ldy,
                  int8_t* q, int64_t ldq, float* q_scale, int64_t n_tok, int64_t n_embd, void* stream);

/* How a block's output b joins the residual stream:
 *   norm: b = the norm above of b (norm_w, norm_eps)
 *   gate: b = b g, g by gate_kind: a token's 1 / (1 + exp(-gate[t])) (taken in 64 bits, rounded once), a channel's
 *         multiplier gate[c], or a value's gate[t ld_gate + c]
 *   out  = residual_scale residual + branch_scale b, rounded to the residual's type
 *   next: the norm above of `out` as stored (next_w, next_eps): the next block's input
 * norm_w and next_w may be NULL (no weights). */
#define XS_GATE_NONE 0
#define XS_GATE_TOKEN 1
#define XS_GATE_CHANNEL 2
#define XS_GATE_VALUE 3
typedef struct xs_block_join_cfg {
    int norm; /* 1: the block's output is normed first */
    const float* norm_w;
    float norm_eps;
    int gate_kind;
    const float* gate;
    int64_t ld_gate;
    float branch_scale, residual_scale;
    const float* next_w;
    float next_eps;
} xs_block_join_cfg_t;

/* The join of rows y: out and, where given, the next block's rows (next, next_type, ld_next) and / or their int8 rows
 * (q, ldq, q_scale).  residual and out are of type r_type, ldr values apart; out may be residual.  next may be y itself
 * (the same type and ld).  n_embd 1 .. 16384. */
int xs_block_join(const xs_block_join_cfg_t* J, const void* y, int y_type, int64_t ldy, const void* residual, void* out,
                  int r_type, int64_t ldr, void* next, int next_type, int64_t ld_next, int8_t* q, int64_t ldq,
                  float* q_scale, int64_t n_tok, int64_t n_embd, void* stream);

/* The join of an MoE layer's parts: a token's block output is the weighted sum of its k rows of `parts` (routing order,
 * n_embd floats each) in rank order, + its row of `shared` once (times 1 / (1 + exp(-shared_gate[t])) where given, taken
 * as the token gate above).  Order and roundings are xs_native_moe_combine_multi's, whose bits the sum has without
 * shared_gate; that entry point takes the gate's sigmoid in fp32, four roundings where this one has one, so that a gated
 * shared row's values may differ by 7 * 2^-24 of themselves before they are added.  k in 1 .. 15. */
int xs_moe_combine_join(const xs_block_join_cfg_t* J, const float* parts, const float* weights, int64_t k,
                        const float* shared, const float* shared_gate, const void* residual, void* out, int r_type,
                        int64_t ldr, void* next, int next_type, int64_t ld_next, int8_t* q, int64_t ldq,
                        float* q_scale, int64_t n_tok, int64_t n_embd, void* stream);

/* Rows of floats to int8 rows.  cols 1 .. 65536. */
int xs_w8a8_quantize(const void* x, int x_type, int64_t ldx, int8_t* q, int64_t ldq, float* q_scale, int64_t rows,
                     int64_t cols, void* stream);

/* y[t, o] = (sum over k of x[t, k] w[o, k]) x_scale[t] w_scale[o]: the sum exact in 32-bit integers, then taken to fp32
 * and multiplied by the token's and by the output's scale, in that order.  x and w are 16-byte aligned, ldx and ldw
 * multiples of 16 bytes, at least n_in rounded up to one and at most 2^23: bytes between n_in and that multiple are read but
 * do not count.  n_in 1 .. 65536, n_tok up to 2^20, n_out up to 2^24. */
int xs_w8a8_gemm(const int8_t* x, int64_t ldx, const float* x_scale, const int8_t* w, int64_t ldw, const float* w_scale,
                 void* y, int y_type, int64_t ldy, int64_t n_tok, int64_t n_in, int64_t n_out, void* stream);

/* The gated pair: h[t, j] = g / (1 + exp(-g)) u with g and u the fp32 products above of row t with the gate rows and with
 * the up rows (n_ff each, both ldw bytes apart).  The bytes of x and of the weights as for xs_w8a8_gemm. */
int xs_w8a8_swiglu(const int8_t* x, int64_t ldx, const float* x_scale, const int8_t* w_gate, const float* gate_scale,
                   const int8_t* w_up, const float* up_scale, int64_t ldw, void* h, int h_type, int64_t ldh,
                   int64_t n_tok, int64_t n_in, int64_t n_ff, void* stream);

#ifdef __cplusplus
}
#endif
#endif
