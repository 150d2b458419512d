/*
 * sam3_seq_amd -- sequence operators around the adapted Linears (gfx950): root-mean-square norm with the residual's addition
 * and an 8-bit output with scales, rotary positions with several axes, attention over packed sequences with grouped heads.
 * They stand beside the trunk's LayerNorm, qkv split + 2-D rotary positions and attention (sam3_vit_amd.h; same library).
 *
 * Conventions as in sam3_lora_amd.h: device pointers unless said otherwise, `stream` = hipStream_t, element types dtype 0 = bf16,
 * 1 = fp32.  Return 0, or -22 (bad argument), -95 (outside what the kernels cover), -12 (workspace too small), -5 (launch
 * error); the text of the last error of the calling thread is sam3_seq_last_error().  Nothing is allocated and the host is
 * never made to wait: every call can be captured into a graph.
 */
#ifndef SAM3_SEQ_AMD_H
#define SAM3_SEQ_AMD_H
#include <stddef.h>
#include <stdint.h>
#ifdef __cplusplus
extern "C" {
#endif

const char* sam3_seq_last_error(void);

/*
 * RMS norm of rows x[M, C] (row pitch ldx elements; residual: ldr), C % 8 == 0, C <= 16384:
 *   h = x + residual (fp32, not rounded; residual NULL: h = x)      rstd = 1 / sqrt(mean(h^2) + eps)      y = h * rstd * weight
 * weight has the activations' type.  Outputs, each NULL or contiguous [M, C]:  y;  h_out (h, rounded once);  h_low [M, C / 8]
 * 16 bits (two bits for each element that bf16 took from h, for the backward's sums; with a bf16 h_out);  rstd_out [M] fp32
 * (what the backward takes);  q8 [M, C] bytes with scales fp32 [M, C / group] (group 32, 64 or 128; 0: [M, 1]):
 *   scale = max(max|y|, 2^-24) / fmt_max over the group's unrounded y,   q8 = fp8(y / scale)   (fmt: sam3_fp8_amd.h)
 * A row with a NaN has NaN in all its outputs but h_out.
 */
int sam3_seq_rms_norm_fwd(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight, void* y, void* h_out,
                          void* h_low, float* rstd_out, void* q8, float* scales, int group, int fmt, int64_t M, int C, float eps, int dtype,
                          void* stream);

/*
 * Gradients: gx = rstd (u - xhat mean(u xhat)) + gh   with u = gy weight, xhat = h rstd;  gw[c] = sum over the rows of gy xhat.
 * h is h_out of the forward (x without a residual), row pitch ldh; h_low (with ldh = C) or NULL; gx is the gradient of x and of the residual.  gy, gh [M, C]
 * contiguous, gh may be NULL.  gx or gw may be NULL.  gw has the weight's type; its sums are fp32, in a fixed order.
 */
size_t sam3_seq_rms_norm_bwd_workspace_bytes(int64_t M, int C);
int sam3_seq_rms_norm_bwd(const void* gy, const void* gh, const void* h, int64_t ldh, const void* h_low, const void* weight,
                          const float* rstd, void* gx, void* gw, int64_t M, int C, int dtype, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Rotary positions with several axes.  q [T, Hq, D], k [T, Hk, D] (k NULL: q alone), strides in elements (token, head; unit inside a
 * head); outputs contiguous.  Pair i (of `pairs`, 2 pairs <= D <= 256) of every head turns by the angle
 * positions[axis[i]][token] * 2 pi * turns[i]; the elements behind the 2 * pairs first are copied.
 *   halves 0: pair i is elements (2i, 2i + 1);  1: elements (i, i + pairs).
 *   positions [axes, T] with strides (axis, token) in elements; pos_type 0 = int32, 1 = int64, 2 = fp32.
 *   axis, turns: HOST arrays of `pairs` entries, read before the call returns.
 * inverse != 0 turns the other way: the gradient of the rotation.  Angles are reduced in 64 bits (turns is: the result is good to
 * fp32 at positions up to 2^30).  D % 8 == 0.
 */
int sam3_seq_rotary(const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh, void* q_out, void* k_out,
                    const void* positions, int64_t pos_sa, int64_t pos_st, int pos_type, int axes, const double* turns,
                    const unsigned char* axis, int pairs, int halves, int inverse, int64_t T, int Hq, int Hk, int D, int dtype,
                    void* stream);

/*
 * Attention over packed sequences with grouped heads.
 *   q [Tq, Hq, D], k, v [Tk, Hk, D], strides (token, head) in elements, unit inside a head, 16-byte alignment throughout; below 2^22, but
 *   those between the heads of k and v, and of q where Hq == Hk, which may be any.  Hq % Hk == 0, D % 8 == 0, D <= 128.
 *   Sequence b of B owns the query rows cu_q[b] .. cu_q[b+1] - 1 and the key rows cu_k[b] .. cu_k[b] + n - 1 with
 *   n = len_k[b], or cu_k[b+1] - cu_k[b] where len_k is NULL (int32, device; cu_q and cu_k
 *   do not decrease; values outside the tensors are clamped to them).
 *   causal: query i of n_q sees the keys j <= i + n - n_q (the last query sees all); otherwise every key.
 *   out [Tq, Hq, D] contiguous;  lse [Tq, Hq] fp32 (natural logarithm; NULL: not wanted).  A row that sees no key gives zeros and
 *   lse = -inf, and so do rows of no sequence.  stats [Tq, Hq, 2] fp32 is what the backward takes (NULL: not wanted).
 * max_q, max_k: the longest lengths if known (they choose the kernels and size the grid; longer sequences are still computed), or Tq and Tk.
 * sam3_seq_attn_workgroups: the workgroups of the forward's main launch (kernel 0) and of the backward's two (1: gq, 2: gk and gv) -- never
 * more than a small multiple of the tiles that Tq or Tk rows in B sequences can have -- or -95 where they exceed what can be launched
 * (2^32 threads: B * Hk in the tens of millions), as the calls do.
 * Key and value rows that a query does not see never enter its result, whatever they hold.
 */
int64_t sam3_seq_attn_workgroups(int kernel, int64_t Tq, int64_t Tk, int B, int Hq, int Hk, int D, int64_t max_q, int64_t max_k, int dtype);
size_t sam3_seq_attn_fwd_workspace_bytes(int64_t Tq, int B, int Hq, int Hk, int D, int64_t max_q, int64_t max_k, int dtype);
int sam3_seq_attn_fwd(const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh, const void* v,
                      int64_t v_st, int64_t v_sh, const int32_t* cu_q, const int32_t* cu_k, const int32_t* len_k, void* out,
                      float* lse, float* stats, int64_t Tq, int64_t Tk, int B, int Hq, int Hk, int D, int64_t max_q, int64_t max_k, int causal,
                      float scale, int dtype, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Its gradients, each sum in a fixed order: gq [Tq, Hq, D], gk, gv [Tk, Hk, D] contiguous, from go [Tq, Hq, D] (strides as q's), out and
 * stats of the forward (contiguous) and the forward's inputs.  gk and gv may both be NULL: not wanted, and not computed.  Rows of no sequence get zeros.  The workspace holds three fp32 for each row.
 */
size_t sam3_seq_attn_bwd_workspace_bytes(int64_t Tq, int Hq);
int sam3_seq_attn_bwd(const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh, const void* v,
                      int64_t v_st, int64_t v_sh, const void* go, int64_t go_st, int64_t go_sh, const void* out, const float* stats,
                      const int32_t* cu_q, const int32_t* cu_k, void* gq, void* gk, void* gv, int64_t Tq, int64_t Tk, int B, int Hq,
                      int Hk, int D, int64_t max_q, int64_t max_k, int causal, float scale, int dtype, void* workspace,
                      size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif
