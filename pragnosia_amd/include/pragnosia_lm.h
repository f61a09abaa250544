/* pragnosia_lm.h -- C ABI of libpragnosia_hip.so, part two: the language model's two ends around the carriers (the
 * token table's lookup with its gradient, and the losses of the head over the vocabulary with theirs).
 *
 * The conventions are pragnosia_hip.h's: device pointers, dense row-major, 16-byte aligned; stream-ordered; nothing
 * allocates or synchronises and nothing records a memset, so every call can be captured; 0 on success, a hipError_t
 * (> 0) if a launch failed, a negative PRAGNOSIA_ERR_* code if the arguments were rejected before anything was launched
 * (pragnosia_error_string names any code). Calls that may overlap each need a workspace of their own. */
#ifndef PRAGNOSIA_LM_H
#define PRAGNOSIA_LM_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ABI version of this header (1); bumped on any change of its entry points. */
int pragnosia_lm_abi_version(void);

/* ---------------------------------------------------------------------------------------------------------
 * Losses of the head l = h W^T over n rows and V classes, with no logits kept: the cross entropy of a label, the
 * distillation loss from a teacher's K top logits, or both from one pass. (The reference's LM forms the logits in
 * chunks and recomputes them, src/model.py:563-567; it distils from no teacher.)
 *
 *   lse_i = log sum_v exp l_iv        ce_i = lse_i - l_{i, y_i}; 0 where y_i is outside [0, V)
 *   p_i   = softmax over k of z_ik / tau, over the entries with ids_ik in [0, V) (an id may repeat); z = -inf: p = 0
 *   lse_t = log sum_v exp(l_iv / tau) P_iv  = sum of p_ik over the k with ids_ik = v
 *   kd_i  = tau^2 sum_v P_iv (log P_iv - l_iv / tau + lse_t_i), tau^2 KL(P_i || softmax(l_i / tau)); 0 where no entry
 *           is left
 *
 * h (n, d) and W (V, d) bf16, d a multiple of 8; y (n) int64 or NULL (no ce); ids (n, K) int64 and z (n, K) fp32, or
 * both NULL with K = 0 (no kd), K at most 1024; at least one of y and ids; tau from 2^-10 to 2^10. n and V at most
 * 2^24, d at most 65536, n K below 2^31. Outputs, all fp32 but `entry`: ce and lse (n) with y; kd, lse_t and psum (n),
 * entry (n, K) int32, p and zl (n, K) with ids -- lse, lse_t, psum (1, or 0 where no entry is left), entry (the id at
 * its first place in the list, or -1), p (an id's whole probability there, or 0) and zl (the student's logit of the
 * entry) are what the backward takes. A NaN among a row's present z makes its kd NaN. */
int64_t pragnosia_head_fwd_workspace_bytes(int64_t n, int64_t V, int64_t d, int64_t K);
int pragnosia_head_fwd(const void* h, const void* W, const int64_t* y, const int64_t* ids, const float* z, float tau,
                       float* ce, float* lse, float* kd, float* lse_t, float* psum, int32_t* entry, float* p, float* zl,
                       void* workspace, int64_t workspace_bytes, int64_t n, int64_t V, int64_t d, int64_t K,
                       void* stream);

/* Backward: from the gradients of ce, lse and kd (n each, fp32, NULL = zero),
 *   dl_iv = (g_ce_i [y_i in range] + g_lse_i) exp(l_iv - lse_i) - g_ce_i [v = y_i]
 *         + tau g_kd_i (psum_i exp(l_iv / tau - lse_t_i) - sum_k p_ik [v = ids_ik])
 * rounded to bf16, then dh = dl W (n, d) bf16 and dW = dl^T h (V, d), bf16 or (dw_f32) fp32; either may be NULL. The
 * logits are formed again in pieces of the vocabulary. Rows whose three gradients are zero get a zero dl whatever h
 * holds there, and a row whose g_kd is zero takes nothing from its p, which may be NaN. */
int64_t pragnosia_head_bwd_workspace_bytes(int64_t n, int64_t V, int64_t d);
int pragnosia_head_bwd(const float* g_ce, const float* g_lse, const float* g_kd, const void* h, const void* W,
                       const int64_t* y, const float* lse, const float* lse_t, const float* psum, const int32_t* entry,
                       const float* p, const float* zl, float tau, void* dh, void* dW, int dw_f32, void* workspace,
                       int64_t workspace_bytes, int64_t n, int64_t V, int64_t d, int64_t K, void* stream);

/* ---------------------------------------------------------------------------------------------------------
 * Rows of a token table: y_i = scale W[ids_i], n rows; an id outside [0, V) gives a zero row. W (V, d) and y (n, d)
 * fp32 or bf16 (w_bf16, y_bf16), d a multiple of 8, n at most 2^27 and V 2^28; ids (n) int64. kept (n) int32 or NULL:
 * the ids in 32 bits for the backward, which then reads half as much (-1 outside the table). n = 0 does nothing. Replaces
 * nn.Embedding of src/model.py:822-826 (scale 1). */
int pragnosia_embed_fwd(const int64_t* ids, const void* W, int w_bf16, float scale, void* y, int y_bf16, int32_t* kept,
                        int64_t n, int64_t V, int64_t d, void* stream);

/* Its gradient: dW[v] = scale sum of g_i over the tokens with ids_i = v, in fp32 in a fixed order, zero where there is
 * none; g (n, d) and dW (V, d) fp32 or bf16; ids (n) int64 (ids_64) or int32, ids outside the table taking no part. No
 * atomics on values, no memset: the same bits each time, also in a captured step. No workspace up to 256 tokens. */
int64_t pragnosia_embed_bwd_workspace_bytes(int64_t n, int64_t V, int64_t d);
int pragnosia_embed_bwd(const void* g, int g_bf16, const void* ids, int ids_64, float scale, void* dW, int w_bf16,
                        void* workspace, int64_t workspace_bytes, int64_t n, int64_t V, int64_t d, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* PRAGNOSIA_LM_H */
