/* pragnosia_gen.h -- C ABI of libpragnosia_hip.so, part three: generation from 4-bit weights under rules (weights rounded
 * to 4 bits and read back, rows times such a weight, penalties, biases and masks on logits and the token they leave).
 *
 * The conventions are pragnosia_hip.h's: device pointers, dense row-major, 16-byte aligned; stream-ordered; nothing
 * allocates or synchronises and nothing records a memset, so every call can be captured; 0 on success, a hipError_t
 * (> 0) if a launch failed, a negative PRAGNOSIA_ERR_* code if the arguments were rejected before anything was launched
 * (pragnosia_error_string names any code). Calls that may overlap each need a workspace of their own. */
#ifndef PRAGNOSIA_GEN_H
#define PRAGNOSIA_GEN_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ABI version of this header (1); bumped on any change of its entry points. */
int pragnosia_gen_abi_version(void);

/* ---------------------------------------------------------------------------------------------------------
 * 4-bit weights. A weight W (N, K), fp32 or bf16 (bf16), becomes codes with one scale for each row's group of `group`
 * columns (32, 64 or 128; the last group may be short):
 *
 *   s = bf16(max |w| / 6) over the group (the quotient rounded to fp32, then to bf16, each to nearest even), NaN where
 *       the group holds an infinity or a NaN
 *   v = the one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (e2m1, codes 0 .. 7, with a sign bit) nearest to w / s, an even code in a
 *       tie, 6 past 6
 *   w is then s v. A group of zeros has s = 0.
 *
 * N at most 2^26, K a multiple of 8 up to 65536. Codes lie in tiles of 16 rows by 128 columns, ceil(K / 128) tiles to a
 * block of rows, 1024 bytes each: lane l of a wave has the 16 bytes at 16 l, row l % 16 of the tile, and its 32-bit
 * word j holds columns 32 j + 8 (l / 16) + 0 .. 7, the first in the lowest four bits. Scales (bf16) lie tile by tile
 * too, 16 rows by 128 / group each, row-major. Rows past N and columns past K hold zeros. */
int64_t pragnosia_fp4_code_bytes(int64_t N, int64_t K);
int64_t pragnosia_fp4_scale_bytes(int64_t N, int64_t K, int64_t group);
int pragnosia_fp4_quantize(const void* W, int bf16, void* codes, void* scales, int64_t N, int64_t K, int64_t group,
                           void* stream);

/* W = s v in fp32 (exact) or bf16 (rounded once). */
int pragnosia_fp4_dequantize(const void* codes, const void* scales, void* W, int bf16, int64_t N, int64_t K,
                             int64_t group, void* stream);

/* y = act(z W^T + bias) + resid for n rows: z = x, or with ln_weight (K) the LayerNorm of x's rows with ln_weight, ln_bias
 * (K, or NULL) and ln_eps; act 0: identity, 1: GELU (erf form); bias (N) and resid (n, N) may be NULL. x (n, K), the
 * norm's, bias, resid and y (n, N) all fp32 or all bf16 (bf16). Sums are fp32; fp32 rows and normalised rows of either type
 * are multiplied whole (as three bf16 parts; what lies below 2^-126 may be lost), other bf16 rows as they are. A group's sum
 * of z v is formed before its scale s, so values of z past 2^118 may overflow. y may be resid, and must not overlap x.
 * n at most 2^24, n N and n K below 2^31. n = 0 does nothing. */
int pragnosia_fp4_linear(const void* x, int bf16, const void* codes, const void* scales, const void* ln_weight,
                         const void* ln_bias, float ln_eps, const void* bias, int act, const void* resid, void* y,
                         int64_t n, int64_t N, int64_t K, int64_t group, void* stream);

/* ---------------------------------------------------------------------------------------------------------
 * Rules on logits l (B, V), fp32 or bf16 (bf16). For row b and word v, in fp32, each step rounded:
 *
 *   a word among history[b][0 .. lengths[b]):   x = l / r if l > 0, else l r             (r = repetition)
 *   c times among [prompt[b] .. lengths[b]):    x -= presence if c > 0, then x -= frequency c
 *   a word of the row's bias list:              x += its value (of the last entry that names it)
 *   a word whose mask bit is clear:             x = -inf
 *
 * history (B, L) int64 with rows history_stride apart, or NULL with L = 0; ids outside [0, V) take no part. lengths and
 * prompt (B) int64: NULL stands for L and 0, values are clamped to [0, L]. Each of the three penalties is an array of B
 * values or, with NULL, the number beside it; r must not be 0. bias_ids (int64) and bias_values (fp32): M entries to a
 * row, rows bias_stride apart (0: all rows share one list); ids outside [0, V) are skipped. mask (S, ceil(V / 32)) 32-bit
 * words, word v's bit v % 32 of word v / 32; state (B) int64 is each row's line of the mask (NULL: line b, or line 0 if
 * S = 1); a negative one leaves the row unmasked, one of S or more masks every word. S = 0: no mask.
 *
 * One of out and tokens is given, the other NULL. out (B, V) in l's type (may be l itself): x, rounded once. tokens (B)
 * int64: the word of the largest x, the lowest among equals, NaN above every number (torch.argmax's rule); -1 where every
 * x is -inf.
 * V at most 2^26, B at most 65535, L at most 2^24, M at most 2^20, L and M of 31 bits together, B V below 2^40. Only tokens
 * take a workspace, of rows past 32761 words. */
int64_t pragnosia_rules_workspace_bytes(int64_t B, int64_t V);
int pragnosia_rules(const void* logits, int bf16, const int64_t* history, int64_t history_stride, int64_t L,
                    const int64_t* lengths, const int64_t* prompt, const float* repetition, float repetition_value,
                    const float* presence, float presence_value, const float* frequency, float frequency_value,
                    const int64_t* bias_ids, const float* bias_values, int64_t M, int64_t bias_stride,
                    const uint32_t* mask, int64_t S, const int64_t* state, void* out, int64_t* tokens, void* workspace,
                    int64_t workspace_bytes, int64_t B, int64_t V, void* stream);

/* What follows a chosen token in a step of generation, for rows b with tokens[b] in [0, V) (others, -1 among them, leave
 * their history and state as they are): with history (B rows of cap entries, history_stride apart) and lengths (B), the
 * token becomes entry lengths[b], which counts one more, while it is below cap; with next (S, V) int32 and state (B), a
 * state s in [0, S) becomes next[s][token]. Each pair may be NULL.
 *
 * With emb (V, d), fp32, for all rows the end of a decode step (pragnosia_decode_tail's, after its argmax):
 * out[c][b] = tok[b] = tokens[b] with c = *ctr_in (out has n_rows rows of B; none past them), p = (*pos_in + 1) mod ctx,
 * h[b] = emb[token] + pemb[p] (fp32; a token outside the table adds nothing), *ctr_out = c + 1, *pos_out = p,
 * p0s[0 .. L - 1] = 1. The two counters are read from one slot and written to another; tok is not tokens. */
int pragnosia_rules_tail(const int64_t* tokens, int64_t* history, int64_t history_stride, int64_t cap, int64_t* lengths,
                         const int32_t* next, int64_t S, int64_t* state, const float* emb, const float* pemb, int64_t d,
                         int64_t ctx, const int64_t* ctr_in, int64_t* ctr_out, const int64_t* pos_in, int64_t* pos_out,
                         int64_t* out, int64_t n_rows, int64_t* tok, float* h, float* p0s, int64_t L, int64_t B, int64_t V,
                         void* stream);

#ifdef __cplusplus
}
#endif
#endif /* PRAGNOSIA_GEN_H */
