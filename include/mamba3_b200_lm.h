/*
 * mamba3_b200_lm.h -- C ABI of the language-model operators around the
 * Mamba-3 decode step: projections with 4-bit weights, and what a token step
 * does with its logits.
 *
 * None of them has a counterpart in the reference, whose decode ends at the
 * layer output.  The conventions of mamba3_b200.h hold: device pointers on
 * the CURRENT device, sizes and strides in ELEMENTS, nothing allocated or
 * synchronised, work enqueued on `stream`, arguments checked on the host
 * before any launch, status codes M3_*, capturable in a CUDA graph after one
 * eager call on the device.  No entry point keeps a workspace, so calls may
 * overlap on several streams.
 */
#ifndef MAMBA3_B200_LM_H
#define MAMBA3_B200_LM_H

#include "mamba3_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Rows and columns of a storage block of a 4-bit weight. */
#define M3_W4_ROWS 16
#define M3_W4_TILE 128

/* y = x W^T with W[n, k] = (code[n, k] - zero[n, k / group]) * scale[n, k / group],
 * code 0..15 and zero 8 where zeros is NULL.
 *   x       (M, K)  x_dtype (f32 / bf16), row stride ldx >= 0, unit column stride
 *   codes   (ceil(N / 16), ceil(K / 128), 16, 16) 32-bit words, contiguous,
 *           16-byte aligned: blocks of 16 rows by 128 columns.  Word 4 t + j
 *           of a block's row holds its columns 32 j + 8 t .. + 7: column + 0,
 *           2, 4, 6 in bits 0, 4, 8, 12, column + 1, 3, 5, 7 in bits 16, 20,
 *           24, 28.  Codes past column K are multiplied with 0 only; those
 *           past row N - 1 reach no output.
 *   scales  (N, ceil(K / group)) s_dtype (f32 / bf16), row stride scale_stride
 *   zeros   (N, ceil(K / group)) bytes 0..15, row stride zero_stride, or NULL
 *   y       (M, N)  y_dtype (f32 / bf16), row stride ldy >= N, unit column stride
 *   group   32, 64 or 128
 * Codes, scales and zeros take less than 4 GB each (M3_ERR_SHAPE).
 * Products are exact (a bf16 x times a small integer; an fp32 x is taken as
 * three bf16 terms, which are all of it from 2^-110 on, and to less than
 * 2^-133 below), sums are fp32, scaled once per group and added in a fixed
 * order: the same call gives the same bits.  The sum of a group before its
 * scale has to stay within fp32's range. */
typedef struct m3_w4_args {
  int32_t M, N, K, group;
  const void *x;      int64_t ldx;          int32_t x_dtype;
  const int32_t *codes;
  const void *scales; int64_t scale_stride; int32_t s_dtype;
  const uint8_t *zeros; int64_t zero_stride;
  void *y;            int64_t ldy;          int32_t y_dtype;
} m3_w4_args;

int m3_linear_w4(const m3_w4_args *args, m3_stream_t stream);

/* Adjustments of a (B, V) matrix of logits, in this order, in fp32, each
 * operation rounded once (no fused multiply-add):
 *   seen in tokens[0 : length]               z = z > 0 ? z / repetition : z * repetition
 *   c times in tokens[prompt_length : length]   z = z - frequency * c
 *   c > 0                                    z = z - presence
 *   always                                   z = z + bias
 *   bit i % 32 of word i / 32 of `allowed` is 0   z = -infinity
 *
 *   logits   (B, V) dtype (f32 / bf16), row stride ld, unit column stride
 *   tokens   (B, T) int32 or int64 (tokens_i64), row stride tokens_stride,
 *            unit column stride; ids outside [0, V) are skipped.  NULL: no
 *            history.
 *   lengths, prompt_lengths   (B,) int32 or int64 (lengths_i64,
 *            prompt_i64), clamped to [0, T]; NULL: T, and 0
 *   repetition, presence, frequency   (B,) f32, or NULL for the scalar *_value
 *   bias     f32, row stride bias_stride (0: one row for all), or NULL
 *   allowed  32-bit words, row stride allowed_stride (0: one row for all),
 *            or NULL: every token
 * m3_process_logits only:
 *   out      (B, V) out_dtype, row stride out_ld; may be `logits` itself
 * m3_next_tokens only (see there):
 *   temperature (B,) f32 or NULL for temperature_value; sample: draw rows
 *            whose temperature is above 0; seeds, positions (B,) int64
 *            (positions may be NULL: 0); ids (B,) int64, logprobs (B,) f32 */
typedef struct m3_logits_args {
  int32_t B, V, T, dtype;
  const void *logits;         int64_t ld;
  const void *tokens;         int64_t tokens_stride;
  const void *lengths, *prompt_lengths;
  int32_t tokens_i64, lengths_i64, prompt_i64, sample;
  const float *repetition, *presence, *frequency;
  float repetition_value, presence_value, frequency_value, temperature_value;
  const float *bias;          int64_t bias_stride;
  const int32_t *allowed;     int64_t allowed_stride;
  void *out;                  int64_t out_ld;
  int32_t out_dtype, reserved;
  const float *temperature;
  const int64_t *seeds, *positions;
  int64_t *ids;
  float *logprobs;
} m3_logits_args;

/* The adjusted logits, rounded once to out_dtype. */
int m3_process_logits(const m3_logits_args *args, m3_stream_t stream);

/* The next token of every row, from the adjusted logits z, which are not
 * stored.
 *   greedy row (sample 0, or a temperature not above 0): the largest z, the
 *     lowest index among equals; logprob = z - log sum exp z
 *   drawn row: the largest z / temperature + noise, noise = -log(-log u);
 *     logprob = z / temperature - log sum exp (z / temperature).  u of token i
 *     is 1 - (w + 1/2) 2^-32, w word i % 4 of block i / 4 of the 4 x 32 bit
 *     counter-based generator of Salmon et al. ("Parallel random numbers: as
 *     easy as 1, 2, 3", SC 2011) with 7 rounds, key = the row's seed (low
 *     word first), counter = (i / 4, position low, position high, 0).  The
 *     comparison is of differences in 64 bits, so that logits of any size
 *     leave the noise its bits, and equal inputs give equal tokens.
 * A NaN that is not masked is taken as the largest (the first one; logprob
 * NaN).  A row with nothing above -infinity gives token 0 and logprob
 * -infinity. */
int m3_next_tokens(const m3_logits_args *args, m3_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* MAMBA3_B200_LM_H */
