/*
 * Decoding operators next to the semiring products of cuasr_b200.h, as C entry points: what a program that decodes
 * sequences step by step does with a product of few rows.
 *
 *   cuasr_b200_q4_product      plus-times product of a few rows with a weight operand held in 4 bits
 *   cuasr_b200_beam_step       max-plus step with back-pointers that keeps the `keep` best continuations of a search
 *                              (cuasr_b200_srgemm_path keeps the one best of every element)
 *   cuasr_b200_reorder_states  state tensors follow those back-pointers
 *
 * The reference has no counterpart.  The conventions are those of cuasr_b200.h: DEVICE pointers owned by the caller,
 * nothing is allocated, freed or synchronised with the host, every launch is asynchronous on `stream`, and return values
 * are cuasr_status_t.  Every call can be captured into a CUDA graph; a replay reads and writes the buffers (and the
 * workspace) of the captured call, so replays that share a workspace or an output must not overlap.
 *
 * `device`: 0 = the current device, d + 1 = device d, made current for the launch and set back before the call
 * returns.  All buffers and the stream belong to that device.
 */
#ifndef CUASR_B200_DECODE_H
#define CUASR_B200_DECODE_H

#include "cuasr_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Y[r, j] = sum over k of X[r, k] * w[j, k],  w[j, k] = scale[j, k / group] * (q[j, k] - zero[j, k / group]).
 *
 * q[j, k] is the low (k even) or high (k odd) half of the byte W[j * ldw + k / 2]; zero is the low half of
 * zeros[j * ld_zeros + k / group], or 8 where `zeros` is NULL.  With x as it is (32-bit values too) and q - zero as the whole
 * number it is, the products are summed in 32 bits by groups, of longer ones by 128, the scale is applied, these are summed in 32 bits, and Y is
 * rounded once.  Weights at their zero point add exactly nothing; infinities and NaN among the values reach the outputs that the formula
 * gives them to.  Of F32 and BF16 values, bits below 2^-133 and products below 2^-120 may count as zero;
 * results below 2^-117 may lose bits.
 * Y must not share bytes with an operand.  The same call gives the same bits every time on one kind of device. */
typedef struct cuasr_b200_q4_args {
  int32_t dtype_x;      /* CUASR_F32, CUASR_F16 or CUASR_BF16 */
  int32_t dtype_y;      /* the same choice */
  int32_t dtype_scale;  /* the same choice */
  int32_t group;        /* values along k that share a scale: a multiple of 32; at least k for one scale per row */
  int32_t m, n, k;      /* X is m x k, W n x k, Y m x n; above 0, n and k at most 2^31 - 2^17, m at most 2 million (655350 rows of
                           32 bits).  Made for m up to 32 or so: every 32 rows of X (10 of 32 bits) read the weights anew */
  int32_t device;
  const void *X;      int64_t ldx;        /* row-major; leading dimensions in elements, at least the row */
  const uint8_t *W;   int64_t ldw;        /* bytes per row, at least (k + 1) / 2; fastest where W and ldw are multiples of 16.  Bytes
                                             between the rows may be read */
  const void *scales; int64_t ld_scales;  /* n x ceil(k / group) */
  const uint8_t *zeros; int64_t ld_zeros; /* n x ceil(k / group), or NULL */
  void *Y;            int64_t ldy;
  void *stream;                           /* cudaStream_t */
} cuasr_b200_q4_args_t;

CUASR_B200_API int cuasr_b200_q4_product_can_implement(const cuasr_b200_q4_args_t *args);
CUASR_B200_API int cuasr_b200_q4_product(const cuasr_b200_q4_args_t *args);

/* One step of `batch` independent beam searches.  A search holds `beams` prefixes with scores; the value of continuing
 * prefix b with token v is
 *
 *   score[b] + logit[b, v]                              (normalise == 0: the inputs are log-probabilities)
 *   score[b] - log(sum over u of exp(logit[b, u])) + logit[b, v]        (normalise != 0)
 *
 * in 64-bit arithmetic, except for the exponentials (32 bits, summed in 32 bits up to 32 at a time, then in 64).
 * A prefix whose finished byte is not 0 has one continuation: `end_token`, with the prefix's own score.  Values of
 * -infinity and NaN are no continuations (a NaN or +infinity among the logits of a prefix thus ends it where they are
 * normalised).
 * The `keep` best values go to out_scores, rounded to 32 bits, with the prefix each continues (parents) and its token:
 * best first, equal values in the order of the prefix, then of the logit (larger first), then of the token.
 * Places left over get -infinity, -1 and -1. */
typedef struct cuasr_b200_beam_args {
  int32_t dtype;                       /* of the logits: CUASR_F32, CUASR_F16 or CUASR_BF16 */
  int32_t normalise;
  int32_t batch, beams, vocab, keep;   /* all above 0; beams at most 1024, keep at most CUASR_B200_BEAM_MAX_KEEP, batch * beams at
                                          most 2^24 */
  int32_t end_token;
  int32_t device;
  const void *logits;                  /* element (s, b, v) at s * batch_stride + b * beam_stride + v */
  int64_t batch_stride, beam_stride;   /* in elements, not negative */
  const float *scores; int64_t ld_scores;            /* batch x beams */
  const uint8_t *finished; int64_t ld_finished;      /* batch x beams, or NULL */
  float *out_scores;   int64_t ld_out_scores;        /* batch x keep; may be `scores` itself, with the same leading
                                                        dimension */
  int32_t *parents;    int64_t ld_parents;           /* batch x keep */
  int32_t *tokens;     int64_t ld_tokens;            /* batch x keep; outputs share no bytes with anything else of the call */
  void *workspace;     size_t workspace_bytes;       /* cuasr_b200_beam_step_workspace_size bytes, 16-byte aligned; any
                                                        content, overwritten */
  void *stream;                                      /* cudaStream_t */
} cuasr_b200_beam_args_t;

#define CUASR_B200_BEAM_MAX_KEEP 64

CUASR_B200_API int cuasr_b200_beam_step_can_implement(const cuasr_b200_beam_args_t *args);
/* Bytes of workspace for these sizes, the same on every device; 0 for invalid arguments (pointers are not looked at). */
CUASR_B200_API size_t cuasr_b200_beam_step_workspace_size(const cuasr_b200_beam_args_t *args);
CUASR_B200_API int cuasr_b200_beam_step(const cuasr_b200_beam_args_t *args);

/* A state tensor of batch x beams x segments x positions x bytes, the last contiguous; all strides in bytes and not
 * negative.  Keys of an attention cache, for instance: segments = heads, positions = tokens, bytes = one head's vector. */
typedef struct cuasr_b200_state {
  const void *src;
  void *dst;
  int64_t src_batch, src_beam, src_segment, src_position;   /* strides */
  int64_t dst_batch, dst_beam, dst_segment, dst_position;
  int64_t bytes;
  int32_t segments, positions;
  int32_t ragged;      /* not 0: only the first lengths[s] positions of search s are in use */
  int32_t reserved;
} cuasr_b200_state_t;

/* dst[s, j] = src[s, parents[s, j]] for the `keep` rows j of every search s and every state: the prefixes' states
 * follow cuasr_b200_beam_step's back-pointers.  Positions behind lengths[s] of a ragged state and rows whose parent is
 * negative (places left over) stay as they were.  A parent of `beams` or more is not followed, and device status 4 is
 * recorded (cuasr_b200_device_status); lengths outside [0, positions] count as the nearer end.
 * In place: dst == src with equal strides, rows that lie apart, keep <= beams, and keep <= CUASR_B200_REORDER_MAX_IN_PLACE.  Otherwise the
 * address ranges of src and dst must not meet.  No state's dst may share bytes with another state of the call (only equal
 * addresses are looked for), and the elements of a dst must lie apart. */
typedef struct cuasr_b200_reorder_args {
  int32_t batch, beams, keep;          /* above 0; keep at most 1024 */
  int32_t n_states;                    /* 0 to CUASR_B200_REORDER_MAX_STATES; 0 does nothing */
  const int32_t *parents; int64_t ld_parents;   /* batch x keep */
  const int32_t *lengths;              /* batch, or NULL where no state is ragged */
  const cuasr_b200_state_t *states;    /* in host memory, read during the call */
  int32_t device;
  int32_t reserved;
  void *stream;                        /* cudaStream_t */
} cuasr_b200_reorder_args_t;

#define CUASR_B200_REORDER_MAX_IN_PLACE 32
#define CUASR_B200_REORDER_MAX_STATES 256

CUASR_B200_API int cuasr_b200_reorder_states_can_implement(const cuasr_b200_reorder_args_t *args);
CUASR_B200_API int cuasr_b200_reorder_states(const cuasr_b200_reorder_args_t *args);

#ifdef __cplusplus
}
#endif
#endif /* CUASR_B200_DECODE_H */
