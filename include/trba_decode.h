/* Beam-search operators of libtrba_b200 (no counterpart in the reference,
 * whose decoder is greedy: src/attn.rs:368-447).  One decoding step is
 *
 *     logits of every (line, beam)      (the caller's decoder)
 *     trba_beam_select                  which (beam, token) pairs survive
 *     trba_beam_reorder                 the states of the beams follow them
 *
 * and trba_beam_sequences turns the tokens and parents of all steps into
 * token sequences.  trba_model_infer_beam (trba_qat.h) runs them for the
 * recogniser's own decoder.
 *
 * All pointers are device pointers of the current device.  The functions
 * only launch kernels on `stream`, without allocation or synchronisation, so
 * they may be captured into CUDA graphs and, each with a workspace of its
 * own, run on several streams at once.  They return 0, -1 for a bad argument
 * (then nothing has run) or a CUDA error code; errors also follow the library
 * policy (trba_last_error / abort on error).  Zero lines is an empty call and
 * returns 0.  Outputs must not overlap the inputs or each other, except where
 * the same buffer is said to do. */
#ifndef TRBA_DECODE_H
#define TRBA_DECODE_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of logits and activations. */
#define TRBA_F32 0
#define TRBA_BF16 1
#define TRBA_F16 2

#define TRBA_MAX_BEAMS 32

/* One selection step.  For every line the `beams` best pairs (b, v) by
 *
 *     scores[b] + logits[b, v] - log(sum_u exp(logits[b, u]))
 *
 * over all its beams b and tokens v, best first; ties go to the lowest
 * (b, v).  logits: [lines * beams, vocab] of `dtype`, row stride ld >= vocab
 * elements; scores: f32 [lines, beams], the beams' log probabilities so far
 * (-inf: the beam is dead, for instance all but the first before the first
 * step); finished: one byte a beam, or NULL for none.  A finished beam's only
 * continuation is `eos`, at an unchanged score; its logits are not read, nor
 * are a dead beam's.
 *
 * Outputs, [lines, beams] each: the new scores; the tokens; the parents
 * (beam index in the line that each slot continues); finished (1 when the
 * token is eos or the parent was finished).  A line with fewer than `beams`
 * continuations above -inf fills the remaining slots with score -inf, token
 * eos (0 when eos < 0), parent = the slot itself, finished 1 (0 when eos <
 * 0).  out_scores / out_finished may be exactly the buffers scores / finished.
 *
 * A logit of NaN counts as -inf (its token is never chosen and adds nothing
 * to the sum).  Where a row holds +inf, its +inf tokens share the
 * probability evenly.  A NaN score counts as a dead beam.  Scores are
 * formed and compared in f64 and rounded to f32 at the end (the exponentials
 * are f32, and so are their sums within a batch of 16 (f32) or 32 (16-bit) of
 * a thread's elements; beyond that f64).
 *
 * beams 1 .. 32, vocab 1 .. 2^30, beams * vocab < 2^31, lines * beams <
 * 2^24, eos in [0, vocab) or -1 for "no end token" (then finished must be
 * NULL).  Long rows need a workspace of trba_beam_select_workspace(...) bytes,
 * aligned to 16 (0 bytes: none, NULL will do), which calls that may overlap
 * must not share; what it holds before and after does not matter. */
long long trba_beam_select_workspace(int dtype, int lines, int beams, int vocab);
int trba_beam_select(const void *logits, int dtype, long long ld, const float *scores, const uint8_t *finished,
                     int lines, int beams, int vocab, int eos, float *out_scores, int32_t *out_tokens,
                     int32_t *out_parents, uint8_t *out_finished, void *workspace, long long workspace_bytes,
                     void *stream);

/* A state tensor whose rows follow the beams, as a strided view
 * [outer][lines * beams][mid][bytes]; strides and sizes in bytes.  A plain
 * [lines * beams, width] matrix has outer = mid = 1 and bytes = width *
 * element size; stacked layers use outer, the filled part of a cache with
 * room for more positions uses mid. */
typedef struct {
    const void *src;
    void *dst;
    long long bytes;
    long long src_row, dst_row;
    long long mid, src_mid, dst_mid;
    long long outer, src_outer, dst_outer;
} trba_beam_state;

/* dst row (l, k) = src row (l, parents[l, k]) for every state, for each of
 * its outer and mid parts, in one launch for up to 16 states.  `states` is a
 * host array, read before the call returns.  No dst may overlap a src or
 * another dst: use two buffers in turn (they may be halves of wider rows).  A
 * state's rows may have up to 2^31 - 2^20 parts of at most 1024 bytes.  A parent outside [0, beams) leaves its dst row as
 * it was. */
int trba_beam_reorder(const trba_beam_state *states, int n_states, const int32_t *parents, int lines, int beams,
                      void *stream);

/* The token sequences that end in the slots of the last step: tokens and
 * parents are [steps, lines, beams] as trba_beam_select wrote them step by
 * step; slot k after step t continues slot parents[t, l, k] after step t - 1
 * (parents[0] is not used).  sequences: [lines, beams, steps], each path's
 * tokens before its first eos, then pad; lengths: [lines, beams], their
 * count.  A path that meets a parent outside [0, beams) ends there: its
 * earlier tokens are unknown, the whole sequence is pad and its length -1. */
int trba_beam_sequences(const int32_t *tokens, const int32_t *parents, int steps, int lines, int beams, int eos,
                        int pad, int32_t *sequences, int32_t *lengths, void *stream);

#ifdef __cplusplus
}
#endif
#endif
