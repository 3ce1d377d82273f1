// C interface of beam search's selection (beam.cu).
//
// logits: rows [groups * beams] of `vocab` numbers, ld elements apart (type 0 bf16, 1 f16, 2 fp32); scores: fp32 [groups, beams], the sums of the
// beams' logarithmic probabilities so far.  A continuation of row r by token t has
//     total = scores[r] + x[r, t] - log(sum over u of exp(x[r, u])),
// with NaN logits and scores taken as minus infinity and plus infinity as the largest fp32 number; a row with ended[r] != 0 has one continuation,
// end_token, with total = scores[r].  For every group the `count` largest totals in descending order, of equal ones the lowest row and then the
// lowest token first: totals (rounded once), rows (in 0 .. groups * beams - 1) and tokens, [groups, count] each.
// scratch: rb_beam_select_scratch_bytes bytes, 16-byte aligned.
#pragma once
#ifdef __cplusplus
extern "C" {
#endif
typedef struct RbBeamSelectArgs {
  const void* logits;
  const float* scores;
  const unsigned char* ended;    // [groups * beams] or NULL
  float* out_scores;
  long long* out_rows;
  long long* out_tokens;
  void* scratch;
  long long ld;
  int groups, beams, vocab, count, type, end_token;
} RbBeamSelectArgs;
long long rb_beam_select_scratch_bytes(int groups, int beams, int vocab, int count, int type);
int rb_beam_select(const RbBeamSelectArgs* args, void* stream);
#ifdef __cplusplus
}
#endif
