// sample_args.h -- argument blocks of the sampling kernels (sample.hip), shared
// with the host launcher (passed by value).
#pragma once
#include <stdint.h>

// Elements of a row that one workgroup of 256 threads takes: 16 a thread, or 4
// where that leaves CUs idle.
#define SAMPLE_MANY 16u
#define SAMPLE_FEW 4u

struct ProbsArgs {
  const float* logits;
  float* probs;
  float* part;  // [row][chunk] {max, sum}
  uint64_t stride;
  uint32_t vocab, chunks;
  float inv_cap, mul;  // 1 / soft-cap (0: none); log2(e) / temperature, times the soft-cap
};

struct VerifyArgs {
  const float *target, *draft;  // [seq][max_draft + 1][vocab], [seq][max_draft][vocab] or null
  const uint32_t *tokens, *n_draft;
  const float *u, *pick;
  uint32_t *out, *accepted;
  double* part;  // [seq][chunk] {weights left, target}
  uint32_t max_draft, vocab, chunks;
};
