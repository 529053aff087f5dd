// Launch records of the operators over rows of logits: processed logits,
// log-probabilities and distillation (jf_process.hip, jf_score.hip,
// jf_distill.hip), and what their host side (jf_scorer.cpp) fills in.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "jf_host.h"

namespace jf {

// A block's 256 threads take a chunk of a row, a few vectors of 16 bytes each.
constexpr uint32_t chunk_tokens(uint32_t dtype, uint32_t vectors) {
  return vectors * 256 * (dtype == 0 ? 4 : 8);
}
// The tokens whose maximum the pass keeps (a power of two that divides a chunk).
constexpr uint32_t kScoreGroup = 64;
constexpr uint32_t kTopLogprobs = 128;    // alternatives a row at most
constexpr uint32_t kTeacherTokens = 256;  // a teacher's list at most: one a thread
// Rows of one launch with alternatives: bounds the groups' scratch.
constexpr uint32_t kTopRows = 512;

// One row's edits, as the host derives them from its policy.
struct ProcessRow {
  uint32_t flags;        // ProcessFlags
  uint32_t penalty_row;  // kNoRow: no penalties
  uint32_t bias_row;     // kNoRow: no biases
  uint32_t mask_row;
  uint32_t extra_count;
  uint32_t extra_offset;
  float repetition;
  float repetition_inverse;
  float presence;
  float frequency;
  uint32_t reserved[2];
};
static_assert(sizeof(ProcessRow) == 48, "process rows are 48 bytes");
enum ProcessFlags : uint32_t { kProcessMasked = 1u, kProcessStops = 2u };
constexpr uint32_t kNoRow = 0xffffffffu;

struct ProcessLaunch {
  const void *logits;
  void *out;
  uint64_t stride, out_stride;
  const ProcessRow *rows;
  uint32_t row_count, vocabulary;
  uint32_t chunks;  // of a row: the launch's own
  uint32_t in_place;
  uint32_t any_masked, all_masked;
  const uint32_t *masks;
  uint64_t mask_stride;
  uint32_t stop0, stop1;
  const PenaltyEntry *pen_entries;
  const uint32_t *pen_offsets;
  uint32_t pen_max_entries;
  const PenaltyEntry *bias_entries;  // {token, bits of the bias}
  const uint32_t *bias_offsets;
  uint32_t bias_max_entries;
  uint32_t buckets;
  const uint32_t *extra;
};

struct ScoreLaunch {
  const void *logits;
  uint64_t stride;
  uint32_t row_count, vocabulary;
  uint32_t vectors;         // a thread: 2 or 4
  uint32_t segments;        // blocks a row, one a chunk
  uint32_t groups;          // groups a row, padded to whole chunks
  const float *temperatures;  // device, or NULL: `temperature` for every row
  float temperature;
  float2 *partials;  // [rows][segments]: maximum, sum of exponentials
  uint32_t *aheads;  // [rows][segments]: tokens ahead of the row's first one
  float *maxima;     // [rows][groups]
  // Log-probabilities.
  const uint32_t *tokens;
  uint32_t token_count;
  uint64_t token_stride;
  float *out_lse;
  float *out_logprobs;
  uint32_t *out_ranks;
  uint32_t top;
  uint32_t *out_top_ids;
  float *out_top_logprobs;
  // Distillation.
  const uint32_t *teacher_ids;
  const float *teacher_values;
  uint64_t teacher_stride;
  uint32_t teacher_count;
  uint32_t normalize;
  float *out_loss;
  float *saved;  // [rows][2 + teacher_count]
};

struct DistillGradLaunch {
  const void *logits;
  uint64_t stride;
  void *grad;
  uint64_t grad_stride;
  uint32_t row_count, vocabulary;
  uint32_t vectors;  // a thread: 2 or 4
  uint32_t chunks;   // blocks a row: the launch's own
  float temperature;
  const uint32_t *teacher_ids;
  uint64_t teacher_stride;
  uint32_t teacher_count;
  const float *saved;
  const float *grad_loss;
  uint64_t grad_loss_stride;
};

// dtypes as JF_DTYPE_*. Each returns a hipError_t. The rows of one launch are
// bounded so that its grid stays below 2^32 threads.
int launch_process(const ProcessLaunch &a, uint32_t dtype, uint32_t out_dtype, void *stream);
// The pass over the rows, and what finishes it.
int launch_score(const ScoreLaunch &a, uint32_t dtype, void *stream);
int launch_logprobs(const ScoreLaunch &a, uint32_t dtype, void *stream);
int launch_distill_loss(const ScoreLaunch &a, uint32_t dtype, void *stream);
int launch_distill_grad(const DistillGradLaunch &a, uint32_t dtype, void *stream);
// Losses and gradients of the same rows at once.
int launch_distill_step(const ScoreLaunch &a, const DistillGradLaunch &g, uint32_t dtype,
                        void *stream);

}  // namespace jf
