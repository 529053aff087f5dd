// Host side of the operators over rows of logits (include/jf_sampler.h,
// "scoring"): argument checks, the bias table, the scorer's scratch and row
// records, and the launches of jf_process.hip, jf_score.hip and
// jf_distill.hip.
#include "jf_scorer.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstring>
#include <new>
#include <string>
#include <utility>
#include <vector>

#include "jf_objects.h"
#include "jf_sampler.h"

namespace {

using namespace jf::host;

constexpr uint32_t kMaxVocabulary = 524288;
constexpr uint32_t kMaxRows = 1u << 22;
// Tokens of one launch at most: the threads of its grid stay below 2^32.
constexpr uint64_t kMaxTokens = 1ull << 33;

constexpr uint32_t kLeastChunk = jf::chunk_tokens(JF_DTYPE_F32, 2);
constexpr uint32_t kMostChunk = jf::chunk_tokens(JF_DTYPE_BF16, 4);
uint32_t blocks_of(uint32_t vocabulary, uint32_t chunk) { return (vocabulary + chunk - 1) / chunk; }
// Rows of one launch at most.
uint32_t launch_rows(uint32_t vocabulary) {
  return (uint32_t)(kMaxTokens / ((uint64_t)blocks_of(vocabulary, kMostChunk) * kMostChunk));
}
size_t element_size(uint32_t dtype) { return dtype == JF_DTYPE_F32 ? 4 : 2; }

// The rows from which a training step takes them whole, a block each, in one
// launch. A short row is done before three launches would be (72,256 tokens, one
// bf16 row 11.1 us against 11.5, 64 rows 12.0 against 13.1, 512 rows 27 against 41).
// A long one keeps its block busy longer than the rows' chunks spread over the GPU
// take (100,003 f32, one row 14.6 against 11.6; 151,936 bf16, 64 rows 21.5 against
// 15.8), unless rows keep nearly half of the CUs busy (96 rows 22.1 against 20.0,
// 128 rows 23.1 against 24.5) or, of the longest, most (248,320 f32, 128 rows 65.2
// against 60.7, 192 rows 105.6 against 92.9; bf16, 128 rows 34.9 against 35.6).
uint32_t whole_rows(uint32_t vocabulary, uint32_t dtype) {
  const uint32_t row_bytes = vocabulary * (uint32_t)element_size(dtype);
  return vocabulary <= 72u << 10 ? 1 : std::max(112u, row_bytes / 5120);
}
// Those of steps by chunks at most: the scorer holds what their forward pass saves
// where the caller does not.
uint32_t chunked_rows(uint32_t vocabulary) { return whole_rows(vocabulary, JF_DTYPE_F32) - 1; }

const void *rows_at(const void *p, uint64_t row, uint64_t stride, uint32_t dtype) {
  return (const uint8_t *)p + row * stride * element_size(dtype);
}
template <class T>
T *at(T *p, uint64_t offset) {
  return p ? p + offset : nullptr;
}

}  // namespace

struct jf_bias_table {
  uint32_t vocabulary = 0;
  uint32_t rows = 0;
  uint32_t max_entries = 0;
  uint32_t buckets = 0;
  int device = 0;
  jf::PenaltyEntry *entries = nullptr;  // [rows][max_entries] {token, bits of the bias}
  uint32_t *offsets = nullptr;          // [rows][buckets + 1]
  // Rows that a failed upload may have left half changed: refused until set.
  std::vector<uint8_t> stale;
  StagingRing staging;
};

struct jf_scorer {
  uint32_t vocabulary = 0;
  uint32_t max_rows = 0;
  int device = 0;
  jf::ProcessRow *rows = nullptr;  // [max_rows]
  float2 *partials = nullptr;      // a chunk each, row by row, of one launch
  uint32_t *aheads = nullptr;      // likewise
  float *maxima = nullptr;         // those of min(max_rows, kTopRows) rows' chunks
  float *saved = nullptr;          // [min(max_rows, chunked_rows)][2 + kTeacherTokens]
  uint64_t workspace_bytes = 0;
  std::vector<jf::ProcessRow> last_rows;  // what the device's rows hold
  std::vector<jf::ProcessRow> host_rows;  // the call's rows, reused across calls
  // A captured call's masks, tables and launches go with its records, which its
  // replays read: they stay as they are, and other records go elsewhere.
  bool rows_captured = false;                    // `rows` are such
  std::vector<jf::ProcessRow *> captured_rows;  // earlier ones, [max_rows] each
  StagingRing staging;
};

extern "C" {

// ---- biases ------------------------------------------------------------------

int jf_bias_table_destroy(jf_bias_table *t) {
  if (!t) return JF_OK;
  t->staging.release();
  (void)hipFree(t->entries);
  (void)hipFree(t->offsets);
  delete t;
  return JF_OK;
}

int jf_bias_table_create(uint32_t vocabulary, uint32_t rows, uint32_t max_entries,
                         jf_bias_table **out) {
  if (!out) return fail(JF_ERR_INVALID_ARGUMENT, "output pointer is null");
  *out = nullptr;
  if (!vocabulary || !rows || !max_entries || max_entries > 0x7fffffffu)
    return fail(JF_ERR_INVALID_ARGUMENT, "invalid bias table geometry");
  if (vocabulary > kMaxVocabulary)
    return fail(JF_ERR_INVALID_ARGUMENT, "vocabulary exceeds 524288 tokens");
  jf_bias_table *t = new (std::nothrow) jf_bias_table;
  if (!t) return fail(JF_ERR_NO_MEMORY, "bias table allocation failed");
  t->vocabulary = vocabulary;
  t->rows = rows;
  t->max_entries = max_entries;
  t->buckets = (vocabulary + jf::kPenaltyBucket - 1) / jf::kPenaltyBucket;
  int rc = JF_OK;
  try {
    t->stale.assign(rows, 0);
  } catch (const std::bad_alloc &) {
    rc = fail(JF_ERR_NO_MEMORY, "bias table allocation failed");
  }
  hipError_t e = hipGetDevice(&t->device);
  if (rc == JF_OK && e != hipSuccess) rc = hip_fail(e, "hipGetDevice");
  const size_t offsets = (size_t)rows * (t->buckets + 1);
  if (rc == JF_OK) rc = device_alloc(&t->entries, (size_t)rows * max_entries, "bias entries");
  if (rc == JF_OK) rc = device_alloc(&t->offsets, offsets, "bias offsets");
  if (rc == JF_OK) {
    e = hipMemset(t->offsets, 0, offsets * sizeof(uint32_t));
    if (e == hipSuccess) e = hipDeviceSynchronize();
    if (e != hipSuccess) rc = hip_fail(e, "bias table init");
  }
  if (rc != JF_OK) {
    jf_bias_table_destroy(t);
    return rc;
  }
  *out = t;
  return JF_OK;
}

int jf_bias_table_set(jf_bias_table *t, uint32_t row, const uint32_t *tokens, const float *biases,
                      uint64_t count, void *stream) {
  if (!t) return fail(JF_ERR_INVALID_ARGUMENT, "bias table is null");
  if (row >= t->rows) return fail(JF_ERR_INVALID_ARGUMENT, "bias row is outside the table");
  if (count && (!tokens || !biases)) return fail(JF_ERR_INVALID_ARGUMENT, "null buffer");
  if (count > t->max_entries)
    return fail(JF_ERR_INVALID_ARGUMENT, "biases exceed the table row");
  int rc = check_device(t->device);
  if (rc != JF_OK) return rc;
  // A replay would upload what the pinned buffers hold by then.
  bool capturing;
  rc = is_capturing((hipStream_t)stream, capturing);
  if (rc != JF_OK) return rc;
  if (capturing) return fail(JF_ERR_LOGIC, "a bias row's upload cannot be captured");
  try {
    std::vector<std::pair<uint32_t, float>> sorted(count);
    for (uint64_t i = 0; i < count; ++i) {
      if (tokens[i] >= t->vocabulary)
        return fail(JF_ERR_INVALID_ARGUMENT, "biased token is outside the vocabulary");
      if (!(biases[i] <= FLT_MAX))
        return fail(JF_ERR_INVALID_ARGUMENT, "a bias is finite or -infinity");
      sorted[i] = {tokens[i], biases[i]};
    }
    std::sort(sorted.begin(), sorted.end(),
              [](const auto &x, const auto &y) { return x.first < y.first; });
    for (uint64_t i = 1; i < count; ++i)
      if (sorted[i].first == sorted[i - 1].first)
        return fail(JF_ERR_INVALID_ARGUMENT, "a token is biased twice in one row");
    std::vector<jf::PenaltyEntry> entries(count);
    std::vector<uint32_t> offsets(t->buckets + 1, 0u);
    for (uint64_t i = 0; i < count; ++i) {
      uint32_t bits;
      std::memcpy(&bits, &sorted[i].second, sizeof(bits));
      entries[i] = {sorted[i].first, bits};
      ++offsets[sorted[i].first / jf::kPenaltyBucket + 1];
    }
    for (uint32_t b = 0; b < t->buckets; ++b) offsets[b + 1] += offsets[b];
    const hipStream_t st = (hipStream_t)stream;
    t->stale[row] = 1;
    rc = t->staging.upload(t->entries + (size_t)row * t->max_entries, entries.data(),
                           count * sizeof(jf::PenaltyEntry), st);
    if (rc == JF_OK)
      rc = t->staging.upload(t->offsets + (size_t)row * (t->buckets + 1), offsets.data(),
                             offsets.size() * sizeof(uint32_t), st);
    if (rc == JF_OK) t->stale[row] = 0;
  } catch (const std::bad_alloc &) {
    return fail(JF_ERR_NO_MEMORY, "bias row allocation failed");
  }
  return rc;
}

// ---- scorer ------------------------------------------------------------------

int jf_scorer_destroy(jf_scorer *s) {
  if (!s) return JF_OK;
  s->staging.release();
  (void)hipFree(s->rows);
  for (jf::ProcessRow *rows : s->captured_rows) (void)hipFree(rows);
  (void)hipFree(s->partials);
  (void)hipFree(s->aheads);
  (void)hipFree(s->maxima);
  (void)hipFree(s->saved);
  delete s;
  return JF_OK;
}

int jf_scorer_create(uint32_t vocabulary, uint32_t max_rows, jf_scorer **out) {
  if (!out) return fail(JF_ERR_INVALID_ARGUMENT, "output pointer is null");
  *out = nullptr;
  if (!vocabulary) return fail(JF_ERR_INVALID_ARGUMENT, "invalid scoring geometry");
  if (vocabulary > kMaxVocabulary)
    return fail(JF_ERR_INVALID_ARGUMENT, "vocabulary exceeds 524288 tokens");
  if (!max_rows || max_rows > kMaxRows)
    return fail(JF_ERR_INVALID_ARGUMENT, "scoring row count is not in 1..4194304");
  jf_scorer *s = new (std::nothrow) jf_scorer;
  if (!s) return fail(JF_ERR_NO_MEMORY, "scorer allocation failed");
  s->vocabulary = vocabulary;
  s->max_rows = max_rows;
  int rc = JF_OK;
  const hipError_t e = hipGetDevice(&s->device);
  if (e != hipSuccess) rc = hip_fail(e, "hipGetDevice");
  // The blocks and groups of one launch's rows, whatever the chunk.
  const uint64_t parts = (uint64_t)std::min(max_rows, launch_rows(vocabulary)) *
                         blocks_of(vocabulary, kLeastChunk);
  const uint64_t maxima = (uint64_t)std::min(max_rows, jf::kTopRows) *
                          blocks_of(vocabulary, kMostChunk) * (kMostChunk / jf::kScoreGroup);
  const uint64_t saved =
      (uint64_t)std::min(max_rows, chunked_rows(vocabulary)) * (2 + jf::kTeacherTokens);
  if (rc == JF_OK) rc = device_alloc(&s->rows, max_rows, "row records");
  if (rc == JF_OK) rc = device_alloc(&s->partials, parts, "row partials");
  if (rc == JF_OK) rc = device_alloc(&s->aheads, parts, "rank partials");
  if (rc == JF_OK) rc = device_alloc(&s->maxima, maxima, "group maxima");
  if (rc == JF_OK) rc = device_alloc(&s->saved, saved, "distillation records");
  if (rc != JF_OK) {
    jf_scorer_destroy(s);
    return rc;
  }
  s->workspace_bytes = max_rows * sizeof(jf::ProcessRow) +
                       parts * (sizeof(float2) + sizeof(uint32_t)) +
                       (maxima + saved) * sizeof(float);
  *out = s;
  return JF_OK;
}

uint64_t jf_scorer_workspace_bytes(const jf_scorer *s) { return s ? s->workspace_bytes : 0; }

// What every call checks of its rows of logits.
static int check_rows(const jf_scorer *s, uint32_t rows, uint32_t dtype, const void *logits,
                      uint64_t stride, const char *what) {
  if (!rows || rows > s->max_rows)
    return fail(JF_ERR_INVALID_ARGUMENT, "invalid scoring batch width");
  if (dtype != JF_DTYPE_F32 && dtype != JF_DTYPE_BF16)
    return fail(JF_ERR_INVALID_ARGUMENT, std::string("unsupported ") + what + " dtype");
  if (!logits) return fail(JF_ERR_INVALID_ARGUMENT, std::string("null ") + what);
  if (rows > 1 && stride < s->vocabulary)
    return fail(JF_ERR_INVALID_ARGUMENT,
                std::string(what) + " row stride is below the vocabulary");
  if ((uintptr_t)logits % element_size(dtype))
    return fail(JF_ERR_INVALID_ARGUMENT,
                std::string(what) + " are not aligned to their element size");
  return JF_OK;
}

// ---- processed logits --------------------------------------------------------

// Leaves the records that a captured call reads to its replays.
static int leave_captured_rows(jf_scorer *s) {
  s->captured_rows.reserve(s->captured_rows.size() + 1);
  jf::ProcessRow *fresh;
  const int rc = device_alloc(&fresh, s->max_rows, "row records");
  if (rc != JF_OK) return rc;
  s->captured_rows.push_back(s->rows);
  s->rows = fresh;
  s->rows_captured = false;
  s->workspace_bytes += s->max_rows * sizeof(jf::ProcessRow);
  return JF_OK;
}

static int fill_process_rows(const jf_scorer *s, const jf_process_args *a,
                             std::vector<jf::ProcessRow> &rows) {
  bool any_constrained = false;
  for (uint32_t r = 0; r < a->rows; ++r) {
    const jf_policy &p = a->policies[r];
    const int rc = jf_policy_validate(&p);
    if (rc != JF_OK) return rc;
    jf::ProcessRow row{};
    row.penalty_row = row.bias_row = jf::kNoRow;
    row.mask_row = a->mask_rows ? a->mask_rows[r] : r;
    if (p.flags & JF_POLICY_CONSTRAINED) {
      row.flags |= jf::kProcessMasked;
      any_constrained = true;
    }
    if (p.flags & JF_POLICY_EXCLUDE_STOP) row.flags |= jf::kProcessStops;
    if (p.repetition != 1.0f || p.presence != 0.0f || p.frequency != 0.0f) {
      if (!a->penalties || !a->penalty_rows || a->penalty_rows[r] >= a->penalties->rows)
        return fail(JF_ERR_INVALID_ARGUMENT, "penalized lane has no penalty table row");
      if (a->penalties->vocabulary != s->vocabulary)
        return fail(JF_ERR_INVALID_ARGUMENT, "penalty table vocabulary differs");
      if (a->penalties->device != s->device)
        return fail(JF_ERR_INVALID_ARGUMENT, "penalty table is on another device");
      if (a->penalties->stale[a->penalty_rows[r]])
        return fail(JF_ERR_LOGIC, "penalty table row is out of date after a failed update; "
                                  "rebuild it");
      row.penalty_row = a->penalty_rows[r];
      row.repetition = p.repetition;
      row.repetition_inverse = std::min(1.0f / p.repetition, FLT_MAX);
      row.presence = p.presence;
      row.frequency = p.frequency;
      row.extra_count = a->extra_counts ? a->extra_counts[r] : 0u;
      if (row.extra_count > (uint32_t)jf::kMaxExtra)
        return fail(JF_ERR_INVALID_ARGUMENT, "more than 16 extra penalty tokens in a row");
      if (row.extra_count && !a->extra_tokens)
        return fail(JF_ERR_INVALID_ARGUMENT, "extra penalty tokens are null");
      const uint64_t offset = !row.extra_count   ? 0
                              : a->extra_offsets ? a->extra_offsets[r]
                                                 : (uint64_t)r * a->extra_stride;
      if (offset > 0xffffffffull - jf::kMaxExtra)
        return fail(JF_ERR_INVALID_ARGUMENT, "extra token offset exceeds 32 bits");
      row.extra_offset = (uint32_t)offset;
    }
    if (a->bias_rows && a->bias_rows[r] != JF_NO_TOKEN) {
      if (!a->biases || a->bias_rows[r] >= a->biases->rows)
        return fail(JF_ERR_INVALID_ARGUMENT, "biased row has no bias table row");
      if (a->biases->vocabulary != s->vocabulary)
        return fail(JF_ERR_INVALID_ARGUMENT, "bias table vocabulary differs");
      if (a->biases->device != s->device)
        return fail(JF_ERR_INVALID_ARGUMENT, "bias table is on another device");
      if (a->biases->stale[a->bias_rows[r]])
        return fail(JF_ERR_LOGIC, "bias table row is out of date after a failed update; set it");
      row.bias_row = a->bias_rows[r];
    }
    rows.push_back(row);
  }
  if (any_constrained &&
      (!a->masks || (a->rows > 1 && a->mask_stride < (s->vocabulary + 31) / 32)))
    return fail(JF_ERR_INVALID_ARGUMENT, "constraint mask buffer is missing or short");
  return JF_OK;
}

int jf_process_logits(jf_scorer *s, const jf_process_args *a, void *stream) {
  if (!s || !a) return fail(JF_ERR_INVALID_ARGUMENT, "null scorer or arguments");
  int rc = check_device(s->device);
  if (rc != JF_OK) return rc;
  rc = check_rows(s, a->rows, a->dtype, a->logits, a->logits_stride, "logits");
  if (rc != JF_OK) return rc;
  rc = check_rows(s, a->rows, a->out_dtype, a->out, a->out_stride, "processed logits");
  if (rc != JF_OK) return rc;
  if (!a->policies) return fail(JF_ERR_INVALID_ARGUMENT, "null policies");
  const bool in_place = a->out == a->logits;
  if (in_place &&
      (a->out_dtype != a->dtype || (a->rows > 1 && a->out_stride != a->logits_stride)))
    return fail(JF_ERR_INVALID_ARGUMENT,
                "logits processed in place keep their dtype and row stride");
  bool capturing;
  rc = is_capturing((hipStream_t)stream, capturing);
  if (rc != JF_OK) return rc;
  try {
    s->host_rows.clear();
    rc = fill_process_rows(s, a, s->host_rows);
    if (rc != JF_OK) return rc;
    // Uploaded only when they change (stream order keeps earlier launches on
    // the records they were enqueued with).
    const size_t bytes = s->host_rows.size() * sizeof(jf::ProcessRow);
    if (s->last_rows.size() < s->host_rows.size() ||
        std::memcmp(s->last_rows.data(), s->host_rows.data(), bytes) != 0) {
      // A replay would upload what the pinned buffer holds by then.
      if (capturing)
        return fail(JF_ERR_LOGIC, "a captured call repeats the rows of the scorer's last call; "
                                  "issue it once before");
      s->last_rows.clear();
      if (s->rows_captured && (rc = leave_captured_rows(s)) != JF_OK) return rc;
      rc = s->staging.upload(s->rows, s->host_rows.data(), bytes, (hipStream_t)stream);
      if (rc != JF_OK) return rc;
      s->last_rows = s->host_rows;
    }
  } catch (const std::bad_alloc &) {
    s->last_rows.clear();
    return fail(JF_ERR_NO_MEMORY, "row record allocation failed");
  }
  s->rows_captured |= capturing;
  const uint64_t stride = a->rows > 1 ? a->logits_stride : s->vocabulary;
  const uint64_t out_stride = a->rows > 1 ? a->out_stride : s->vocabulary;
  const uint32_t most = launch_rows(s->vocabulary);
  const auto masked = [](const jf::ProcessRow &p) { return p.flags != 0; };
  const bool any_masked = std::any_of(s->host_rows.begin(), s->host_rows.end(), masked);
  const bool all_masked = std::all_of(s->host_rows.begin(), s->host_rows.end(), masked);
  for (uint32_t r = 0; r < a->rows; r += most) {
    jf::ProcessLaunch L{};
    L.logits = rows_at(a->logits, r, stride, a->dtype);
    L.out = (void *)rows_at(a->out, r, out_stride, a->out_dtype);
    L.stride = stride;
    L.out_stride = out_stride;
    L.rows = s->rows + r;
    L.row_count = std::min(most, a->rows - r);
    L.vocabulary = s->vocabulary;
    L.in_place = in_place ? 1u : 0u;
    L.any_masked = any_masked ? 1u : 0u;
    L.all_masked = all_masked ? 1u : 0u;
    L.masks = a->masks;
    L.mask_stride = a->mask_stride;
    L.stop0 = a->stop_token_0;
    L.stop1 = a->stop_token_1;
    if (a->penalties) {
      L.pen_entries = (const jf::PenaltyEntry *)a->penalties->entries;
      L.pen_offsets = a->penalties->offsets;
      L.pen_max_entries = a->penalties->max_entries;
    }
    if (a->biases) {
      L.bias_entries = a->biases->entries;
      L.bias_offsets = a->biases->offsets;
      L.bias_max_entries = a->biases->max_entries;
    }
    L.buckets = (s->vocabulary + jf::kPenaltyBucket - 1) / jf::kPenaltyBucket;
    L.extra = a->extra_tokens;
    const int e = jf::launch_process(L, a->dtype, a->out_dtype, stream);
    if (e != hipSuccess) return hip_fail((hipError_t)e, "processed logits launch");
  }
  return JF_OK;
}

// ---- the pass over a row -----------------------------------------------------

// The vectors a thread takes of a row at a time, two while four would leave the
// GPU with few blocks (20 alternatives of one f32 row x 151,936: 8.4 us against
// 8.8, of 64 rows 17.4 against 15.5; of 8 bf16 rows 9.9 against 10.0, of 64 rows
// 15.0 against 14.7; gradients of 32 bf16 rows x 100,003 4.6 against 5.2).
static uint32_t chunk_vectors(uint32_t rows, uint32_t vocabulary, uint32_t dtype) {
  const uint64_t tokens = (uint64_t)rows * vocabulary;
  return tokens <= (dtype == JF_DTYPE_F32 ? 1u << 20 : 8u << 20) ? 2 : 4;
}

static jf::ScoreLaunch score_rows(const jf_scorer *s, const void *logits, uint64_t stride,
                                  uint32_t dtype, uint32_t first, uint32_t rows) {
  jf::ScoreLaunch L{};
  L.logits = rows_at(logits, first, stride, dtype);
  L.stride = stride;
  L.row_count = rows;
  L.vocabulary = s->vocabulary;
  L.vectors = chunk_vectors(rows, s->vocabulary, dtype);
  const uint32_t chunk = jf::chunk_tokens(dtype, L.vectors);
  L.segments = blocks_of(s->vocabulary, chunk);
  L.groups = L.segments * (chunk / jf::kScoreGroup);
  L.temperature = 1.0f;
  // Launches of one call follow one another on its stream: each takes the
  // scratch of the first rows again.
  L.partials = s->partials;
  L.aheads = s->aheads;
  L.maxima = s->maxima;
  return L;
}

// ---- log-probabilities -------------------------------------------------------

int jf_logprobs(jf_scorer *s, const jf_logprobs_args *a, void *stream) {
  if (!s || !a) return fail(JF_ERR_INVALID_ARGUMENT, "null scorer or arguments");
  int rc = check_device(s->device);
  if (rc != JF_OK) return rc;
  rc = check_rows(s, a->rows, a->dtype, a->logits, a->logits_stride, "logits");
  if (rc != JF_OK) return rc;
  if (a->top > jf::kTopLogprobs)
    return fail(JF_ERR_INVALID_ARGUMENT, "more than 128 alternatives in a row");
  if (a->top && (!a->out_top_ids || !a->out_top_logprobs))
    return fail(JF_ERR_INVALID_ARGUMENT, "alternatives need ids and log-probabilities");
  if (a->token_count && (!a->tokens || !a->out_logprobs))
    return fail(JF_ERR_INVALID_ARGUMENT, "scored tokens need ids and log-probabilities");
  if (a->token_count && a->rows > 1 && a->token_stride < a->token_count)
    return fail(JF_ERR_INVALID_ARGUMENT, "token row stride is below the token count");
  if (a->out_ranks && !a->token_count)
    return fail(JF_ERR_INVALID_ARGUMENT, "ranks need scored tokens");
  if (!a->top && !a->token_count && !a->out_lse)
    return fail(JF_ERR_INVALID_ARGUMENT, "nothing to score");
  const uint64_t stride = a->rows > 1 ? a->logits_stride : s->vocabulary;
  const uint32_t most = a->top ? jf::kTopRows : launch_rows(s->vocabulary);
  for (uint32_t r = 0; r < a->rows; r += most) {
    jf::ScoreLaunch L = score_rows(s, a->logits, stride, a->dtype, r, std::min(most, a->rows - r));
    L.temperatures = at(a->temperatures, r);
    L.tokens = at(a->tokens, r * a->token_stride);
    L.token_count = a->token_count;
    L.token_stride = a->rows > 1 ? a->token_stride : 0;
    L.out_lse = at(a->out_lse, r);
    L.out_logprobs = at(a->out_logprobs, (uint64_t)r * a->token_count);
    L.out_ranks = at(a->out_ranks, r);
    L.top = a->top;
    L.out_top_ids = at(a->out_top_ids, (uint64_t)r * a->top);
    L.out_top_logprobs = at(a->out_top_logprobs, (uint64_t)r * a->top);
    int e = jf::launch_score(L, a->dtype, stream);
    if (e == hipSuccess) e = jf::launch_logprobs(L, a->dtype, stream);
    if (e != hipSuccess) return hip_fail((hipError_t)e, "log-probabilities launch");
  }
  return JF_OK;
}

// ---- distillation ------------------------------------------------------------

// `forward`, `backward`: the passes the call makes.
static int check_distill(const jf_scorer *s, const jf_distill_args *a, bool forward,
                         bool backward) {
  int rc = check_device(s->device);
  if (rc != JF_OK) return rc;
  rc = check_rows(s, a->rows, a->dtype, a->logits, a->logits_stride, "logits");
  if (rc != JF_OK) return rc;
  if (!a->teacher_count || a->teacher_count > jf::kTeacherTokens)
    return fail(JF_ERR_INVALID_ARGUMENT, "a teacher's list holds 1..256 tokens");
  if (!a->teacher_ids || (forward && !a->teacher_values))
    return fail(JF_ERR_INVALID_ARGUMENT, "a teacher's list needs ids and values");
  if (a->rows > 1 && a->teacher_stride < a->teacher_count)
    return fail(JF_ERR_INVALID_ARGUMENT, "teacher row stride is below the teacher count");
  if (!std::isfinite(a->temperature) || a->temperature < FLT_MIN)
    return fail(JF_ERR_INVALID_ARGUMENT,
                "distillation requires a finite temperature of at least FLT_MIN");
  if (forward && !a->out_loss) return fail(JF_ERR_INVALID_ARGUMENT, "null losses");
  if (!backward) return JF_OK;
  if (!a->grad_loss) return fail(JF_ERR_INVALID_ARGUMENT, "null loss gradients");
  if (!forward && !a->saved)
    return fail(JF_ERR_INVALID_ARGUMENT, "the backward pass needs what the forward pass saved");
  rc = check_rows(s, a->rows, a->dtype, a->grad, a->grad_stride, "gradients");
  if (rc != JF_OK) return rc;
  if (a->grad == a->logits && a->rows > 1 && a->grad_stride != a->logits_stride)
    return fail(JF_ERR_INVALID_ARGUMENT, "gradients in place of the logits keep their row stride");
  return JF_OK;
}

static int distill(jf_scorer *s, const jf_distill_args *a, bool forward, bool backward,
                   void *stream) {
  if (!s || !a) return fail(JF_ERR_INVALID_ARGUMENT, "null scorer or arguments");
  const int rc = check_distill(s, a, forward, backward);
  if (rc != JF_OK) return rc;
  const uint64_t stride = a->rows > 1 ? a->logits_stride : s->vocabulary;
  const uint64_t grad_stride = a->rows > 1 ? a->grad_stride : s->vocabulary;
  const uint32_t K = a->teacher_count;
  const uint32_t most = launch_rows(s->vocabulary);
  for (uint32_t r = 0; r < a->rows; r += most) {
    const uint32_t n = std::min(most, a->rows - r);
    float *saved = a->saved ? a->saved + (uint64_t)r * (2 + K) : backward ? s->saved : nullptr;
    jf::ScoreLaunch L = score_rows(s, a->logits, stride, a->dtype, r, n);
    jf::DistillGradLaunch G{};
    L.temperature = G.temperature = a->temperature;
    L.teacher_ids = G.teacher_ids = a->teacher_ids + r * a->teacher_stride;
    L.teacher_stride = G.teacher_stride = a->teacher_stride;
    L.teacher_count = G.teacher_count = K;
    L.saved = saved;
    G.saved = saved;
    if (forward) {
      L.out_lse = at(a->out_lse, r);
      L.teacher_values = a->teacher_values + r * a->teacher_stride;
      L.normalize = a->normalize ? 1u : 0u;
      L.out_loss = a->out_loss + r;
    }
    if (backward) {
      G.logits = L.logits;
      G.stride = stride;
      G.grad = (void *)rows_at(a->grad, r, grad_stride, a->dtype);
      G.grad_stride = grad_stride;
      G.row_count = n;
      G.vocabulary = s->vocabulary;
      G.vectors = L.vectors;
      G.grad_loss = a->grad_loss + r * a->grad_loss_stride;
      G.grad_loss_stride = a->grad_loss_stride;
    }
    int e = hipSuccess;
    if (forward && backward && n >= whole_rows(s->vocabulary, a->dtype)) {
      L.saved = a->saved ? saved : nullptr;
      e = jf::launch_distill_step(L, G, a->dtype, stream);
    } else {
      if (forward) e = jf::launch_score(L, a->dtype, stream);
      if (forward && e == hipSuccess) e = jf::launch_distill_loss(L, a->dtype, stream);
      if (backward && e == hipSuccess) e = jf::launch_distill_grad(G, a->dtype, stream);
    }
    if (e != hipSuccess) return hip_fail((hipError_t)e, "distillation launch");
  }
  return JF_OK;
}

int jf_distill(jf_scorer *s, const jf_distill_args *a, void *stream) {
  return distill(s, a, true, false, stream);
}
int jf_distill_backward(jf_scorer *s, const jf_distill_args *a, void *stream) {
  return distill(s, a, false, true, stream);
}
int jf_distill_step(jf_scorer *s, const jf_distill_args *a, void *stream) {
  return distill(s, a, true, true, stream);
}

}  // extern "C"
