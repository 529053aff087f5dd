// Host side of the losses of drawn tokens (include/jf_sampler.h): argument checks
// and the launches of jf_learn.hip, over a scorer's scratch.
#include "jf_learn.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "jf_scorer_host.h"

namespace {

using namespace jf::host;

constexpr uint32_t kMaxPairs = 1u << 22;
// Rows of a preference call that the pairs' launch works out itself, a thread each: one
// pair may hold them all, in four turns of its block.
constexpr uint32_t kPairRows = 1024;
// Rows below which they are always taken by chunks: the pairs' launch, which there is
// anyway, joins them (48 f32 rows x 32,000 8.4 us against 8.9, 150 rows 10.3 against 9.9).
constexpr uint32_t kWholePairRows = 144;

// What both losses' calls share.
struct Rows {
  uint32_t rows, dtype;
  const void *logits;
  uint64_t stride;
  float temperature;
  const uint32_t *tokens;
  float *saved;
  const float *grad_loss;
  uint64_t grad_loss_stride;
  void *grad;
  uint64_t grad_stride;
};
template <class Args>
Rows rows_of(const Args *a) {
  return {a->rows,  a->dtype,     a->logits,           a->logits_stride, a->temperature, a->tokens,
          a->saved, a->grad_loss, a->grad_loss_stride, a->grad,          a->grad_stride};
}

int check_learned(const jf_scorer *s, const Rows &a, bool saved, bool backward) {
  int rc = check_device(s->device);
  if (rc != JF_OK) return rc;
  rc = check_rows(s, a.rows, a.dtype, a.logits, a.stride, "logits");
  if (rc != JF_OK) return rc;
  if (!std::isfinite(a.temperature) || a.temperature < FLT_MIN)
    return fail(JF_ERR_INVALID_ARGUMENT,
                "a loss requires a finite temperature of at least FLT_MIN");
  if (!a.tokens) return fail(JF_ERR_INVALID_ARGUMENT, "null tokens");
  if (saved && !a.saved)
    return fail(JF_ERR_INVALID_ARGUMENT, "the loss needs a place for what its passes share");
  if ((uintptr_t)a.saved % sizeof(jf::LearnedRow))
    return fail(JF_ERR_INVALID_ARGUMENT, "rows' records are not aligned to 16 bytes");
  if (!backward) return JF_OK;
  if (!a.grad_loss) return fail(JF_ERR_INVALID_ARGUMENT, "null loss gradients");
  rc = check_rows(s, a.rows, a.dtype, a.grad, a.grad_stride, "gradients");
  if (rc != JF_OK) return rc;
  if (a.grad == a.logits && a.rows > 1 && a.grad_stride != a.stride)
    return fail(JF_ERR_INVALID_ARGUMENT, "gradients in place of the logits keep their row stride");
  return JF_OK;
}

uint64_t row_stride(const jf_scorer *s, uint32_t rows, uint64_t stride) {
  return rows > 1 ? stride : s->vocabulary;
}

// The pass over rows [first, first + count), whose records go to `saved`.
jf::LearnLaunch score_launch(const jf_scorer *s, const Rows &a, uint32_t first, uint32_t count,
                             jf::LearnedRow *saved) {
  const uint64_t stride = row_stride(s, a.rows, a.stride);
  jf::LearnLaunch L{};
  L.logits = rows_at(a.logits, first, stride, a.dtype);
  L.stride = stride;
  L.tokens = a.tokens + first;
  L.row_count = count;
  L.vocabulary = s->vocabulary;
  L.vectors = chunk_vectors(count, s->vocabulary, a.dtype);
  // Many f32 tokens: as large a chunk as bf16's, of which fewer are joined (1000 rows x
  // 248,320 171 -> 166 us, 200 rows 39.6 -> 38.9; 48 rows x 100,003 9.8 -> 10.2, so not there).
  if (a.dtype == JF_DTYPE_F32 && (uint64_t)count * s->vocabulary >= 24u << 20) L.vectors = 8;
  L.segments = blocks_of(s->vocabulary, jf::chunk_tokens(a.dtype, L.vectors));
  L.temperature = a.temperature;
  L.partials = s->partials;
  L.means = (float *)s->aheads;  // a float a chunk; no ranks are counted
  L.saved = saved;
  return L;
}

jf::LearnGradLaunch grad_launch(const jf_scorer *s, const Rows &a, uint32_t first, uint32_t count,
                                const jf::LearnedRow *saved) {
  const uint64_t stride = row_stride(s, a.rows, a.stride);
  jf::LearnGradLaunch G{};
  G.logits = rows_at(a.logits, first, stride, a.dtype);
  G.stride = stride;
  G.grad_stride = row_stride(s, a.rows, a.grad_stride);
  G.grad = (void *)rows_at(a.grad, first, G.grad_stride, a.dtype);
  G.tokens = a.tokens + first;
  G.saved = saved;
  G.grad_loss = a.grad_loss;
  G.grad_loss_stride = a.grad_loss_stride;
  G.row_count = count;
  G.vocabulary = s->vocabulary;
  G.vectors = chunk_vectors(count, s->vocabulary, a.dtype);
  G.temperature = a.temperature;
  return G;
}

// Whether a forward pass takes rows whole: not where a row's block would be on its way
// longer than the row's chunks take, spread over the GPU (bf16 x 100,003, 64 rows 10.1 us
// against 8.6, 128 rows 10.3 against 10.6; f32, 32 rows 9.4 against 8.1, 96 rows 9.8 against
// 11.5); nor where so much is left to the last rows' blocks that it weighs more than the
// launch saved (300 bf16 rows x 151,936 24.2 against 21.3, 1100 rows 63 against 60; f32 x
// 151,936 39 against 36, 118 against 114; but bf16 x 100,003 1500 rows 57.5 against 57.6,
// 3000 rows 105 against 111).
bool whole_rows(uint32_t rows, uint32_t vocabulary, uint32_t dtype) {
  if (vocabulary <= 72u << 10) return true;
  if (dtype == JF_DTYPE_BF16) return vocabulary <= 128u << 10 && rows >= 128;
  return vocabulary <= 104u << 10 && rows >= 80;
}
// Their threads: 512, which ask for more at once, where they fill their vectors and there
// are few rows (16 f32 rows x 32,000 6.1 us, 6.5 with 256); 256, of which more rows are under
// way, where rows are many or short (600 bf16 rows x 64,000 17.0 us, 18.8 with 512; 4096 x
// 8000 15.5, 24).
uint32_t rows_threads(uint32_t rows, uint32_t vocabulary, uint32_t dtype) {
  const uint32_t bytes = vocabulary * (uint32_t)element_size(dtype);
  return bytes <= 24u << 10 || (bytes <= 128u << 10 && rows > 256) ? 256 : 512;
}

// ---- a row's own loss -----------------------------------------------------------

// A step of whole rows: 1024 threads a row where two rows on a CU would leave most of
// each to the caches (512 f32 rows x 151,936 127 us against 140, x 248,320 207 against
// 248; bf16 105 against 113, but of 151,936 tokens 66 against 65, and 2048 rows, a
// quarter of them without a token, 242 against 233).
uint32_t step_threads(uint32_t vocabulary, uint32_t dtype) {
  return vocabulary * (uint32_t)element_size(dtype) > 320u << 10 ? 1024 : 512;
}
// Floats (or ids) that a call reads or writes.
struct Floats {
  const void *begin;
  uint64_t count;
};
bool meet(const Floats &x, const Floats &y) {
  return x.begin && y.begin &&
         (uintptr_t)x.begin < (uintptr_t)y.begin + y.count * sizeof(float) &&
         (uintptr_t)y.begin < (uintptr_t)x.begin + x.count * sizeof(float);
}
template <size_t N>
bool meet(const Floats (&outputs)[N], const Floats &in) {
  return std::any_of(outputs, outputs + N, [&](const Floats &out) { return meet(out, in); });
}
// Whether outputs are in the place of what launches behind theirs read: the tokens, and
// for gradients the losses'.
template <size_t N>
bool meet_late(const Floats (&outputs)[N], const Rows &a, uint64_t losses, bool gradients) {
  return meet(outputs, {a.tokens, a.rows}) ||
         (gradients && meet(outputs, {a.grad_loss, (losses - 1) * a.grad_loss_stride + 1}));
}

bool outputs_meet(const jf_clipped_args *a, const float *in) {
  const uint64_t n = a->rows;
  return meet({{a->out_loss, n}, {a->out_logprobs, n}, {a->out_kl, n}, {a->out_entropy, n},
               {a->saved, 4 * n}}, {in, n});
}

// The blocks of a step that share a row (16 f32 rows x 32,000 with entropies: one 9.3 us,
// two 8.2, four 8.2, eight 8.8; one row 9.0, 7.9, 7.5, 7.2; 64 rows 9.8, 9.7, 11.2; 64 bf16
// rows 9.0, 8.4, 9.2). Not where one of them would write what another one reads.
uint32_t step_blocks(uint32_t rows, const jf_clipped_args *a) {
  if (rows > 64 || a->grad == a->logits || outputs_meet(a, a->advantages) ||
      outputs_meet(a, a->old_logprobs) || outputs_meet(a, a->reference_logprobs))
    return 1;
  return rows <= 4 ? 8 : rows <= 24 ? 4 : 2;
}
// Whether a step takes rows whole: always where a row is short (one f32 row x 32,000 with
// entropies in eight blocks 7.2 us, 8.3 by chunks, x 40,000 8.1 against 7.9, 16 rows 9.5
// against 8.6), and from where the rows keep the CUs busy. Entropies cost whole rows more
// than chunks, so that one rule for both comes late without them and, by up to 5%, early
// with them. Whole against chunks, without and with entropies: f32 x 48,000, 64 rows 11.3
// against 10.1, 12.7 against 11.1; 96 rows 12.1, 13.7; 14.0, 14.8; x 100,003, 80 rows 20.2,
// 20.5; 23.8, 22.7; 96 rows 20.8, 22.5; 24.3, 24.5; x 151,936, 96 rows 28.5, 31.9; 33.0,
// 32.8; of the longest, with them, 192 rows 95, 91; 256 rows 112, 118. bf16 x 64,000, 112
// rows 11.8, 12.9; 14.5, 14.4; 128 rows 12.0, 13.6; 14.7, 15.1; x 100,003, 160 rows 21.2,
// 21.3; 25.5, 23.3; 176 rows 21.7, 22.6; 25.9, 24.6; 200 rows 22.1, 24.2; 26.4, 26.2; x
// 151,936, 176 rows 28.3, 31.4; 33.8, 33.1.
bool whole_step(uint32_t rows, uint32_t vocabulary, uint32_t dtype) {
  const bool bf16 = dtype == JF_DTYPE_BF16;
  if (vocabulary <= 36u << 10) return true;
  return rows >= (bf16 ? vocabulary <= 66u << 10 ? 112 : 176 : vocabulary <= 200000 ? 96 : 224);
}
// Tokens of a step by chunks up to which the rows' own losses come with the gradients: each
// block joins its row's sums, while the GPU has room for all of them at once (one f32 row x
// 100,003 11.3 -> 7.7 us, 16 rows 10.9 -> 10.1, 32 rows 12.9 -> 13.0; 16 bf16 rows x 151,936
// 10.9 -> 10.3, 32 rows 12.2 -> 12.9; 32 f32 rows x 70,000, otherwise whole and then the
// gradients, 14.4 -> 11.5).
constexpr uint64_t kOwnTokens = 3u << 20;

bool is_bound(float v) { return v >= 0.0f; }  // +infinity: none

int clipped(jf_scorer *s, const jf_clipped_args *a, bool forward, bool backward, void *stream) {
  if (!s || !a) return fail(JF_ERR_INVALID_ARGUMENT, "null scorer or arguments");
  const Rows rows = rows_of(a);
  const int rc = check_learned(s, rows, backward, backward);
  if (rc != JF_OK) return rc;
  if (!std::isfinite(a->entropy_weight))
    return fail(JF_ERR_INVALID_ARGUMENT, "entropy weight is not finite");
  if (forward) {
    if (!a->advantages) return fail(JF_ERR_INVALID_ARGUMENT, "null advantages");
    if (!a->out_loss) return fail(JF_ERR_INVALID_ARGUMENT, "null losses");
    if (!is_bound(a->clip_low) || !is_bound(a->clip_high))
      return fail(JF_ERR_INVALID_ARGUMENT, "clip bounds are not in 0..infinity");
    if (!std::isfinite(a->kl_weight))
      return fail(JF_ERR_INVALID_ARGUMENT, "KL weight is not finite");
    if (!a->reference_logprobs && (a->kl_weight != 0.0f || a->out_kl))
      return fail(JF_ERR_INVALID_ARGUMENT, "a KL term needs the reference's log-probabilities");
  }
  const bool step = forward && backward;
  const uint64_t count = a->rows;
  const bool late = step && meet_late({{a->out_loss, count}, {a->out_logprobs, count},
                                       {a->out_kl, count}, {a->out_entropy, count},
                                       {a->saved, 4 * count}}, rows, count, true);
  const uint32_t most = launch_rows(s->vocabulary);
  for (uint32_t r = 0; r < a->rows; r += most) {
    const uint32_t n = std::min(most, a->rows - r);
    jf::LearnedRow *saved = at((jf::LearnedRow *)a->saved, r);
    jf::LearnLaunch L{};
    jf::LearnGradLaunch G{};
    if (forward) {
      L = score_launch(s, rows, r, n, saved);
      L.entropy = a->entropy_weight != 0.0f || a->out_entropy ? 1u : 0u;
      L.advantages = a->advantages + r;
      L.old_logprobs = at(a->old_logprobs, r);
      L.reference = at(a->reference_logprobs, r);
      L.clip_low = a->clip_low;
      L.clip_high = a->clip_high;
      L.kl_weight = a->kl_weight;
      L.entropy_weight = a->entropy_weight;
      L.out_loss = a->out_loss + r;
      L.out_logprobs = at(a->out_logprobs, r);
      L.out_kl = at(a->out_kl, r);
      L.out_entropy = at(a->out_entropy, r);
    }
    if (backward) {
      G = grad_launch(s, rows, r, n, saved);
      G.grad_loss += r * a->grad_loss_stride;
      G.entropy_weight = a->entropy_weight;
    }
    int e = hipSuccess;
    G.blocks = step && !late ? step_blocks(n, a) : 1;
    if (step && (late || whole_step(n, s->vocabulary, a->dtype))) {
      const uint32_t threads = G.blocks > 1 ? 512 : step_threads(s->vocabulary, a->dtype);
      e = jf::launch_clipped_step(L, G, a->dtype, threads, stream);
    } else {
      const bool own = G.blocks > 1 && (uint64_t)n * s->vocabulary <= kOwnTokens;
      if (forward && !own && whole_rows(n, s->vocabulary, a->dtype)) {
        e = jf::launch_learn_rows(L, false, a->dtype, rows_threads(n, s->vocabulary, a->dtype),
                                  stream);
      } else if (forward) {
        e = jf::launch_learn_score(L, a->dtype, stream);
        if (!own && e == hipSuccess) e = jf::launch_clipped_rows(L, a->dtype, stream);
      }
      if (backward && e == hipSuccess)
        e = jf::launch_learn_grad(G, own ? &L : nullptr, a->dtype, stream);
    }
    if (e != hipSuccess) return hip_fail((hipError_t)e, "clipped loss launch");
  }
  return JF_OK;
}

// ---- pairs of sequences ------------------------------------------------------------

int preference(jf_scorer *s, const jf_preference_args *a, bool forward, bool backward,
               void *stream) {
  if (!s || !a) return fail(JF_ERR_INVALID_ARGUMENT, "null scorer or arguments");
  const Rows rows = rows_of(a);
  const int rc = check_learned(s, rows, true, backward);
  if (rc != JF_OK) return rc;
  if (!a->pairs || a->pairs > kMaxPairs)
    return fail(JF_ERR_INVALID_ARGUMENT, "pair count is not in 1..4194304");
  if (forward) {
    if (!a->offsets) return fail(JF_ERR_INVALID_ARGUMENT, "null sequence offsets");
    if (!a->out_loss) return fail(JF_ERR_INVALID_ARGUMENT, "null losses");
    if (a->loss > JF_PREFERENCE_SQUARED)
      return fail(JF_ERR_INVALID_ARGUMENT, "unknown preference loss");
    if (!std::isfinite(a->beta) || !(a->beta > 0.0f))
      return fail(JF_ERR_INVALID_ARGUMENT, "beta is not positive and finite");
    if (!std::isfinite(a->margin)) return fail(JF_ERR_INVALID_ARGUMENT, "margin is not finite");
    if (!(a->smoothing >= 0.0f && a->smoothing <= 1.0f))
      return fail(JF_ERR_INVALID_ARGUMENT, "smoothing is not in 0..1");
  }
  const uint64_t count = a->rows;
  if (forward &&
      meet_late({{a->out_loss, a->pairs}, {a->out_scores, 2ull * a->pairs},
                 {a->out_logprobs, count}, {a->saved, 4 * count}}, rows, a->pairs, backward))
    return fail(JF_ERR_INVALID_ARGUMENT,
                "outputs share elements with the tokens or the losses' gradients");
  jf::LearnedRow *saved = (jf::LearnedRow *)a->saved;
  const uint32_t most = launch_rows(s->vocabulary);
  int e = hipSuccess;
  if (forward) {
    jf::LearnLaunch L{};
    const bool whole = a->rows >= kWholePairRows &&
                       whole_rows(std::min(most, a->rows), s->vocabulary, a->dtype);
    const bool with_rows = !whole && a->rows <= std::min(most, kPairRows);
    for (uint32_t r = 0; r < a->rows && e == hipSuccess; r += most) {
      L = score_launch(s, rows, r, std::min(most, a->rows - r), saved + r);
      L.reference = at(a->reference_logprobs, r);
      L.out_logprobs = at(a->out_logprobs, r);
      if (whole) {
        e = jf::launch_learn_rows(L, true, a->dtype,
                                  rows_threads(L.row_count, s->vocabulary, a->dtype), stream);
        continue;
      }
      e = jf::launch_learn_score(L, a->dtype, stream);
      if (!with_rows && e == hipSuccess) e = jf::launch_pair_rows(L, a->dtype, stream);
    }
    jf::PairLaunch P{};
    P.saved = saved;
    P.tokens = a->tokens;
    P.rows = a->rows;
    P.vocabulary = s->vocabulary;
    P.pairs = a->pairs;
    P.offsets = a->offsets;
    P.loss = a->loss;
    P.mean = a->mean ? 1u : 0u;
    P.beta = a->beta;
    P.margin = a->margin;
    P.smoothing = a->smoothing;
    P.out_loss = a->out_loss;
    P.out_scores = a->out_scores;
    if (e == hipSuccess) e = jf::launch_pairs(P, L, with_rows, a->dtype, stream);
  }
  if (backward) {
    for (uint32_t r = 0; r < a->rows && e == hipSuccess; r += most) {
      jf::LearnGradLaunch G = grad_launch(s, rows, r, std::min(most, a->rows - r), saved + r);
      G.pairs = a->pairs;
      e = jf::launch_learn_grad(G, nullptr, a->dtype, stream);
    }
  }
  if (e != hipSuccess) return hip_fail((hipError_t)e, "preference loss launch");
  return JF_OK;
}

}  // namespace

extern "C" {

int jf_clipped_loss(jf_scorer *s, const jf_clipped_args *a, void *stream) {
  return clipped(s, a, true, false, stream);
}
int jf_clipped_loss_backward(jf_scorer *s, const jf_clipped_args *a, void *stream) {
  return clipped(s, a, false, true, stream);
}
int jf_clipped_loss_step(jf_scorer *s, const jf_clipped_args *a, void *stream) {
  return clipped(s, a, true, true, stream);
}

int jf_preference_loss(jf_scorer *s, const jf_preference_args *a, void *stream) {
  return preference(s, a, true, false, stream);
}
int jf_preference_loss_backward(jf_scorer *s, const jf_preference_args *a, void *stream) {
  return preference(s, a, false, true, stream);
}
int jf_preference_loss_step(jf_scorer *s, const jf_preference_args *a, void *stream) {
  return preference(s, a, true, true, stream);
}

}  // extern "C"
