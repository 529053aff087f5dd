// Losses of drawn tokens on gfx950. With t_j = (x_j - m) / T, m a row's maximum,
// S = sum exp t_j, p_j = exp(t_j) / S, a its token, lp = t_a - ln S and
// E = sum p_j t_j, the entropy is ln S - E and ln p_j + H = t_j - E. A loss of
// slope G by lp and weight h of the entropy has
//   dx_j = g / T * (G [j = a] + p_j (h (t_j - E) - G)),
// so a backward pass reads the logits once, writes the gradient once, and needs
// four numbers a row.
//
// Forward: a block takes a row that has a token (others are not read), or a chunk of
// one, of which it leaves maximum and sum for a wave that joins them; one lane works
// the token out, in 64 bits. A pair's block then adds its rows' distances from the
// reference, in 64 bits, and leaves the slope with each row.
//
// Memory bounds all of it but small calls, which wait for it: reads reach 5.0 to 5.8
// TB/s, the backward pass 5.5 to 6.2, read and written.
#include <hip/hip_runtime.h>

#include "jf_learn.h"
#include "jf_logits.h"

namespace jf {

namespace {

constexpr float kLn2 = 0.693147180559945309f;
// An exponent (of 2) below which nothing is left of an exponential; what is far
// below it, -infinity among it, is taken as this, so that products with it are 0.
constexpr float kNoExponent = -1e4f;

__device__ __forceinline__ float bounded(float t) { return __builtin_fmaxf(t, kNoExponent); }

// A running maximum m, sum s of exponentials e = 2^u, u = (x - m) c, and sum w of
// e u.
struct MaxSums {
  float m, s, w;
};
// Its sums for the maximum r, which is at least m.
__device__ __forceinline__ MaxSums from(const MaxSums &p, float r, float c) {
  const float u = (p.m - r) * c, f = __builtin_amdgcn_exp2f(u);
  return {r, p.s * f, (p.w + p.s * bounded(u)) * f};
}
__device__ __forceinline__ MaxSums join(const MaxSums &p, const MaxSums &q, float c) {
  const float m = __builtin_fmaxf(p.m, q.m), r = finite_reference(m);
  const MaxSums a = from(p, r, c), b = from(q, r, c);
  return {m, a.s + b.s, a.w + b.w};
}
template <bool ENTROPY>
__device__ __forceinline__ MaxSums wave_join(const MaxSums &p, float c) {
  const float m = wave_max_f32(p.m);
  const MaxSums a = from(p, finite_reference(m), c);
  return {m, wave_sum_f32(a.s), ENTROPY ? wave_sum_f32(a.w) : 0.0f};
}

// A row's, in 64 bits where its blocks' or waves' come together: each of theirs has been
// rounded at its own share of the row, an addition in 32 bits would be at the whole
// (log-probabilities among 151,936 tokens off by 6.0e-8, 9.2e-8 with 32 bits; the blocks'
// own sums in 64 bits would leave 4.8e-8 and cost 4% of a call).
struct RowSums {
  float m;
  double s;
  float w;
};
template <bool ENTROPY>
__device__ __forceinline__ RowSums whole(const MaxSums &p, float c) {
  const float m = wave_max_f32(p.m);
  const MaxSums a = from(p, finite_reference(m), c);
  return {m, wave_sum_f64(a.s), ENTROPY ? wave_sum_f32(a.w) : 0.0f};
}

// Functions in 64 bits, off by less than 2^-40 of the result: a lane goes through them
// alone while its wave waits, and those of the last bit take several times as long (a
// step of 16 f32 rows x 32,000 7.8 -> 7.6 us).
__device__ __forceinline__ double inverse_of(double v) {
  double r = __builtin_amdgcn_rcp(v);
  r = __builtin_fma(__builtin_fma(-v, r, 1.0), r, r);
  return __builtin_fma(__builtin_fma(-v, r, 1.0), r, r);
}
// The N first terms of atanh z / z, by y = z^2: 1 + y / 3 + y^2 / 5 ...
template <int N>
__device__ __forceinline__ double atanh_series(double y) {
  double sum = 1.0 / (2 * N - 1);
#pragma unroll
  for (int n = N - 2; n >= 0; --n) sum = __builtin_fma(sum, y, 1.0 / (2 * n + 1));
  return sum;
}
// ln v of a number of at least 2^-1022, infinity or NaN, by v = 2^k m, m in
// (sqrt(1/2), sqrt(2)], and ln m = 2 atanh((m - 1) / (m + 1)); ln 0 is -infinity.
__device__ __forceinline__ double log_of(double v) {
  int k = __builtin_amdgcn_frexp_exp(v);
  double m = __builtin_amdgcn_frexp_mant(v);
  const bool low = m <= 0.70710678118654752;
  m = low ? m + m : m;
  k = low ? k - 1 : k;
  const double z = (m - 1.0) * inverse_of(m + 1.0);
  const double whole = __builtin_fma((double)k, 0.693147180559945309417,
                                     (z + z) * atanh_series<8>(z * z));
  return v == 0.0 ? -__builtin_inf() : v == __builtin_inf() ? v : whole;
}
// ln(1 + v), 0 <= v <= 1, as 2 atanh(v / (2 + v)).
__device__ __forceinline__ double log1_of(double v) {
  const double z = v * inverse_of(2.0 + v);
  return (z + z) * atanh_series<13>(z * z);
}
// e^v: whole, less 1, and less 1 + v; by v = k ln 2 + r, |r| <= ln 2 / 2, and the series of
// e^r, whose terms from r^2 on are `over`.
struct Exponential {
  double whole, less, over;
};
__device__ __forceinline__ Exponential exp_of(double v) {
  // Past these there is nothing or infinity left; NaN has no order.
  const double x = v > 800.0 ? 800.0 : v < -800.0 ? -800.0 : v;
  const double k = __builtin_rint(x * 1.44269504088896340736);
  const double r = __builtin_fma(-k, 0.693147180559945309417, x);
  double sum = 1.0 / 39916800.0;  // 11!
  const double inverses[9] = {1.0 / 2,    1.0 / 6,     1.0 / 24,     1.0 / 120,    1.0 / 720,
                              1.0 / 5040, 1.0 / 40320, 1.0 / 362880, 1.0 / 3628800};
#pragma unroll
  for (int n = 8; n >= 0; --n) sum = __builtin_fma(sum, r, inverses[n]);
  const double over = sum * r * r;
  const double whole = __builtin_ldexp(1.0 + r + over, k == k ? (int)k : 0);
  if (k == 0.0) return {whole, r + over, over};
  const double less = whole - 1.0;
  return {whole, less, less == __builtin_inf() ? less : less - v};
}

// Adds N (even) vectors, for the maximum r; BOUNDED: tokens of -infinity may be among
// them, whose exponent times their 0 is no number. A vector's sums start from 0 and are
// added in pairs: in one chain over a row the tokens behind a likely one lose bits to it
// (log-probabilities of 2048 steps off by 6e-7, of which 4e-7 one way; 1.4e-7 so, the
// rounding of what is stored).
template <int DT, bool ENTROPY, bool BOUNDED, uint32_t N>
__device__ __forceinline__ void add_vectors(MaxSums &run, const LogitWords (&w)[N], float r,
                                            float c) {
  float s[N], t[N];
#pragma unroll
  for (uint32_t j = 0; j < N; ++j) {
    float v[Logits<DT>::VEC];
    unpack<DT>(w[j], v);
    s[j] = t[j] = 0.0f;
#pragma unroll
    for (uint32_t e = 0; e < Logits<DT>::VEC; ++e) {
      const float u = (v[e] - r) * c, p = __builtin_amdgcn_exp2f(u);
      s[j] += p;
      if constexpr (ENTROPY) t[j] = __builtin_fmaf(p, BOUNDED ? bounded(u) : u, t[j]);
    }
  }
  float whole = s[0] + s[1], product = t[0] + t[1];
#pragma unroll
  for (uint32_t j = 2; j < N; j += 2) {
    whole += s[j] + s[j + 1];
    product += t[j] + t[j + 1];
  }
  run.s += whole;
  if constexpr (ENTROPY) run.w += product;
}

template <int DT, uint32_t N, bool ENTROPY>
__global__ __launch_bounds__(256) void learn_score_kernel(LearnLaunch a) {
  constexpr uint32_t CHUNK = N * kSlab<DT>;
  __shared__ MaxSums wave_part[4];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  const uint32_t row = blockIdx.x / a.segments, segment = blockIdx.x - row * a.segments;
  const uint32_t V = a.vocabulary;
  const auto *x = row_of<DT>(a.logits, (uint64_t)row * a.stride);
  LogitWords w[N];
  // Small calls wait for memory, not for its rate: the chunk is asked for beside the
  // token, which then says whether it is of any use.
  constexpr bool AHEAD = N == 2;
  if (!AHEAD && a.tokens[row] >= V) return;
  load_chunk<DT>(x, segment * CHUNK, V, kPastMinusInfinity<DT>, w);
  if (AHEAD && a.tokens[row] >= V) return;
  const float c = kLog2e / a.temperature;
  float top = vector_max<DT>(w[0]);
#pragma unroll
  for (uint32_t j = 1; j < N; ++j) top = loaded_max(top, vector_max<DT>(w[j]));
  const float r = finite_reference(top);
  MaxSums run{top, 0.0f, 0.0f};
  // Past a row's end a chunk has -infinity (1000 bf16 rows x 151,936: 63 us a call, 66
  // where that was found below).
  const bool bounds = ENTROPY && segment * CHUNK + CHUNK > V;
  if (bounds)
    add_vectors<DT, ENTROPY, true>(run, w, r, c);
  else
    add_vectors<DT, ENTROPY, false>(run, w, r, c);
  if constexpr (ENTROPY) {
    // -infinity among its tokens: again, which few chunks need (the same call: 68.7 us with
    // every exponent bounded).
    if (ballot(!bounds && run.w != run.w)) {
      run = MaxSums{top, 0.0f, 0.0f};
      // Unpacked anew: kept from above they would take twice the registers.
#pragma unroll
      for (uint32_t j = 0; j < N; ++j) asm volatile("" : "+v"(w[j]));
      add_vectors<DT, ENTROPY, true>(run, w, r, c);
    }
  }
  run = wave_join<ENTROPY>(run, c);
  if (lane == 0) wave_part[wave] = run;
  __syncthreads();
  if (tid == 0) {
    const MaxSums total = join(join(wave_part[0], wave_part[1], c),
                               join(wave_part[2], wave_part[3], c), c);
    const uint64_t at = (uint64_t)row * a.segments + segment;
    a.partials[at] = make_float2(total.m, total.s);
    if constexpr (ENTROPY) a.means[at] = total.w;
  }
}

// A lane's first block of a row; of a row without a token, anything.
template <bool ENTROPY>
__device__ __forceinline__ MaxSums row_part(const LearnLaunch &a, uint32_t row) {
  const uint32_t g = threadIdx.x & 63u;
  if (g >= a.segments) return MaxSums{-__builtin_inff(), 0.0f, 0.0f};
  const uint64_t at = (uint64_t)row * a.segments + g;
  const float2 v = a.partials[at];
  return MaxSums{v.x, v.y, ENTROPY ? a.means[at] : 0.0f};
}
// A row's sums from its blocks', every lane of the wave; `run` is the lane's row_part,
// asked for before the row's token is known.
template <bool ENTROPY>
__device__ __forceinline__ RowSums row_sums(const LearnLaunch &a, uint32_t row, MaxSums run,
                                            float c) {
  for (uint32_t g = (threadIdx.x & 63u) + 64; g < a.segments; g += 64) {
    const uint64_t at = (uint64_t)row * a.segments + g;
    const float2 v = a.partials[at];
    run = join(run, MaxSums{v.x, v.y, ENTROPY ? a.means[at] : 0.0f}, c);
  }
  return whole<ENTROPY>(run, c);
}

// ln q of a token of logit x: with the row's sums in fp32, in 64 bits, since what
// follows from it is its small distance from another log-probability. The sum's exponents
// are by a rounded c, so the token's is too, by the same share of its own: then the
// rounding weighs its distance from the mean exponent, which is 0 on the average of drawn
// tokens, where by 1 / T alone it would weigh the mean, the same way in every row of a
// sequence. An exponent below -16, which no mean is near, takes the share of -16.
__device__ __forceinline__ double token_logprob(float x, const RowSums &total, float temperature) {
  // A token of logit -infinity has no probability, whatever else the row holds
  // but NaN.
  if (x == -__builtin_inff() && total.s == total.s) return -__builtin_inf();
  const double share = __builtin_fma((double)(kLog2e / temperature) * 0.693147180559945309417,
                                     (double)temperature, -1.0);
  const double t = ((double)x - (double)total.m) * inverse_of((double)temperature);
  return __builtin_fma(fmax(t, -16.0), share, t) - log_of(total.s);
}
__device__ __forceinline__ float inverse_sum(const RowSums &total) {
  return total.s == 0.0 ? 0.0f : 1.0f / (float)total.s;
}

// What a row's own loss takes beside its logits.
struct RowTerms {
  float x, advantage, old, reference;
};
__device__ __forceinline__ RowTerms row_terms(const LearnLaunch &a, uint32_t row, float x) {
  return {x, a.advantages[row], a.old_logprobs ? a.old_logprobs[row] : 0.0f,
          a.reference ? a.reference[row] : 0.0f};
}

// The outputs of a row without a token.
__device__ __forceinline__ void put_nothing(const LearnLaunch &a, uint32_t row) {
  a.out_loss[row] = 0.0f;
  if (a.out_logprobs) a.out_logprobs[row] = 0.0f;
  if (a.out_kl) a.out_kl[row] = 0.0f;
  if (a.out_entropy) a.out_entropy[row] = 0.0f;
  if (a.saved) a.saved[row] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
}

// A row's own loss from its sums, every lane alike, and its record; `put`: the
// lane that writes them.
template <bool ENTROPY>
__device__ __forceinline__ LearnedRow clipped_row(const LearnLaunch &a, uint32_t row,
                                                  const RowTerms &terms, const RowSums &total,
                                                  bool put) {
  const double lp = token_logprob(terms.x, total, a.temperature);
  const double A = terms.advantage;
  const double ratio = a.old_logprobs ? exp_of(lp - (double)terms.old).whole : 1.0;
  const double held =
      fmin(fmax(ratio, 1.0 - (double)a.clip_low), 1.0 + (double)a.clip_high);
  // At a bound the ratio is not held back; NaN has neither order.
  const bool stopped = held * A < ratio * A;
  double loss = -(stopped ? held * A : ratio * A), slope = stopped ? 0.0 : -ratio * A;
  if (a.reference) {
    const Exponential grown = exp_of((double)terms.reference - lp);
    if (put && a.out_kl) a.out_kl[row] = (float)grown.over;
    if (a.kl_weight != 0.0f) {
      loss += (double)a.kl_weight * grown.over;
      slope -= (double)a.kl_weight * grown.less;
    }
  }
  const float inv = inverse_sum(total);
  float mean = 0.0f;
  if constexpr (ENTROPY) {
    // A row that leaves nothing has no entropy.
    mean = kLn2 * total.w * inv;
    const float entropy = total.s == 0.0 ? 0.0f : (float)(log_of(total.s) - (double)mean);
    if (put && a.out_entropy) a.out_entropy[row] = entropy;
    if (a.entropy_weight != 0.0f) loss -= (double)a.entropy_weight * (double)entropy;
  }
  const LearnedRow record = make_float4(total.m, inv, (float)slope, mean);
  if (put) {
    // Also where no ratio has made it so: a trainer looks for NaN in its losses.
    a.out_loss[row] = lp != lp ? (float)lp : (float)loss;
    if (a.out_logprobs) a.out_logprobs[row] = (float)lp;
    if (a.saved) a.saved[row] = record;
  }
  return record;
}

// One wave a row.
template <int DT, bool ENTROPY>
__global__ __launch_bounds__(64) void clipped_rows_kernel(LearnLaunch a) {
  const uint32_t row = blockIdx.x, lane = threadIdx.x;
  const MaxSums part = row_part<ENTROPY>(a, row);
  const uint32_t token = a.tokens[row];
  if (token >= a.vocabulary) {
    if (lane == 0) put_nothing(a, row);
    return;
  }
  const RowTerms terms =
      row_terms(a, row, logit_value(row_of<DT>(a.logits, (uint64_t)row * a.stride)[token]));
  const RowSums total = row_sums<ENTROPY>(a, row, part, kLog2e / a.temperature);
  if (lane == 0) clipped_row<ENTROPY>(a, row, terms, total, true);
}

// A pair's row without a token; and the outputs of one with a token, whose distance
// from the reference is returned.
__device__ __forceinline__ void put_no_pair(const LearnLaunch &a, uint32_t row) {
  if (a.out_logprobs) a.out_logprobs[row] = 0.0f;
  a.saved[row] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
}
__device__ __forceinline__ double put_pair_row(const LearnLaunch &a, uint32_t row, float x,
                                               const RowSums &total) {
  const double lp = token_logprob(x, total, a.temperature);
  const double gap = a.reference ? lp - (double)a.reference[row] : lp;
  if (a.out_logprobs) a.out_logprobs[row] = (float)lp;
  // The distance as its bits, in the last two floats, until the pair's block takes it.
  const uint64_t bits = __builtin_bit_cast(uint64_t, gap);
  a.saved[row] = make_float4(total.m, inverse_sum(total), u2f((uint32_t)bits),
                             u2f((uint32_t)(bits >> 32)));
  return gap;
}

// One wave a row.
template <int DT>
__global__ __launch_bounds__(64) void pair_rows_kernel(LearnLaunch a) {
  const uint32_t row = blockIdx.x, lane = threadIdx.x;
  const MaxSums part = row_part<false>(a, row);
  const uint32_t token = a.tokens[row];
  if (token >= a.vocabulary) {
    if (lane == 0) put_no_pair(a, row);
    return;
  }
  const float x = logit_value(row_of<DT>(a.logits, (uint64_t)row * a.stride)[token]);
  const RowSums total = row_sums<false>(a, row, part, kLog2e / a.temperature);
  if (lane == 0) put_pair_row(a, row, x, total);
}

// The same of one row in one thread; whether it has a token.
template <int DT>
__device__ __forceinline__ bool pair_row(const LearnLaunch &a, uint32_t row, double &gap) {
  const uint32_t token = a.tokens[row];
  if (token >= a.vocabulary) {
    put_no_pair(a, row);
    return false;
  }
  const float x = logit_value(row_of<DT>(a.logits, (uint64_t)row * a.stride)[token]);
  const float2 *parts = a.partials + (uint64_t)row * a.segments;
  const float c = kLog2e / a.temperature;
  float m = parts[0].x;
#pragma unroll 8
  for (uint32_t g = 1; g < a.segments; ++g) m = __builtin_fmaxf(m, parts[g].x);
  const float r = finite_reference(m);
  double s = 0.0;
#pragma unroll 8
  for (uint32_t g = 0; g < a.segments; ++g) s += parts[g].y * exp_below(parts[g].x, r, c);
  gap = put_pair_row(a, row, x, RowSums{m, s, 0.0f});
  return true;
}

constexpr uint32_t kPairThreads = 256;

// One block a pair, and one more for the rows of no sequence. ROWS: the rows of a call
// of few are worked out here, a thread each, instead of in a launch of their own before
// (48 rows: 13.9 -> 11.3 us a step).
template <int DT, bool ROWS>
__global__ __launch_bounds__(kPairThreads) void pairs_kernel(PairLaunch a, LearnLaunch l) {
  constexpr uint32_t WAVES = kPairThreads / 64;
  __shared__ double sums[2][WAVES];
  __shared__ uint32_t counts[2][WAVES];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, pair = blockIdx.x;
  if (pair == a.pairs) {
    const uint32_t first = min(a.offsets[0], a.rows);
    const uint32_t last = min(a.offsets[2 * a.pairs], a.rows);
    const auto none = [&](uint32_t r) {
      double gap;
      if (ROWS) pair_row<DT>(l, r, gap);
      a.saved[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    };
    for (uint32_t r = tid; r < first; r += kPairThreads) none(r);
    for (uint32_t r = max(first, last) + tid; r < a.rows; r += kPairThreads) none(r);
    return;
  }
  // Offsets past the rows end there, and a sequence that falls is empty.
  const uint32_t from = min(a.offsets[2 * pair], a.rows);
  const uint32_t middle = min(a.offsets[2 * pair + 1], a.rows);
  const uint32_t to = min(a.offsets[2 * pair + 2], a.rows);
  // Both sequences' rows at once: those of the first, then of the second, also where
  // the two do not follow one another.
  const uint32_t first = from < middle ? middle - from : 0, second = middle < to ? to - middle : 0;
  const auto row_at = [&](uint32_t i) { return i < first ? from + i : middle + (i - first); };
  double own[2] = {0.0, 0.0};
  uint32_t own_count[2] = {0, 0};
  for (uint32_t i = tid; i < first + second; i += kPairThreads) {
    const uint32_t r = row_at(i);
    double gap;
    if constexpr (ROWS) {
      if (!pair_row<DT>(l, r, gap)) continue;
    } else {
      if (a.tokens[r] >= a.vocabulary) continue;
      const float4 v = a.saved[r];
      gap = __builtin_bit_cast(double, (uint64_t)f2u(v.z) | (uint64_t)f2u(v.w) << 32);
    }
    if (i < first) {
      own[0] += gap;
      ++own_count[0];
    } else {
      own[1] += gap;
      ++own_count[1];
    }
  }
#pragma unroll
  for (uint32_t q = 0; q < 2; ++q) {
    const double sum = wave_sum_f64(own[q]);
    const uint32_t count = wave_sum_u32(own_count[q]);
    if (lane == 0) {
      sums[q][wave] = sum;
      counts[q][wave] = count;
    }
  }
  __syncthreads();
  double score[2], share[2];
  uint32_t tokens = 0;
#pragma unroll
  for (uint32_t q = 0; q < 2; ++q) {
    double sum = 0.0;
    uint32_t count = 0;
#pragma unroll
    for (uint32_t w = 0; w < WAVES; ++w) {
      sum += sums[q][w];
      count += counts[q][w];
    }
    share[q] = a.mean && count ? 1.0 / (double)count : 1.0;
    score[q] = sum * share[q];
    tokens += count;
  }
  const double beta = a.beta, u = beta * (score[0] - score[1]) - (double)a.margin;
  double loss, slope;
  if (a.loss == 1) {  // hinge
    loss = u < 1.0 ? 1.0 - u : u != u ? u : 0.0;
    slope = u < 1.0 ? -1.0 : u != u ? u : 0.0;
  } else if (a.loss == 2) {  // squared
    const double d = (u - 0.5) / beta;
    loss = d * d;
    slope = 2.0 * d / beta;
  } else {
    // ln(1 + exp(-u)) and ln(1 + exp(u)), and the logistic function of both.
    const double e = exp_of(-fabs(u)).whole, l = log1_of(e), large = inverse_of(1.0 + e),
                 small = e * large;
    const double smoothing = a.smoothing;
    const double against = (u > 0.0 ? 0.0 : -u) + l, with = (u > 0.0 ? u : 0.0) + l;
    const double fall = u > 0.0 ? small : large, rise = u > 0.0 ? large : small;
    loss = slope = 0.0;
    if (smoothing != 1.0) {
      loss += (1.0 - smoothing) * against;
      slope -= (1.0 - smoothing) * fall;
    }
    if (smoothing != 0.0) {
      loss += smoothing * with;
      slope += smoothing * rise;
    }
  }
  if (tid == 0) {
    a.out_loss[pair] = tokens ? (float)loss : 0.0f;
    if (a.out_scores) {
      a.out_scores[2 * pair] = (float)score[0];
      a.out_scores[2 * pair + 1] = (float)score[1];
    }
  }
  const float up = (float)(beta * slope * share[0]), down = (float)(-beta * slope * share[1]);
  for (uint32_t i = tid; i < first + second; i += kPairThreads) {
    const uint32_t r = row_at(i);
    if (a.tokens[r] >= a.vocabulary) continue;
    float *v = (float *)(a.saved + r);
    v[2] = i < first ? up : down;
    v[3] = u2f(pair);
  }
}

// A row's gradient by its record and its loss's gradient.
template <bool ENTROPY>
struct Slopes {
  float m, c, share, flat, steep;
  bool any;  // of the row's tokens but its own

  __device__ __forceinline__ Slopes(const LearnedRow &r, float scale, float c, float entropy_weight)
      : m(r.x), c(c), share(scale * r.z) {
    const float weight = scale * r.y;
    // A loss that nothing follows from has no gradient, also where its row's sum is NaN.
    any = scale != 0.0f && weight != 0.0f;
    // p_j (h (t_j - E) - G) as e_j (flat + steep u_j), u_j the exponents of 2.
    flat = ENTROPY ? -weight * (r.z + entropy_weight * r.w) : -share * r.y;
    steep = ENTROPY ? weight * entropy_weight * kLn2 : 0.0f;
  }
  __device__ __forceinline__ float operator()(float x) const {
    const float u = (x - m) * c, p = __builtin_amdgcn_exp2f(u);
    // The exponent by its exponential first, which leaves the range less than its
    // product with the weights would.
    return ENTROPY ? __builtin_fmaf(p * bounded(u), steep, p * flat) : p * flat;
  }
};

// A vector of a row's gradient; `token` is the row's from the vector's first on.
template <int DT, bool ENTROPY>
__device__ __forceinline__ LogitWords gradient(const Slopes<ENTROPY> &s, const LogitWords &w,
                                               uint32_t token) {
  constexpr uint32_t VEC = Logits<DT>::VEC;
  float v[VEC];
  if (s.any) {
    unpack<DT>(w, v);
#pragma unroll
    for (uint32_t e = 0; e < VEC; ++e) v[e] = s(v[e]);
  } else {
#pragma unroll
    for (uint32_t e = 0; e < VEC; ++e) v[e] = 0.0f;
  }
  if (token < VEC) {
#pragma unroll
    for (uint32_t e = 0; e < VEC; ++e)
      if (token == e) v[e] += s.share;
  }
  return pack<DT>(v);
}

// Losses and gradients of whole rows, a block each. 512 threads: two blocks on a CU, of
// which one reads while the other computes or writes. 1024: one, which holds twice as
// much of its row. Some quads of vectors a thread stay in registers from the first pass
// to the second, the rest is read again through the caches. Vectors count from the
// gradient's last line before the row (see jf_distill.hip).
//
// SHARED: few rows leave most CUs idle. Several blocks then take a row's sums, each all of
// them, and write the gradient's vectors by turns, the first block the row's numbers too
// (16 f32 rows x 32,000 7.6 -> 6.8 us, one with entropies 9.0 -> 7.2). A kernel of its own:
// the turns cost one of many rows 3%.
constexpr uint32_t kQuad = 4;  // vectors a thread loads, adds and stores together
constexpr uint32_t kHeld = 3;  // of them held: what the registers take

template <int DT, bool ENTROPY, uint32_t THREADS, bool SHARED>
__global__ __launch_bounds__(THREADS, 4) void clipped_step_kernel(LearnLaunch a,
                                                                  LearnGradLaunch g) {
  constexpr uint32_t VEC = Logits<DT>::VEC, SLAB = THREADS * VEC, QUAD = kQuad * SLAB,
                     HELD = kHeld, WAVES = THREADS / 64;
  using Words = typename Logits<DT>::Words;
  __shared__ MaxSums part[WAVES];
  const uint32_t tid = threadIdx.x, wave = tid >> 6, lane = tid & 63u;
  const uint32_t blocks = SHARED ? g.blocks : 1;
  const uint32_t row = blockIdx.x >> __builtin_ctz(blocks), block = blockIdx.x & (blocks - 1);
  const uint32_t token = a.tokens[row];
  const auto *logits = row_of<DT>(a.logits, (uint64_t)row * a.stride);
  auto *grad = row_of<DT>(g.grad, (uint64_t)row * g.grad_stride);
  const uint32_t before = (uint32_t)((uintptr_t)grad % 128 / sizeof(*grad));
  const auto *z = logits - before;
  auto *dz = grad - before;
  const uint32_t V = before + a.vocabulary, quads = V / QUAD;
  const auto put = [&](uint32_t at, const LogitWords &d) {
    if (at >= before && at + VEC <= V)
      __builtin_nontemporal_store(d, (Words *)(dz + at));
    else if (at < V)
      store_words<DT>(dz, at, V, d, before);
  };
  if (token >= a.vocabulary) {
    // Every wave has the token before the row's numbers are written, which may take its
    // place: a wave that found 0 there would learn from the row.
    __syncthreads();
    if (tid == 0 && block == 0) put_nothing(a, row);
    const LogitWords zero{};
    for (uint32_t at = block * SLAB + tid * VEC; at < V; at += blocks * SLAB) put(at, zero);
    return;
  }
  const auto load = [&](uint32_t quad, LogitWords (&w)[kQuad]) {
#pragma unroll
    for (uint32_t j = 0; j < kQuad; ++j)
      w[j] = *(const Words *)(z + quad * QUAD + j * SLAB + tid * VEC);
  };
  // `rest`: the vectors past the last whole quad.
  LogitWords held[HELD][kQuad], rest[kQuad];
#pragma unroll
  for (uint32_t q = 0; q < HELD; ++q) {
    if (q >= quads) break;
    if (q == 0 && tid * VEC < before) {
      // The row's first line: the first vectors of its first wave.
      held[0][0] = load_words<DT>(z, tid * VEC, V, kPastMinusInfinity<DT>, before);
#pragma unroll
      for (uint32_t j = 1; j < kQuad; ++j)
        held[0][j] = *(const Words *)(z + j * SLAB + tid * VEC);
    } else {
      load(q, held[q]);
    }
  }
#pragma unroll
  for (uint32_t j = 0; j < kQuad; ++j)
    rest[j] = load_words<DT>(z, quads * QUAD + j * SLAB + tid * VEC, V, kPastMinusInfinity<DT>,
                             before);
  RowTerms terms = row_terms(a, row, logit_value(logits[token]));
  float loss_gradient = g.grad_loss[(uint64_t)row * g.grad_loss_stride];
  const float c = kLog2e / a.temperature;
  MaxSums run{-__builtin_inff(), 0.0f, 0.0f};
  const auto add = [&](const LogitWords (&w)[kQuad]) {
    float grown = run.m;
#pragma unroll
    for (uint32_t j = 0; j < kQuad; ++j) grown = loaded_max(grown, vector_max<DT>(w[j]));
    const float r = finite_reference(grown);
    run = from(run, r, c);
    run.m = grown;
    add_vectors<DT, ENTROPY, true>(run, w, r, c);
  };
  // What is not held is on its way beside the sums (1000 f32 rows x 64,000 107 -> 101 us, 1024
  // x 151,936 265 -> 259), where the registers take that: not beside unpacked bf16.
  constexpr bool AHEAD = DT == 0;
  LogitWords next[kQuad];
  if (AHEAD && HELD < quads) load(HELD, next);
  if (AHEAD) add(rest);
#pragma unroll
  for (uint32_t q = 0; q < HELD; ++q)
    if (q < quads) add(held[q]);
  for (uint32_t q = HELD; q < quads; ++q) {
    LogitWords w[kQuad];
    if constexpr (AHEAD) {
#pragma unroll
      for (uint32_t j = 0; j < kQuad; ++j) w[j] = next[j];
      if (q + 1 < quads) load(q + 1, next);
    } else {
      load(q, w);
    }
    add(w);
  }
  if (!AHEAD) add(rest);
  run = wave_join<ENTROPY>(run, c);
  if (lane == 0) part[wave] = run;
  // What the row takes is here before any wave writes its gradient or its numbers, in
  // whose place some of it may be.
  asm volatile("" : "+v"(terms.x), "+v"(terms.advantage), "+v"(terms.old), "+v"(terms.reference));
  asm volatile("" : "+v"(loss_gradient));
  __syncthreads();
  // The held words anew, or the compiler keeps the values it unpacked above, two
  // registers a word.
#pragma unroll
  for (uint32_t q = 0; q < HELD; ++q)
#pragma unroll
    for (uint32_t j = 0; j < kQuad; ++j) asm volatile("" : "+v"(held[q][j]));
  const RowSums total = whole<ENTROPY>(
      lane < WAVES ? part[lane] : MaxSums{-__builtin_inff(), 0.0f, 0.0f}, c);
  const LearnedRow record = clipped_row<ENTROPY>(a, row, terms, total, tid == 0 && block == 0);
  // A loss without a slope, also where only its entropy is asked for.
  const bool sloped = record.z != 0.0f || (ENTROPY && a.entropy_weight != 0.0f);
  const float scale = sloped ? loss_gradient / a.temperature : 0.0f;
  const Slopes<ENTROPY> slopes(record, scale, c, a.entropy_weight);
  const uint32_t at_token = scale != 0.0f ? token + before : 0xffffffffu;
  // Whether a vector is the block's to write.
  const auto own = [&](uint32_t quad, uint32_t j) {
    return !SHARED || ((quad * kQuad + j) & (blocks - 1)) == block;
  };
  const auto put_quad = [&](uint32_t quad, const LogitWords (&w)[kQuad]) {
#pragma unroll
    for (uint32_t j = 0; j < kQuad; ++j) {
      if (!own(quad, j)) continue;
      const uint32_t at = quad * QUAD + j * SLAB + tid * VEC;
      put(at, gradient<DT>(slopes, w[j], at_token - at));
    }
  };
  // The quads read again come first, the last read before the others.
  for (uint32_t q = quads; q-- > HELD;) {
    LogitWords w[kQuad];
#pragma unroll
    for (uint32_t j = 0; j < kQuad; ++j)
      if (own(q, j)) w[j] = *(const Words *)(z + q * QUAD + j * SLAB + tid * VEC);
    put_quad(q, w);
  }
#pragma unroll
  for (uint32_t q = 0; q < HELD; ++q)
    if (q < quads) put_quad(q, held[q]);
  put_quad(quads, rest);
}

// The forward pass of whole rows, a block each: a quad of vectors a thread is added while
// the next is on its way, which takes a row faster than its chunks' sums and a launch that
// joins them (losses of 4096 bf16 rows x 32,000 58.3 -> 48.5 us, of 512 x 100,003, a third
// without a token, 21.2 -> 20.1, of 16 f32 rows x 32,000 7.5 -> 6.2). PAIRS: the rows are
// those of pairs of sequences. Vectors count from the last line before the row.
template <int DT, bool ENTROPY, bool PAIRS, uint32_t THREADS>
__global__ __launch_bounds__(THREADS, 6) void learn_rows_kernel(LearnLaunch a) {
  constexpr uint32_t VEC = Logits<DT>::VEC, SLAB = THREADS * VEC, QUAD = kQuad * SLAB,
                     WAVES = THREADS / 64;
  using Words = typename Logits<DT>::Words;
  __shared__ MaxSums part[WAVES];
  const uint32_t tid = threadIdx.x, wave = tid >> 6, lane = tid & 63u, row = blockIdx.x;
  const uint32_t token = a.tokens[row];
  if (token >= a.vocabulary) {
    // As in a step: every wave has the token before the row's numbers may take its place.
    __syncthreads();
    if (tid) return;
    if constexpr (PAIRS)
      put_no_pair(a, row);
    else
      put_nothing(a, row);
    return;
  }
  const auto *logits = row_of<DT>(a.logits, (uint64_t)row * a.stride);
  const uint32_t before = (uint32_t)((uintptr_t)logits % 128 / sizeof(*logits));
  const auto *z = logits - before;
  const uint32_t V = before + a.vocabulary, quads = V / QUAD;
  // The vectors past the last whole quad, two at a time where there are any. They are the
  // first to be added: behind the others they would have nothing on its way beside them.
  LogitWords rest[kQuad], next[kQuad];
  const auto load_end = [&](uint32_t at) {
    return load_words<DT>(z, at, V, kPastMinusInfinity<DT>, before);
  };
#pragma unroll
  for (uint32_t j = 0; j < kQuad; ++j)
    if (quads * QUAD + j / 2 * 2 * SLAB < V)
      rest[j] = load_end(quads * QUAD + j * SLAB + tid * VEC);
  const auto load = [&](uint32_t quad) {
#pragma unroll
    for (uint32_t j = 0; j < kQuad; ++j)
      next[j] = *(const Words *)(z + quad * QUAD + j * SLAB + tid * VEC);
  };
  if (quads && tid * VEC < before) {
    // The row's first line: the first vectors of its first wave.
    next[0] = load_end(tid * VEC);
#pragma unroll
    for (uint32_t j = 1; j < kQuad; ++j) next[j] = *(const Words *)(z + j * SLAB + tid * VEC);
  } else if (quads) {
    load(0);
  }
  const float x = logit_value(logits[token]);
  RowTerms terms{x, 0.0f, 0.0f, 0.0f};
  if constexpr (!PAIRS) terms = row_terms(a, row, x);
  const float c = kLog2e / a.temperature;
  MaxSums run{-__builtin_inff(), 0.0f, 0.0f};
  const auto add = [&]<uint32_t N>(const LogitWords(&w)[N]) {
    float grown = run.m;
#pragma unroll
    for (uint32_t j = 0; j < N; ++j) grown = loaded_max(grown, vector_max<DT>(w[j]));
    const float r = finite_reference(grown);
    run = from(run, r, c);
    run.m = grown;
    // Every exponent bounded: beside the next quad there are no registers for a second try
    // (4096 bf16 rows x 32,000 with entropies 53 us, 57 with one).
    add_vectors<DT, ENTROPY, true>(run, w, r, c);
  };
#pragma unroll
  for (uint32_t j = 0; j < kQuad; j += 2) {
    if (quads * QUAD + j * SLAB >= V) break;
    const LogitWords w[2] = {rest[j], rest[j + 1]};
    add(w);
  }
#pragma unroll 1
  for (uint32_t q = 0; q < quads; ++q) {
    LogitWords w[kQuad];
#pragma unroll
    for (uint32_t j = 0; j < kQuad; ++j) w[j] = next[j];
    if (q + 1 < quads) load(q + 1);
    add(w);
  }
  run = wave_join<ENTROPY>(run, c);
  if (lane == 0) part[wave] = run;
  // What the row takes is here before any number of its is written, in whose place some
  // of it may be.
  asm volatile("" : "+v"(terms.x), "+v"(terms.advantage), "+v"(terms.old), "+v"(terms.reference));
  __syncthreads();
  if (wave) return;
  const RowSums total = whole<ENTROPY>(
      lane < WAVES ? part[lane] : MaxSums{-__builtin_inff(), 0.0f, 0.0f}, c);
  if (lane) return;
  if constexpr (PAIRS)
    put_pair_row(a, row, terms.x, total);
  else
    clipped_row<ENTROPY>(a, row, terms, total, true);
}

// Bytes of rows from which the last cache (256 MB) holds part of them only.
constexpr uint64_t kLastCache = 300ull << 20;

// The gradient of a chunk of a row. LINES: chunks count from the gradient's last
// line before the row, for rows that start within one (see jf_distill.hip). OWN: a step's
// rows by chunks, whose sums each wave of each block joins for itself, in place of a launch
// between (one f32 row x 100,003 11.3 -> 7.7 us).
template <int DT, uint32_t N, bool LINES, bool ENTROPY, bool OWN>
__global__ __launch_bounds__(256) void learn_grad_kernel(LearnGradLaunch a, LearnLaunch l) {
  constexpr uint32_t VEC = Logits<DT>::VEC, SLAB = kSlab<DT>, CHUNK = N * SLAB;
  const uint32_t tid = threadIdx.x;
  // From the last row on where the rows do not fit the last cache: the forward pass has
  // left the last ones there (2000 bf16 rows x 151,936, both passes: 259 us, 284 from the
  // first row on).
  const uint32_t block = a.backwards ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
  const uint32_t row = block / a.chunks, chunk = block - row * a.chunks;
  const uint32_t base = chunk * CHUNK;
  const auto *z = row_of<DT>(a.logits, (uint64_t)row * a.stride);
  auto *dz = row_of<DT>(a.grad, (uint64_t)row * a.grad_stride);
  const uint32_t before = LINES ? (uint32_t)((uintptr_t)dz % 128 / sizeof(*dz)) : 0;
  const uint32_t V = before + a.vocabulary;
  if (LINES && base >= V) return;  // not every row reaches the last chunk
  z -= before;
  dz -= before;
  LearnedRow saved{};
  if constexpr (!OWN) saved = a.saved[row];
  const uint32_t token = a.tokens[row];
  // A row without a token has no slope, and no gradient whatever the losses'.
  const bool learned = token < a.vocabulary && (OWN || ENTROPY || saved.z != 0.0f);
  LogitWords w[N];
  if (learned) load_chunk<DT>(z, base, V, 0, w, before);
  float scale = 0.0f;
  if constexpr (OWN) {
    const bool put = chunk == 0 && tid == 0;
    if (learned) {
      const MaxSums part = row_part<ENTROPY>(l, row);
      const RowTerms terms = row_terms(l, row, logit_value(z[before + token]));
      const float loss_gradient = a.grad_loss[(uint64_t)row * a.grad_loss_stride];
      const RowSums total = row_sums<ENTROPY>(l, row, part, kLog2e / a.temperature);
      saved = clipped_row<ENTROPY>(l, row, terms, total, put);
      // As a step of whole rows.
      const bool sloped = saved.z != 0.0f || (ENTROPY && a.entropy_weight != 0.0f);
      scale = sloped ? loss_gradient / a.temperature : 0.0f;
    } else if (put) {
      put_nothing(l, row);
    }
  } else if (learned) {
    const uint32_t loss = a.pairs ? f2u(saved.w) : row;
    if (!a.pairs || loss < a.pairs)
      scale = a.grad_loss[(uint64_t)loss * a.grad_loss_stride] / a.temperature;
  }
  const Slopes<ENTROPY> slopes(saved, scale, kLog2e / a.temperature, a.entropy_weight);
  const uint32_t at_token = scale != 0.0f ? token + before : 0xffffffffu;
#pragma unroll
  for (uint32_t j = 0; j < N; ++j) {
    const uint32_t at = base + j * SLAB + tid * VEC;
    if (at >= V) continue;
    const LogitWords d = gradient<DT>(slopes, w[j], at_token - at);
    if (at >= before && at + VEC <= V)
      __builtin_nontemporal_store(d, (typename Logits<DT>::Words *)(dz + at));
    else
      store_words<DT>(dz, at, V, d, before);
  }
}

}  // namespace

int launch_learn_score(const LearnLaunch &a, uint32_t dtype, void *stream) {
  const dim3 grid(a.row_count * a.segments), block(256);
  const hipStream_t st = (hipStream_t)stream;
  const bool entropy = a.entropy != 0;
#define JF_LEARN(DT, N, ENTROPY)                              \
  if (dtype == DT && a.vectors == N && entropy == ENTROPY)    \
  hipLaunchKernelGGL((learn_score_kernel<DT, N, ENTROPY>), grid, block, 0, st, a)
  JF_LEARN(0, 2, false);
  JF_LEARN(0, 2, true);
  JF_LEARN(0, 4, false);
  JF_LEARN(0, 4, true);
  JF_LEARN(0, 8, false);
  JF_LEARN(0, 8, true);
  JF_LEARN(1, 2, false);
  JF_LEARN(1, 2, true);
  JF_LEARN(1, 4, false);
  JF_LEARN(1, 4, true);
#undef JF_LEARN
  return (int)hipGetLastError();
}

int launch_clipped_rows(const LearnLaunch &a, uint32_t dtype, void *stream) {
  const dim3 rows(a.row_count), block(64);
  const hipStream_t st = (hipStream_t)stream;
  const bool entropy = a.entropy != 0;
  if (dtype == 0 && entropy)
    hipLaunchKernelGGL((clipped_rows_kernel<0, true>), rows, block, 0, st, a);
  else if (dtype == 0)
    hipLaunchKernelGGL((clipped_rows_kernel<0, false>), rows, block, 0, st, a);
  else if (entropy)
    hipLaunchKernelGGL((clipped_rows_kernel<1, true>), rows, block, 0, st, a);
  else
    hipLaunchKernelGGL((clipped_rows_kernel<1, false>), rows, block, 0, st, a);
  return (int)hipGetLastError();
}

int launch_learn_rows(const LearnLaunch &a, bool pairs, uint32_t dtype, uint32_t threads,
                      void *stream) {
  const dim3 rows(a.row_count), block(threads);
  const hipStream_t st = (hipStream_t)stream;
  const bool entropy = a.entropy != 0;
#define JF_ROWS(DT, ENTROPY, PAIRS)                                                            \
  if (dtype == DT && entropy == ENTROPY && pairs == PAIRS && threads == 256)                   \
    hipLaunchKernelGGL((learn_rows_kernel<DT, ENTROPY, PAIRS, 256>), rows, block, 0, st, a);   \
  if (dtype == DT && entropy == ENTROPY && pairs == PAIRS && threads == 512)                   \
  hipLaunchKernelGGL((learn_rows_kernel<DT, ENTROPY, PAIRS, 512>), rows, block, 0, st, a)
  JF_ROWS(0, false, false);
  JF_ROWS(0, true, false);
  JF_ROWS(0, false, true);
  JF_ROWS(1, false, false);
  JF_ROWS(1, true, false);
  JF_ROWS(1, false, true);
#undef JF_ROWS
  return (int)hipGetLastError();
}

int launch_clipped_step(const LearnLaunch &a, const LearnGradLaunch &g, uint32_t dtype,
                        uint32_t threads, void *stream) {
  const dim3 rows(a.row_count * g.blocks), block(threads);
  const hipStream_t st = (hipStream_t)stream;
  const bool entropy = a.entropy != 0;
#define JF_STEP(DT, ENTROPY, THREADS, SHARED)                                              \
  if (dtype == DT && entropy == ENTROPY && threads == THREADS && (g.blocks > 1) == SHARED) \
  hipLaunchKernelGGL((clipped_step_kernel<DT, ENTROPY, THREADS, SHARED>), rows, block, 0, st, a, g)
  JF_STEP(0, false, 512, false);
  JF_STEP(0, true, 512, false);
  JF_STEP(1, false, 512, false);
  JF_STEP(1, true, 512, false);
  JF_STEP(0, false, 512, true);
  JF_STEP(0, true, 512, true);
  JF_STEP(1, false, 512, true);
  JF_STEP(1, true, 512, true);
  JF_STEP(0, false, 1024, false);
  JF_STEP(0, true, 1024, false);
  JF_STEP(1, false, 1024, false);
  JF_STEP(1, true, 1024, false);
#undef JF_STEP
  return (int)hipGetLastError();
}

int launch_pair_rows(const LearnLaunch &a, uint32_t dtype, void *stream) {
  const dim3 rows(a.row_count), block(64);
  if (dtype == 0)
    hipLaunchKernelGGL((pair_rows_kernel<0>), rows, block, 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL((pair_rows_kernel<1>), rows, block, 0, (hipStream_t)stream, a);
  return (int)hipGetLastError();
}

int launch_pairs(const PairLaunch &a, const LearnLaunch &rows, bool with_rows, uint32_t dtype,
                 void *stream) {
  const dim3 grid(a.pairs + 1), block(kPairThreads);
  const hipStream_t st = (hipStream_t)stream;
  if (!with_rows)
    hipLaunchKernelGGL((pairs_kernel<0, false>), grid, block, 0, st, a, rows);
  else if (dtype == 0)
    hipLaunchKernelGGL((pairs_kernel<0, true>), grid, block, 0, st, a, rows);
  else
    hipLaunchKernelGGL((pairs_kernel<1, true>), grid, block, 0, st, a, rows);
  return (int)hipGetLastError();
}

int launch_learn_grad(const LearnGradLaunch &rows, const LearnLaunch *own, uint32_t dtype,
                      void *stream) {
  LearnGradLaunch a = rows;
  const uint32_t size = dtype == 0 ? 4 : 2, chunk = chunk_tokens(dtype, a.vectors);
  // Rows that start within a line may reach a chunk more.
  const bool lines = (uintptr_t)a.grad % 128 != 0 ||
                     (a.row_count > 1 && a.grad_stride * size % 128 != 0);
  a.chunks = (a.vocabulary + (lines ? 128 / size - 1 : 0) + chunk - 1) / chunk;
  a.backwards = (uint64_t)a.row_count * a.vocabulary * size > kLastCache ? 1u : 0u;
  const dim3 grid(a.row_count * a.chunks), block(256);
  const hipStream_t st = (hipStream_t)stream;
  const bool entropy = own ? own->entropy != 0 : a.entropy_weight != 0.0f;
  const LearnLaunch l = own ? *own : LearnLaunch{};
#define JF_GRAD(DT, N, LINES, ENTROPY)                                                        \
  if (dtype == DT && a.vectors == N && lines == LINES && entropy == ENTROPY && own)           \
    hipLaunchKernelGGL((learn_grad_kernel<DT, N, LINES, ENTROPY, true>), grid, block, 0, st, a, l); \
  if (dtype == DT && a.vectors == N && lines == LINES && entropy == ENTROPY && !own)          \
  hipLaunchKernelGGL((learn_grad_kernel<DT, N, LINES, ENTROPY, false>), grid, block, 0, st, a, l)
#define JF_GRADS(DT, N)         \
  JF_GRAD(DT, N, false, false); \
  JF_GRAD(DT, N, false, true);  \
  JF_GRAD(DT, N, true, false);  \
  JF_GRAD(DT, N, true, true)
  JF_GRADS(0, 2);
  JF_GRADS(0, 4);
  JF_GRADS(1, 2);
  JF_GRADS(1, 4);
#undef JF_GRADS
#undef JF_GRAD
  return (int)hipGetLastError();
}

}  // namespace jf
