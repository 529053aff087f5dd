// Log-probabilities and the distillation's forward pass on gfx950: one pass
// over a row's logits for its maximum m and s = sum exp((x - m) / T), then a
// finish over a few words of the row.
//
// The pass. A block takes a segment of a row, a chunk of 8192 tokens at a time
// in registers. A thread holds 32 values of a chunk, takes their maximum and
// adds their exponentials against its running one (rescaled when it grows);
// waves and then the block join theirs. The row's first token's rank needs
// only its logit, read up front: a count of the values ahead of it.
//
// The best tokens without a second pass. The pass also keeps the maximum of
// every group of 64 consecutive tokens. The k best tokens of a row, in the
// order (logit down, id up), lie in its k best groups, ordered by (maximum
// down, group up): a token in a group behind k others has k group maxima ahead
// of it, ties included, since ids of an earlier group are lower. So the finish
// reads 1/64 of the row in maxima, and then k groups.
#include <hip/hip_runtime.h>

#include "jf_logits.h"

namespace jf {

namespace {

constexpr float kLog2e = 1.44269504088896341f;

// A row's temperature: the sampler's 0 (a greedy row) and anything that is no
// temperature leave the logits as they are.
__device__ __forceinline__ float inverse_temperature(const ScoreLaunch &a, uint32_t row) {
  const float t = a.temperatures ? a.temperatures[row] : a.temperature;
  return t >= __FLT_MIN__ && t < __builtin_inff() ? 1.0f / t : 1.0f;
}

// A running maximum and sum of exponentials. Nothing yet, or nothing but
// -infinity: m = -infinity, s = 0. A NaN, or +infinity, makes s NaN for good.
struct MaxSum {
  float m, s;
};
// exp((x - m) / T) with c = log2(e) / T; m is at least x, and not -infinity.
__device__ __forceinline__ float exp_below(float x, float m, float c) {
  return __builtin_amdgcn_exp2f((x - m) * c);
}
__device__ __forceinline__ float finite_reference(float m) {
  return m == -__builtin_inff() ? 0.0f : m;
}
__device__ __forceinline__ MaxSum join(MaxSum p, MaxSum q, float c) {
  const float m = __builtin_fmaxf(p.m, q.m), r = finite_reference(m);
  return {m, p.s * exp_below(p.m, r, c) + q.s * exp_below(q.m, r, c)};
}
template <int M>
__device__ __forceinline__ MaxSum join_xor(MaxSum p, float c) {
  return join(p, MaxSum{xor_f32<M>(p.m), xor_f32<M>(p.s)}, c);
}
__device__ __forceinline__ MaxSum wave_join(MaxSum p, float c) {
  const float m = wave_max_f32(p.m);
  float s = p.s * exp_below(p.m, finite_reference(m), c);
  s += xor_f32<1>(s);
  s += xor_f32<2>(s);
  s += xor_f32<4>(s);
  s += xor_f32<8>(s);
  s += xor_f32<16>(s);
  s += xor_f32<32>(s);
  return {m, s};
}

// The least float above x; a NaN, which nothing reaches, above +infinity and
// NaN.
__device__ __forceinline__ float next_up(float x) {
  if (!(x < __builtin_inff())) return __builtin_nanf("");
  const uint32_t u = f2u(x);
  return u2f((u << 1) == 0 ? 1u : (u & 0x80000000u) ? u - 1 : u + 1);
}

// A logit's place in the order of alternatives: larger first; 0 for tokens
// that are never listed (-infinity and NaN).
__device__ __forceinline__ uint32_t listed_key(float x) {
  return x > -__builtin_inff() ? logit_key(x) : 0u;
}

template <int DT, bool TOP, bool RANK>
__global__ __launch_bounds__(256) void score_kernel(ScoreLaunch a) {
  constexpr uint32_t VEC = Logits<DT>::VEC, SLAB = kSlab<DT>, LOADS = kLoads<DT>;
  __shared__ MaxSum wave_part[4];
  __shared__ uint32_t wave_ahead[4];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  const uint32_t row = blockIdx.x / a.segments, segment = blockIdx.x - row * a.segments;
  const uint32_t V = a.vocabulary;
  const auto *x = row_of<DT>(a.logits, (uint64_t)row * a.stride);
  const float c = inverse_temperature(a, row) * kLog2e;
  uint32_t target = 0xffffffffu;
  float at_target = 0.0f, above_target = 0.0f;
  uint32_t ahead = 0;
  if constexpr (RANK) {
    target = a.tokens[(uint64_t)row * a.token_stride];
    if (target < V) {
      at_target = logit_value(x[target]);
      above_target = next_up(at_target);
    }
  }
  MaxSum run{-__builtin_inff(), 0.0f};
  const uint32_t first = segment * a.segment_chunks;
  const uint32_t last = min(first + a.segment_chunks, (V + kScoreChunk - 1) / kScoreChunk);
  for (uint32_t chunk = first; chunk < last; ++chunk) {
    const uint32_t base = chunk * kScoreChunk;
    LogitWords w[LOADS];
    if (base + kScoreChunk <= V) {
#pragma unroll
      for (uint32_t j = 0; j < LOADS; ++j)
        w[j] = *(const typename Logits<DT>::Words *)(x + base + j * SLAB + tid * VEC);
    } else {
#pragma unroll
      for (uint32_t j = 0; j < LOADS; ++j)
        w[j] = load_words<DT>(x, base + j * SLAB + tid * VEC, V, kPastMinusInfinity<DT>);
    }
    float part[LOADS], m = -__builtin_inff();
#pragma unroll
    for (uint32_t j = 0; j < LOADS; ++j) {
      float v[VEC];
      unpack<DT>(w[j], v);
      part[j] = v[0];
#pragma unroll
      for (uint32_t e = 1; e < VEC; ++e) part[j] = __builtin_fmaxf(part[j], v[e]);
      m = __builtin_fmaxf(m, part[j]);
    }
    // A NaN maximum: every value of the thread is NaN.
    const float grown = __builtin_fmaxf(run.m, m), r = finite_reference(grown);
    float s = run.s * exp_below(run.m, r, c);
#pragma unroll
    for (uint32_t j = 0; j < LOADS; ++j) {
      float v[VEC];
      unpack<DT>(w[j], v);
#pragma unroll
      for (uint32_t e = 0; e < VEC; ++e) s += exp_below(v[e], r, c);
    }
    run = {grown, s};
    if constexpr (RANK) {
      if (target < V) {
        // Ids before the target's are ahead of it at equal logits too.
        const bool mixed = target - base < kScoreChunk;
        const float least = base < target ? at_target : above_target;
#pragma unroll
        for (uint32_t j = 0; j < LOADS; ++j) {
          float v[VEC];
          unpack<DT>(w[j], v);
#pragma unroll
          for (uint32_t e = 0; e < VEC; ++e) {
            const float from =
                mixed && base + j * SLAB + tid * VEC + e >= target ? above_target : least;
            ahead += v[e] >= from ? 1u : 0u;
          }
        }
      }
    }
    if constexpr (TOP) {
      // A group's 64 tokens lie in 16 (f32) or 8 (bf16) neighbouring lanes.
      float *maxima = a.maxima + (uint64_t)row * a.groups + chunk * kScoreChunkGroups;
#pragma unroll
      for (uint32_t j = 0; j < LOADS; ++j) {
        float g = part[j];
        g = __builtin_fmaxf(g, xor_f32<1>(g));
        g = __builtin_fmaxf(g, xor_f32<2>(g));
        g = __builtin_fmaxf(g, xor_f32<4>(g));
        if constexpr (DT == 0) g = __builtin_fmaxf(g, xor_f32<8>(g));
        if (tid % (kScoreGroup / VEC) == 0)
          maxima[(j * SLAB + tid * VEC) / kScoreGroup] = g;
      }
    }
  }
  run = wave_join(run, c);
  if constexpr (RANK) ahead = wave_sum_u32(ahead);
  if (lane == 0) {
    wave_part[wave] = run;
    wave_ahead[wave] = ahead;
  }
  __syncthreads();
  if (tid == 0) {
    const MaxSum all = join(join(wave_part[0], wave_part[1], c),
                            join(wave_part[2], wave_part[3], c), c);
    const uint64_t at = (uint64_t)row * a.segments + segment;
    a.partials[at] = make_float2(all.m, all.s);
    if constexpr (RANK)
      a.aheads[at] = wave_ahead[0] + wave_ahead[1] + wave_ahead[2] + wave_ahead[3];
  }
}

// ---- finish -----------------------------------------------------------------

// The row's maximum and sum from its segments' (every lane of the wave gets
// them). A row has at most 64 segments.
__device__ __forceinline__ MaxSum row_total(const ScoreLaunch &a, uint32_t row, float c) {
  MaxSum p{-__builtin_inff(), 0.0f};
  const uint32_t lane = threadIdx.x & 63u;
  if (lane < a.segments) {
    const float2 v = a.partials[(uint64_t)row * a.segments + lane];
    p = {v.x, v.y};
  }
  return wave_join(p, c);
}

// A row's totals as its outputs take them.
struct RowScore {
  float m, inv_t, log_sum;
  __device__ __forceinline__ float logprob(float x) const {
    // No token: -infinity has no probability, whatever the row.
    return x == -__builtin_inff() ? x : (x - m) * inv_t - log_sum;
  }
  __device__ __forceinline__ float lse() const {
    // ln 0: the row leaves nothing (a row of NaN has one for its sum).
    return log_sum == -__builtin_inff() ? log_sum : m * inv_t + log_sum;
  }
};

constexpr uint32_t kMostItems = 32;  // groups, and then tokens, a thread holds at most

struct TopLds {
  uint4 key[64];  // the threads' best keys
  uint32_t list_key[kMostItems * (kTopLogprobs - 1) + 1];
  uint32_t list_id[kMostItems * (kTopLogprobs - 1) + 1];
  uint32_t best[kTopLogprobs];
  uint32_t bound_key, bound_id, ahead, ties, count;
};

// Lists in LDS, in no order, the block's items at or ahead of the k-th of its
// threads' best items, in the order (key down, id up); key 0 is no item, and
// with fewer than k threads that have an item every one is listed. So the list
// holds the block's k best items. An item on it belongs to one of those k
// threads, the k-th of which has no other one there: at most
// (k - 1) * kMostItems + 1 items. Returns their number.
template <uint32_t N>
__device__ __forceinline__ uint32_t list_best(TopLds &s, uint32_t k, const uint32_t (&key)[N],
                                              const uint32_t (&id)[N]) {
  static_assert(N <= kMostItems);
  const uint32_t tid = threadIdx.x;
  uint32_t best = 0, best_id = 0;
#pragma unroll
  for (uint32_t i = 0; i < N; ++i)
    if (key[i] > best || (key[i] == best && key[i] && id[i] < best_id)) {
      best = key[i];
      best_id = id[i];
    }
  __syncthreads();  // what an earlier call left has been read
  ((uint32_t *)s.key)[tid] = best;
  if (tid == 0) {
    s.bound_key = 0xffffffffu;
    s.bound_id = 0;
    s.ties = s.count = 0;
  }
  const uint32_t threads = (uint32_t)__syncthreads_count(best != 0);
  uint32_t bound_key = 1, bound_id = 0xffffffffu;  // everything
  if (threads >= k) {
    uint32_t ahead = 0;
    for (uint32_t t = 0; t < 64; ++t) {
      const uint4 other = s.key[t];
      ahead += other.x > best;
      ahead += other.y > best;
      ahead += other.z > best;
      ahead += other.w > best;
    }
    // The k-th best key is the least with fewer than k ahead of it.
    if (ahead < k) atomicMin(&s.bound_key, best);
    __syncthreads();
    bound_key = s.bound_key;
    const bool tie = best == bound_key;
    if (tie) {
      s.list_id[atomicAdd(&s.ties, 1u)] = best_id;
      s.ahead = ahead;  // the same for every tie
    }
    __syncthreads();
    // Of the threads at that key, the one whose id is k - ahead in order.
    const uint32_t ties = s.ties, place = k - 1 - s.ahead;
    if (tie) {
      uint32_t lower = 0;
      for (uint32_t t = 0; t < ties; ++t) lower += s.list_id[t] < best_id;
      if (lower == place) s.bound_id = best_id;
    }
    __syncthreads();
    bound_id = s.bound_id;
  }
#pragma unroll
  for (uint32_t i = 0; i < N; ++i)
    if (key[i] > bound_key || (key[i] == bound_key && id[i] <= bound_id)) {
      const uint32_t at = atomicAdd(&s.count, 1u);
      s.list_key[at] = key[i];
      s.list_id[at] = id[i];
    }
  __syncthreads();
  return s.count;
}

// The place of list item i among the n listed ones.
__device__ __forceinline__ uint32_t place_of(const TopLds &s, uint32_t n, uint32_t key,
                                             uint32_t id) {
  uint32_t place = 0;
  for (uint32_t j = 0; j < n; ++j) {
    const uint32_t other = s.list_key[j];
    place += other > key || (other == key && s.list_id[j] < id) ? 1u : 0u;
  }
  return place;
}

// The row's best groups into s.best; returns their number, at most
// kTopLogprobs and at least the k best.
template <uint32_t N>
__device__ __forceinline__ uint32_t best_groups(TopLds &s, const float *maxima, uint32_t groups,
                                                uint32_t k) {
  const uint32_t tid = threadIdx.x;
  uint32_t key[N], id[N];
#pragma unroll
  for (uint32_t i = 0; i < N; ++i) {
    id[i] = i * 256 + tid;
    key[i] = id[i] < groups ? listed_key(maxima[id[i]]) : 0u;
  }
  const uint32_t n = list_best(s, k, key, id);
  if (n <= kTopLogprobs) {
    if (tid < n) s.best[tid] = s.list_id[tid];
  } else {
    for (uint32_t i = tid; i < n; i += 256) {
      const uint32_t place = place_of(s, n, s.list_key[i], s.list_id[i]);
      if (place < k) s.best[place] = s.list_id[i];
    }
  }
  __syncthreads();
  return n <= kTopLogprobs ? n : k;
}

// The row's k best tokens from its best groups: a wave reads a group a load.
template <int DT, uint32_t N>
__device__ __forceinline__ void best_tokens(TopLds &s, const ScoreLaunch &a, uint32_t row,
                                            const typename Logits<DT>::Element *x, uint32_t n,
                                            const RowScore &score) {
  const uint32_t tid = threadIdx.x, k = a.top;
  uint32_t key[N], id[N];
#pragma unroll
  for (uint32_t i = 0; i < N; ++i) {
    const uint32_t slot = i * 4 + (tid >> 6);
    id[i] = slot < n ? s.best[slot] * kScoreGroup + (tid & 63u) : 0xffffffffu;
    key[i] = id[i] < a.vocabulary ? listed_key(logit_value(x[id[i]])) : 0u;
  }
  const uint32_t m = list_best(s, k, key, id);
  uint32_t *ids = a.out_top_ids + (uint64_t)row * k;
  float *logprobs = a.out_top_logprobs + (uint64_t)row * k;
  for (uint32_t i = tid; i < m; i += 256) {
    const uint32_t item = s.list_key[i], token = s.list_id[i];
    const uint32_t place = place_of(s, m, item, token);
    if (place < k) {
      ids[place] = token;
      logprobs[place] = score.logprob(key_logit(item));
    }
  }
  for (uint32_t i = m + tid; i < k; i += 256) {
    ids[i] = kNoToken;
    logprobs[i] = -__builtin_inff();
  }
}

// One row a block: 256 threads with alternatives, otherwise a wave.
template <int DT, bool TOP>
__global__ __launch_bounds__(TOP ? 256 : 64) void logprobs_kernel(ScoreLaunch a) {
  constexpr uint32_t THREADS = TOP ? 256 : 64;
  const uint32_t tid = threadIdx.x, row = blockIdx.x;
  const auto *x = row_of<DT>(a.logits, (uint64_t)row * a.stride);
  const float inv_t = inverse_temperature(a, row);
  const MaxSum total = row_total(a, row, inv_t * kLog2e);
  const RowScore score{total.m, inv_t, logf(total.s)};
  if (tid == 0 && a.out_lse) a.out_lse[row] = score.lse();
  for (uint32_t i = tid; i < a.token_count; i += THREADS) {
    const uint32_t token = a.tokens[(uint64_t)row * a.token_stride + i];
    const bool known = token < a.vocabulary;
    if (a.out_logprobs)
      a.out_logprobs[(uint64_t)row * a.token_count + i] =
          known ? score.logprob(logit_value(x[token])) : -__builtin_inff();
    if (i == 0 && a.out_ranks) {
      uint32_t rank = 1;
      for (uint32_t g = 0; g < a.segments; ++g) rank += a.aheads[(uint64_t)row * a.segments + g];
      a.out_ranks[row] = known ? rank : 0u;
    }
  }
  if constexpr (TOP) {
    __shared__ TopLds s;
    const float *maxima = a.maxima + (uint64_t)row * a.groups;
    uint32_t n;
    if (a.groups <= 8 * 256)
      n = best_groups<8>(s, maxima, a.groups, a.top);
    else if (a.groups <= 16 * 256)
      n = best_groups<16>(s, maxima, a.groups, a.top);
    else
      n = best_groups<kMostItems>(s, maxima, a.groups, a.top);
    if (n <= 8 * 4)
      best_tokens<DT, 8>(s, a, row, x, n, score);
    else
      best_tokens<DT, kMostItems>(s, a, row, x, n, score);
  }
}

__device__ __forceinline__ float block_max(float v, float *lds) {
  v = wave_max_f32(v);
  __syncthreads();
  if ((threadIdx.x & 63u) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return __builtin_fmaxf(__builtin_fmaxf(lds[0], lds[1]), __builtin_fmaxf(lds[2], lds[3]));
}
__device__ __forceinline__ float block_sum(float v, float *lds) {
  v += xor_f32<1>(v);
  v += xor_f32<2>(v);
  v += xor_f32<4>(v);
  v += xor_f32<8>(v);
  v += xor_f32<16>(v);
  v += xor_f32<32>(v);
  __syncthreads();
  if ((threadIdx.x & 63u) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

// The distillation's loss of one row a block, one listed token a thread:
// sum p_k (ln p_k - ln q_k), and what the backward pass takes: the row's
// maximum, the list's mass over the row's sum, and each slot's probability
// (-1: no token, or one that an earlier slot lists).
template <int DT>
__global__ __launch_bounds__(256) void distill_loss_kernel(ScoreLaunch a) {
  __shared__ uint32_t listed[kTeacherTokens];
  __shared__ float lds[4];
  const uint32_t tid = threadIdx.x, row = blockIdx.x, K = a.teacher_count;
  const auto *x = row_of<DT>(a.logits, (uint64_t)row * a.stride);
  const float inv_t = 1.0f / a.temperature;
  uint32_t id = kNoToken;
  float value = -__builtin_inff(), logit = 0.0f;
  if (tid < K) {
    id = a.teacher_ids[(uint64_t)row * a.teacher_stride + tid];
    value = a.teacher_values[(uint64_t)row * a.teacher_stride + tid];
  }
  const MaxSum total = row_total(a, row, inv_t * kLog2e);
  const RowScore score{total.m, inv_t, logf(total.s)};
  listed[tid] = id;
  __syncthreads();
  bool valid = id < a.vocabulary;
  if (valid) logit = logit_value(x[id]);
  for (uint32_t k = 0; k < K; ++k) valid = valid && !(k < tid && listed[k] == id);
  float log_p = valid ? value : -__builtin_inff();
  if (a.normalize) {
    log_p *= inv_t;
    log_p -= finite_reference(block_max(log_p, lds));
    const float log_sum = logf(block_sum(expf(log_p), lds));
    // -infinity stays: a list of nothing else has no mass.
    if (log_p != -__builtin_inff()) log_p -= log_sum;
  }
  const float p = valid ? expf(log_p) : 0.0f;
  // A token of no teacher probability adds nothing, whatever the student's.
  const float loss = block_sum(p == 0.0f ? 0.0f : p * (log_p - score.logprob(logit)), lds);
  const float mass = block_sum(p, lds);
  if (tid == 0) {
    a.out_loss[row] = loss;
    if (a.out_lse) a.out_lse[row] = score.lse();
  }
  if (a.saved) {
    float *saved = a.saved + (uint64_t)row * (2 + K);
    if (tid == 0) {
      saved[0] = total.m;
      // No list, or no student probability anywhere: no exponentials to add.
      saved[1] = mass == 0.0f || total.s == 0.0f ? 0.0f : mass / total.s;
    }
    if (tid < K) saved[2 + tid] = valid ? p : -1.0f;
  }
}

}  // namespace

int launch_score(const ScoreLaunch &a, uint32_t dtype, void *stream) {
  const hipStream_t st = (hipStream_t)stream;
  const dim3 grid(a.row_count * a.segments), block(256);
  const bool top = a.top != 0, rank = a.out_ranks != nullptr;
#define JF_SCORE(DT, TOP, RANK)                                                        \
  if (dtype == DT && top == TOP && rank == RANK)                                       \
  hipLaunchKernelGGL((score_kernel<DT, TOP, RANK>), grid, block, 0, st, a)
  JF_SCORE(0, false, false);
  JF_SCORE(0, false, true);
  JF_SCORE(0, true, false);
  JF_SCORE(0, true, true);
  JF_SCORE(1, false, false);
  JF_SCORE(1, false, true);
  JF_SCORE(1, true, false);
  JF_SCORE(1, true, true);
#undef JF_SCORE
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  const dim3 rows(a.row_count);
  if (a.teacher_ids) {
    if (dtype == 0)
      hipLaunchKernelGGL((distill_loss_kernel<0>), rows, block, 0, st, a);
    else
      hipLaunchKernelGGL((distill_loss_kernel<1>), rows, block, 0, st, a);
  } else if (top) {
    if (dtype == 0)
      hipLaunchKernelGGL((logprobs_kernel<0, true>), rows, block, 0, st, a);
    else
      hipLaunchKernelGGL((logprobs_kernel<1, true>), rows, block, 0, st, a);
  } else {
    if (dtype == 0)
      hipLaunchKernelGGL((logprobs_kernel<0, false>), rows, dim3(64), 0, st, a);
    else
      hipLaunchKernelGGL((logprobs_kernel<1, false>), rows, dim3(64), 0, st, a);
  }
  return (int)hipGetLastError();
}

}  // namespace jf
