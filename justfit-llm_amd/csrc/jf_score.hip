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
    load_chunk<DT>(x, base, V, kPastMinusInfinity<DT>, w);
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
// Lists of up to this many alternatives are cut by the best items of 64 quads
// of lanes, longer ones by those of the 256 threads: a cut by fewer units is
// quicker to find and lists more items.
constexpr uint32_t kQuadTop = 32;
constexpr uint32_t kListItems = kMostItems * (kTopLogprobs - 1) + 1;
static_assert(4 * kMostItems * (kQuadTop - 1) + 1 <= kListItems);
constexpr uint32_t kIdBits = 20;  // tokens and groups are below 2^20

struct TopList {
  uint32_t unit_key[256], unit_id[256];
  uint2 item[kListItems];  // key, id
  uint32_t count;
};

// The k-th largest (from 1) of the wave's 64 * U values below 2^BITS, found
// bit by bit: the largest t that k values reach.
template <uint32_t U, int BITS>
__device__ __forceinline__ uint32_t kth_largest(const uint32_t (&v)[U], uint32_t k) {
  uint32_t t = 0;
#pragma unroll 4
  for (int b = BITS - 1; b >= 0; --b) {
    const uint32_t trial = t | 1u << b;
    uint32_t reach = 0;
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) reach += (uint32_t)__popcll(ballot(v[u] >= trial));
    if (reach >= k) t = trial;
  }
  return t;
}

// Lists in LDS, in no order, the block's items at or ahead of the k-th of its
// units' best items (a unit: four lanes, or with U = 4 one thread), in the
// order (key down, id up); key 0 is no item, and with fewer than k units that
// have an item every one is listed. So the list holds the block's k best items.
// An item on it belongs to one of those k units, the k-th of which has no other
// one there: at most (k - 1) * 4 / U * N + 1 items. Returns their number.
// s.count is 0 on entry, ordered by a barrier.
template <uint32_t N, uint32_t U>
__device__ __forceinline__ uint32_t list_best(TopList &s, uint32_t k, const uint32_t (&key)[N],
                                              const uint32_t (&id)[N]) {
  static_assert(N <= kMostItems && (U == 1 || U == 4));
  const uint32_t tid = threadIdx.x, lane = tid & 63u;
  uint32_t best = 0, best_id = 0;
  const auto take = [&](uint32_t other, uint32_t other_id) {
    if (other > best || (other == best && other_id < best_id)) {
      best = other;
      best_id = other_id;
    }
  };
#pragma unroll
  for (uint32_t i = 0; i < N; ++i) take(key[i], id[i]);
  const uint32_t own = best, own_id = best_id;
  if constexpr (U == 1) {
    take(xor_u32<1>(best), xor_u32<1>(best_id));
    take(xor_u32<2>(best), xor_u32<2>(best_id));
    if (tid % 4 == 0) {
      s.unit_key[tid / 4] = best;
      s.unit_id[tid / 4] = best_id;
    }
  } else {
    s.unit_key[tid] = best;
    s.unit_id[tid] = best_id;
  }
  __syncthreads();
  // Every wave finds the cut by itself.
  uint32_t unit[U], unit_id[U], present = 0;
#pragma unroll
  for (uint32_t u = 0; u < U; ++u) {
    unit[u] = s.unit_key[lane * U + u];
    unit_id[u] = s.unit_id[lane * U + u];
    present += (uint32_t)__popcll(ballot(unit[u] != 0));
  }
  uint32_t cut = 1, cut_id = 0xffffffffu;  // everything
  if (present >= k) {
    cut = kth_largest<U, 32>(unit, k);
    uint32_t ahead = 0, ties = 0, tie_id[U], last = 0;
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      ahead += (uint32_t)__popcll(ballot(unit[u] > cut));
      ties += (uint32_t)__popcll(ballot(unit[u] == cut));
      // Ids from the top down, so that the lowest is the largest.
      tie_id[u] = unit[u] == cut ? (1u << kIdBits) - 1u - unit_id[u] : 0u;
      last = max(last, unit[u] == cut ? unit_id[u] : 0u);
    }
    if (ahead + ties == k)
      cut_id = wave_max_u32(last);
    else
      cut_id = (1u << kIdBits) - 1u - kth_largest<U, kIdBits>(tie_id, k - ahead);
  }
  if (own > cut || (own == cut && own_id <= cut_id)) {
#pragma unroll
    for (uint32_t i = 0; i < N; ++i)
      if (key[i] > cut || (key[i] == cut && id[i] <= cut_id))
        s.item[atomicAdd(&s.count, 1u)] = make_uint2(key[i], id[i]);
  }
  __syncthreads();
  return s.count;
}

// The place of an item among the n listed ones.
__device__ __forceinline__ uint32_t place_of(const TopList &s, uint32_t n, uint2 item) {
  uint32_t place = 0;
#pragma unroll 8
  for (uint32_t j = 0; j < n; ++j) {
    const uint2 other = s.item[j];
    place += other.x > item.x || (other.x == item.x && other.y < item.y) ? 1u : 0u;
  }
  return place;
}

// The row's best groups; `best` receives them. Returns their number, at most
// kTopLogprobs, the k best among them.
template <uint32_t N, uint32_t U>
__device__ __forceinline__ uint32_t best_groups(TopList &s, uint32_t *best, const float *maxima,
                                                uint32_t groups, uint32_t k) {
  const uint32_t tid = threadIdx.x;
  float m[N];
#pragma unroll
  for (uint32_t i = 0; i < N; ++i)
    m[i] = maxima[min(i * 256 + tid, groups - 1)];
  uint32_t key[N], id[N];
#pragma unroll
  for (uint32_t i = 0; i < N; ++i) {
    id[i] = i * 256 + tid;
    key[i] = id[i] < groups ? listed_key(m[i]) : 0u;
  }
  const uint32_t n = list_best<N, U>(s, k, key, id);
  if (n <= kTopLogprobs) {
    if (tid < n) best[tid] = s.item[tid].y;
  } else {
    for (uint32_t i = tid; i < n; i += 256) {
      const uint32_t place = place_of(s, n, s.item[i]);
      if (place < k) best[place] = s.item[i].y;
    }
  }
  __syncthreads();
  if (tid == 0) s.count = 0;  // ordered by the next list's barrier before its items
  return n <= kTopLogprobs ? n : k;
}

// The row's k best tokens from its n best groups: a wave reads a group a load.
template <int DT, uint32_t N, uint32_t U>
__device__ __forceinline__ void best_tokens(TopList &s, const uint32_t *best, const ScoreLaunch &a,
                                            uint32_t row, const typename Logits<DT>::Element *x,
                                            uint32_t n, const RowScore &score) {
  const uint32_t tid = threadIdx.x, k = a.top;
  float v[N];
  uint32_t key[N], id[N];
#pragma unroll
  for (uint32_t i = 0; i < N; ++i) {
    const uint32_t slot = i * 4 + (tid >> 6);
    id[i] = best[min(slot, n - 1)] * kScoreGroup + (tid & 63u);
    v[i] = logit_value(x[min(id[i], a.vocabulary - 1)]);
  }
#pragma unroll
  for (uint32_t i = 0; i < N; ++i)
    key[i] = i * 4 + (tid >> 6) < n && id[i] < a.vocabulary ? listed_key(v[i]) : 0u;
  const uint32_t m = list_best<N, U>(s, k, key, id);
  uint32_t *ids = a.out_top_ids + (uint64_t)row * k;
  float *logprobs = a.out_top_logprobs + (uint64_t)row * k;
  for (uint32_t i = tid; i < m; i += 256) {
    const uint2 item = s.item[i];
    const uint32_t place = place_of(s, m, item);
    if (place < k) {
      ids[place] = item.y;
      logprobs[place] = score.logprob(key_logit(item.x));
    }
  }
  for (uint32_t i = m + tid; i < k; i += 256) {
    ids[i] = kNoToken;
    logprobs[i] = -__builtin_inff();
  }
}

template <int DT, uint32_t U>
__device__ __forceinline__ void row_best(TopList &s, uint32_t *best, const ScoreLaunch &a,
                                         uint32_t row, const typename Logits<DT>::Element *x,
                                         const RowScore &score) {
  const float *maxima = a.maxima + (uint64_t)row * a.groups;
  uint32_t n;
  if (a.groups <= 10 * 256)
    n = best_groups<10, U>(s, best, maxima, a.groups, a.top);
  else if (a.groups <= 16 * 256)
    n = best_groups<16, U>(s, best, maxima, a.groups, a.top);
  else
    n = best_groups<kMostItems, U>(s, best, maxima, a.groups, a.top);
  if (n == 0) {  // nothing to list
    for (uint32_t i = threadIdx.x; i < a.top; i += 256) {
      a.out_top_ids[(uint64_t)row * a.top + i] = kNoToken;
      a.out_top_logprobs[(uint64_t)row * a.top + i] = -__builtin_inff();
    }
  } else if (U == 1 && n <= 8 * 4) {
    best_tokens<DT, 8, U>(s, best, a, row, x, n, score);
  } else {
    best_tokens<DT, kMostItems, U>(s, best, a, row, x, n, score);
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
    a.out_logprobs[(uint64_t)row * a.token_count + i] =
        token < a.vocabulary ? score.logprob(logit_value(x[token])) : -__builtin_inff();
  }
  if (a.out_ranks && tid < 64) {
    const uint32_t ahead =
        wave_sum_u32(tid < a.segments ? a.aheads[(uint64_t)row * a.segments + tid] : 0u);
    if (tid == 0)
      a.out_ranks[row] =
          a.tokens[(uint64_t)row * a.token_stride] < a.vocabulary ? ahead + 1u : 0u;
  }
  if constexpr (TOP) {
    __shared__ TopList s;
    __shared__ uint32_t best[kTopLogprobs];
    if (tid == 0) s.count = 0;
    __syncthreads();
    if (a.top <= kQuadTop)
      row_best<DT, 1>(s, best, a, row, x, score);
    else
      row_best<DT, 4>(s, best, a, row, x, score);
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
