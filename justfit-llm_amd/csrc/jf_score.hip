// Log-probabilities and the distillation's forward pass on gfx950: one pass
// over a row's logits for its maximum m and s = sum exp((x - m) / T), then a
// finish over a few words of the row.
//
// The pass. A block takes one chunk of a row in registers, 8 to 32 values a
// thread, which takes their maximum and adds their exponentials against it;
// waves and then the block join theirs. The row's first token's rank needs
// only its logit, read up front: a count of the values ahead of it. Reading
// bounds it: 2048 rows x 151,936 bf16, 622 MB, take 103 us without
// alternatives (6 TB/s), 256 rows x 248,320 with the groups' maxima 26.8 (4.9).
//
// The finish is a launch of its own, 4 to 6 us for few rows: a block that
// counts the row's others in and finishes behind the last of them makes every
// block publish its part first, and 1024 losses of 151,936 took 105 us so, 59
// in two launches. (Not timed for a few rows.)
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

// A row's temperature: the sampler's 0 (a greedy row) and anything that is no
// temperature leave the logits as they are.
__device__ __forceinline__ float inverse_temperature(const ScoreLaunch &a, uint32_t row) {
  const float t = a.temperatures ? a.temperatures[row] : a.temperature;
  return t >= __FLT_MIN__ && t < __builtin_inff() ? 1.0f / t : 1.0f;
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

// That of the least finite logit.
constexpr uint32_t kLeastKey = 0x00800000u;

// ---- the best tokens ----------------------------------------------------------

// Element i of a row at a uniform address, by a 32-bit offset (a row's bytes
// stay below 2^22): one address register a load.
template <class T>
__device__ __forceinline__ const T *element(const T *row, uint32_t i) {
  return (const T *)((const char *)row + (uint32_t)(i * sizeof(T)));
}

// A row's block: eight waves list its alternatives, one takes its totals.
constexpr uint32_t kListWaves = 8;
constexpr uint32_t kListThreads = kListWaves * 64;
constexpr uint32_t kTopWaves = kListWaves + 1;
constexpr uint32_t kMostItems = 16;  // groups a thread holds at most
constexpr uint32_t kWaveGroups = 128;  // groups a wave lists at most
// Tokens a wave lists at most. A row whose best tokens are neighbours lists most
// of their groups' tokens: ids in the order of their frequency come to hundreds.
constexpr uint32_t kWaveItems = 512;
// Lists of up to this many alternatives are cut by the best groups of 64 units of
// eight lanes, longer ones by those of 256 pairs: a cut by fewer units is
// quicker to find and lists more groups (64 rows x 151,936 in f32: 5 alternatives
// 14.3 us by the larger units, 16.0 by pairs; 20 15.3 and 16.7; 33 16.4 and 17.4;
// 48 19.8 and 17.9).
constexpr uint32_t kShortTop = 32;

struct TopLds {
  uint64_t item[kListWaves][kWaveItems + 8];  // each wave's tokens, then 0 up to a multiple of 8
  uint32_t unit[256];                // the units' best keys
  uint16_t group[kListWaves][kWaveGroups];
  uint32_t best[kTopLogprobs];
  uint64_t wave[2][kTopWaves];
  uint32_t count[kListWaves];
  uint32_t crowded;
  RowScore score;
};

// The group whose maximum is the i-th of its row: a chunk's groups are stored in
// the order (lanes, vector), the pass's own (score_kernel).
template <int DT>
__device__ __forceinline__ uint32_t group_at(const ScoreLaunch &a, uint32_t i) {
  // Of a chunk: 2^lv vectors of 2^ls groups.
  constexpr uint32_t ls = DT == 0 ? 4 : 5;
  static_assert(kSlab<DT> / kScoreGroup == 1u << ls);
  const uint32_t lv = a.vectors == 4 ? 2 : 1;
  const uint32_t within = i & ((1u << (lv + ls)) - 1u);
  return i - within + ((within & ((1u << lv) - 1u)) << ls) + (within >> lv);
}
// An item as one number, larger ones ahead: its key, then the lower id.
__device__ __forceinline__ uint64_t item_of(uint32_t key, uint32_t id) {
  return (uint64_t)key << 32 | (0xffffffffu - id);
}
__device__ __forceinline__ uint32_t item_id(uint64_t item) { return 0xffffffffu - (uint32_t)item; }

// The k-th largest (from 1) of the wave's 64 * U values, down to its top BITS
// bits, two bits a step: the largest such t that k values reach.
template <uint32_t U, int BITS>
__device__ __forceinline__ uint32_t kth_largest(const uint32_t (&v)[U], uint32_t k) {
  static_assert(BITS % 2 == 0);
  uint32_t t = 0;
  for (int b = 30; b > 30 - BITS; b -= 2) {
    uint32_t reach[3] = {};
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
#pragma unroll
      for (uint32_t q = 0; q < 3; ++q)
        reach[q] += (uint32_t)__popcll(ballot(v[u] >= (t | (q + 1) << b)));
    }
    t |= (reach[2] >= k ? 3u : reach[1] >= k ? 2u : reach[0] >= k ? 1u : 0u) << b;
  }
  return t;
}

// A search for the k-th largest of some values, two bits a step from bits b and
// b + 1 down: t is the largest prefix so far that k of them reach.
struct Search {
  uint32_t t;
  int b;
  // After a step's counts of the values that reach t with 1, 2 and 3 in its bits.
  __device__ __forceinline__ void take(uint32_t one, uint32_t two, uint32_t three, uint32_t k) {
    t |= (three >= k ? 3u : two >= k ? 2u : one >= k ? 1u : 0u) << b;
    b -= 2;
  }
};
// The search among at least k values from `least` to `most`: the bits that they
// share are no steps.
__device__ __forceinline__ Search search_between(uint32_t least, uint32_t most) {
  if (least == most) return {most, -2};
  const int b = (31 - __builtin_clz(least ^ most)) & ~1;
  return {b == 30 ? 0u : most >> (b + 2) << (b + 2), b};
}
// A lane's part of a step's counts: those of 1 and, shifted by 16, of 2; of 3.
// (For many values a lane; for few, counting a ballot's bits each is quicker.)
template <uint32_t M>
__device__ __forceinline__ void count_reach(const uint32_t (&v)[M], const Search &f,
                                            uint32_t &low, uint32_t &high) {
  uint32_t reach[3] = {};
#pragma unroll
  for (uint32_t m = 0; m < M; ++m) {
#pragma unroll
    for (uint32_t q = 0; q < 3; ++q) reach[q] += v[m] >= (f.t | (q + 1) << f.b) ? 1u : 0u;
  }
  low = reach[0] | reach[1] << 16;
  high = reach[2];
}
// A lane's least value but 0, and its largest.
template <uint32_t M>
__device__ __forceinline__ void extent(const uint32_t (&v)[M], uint32_t &least, uint32_t &most) {
  least = 0xffffffffu;
  most = 0;
#pragma unroll
  for (uint32_t m = 0; m < M; ++m) {
    least = v[m] && v[m] < least ? v[m] : least;
    most = max(most, v[m]);
  }
}

// The search through the whole block's values, to their last bit.
template <uint32_t M>
__device__ __forceinline__ uint32_t block_kth_largest(TopLds &s, const uint32_t (&v)[M],
                                                      Search f, uint32_t k, uint32_t &phase) {
  static_assert(kTopWaves * 64 * M < 1u << 16);
#pragma unroll 1
  while (f.b >= 0) {
    uint32_t low, high;
    count_reach(v, f, low, high);
    low = wave_sum_u32(low);
    high = wave_sum_u32(high);
    // Two rows of counts in turn: a step's are read before the next but one's.
    uint64_t *counts = s.wave[phase];
    phase ^= 1u;
    if ((threadIdx.x & 63u) == 0) counts[threadIdx.x >> 6] = low | (uint64_t)high << 32;
    __syncthreads();
    uint64_t all = 0;
#pragma unroll
    for (uint32_t w = 0; w < kTopWaves; ++w) all += counts[w];
    f.take((uint32_t)all & 0xffffu, (uint32_t)all >> 16, (uint32_t)(all >> 32), k);
  }
  return f.t;
}
// The k-th largest of the block's keys; 0 if fewer of them are not 0.
template <uint32_t M>
__device__ __forceinline__ uint32_t block_kth_key(TopLds &s, const uint32_t (&key)[M], uint32_t k,
                                                  uint32_t &phase) {
  uint32_t least, most, keys = 0;
  extent(key, least, most);
#pragma unroll
  for (uint32_t m = 0; m < M; ++m) keys += key[m] ? 1u : 0u;
  least = wave_min_u32(least);
  most = wave_max_u32(most);
  keys = wave_sum_u32(keys);
  uint32_t(*waves)[kTopWaves] = (uint32_t(*)[kTopWaves])s.unit;  // no longer read
  if ((threadIdx.x & 63u) == 0) {
    const uint32_t w = threadIdx.x >> 6;
    waves[0][w] = least;
    waves[1][w] = most;
    waves[2][w] = keys;
  }
  __syncthreads();
  keys = 0;
#pragma unroll
  for (uint32_t w = 0; w < kTopWaves; ++w) {
    least = min(least, waves[0][w]);
    most = max(most, waves[1][w]);
    keys += waves[2][w];
  }
  return keys < k ? 0u : block_kth_largest(s, key, search_between(least, most), k, phase);
}

// The block's `k` best of M keys a thread, each with an id (0 is no key), to
// put(place, key, id) of their threads, in no order; returns how many.
// Whatever the ties: the k-th key, then the k-th of the ids that have it.
template <uint32_t M, int ID_BITS, class Id, class Put>
__device__ __forceinline__ uint32_t pick_best(TopLds &s, const uint32_t (&key)[M], uint32_t k,
                                              uint32_t &phase, const Id &id_of, const Put &put) {
  constexpr uint32_t AHEAD = (1u << ID_BITS) - 1u;  // above every id's number
  if (threadIdx.x == 0) s.count[0] = 0;
  const uint32_t t = block_kth_key(s, key, k, phase);
  uint32_t number[M];
#pragma unroll
  for (uint32_t m = 0; m < M; ++m)
    number[m] = key[m] > t ? AHEAD : key[m] == t && t ? AHEAD - 1u - id_of(m) : 0u;
  const uint32_t cut =
      max(block_kth_largest(s, number, Search{0u, ID_BITS - 2}, k, phase), 1u);
#pragma unroll
  for (uint32_t m = 0; m < M; ++m)
    if (number[m] >= cut) put(atomicAdd(&s.count[0], 1u), key[m], id_of(m));
  __syncthreads();
  const uint32_t n = s.count[0];
  __syncthreads();
  return n;
}

// One alternative of a row at its place.
__device__ __forceinline__ void put_best(const ScoreLaunch &a, uint32_t row, uint32_t place,
                                         uint64_t item, const RowScore &score) {
  const uint64_t at = (uint64_t)row * a.top + place;
  a.out_top_ids[at] = item_id(item);
  a.out_top_logprobs[at] = score.logprob(key_logit((uint32_t)(item >> 32)));
}

// The alternatives of a row whose best groups or tokens crowd the lists (many
// equal maxima, as of a constant row, one masked by a lowest value down to fewer
// than k tokens, or one that falls from its first token on): its k best groups,
// then their k best tokens. Returns how many there are. 64 rows x 151,936 in
// f32, constant: 20 alternatives 32 us, 128 of them 36, and masked by the lowest
// value 60 and 65 (in random order 13 and 21; in k rounds of a maximum each 67
// and 975).
template <int DT, uint32_t N>
__device__ __forceinline__ uint32_t crowded_best(TopLds &s, const ScoreLaunch &a, uint32_t row,
                                              const typename Logits<DT>::Element *x,
                                              const float *maxima) {
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  uint32_t phase = 0, n;
  {
    uint32_t key[N];
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) {
      const uint32_t at = i * kListThreads + tid;
      key[i] = tid < kListThreads && at < a.groups ? listed_key(*element(maxima, at)) : 0u;
    }
    n = pick_best<N, 14>(
        s, key, a.top, phase, [&](uint32_t i) { return group_at<DT>(a, i * kListThreads + tid); },
        [&](uint32_t place, uint32_t, uint32_t id) { s.best[place] = id; });
  }
  if (n == 0) return 0;
  constexpr uint32_t EACH = (kTopLogprobs + kTopWaves - 1) / kTopWaves;  // groups a wave
  uint32_t key[EACH];
  const auto id_of = [&](uint32_t i) {
    return s.best[min(i * kTopWaves + wave, n - 1)] * kScoreGroup + lane;
  };
  float v[EACH];
#pragma unroll
  for (uint32_t i = 0; i < EACH; ++i)
    v[i] = logit_value(*element(x, min(id_of(i), a.vocabulary - 1)));
#pragma unroll
  for (uint32_t i = 0; i < EACH; ++i)
    key[i] = i * kTopWaves + wave < n && id_of(i) < a.vocabulary ? listed_key(v[i]) : 0u;
  uint64_t *items = s.item[0];
  const uint32_t listed = pick_best<EACH, 20>(
      s, key, a.top, phase, id_of,
      [&](uint32_t place, uint32_t key, uint32_t id) { items[place] = item_of(key, id); });
  if (tid < listed) {
    const uint64_t item = items[tid];
    uint32_t place = 0;
    for (uint32_t i = 0; i < listed; ++i) place += items[i] > item ? 1u : 0u;
    put_best(a, row, place, item, s.score);
  }
  return listed;
}

// The wave's own groups whose maxima reach the k-th best of the units', and of
// their tokens those that reach it, into its lists. A unit is eight lanes (U = 1:
// 64 units) or two (U = 4: 256 of them). At least k groups reach that
// cut, and so the row's k best tokens do; few others where the best groups lie
// in different units. The cut's last bits are left out (each is half a step of
// the search): of an f32 key the last 10, a bf16 key has 16.
template <int DT, uint32_t N, uint32_t U>
__device__ __forceinline__ void list_wave(TopLds &s, const ScoreLaunch &a,
                                          const typename Logits<DT>::Element *x,
                                          const uint32_t (&key)[N]) {
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, k = a.top;
  uint32_t unit[U], present = 0;
#pragma unroll
  for (uint32_t u = 0; u < U; ++u) {
    unit[u] = s.unit[lane * U + u];
    present += (uint32_t)__popcll(ballot(unit[u] != 0));
  }
  // With fewer than k units that have a group, every group is listed.
  uint32_t cut = 1;
  if (present >= k) cut = max(kth_largest<U, DT == 0 ? 22 : 16>(unit, k), 1u);
  uint32_t n = 0, tokens = 0;
#pragma unroll
  for (uint32_t i = 0; i < N; ++i) {
    const bool take = key[i] >= cut;
    const uint64_t lanes = ballot(take);
    if (!lanes) continue;
    const uint32_t at = n + mbcnt(lanes);
    if (take && at < kWaveGroups) s.group[wave][at] = (uint16_t)(i * kListThreads + tid);
    n += (uint32_t)__popcll(lanes);
  }
  __builtin_amdgcn_wave_barrier();  // the wave's own list, in order
  bool fits = n <= kWaveGroups;
  if (fits) {
    constexpr uint32_t AHEAD = 8;  // groups asked for at once
    const float least = key_logit(max(cut, kLeastKey));
#pragma unroll 1
    for (uint32_t first = 0; first < n; first += AHEAD) {
      // A lane's group is a load's for all.
      const uint32_t mine = group_at<DT>(a, s.group[wave][min(first + lane % AHEAD, n - 1)]);
      float v[AHEAD];
#pragma unroll
      for (uint32_t i = 0; i < AHEAD; ++i) {
        const uint32_t base = __builtin_amdgcn_readlane(mine, i) * kScoreGroup;
        v[i] = logit_value(*element(x + base, min(lane, a.vocabulary - 1 - base)));
      }
#pragma unroll
      for (uint32_t i = 0; i < AHEAD; ++i) {
        if (first + i >= n) break;
        const uint32_t base = __builtin_amdgcn_readlane(mine, i) * kScoreGroup;
        const bool take = v[i] >= least && lane < a.vocabulary - base;
        const uint64_t lanes = ballot(take);
        const uint32_t at = tokens + mbcnt(lanes);
        if (take && at < kWaveItems) s.item[wave][at] = item_of(logit_key(v[i]), base + lane);
        tokens += (uint32_t)__popcll(lanes);
      }
    }
    fits = tokens <= kWaveItems;
  }
  if (fits && lane < 8) s.item[wave][tokens + lane] = 0;
  if (lane == 0) {
    s.count[wave] = tokens;
    if (!fits) s.crowded = 1;
  }
}

// Every item's place is the number of items ahead of it: eight lanes take R items
// at a time, a wave's list each.
template <uint32_t R>
__device__ __forceinline__ void place_items(const TopLds &s, const ScoreLaunch &a, uint32_t row,
                                            uint32_t listed) {
  constexpr uint32_t STEP = kTopWaves * 64 / kListWaves;
  const uint32_t tid = threadIdx.x, own = s.count[tid % kListWaves];
  const uint64_t *list = s.item[tid % kListWaves];
  const RowScore score = s.score;
  for (uint32_t first = 0; first < listed; first += R * STEP) {
    uint64_t item[R];
    uint32_t place[R] = {};
#pragma unroll
    for (uint32_t r = 0; r < R; ++r) {
      const uint32_t i = first + r * STEP + tid / kListWaves;
      uint32_t w = 0, at = i;
#pragma unroll
      for (uint32_t j = 0; j + 1 < kListWaves; ++j) {
        const uint32_t n = s.count[j];
        const bool past = w == j && at >= n;
        at -= past ? n : 0u;
        w += past ? 1u : 0u;
      }
      item[r] = i < listed ? s.item[w][at] : 0ull;
    }
#pragma unroll 1
    for (uint32_t j = 0; j < own; j += 8) {
#pragma unroll
      for (uint32_t e = 0; e < 8; ++e) {
        const uint64_t other = list[j + e];
#pragma unroll
        for (uint32_t r = 0; r < R; ++r) place[r] += other > item[r] ? 1u : 0u;
      }
    }
#pragma unroll
    for (uint32_t r = 0; r < R; ++r) {
      place[r] += xor_u32<1>(place[r]);
      place[r] += xor_u32<2>(place[r]);
      place[r] += xor_u32<4>(place[r]);
      if (item[r] && place[r] < a.top && tid % kListWaves == 0)
        put_best(a, row, place[r], item[r], score);
    }
  }
}

// ---- finish -------------------------------------------------------------------

// A row's totals and its tokens' log-probabilities by one wave. What they are
// worked out from is asked for at once, the lane's first token among it.
template <int DT>
struct RowWave {
  float inv_t;
  MaxSum part;
  uint32_t token, ahead;

  __device__ __forceinline__ void load(const ScoreLaunch &a, uint32_t row) {
    const uint32_t lane = threadIdx.x & 63u;
    part = row_part(a, row);
    token = lane < a.token_count ? a.tokens[(uint64_t)row * a.token_stride + lane] : kNoToken;
    ahead = 0;
    if (a.out_ranks) {
      for (uint32_t g = lane; g < a.segments; g += 64)
        ahead += a.aheads[(uint64_t)row * a.segments + g];
    }
    inv_t = inverse_temperature(a, row);
  }
  __device__ __forceinline__ RowScore put(const ScoreLaunch &a, uint32_t row,
                                          const typename Logits<DT>::Element *x) const {
    const uint32_t lane = threadIdx.x & 63u;
    float logit = token < a.vocabulary ? logit_value(x[token]) : -__builtin_inff();
    const MaxSum total = row_total(a, row, part, inv_t * kLog2e);
    const RowScore score{total.m, inv_t, logf(total.s)};
    if (lane == 0 && a.out_lse) a.out_lse[row] = score.lse();
    uint32_t id = token;
    for (uint32_t i = lane; i < a.token_count; i += 64) {
      if (i != lane) {
        id = a.tokens[(uint64_t)row * a.token_stride + i];
        logit = id < a.vocabulary ? logit_value(x[id]) : -__builtin_inff();
      }
      a.out_logprobs[(uint64_t)row * a.token_count + i] = score.logprob(logit);
    }
    if (a.out_ranks) {
      const uint32_t rank = wave_sum_u32(ahead) + 1u;
      if (lane == 0) a.out_ranks[row] = token < a.vocabulary ? rank : 0u;
    }
    return score;
  }
};

// One row a wave.
template <int DT>
__global__ __launch_bounds__(64) void logprobs_kernel(ScoreLaunch a) {
  const uint32_t row = blockIdx.x;
  const auto *x = row_of<DT>(a.logits, (uint64_t)row * a.stride);
  RowWave<DT> wave;
  wave.load(a, row);
  wave.put(a, row, x);
}

// One row a block, with alternatives: up to N groups a thread. The last wave
// takes the row's totals and tokens while the others list.
template <int DT, uint32_t N>
__global__ __launch_bounds__(kTopWaves * 64) void alternatives_kernel(ScoreLaunch a) {
  static_assert(N <= kMostItems);
  __shared__ TopLds s;
  const uint32_t tid = threadIdx.x, row = blockIdx.x, k = a.top;
  const auto *x = row_of<DT>(a.logits, (uint64_t)row * a.stride);
  const float *maxima = a.maxima + (uint64_t)row * a.groups;
  uint32_t key[N];
  RowWave<DT> totals;
  if (tid < kListThreads) {
    float m[N];
#pragma unroll
    for (uint32_t i = 0; i < N; ++i)
      m[i] = *element(maxima, min(i * kListThreads + tid, a.groups - 1));
    uint32_t best = 0;
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) {
      key[i] = i * kListThreads + tid < a.groups ? listed_key(m[i]) : 0u;
      best = max(best, key[i]);
    }
    best = max(best, xor_u32<1>(best));
    if (k <= kShortTop) {
      best = max(best, xor_u32<2>(best));
      best = max(best, xor_u32<4>(best));
      if (tid % 8 == 0) s.unit[tid / 8] = best;
    } else {
      if (tid % 2 == 0) s.unit[tid / 2] = best;
    }
  } else {
    totals.load(a, row);
  }
  if (tid == 0) s.crowded = 0;
  __syncthreads();
  if (tid >= kListThreads) {
    const RowScore score = totals.put(a, row, x);
    if (tid == kListThreads) s.score = score;
  } else if (k <= kShortTop) {
    list_wave<DT, N, 1>(s, a, x, key);
  } else {
    list_wave<DT, N, 4>(s, a, x, key);
  }
  __syncthreads();
  uint32_t listed = 0;
  if (!s.crowded) {
#pragma unroll
    for (uint32_t w = 0; w < kListWaves; ++w) listed += s.count[w];
    if (k <= kShortTop)
      place_items<1>(s, a, row, listed);
    else
      place_items<3>(s, a, row, listed);
  } else {
    listed = crowded_best<DT, N>(s, a, row, x, maxima);
  }
  for (uint32_t i = listed + tid; i < k; i += kTopWaves * 64) {
    a.out_top_ids[(uint64_t)row * k + i] = kNoToken;
    a.out_top_logprobs[(uint64_t)row * k + i] = -__builtin_inff();
  }
}

// ---- the pass -----------------------------------------------------------------

// Each value's maximum with a neighbour's (as loaded_max takes it). A lane reads
// its neighbour two instructions after the value was written at the earliest:
// hence the wait in front.
#define JF_MAX_DPP(V, CTRL) "v_max_f32_dpp " V ", " V ", " V " " CTRL " row_mask:0xf bank_mask:0xf\n"
#define JF_MAX_STEP(NAME, CTRL)                                                                 \
  template <uint32_t N>                                                                         \
  __device__ __forceinline__ void NAME(float (&g)[N]) {                                         \
    static_assert(N == 2 || N == 4);                                                            \
    if constexpr (N == 2)                                                                       \
      asm("s_nop 1\n" JF_MAX_DPP("%0", CTRL) JF_MAX_DPP("%1", CTRL) : "+v"(g[0]), "+v"(g[1]));  \
    else                                                                                        \
      asm("s_nop 1\n" JF_MAX_DPP("%0", CTRL) JF_MAX_DPP("%1", CTRL) JF_MAX_DPP("%2", CTRL)      \
              JF_MAX_DPP("%3", CTRL)                                                            \
          : "+v"(g[0]), "+v"(g[1]), "+v"(g[2]), "+v"(g[3]));                                    \
  }
JF_MAX_STEP(max_pairs, "quad_perm:[1,0,3,2]")
JF_MAX_STEP(max_quads, "quad_perm:[2,3,0,1]")
JF_MAX_STEP(max_eights, "row_half_mirror")  // of quads that agree
JF_MAX_STEP(max_sixteens, "row_mirror")     // of eights that agree
#undef JF_MAX_STEP
#undef JF_MAX_DPP

// A block's chunk of a row, N slabs.
template <int DT, uint32_t N, bool RANK, bool TOP>
__global__ __launch_bounds__(256) void score_kernel(ScoreLaunch a) {
  constexpr uint32_t VEC = Logits<DT>::VEC, SLAB = kSlab<DT>, CHUNK = N * SLAB;
  __shared__ MaxSum wave_part[4];
  __shared__ uint32_t wave_ahead[4];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  const uint32_t row = blockIdx.x / a.segments, segment = blockIdx.x - row * a.segments;
  const uint32_t V = a.vocabulary;
  const auto *x = row_of<DT>(a.logits, (uint64_t)row * a.stride);
  // The chunk first: what the row's temperature and target are is asked for
  // while it arrives.
  const uint32_t base = segment * CHUNK;
  LogitWords w[N];
  load_chunk<DT>(x, base, V, kPastMinusInfinity<DT>, w);
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
  float part[N];
#pragma unroll
  for (uint32_t j = 0; j < N; ++j) part[j] = vector_max<DT>(w[j]);
  add_vectors<DT>(run, w, part, c);
  if constexpr (RANK) {
    if (target < V) {
      // Ids before the target's are ahead of it at equal logits too.
      const bool mixed = target - base < CHUNK;
      const float least = base < target ? at_target : above_target;
#pragma unroll
      for (uint32_t j = 0; j < N; ++j) {
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
    // A group's 64 tokens lie in 16 (f32) or 8 (bf16) neighbouring lanes, of
    // which the j-th writes the group of vector j: a wave's store is a run.
    constexpr uint32_t LANES = kScoreGroup / VEC;
    if (ballot(run.s != run.s)) {
      // A NaN among them: a signalling one has taken others' places.
#pragma unroll
      for (uint32_t j = 0; j < N; ++j) {
        float v[VEC];
        unpack<DT>(w[j], v);
        part[j] = -__builtin_inff();
#pragma unroll
        for (uint32_t e = 0; e < VEC; ++e) part[j] = v[e] > part[j] ? v[e] : part[j];
      }
    }
    max_pairs(part);
    max_quads(part);
    max_eights(part);
    if constexpr (DT == 0) max_sixteens(part);
    float own = part[0];
#pragma unroll
    for (uint32_t j = 1; j < N; ++j) own = tid % LANES == j ? part[j] : own;
    if (tid % LANES < N)
      a.maxima[(uint64_t)row * a.groups + base / kScoreGroup + tid / LANES * N + tid % LANES] =
          own;
  }
  run = wave_join(run, c);
  if constexpr (RANK) ahead = wave_sum_u32(ahead);
  if (lane == 0) {
    wave_part[wave] = run;
    wave_ahead[wave] = ahead;
  }
  __syncthreads();
  if (tid == 0) {
    const MaxSum total = join(join(wave_part[0], wave_part[1], c),
                              join(wave_part[2], wave_part[3], c), c);
    const uint64_t at = (uint64_t)row * a.segments + segment;
    a.partials[at] = make_float2(total.m, total.s);
    if constexpr (RANK)
      a.aheads[at] = wave_ahead[0] + wave_ahead[1] + wave_ahead[2] + wave_ahead[3];
  }
}

// The places for groups that a thread holds: it asks for all of them, there or
// not (64 rows x 32,000 tokens, a group a thread: 10.3 us with 8 places, 10.9 with
// 16; x 151,936, five of them: 15.5 and 15.9; with 6 or 2 no less).
template <int DT>
void launch_alternatives(const ScoreLaunch &a, hipStream_t stream) {
  const dim3 rows(a.row_count), block(kTopWaves * 64);
  if (a.groups <= 8 * kListThreads)
    hipLaunchKernelGGL((alternatives_kernel<DT, 8>), rows, block, 0, stream, a);
  else
    hipLaunchKernelGGL((alternatives_kernel<DT, kMostItems>), rows, block, 0, stream, a);
}

}  // namespace

int launch_score(const ScoreLaunch &a, uint32_t dtype, void *stream) {
  const dim3 grid(a.row_count * a.segments);
  const bool top = a.top != 0, rank = a.out_ranks != nullptr;
#define JF_SCORE(DT, N, RANK, TOP)                                     \
  if (dtype == DT && a.vectors == N && rank == RANK && top == TOP)     \
  hipLaunchKernelGGL((score_kernel<DT, N, RANK, TOP>), grid, dim3(256), 0, (hipStream_t)stream, a)
#define JF_SCORE_ALL(DT, N)      \
  JF_SCORE(DT, N, false, false); \
  JF_SCORE(DT, N, false, true);  \
  JF_SCORE(DT, N, true, false);  \
  JF_SCORE(DT, N, true, true)
  JF_SCORE_ALL(0, 2);
  JF_SCORE_ALL(0, 4);
  JF_SCORE_ALL(1, 2);
  JF_SCORE_ALL(1, 4);
#undef JF_SCORE_ALL
#undef JF_SCORE
  return (int)hipGetLastError();
}

int launch_logprobs(const ScoreLaunch &a, uint32_t dtype, void *stream) {
  const hipStream_t st = (hipStream_t)stream;
  if (a.top && dtype == 0)
    launch_alternatives<0>(a, st);
  else if (a.top)
    launch_alternatives<1>(a, st);
  else if (dtype == 0)
    hipLaunchKernelGGL((logprobs_kernel<0>), dim3(a.row_count), dim3(64), 0, st, a);
  else
    hipLaunchKernelGGL((logprobs_kernel<1>), dim3(a.row_count), dim3(64), 0, st, a);
  return (int)hipGetLastError();
}

}  // namespace jf
