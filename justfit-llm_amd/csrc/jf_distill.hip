// Distillation on gfx950: with q = softmax(z / T) over the vocabulary and p over
// a row's listed tokens, the loss sum p_k (ln p_k - ln q_k) and
//   dz_j = g / T * (P / S * exp((z_j - m) / T) - [j listed] p_j),
// m the row's maximum, S its sum of exponentials, P = sum p_k.
//
// Forward: the pass of jf_score.hip leaves the rows' maxima and sums, and one
// wave a row works out the list. Backward: one read of the logits and one write
// of the gradient; a block takes a chunk of a row. A listed token in the chunk
// is marked in a bitmap and its place in the list left in a byte map, so the
// lane that holds the token subtracts p in registers and every element is
// stored once (also where the gradient overwrites the logits).
//
// Both at once, for short rows and for many: a block takes a whole row, reads it for m and S,
// and takes it again for the gradient, a third of a 300 KB row from registers,
// the rest from the caches. What the caches serve counts as well (their fabric
// carries about 6 TB/s, read and written), so what is held is time: 2048 rows x
// 151,936 bf16, 622 MB read and as much written, take 260 us; reading every row
// twice 290, and the passes apart 353. Holding the whole row takes a CU's
// registers for one block, which then reads, computes and writes in turn: 280.
// The listed tokens' elements are stored once more behind the row's: looking
// every vector's up cost 40 us.
//
// Gradients go past the caches (nontemporal stores; 256 rows: 32 us against 41),
// which keeps the rows being read there.
#include <hip/hip_runtime.h>

#include "jf_logits.h"

namespace jf {

namespace {

// P / S; 0 with no list, or no student probability anywhere: then there are no
// exponentials to add.
__device__ __forceinline__ float list_weight(float mass, const MaxSum &total) {
  return mass == 0.0f || total.s == 0.0f ? 0.0f : mass / total.s;
}

constexpr uint32_t kHolderBits = 11, kHolders = 1u << kHolderBits;
static_assert(kTeacherTokens <= 256, "a slot is a byte");

// A row's list, worked out by one wave, SLOTS slots a lane: slot i * 64 + lane
// is element i of its lane.
template <int DT, uint32_t SLOTS>
struct Teacher {
  uint32_t id[SLOTS];
  float logit[SLOTS], log_p[SLOTS], p[SLOTS];
  bool valid[SLOTS];  // a token, and its first slot
  float mass;

  // `holder` is LDS of kHolders bytes.
  __device__ __forceinline__ void load(const ScoreLaunch &a, uint32_t row,
                                       const typename Logits<DT>::Element *x, float inv_t,
                                       uint8_t *holder) {
    const uint32_t lane = threadIdx.x & 63u, K = a.teacher_count;
    float value[SLOTS];
#pragma unroll
    for (uint32_t i = 0; i < SLOTS; ++i) {
      const uint32_t k = i * 64 + lane;
      id[i] = kNoToken;
      value[i] = -__builtin_inff();
      if (k < K) {
        id[i] = a.teacher_ids[(uint64_t)row * a.teacher_stride + k];
        value[i] = a.teacher_values[(uint64_t)row * a.teacher_stride + k];
      }
      valid[i] = id[i] < a.vocabulary;
      logit[i] = valid[i] ? logit_value(x[id[i]]) : 0.0f;
    }
    keep_first(holder);
    float most = -__builtin_inff();
#pragma unroll
    for (uint32_t i = 0; i < SLOTS; ++i) {
      log_p[i] = valid[i] ? value[i] : -__builtin_inff();
      most = __builtin_fmaxf(most, log_p[i]);
    }
    if (a.normalize) {
      // Apart from the largest before the scale: their common offset costs no
      // bits, and u / T may pass the range.
      most = finite_reference(wave_max_f32(most));
      float sum = 0.0f;
#pragma unroll
      for (uint32_t i = 0; i < SLOTS; ++i) {
        log_p[i] = (log_p[i] - most) * inv_t;
        sum += expf(log_p[i]);
      }
      sum = logf(wave_sum_f32(sum));
      // -infinity stays: a list of nothing else has no mass.
#pragma unroll
      for (uint32_t i = 0; i < SLOTS; ++i)
        if (log_p[i] != -__builtin_inff()) log_p[i] -= sum;
    }
    mass = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < SLOTS; ++i) {
      p[i] = valid[i] ? expf(log_p[i]) : 0.0f;
      mass += p[i];
    }
    mass = wave_sum_f32(mass);
  }

  // Drops the slots whose token an earlier one lists. Every slot writes itself
  // down at its token's place in a table: all but one of those that share a token
  // then find another one there, as few others do, and each such token is looked
  // up among all slots. (Comparing every slot with every one before it took 98
  // slots a row 5 us.)
  __device__ __forceinline__ void keep_first(uint8_t *holder) {
    const uint32_t lane = threadIdx.x & 63u;
    const auto place = [&](uint32_t i) { return id[i] * 2654435761u >> (32 - kHolderBits); };
#pragma unroll
    for (uint32_t i = 0; i < SLOTS; ++i)
      if (valid[i]) holder[place(i)] = (uint8_t)(i * 64 + lane);
    __builtin_amdgcn_wave_barrier();  // the wave's own LDS, in order
    uint64_t look[SLOTS];
#pragma unroll
    for (uint32_t i = 0; i < SLOTS; ++i)
      look[i] = ballot(valid[i] && holder[place(i)] != (uint8_t)(i * 64 + lane));
#pragma unroll
    for (uint32_t i = 0; i < SLOTS; ++i) {
      while (look[i]) {
        const uint32_t token = readlane_u32(id[i], __builtin_ctzll(look[i]));
        bool first = true;
#pragma unroll
        for (uint32_t j = 0; j < SLOTS; ++j) {
          const bool same = valid[j] && id[j] == token;
          const uint64_t lanes = ballot(same);
          valid[j] = valid[j] && !(same && !(first && lane == (uint32_t)__builtin_ctzll(lanes)));
          first = first && !lanes;
          look[j] &= ~lanes;
        }
      }
    }
  }

  // The row's outputs, and what the backward pass takes: the maximum, the
  // list's mass over the sum, and each slot's probability (-1: no token, or
  // one that an earlier slot lists).
  __device__ __forceinline__ void put(const ScoreLaunch &a, uint32_t row, const MaxSum &total,
                                      const RowScore &score) const {
    const uint32_t lane = threadIdx.x & 63u, K = a.teacher_count;
    float loss = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < SLOTS; ++i)
      // A token of no teacher probability adds nothing, whatever the student's.
      if (p[i] != 0.0f) loss += p[i] * (log_p[i] - score.logprob(logit[i]));
    loss = wave_sum_f32(loss);
    if (lane == 0) {
      a.out_loss[row] = loss;
      if (a.out_lse) a.out_lse[row] = score.lse();
    }
    if (!a.saved) return;
    float *saved = a.saved + (uint64_t)row * (2 + K);
    if (lane == 0) {
      saved[0] = total.m;
      saved[1] = list_weight(mass, total);
    }
#pragma unroll
    for (uint32_t i = 0; i < SLOTS; ++i)
      if (i * 64 + lane < K) saved[2 + i * 64 + lane] = valid[i] ? p[i] : -1.0f;
  }
};

template <int DT, uint32_t SLOTS>
__global__ __launch_bounds__(64) void distill_loss_kernel(ScoreLaunch a) {
  __shared__ uint8_t holder[kHolders];
  const uint32_t row = blockIdx.x;
  const auto *x = row_of<DT>(a.logits, (uint64_t)row * a.stride);
  const float inv_t = 1.0f / a.temperature;
  const MaxSum part = row_part(a, row);
  Teacher<DT, SLOTS> t;
  t.load(a, row, x, inv_t, holder);
  const MaxSum total = row_total(a, row, part, inv_t * kLog2e);
  t.put(a, row, total, RowScore{total.m, inv_t, logf(total.s)});
}

// A training step's block: two of them on a CU, so that one reads while the
// other computes or writes.
constexpr uint32_t kStepThreads = 512;
constexpr uint32_t kStepWaves = kStepThreads / 64;
constexpr uint32_t kQuad = 4;       // vectors a thread loads, adds and stores together
// Of them held from the first pass to the second: what the registers take
// beside a list of SLOTS a lane.
template <uint32_t SLOTS>
constexpr uint32_t kHeld = SLOTS == 1 ? 3 : 2;

template <int DT, uint32_t SLOTS>
__global__ __launch_bounds__(kStepThreads, 4) void distill_step_kernel(ScoreLaunch a,
                                                                       DistillGradLaunch g) {
  constexpr uint32_t VEC = Logits<DT>::VEC, SLAB = kStepThreads * VEC, QUAD = kQuad * SLAB,
                     HELD = kHeld<SLOTS>;
  using Words = typename Logits<DT>::Words;
  __shared__ uint8_t holder[kHolders];
  __shared__ MaxSum part[kStepWaves];
  __shared__ float mass;
  const uint32_t tid = threadIdx.x, wave = tid >> 6, lane = tid & 63u, row = blockIdx.x;
  const auto *logits = row_of<DT>(a.logits, (uint64_t)row * a.stride);
  auto *grad = row_of<DT>(g.grad, (uint64_t)row * g.grad_stride);
  // Vectors count from the gradient's last line before the row, `before` elements
  // ahead of it, so that every store covers whole lines: a row that starts within
  // one is stored in parts of lines otherwise (2048 rows x 151,935 bf16: 324 us,
  // 271 so). Nothing ahead of the row is read or written.
  const uint32_t before = (uint32_t)((uintptr_t)grad % 128 / sizeof(*grad));
  const auto *z = logits - before;
  auto *dz = grad - before;
  const uint32_t V = before + a.vocabulary, quads = V / QUAD;
  const float inv_t = 1.0f / a.temperature, c = inv_t * kLog2e;
  const float scale = g.grad_loss[(uint64_t)row * g.grad_loss_stride] * inv_t;
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
  // The first wave works the list out while the row arrives.
  Teacher<DT, SLOTS> t;
  if (wave == 0) {
    t.load(a, row, logits, inv_t, holder);
    if (lane == 0) mass = t.mass;
  }
  MaxSum run{-__builtin_inff(), 0.0f};
  const auto add = [&](const LogitWords (&w)[kQuad]) {
    float top[kQuad];
#pragma unroll
    for (uint32_t j = 0; j < kQuad; ++j) top[j] = vector_max<DT>(w[j]);
    add_vectors<DT>(run, w, top, c);
  };
#pragma unroll
  for (uint32_t q = 0; q < HELD; ++q)
    if (q < quads) add(held[q]);
  for (uint32_t q = HELD; q < quads; ++q) {
    LogitWords w[kQuad];
    load(q, w);
    add(w);
  }
  add(rest);
  run = wave_join(run, c);
  if (lane == 0) part[wave] = run;
  __syncthreads();
  // The held words anew, or the compiler keeps the values it unpacked above,
  // two registers a word.
#pragma unroll
  for (uint32_t q = 0; q < HELD; ++q)
#pragma unroll
    for (uint32_t j = 0; j < kQuad; ++j) asm volatile("" : "+v"(held[q][j]));
  MaxSum total = lane < kStepWaves ? part[lane] : MaxSum{-__builtin_inff(), 0.0f};
  total = wave_join(total, c);
  // A row with no list, or whose loss nothing follows from, has no gradient.
  const float m = total.m, listed_weight = list_weight(mass, total);
  const float weight = scale * listed_weight;
  const bool any = listed_weight != 0.0f && scale != 0.0f;
  const auto pulled = [&](float logit) { return any ? weight * exp_below(logit, m, c) : 0.0f; };
  const auto gradient = [&](const LogitWords &w) {
    float v[VEC];
    unpack<DT>(w, v);
#pragma unroll
    for (uint32_t e = 0; e < VEC; ++e) v[e] = pulled(v[e]);
    return pack<DT>(v);
  };
  const auto put = [&](uint32_t quad, const LogitWords (&w)[kQuad]) {
#pragma unroll
    for (uint32_t j = 0; j < kQuad; ++j) {
      const uint32_t token = quad * QUAD + j * SLAB + tid * VEC;
      const LogitWords d = gradient(w[j]);
      if (j == 0 && token < before)
        store_words<DT>(dz, token, V, d, before);
      else
        __builtin_nontemporal_store(d, (Words *)(dz + token));
    }
  };
  // The quads read again come first, the last read before the others.
  for (uint32_t q = quads; q-- > HELD;) {
    LogitWords w[kQuad];
    load(q, w);
    put(q, w);
  }
#pragma unroll
  for (uint32_t q = 0; q < HELD; ++q)
    if (q < quads) put(q, held[q]);
#pragma unroll
  for (uint32_t j = 0; j < kQuad; ++j) {
    const uint32_t token = quads * QUAD + j * SLAB + tid * VEC;
    if (token < V) store_words<DT>(dz, token, V, gradient(rest[j]), before);
  }
  if (wave == 0) t.put(a, row, total, RowScore{total.m, inv_t, logf(total.s)});
  // The listed tokens' elements anew, once every store above has completed.
  wait_memory();
  __syncthreads();
  if (wave == 0 && scale != 0.0f) {
#pragma unroll
    for (uint32_t i = 0; i < SLOTS; ++i)
      if (!(t.p[i] <= 0.0f)) grad[t.id[i]] = logit_of<DT>(pulled(t.logit[i]) - scale * t.p[i]);
  }
}

// LINES: chunks count from the gradient's last line before the row, as above, for
// rows that start within one (512 f32 rows x 151,935: 108.0 us, 113.5 otherwise; 96
// x 100,003 13.3 and 13.8; aligned rows take either way's time).
template <int DT, uint32_t N, bool LINES>
__global__ __launch_bounds__(256) void distill_grad_kernel(DistillGradLaunch a) {
  constexpr uint32_t VEC = Logits<DT>::VEC, SLAB = kSlab<DT>, CHUNK = N * SLAB;
  __shared__ uint32_t listed[CHUNK / 32];
  __shared__ uint8_t slot[CHUNK];  // read at listed tokens only
  __shared__ float share[kTeacherTokens];
  const uint32_t tid = threadIdx.x;
  const uint32_t row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks;
  const uint32_t base = chunk * CHUNK, K = a.teacher_count;
  const auto *z = row_of<DT>(a.logits, (uint64_t)row * a.stride);
  auto *dz = row_of<DT>(a.grad, (uint64_t)row * a.grad_stride);
  const uint32_t before = LINES ? (uint32_t)((uintptr_t)dz % 128 / sizeof(*dz)) : 0;
  const uint32_t V = before + a.vocabulary;
  if (LINES && base >= V) return;  // not every row reaches the last chunk
  z -= before;
  dz -= before;
  const float *saved = a.saved + (uint64_t)row * (2 + K);
  const float inv_t = 1.0f / a.temperature, c = inv_t * kLog2e;
  const float scale = a.grad_loss[(uint64_t)row * a.grad_loss_stride] * inv_t;
  const float m = saved[0], listed_weight = saved[1], weight = scale * listed_weight;
  // A row with no list, or whose loss nothing follows from, has no gradient.
  const bool any = listed_weight != 0.0f && scale != 0.0f;
  LogitWords w[N];
  if (any) load_chunk<DT>(z, base, V, 0, w, before);
  if (tid < CHUNK / 32) listed[tid] = 0;
  __syncthreads();
  if (tid < K && scale != 0.0f) {
    const uint32_t id = a.teacher_ids[(uint64_t)row * a.teacher_stride + tid];
    const uint32_t at = id + before - base;
    const float p = saved[2 + tid];
    // A token of no probability has no share, also of a gradient that is not finite.
    if (at < CHUNK && id < a.vocabulary && !(p <= 0.0f)) {
      share[tid] = scale * p;
      slot[at] = (uint8_t)tid;
      atomicOr(&listed[at >> 5], 1u << (at & 31u));
    }
  }
  __syncthreads();
#pragma unroll
  for (uint32_t j = 0; j < N; ++j) {
    const uint32_t at = j * SLAB + tid * VEC, token = base + at;
    if (token >= V) continue;
    float v[VEC];
    if (any) {
      unpack<DT>(w[j], v);
#pragma unroll
      for (uint32_t e = 0; e < VEC; ++e)
        v[e] = weight * exp_below(v[e], m, c);
    } else {
#pragma unroll
      for (uint32_t e = 0; e < VEC; ++e) v[e] = 0.0f;
    }
    const uint32_t bits = (listed[at >> 5] >> (at & 31u)) & ((1u << VEC) - 1u);
    if (bits) {
#pragma unroll
      for (uint32_t e = 0; e < VEC; ++e)
        if (bits >> e & 1u) v[e] -= share[slot[at + e]];
    }
    if (token >= before && token + VEC <= V)
      __builtin_nontemporal_store(pack<DT>(v), (typename Logits<DT>::Words *)(dz + token));
    else
      store_words<DT>(dz, token, V, pack<DT>(v), before);
  }
}

}  // namespace

int launch_distill_loss(const ScoreLaunch &a, uint32_t dtype, void *stream) {
  const dim3 rows(a.row_count), block(64);
  const hipStream_t st = (hipStream_t)stream;
  const bool one = a.teacher_count <= 64;
  if (dtype == 0 && one)
    hipLaunchKernelGGL((distill_loss_kernel<0, 1>), rows, block, 0, st, a);
  else if (dtype == 0)
    hipLaunchKernelGGL((distill_loss_kernel<0, 4>), rows, block, 0, st, a);
  else if (one)
    hipLaunchKernelGGL((distill_loss_kernel<1, 1>), rows, block, 0, st, a);
  else
    hipLaunchKernelGGL((distill_loss_kernel<1, 4>), rows, block, 0, st, a);
  return (int)hipGetLastError();
}

int launch_distill_step(const ScoreLaunch &a, const DistillGradLaunch &g, uint32_t dtype,
                        void *stream) {
  const dim3 rows(a.row_count), block(kStepThreads);
  const hipStream_t st = (hipStream_t)stream;
  const bool one = a.teacher_count <= 64;
  if (dtype == 0 && one)
    hipLaunchKernelGGL((distill_step_kernel<0, 1>), rows, block, 0, st, a, g);
  else if (dtype == 0)
    hipLaunchKernelGGL((distill_step_kernel<0, 4>), rows, block, 0, st, a, g);
  else if (one)
    hipLaunchKernelGGL((distill_step_kernel<1, 1>), rows, block, 0, st, a, g);
  else
    hipLaunchKernelGGL((distill_step_kernel<1, 4>), rows, block, 0, st, a, g);
  return (int)hipGetLastError();
}

int launch_distill_grad(const DistillGradLaunch &rows, uint32_t dtype, void *stream) {
  DistillGradLaunch a = rows;
  const uint32_t size = dtype == 0 ? 4 : 2, chunk = chunk_tokens(dtype, a.vectors);
  // Rows that start within a line may reach a chunk more.
  const bool lines = (uintptr_t)a.grad % 128 != 0 ||
                     (a.row_count > 1 && a.grad_stride * size % 128 != 0);
  a.chunks = (a.vocabulary + (lines ? 128 / size - 1 : 0) + chunk - 1) / chunk;
  const dim3 grid(a.row_count * a.chunks), block(256);
  const hipStream_t st = (hipStream_t)stream;
#define JF_GRAD(DT, N, LINES)                                \
  if (dtype == DT && a.vectors == N && lines == LINES)       \
  hipLaunchKernelGGL((distill_grad_kernel<DT, N, LINES>), grid, block, 0, st, a)
  JF_GRAD(0, 2, false);
  JF_GRAD(0, 2, true);
  JF_GRAD(0, 4, false);
  JF_GRAD(0, 4, true);
  JF_GRAD(1, 2, false);
  JF_GRAD(1, 2, true);
  JF_GRAD(1, 4, false);
  JF_GRAD(1, 4, true);
#undef JF_GRAD
  return (int)hipGetLastError();
}

}  // namespace jf
