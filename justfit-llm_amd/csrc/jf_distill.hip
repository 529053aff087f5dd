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
// Both at once, for many rows: a block takes a whole row, reads it for m and S
// and reads it again for the gradient. The rows in flight (two a CU) fit the
// Infinity Cache, which serves the second reading, so HBM sees one read and one
// write.
#include <hip/hip_runtime.h>

#include "jf_logits.h"

namespace jf {

namespace {

// A row's list, worked out by one wave, SLOTS slots a lane: slot i * 64 + lane
// is element i of its lane.
template <int DT, uint32_t SLOTS>
struct Teacher {
  uint32_t id[SLOTS];
  float logit[SLOTS], log_p[SLOTS], p[SLOTS];
  bool valid[SLOTS];  // a token, and its first slot
  float mass;

  // `listed` is LDS for 64 * SLOTS ids.
  __device__ __forceinline__ void load(const ScoreLaunch &a, uint32_t row,
                                       const typename Logits<DT>::Element *x, float inv_t,
                                       uint32_t *listed) {
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
      listed[k] = id[i];
    }
    __builtin_amdgcn_wave_barrier();  // the wave's own LDS, in order
#pragma unroll 8
    for (uint32_t k = 0; k < K; ++k) {
      const uint32_t other = listed[k];
#pragma unroll
      for (uint32_t i = 0; i < SLOTS; ++i)
        valid[i] = valid[i] && !(k < i * 64 + lane && other == id[i]);
    }
    float first = -__builtin_inff();
#pragma unroll
    for (uint32_t i = 0; i < SLOTS; ++i) {
      log_p[i] = valid[i] ? value[i] : -__builtin_inff();
      if (a.normalize) log_p[i] *= inv_t;
      first = __builtin_fmaxf(first, log_p[i]);
    }
    if (a.normalize) {
      first = finite_reference(wave_max_f32(first));
      float sum = 0.0f;
#pragma unroll
      for (uint32_t i = 0; i < SLOTS; ++i) {
        log_p[i] -= first;
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
      saved[1] = weight(total);
    }
#pragma unroll
    for (uint32_t i = 0; i < SLOTS; ++i)
      if (i * 64 + lane < K) saved[2 + i * 64 + lane] = valid[i] ? p[i] : -1.0f;
  }
  // P / S; 0 with no list, or no student probability anywhere: then there are
  // no exponentials to add.
  __device__ __forceinline__ float weight(const MaxSum &total) const {
    return mass == 0.0f || total.s == 0.0f ? 0.0f : mass / total.s;
  }
};

template <int DT, uint32_t SLOTS>
__global__ __launch_bounds__(64) void distill_loss_kernel(ScoreLaunch a) {
  __shared__ uint32_t listed[64 * SLOTS];
  const uint32_t row = blockIdx.x;
  const auto *x = row_of<DT>(a.logits, (uint64_t)row * a.stride);
  const float inv_t = 1.0f / a.temperature;
  Teacher<DT, SLOTS> t;
  t.load(a, row, x, inv_t, listed);
  const MaxSum total = row_total(a, row, inv_t * kLog2e);
  t.put(a, row, total, RowScore{total.m, inv_t, logf(total.s)});
}

constexpr uint32_t kStepThreads = 1024;
constexpr uint32_t kStepWaves = kStepThreads / 64;
constexpr uint32_t kStepLoads = 2;  // vectors a thread has in flight

template <int DT, uint32_t SLOTS>
__global__ __launch_bounds__(kStepThreads, 8) void distill_step_kernel(ScoreLaunch a,
                                                                       DistillGradLaunch g) {
  constexpr uint32_t VEC = Logits<DT>::VEC, SLAB = kStepThreads * VEC;
  extern __shared__ uint32_t marked[];  // a bit a token
  __shared__ uint32_t listed[64 * SLOTS];
  __shared__ float share[64 * SLOTS];
  __shared__ MaxSum part[kStepWaves];
  __shared__ float weight;
  const uint32_t tid = threadIdx.x, wave = tid >> 6, lane = tid & 63u, row = blockIdx.x;
  const uint32_t V = a.vocabulary;
  const auto *z = row_of<DT>(a.logits, (uint64_t)row * a.stride);
  auto *dz = row_of<DT>(g.grad, (uint64_t)row * g.grad_stride);
  const float inv_t = 1.0f / a.temperature, c = inv_t * kLog2e;
  const float scale = g.grad_loss[(uint64_t)row * g.grad_loss_stride] * inv_t;
  for (uint32_t i = tid; i < (V + 31) / 32; i += kStepThreads) marked[i] = 0;
  MaxSum run{-__builtin_inff(), 0.0f};
  for (uint32_t base = 0; base < V; base += kStepLoads * SLAB) {
    LogitWords w[kStepLoads];
    float top[kStepLoads];
    if (base + kStepLoads * SLAB <= V) {
#pragma unroll
      for (uint32_t j = 0; j < kStepLoads; ++j)
        w[j] = *(const typename Logits<DT>::Words *)(z + base + j * SLAB + tid * VEC);
    } else {
#pragma unroll
      for (uint32_t j = 0; j < kStepLoads; ++j)
        w[j] = load_words<DT>(z, base + j * SLAB + tid * VEC, V, kPastMinusInfinity<DT>);
    }
#pragma unroll
    for (uint32_t j = 0; j < kStepLoads; ++j) top[j] = vector_max<DT>(w[j]);
    add_vectors<DT>(run, w, top, c);
  }
  run = wave_join(run, c);
  if (lane == 0) part[wave] = run;
  __syncthreads();
  MaxSum total = lane < kStepWaves ? part[lane] : MaxSum{-__builtin_inff(), 0.0f};
  total = wave_join(total, c);
  if (wave == 0) {
    Teacher<DT, SLOTS> t;
    t.load(a, row, z, inv_t, listed);
    t.put(a, row, total, RowScore{total.m, inv_t, logf(total.s)});
    if (lane == 0) weight = scale * t.weight(total);
#pragma unroll
    for (uint32_t i = 0; i < SLOTS; ++i) {
      share[i * 64 + lane] = t.valid[i] ? scale * t.p[i] : 0.0f;
      if (t.valid[i] && scale != 0.0f) atomicOr(&marked[t.id[i] >> 5], 1u << (t.id[i] & 31u));
    }
  }
  __syncthreads();
  const float weight_ = weight;
  // A row with no list, or whose loss nothing follows from, has no gradient.
  const bool any = weight_ != 0.0f && scale != 0.0f;
  const float m = total.m;
  for (uint32_t base = 0; base < V; base += kStepLoads * SLAB) {
    LogitWords w[kStepLoads];
    if (any) {
      if (base + kStepLoads * SLAB <= V) {
#pragma unroll
        for (uint32_t j = 0; j < kStepLoads; ++j)
          w[j] = *(const typename Logits<DT>::Words *)(z + base + j * SLAB + tid * VEC);
      } else {
#pragma unroll
        for (uint32_t j = 0; j < kStepLoads; ++j)
          w[j] = load_words<DT>(z, base + j * SLAB + tid * VEC, V, 0);
      }
    }
#pragma unroll
    for (uint32_t j = 0; j < kStepLoads; ++j) {
      const uint32_t token = base + j * SLAB + tid * VEC;
      if (token >= V) continue;
      float v[VEC];
      if (any) {
        unpack<DT>(w[j], v);
#pragma unroll
        for (uint32_t e = 0; e < VEC; ++e)
          v[e] = weight_ * exp_below(v[e], m, c);
      } else {
#pragma unroll
        for (uint32_t e = 0; e < VEC; ++e) v[e] = 0.0f;
      }
      const uint32_t bits = (marked[token >> 5] >> (token & 31u)) & ((1u << VEC) - 1u);
      if (bits) {
#pragma unroll
        for (uint32_t e = 0; e < VEC; ++e)
          if (bits >> e & 1u) {
            uint32_t k = 0;
            while (listed[k] != token + e) ++k;
            v[e] -= share[k];
          }
      }
      store_words<DT>(dz, token, V, pack<DT>(v));
    }
  }
}

template <int DT>
__global__ __launch_bounds__(256) void distill_grad_kernel(DistillGradLaunch a) {
  constexpr uint32_t VEC = Logits<DT>::VEC, SLAB = kSlab<DT>, LOADS = kLoads<DT>;
  __shared__ uint32_t listed[kScoreChunk / 32];
  __shared__ uint8_t slot[kScoreChunk];  // read at listed tokens only
  __shared__ float share[kTeacherTokens];
  const uint32_t tid = threadIdx.x;
  const uint32_t row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks;
  const uint32_t base = chunk * kScoreChunk, V = a.vocabulary, K = a.teacher_count;
  const auto *z = row_of<DT>(a.logits, (uint64_t)row * a.stride);
  auto *dz = row_of<DT>(a.grad, (uint64_t)row * a.grad_stride);
  const float *saved = a.saved + (uint64_t)row * (2 + K);
  const float inv_t = 1.0f / a.temperature, c = inv_t * kLog2e;
  const float scale = a.grad_loss[(uint64_t)row * a.grad_loss_stride] * inv_t;
  const float m = saved[0], weight = scale * saved[1];
  // A row with no list, or whose loss nothing follows from, is not read.
  const bool read = weight != 0.0f && scale != 0.0f;
  LogitWords w[LOADS];
  if (read) load_chunk<DT>(z, base, V, 0, w);
  listed[tid] = 0;
  __syncthreads();
  if (tid < K && scale != 0.0f) {
    const uint32_t id = a.teacher_ids[(uint64_t)row * a.teacher_stride + tid], at = id - base;
    const float p = saved[2 + tid];
    if (at < kScoreChunk && id < V && p >= 0.0f) {
      share[tid] = scale * p;
      slot[at] = (uint8_t)tid;
      atomicOr(&listed[at >> 5], 1u << (at & 31u));
    }
  }
  __syncthreads();
#pragma unroll
  for (uint32_t j = 0; j < LOADS; ++j) {
    const uint32_t at = j * SLAB + tid * VEC, token = base + at;
    if (token >= V) continue;
    float v[VEC];
    if (read) {
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
    store_words<DT>(dz, token, V, pack<DT>(v));
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
  const uint32_t bits = (a.vocabulary + 31) / 32 * sizeof(uint32_t);  // 64 KB at most
  const bool one = a.teacher_count <= 64;
  if (dtype == 0 && one)
    hipLaunchKernelGGL((distill_step_kernel<0, 1>), rows, block, bits, st, a, g);
  else if (dtype == 0)
    hipLaunchKernelGGL((distill_step_kernel<0, 4>), rows, block, bits, st, a, g);
  else if (one)
    hipLaunchKernelGGL((distill_step_kernel<1, 1>), rows, block, bits, st, a, g);
  else
    hipLaunchKernelGGL((distill_step_kernel<1, 4>), rows, block, bits, st, a, g);
  return (int)hipGetLastError();
}

int launch_distill_grad(const DistillGradLaunch &a, uint32_t dtype, void *stream) {
  const dim3 grid(a.row_count * a.chunks), block(256);
  if (dtype == 0)
    hipLaunchKernelGGL((distill_grad_kernel<0>), grid, block, 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL((distill_grad_kernel<1>), grid, block, 0, (hipStream_t)stream, a);
  return (int)hipGetLastError();
}

}  // namespace jf
