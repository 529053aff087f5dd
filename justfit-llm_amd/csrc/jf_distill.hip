// The distillation's backward pass on gfx950:
//   dz_j = g / T * (P / S * exp((z_j - m) / T) - [j listed] p_j),
// with the row's maximum m, P / S (the list's mass over the sum of
// exponentials) and the listed probabilities as the forward pass saved them.
//
// One read of the logits and one write of the gradient; a block takes a chunk
// of a row. Each of the list's slots is a thread's: a slot whose token lies in
// the chunk marks it in a bitmap and leaves its place in the list in a byte
// map, so the lane that holds the token subtracts p in registers and every
// element is stored once (also where the gradient overwrites the logits).
#include <hip/hip_runtime.h>

#include "jf_logits.h"

namespace jf {

namespace {

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
  const float inv_t = 1.0f / a.temperature, c = inv_t * 1.44269504088896341f;
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
        v[e] = weight * __builtin_amdgcn_exp2f((v[e] - m) * c);
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

int launch_distill_grad(const DistillGradLaunch &a, uint32_t dtype, void *stream) {
  const dim3 grid(a.row_count * a.chunks), block(256);
  if (dtype == 0)
    hipLaunchKernelGGL((distill_grad_kernel<0>), grid, block, 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL((distill_grad_kernel<1>), grid, block, 0, (hipStream_t)stream, a);
  return (int)hipGetLastError();
}

}  // namespace jf
