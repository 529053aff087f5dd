// Processed logits on gfx950: y = mask(bias(penalize(x))) of every token of a
// row, written out or in place. penalize is the selection's own (jf_device.h),
// so a sampler that reads y draws from the distribution that the selection
// with the same policy draws from.
//
// Only a few tokens of a row are edited: the row's penalty entries, its extra
// tokens and its biases, sorted lists in buckets of 2048 tokens. A block takes
// one chunk of a row. It works the chunk's edited values out first, in fp32,
// in three steps with a barrier between them (penalties, extra tokens that the
// table does not hold, biases on what the first two left), into an LDS tile
// that is written only at those tokens, with a bitmap of them; then the
// chunk's vectors go from registers to the output, each lane replacing what
// the bitmap and the mask words say.
//
// A vector is loaded only if one of its tokens is admitted and not edited, and
// in place written only if one of them changes: a grammar's row, which drops
// nearly all of its tokens, is written without being read, and an unmasked row
// in place touches nothing but its edits.
#include <hip/hip_runtime.h>

#include "jf_logits.h"

namespace jf {

namespace {

struct ProcessLds {
  float value[kScoreChunk];              // written and read at edited tokens only
  uint32_t edited[kScoreChunk / 32];
  uint32_t admitted[kScoreChunk / 32];
  uint32_t extras[16];
};

// VEC bits of a bitmap from token `at` of the chunk (a multiple of VEC).
template <uint32_t VEC>
__device__ __forceinline__ uint32_t bits_at(const uint32_t *map, uint32_t at) {
  return (map[at >> 5] >> (at & 31u)) & ((1u << VEC) - 1u);
}

template <int DI, int DO>
__global__ __launch_bounds__(256) void process_kernel(ProcessLaunch a) {
  constexpr uint32_t VEC = Logits<DI>::VEC, SLAB = kSlab<DI>, LOADS = kLoads<DI>;
  constexpr uint32_t ALL = (1u << VEC) - 1u;
  __shared__ ProcessLds s;
  const uint32_t tid = threadIdx.x;
  const uint32_t row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks;
  const uint32_t base = chunk * kScoreChunk, V = a.vocabulary;
  const ProcessRow p = a.rows[row];
  const auto *x = row_of<DI>(a.logits, (uint64_t)row * a.stride);
  auto *y = row_of<DO>(a.out, (uint64_t)row * a.out_stride);
  const bool masked = (p.flags & (kProcessMasked | kProcessStops)) != 0;

  // An unmasked row that is written elsewhere needs every vector: ask first.
  const bool whole = !masked && !a.in_place;
  LogitWords w[LOADS];
  if (whole) load_chunk<DI>(x, base, V, 0, w);

  uint32_t pen0 = 0, pen1 = 0, bias0 = 0, bias1 = 0;
  const uint32_t b0 = chunk * (kScoreChunk / kPenaltyBucket);
  const uint32_t b1 = min(b0 + kScoreChunk / kPenaltyBucket, a.buckets);
  if (p.penalty_row != kNoRow) {
    const uint32_t *off = a.pen_offsets + (uint64_t)p.penalty_row * (a.buckets + 1);
    pen0 = off[b0];
    pen1 = off[b1];
  }
  if (p.bias_row != kNoRow) {
    const uint32_t *off = a.bias_offsets + (uint64_t)p.bias_row * (a.buckets + 1);
    bias0 = off[b0];
    bias1 = off[b1];
  }
  s.edited[tid] = 0;
  if (masked) {
    // Tokens past the vocabulary are never stored; words past it not read.
    const uint32_t word = base / 32 + tid;
    uint32_t bits = 0xffffffffu;
    if ((p.flags & kProcessMasked) && word < (V + 31) / 32)
      bits = a.masks[(uint64_t)p.mask_row * a.mask_stride + word];
    if (p.flags & kProcessStops) {
      if (a.stop0 / 32 == word) bits &= ~(1u << (a.stop0 % 32));
      if (a.stop1 / 32 == word) bits &= ~(1u << (a.stop1 % 32));
    }
    s.admitted[tid] = bits;
  }
  if (tid < p.extra_count) s.extras[tid] = a.extra[p.extra_offset + tid];
  const bool edits = pen1 > pen0 || bias1 > bias0 || p.extra_count;
  if (edits || masked) __syncthreads();
  // A dropped token's edits are not worked out, nor its logit read.
  const auto dropped = [&](uint32_t at) {
    return masked && !(s.admitted[at >> 5] >> (at & 31u) & 1u);
  };
  if (pen1 > pen0) {
    const PenaltyEntry *list = a.pen_entries + (uint64_t)p.penalty_row * a.pen_max_entries;
    for (uint32_t i = pen0 + tid; i < pen1; i += 256) {
      const PenaltyEntry e = list[i];
      const uint32_t at = e.token - base;
      if (dropped(at)) continue;
      uint32_t count = e.word & kCountMask;
      for (uint32_t k = 0; k < p.extra_count; ++k) count += s.extras[k] == e.token;
      s.value[at] = penalize(logit_value(x[e.token]), count, p.repetition, p.repetition_inverse,
                             p.presence, p.frequency);
      atomicOr(&s.edited[at >> 5], 1u << (at & 31u));
    }
  }
  if (p.extra_count) {
    // Extra tokens outside the table, each at its first place in the list.
    __syncthreads();
    if (tid < p.extra_count) {
      const uint32_t token = s.extras[tid], at = token - base;
      bool take = token < V && at < kScoreChunk && !dropped(at) &&
                  !(s.edited[at >> 5] >> (at & 31u) & 1u);
      uint32_t count = 0;
      for (uint32_t k = 0; k < p.extra_count; ++k) {
        count += s.extras[k] == token;
        take = take && !(k < tid && s.extras[k] == token);
      }
      // One wave holds all of them: its reads of the bitmap come before this.
      if (take) {
        s.value[at] = penalize(logit_value(x[token]), count, p.repetition, p.repetition_inverse,
                               p.presence, p.frequency);
        atomicOr(&s.edited[at >> 5], 1u << (at & 31u));
      }
    }
  }
  if (bias1 > bias0) {
    __syncthreads();
    const PenaltyEntry *list = a.bias_entries + (uint64_t)p.bias_row * a.bias_max_entries;
    for (uint32_t i = bias0 + tid; i < bias1; i += 256) {
      const PenaltyEntry e = list[i];
      const uint32_t at = e.token - base;
      if (dropped(at)) continue;
      const float bias = u2f(e.word);
      // Only this token's own bias can set its bit meanwhile.
      const float v = s.edited[at >> 5] >> (at & 31u) & 1u ? s.value[at] : logit_value(x[e.token]);
      // A ban holds whatever the logit.
      s.value[at] = bias == -__builtin_inff() ? bias : v + bias;
      atomicOr(&s.edited[at >> 5], 1u << (at & 31u));
    }
  }
  if (edits) __syncthreads();

  if (!whole) {
#pragma unroll
    for (uint32_t j = 0; j < LOADS; ++j) {
      const uint32_t at = j * SLAB + tid * VEC, token = base + at;
      if (token >= V) continue;
      const uint32_t edited = edits ? bits_at<VEC>(s.edited, at) : 0u;
      const uint32_t admitted = masked ? bits_at<VEC>(s.admitted, at) : ALL;
      const bool write = !a.in_place || edited || admitted != ALL;
      w[j] = LogitWords{};
      if (write && (admitted & ~edited)) w[j] = load_words<DI>(x, token, V, 0);
    }
  }
#pragma unroll
  for (uint32_t j = 0; j < LOADS; ++j) {
    const uint32_t at = j * SLAB + tid * VEC, token = base + at;
    if (token >= V) continue;
    const uint32_t edited = edits ? bits_at<VEC>(s.edited, at) : 0u;
    const uint32_t admitted = masked ? bits_at<VEC>(s.admitted, at) : ALL;
    if (a.in_place && !edited && admitted == ALL) continue;
    if (DI == DO && !edited && admitted == ALL) {
      store_words<DO>(y, token, V, w[j]);
      continue;
    }
    float v[VEC];
    unpack<DI>(w[j], v);
#pragma unroll
    for (uint32_t e = 0; e < VEC; ++e) {
      if (edited >> e & 1u) v[e] = s.value[at + e];
      if (!(admitted >> e & 1u)) v[e] = -__builtin_inff();
    }
    if constexpr (DI == DO) {
      store_words<DO>(y, token, V, pack<DO>(v));
    } else if constexpr (DI == 1) {
      float half[4];
#pragma unroll
      for (uint32_t h = 0; h < 2; ++h) {
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) half[e] = v[h * 4 + e];
        if (token + h * 4 < V) store_words<0>(y, token + h * 4, V, pack<0>(half));
      }
    } else if (token + VEC <= V) {
      typedef uint32_t Pair __attribute__((ext_vector_type(2)));
      typedef Pair PairAt2 __attribute__((aligned(2)));
      *(PairAt2 *)(y + token) = Pair{floats_to_bf16(v[0], v[1]), floats_to_bf16(v[2], v[3])};
    } else {
#pragma unroll
      for (uint32_t e = 0; e < VEC; ++e)
        if (token + e < V) y[token + e] = logit_of<DO>(v[e]);
    }
  }
}

}  // namespace

int launch_process(const ProcessLaunch &a, uint32_t dtype, uint32_t out_dtype, void *stream) {
  const dim3 grid(a.row_count * a.chunks), block(256);
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == 0 && out_dtype == 0)
    hipLaunchKernelGGL((process_kernel<0, 0>), grid, block, 0, st, a);
  else if (dtype == 0)
    hipLaunchKernelGGL((process_kernel<0, 1>), grid, block, 0, st, a);
  else if (out_dtype == 0)
    hipLaunchKernelGGL((process_kernel<1, 0>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((process_kernel<1, 1>), grid, block, 0, st, a);
  return (int)hipGetLastError();
}

}  // namespace jf
