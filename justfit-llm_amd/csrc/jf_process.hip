// Processed logits on gfx950: y = mask(bias(penalize(x))) of every token of a
// row, written out or in place. penalize is the selection's own (jf_device.h),
// so a sampler that reads y draws from the distribution that the selection
// with the same policy draws from.
//
// Only a few tokens of a row are edited: the row's penalty entries, its extra
// tokens and its biases, lists sorted by token. A block takes one chunk of a
// row. Each list's entries of the chunk go to LDS in their order, a thread an
// entry: a penalty entry as its finished value (it reads its own logit), a bias
// as it is, with a bitmap of the list's tokens and, for each of its words, the
// place of the word's first entry. Then the chunk's vectors go from registers
// to the output; the lane that holds an edited token finds its entry by the
// word's first place and the bits before it. That keeps a block at 13 KB of
// LDS, eight blocks on a CU: what bounds the kernel is the chain of dependent
// loads (row record, list bounds and mask, entries and vectors, entries'
// logits), and the chunks in flight hide it. (A tile of 8192 values in LDS held
// four blocks: 256 masked rows x 248,320 bf16 took 73 us.)
//
// A vector is loaded only if one of its tokens is admitted, and in place
// written only if one of them changes: a grammar's row, which drops nearly all
// of its tokens, is written without being read, and an unmasked row in place
// touches nothing but the vectors of its edits.
#include <hip/hip_runtime.h>

#include "jf_kernels.h"
#include "jf_logits.h"

namespace jf {

namespace {

constexpr uint32_t kMapWords = kScoreChunk / 32;
constexpr uint32_t kStaged = 1024;  // a list's entries in LDS; later ones stay in memory

// A list's entries of the chunk.
struct ListLds {
  uint32_t bits[kMapWords];
  uint16_t first[kMapWords];  // of a word with any bit
  float value[kStaged];
};
struct ProcessLds {
  ListLds penalty, bias;
  uint32_t admitted[kMapWords];
  uint32_t extra_bits[kMapWords];  // extra tokens that the table does not hold
  uint32_t extras[kMaxExtra];
  float extra_value[kMaxExtra];
};

// VEC bits of a bitmap from token `at` of the chunk (a multiple of VEC).
template <uint32_t VEC>
__device__ __forceinline__ uint32_t bits_at(const uint32_t *map, uint32_t at) {
  return (map[at >> 5] >> (at & 31u)) & ((1u << VEC) - 1u);
}
__device__ __forceinline__ bool bit_at(const uint32_t *map, uint32_t at) {
  return map[at >> 5] >> (at & 31u) & 1u;
}
// The place in its list's chunk of the entry of token `at`, which it holds.
__device__ __forceinline__ uint32_t place_at(const ListLds &l, uint32_t at) {
  return l.first[at >> 5] + __popc(l.bits[at >> 5] & ((1u << (at & 31u)) - 1u));
}
// Entry i of a list's chunk: its bit, and its place if it begins a word.
__device__ __forceinline__ void mark(ListLds &l, const PenaltyEntry *list, uint32_t i,
                                     uint32_t token, uint32_t base) {
  const uint32_t at = token - base;
  atomicOr(&l.bits[at >> 5], 1u << (at & 31u));
  if (i == 0 || (list[i - 1].token - base) >> 5 != at >> 5) l.first[at >> 5] = (uint16_t)i;
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

  uint32_t pen0 = 0, pens = 0, bias0 = 0, biases = 0;
  const uint32_t b0 = chunk * (kScoreChunk / kPenaltyBucket);
  const uint32_t b1 = min(b0 + kScoreChunk / kPenaltyBucket, a.buckets);
  if (p.penalty_row != kNoRow) {
    const uint32_t *off = a.pen_offsets + (uint64_t)p.penalty_row * (a.buckets + 1);
    pen0 = off[b0];
    pens = off[b1] - pen0;
  }
  if (p.bias_row != kNoRow) {
    const uint32_t *off = a.bias_offsets + (uint64_t)p.bias_row * (a.buckets + 1);
    bias0 = off[b0];
    biases = off[b1] - bias0;
  }
  s.penalty.bits[tid] = s.bias.bits[tid] = s.extra_bits[tid] = 0;
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
  const bool edits = pens || biases || p.extra_count;
  if (edits || masked) __syncthreads();
  if (!whole && !a.in_place) {
#pragma unroll
    for (uint32_t j = 0; j < LOADS; ++j) {
      const uint32_t at = j * SLAB + tid * VEC;
      w[j] = LogitWords{};
      if (base + at < V && bits_at<VEC>(s.admitted, at)) w[j] = load_words<DI>(x, base + at, V, 0);
    }
  }
  const PenaltyEntry *pen_list =
      a.pen_entries + (uint64_t)p.penalty_row * a.pen_max_entries + pen0;
  const PenaltyEntry *bias_list =
      a.bias_entries + (uint64_t)p.bias_row * a.bias_max_entries + bias0;
  const auto penalized = [&](const PenaltyEntry &e, float logit) {
    uint32_t count = e.word & kCountMask;
    for (uint32_t k = 0; k < p.extra_count; ++k) count += s.extras[k] == e.token;
    return penalize(logit, count, p.repetition, p.repetition_inverse, p.presence, p.frequency);
  };
  for (uint32_t i = tid; i < biases; i += 256) {
    const PenaltyEntry e = bias_list[i];
    mark(s.bias, bias_list, i, e.token, base);
    if (i < kStaged) s.bias.value[i] = u2f(e.word);
  }
  for (uint32_t i = tid; i < pens; i += 256) {
    const PenaltyEntry e = pen_list[i];
    mark(s.penalty, pen_list, i, e.token, base);
    // A dropped token's value is never taken, nor its logit read.
    if (i < kStaged && !(masked && !bit_at(s.admitted, e.token - base)))
      s.penalty.value[i] = penalized(e, logit_value(x[e.token]));
  }
  if (p.extra_count) {
    __syncthreads();
    if (tid < p.extra_count) {
      const PenaltyEntry e{s.extras[tid], 0};
      const uint32_t at = e.token - base;
      if (e.token < V && at < kScoreChunk && !bit_at(s.penalty.bits, at)) {
        // A token that comes more than once leaves the same value each time.
        s.extra_value[tid] = penalized(e, logit_value(x[e.token]));
        atomicOr(&s.extra_bits[at >> 5], 1u << (at & 31u));
      }
    }
  }
  if (edits) __syncthreads();

  // The tokens of a vector that some list edits.
  const auto edited_at = [&](uint32_t at) {
    return edits ? bits_at<VEC>(s.penalty.bits, at) | bits_at<VEC>(s.bias.bits, at) |
                       bits_at<VEC>(s.extra_bits, at)
                 : 0u;
  };
  if (a.in_place) {
#pragma unroll
    for (uint32_t j = 0; j < LOADS; ++j) {
      const uint32_t at = j * SLAB + tid * VEC;
      w[j] = LogitWords{};
      if (base + at >= V) continue;
      const uint32_t admitted = masked ? bits_at<VEC>(s.admitted, at) : ALL;
      if (admitted && (admitted != ALL || edited_at(at)))
        w[j] = load_words<DI>(x, base + at, V, 0);
    }
    // A neighbour's edit reads no logit that this block writes: every read of
    // a list's logit came before the barrier above.
  }
#pragma unroll
  for (uint32_t j = 0; j < LOADS; ++j) {
    const uint32_t at = j * SLAB + tid * VEC, token = base + at;
    if (token >= V) continue;
    const uint32_t admitted = masked ? bits_at<VEC>(s.admitted, at) : ALL;
    const uint32_t edited = edited_at(at) & admitted;
    if (a.in_place && !edited && admitted == ALL) continue;
    if (DI == DO && !edited && admitted == ALL) {
      store_words<DO>(y, token, V, w[j]);
      continue;
    }
    float v[VEC];
    unpack<DI>(w[j], v);
    if (edited) {
#pragma unroll
      for (uint32_t e = 0; e < VEC; ++e) {
        if (!(edited >> e & 1u)) continue;
        if (bit_at(s.penalty.bits, at + e)) {
          const uint32_t i = place_at(s.penalty, at + e);
          v[e] = i < kStaged ? s.penalty.value[i] : penalized(pen_list[i], v[e]);
        } else if (bit_at(s.extra_bits, at + e)) {
          uint32_t k = 0;
          while (s.extras[k] != token + e) ++k;
          v[e] = s.extra_value[k];
        }
        if (bit_at(s.bias.bits, at + e)) {
          const uint32_t i = place_at(s.bias, at + e);
          const float bias = i < kStaged ? s.bias.value[i] : u2f(bias_list[i].word);
          // A ban holds whatever the logit.
          v[e] = bias == -__builtin_inff() ? bias : v[e] + bias;
        }
      }
    }
#pragma unroll
    for (uint32_t e = 0; e < VEC; ++e)
      if (!(admitted >> e & 1u)) v[e] = -__builtin_inff();
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
