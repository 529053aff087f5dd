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
// LDS, eight blocks on a CU: what bounds a call of few rows is the chain of
// dependent loads (row record, list bounds and mask, entries and vectors,
// entries' logits), and the chunks in flight hide it in larger ones. (A tile of
// 8192 values in LDS held four blocks: 256 masked rows x 248,320 bf16 took 73
// us, 46.7 as here; with nontemporal stores, 28.7.)
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

constexpr uint32_t kStaged = 1024;  // a list's entries in LDS; later ones stay in memory

// A list's entries of the chunk.
template <uint32_t CHUNK>
struct ListLds {
  uint32_t bits[CHUNK / 32];
  uint16_t first[CHUNK / 32];  // of a word with any bit
  float value[kStaged];
};
template <uint32_t CHUNK>
struct ProcessLds {
  ListLds<CHUNK> penalty, bias;
  uint32_t admitted[CHUNK / 32];
  uint32_t extra_bits[CHUNK / 32];  // extra tokens that the table does not hold
  uint32_t extras[kMaxExtra];
  float extra_value[kMaxExtra];
};

// VEC tokens of a row of type DT as a lane loads or stores them: 16 bytes, or 8
// bytes of bf16 where the other side is f32, so that a wave's loads and its
// stores both cover whole lines. BELOW: a token may be below 0, modulo 2^32; there
// is nothing, as past the vocabulary.
template <int DT, uint32_t VEC, bool BELOW>
struct Tokens {
  using Element = typename Logits<DT>::Element;
  static constexpr uint32_t WORDS = VEC * sizeof(Element) / 4;
  typedef uint32_t Words __attribute__((ext_vector_type(WORDS)));
  typedef Words WordsAt __attribute__((aligned(sizeof(Element))));

  static __device__ __forceinline__ bool within(uint32_t token, uint32_t V) {
    return (!BELOW || token < V) && token + VEC <= V;
  }
  static __device__ __forceinline__ Words load(const Element *row, uint32_t token, uint32_t V) {
    if (within(token, V)) return *(const WordsAt *)(row + token);
    Words w{};
#pragma unroll
    for (uint32_t e = 0; e < VEC; ++e)
      if (token + e < V) {
        if constexpr (DT == 0)
          w[e] = f2u(row[token + e]);
        else
          w[e / 2] |= (uint32_t)row[token + e] << (16 * (e & 1));
      }
    return w;
  }
  template <bool NT>
  static __device__ __forceinline__ void store(Element *row, uint32_t token, uint32_t V, Words w) {
    if (within(token, V)) {
      if constexpr (NT)
        __builtin_nontemporal_store(w, (WordsAt *)(row + token));
      else
        *(WordsAt *)(row + token) = w;
      return;
    }
#pragma unroll
    for (uint32_t e = 0; e < VEC; ++e)
      if (token + e < V) {
        if constexpr (DT == 0)
          row[token + e] = u2f(w[e]);
        else
          row[token + e] = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
      }
  }
  static __device__ __forceinline__ void unpack(Words w, float (&v)[VEC]) {
#pragma unroll
    for (uint32_t e = 0; e < VEC; ++e) {
      if constexpr (DT == 0)
        v[e] = u2f(w[e]);
      else
        v[e] = u2f(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    }
  }
  static __device__ __forceinline__ Words pack(const float (&v)[VEC]) {
    Words w;
#pragma unroll
    for (uint32_t i = 0; i < WORDS; ++i) {
      if constexpr (DT == 0)
        w[i] = f2u(v[i]);
      else
        w[i] = floats_to_bf16(v[2 * i], v[2 * i + 1]);
    }
    return w;
  }
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
template <class List>
__device__ __forceinline__ uint32_t place_at(const List &l, uint32_t at) {
  return l.first[at >> 5] + __popc(l.bits[at >> 5] & ((1u << (at & 31u)) - 1u));
}
// Entry i of a list, token `at` of the chunk: its bit, and its place if it begins
// a word.
template <class List>
__device__ __forceinline__ void mark(List &l, const PenaltyEntry *list, uint32_t i, uint32_t at,
                                     uint32_t base) {
  atomicOr(&l.bits[at >> 5], 1u << (at & 31u));
  if (i == 0 || (list[i - 1].token - base) >> 5 != at >> 5) l.first[at >> 5] = (uint16_t)i;
}

// How a call's outputs are stored: kPast: past the caches (nontemporal); kLines:
// also in whole lines, of rows that start within one.
enum Stores { kCached, kPast, kLines };

// A chunk of N vectors a thread.
template <int DI, int DO, uint32_t N, Stores STORES>
__global__ __launch_bounds__(256) void process_kernel(ProcessLaunch a) {
  constexpr uint32_t VEC = DI == 1 && DO == 1 ? 8 : 4, SLAB = 256 * VEC, CHUNK = N * SLAB;
  constexpr uint32_t ALL = (1u << VEC) - 1u;
  static_assert(CHUNK % kPenaltyBucket == 0 && CHUNK / 32 <= 256);
  constexpr bool NT = STORES != kCached, BELOW = STORES == kLines;
  using In = Tokens<DI, VEC, BELOW>;
  using Out = Tokens<DO, VEC, BELOW>;
  __shared__ ProcessLds<CHUNK> s;
  const uint32_t tid = threadIdx.x;
  const uint32_t row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks;
  const uint32_t V = a.vocabulary;
  const auto *x = row_of<DI>(a.logits, (uint64_t)row * a.stride);
  auto *y = row_of<DO>(a.out, (uint64_t)row * a.out_stride);
  // Whole lines: chunks count from the output's last line before the row; the
  // first one's `base` is then below 0, modulo 2^32.
  const uint32_t before = BELOW ? (uint32_t)((uintptr_t)y % 128 / sizeof(*y)) : 0;
  const uint32_t base = chunk * CHUNK - before;
  if (BELOW && chunk && base >= V) return;  // not every row reaches the last chunk
  // Whether any token of a vector is the row's.
  const auto inside = [&](uint32_t token) {
    return token < V || (BELOW && 0u - token < VEC);
  };
  typename In::Words w[N];
  const auto load_all = [&] {
    if ((!BELOW || base < V) && base + CHUNK <= V) {
#pragma unroll
      for (uint32_t j = 0; j < N; ++j)
        w[j] = *(const typename In::WordsAt *)(x + base + j * SLAB + tid * VEC);
    } else {
#pragma unroll
      for (uint32_t j = 0; j < N; ++j) w[j] = In::load(x, base + j * SLAB + tid * VEC, V);
    }
  };
  // An unmasked row that is written elsewhere needs every vector: asked for
  // before anything else, the row's record too where no row is masked.
  const bool early = !a.any_masked && !a.in_place;
  if (early) load_all();
  const ProcessRow p = a.rows[row];
  const bool masked = (p.flags & (kProcessMasked | kProcessStops)) != 0;
  const bool whole = !masked && !a.in_place;
  if (whole && !early) load_all();

  uint32_t pen0 = 0, pens = 0, bias0 = 0, biases = 0;
  const uint32_t b0 = (BELOW && !chunk ? 0 : base) / kPenaltyBucket;
  const uint32_t b1 = min((base + CHUNK + kPenaltyBucket - 1) / kPenaltyBucket, a.buckets);
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
  const bool has_word = tid < CHUNK / 32;
  if (has_word) s.penalty.bits[tid] = s.bias.bits[tid] = s.extra_bits[tid] = 0;
  if (masked && has_word) {
    // Tokens outside the vocabulary are never stored; words outside it not read.
    uint32_t bits = 0xffffffffu;
    if (p.flags & kProcessMasked) {
      const uint32_t *mask = a.masks + (uint64_t)p.mask_row * a.mask_stride;
      const uint32_t words = (V + 31) / 32;
      const int32_t token = (int32_t)(base + tid * 32);
      const uint32_t word = (uint32_t)(token >> 5), shift = token & 31;
      bits = word < words ? mask[word] : 0xffffffffu;
      if (BELOW && shift) {
        const uint32_t next = word + 1 < words ? mask[word + 1] : 0xffffffffu;
        bits = bits >> shift | next << (32 - shift);
      }
    }
    if (p.flags & kProcessStops) {
      const uint32_t at0 = a.stop0 - base, at1 = a.stop1 - base;
      if (at0 >> 5 == tid) bits &= ~(1u << (at0 & 31u));
      if (at1 >> 5 == tid) bits &= ~(1u << (at1 & 31u));
    }
    s.admitted[tid] = bits;
  }
  if (tid < p.extra_count) s.extras[tid] = a.extra[p.extra_offset + tid];
  const bool edits = pens || biases || p.extra_count;
  if (edits || masked) __syncthreads();
  if (!whole && !a.in_place) {
#pragma unroll
    for (uint32_t j = 0; j < N; ++j) {
      const uint32_t at = j * SLAB + tid * VEC;
      w[j] = typename In::Words{};
      if (inside(base + at) && bits_at<VEC>(s.admitted, at)) w[j] = In::load(x, base + at, V);
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
    const uint32_t at = e.token - base;
    if (BELOW && at >= CHUNK) continue;  // of a bucket that the chunk shares
    mark(s.bias, bias_list, i, at, base);
    if (i < kStaged) s.bias.value[i] = u2f(e.word);
  }
  for (uint32_t i = tid; i < pens; i += 256) {
    const PenaltyEntry e = pen_list[i];
    const uint32_t at = e.token - base;
    if (BELOW && at >= CHUNK) continue;
    mark(s.penalty, pen_list, i, at, base);
    // A dropped token's value is never taken, nor its logit read.
    if (i < kStaged && !(masked && !bit_at(s.admitted, at)))
      s.penalty.value[i] = penalized(e, logit_value(x[e.token]));
  }
  if (p.extra_count) {
    __syncthreads();
    if (tid < p.extra_count) {
      const PenaltyEntry e{s.extras[tid], 0};
      const uint32_t at = e.token - base;
      if (e.token < V && at < CHUNK && !bit_at(s.penalty.bits, at)) {
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
    for (uint32_t j = 0; j < N; ++j) {
      const uint32_t at = j * SLAB + tid * VEC;
      w[j] = typename In::Words{};
      if (!inside(base + at)) continue;
      const uint32_t admitted = masked ? bits_at<VEC>(s.admitted, at) : ALL;
      if (admitted && (admitted != ALL || edited_at(at)))
        w[j] = In::load(x, base + at, V);
    }
    // A neighbour's edit reads no logit that this block writes: every read of
    // a list's logit came before the barrier above.
  }
#pragma unroll
  for (uint32_t j = 0; j < N; ++j) {
    const uint32_t at = j * SLAB + tid * VEC, token = base + at;
    if (!inside(token)) continue;
    const uint32_t admitted = masked ? bits_at<VEC>(s.admitted, at) : ALL;
    const uint32_t edited = edited_at(at) & admitted;
    if (a.in_place && !edited && admitted == ALL) continue;
    if constexpr (DI == DO) {
      if (!edited && admitted == ALL) {
        Out::template store<NT>(y, token, V, w[j]);
        continue;
      }
    }
    float v[VEC];
    In::unpack(w[j], v);
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
    Out::template store<NT>(y, token, V, Out::pack(v));
  }
}

// Outputs of more than this go past the caches (nontemporal stores): alone, 256
// masked rows x 248,320 bf16 take 28.7 us so, 46.5 otherwise, and 67.3 or 67.6
// with a pass that reads them behind; 64 rows x 151,936 in f32, 39 MB, 15.0 or
// 16.3, and 26.0 or 26.5. A smaller output is found there by its reader: 16 such
// rows 6.6 or 7.3, but 14.7 or 14.2 with the reader. Such stores of parts of lines
// are dear: rows that start within a line take them whole at the price of masks
// that shift and vectors that begin below the row (256 masked rows x 248,319 bf16
// 34.9 us without, 31.2 so; but 256 bf16 rows x 151,936 to f32, aligned, 40.4
// without, 44.3 so).
constexpr uint64_t kCachedOutput = 24u << 20;

template <int DI, int DO, uint32_t CHUNK>
void launch_chunks(ProcessLaunch a, hipStream_t stream) {
  constexpr uint32_t N = CHUNK / (256 * (DI == 1 && DO == 1 ? 8 : 4));
  constexpr uint32_t SIZE = sizeof(typename Logits<DO>::Element);
  const bool past = (uint64_t)a.row_count * a.vocabulary * SIZE > kCachedOutput;
  const bool lines = past && ((uintptr_t)a.out % 128 != 0 ||
                              (a.row_count > 1 && a.out_stride * SIZE % 128 != 0));
  // A row that starts within a line may reach a chunk more.
  const uint32_t before = lines ? 128 / SIZE - 1 : 0;
  a.chunks = (a.vocabulary + before + CHUNK - 1) / CHUNK;
  const dim3 grid(a.row_count * a.chunks), block(256);
  if (lines)
    hipLaunchKernelGGL((process_kernel<DI, DO, N, kLines>), grid, block, 0, stream, a);
  else if (past)
    hipLaunchKernelGGL((process_kernel<DI, DO, N, kPast>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((process_kernel<DI, DO, N, kCached>), grid, block, 0, stream, a);
}

// Small chunks while there are few, for blocks on every CU (16 rows x 151,936:
// 6.6 us in chunks of 2048 tokens, 7.8 of 4096, 11.0 of 8192; 48 rows 12.4, 11.0
// and 13.3; 128 rows 25.7, 23.4 and 26.0). Masked rows are mostly written without
// being read, and then a chunk's cost is that of its block: 256 such rows x
// 248,320 bf16 48.3, 33.2 and 28.6.
template <int DI, int DO>
void launch_types(const ProcessLaunch &a, hipStream_t stream) {
  const uint64_t tokens = (uint64_t)a.row_count * a.vocabulary;
  if (tokens <= 512u * 8192u)
    launch_chunks<DI, DO, 2048>(a, stream);
  else if (a.all_masked && tokens > 2048u * 8192u)
    launch_chunks<DI, DO, 8192>(a, stream);
  else
    launch_chunks<DI, DO, 4096>(a, stream);
}

}  // namespace

int launch_process(const ProcessLaunch &a, uint32_t dtype, uint32_t out_dtype, void *stream) {
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == 0 && out_dtype == 0)
    launch_types<0, 0>(a, st);
  else if (dtype == 0)
    launch_types<0, 1>(a, st);
  else if (out_dtype == 0)
    launch_types<1, 0>(a, st);
  else
    launch_types<1, 1>(a, st);
  return (int)hipGetLastError();
}

}  // namespace jf
