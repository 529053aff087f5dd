// The global norm of many tensors' gradients, and their clipping, on gfx950:
// n = sqrt(sum g^2) (or max |g|) over all of them, then g min(1, limit / (n + 1e-6)).
//
// Two passes over the same chunks of the same table of tensors. The first leaves a
// part of the norm a block; the second adds the parts up in every block (in the same
// order) and takes the chunks from the last to the first, since the last may still be
// in the caches. Squares are added in 64 bits: their range is twice that of an f32
// gradient, and the order of blocks costs no bits that a norm in fp32 has.
//
// Memory bounds both: 500M bf16 elements in 290 tensors, norm 174 us (6 TB/s without
// the launches beside it), norm and clipping 526. Blocks take chunks by turns, so that
// all of them read at one place of memory (a run of chunks a block: 602 us), which makes
// every chunk one of another tensor: the table is in LDS, where looking a chunk up
// costs little, and the next chunk's loads are out while one is worked on.
//
// The table is up to 124 entries in the kernel arguments, or more of them put
// together in device memory by launches that carry 160 tensors each, 2.3 us a launch:
// nothing is copied from host memory, so a captured call replays with its own tensors.
#include <hip/hip_runtime.h>

#include "jf_gradients.h"
#include "jf_logits.h"

namespace jf {

namespace {

constexpr uint32_t kThreads = 256, kWaves = kThreads / 64;
// Entries in LDS; a longer table is looked up in device memory.
constexpr uint32_t kTableLds = 1024;

// Parts are joined by sums, or as the largest bits of a magnitude: NaN is above
// infinity there, and so is kept.
template <bool MAX>
struct Part;
template <>
struct Part<false> {
  double v = 0.0;
  __device__ __forceinline__ void add(float x) {
    const double d = (double)x;
    v = __builtin_fma(d, d, v);
  }
  __device__ __forceinline__ void join(double p) { v += p; }
  __device__ __forceinline__ double wave() const { return wave_sum_f64(v); }
  __device__ __forceinline__ static double norm(double v) { return sqrt(v); }
};
template <>
struct Part<true> {
  uint32_t v = 0;
  __device__ __forceinline__ void add(float x) { v = max(v, f2u(x) & 0x7fffffffu); }
  __device__ __forceinline__ void join(double p) { v = max(v, (uint32_t)p); }
  __device__ __forceinline__ double wave() const { return (double)wave_max_u32(v); }
  __device__ __forceinline__ static double norm(double v) { return (double)u2f((uint32_t)v); }
};

// A block's part from its threads' (every thread).
template <bool MAX>
__device__ __forceinline__ double block_part(const Part<MAX> &p, double *waves) {
  const double w = p.wave();
  if ((threadIdx.x & 63u) == 0) waves[threadIdx.x >> 6] = w;
  __syncthreads();
  Part<MAX> all;
#pragma unroll
  for (uint32_t i = 0; i < kWaves; ++i) all.join(waves[i]);
  return (double)all.v;
}

// ---- the table ---------------------------------------------------------------------

template <bool LDS>
struct Table;
template <>
struct Table<true> {
  struct Memory {
    GradientEntry entries[kTableLds];
    uint32_t first[kTableLds];
  };
  const Memory &m;
  uint32_t tensors;
  __device__ __forceinline__ uint32_t first(uint32_t i) const { return m.first[i]; }
  __device__ __forceinline__ const GradientEntry &entry(uint32_t i) const { return m.entries[i]; }
  // Every thread of the block, before the first use.
  __device__ __forceinline__ static Table load(const GradientLaunch &a, const GradientEntry *from,
                                               Memory &m) {
    for (uint32_t i = threadIdx.x; i < a.tensors; i += kThreads) {
      const GradientEntry e = from[i];
      m.entries[i] = e;
      m.first[i] = e.first;
    }
    __syncthreads();
    return {m, a.tensors};
  }
};
template <>
struct Table<false> {
  struct Memory {};
  const GradientEntry *from;
  uint32_t tensors;
  __device__ __forceinline__ uint32_t first(uint32_t i) const { return from[i].first; }
  __device__ __forceinline__ const GradientEntry &entry(uint32_t i) const { return from[i]; }
  __device__ __forceinline__ static Table load(const GradientLaunch &a, const GradientEntry *from,
                                               Memory &) {
    return {from, a.tensors};
  }
};

// The entries among the kernel arguments, behind the launch record: their address,
// since one by an index would be copied to private memory first.
struct KernelArgs {
  GradientLaunch a;
  GradientArgs entries;
};
static_assert(sizeof(KernelArgs) <= 4096);
__device__ __forceinline__ const GradientEntry *table_of(const GradientLaunch &a) {
  uint64_t u = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(u));
  return a.table ? a.table : (const GradientEntry *)(u + __builtin_offsetof(KernelArgs, entries));
}

// The elements of a tensor's first line that are none of its, and its chunks.
__device__ __forceinline__ uint32_t elements_before(const GradientTensor &t) {
  return (uint32_t)((uintptr_t)t.out % 128) >>
         (t.count_types >> kGradientTypeShift & kGradientOutBf16 ? 1 : 2);
}
__device__ __forceinline__ uint64_t end_of(const GradientTensor &t) {
  return elements_before(t) + (t.count_types & ((1ull << kGradientTypeShift) - 1));
}

// One wave: three tensors a lane at most.
__global__ __launch_bounds__(64) void gradient_table_kernel(GradientTableArgs a) {
  constexpr uint32_t EACH = (kGradientTableArgs + 63) / 64;
  uint64_t u = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(u));
  const auto *tensors = ((const GradientTableArgs *)u)->tensors;
  GradientTensor t[EACH];
  uint32_t at[EACH], chunks[EACH];
#pragma unroll
  for (uint32_t k = 0; k < EACH; ++k) {
    at[k] = k * 64 + threadIdx.x;
    t[k] = tensors[at[k] < a.count ? at[k] : 0];
  }
  uint32_t first = a.first;
#pragma unroll
  for (uint32_t k = 0; k < EACH; ++k) {
    chunks[k] =
        at[k] < a.count ? (uint32_t)((end_of(t[k]) + kGradientChunk - 1) / kGradientChunk) : 0;
    const uint32_t sum = wave_incl_scan_u32(chunks[k]);
    if (at[k] < a.count) a.table[at[k]] = GradientEntry{t[k], first + sum - chunks[k], 0};
    first += readlane_u32(sum, 63);
  }
}

// ---- chunks --------------------------------------------------------------------------

__device__ __forceinline__ uint64_t uniform(uint64_t v) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v) |
         (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32)) << 32;
}

// A chunk of a tensor: where its elements are, first .. last - 1 of kGradientChunk,
// and the tensor's types. Every wave alike.
struct Place {
  uintptr_t grad, out;
  uint32_t first, last, types;
  __device__ __forceinline__ bool whole() const { return first == 0 && last == kGradientChunk; }
};

template <bool LDS>
__device__ __forceinline__ Place place_of(const Table<LDS> &table, uint32_t chunk) {
  // The entry that holds it: 64 of them are looked at at a time, evenly apart.
  const uint32_t lane = threadIdx.x & 63u;
  uint32_t lo = 0, n = table.tensors;
  while (n > 1) {
    const uint32_t step = (n + 63) / 64, at = lane * step;
    const uint32_t reach =
        (uint32_t)__popcll(ballot(at < n && table.first(lo + (at < n ? at : 0)) <= chunk));
    const uint32_t skip = (reach - 1) * step;
    lo += skip;
    n = min(step, n - skip);
  }
  const GradientEntry &e = table.entry(lo);
  const uint64_t count_types = uniform(e.tensor.count_types);
  const uint32_t in_tensor = chunk - (uint32_t)__builtin_amdgcn_readfirstlane((int)e.first);
  Place p;
  p.types = (uint32_t)(count_types >> kGradientTypeShift);
  const uint32_t in_shift = p.types & kGradientBf16 ? 1 : 2;
  const uint32_t out_shift = p.types & kGradientOutBf16 ? 1 : 2;
  const uint64_t out = uniform((uint64_t)e.tensor.out);
  // Elements count from the tensor's last line before it.
  const uint32_t before = (uint32_t)(out % 128) >> out_shift;
  const uint64_t at = (uint64_t)in_tensor * kGradientChunk;
  const uint64_t end = before + (count_types & ((1ull << kGradientTypeShift) - 1)) - at;
  p.first = in_tensor ? 0 : before;
  p.last = end < kGradientChunk ? (uint32_t)end : kGradientChunk;
  p.grad = uniform((uint64_t)e.tensor.grad) + ((at - before) << in_shift);
  p.out = out + ((at - before) << out_shift);
  return p;
}

// An address that is none of LDS: the loads from one that may be wait for what LDS
// does, and what LDS does for them.
template <class T>
__device__ __forceinline__ T *in_memory(uintptr_t p) {
  return (T *)(__attribute__((address_space(1))) T *)p;
}

// A thread's vectors of a chunk as they are in memory: eight of 16 bytes (f32), four
// (bf16), or eight of 8 (bf16 on its way to f32, whose vectors are of four elements).
struct Vectors {
  LogitWords w[8];
};
static_assert(kGradientChunk == 8 * kThreads * 4);

template <int DT, uint32_t VEC>
__device__ __forceinline__ LogitWords load_vector(const typename Logits<DT>::Element *p) {
  if constexpr (DT == 1 && VEC == 4) {
    struct Pair {
      uint32_t w[2];
    } __attribute__((packed, aligned(2)));
    const Pair v = *(const Pair *)p;
    return LogitWords{v.w[0], v.w[1], 0, 0};
  } else {
    return *(const typename Logits<DT>::Words *)p;
  }
}
// Of a whole chunk.
template <int DT, uint32_t VEC>
__device__ __forceinline__ Vectors load_whole(const Place &p) {
  constexpr uint32_t SLAB = kThreads * VEC, N = kGradientChunk / SLAB;
  const auto *row = in_memory<const typename Logits<DT>::Element>(p.grad);
  Vectors v;
#pragma unroll
  for (uint32_t j = 0; j < N; ++j)
    v.w[j] = load_vector<DT, VEC>(row + j * SLAB + threadIdx.x * VEC);
  return v;
}
// Of one that is not; 0 beside its tensor's elements.
template <int DT, uint32_t VEC>
__device__ __forceinline__ Vectors load_part(const Place &p) {
  constexpr uint32_t SLAB = kThreads * VEC, N = kGradientChunk / SLAB;
  const auto *row = in_memory<const typename Logits<DT>::Element>(p.grad);
  Vectors v;
#pragma unroll
  for (uint32_t j = 0; j < N; ++j) {
    const uint32_t at = j * SLAB + threadIdx.x * VEC;
    if constexpr (DT == 1 && VEC == 4) {
      const auto one = [&](uint32_t i) -> uint32_t {
        return i >= p.first && i < p.last ? row[i] : 0;
      };
      v.w[j] = LogitWords{one(at) | one(at + 1) << 16, one(at + 2) | one(at + 3) << 16, 0, 0};
    } else {
      v.w[j] = load_words<DT>(row, at, p.last, 0, p.first);
    }
  }
  return v;
}
template <int DT>
__device__ __forceinline__ float value(const LogitWords &w, uint32_t e) {
  if constexpr (DT == 0) return u2f(w[e]);
  return u2f(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
}

template <int DT, bool MAX>
__device__ __forceinline__ void add_vectors(Part<MAX> &part, const Vectors &v) {
  constexpr uint32_t VEC = Logits<DT>::VEC, N = kGradientChunk / (kThreads * VEC);
#pragma unroll
  for (uint32_t j = 0; j < N; ++j)
#pragma unroll
    for (uint32_t e = 0; e < VEC; ++e) part.add(value<DT>(v.w[j], e));
}

template <int IN, int OUT, uint32_t VEC>
__device__ __forceinline__ void store_vectors(const Vectors &v, const Place &p, float scale) {
  constexpr uint32_t SLAB = kThreads * VEC, N = kGradientChunk / SLAB;
  auto *row = in_memory<typename Logits<OUT>::Element>(p.out);
  const bool whole = p.whole();
#pragma unroll
  for (uint32_t j = 0; j < N; ++j) {
    const uint32_t at = j * SLAB + threadIdx.x * VEC;
    float s[VEC];
#pragma unroll
    for (uint32_t e = 0; e < VEC; ++e) s[e] = value<IN>(v.w[j], e) * scale;
    if (whole || (at >= p.first && at + VEC <= p.last)) {
      if constexpr (OUT == 1 && VEC == 4) {
        typedef uint32_t Pair __attribute__((ext_vector_type(2)));
        __builtin_nontemporal_store(Pair{floats_to_bf16(s[0], s[1]), floats_to_bf16(s[2], s[3])},
                                    (Pair *)(row + at));
      } else {
        __builtin_nontemporal_store(pack<OUT>(s), (LogitWords *)(row + at));
      }
    } else {
#pragma unroll
      for (uint32_t e = 0; e < VEC; ++e)
        if (at + e >= p.first && at + e < p.last) row[at + e] = logit_of<OUT>(s[e]);
    }
  }
}

// A call's tensors are mostly of the same types: kernels of their own, in which the
// next chunk's loads have one place in the code and so are not waited for where
// several places' meet (a type, or a chunk that is not whole). kMixed: any types, and
// no chunk is asked for ahead.
constexpr int kMixed = 2;
template <int IN>
__device__ __forceinline__ bool is_bf16(const Place &p) {
  return IN == kMixed ? (p.types & kGradientBf16) != 0 : IN == 1;
}
// The vectors of a chunk at its use: `v` where it was asked for ahead.
template <int IN, int DT, uint32_t VEC>
__device__ __forceinline__ Vectors own(const Vectors &v, const Place &p) {
  if (!p.whole()) return load_part<DT, VEC>(p);
  if constexpr (IN == kMixed)
    return load_whole<DT, VEC>(p);
  else
    return v;
}
template <int OUT>
__device__ __forceinline__ bool is_out_bf16(const Place &p) {
  return OUT == kMixed ? (p.types & kGradientOutBf16) != 0 : OUT == 1;
}

// The block's chunks: take(place) asks for a whole one's vectors, use(place, vectors)
// works on a chunk while the next one is on its way; what is not whole it loads for
// itself. `go` is asked once, with the first under way.
template <bool LDS, class Take, class Go, class Use>
__device__ __forceinline__ void each_chunk(const Table<LDS> &table, uint32_t chunks, bool backwards,
                                           const Take &take, const Go &go, const Use &use) {
  uint32_t n = blockIdx.x;
  const auto place = [&](uint32_t i) { return place_of(table, backwards ? chunks - 1 - i : i); };
  Place here = place(n);
  Vectors now{}, next{};
  if (here.whole()) now = take(here);
  if (!go()) return;
  while (true) {
    n += gridDim.x;
    const bool more = n < chunks;
    Place there{};
    if (more) {
      there = place(n);
      if (there.whole()) next = take(there);
    }
    use(here, now);
    if (!more) return;
    here = there;
    now = next;
  }
}

template <int DT, bool MAX, bool LDS>
__global__ __launch_bounds__(kThreads, 3) void gradient_parts_kernel(GradientLaunch a,
                                                                     GradientArgs entries) {
  __shared__ typename Table<LDS>::Memory memory;
  __shared__ double waves[kWaves];
  const auto table = Table<LDS>::load(a, table_of(a), memory);
  Part<MAX> part;
  each_chunk(
      table, a.chunks, false,
      [](const Place &p) {
        if constexpr (DT == kMixed)
          return Vectors{};
        else
          return load_whole<DT, Logits<DT>::VEC>(p);
      },
      [] { return true; },
      [&](const Place &p, const Vectors &v) {
        if (is_bf16<DT>(p))
          add_vectors<1>(part, own<DT, 1, 8>(v, p));
        else
          add_vectors<0>(part, own<DT, 0, 4>(v, p));
      });
  const double all = block_part(part, waves);
  if (threadIdx.x == 0) a.parts[blockIdx.x] = all;
}

// The norm of the parts, in every thread; the parts may be asked for before.
constexpr uint32_t kPartsEach = kGradientParts / kThreads;
static_assert(kGradientParts % kThreads == 0);
struct Parts {
  double v[kPartsEach];  // 0 adds nothing in either order
};
__device__ __forceinline__ Parts load_parts(const GradientLaunch &a) {
  Parts p;
#pragma unroll
  for (uint32_t k = 0; k < kPartsEach; ++k) {
    const uint32_t i = k * kThreads + threadIdx.x;
    p.v[k] = i < a.part_count ? a.parts[i] : 0.0;
  }
  return p;
}
template <bool MAX>
__device__ __forceinline__ double joined_norm(const Parts &p, double *waves) {
  Part<MAX> part;
#pragma unroll
  for (uint32_t k = 0; k < kPartsEach; ++k) part.join(p.v[k]);
  return Part<MAX>::norm(block_part(part, waves));
}
__device__ __forceinline__ double joined_norm(const GradientLaunch &a, const Parts &p,
                                              double *waves) {
  return a.max_order ? joined_norm<true>(p, waves) : joined_norm<false>(p, waves);
}

__global__ __launch_bounds__(kThreads) void gradient_norm_kernel(GradientLaunch a) {
  __shared__ double waves[kWaves];
  const double norm = joined_norm(a, load_parts(a), waves);
  if (threadIdx.x == 0) a.norm[0] = (float)norm;
}

template <int IN, int OUT, bool LDS>
__global__ __launch_bounds__(kThreads, 3) void gradient_scale_kernel(GradientLaunch a,
                                                                     GradientArgs entries) {
  __shared__ typename Table<LDS>::Memory memory;
  __shared__ double waves[kWaves];
  // The parts, the table and the first chunk are on their way together.
  Parts parts{};
  double norm = 0.0;
  if (a.norm_given)
    norm = (double)a.norm[0];
  else
    parts = load_parts(a);
  const auto table = Table<LDS>::load(a, table_of(a), memory);
  float scale = 0.0f;
  // Gradients in place stay where the scale is 1.
  const auto stays = [&](const Place &p) {
    return scale == 1.0f && !(p.types & kGradientOutElsewhere);
  };
  each_chunk(
      table, a.chunks, true,
      [&](const Place &p) {
        if constexpr (IN == kMixed)
          return Vectors{};
        else
          return load_whole<IN, IN == 1 && OUT == 1 ? 8 : 4>(p);
      },
      [&] {
        if (!a.norm_given) {
          norm = joined_norm(a, parts, waves);
          if (blockIdx.x == 0 && threadIdx.x == 0) a.norm[0] = (float)norm;
        }
        const double limit = (double)a.max_norm / (norm + 1e-6);
        scale = limit >= 1.0 ? 1.0f : (float)limit;
        return scale != 1.0f || a.any_elsewhere;
      },
      [&](const Place &p, const Vectors &v) {
        if (stays(p)) return;
        if (!is_bf16<IN>(p)) {
          if (is_out_bf16<OUT>(p))
            store_vectors<0, 1, 4>(own<IN, 0, 4>(v, p), p, scale);
          else
            store_vectors<0, 0, 4>(own<IN, 0, 4>(v, p), p, scale);
        } else if (is_out_bf16<OUT>(p)) {
          store_vectors<1, 1, 8>(own<IN, 1, 8>(v, p), p, scale);
        } else {
          store_vectors<1, 0, 4>(own<IN, 1, 4>(v, p), p, scale);
        }
      });
}

}  // namespace

int launch_gradient_table(const GradientTableArgs &a, void *stream) {
  hipLaunchKernelGGL(gradient_table_kernel, dim3(1), dim3(64), 0, (hipStream_t)stream, a);
  return (int)hipGetLastError();
}

int launch_gradient_parts(const GradientLaunch &a, const GradientArgs &entries, void *stream) {
  const dim3 grid(a.part_count), block(kThreads);
  const hipStream_t st = (hipStream_t)stream;
  const bool lds = a.tensors <= kTableLds;
  const int in = a.types & kGradientMixed ? kMixed : a.types & kGradientBf16 ? 1 : 0;
#define JF_PARTS(DT, MAX, LDS)                                                             \
  if (in == DT && (a.max_order != 0) == MAX && lds == LDS)                                 \
  hipLaunchKernelGGL((gradient_parts_kernel<DT, MAX, LDS>), grid, block, 0, st, a, entries)
#define JF_PARTS_ALL(DT)       \
  JF_PARTS(DT, false, false);  \
  JF_PARTS(DT, false, true);   \
  JF_PARTS(DT, true, false);   \
  JF_PARTS(DT, true, true)
  JF_PARTS_ALL(0);
  JF_PARTS_ALL(1);
  JF_PARTS_ALL(kMixed);
#undef JF_PARTS_ALL
#undef JF_PARTS
  return (int)hipGetLastError();
}

int launch_gradient_norm(const GradientLaunch &a, void *stream) {
  hipLaunchKernelGGL(gradient_norm_kernel, dim3(1), dim3(kThreads), 0, (hipStream_t)stream, a);
  return (int)hipGetLastError();
}

int launch_gradient_scale(const GradientLaunch &a, const GradientArgs &entries, void *stream) {
  const dim3 grid(a.part_count), block(kThreads);
  const hipStream_t st = (hipStream_t)stream;
  const bool lds = a.tensors <= kTableLds;
  const bool in = a.types & kGradientBf16, out = a.types & kGradientOutBf16;
  // f32 gradients that are narrowed go with the mixed ones.
  const bool mixed = (a.types & kGradientMixed) || (!in && out);
#define JF_SCALE(IN, OUT, COND)                                                             \
  if ((COND) && lds)                                                                        \
    hipLaunchKernelGGL((gradient_scale_kernel<IN, OUT, true>), grid, block, 0, st, a, entries); \
  else if (COND)                                                                            \
  hipLaunchKernelGGL((gradient_scale_kernel<IN, OUT, false>), grid, block, 0, st, a, entries)
  JF_SCALE(0, 0, !mixed && !in);
  JF_SCALE(1, 0, !mixed && in && !out);
  JF_SCALE(1, 1, !mixed && in && out);
  JF_SCALE(kMixed, kMixed, mixed);
#undef JF_SCALE
  return (int)hipGetLastError();
}

}  // namespace jf
