// Device access to rows of logits, f32 (DT 0) or bf16 (DT 1), for the
// operators that read or write whole rows: 16-byte vectors at any element's
// alignment, in chunks of N slabs of 256 vectors: element e of thread tid's j-th
// vector is token j * SLAB + tid * VEC + e of the chunk.
#pragma once

#include "jf_device.h"
#include "jf_scorer.h"

namespace jf {

typedef uint32_t LogitWords __attribute__((ext_vector_type(4)));
typedef LogitWords LogitWordsAt4 __attribute__((aligned(4)));
typedef LogitWords LogitWordsAt2 __attribute__((aligned(2)));

template <int DT>
struct Logits;
template <>
struct Logits<0> {
  using Element = float;
  using Words = LogitWordsAt4;
  static constexpr uint32_t VEC = 4;
};
template <>
struct Logits<1> {
  using Element = uint16_t;
  using Words = LogitWordsAt2;
  static constexpr uint32_t VEC = 8;
};
template <int DT>
constexpr uint32_t kSlab = 256 * Logits<DT>::VEC;

template <int DT>
__device__ __forceinline__ const typename Logits<DT>::Element *row_of(const void *logits,
                                                                      uint64_t at) {
  return (const typename Logits<DT>::Element *)logits + at;
}
template <int DT>
__device__ __forceinline__ typename Logits<DT>::Element *row_of(void *logits, uint64_t at) {
  return (typename Logits<DT>::Element *)logits + at;
}

__device__ __forceinline__ float logit_value(float x) { return x; }
__device__ __forceinline__ float logit_value(uint16_t x) { return bf16_to_float(x); }

// Two values rounded to bf16 (to nearest, ties to even; a NaN stays one), the
// first in the low half: one conversion instruction.
__device__ __forceinline__ uint32_t floats_to_bf16(float lo, float hi) {
  typedef float Floats __attribute__((ext_vector_type(2)));
  typedef __bf16 Halves __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((Floats{lo, hi}), Halves));
}
template <int DT>
__device__ __forceinline__ typename Logits<DT>::Element logit_of(float x) {
  if constexpr (DT == 0)
    return x;
  else
    return (uint16_t)floats_to_bf16(x, x);
}

// The VEC values of one vector.
template <int DT>
__device__ __forceinline__ void unpack(const LogitWords &w, float (&v)[Logits<DT>::VEC]) {
  if constexpr (DT == 0) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = u2f(w[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = u2f(w[e] << 16);
      v[2 * e + 1] = u2f(w[e] & 0xffff0000u);
    }
  }
}
template <int DT>
__device__ __forceinline__ LogitWords pack(const float (&v)[Logits<DT>::VEC]) {
  LogitWords w;
  if constexpr (DT == 0) {
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = f2u(v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = floats_to_bf16(v[2 * e], v[2 * e + 1]);
  }
  return w;
}

// The vector at `token` of a row of `vocabulary` tokens, of which the first
// `before` are none; those and the ones past its end hold the bits `past`.
template <int DT>
__device__ __forceinline__ LogitWords load_words(const typename Logits<DT>::Element *row,
                                                 uint32_t token, uint32_t vocabulary,
                                                 uint32_t past, uint32_t before = 0) {
  if (token >= before && token + Logits<DT>::VEC <= vocabulary)
    return *(const typename Logits<DT>::Words *)(row + token);
  const auto at = [&](uint32_t t) -> uint32_t {
    if (t < before || t >= vocabulary) return past;
    if constexpr (DT == 0)
      return f2u(row[t]);
    else
      return row[t];
  };
  LogitWords w;
#pragma unroll
  for (uint32_t e = 0; e < 4; ++e) {
    if constexpr (DT == 0)
      w[e] = at(token + e);
    else
      w[e] = at(token + 2 * e) | at(token + 2 * e + 1) << 16;
  }
  return w;
}
// A thread's vectors of the chunk of N slabs at `base`, likewise. One branch for the
// chunk: with one a vector the compiler keeps every vector's ways apart in
// registers.
template <int DT, uint32_t N>
__device__ __forceinline__ void load_chunk(const typename Logits<DT>::Element *row, uint32_t base,
                                           uint32_t vocabulary, uint32_t past,
                                           LogitWords (&w)[N], uint32_t before = 0) {
  const uint32_t token = base + threadIdx.x * Logits<DT>::VEC;
  if (base >= before && base + N * kSlab<DT> <= vocabulary) {
#pragma unroll
    for (uint32_t j = 0; j < N; ++j)
      w[j] = *(const typename Logits<DT>::Words *)(row + token + j * kSlab<DT>);
  } else {
#pragma unroll
    for (uint32_t j = 0; j < N; ++j)
      w[j] = load_words<DT>(row, token + j * kSlab<DT>, vocabulary, past, before);
  }
}
// The bits of -infinity for `past`.
template <int DT>
constexpr uint32_t kPastMinusInfinity = DT == 0 ? 0xff800000u : 0xff80u;

// The values of a vector into tokens [token, token + VEC) of a row, those
// past its end and its first `before` left out.
template <int DT>
__device__ __forceinline__ void store_words(typename Logits<DT>::Element *row, uint32_t token,
                                            uint32_t vocabulary, const LogitWords &w,
                                            uint32_t before = 0) {
  if (token >= before && token + Logits<DT>::VEC <= vocabulary) {
    *(typename Logits<DT>::Words *)(row + token) = w;
    return;
  }
#pragma unroll
  for (uint32_t e = 0; e < Logits<DT>::VEC; ++e)
    if (token + e >= before && token + e < vocabulary) {
      if constexpr (DT == 0)
        row[token + e] = u2f(w[e]);
      else
        row[token + e] = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
    }
}

// ---- softmax statistics ---------------------------------------------------------

constexpr float kLog2e = 1.44269504088896341f;

__device__ __forceinline__ float wave_sum_f32(float v) {
  v += xor_f32<1>(v);
  v += xor_f32<2>(v);
  v += xor_f32<4>(v);
  v += xor_f32<8>(v);
  v += xor_f32<16>(v);
  v += xor_f32<32>(v);
  return v;
}

// Maxima of values as they are loaded: fmax quiets each of its operands first,
// an instruction a value. A quiet NaN is passed over; a signalling one may
// take others' places, but then the sum of their exponentials is NaN as well.
__device__ __forceinline__ float loaded_max(float a, float b) {
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
__device__ __forceinline__ float loaded_max(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
template <int DT>
__device__ __forceinline__ float vector_max(const LogitWords &w) {
  float v[Logits<DT>::VEC];
  unpack<DT>(w, v);
  float m = loaded_max(v[0], v[1], v[2]);
  if constexpr (DT == 0) return loaded_max(m, v[3]);
  m = loaded_max(m, v[3], v[4]);
  return loaded_max(loaded_max(m, v[5], v[6]), v[7]);
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
__device__ __forceinline__ MaxSum wave_join(MaxSum p, float c) {
  const float m = wave_max_f32(p.m);
  return {m, wave_sum_f32(p.s * exp_below(p.m, finite_reference(m), c))};
}
// Adds a thread's N vectors, whose maxima are `part`.
template <int DT, uint32_t N>
__device__ __forceinline__ void add_vectors(MaxSum &run, const LogitWords (&w)[N],
                                            const float (&part)[N], float c) {
  float grown = run.m;
#pragma unroll
  for (uint32_t j = 0; j < N; ++j) grown = loaded_max(grown, part[j]);
  const float r = finite_reference(grown);
  float s = run.s * exp_below(run.m, r, c);
#pragma unroll
  for (uint32_t j = 0; j < N; ++j) {
    float v[Logits<DT>::VEC];
    unpack<DT>(w[j], v);
#pragma unroll
    for (uint32_t e = 0; e < Logits<DT>::VEC; ++e) s += exp_below(v[e], r, c);
  }
  run = {grown, s};
}

// A lane's first block of a row.
__device__ __forceinline__ MaxSum row_part(const ScoreLaunch &a, uint32_t row) {
  const uint32_t lane = threadIdx.x & 63u;
  if (lane >= a.segments) return MaxSum{-__builtin_inff(), 0.0f};
  const float2 v = a.partials[(uint64_t)row * a.segments + lane];
  return MaxSum{v.x, v.y};
}
// The row's maximum and sum from its blocks' (every lane of the wave); `p` is
// the lane's row_part, which may have been asked for before.
__device__ __forceinline__ MaxSum row_total(const ScoreLaunch &a, uint32_t row, MaxSum p,
                                            float c) {
  for (uint32_t g = (threadIdx.x & 63u) + 64; g < a.segments; g += 64) {
    const float2 v = a.partials[(uint64_t)row * a.segments + g];
    p = join(p, MaxSum{v.x, v.y}, c);
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

}  // namespace jf
