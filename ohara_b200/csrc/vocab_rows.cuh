// What the row kernels over given logits (vocab_rows.cu) and the kernels that make the logits
// themselves (vocab_gemm_sm100.cu) have in common: packed arithmetic, the running statistics of a
// softmax, a row's distillation loss and the coefficients of a row's gradient.
#pragma once

#include "api.h"
#include "common.cuh"

namespace ob {
namespace vocab {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// A teacher's mass outside its list of up to this much is the rounding of the list's sum (K terms of
// relative error 2^-24 and the teacher's own) and counts as none: the student may have no token there.
constexpr float kLeastRest = 1e-6f;

// Two floats in one register pair: sm_100 adds, multiplies and fuses them with one instruction.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 both(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float quiet_nan() { return __uint_as_float(0x7fffffffu); }

// ---------------------------------------------------------------------------------------------
// Running statistics of the softmax of scaled logits (c = log2(e) / T): `m` the maximum seen (-inf:
// nothing finite yet), `s` the sum of e = 2^((x - m) c), and `w` by kind
//   kSum      nothing
//   kEntropy  the sum of e (x - m)
//   kSplit    the sum of e over the tokens outside the teacher's list; `s` is the sum inside it
// ---------------------------------------------------------------------------------------------
enum Kind { kSum, kEntropy, kSplit };

struct Stats {
  float m, s, w;
};

__device__ __forceinline__ float reference_of(float m) { return m == -INFINITY ? 0.f : m; }

// Moves the sums from maximum `a.m` to `m` (>= a.m).
template <Kind K>
__device__ __forceinline__ void rebase(Stats& a, float m, float c) {
  if (m == a.m) return;
  const float shift = a.m - m;  // < 0; -inf while nothing was seen or where the gap overflows
  const float f = fast_exp2(shift * c);
  if (f == 0.f) {
    // an empty or vanished sum becomes zero (0 * inf below would not), a NaN stays
    a.s = a.s == a.s ? 0.f : a.s;
    if (K != kSum) a.w = a.w == a.w ? 0.f : a.w;
  } else {
    if (K == kEntropy) a.w = f * fmaf(a.s, shift, a.w);
    if (K == kSplit) a.w *= f;
    a.s *= f;
  }
  a.m = m;
}

// One maximum for the warp first, so that every lane moves its sums once.
template <Kind K>
__device__ __forceinline__ Stats warp_merge(Stats a, float c) {
  rebase<K>(a, warp_max(a.m), c);
  a.s = warp_sum(a.s);
  if (K != kSum) a.w = warp_sum(a.w);
  return a;
}

// ---------------------------------------------------------------------------------------------
// A row's distillation loss, by one warp
// ---------------------------------------------------------------------------------------------
// A lane's share of the teacher's list: entries lane, lane + 32, ...
constexpr int kEntriesPerLane = kMaxAlternatives / 32;

// Does the list teach anything? (the whole warp asks) An empty one, or without the tail one whose
// entries all have probability 0, leaves the row out.
__device__ __forceinline__ bool list_counts(const DistillationArgs& p, int64_t row) {
  bool counts = false;
  for (int k = threadIdx.x & 31; k < p.top; k += 32)
    counts |= p.tokens[row * p.top + k] >= 0 && (p.tail || p.teacher[row * p.top + k] != -INFINITY);
  return __any_sync(0xffffffffu, counts);
}
__device__ __forceinline__ void skip_row(const DistillationArgs& p, int64_t row) {
  p.loss[row] = 0.f;
  p.stats[row] = make_float4(0.f, INFINITY, 0.f, 0.f);
}

// `value`: log-probabilities (-inf where there is no entry), `picked`: the entries' logits (NaN for a
// token outside the vocabulary), `total` / `outside`: sums of e over all / the unlisted tokens.
template <bool TAIL>
__device__ __forceinline__ void finish_distillation(const DistillationArgs& p, int64_t row,
                                                    const float (&value)[kEntriesPerLane],
                                                    const float (&picked)[kEntriesPerLane], float ref,
                                                    float total, float outside) {
  const float log_s = logf(total);
  float list_log = 0.f;  // log-sum of the list, which renormalises it
  if (!TAIL) {
    float high = -INFINITY;
#pragma unroll
    for (int i = 0; i < kEntriesPerLane; ++i) high = fmaxf(high, value[i]);
    high = warp_max(high);
    float mass = 0.f;
#pragma unroll
    for (int i = 0; i < kEntriesPerLane; ++i) mass += expf(value[i] - high);
    list_log = high + logf(warp_sum(mass));
  }
  float loss = 0.f, mass = 0.f;
#pragma unroll
  for (int i = 0; i < kEntriesPerLane; ++i) {
    const float log_p = value[i] - list_log;
    const float weight = expf(log_p);
    mass += weight;
    if (weight != 0.f) loss += weight * (log_p - fmaf(picked[i] - ref, p.inv_temperature, -log_s));
  }
  loss = warp_sum(loss);
  mass = warp_sum(mass);
  if (TAIL) {
    const float rest = 1.f - mass;
    if (!(rest <= kLeastRest)) loss += rest * (logf(rest) - (logf(outside) - log_s));
  }
  if ((threadIdx.x & 31) == 0) {
    p.loss[row] = loss;
    // a NaN loss has a NaN gradient, also where it comes from a token outside the vocabulary
    p.stats[row] = make_float4(ref, loss == loss ? total : loss, TAIL ? mass : list_log, outside);
  }
}

// ---------------------------------------------------------------------------------------------
// A row's gradient
// ---------------------------------------------------------------------------------------------
// Both operators' gradients are  e (slope t + level)  with t = (x - ref) c and e = 2^t for the tokens
// that no entry names, and  e (slope t + level_named) + the entries' weights  for the others.
struct GradRow {
  bool zero;  // nothing was asked for, whatever the logits hold
  float ref, slope, level, level_named;
};

// `g_top`: sum of the top list's incoming gradients, `any_top`: one of them is not 0.
template <bool DISTILL>
__device__ __forceinline__ GradRow grad_row(const VocabGradArgs& p, int64_t row, float g_top, bool any_top) {
  const float4 st = p.stats[row];
  GradRow r{st.y == INFINITY, st.x, 0.f, 0.f, 0.f};  // the forward pass skipped the row
  if (r.zero) return r;
  const float total = st.y;
  if (DISTILL) {
    const float g = p.grad[row] * p.inv_temperature;
    r.zero = g == 0.f;
    float mass = 1.f, rest = 0.f;
    if (p.tail) {
      rest = 1.f - st.z <= kLeastRest ? 0.f : 1.f - st.z;
      mass = st.z + rest;
    }
    r.level_named = g * mass / total;
    // without outside mass every unnamed token has e = 0
    r.level = (rest > 0.f && st.w > 0.f) ? g * (mass / total - rest / st.w) : r.level_named;
  } else {
    float g = p.grad != nullptr ? p.grad[row] : 0.f;
    if (g != 0.f) {
      const int64_t token = p.tokens[row];
      if (token < 0 || token >= p.vocab) g = quiet_nan();
    }
    const float gh = p.grad_entropy != nullptr ? p.grad_entropy[row] : 0.f;
    r.zero = g == 0.f && gh == 0.f && !any_top;
    const float inv = p.inv_temperature / total;
    r.level = r.level_named = -inv * (g + g_top + gh * (st.z - logf(total)));
    r.slope = -inv * gh * kLn2;
  }
  if (r.zero) r.slope = r.level = r.level_named = 0.f;
  return r;
}

// What entry k (the target; an entry of the teacher's list) adds to its token.
template <bool DISTILL>
__device__ __forceinline__ float entry_weight(const VocabGradArgs& p, int64_t row, int k) {
  const float g = p.grad != nullptr ? p.grad[row] * p.inv_temperature : 0.f;
  if (!DISTILL) return g;
  const float value = p.teacher[row * p.top + k];
  return -g * expf(p.tail ? value : value - p.stats[row].z);
}

// e is 0 from t = -150 down; the clamp keeps `slope t` finite there (masked logits: t = -inf).
__device__ __forceinline__ float grad_exponent(float x, float ref, float c) {
  return fmaxf((x - ref) * c, -1.0e4f);
}

}  // namespace vocab
}  // namespace ob
