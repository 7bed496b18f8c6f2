// The running statistics behind log probabilities and entropies (token_logprobs.cu states the formulas): a part's largest entry m, L = sum
// exp(x - m) and T = sum exp(x - m) (x - m), and how two parts meet.
#pragma once

#include "common.cuh"

struct Stats { float m, l, t; };

__device__ __forceinline__ float lp_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lp_exp(float d) { return lp_exp2(d * 1.4426950408889634f); }
// Both parts on the larger reference.  (A part that has seen no finite entry has m = -inf, L = T = 0.)
__device__ __forceinline__ Stats lp_join(const Stats& a, const Stats& b) {
  const float m = fmaxf(a.m, b.m), base = m == -INFINITY ? 0.f : m;
  const float da = fmaxf(a.m - base, -1e30f), db = fmaxf(b.m - base, -1e30f);
  const float wa = lp_exp(da), wb = lp_exp(db);
  // (a weight of zero meets a distance of 1e30 here: L is then 0 or its part is)
  return Stats{m, fmaf(a.l, wa, b.l * wb), wa * fmaf(a.l, wa > 0.f ? da : 0.f, a.t) + wb * fmaf(b.l, wb > 0.f ? db : 0.f, b.t)};
}
